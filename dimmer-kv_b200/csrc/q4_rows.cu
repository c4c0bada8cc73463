// q4_rows.cu — keys and values into the cells of the paged 4-bit cache, and back (dkv_q4_append, dkv_q4_read).
//
// A lane takes eight dimensions of a token (one 16-byte load or store; q4_cells.cuh quantises). Memory bound: 2
// bytes read and 0.56 written per element, and the reverse.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace {

using q4::Cells;
constexpr int kRowThreads = 256;

// One lane: 8 dimensions (the j-th eight of its row) of one token's keys (z = 0) or values (z = 1).
template <int D, bool F16>
__global__ void __launch_bounds__(kRowThreads) q4_append_kernel(const dkv_q4_rows_args a) {
  if (__any_sync(0xffffffffu, status_at_entry(a.status) != 0)) return;  // one answer for the warp's shuffles
  constexpr int kLanes = D / 8;  // lanes of a row
  using C = Cells<D>;
  const int64_t rows = static_cast<int64_t>(a.n_seq) * a.q_len * a.n_kv_heads;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / kLanes;
  const int j = threadIdx.x % kLanes;
  const bool is_value = blockIdx.y != 0;
  int slot = -1;
  int64_t src = 0;
  int head = 0;
  if (row < rows) {
    const int64_t token = row / a.n_kv_heads;
    head = static_cast<int>(row - token * a.n_kv_heads);
    const int s = static_cast<int>(token / a.q_len), i = static_cast<int>(token - static_cast<int64_t>(s) * a.q_len);
    slot = a.slots[token];
    const int64_t* st = is_value ? a.v_stride : a.k_stride;
    src = s * st[0] + head * st[1] + i * st[2] + j * 8;
    if (slot >= a.n_pages * q4::kPage) {
      record_error(a.status, kSiteQ4Rows + kErrBadDescriptor);
      slot = -1;
    }
  }
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0) raw = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(is_value ? a.value : a.key) + src);
  const q4::Cell8 c = q4::quantise8<F16>(raw);
  if (!c.fits) record_error(a.status, kSiteQ4Rows + kErrCellRange);
  if (slot < 0) return;
  uint8_t* page = a.cells + (static_cast<int64_t>(slot / q4::kPage) * a.n_kv_heads + head) * C::kBytes;
  if (is_value) q4::store_value8<D>(page, slot % q4::kPage, j, c);
  else q4::store_key8<D>(page, slot % q4::kPage, j, c);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kRowThreads) q4_read_kernel(const dkv_q4_rows_args a) {
  constexpr int kLanes = D / 8;
  using C = Cells<D>;
  const bool failed = status_at_entry(a.status) != 0;
  const int64_t rows = static_cast<int64_t>(a.n_seq) * a.q_len * a.n_kv_heads;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / kLanes;
  const int j = threadIdx.x % kLanes;
  const bool is_value = blockIdx.y != 0;
  if (row >= rows) return;
  // heads outermost: neighbouring rows are neighbouring tokens of one head, as key and value are laid out
  const int64_t per_seq = static_cast<int64_t>(a.n_kv_heads) * a.q_len;
  const int s = static_cast<int>(row / per_seq);
  const int head = static_cast<int>((row - s * per_seq) / a.q_len);
  const int i = static_cast<int>(row - s * per_seq - static_cast<int64_t>(head) * a.q_len);
  int slot = a.slots[static_cast<int64_t>(s) * a.q_len + i];
  if (slot >= a.n_pages * q4::kPage) {
    record_error(a.status, kSiteQ4Rows + kErrBadDescriptor);
    slot = -1;
  }
  const int64_t* st = is_value ? a.v_stride : a.k_stride;
  uint16_t* dst = static_cast<uint16_t*>(is_value ? a.value : a.key) + s * st[0] + head * st[1] + i * st[2] + j * 8;
  uint32_t out[4] = {0u, 0u, 0u, 0u};
  if (slot >= 0 && !failed) {
    const uint8_t* page = a.cells + (static_cast<int64_t>(slot / q4::kPage) * a.n_kv_heads + head) * C::kBytes;
    const int r = slot % q4::kPage;
    uint32_t codes, scale_low;
    if (!is_value) {
      codes = *reinterpret_cast<const uint32_t*>(page + C::key_word(r, j));
      scale_low = *reinterpret_cast<const uint32_t*>(page + C::key_head(r, j / 8));
    } else {
      const uint8_t* w = page + C::value_words(r >> 1, j) + 2 * (r & 1);
      codes = *reinterpret_cast<const uint16_t*>(w) |
              static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(w + 4)) << 16;
      scale_low = *reinterpret_cast<const uint32_t*>(page + C::value_head(r, j / 8));
    }
    const float scale = __half2float(__ushort_as_half(static_cast<uint16_t>(scale_low)));
    const float low = __half2float(__ushort_as_half(static_cast<uint16_t>(scale_low >> 16)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // code * scale is exact in float32 (4 and 11 bits): one rounding to float32, one to 16 bits
      const float v = __fmaf_rn(static_cast<float>((codes >> (4 * e)) & 15u), scale, low);
      out[e >> 1] |= static_cast<uint32_t>(q4::to16<F16>(v)) << (16 * (e & 1));
    }
  }
  *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
}

int check_rows(const dkv_q4_rows_args* a) {
  if (a == nullptr || a->cells == nullptr || a->slots == nullptr || a->key == nullptr || a->value == nullptr ||
      a->status == nullptr || a->n_pages < 1 || a->n_kv_heads < 1 || a->n_seq < 0 || a->q_len < 0)
    return DKV_ERR_ARGS;
  if (a->head_dim != 64 && a->head_dim != 128) return DKV_ERR_CONFIG;
  if (static_cast<int64_t>(a->n_pages) * q4::kPage > INT32_MAX) return DKV_ERR_CONFIG;
  if (reinterpret_cast<uintptr_t>(a->cells) % 16 || reinterpret_cast<uintptr_t>(a->key) % 16 ||
      reinterpret_cast<uintptr_t>(a->value) % 16)
    return DKV_ERR_ARGS;
  for (int k = 0; k < 3; ++k)
    if (a->k_stride[k] % 8 || a->v_stride[k] % 8) return DKV_ERR_ARGS;
  return DKV_OK;
}

}  // namespace
}  // namespace dkv

extern "C" {

int64_t dkv_q4_page_bytes(int32_t head_dim) {
  return head_dim == 128 ? dkv::Cells<128>::kBytes : head_dim == 64 ? dkv::Cells<64>::kBytes : -1;
}

int dkv_q4_append(const dkv_q4_rows_args* a, void* stream) {
  const int rc = dkv::check_rows(a);
  if (rc != DKV_OK) return rc;
  const int64_t lanes = static_cast<int64_t>(a->n_seq) * a->q_len * a->n_kv_heads * (a->head_dim / 8);
  if (lanes == 0) return DKV_OK;
  const int64_t blocks = (lanes + dkv::kRowThreads - 1) / dkv::kRowThreads;
  if (blocks > INT32_MAX) return DKV_ERR_CONFIG;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kernel = a->head_dim == 128 ? (a->fp16 ? dkv::q4_append_kernel<128, true> : dkv::q4_append_kernel<128, false>)
                                   : (a->fp16 ? dkv::q4_append_kernel<64, true> : dkv::q4_append_kernel<64, false>);
  kernel<<<grid, dkv::kRowThreads, 0, st>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

int dkv_q4_read(const dkv_q4_rows_args* a, void* stream) {
  const int rc = dkv::check_rows(a);
  if (rc != DKV_OK) return rc;
  const int64_t lanes = static_cast<int64_t>(a->n_seq) * a->q_len * a->n_kv_heads * (a->head_dim / 8);
  if (lanes == 0) return DKV_OK;
  const int64_t blocks = (lanes + dkv::kRowThreads - 1) / dkv::kRowThreads;
  if (blocks > INT32_MAX) return DKV_ERR_CONFIG;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kernel = a->head_dim == 128 ? (a->fp16 ? dkv::q4_read_kernel<128, true> : dkv::q4_read_kernel<128, false>)
                                   : (a->fp16 ? dkv::q4_read_kernel<64, true> : dkv::q4_read_kernel<64, false>);
  kernel<<<grid, dkv::kRowThreads, 0, st>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

}  // extern "C"
