// q4_rows.cu — keys and values into the cells of the paged 4-bit cache, and back (dkv_q4_append, dkv_q4_read).
//
// A lane takes 16 dimensions of a token's key and value, or 32 to store many (q4_cells.cuh quantises). 2 bytes are read
// and 0.56 written per element, and the reverse. Storing is bound by its instructions: what a lane does once for its part
// of a group (its place, the group's scale) it then does for twice as much.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_launch.h"
#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace {

using q4::Cells;
constexpr int kRowThreads = 256;
constexpr int kReadDims = 16;  // of a lane

// A lane's place: the j-th D / kLanes dimensions of token i of a conversation's KV head. Rows run over tokens fastest, so a
// warp holds neighbouring tokens of one head: whole lines of the key cells, and both tokens of a value pair.
struct Place {
  int seq, head, i, j, slot;  // slot -1: no token
};

template <int kLanes>
__device__ __forceinline__ Place place_of(const dkv_q4_rows_args& a) {
  const uint32_t row = (blockIdx.x * kRowThreads + threadIdx.x) / kLanes;
  const uint32_t q_len = a.q_len, heads = a.n_kv_heads;
  const uint32_t line = row / q_len;
  Place p;
  p.j = threadIdx.x % kLanes;
  p.i = static_cast<int>(row - line * q_len);
  p.seq = static_cast<int>(line / heads);
  p.head = static_cast<int>(line - p.seq * heads);
  p.slot = p.seq < a.n_seq ? a.slots[static_cast<int64_t>(p.seq) * a.q_len + p.i] : -1;
  if (p.slot >= a.n_pages * q4::kPage) {
    record_error(a.status, kSiteQ4Rows + kErrBadDescriptor);
    p.slot = -1;
  }
  return p;
}

template <int D, int DIMS, bool F16>
__global__ void __launch_bounds__(kRowThreads) q4_append_kernel(const __grid_constant__ dkv_q4_rows_args a) {
  using C = Cells<D>;
  constexpr int H = DIMS / 8, kLanes = D / DIMS;  // DIMS: of a lane
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // an attention that reads these cells begins to set up
  const Place p = place_of<kLanes>(a);
  uint4 key[H], value[H];
#pragma unroll
  for (int h = 0; h < H; ++h) key[h] = value[h] = make_uint4(0u, 0u, 0u, 0u);
  if (p.slot >= 0) {
    const uint4* ks = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.key) + p.seq * a.k_stride[0] +
                                                     p.head * a.k_stride[1] + p.i * a.k_stride[2] + p.j * DIMS);
    const uint4* vs = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.value) + p.seq * a.v_stride[0] +
                                                     p.head * a.v_stride[1] + p.i * a.v_stride[2] + p.j * DIMS);
#pragma unroll
    for (int h = 0; h < H; ++h) key[h] = ks[h], value[h] = vs[h];
  }
  // one answer for the warp's shuffles: nothing to do for it, or nothing to be done
  if (__all_sync(0xffffffffu, p.slot < 0) || __any_sync(0xffffffffu, status_at_entry(a.status) != 0)) return;
  const q4::CellPart<H> k = q4::quantise<F16>(key), v = q4::quantise<F16>(value);
  if (!k.fits || !v.fits) record_error(a.status, kSiteQ4Rows + kErrCellRange);
  // the other token of the pair, where the lanes beside hold it: its codes of the half of the eights that this lane writes
  const int there = __shfl_xor_sync(0xffffffffu, p.slot, kLanes);
  const int beside = __shfl_xor_sync(0xffffffffu, p.i, kLanes);
  const bool first = (threadIdx.x & kLanes) == 0;
  uint32_t other[H / 2];
#pragma unroll
  for (int h = 0; h < H / 2; ++h) other[h] = __shfl_xor_sync(0xffffffffu, first ? v.codes[H / 2 + h] : v.codes[h], kLanes);
  if (p.slot < 0) return;
  uint8_t* page = a.cells + (static_cast<int64_t>(p.slot / q4::kPage) * a.n_kv_heads + p.head) * C::kBytes;
  const int r = p.slot % q4::kPage;
  q4::store_key<D>(page, r, p.j, k);
  const int step = first ? 1 : -1;
  if (there >= 0 && there == p.slot + step && beside == p.i + step && (r & 1) == (first ? 0 : 1)) {
    // the even token's lane writes the first half of the eights of both, the odd one's the second
#pragma unroll
    for (int h = 0; h < H / 2; ++h) {
      const uint32_t even = first ? v.codes[h] : other[h], odd = first ? other[h] : v.codes[H / 2 + h];
      *reinterpret_cast<uint2*>(page + C::value_words(r >> 1, H * p.j + (first ? 0 : H / 2) + h)) =
          make_uint2(__byte_perm(even, odd, 0x5410), __byte_perm(even, odd, 0x7632));
    }
    q4::store_value_head<D>(page, r, p.j, v);
  } else {
    q4::store_value<D>(page, r, p.j, v);
  }
}

// 8 codes to the 16-bit values that they stand for.
template <bool F16>
__device__ __forceinline__ uint4 values_of(uint32_t codes, uint32_t scale_low) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&scale_low));
  uint32_t out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // code * scale is exact in float32 (4 and 11 bits): one rounding to float32, one to 16 bits
    const float c0 = __uint_as_float(0x4b000000u | ((codes >> (8 * e)) & 15u)) - 8388608.f;
    const float c1 = __uint_as_float(0x4b000000u | ((codes >> (8 * e + 4)) & 15u)) - 8388608.f;
    const float x = __fmaf_rn(c0, f.x, f.y), y = __fmaf_rn(c1, f.x, f.y);
    if constexpr (F16) {
      const __half2 h = __floats2half2_rn(x, y);
      out[e] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      out[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kRowThreads) q4_read_kernel(const __grid_constant__ dkv_q4_rows_args a) {
  using C = Cells<D>;
  const Place p = place_of<D / kReadDims>(a);
  if (p.seq >= a.n_seq) return;
  uint4 key[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)}, value[2] = {key[0], key[0]};
  if (p.slot >= 0 && status_at_entry(a.status) == 0) {
    const uint8_t* page = a.cells + (static_cast<int64_t>(p.slot / q4::kPage) * a.n_kv_heads + p.head) * C::kBytes;
    const int r = p.slot % q4::kPage;
    const uint2 codes = *reinterpret_cast<const uint2*>(page + C::key_word(r, 2 * p.j));
    const uint32_t key_head = *reinterpret_cast<const uint32_t*>(page + C::key_head(r, p.j / 4));
    const uint32_t value_head = *reinterpret_cast<const uint32_t*>(page + C::value_head(r, p.j / 4));
    const uint32_t half = r & 1 ? 0x7632 : 0x5410;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint2 w = *reinterpret_cast<const uint2*>(page + C::value_words(r >> 1, 2 * p.j + h));
      value[h] = values_of<F16>(__byte_perm(w.x, w.y, half), value_head);
    }
    key[0] = values_of<F16>(codes.x, key_head);
    key[1] = values_of<F16>(codes.y, key_head);
  }
  uint4* ks = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.key) + p.seq * a.k_stride[0] + p.head * a.k_stride[1] +
                                       p.i * a.k_stride[2] + p.j * 16);
  uint4* vs = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.value) + p.seq * a.v_stride[0] + p.head * a.v_stride[1] +
                                       p.i * a.v_stride[2] + p.j * 16);
  ks[0] = key[0], ks[1] = key[1], vs[0] = value[0], vs[1] = value[1];
}

int check_rows(const dkv_q4_rows_args* a) {
  if (a == nullptr || a->cells == nullptr || a->status == nullptr || a->n_pages < 1 || a->n_kv_heads < 1 ||
      a->n_seq < 0 || a->q_len < 0)
    return DKV_ERR_ARGS;
  if (a->head_dim != 64 && a->head_dim != 128) return DKV_ERR_CONFIG;
  if (static_cast<int64_t>(a->n_pages) * q4::kPage > INT32_MAX) return DKV_ERR_CONFIG;
  if (a->n_seq == 0 || a->q_len == 0) return DKV_OK;  // tensors without an element have no address
  if (a->slots == nullptr || a->key == nullptr || a->value == nullptr) return DKV_ERR_ARGS;
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
  const int64_t dims = static_cast<int64_t>(a->n_seq) * a->q_len * a->n_kv_heads * a->head_dim;
  if (dims == 0) return DKV_OK;
  if (dims / 16 > INT32_MAX) return DKV_ERR_CONFIG;
  // 16 dimensions per lane while the lanes fit the GPU at once (16 tokens of 8 heads of 64: 7.1 us with the read, 8.2 with
  // 32), 32 where there are more (16 prompts of up to 4095 tokens of 8 heads of 128: 82 us, 93 with 16).
  const bool few = dims / 16 <= dkv::device_sms() * 2048;
  const int64_t lanes = dims / (few ? 16 : 32);
  const dim3 grid(static_cast<unsigned>((lanes + dkv::kRowThreads - 1) / dkv::kRowThreads));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define DKV_Q4_APPEND(D, DIMS) (a->fp16 ? dkv::q4_append_kernel<D, DIMS, true> : dkv::q4_append_kernel<D, DIMS, false>)
  auto kernel = a->head_dim == 128 ? (few ? DKV_Q4_APPEND(128, 16) : DKV_Q4_APPEND(128, 32))
                                   : (few ? DKV_Q4_APPEND(64, 16) : DKV_Q4_APPEND(64, 32));
#undef DKV_Q4_APPEND
  kernel<<<grid, dkv::kRowThreads, 0, st>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

int dkv_q4_read(const dkv_q4_rows_args* a, void* stream) {
  const int rc = dkv::check_rows(a);
  if (rc != DKV_OK) return rc;
  const int64_t lanes = static_cast<int64_t>(a->n_seq) * a->q_len * a->n_kv_heads * (a->head_dim / dkv::kReadDims);
  if (lanes == 0) return DKV_OK;
  const int64_t blocks = (lanes + dkv::kRowThreads - 1) / dkv::kRowThreads;
  if (lanes > INT32_MAX) return DKV_ERR_CONFIG;
  const dim3 grid(static_cast<unsigned>(blocks));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kernel = a->head_dim == 128 ? (a->fp16 ? dkv::q4_read_kernel<128, true> : dkv::q4_read_kernel<128, false>)
                                   : (a->fp16 ? dkv::q4_read_kernel<64, true> : dkv::q4_read_kernel<64, false>);
  kernel<<<grid, dkv::kRowThreads, 0, st>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

}  // extern "C"
