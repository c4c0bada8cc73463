// q4_rows.cu — keys and values into the cells of the paged 4-bit cache, and back (dkv_q4_append, dkv_q4_read).
//
// Eight lanes hold a group of 64 dimensions, eight dimensions each (one 16-byte load): the group's minimum and
// maximum are three shuffles, and a lane's eight key codes are exactly one word of the key cell, its value codes
// the halves of two words of the pair's. Memory bound: 2 bytes read and 0.56 written per element.
//
// The code is the nearest whole number to the true quotient (x - low) / scale, not to its float32 rounding: the
// float32 quotient, off by less than 2^-18, decides unless it lies within 2^-16 of a half; then the border
// low + (c + 1/2) * scale, which float64 holds exactly (two float16 numbers, exponents -25 .. 15, and 5 bits),
// is compared with x. So the codes do not depend on how a device rounds a division.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace {

using q4::Cells;
constexpr int kRowThreads = 256;

template <bool F16>
__device__ __forceinline__ float from16(uint16_t v) {
  return F16 ? __half2float(__ushort_as_half(v)) : __bfloat162float(__ushort_as_bfloat16(v));
}
template <bool F16>
__device__ __forceinline__ uint16_t to16(float v) {
  return F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Nearest whole number of 0..15 to (x - low) / scale, ties to even; inv = 1 / scale to float32 accuracy.
__device__ __forceinline__ uint32_t code_of(float x, float low, float scale, float inv) {
  const float q = __fmul_rn(__fsub_rn(x, low), inv);
  float c = rintf(q);
  const float below = floorf(q);
  if (fabsf(q - below - 0.5f) < 0x1p-16f && q > -1.f && q < 16.f) {
    const double border = static_cast<double>(low) + (static_cast<double>(below) + 0.5) * static_cast<double>(scale);
    const double xd = static_cast<double>(x);
    const bool up = xd > border || (xd == border && (static_cast<int>(below) & 1));
    c = up ? below + 1.f : below;
  }
  return static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f));
}

// One lane: 8 dimensions (the j-th eight of its row) of one token's keys (z = 0) or values (z = 1).
template <int D, bool F16>
__global__ void __launch_bounds__(kRowThreads) q4_append_kernel(const dkv_q4_rows_args a) {
  if (status_at_entry(a.status) != 0) return;
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
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = from16<F16>(static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1))));
  float lo = x[0], hi = x[0];
  bool fits = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    fits = fits && fabsf(x[e]) <= q4::kCellMax;  // false for a NaN
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  if (!fits) record_error(a.status, kSiteQ4Rows + kErrCellRange);
  if (slot < 0) return;
  const __half low_h = __float2half_rn(lo);
  const float low = __half2float(low_h);
  const __half scale_h = __float2half_rn(__fdiv_rn(__fsub_rn(hi, low), 15.f));
  const float scale = __half2float(scale_h);
  const float inv = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) codes |= code_of(x[e], low, scale, inv) << (4 * e);
  if (!(scale > 0.f)) codes = 0;
  uint8_t* page = a.cells + (static_cast<int64_t>(slot / q4::kPage) * a.n_kv_heads + head) * C::kBytes;
  const int r = slot % q4::kPage;
  if (!is_value) {
    *reinterpret_cast<uint32_t*>(page + C::key_word(r, j)) = codes;
    if (j % 8 == 0)
      *reinterpret_cast<uint32_t*>(page + C::key_head(r, j / 8)) =
          static_cast<uint32_t>(__half_as_ushort(scale_h)) | static_cast<uint32_t>(__half_as_ushort(low_h)) << 16;
  } else {
    const int pair = r >> 1, odd = r & 1;
    *reinterpret_cast<uint16_t*>(page + C::value_word(pair, 2 * j) + 2 * odd) = static_cast<uint16_t>(codes);
    *reinterpret_cast<uint16_t*>(page + C::value_word(pair, 2 * j + 1) + 2 * odd) = static_cast<uint16_t>(codes >> 16);
    if (j % 8 == 0) {
      uint8_t* h = page + C::value_head(pair, j / 8) + 2 * odd;
      *reinterpret_cast<uint16_t*>(h) = __half_as_ushort(scale_h);
      *reinterpret_cast<uint16_t*>(h + 4) = __half_as_ushort(low_h);
    }
  }
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
      const int pair = r >> 1, odd = r & 1;
      codes = *reinterpret_cast<const uint16_t*>(page + C::value_word(pair, 2 * j) + 2 * odd) |
              static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(page + C::value_word(pair, 2 * j + 1) + 2 * odd))
                  << 16;
      const uint8_t* h = page + C::value_head(pair, j / 8) + 2 * odd;
      scale_low = *reinterpret_cast<const uint16_t*>(h) |
                  static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(h + 4)) << 16;
    }
    const float scale = __half2float(__ushort_as_half(static_cast<uint16_t>(scale_low)));
    const float low = __half2float(__ushort_as_half(static_cast<uint16_t>(scale_low >> 16)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // code * scale is exact in float32 (4 and 11 bits): one rounding to float32, one to 16 bits
      const float v = __fmaf_rn(static_cast<float>((codes >> (4 * e)) & 15u), scale, low);
      out[e >> 1] |= static_cast<uint32_t>(to16<F16>(v)) << (16 * (e & 1));
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
