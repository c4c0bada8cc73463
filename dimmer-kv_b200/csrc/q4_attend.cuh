// q4_attend.cuh — what the kernels of dkv_q4_attend share.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dkv_launch.h"
#include "dkv_ptx.cuh"
#include "q4_cells.cuh"

namespace dkv {
namespace q4 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBias = 7.f;    // probabilities are scaled by 2^7
constexpr float kSlack = 8.f;   // the reference maximum may lag by 2^8: 2^(7 + 8) < 65504

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }

// Tokens that conversation s attends over (0 if it has no new token).
__device__ __forceinline__ int tokens_of(const dkv_q4_attend_args& a, int s) {
  const int start = a.starts[s], len = min(a.lengths[s], a.max_blocks * kPage);
  return start >= 0 && len > start ? len : 0;
}
__device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// How a line of `total` places is dealt to the workers: worker w has [total * w / workers, total * (w + 1) / workers).
struct Deal {
  int64_t total;
  int workers;
  __device__ __forceinline__ Deal(int64_t total_, int workers_)
      : total(total_), workers(static_cast<int>(total_ < workers_ ? total_ : workers_)) {}
  __device__ __forceinline__ int64_t begin(int w) const {
    const int64_t x = total * w;
    return x <= 0xffffffffll ? static_cast<uint32_t>(x) / static_cast<uint32_t>(workers) : x / workers;
  }
  // The worker that has place x; none is without a place.
  __device__ __forceinline__ int owner(int64_t x) const {
    const int64_t y = (x + 1) * workers - 1;
    return static_cast<int>(y <= 0xffffffffll ? static_cast<uint32_t>(y) / static_cast<uint32_t>(total) : y / total);
  }
};

template <bool F16>
__device__ __forceinline__ void store_out4(const dkv_q4_attend_args& a, int64_t at, float x, float y, float z, float w) {
  if (a.out_f32)
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x, y, z, w);
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(static_cast<uint32_t>(to16<F16>(x)) | static_cast<uint32_t>(to16<F16>(y)) << 16,
                   static_cast<uint32_t>(to16<F16>(z)) | static_cast<uint32_t>(to16<F16>(w)) << 16);
}

// A partial result in the workspace: per slot (two per worker) [rows][D] of O, then [rows][4] with (reference, l).
__host__ __device__ __forceinline__ int64_t slot_floats(int rows, int d) { return static_cast<int64_t>(rows) * (d + 4); }

// Query rows of a KV head (all new tokens' rows of its query heads).
inline int rows_of(const dkv_q4_attend_args& a) { return a.q_len * (a.n_q_heads / a.n_kv_heads); }

// q4_prefill.cu
bool prefill_takes(const dkv_q4_attend_args& a);
int64_t prefill_floats(const dkv_q4_attend_args& a);
int run_prefill(const dkv_q4_attend_args& a, cudaStream_t stream);

}  // namespace q4
}  // namespace dkv
