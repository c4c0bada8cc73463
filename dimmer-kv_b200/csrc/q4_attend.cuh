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

// a / b: lines shorter than 2^32 / workers, all but the largest, do with 32 bits; the others' division is kept out of line
// (CALL), for kernels of a few microseconds wait for their code, but for the kernel that deals out registers: a call in it
// would hold every role to the registers of the launch (q4_prefill_kernel: 74 us without, 81 with).
static __device__ __noinline__ int64_t divide64(int64_t a, int64_t b) { return a / b; }
template <bool CALL>
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (a <= 0xffffffffll && b <= 0xffffffffll) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return CALL ? divide64(a, b) : a / b;
}

// How a line of `total` places is dealt to the workers: worker w has [total * w / workers, total * (w + 1) / workers).
template <bool CALL>
struct DealOf {
  int64_t total;
  int workers;
  __device__ __forceinline__ DealOf(int64_t total_, int workers_)
      : total(total_), workers(static_cast<int>(total_ < workers_ ? total_ : workers_)) {}
  __device__ __forceinline__ int64_t begin(int w) const { return divide<CALL>(total * w, workers); }
};
using Deal = DealOf<true>;

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

// Behind the slots, per unit: the slot of its first piece, written by the worker that has it, and the worker of its last.
__device__ __forceinline__ int2* unit_record(const dkv_q4_attend_args& a, int workers, int rows, int64_t unit) {
  return reinterpret_cast<int2*>(a.workspace + 2 * static_cast<int64_t>(workers) * slot_floats(rows, a.head_dim)) + unit;
}
__device__ __forceinline__ void record_unit(int2* by, int worker, bool second_slot, bool begins, bool ends) {
  if (begins) by->x = 2 * worker + second_slot;
  if (ends) by->y = worker;
}

// The partial results of one unit: worker w0 + k left the unit's piece in slot(k). The unit is the last segment of w0 unless
// w0 begins with it (its second slot), and the first segment of the others.
struct Pieces {
  const float *first, *rest;
  int64_t stride;
  int n;
  Pieces() = default;
  __device__ __forceinline__ Pieces(const dkv_q4_attend_args& a, int2 by, int workers, int rows, int d) {
    stride = slot_floats(rows, d);
    first = a.workspace + by.x * stride;
    rest = a.workspace + (by.x & ~1) * stride;
    n = by.x >= 0 && by.y < workers ? max(0, by.y - (by.x >> 1) + 1) : 0;  // (unwritten records only after an error)
  }
  __device__ __forceinline__ const float* slot(int k) const { return k == 0 ? first : rest + 2 * k * stride; }
};

template <int N>
__device__ __forceinline__ void load_row(const float* at, float (&x)[N]) {
  if constexpr (N == 4) {
    const float4 u = *reinterpret_cast<const float4*>(at);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
  } else {
    const float2 u = *reinterpret_cast<const float2*>(at);
    x[0] = u.x, x[1] = u.y;
  }
}

// Joins the pieces of row `row` of a unit: a warp, D / 32 dimensions per lane. References are where the sums' factor is
// 2^-reference (SIGN = 1: q4_prefill's maxima) or 2^reference (-1: q4_decode's negated ones).
template <int D, int SIGN, int UNROLL, int AHEAD>
__device__ __forceinline__ void join_row(const Pieces& p, int rows, int row, float (&sum)[D / 32]) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum[e] = 0.f;
  float den = 0.f, ref = -INFINITY;
  for (int base = 0; base < p.n; base += 32) {
    // the factors of 32 pieces, one per lane, then their sums with no load waiting for another; the loads of the first
    // AHEAD pieces are under way with the factors'
    const int n = min(32, p.n - base);
    float ahead[AHEAD > 0 ? AHEAD : 1][kPer];
#pragma unroll
    for (int w = 0; w < AHEAD; ++w) load_row<kPer>(p.slot(base + min(w, n - 1)) + row * D + lane * kPer, ahead[w]);
    const float2 s = lane < n ? *reinterpret_cast<const float2*>(p.slot(base + lane) + rows * D + row * 4) : make_float2(0.f, 0.f);
    const float mine = s.y == 0.f ? -INFINITY : SIGN * s.x;  // a piece that saw no token of this row has no say
    float now = fmaxf(ref, mine);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d));
    const float f = mine == -INFINITY ? 0.f : exp2_fast(mine - now);
    float add = s.y * f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
    const float keep = ref == -INFINITY ? 0.f : exp2_fast(ref - now);
    den = fmaf(den, keep, add);
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum[e] *= keep;
    ref = now;
#pragma unroll
    for (int w = 0; w < AHEAD; ++w) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] = w < n ? fmaf(ahead[w][e], fw, sum[e]) : sum[e];
    }
#pragma unroll UNROLL
    for (int w = AHEAD; w < n; ++w) {
      float o[kPer];
      load_row<kPer>(p.slot(base + w) + row * D + lane * kPer, o);
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int e = 0; e < kPer; ++e) sum[e] = fmaf(o[e], fw, sum[e]);
    }
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum[e] *= inv;
}

// A lane's D / 32 dimensions of an output row that begins at `at`.
template <int D, bool F16>
__device__ __forceinline__ void store_row(const dkv_q4_attend_args& a, int64_t at, const float (&v)[D / 32]) {
  at += (threadIdx.x & 31) * (D / 32);
  if constexpr (D == 128) {
    store_out4<F16>(a, at, v[0], v[1], v[2], v[3]);
  } else if (a.out_f32) {
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(v[0], v[1]);
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at) =
        static_cast<uint32_t>(to16<F16>(v[0])) | static_cast<uint32_t>(to16<F16>(v[1])) << 16;
  }
}

// Query rows of a KV head (all new tokens' rows of its query heads).
inline int rows_of(const dkv_q4_attend_args& a) { return a.q_len * (a.n_q_heads / a.n_kv_heads); }

// q4_prefill.cu
bool prefill_takes(const dkv_q4_attend_args& a);
int64_t prefill_floats(const dkv_q4_attend_args& a);
int run_prefill(const dkv_q4_attend_args& a, bool appended, cudaStream_t stream);

}  // namespace q4
}  // namespace dkv
