// logits.cu — the choice of the next token (dkv_logit_rules): penalties for repeated tokens, biases and a grammar
// mask on a row of logits, and its largest entry.
//
// Eight CTAs of a cluster share a row, each a slice of the vocabulary. A CTA counts the history's tokens of its
// slice in shared memory (one word per token: bit 31 = seen in the prompt, the low bits = times generated; integer
// atomics, so the order does not matter), then passes over the slice's logits once: read, adjust, write, and keep
// the largest as a 64-bit key (the float's order above, the inverted token below, so that equal values give the
// lowest token). The slices' keys meet in distributed shared memory: one launch, no workspace in memory. Every
// step is a single float32 operation with the rounding that the header's formulas state (no contraction), so that
// the choice between near-equal tokens does not depend on the compiler. Bound by the logits' bytes.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dimmer_kv.h"
#include "dkv_ptx.cuh"

namespace dkv {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kRuleSplits = 8;       // CTAs of a row
constexpr int kSlice = 16384;        // tokens that a CTA counts at a time
constexpr int kMaxBias = 1024;

__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
  if (x == -INFINITY) return 0ull;
  uint32_t b = __float_as_uint(x);
  b = x != x ? 0xffffffffu : (x == 0.f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u));
  return static_cast<uint64_t>(b) << 32 | (0xffffffffu - token);
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if constexpr (DT == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if constexpr (DT == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

// Four logits from an address that is a multiple of four elements.
template <int DT>
__device__ __forceinline__ void logits4(const void* p, int64_t i, float (&x)[4]) {
  if constexpr (DT == 2) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[2] = {v.x, v.y};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t h = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
      x[e] = DT == 0 ? __bfloat162float(__ushort_as_bfloat16(h)) : __half2float(__ushort_as_half(h));
    }
  }
}

struct RowRules {
  float repetition, frequency, presence;
};

__device__ __forceinline__ float adjust(float x, uint32_t word, float bias, bool biased, bool allowed, const RowRules& r) {
  if (word != 0) {
    x = x > 0.f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    const uint32_t made = word & 0x7fffffffu;
    if (made != 0) {
      x = __fsub_rn(x, __fmul_rn(r.frequency, static_cast<float>(made)));
      x = __fsub_rn(x, r.presence);
    }
  }
  if (biased) x = __fadd_rn(x, bias);
  return allowed ? x : -INFINITY;
}

template <int DT>
__global__ void __cluster_dims__(kRuleSplits, 1, 1) __launch_bounds__(kRuleThreads)
logit_rules_kernel(const dkv_logits_args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t keys[kRuleThreads / 32];
  __shared__ uint64_t slice_key;
  uint32_t* count = reinterpret_cast<uint32_t*>(smem);
  float* bias = reinterpret_cast<float*>(smem + kSlice * 4);  // only with biases
  const int row = blockIdx.x / kRuleSplits, rank = blockIdx.x % kRuleSplits;
  const int tid = threadIdx.x;
  const bool failed = cta_failed_at_entry(a.status);
  const int length = failed ? 0 : max(0, min(a.lengths[row], a.capacity));
  const int prompt = a.prompts[row];
  const int32_t* hist = a.history + static_cast<int64_t>(row) * a.capacity;
  const RowRules rules = {a.repetition[row], a.frequency[row], a.presence[row]};
  const uint32_t* allowed = a.allowed ? a.allowed + static_cast<int64_t>(row) * ((a.vocab + 31) / 32) : nullptr;
  const int esize = DT == 2 ? 4 : 2;
  const uint8_t* in = static_cast<const uint8_t*>(a.logits) + row * a.row_stride * esize;
  float* out = a.adjusted ? a.adjusted + static_cast<int64_t>(row) * a.vocab : nullptr;
  // Four tokens at a time where the row starts on their boundary.
  const bool wide = reinterpret_cast<uintptr_t>(in) % (4 * esize) == 0 &&
                    (out == nullptr || reinterpret_cast<uintptr_t>(out) % 16 == 0);
  const int per = ((a.vocab + kRuleSplits - 1) / kRuleSplits + 31) / 32 * 32;  // tokens of a CTA
  const int end = min(a.vocab, (rank + 1) * per);
  uint64_t best = 0;
  for (int lo = rank * per; lo < end && !failed; lo += kSlice) {
    const int n = min(kSlice, end - lo);
    __syncthreads();
    for (int i = tid; i < (n + 3) / 4; i += kRuleThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (a.n_bias)
      for (int i = tid; i < (n + 3) / 4; i += kRuleThreads)
        reinterpret_cast<float4*>(bias)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    for (int i = tid; i < length; i += kRuleThreads) {
      const uint32_t at = static_cast<uint32_t>(hist[i]) - static_cast<uint32_t>(lo);
      if (at < static_cast<uint32_t>(n)) {
        if (i < prompt) atomicOr(&count[at], 0x80000000u);
        else atomicAdd(&count[at], 1u);
      }
    }
    if (a.n_bias) {
      const int32_t* ids = a.bias_ids + static_cast<int64_t>(row) * a.n_bias;
      const float* vals = a.bias_values + static_cast<int64_t>(row) * a.n_bias;
      for (int i = tid; i < a.n_bias; i += kRuleThreads) {
        const int id = ids[i];
        const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(lo);
        if (at >= static_cast<uint32_t>(n)) continue;
        // the first entry of a token adds up all of them, in their order
        bool first = true;
        for (int k = 0; k < i && first; ++k) first = ids[k] != id;
        if (!first) continue;
        float sum = vals[i];
        for (int k = i + 1; k < a.n_bias; ++k)
          if (ids[k] == id) sum = __fadd_rn(sum, vals[k]);
        bias[at] = sum;
      }
    }
    __syncthreads();
    const int n4 = wide ? n / 4 : 0;
    for (int q = tid; q < n4; q += kRuleThreads) {
      const int token = lo + q * 4;
      float x[4];
      logits4<DT>(in, token, x);
      const uint4 w = reinterpret_cast<const uint4*>(count)[q];
      const float4 b = a.n_bias ? reinterpret_cast<const float4*>(bias)[q] : make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t ok = allowed ? allowed[token >> 5] >> (token & 31) : 0xfu;
      x[0] = adjust(x[0], w.x, b.x, b.x != 0.f, ok & 1u, rules);
      x[1] = adjust(x[1], w.y, b.y, b.y != 0.f, ok & 2u, rules);
      x[2] = adjust(x[2], w.z, b.z, b.z != 0.f, ok & 4u, rules);
      x[3] = adjust(x[3], w.w, b.w, b.w != 0.f, ok & 8u, rules);
      if (out) *reinterpret_cast<float4*>(out + token) = make_float4(x[0], x[1], x[2], x[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t key = order_key(x[e], token + e);
        best = key > best ? key : best;
      }
    }
    for (int i = n4 * 4 + tid; i < n; i += kRuleThreads) {
      const int token = lo + i;
      const float b = a.n_bias ? bias[i] : 0.f;
      const bool ok = allowed == nullptr || (allowed[token >> 5] >> (token & 31)) & 1u;
      const float x = adjust(logit_at<DT>(in, token), count[i], b, b != 0.f, ok, rules);
      if (out) out[token] = x;
      const uint64_t key = order_key(x, token);
      best = key > best ? key : best;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, best, d);
    best = other > best ? other : best;
  }
  if ((tid & 31) == 0) keys[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kRuleThreads / 32; ++w) best = keys[w] > best ? keys[w] : best;
    slice_key = best;
  }
  __syncthreads();
  cluster_sync_all();  // every CTA's key is there, and every CTA has read the history
  if (rank == 0 && tid < 32) {
    uint64_t key = 0;
    if (tid < kRuleSplits) {
      const uint32_t addr = mapa_shared(smem_u32(&slice_key), tid);
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(addr) : "memory");
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, d);
      key = other > key ? other : key;
    }
    if (tid == 0) {
      const int64_t token = key == 0 ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
      a.tokens[row] = token;
      if (a.append && token >= 0 && !failed) {
        const int at = a.lengths[row];
        if (at >= 0 && at < a.capacity) {
          a.history[static_cast<int64_t>(row) * a.capacity + at] = static_cast<int32_t>(token);
          a.lengths[row] = at + 1;
        } else {
          record_error(a.status, kErrHistory);
        }
      }
    }
  }
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its key is read
}

}  // namespace
}  // namespace dkv

extern "C" int dkv_logit_rules(const dkv_logits_args* a, void* stream) {
  if (a == nullptr || a->logits == nullptr || a->history == nullptr || a->lengths == nullptr || a->prompts == nullptr ||
      a->repetition == nullptr || a->frequency == nullptr || a->presence == nullptr || a->tokens == nullptr ||
      a->status == nullptr)
    return DKV_ERR_ARGS;
  if (a->n_rows < 0 || a->vocab < 1 || a->capacity < 1 || a->n_bias < 0 || a->row_stride < 0 || a->dtype < 0 ||
      a->dtype > 2 || (a->n_bias > 0 && (a->bias_ids == nullptr || a->bias_values == nullptr)))
    return DKV_ERR_ARGS;
  if (a->n_bias > dkv::kMaxBias || a->vocab > (1 << 30) || a->n_rows > (INT32_MAX / dkv::kRuleSplits))
    return DKV_ERR_CONFIG;
  if (a->n_rows == 0) return DKV_OK;
  auto kernel = a->dtype == 0 ? dkv::logit_rules_kernel<0> : a->dtype == 1 ? dkv::logit_rules_kernel<1> : dkv::logit_rules_kernel<2>;
  const int bytes = dkv::kSlice * (a->n_bias ? 8 : 4);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dkv::kSlice * 8) != cudaSuccess)
    return DKV_ERR_CUDA;
  kernel<<<a->n_rows * dkv::kRuleSplits, dkv::kRuleThreads, bytes, static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}
