// logits.cu — the choice of the next token (dkv_logit_rules): penalties for repeated tokens, biases and a grammar
// mask on a row of logits, and its largest entry.
//
// The four or eight CTAs of a cluster share a row, each a slice of the vocabulary. The few tokens that a rule touches (those of
// the history, and the biased ones) are separated from the many that none does: a CTA counts its slice's in
// shared memory (a few flag bits and the times generated in one word per token; integer atomics, so their order
// does not matter) and lists each at its first count. Then one pass over the slice, loaded ahead of the counting,
// writes the untouched tokens with the mask alone, and a second, dense one goes over the list. The largest entry
// is a 64-bit key (the float's order above, the inverted token below, so that equal values give the lowest
// token); the slices' keys meet in distributed shared memory: one launch, no workspace in memory. Every step is a
// single float32 operation with the rounding that the header's formulas state (no contraction), so that the choice
// between near-equal tokens does not depend on the compiler. Bound by the logits' bytes.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/dimmer_kv.h"
#include "dkv_launch.h"
#include "dkv_ptx.cuh"
#include "dkv_serving.h"

namespace dkv {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kMaxSplits = 8;        // CTAs of a row
constexpr int kVec = 8;              // tokens that a thread loads at a time
constexpr int kMaxSlice = 32768;     // tokens that a CTA takes at a time, at most
constexpr int kPast = 8;             // tokens of the history that a thread holds
constexpr int kMaxBias = 1024;

// A token's word: seen in the prompt, biased, and the times generated. 16 bits where the history is short enough.
template <typename W>
struct Word {
  static constexpr uint32_t kSeen = 1u << (8 * sizeof(W) - 1), kBiased = kSeen >> 1, kCount = kBiased - 1;
  // Adds to the word of token `at`; true for the first to touch it.
  static __device__ __forceinline__ bool add(W* words, uint32_t at, uint32_t flag, bool counted) {
    uint32_t* w = reinterpret_cast<uint32_t*>(words) + (sizeof(W) == 2 ? at >> 1 : at);
    const int sh = sizeof(W) == 2 ? 16 * (at & 1) : 0;
    const uint32_t old = counted ? atomicAdd(w, 1u << sh) : atomicOr(w, flag << sh);
    return ((old >> sh) & (sizeof(W) == 2 ? 0xffffu : 0xffffffffu)) == 0;
  }
};

constexpr uint64_t kFailedKey = ~0ull;  // above every token's key: a CTA that found the status word set and did no work

__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
  if (x == -INFINITY) return 0ull;
  uint32_t b = __float_as_uint(x);
  b = x != x ? 0xfffffffeu : (x == 0.f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u));
  return static_cast<uint64_t>(b) << 32 | (0xffffffffu - token);
}

__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if constexpr (DT == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if constexpr (DT == 1) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

// The places of the lanes with `fresh` go to the end of the list, with one addition for the warp.
__device__ __forceinline__ void append_place(bool fresh, uint32_t place, uint16_t* list, int* listed) {
  const uint32_t who = __ballot_sync(0xffffffffu, fresh);
  if (who == 0) return;
  const int lane = threadIdx.x & 31;
  int at = 0;
  if (lane == 0) at = atomicAdd(listed, __popc(who));
  at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
  if (fresh) list[at] = static_cast<uint16_t>(place);
}

struct RowRules {
  float repetition, frequency, presence;
};

template <int DT>
struct Raw {  // kVec logits as they lie in memory
  uint4 v[DT == 2 ? 2 : 1];
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[DT == 2].x, v[DT == 2].y, v[DT == 2].z, v[DT == 2].w};
    if constexpr (DT == 2) return __uint_as_float(w[e]);
    const uint16_t h = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
    return DT == 0 ? __bfloat162float(__ushort_as_bfloat16(h)) : __half2float(__ushort_as_half(h));
  }
};

template <int DT, typename W>
__global__ void __launch_bounds__(kRuleThreads, 2)
logit_rules_kernel(const __grid_constant__ dkv_logits_args a, int splits, int slice) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t keys[kRuleThreads / 32];
  __shared__ uint64_t slice_key;
  __shared__ int listed;
  __shared__ __align__(16) int32_t ids[kMaxBias];  // the row's biases
  __shared__ __align__(16) float values[kMaxBias];
  W* words = reinterpret_cast<W*>(smem);  // [slice + 32]
  uint32_t* mask = reinterpret_cast<uint32_t*>(smem + (slice + 32) * sizeof(W));  // [slice / 32 + 4], the slice's grammar
  uint16_t* list = reinterpret_cast<uint16_t*>(mask + slice / 32 + 4);
  const int row = blockIdx.x / splits, rank = blockIdx.x % splits;
  const int tid = threadIdx.x;
  constexpr int kSize = DT == 2 ? 4 : 2, kHeld = DT == 2 ? 2 : 4;  // loads that a thread has under way
  const uint8_t* in = static_cast<const uint8_t*>(a.logits) + row * a.row_stride * kSize;
  float* out = a.adjusted ? a.adjusted + static_cast<int64_t>(row) * a.vocab : nullptr;
  const uint32_t* allowed = a.allowed ? a.allowed + static_cast<int64_t>(row) * ((a.vocab + 31) / 32) : nullptr;
  const int per = ((a.vocab + splits - 1) / splits + 31) / 32 * 32;  // tokens of a CTA
  const int end = min(a.vocab, (rank + 1) * per);
  const int length = max(0, min(a.lengths[row], a.capacity));
  const int prompt = a.prompts[row];
  const int32_t* hist = a.history + static_cast<int64_t>(row) * a.capacity;
  const RowRules rules = {a.repetition[row], a.frequency[row], a.presence[row]};
  // The history comes kPast tokens a thread at a time, all of them under way before the first is counted.
  int32_t past[kPast];
  auto fetch_past = [&](int base) {
#pragma unroll
    for (int k = 0; k < kPast; ++k) {
      const int i = base + k * kRuleThreads + tid;
      past[k] = i < length ? hist[i] : -1;
    }
  };
  fetch_past(0);
  for (int i = tid; i < a.n_bias; i += kRuleThreads) {
    ids[i] = a.bias_ids[static_cast<int64_t>(row) * a.n_bias + i];
    values[i] = a.bias_values[static_cast<int64_t>(row) * a.n_bias + i];
  }
  const bool failed = cta_failed_at_entry(a.status);  // a barrier of the CTA
  uint64_t best = 0;
  float top = -INFINITY;  // of the thread's untouched tokens, in ascending order: the first of equal ones stays
  int top_at = 0;
  for (int lo = rank * per; lo < end && !failed; lo += slice) {
    const int n = min(slice, end - lo);
    // Place p of the slice is token lo - pad + p: vectors of kVec places start on 16-byte boundaries of the logits.
    const int pad = static_cast<int>(reinterpret_cast<uintptr_t>(in + static_cast<int64_t>(lo) * kSize) / kSize % kVec);
    const int first = lo - pad, last = pad + n;
    const bool out_wide = out != nullptr && reinterpret_cast<uintptr_t>(out + first) % 16 == 0;
    // ---- the first of the slice's logits, on their way while the words are made
    Raw<DT> raw[kHeld];
    auto fetch = [&](int p, Raw<DT>& r) {
      if (p >= pad && p + kVec <= last) {
        const uint4* src = reinterpret_cast<const uint4*>(in + static_cast<int64_t>(first + p) * kSize);
#pragma unroll
        for (int h = 0; h < (DT == 2 ? 2 : 1); ++h) r.v[h] = src[h];
      }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) fetch((k * kRuleThreads + tid) * kVec, raw[k]);
    __syncthreads();
    const int masks = allowed ? (n + 31) / 32 : -1;
    for (int i = tid; i <= masks; i += kRuleThreads) mask[i] = i < masks ? allowed[lo / 32 + i] : 0u;
    const int fill = ((n + 32) * static_cast<int>(sizeof(W)) + 15) / 16;
    for (int i = tid; i < fill; i += kRuleThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) listed = 0;
    __syncthreads();
    for (int base = 0; base < length; base += kPast * kRuleThreads) {
      if (base > 0 || lo != rank * per) fetch_past(base);
#pragma unroll
      for (int k = 0; k < kPast; ++k) {
        const uint32_t at = static_cast<uint32_t>(past[k]) - static_cast<uint32_t>(lo);
        const uint32_t place = at + pad;
        const bool fresh = at < static_cast<uint32_t>(n) &&
                           Word<W>::add(words, place, Word<W>::kSeen, base + k * kRuleThreads + tid >= prompt);
        append_place(fresh, place, list, &listed);
      }
    }
    for (int base = 0; base < a.n_bias; base += kRuleThreads) {
      const int i = base + tid;
      const uint32_t at = i < a.n_bias ? static_cast<uint32_t>(ids[i]) - static_cast<uint32_t>(lo) : 0xffffffffu;
      const uint32_t place = at + pad;
      const bool fresh = at < static_cast<uint32_t>(n) && Word<W>::add(words, place, Word<W>::kBiased, false);
      append_place(fresh, place, list, &listed);
    }
    __syncthreads();
    // ---- the untouched tokens (what is written for the others is overwritten below)
    for (int k0 = 0; k0 * kRuleThreads * kVec < last; k0 += kHeld)
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int p = ((k0 + k) * kRuleThreads + tid) * kVec;
      if (p >= last) break;
      const int token = first + p;
      const bool whole = p >= pad && p + kVec <= last;
      float x[kVec];
      if (whole) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = raw[k].get(e);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[e] = p + e >= pad && p + e < last ? logit_at<DT>(in, token + e) : -INFINITY;
      }
      fetch(p + kHeld * kRuleThreads * kVec, raw[k]);
      if (allowed) {
        const int at = max(p - pad, 0);
        const uint32_t ok = __funnelshift_r(mask[at >> 5], mask[(at >> 5) + 1], at & 31) << (at - (p - pad));
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (!(ok & (1u << e))) x[e] = -INFINITY;
      }
      if (whole && out_wide) {
        reinterpret_cast<float4*>(out + token)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(out + token)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else if (out != nullptr) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (p + e >= pad && p + e < last) out[token + e] = x[e];
      }
      uint32_t any = 0;
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(W)) / 2; ++h) {
        const uint4 w = reinterpret_cast<const uint4*>(words + p)[h];
        any |= w.x | w.y | w.z | w.w;
      }
      if (any != 0) {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (words[p + e] != 0) x[e] = -INFINITY;
      }
      float m = x[0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) m = max_nan(m, x[e]);
      if (!(m <= top)) {  // larger, or a NaN: rare
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (top == top && !(x[e] <= top)) {
            top = x[e];
            top_at = token + e;
          }
      }
    }
    __syncthreads();
    // ---- the touched ones
    auto finish = [&](int token, uint32_t word, float bias) {
      float x = logit_at<DT>(in, token);
      if (word & ~Word<W>::kBiased) {
        x = x > 0.f ? __fdiv_rn(x, rules.repetition) : __fmul_rn(x, rules.repetition);
        const uint32_t made = word & Word<W>::kCount;
        if (made != 0) {
          x = __fsub_rn(x, __fmul_rn(rules.frequency, static_cast<float>(made)));
          x = __fsub_rn(x, rules.presence);
        }
      }
      if (word & Word<W>::kBiased) x = __fadd_rn(x, bias);
      if (allowed && !((mask[(token - lo) >> 5] >> (token & 31)) & 1u)) x = -INFINITY;
      if (out) out[token] = x;
      const uint64_t key = order_key(x, token);
      best = key > best ? key : best;
    };
    for (int i = tid; i < listed; i += kRuleThreads) {
      const int p = list[i];
      const uint32_t word = words[p];
      if (!(word & Word<W>::kBiased)) finish(first + p, word, 0.f);
    }
    // The first entry of a biased token takes it, with the sum of all its entries in their order. The last warps begin:
    // the list keeps the first ones busy.
    for (int i = kRuleThreads - 1 - tid; i < a.n_bias; i += kRuleThreads) {
      const int id = ids[i];
      const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(lo);
      if (at >= static_cast<uint32_t>(n)) continue;
      bool before = false;
      float sum = 0.f;
#pragma unroll 8
      for (int k = 0; k < a.n_bias; ++k) {
        const bool same = ids[k] == id;
        before = before || (same && k < i);
        sum = same ? __fadd_rn(sum, values[k]) : sum;
      }
      if (!before) finish(id, words[at + pad], sum);
    }
  }
  const uint64_t top_key = order_key(top, top_at);
  best = top_key > best ? top_key : best;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, best, d);
    best = other > best ? other : best;
  }
  // A row of the same launch may have set the status word in between, seen by some CTAs of this row and not by others: one
  // that did no work leaves the row without a token, for what the others found is of a part of the vocabulary.
  if (failed) best = kFailedKey;
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
    if (tid < splits) {
      const uint32_t addr = mapa_shared(smem_u32(&slice_key), tid);
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(addr) : "memory");
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, d);
      key = other > key ? other : key;
    }
    if (tid == 0) {
      const int64_t token =
          key == 0 || key == kFailedKey ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
      a.tokens[row] = token;
      if (a.append && token >= 0) {
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

template <int DT, typename W>
int launch_rules(const dkv_logits_args& a, cudaStream_t stream) {
  // Where clusters of eight would come in a second wave of CTAs, clusters of four with slices twice as long do not (two
  // CTAs per SM), and go through the history half as often: 64 rows of 128256 took 24 us against 34, 40 rows 24
  // against 31; one row has 8.0 us with eight. 32-bit words allow half the slice.
  const int splits = a.n_rows * kMaxSplits <= 2 * device_sms() ? kMaxSplits : kMaxSplits / 2;
  const int most = sizeof(W) == 2 ? kMaxSlice : kMaxSlice / 2;
  const int per = ((a.vocab + splits - 1) / splits + 31) / 32 * 32;
  const int slice = per < most ? per : most;
  // Every touched token of a slice has a place in the list.
  const int64_t touched = static_cast<int64_t>(a.capacity) + a.n_bias;
  const int room = static_cast<int>(touched < slice ? touched : slice);
  auto kernel = logit_rules_kernel<DT, W>;
  static std::atomic<uint64_t> done{0};
  if (!allow_shared(kernel, (most + 40) * static_cast<int>(sizeof(W)) + most * 2 + most / 8 + 32, done)) return DKV_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.n_rows * splits);
  cfg.blockDim = dim3(kRuleThreads);
  cfg.dynamicSmemBytes = (slice + 32) * static_cast<int>(sizeof(W)) + slice / 8 + 16 + (room * 2 + 15) / 16 * 16 + 16;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, splits, slice) == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
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
  if (a->n_bias > dkv::kMaxBias || a->vocab > (1 << 30) || a->n_rows > (INT32_MAX / dkv::kMaxSplits))
    return DKV_ERR_CONFIG;
  if (a->n_rows == 0) return DKV_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 14 bits count what a history of at most 16383 tokens can repeat; the halved words leave room for twice the CTAs.
  if (a->capacity <= 16383)
    return a->dtype == 0   ? dkv::launch_rules<0, uint16_t>(*a, st)
           : a->dtype == 1 ? dkv::launch_rules<1, uint16_t>(*a, st)
                           : dkv::launch_rules<2, uint16_t>(*a, st);
  return a->dtype == 0   ? dkv::launch_rules<0, uint32_t>(*a, st)
         : a->dtype == 1 ? dkv::launch_rules<1, uint32_t>(*a, st)
                         : dkv::launch_rules<2, uint32_t>(*a, st);
}
