// pages.cu — block tables and slot maps of the paged 4-bit cache, built on the GPU from the conversations'
// lengths (dkv_page_plan, dkv_page_trim, dkv_page_slots).
//
// One plan: have_s = ceil(len_s / 64), need_s = ceil((len_s + new_s) / 64); the exclusive sum of need - have
// over the conversations ranks every page to take, and the page of rank r is free[n_free - 1 - r]. A token's slot
// is its page * 64 + its place. A trim ranks the pages that it releases the same way and puts rank r of R at
// free[n_free + R - 1 - r], so that the first released is on top and trim(starts) undoes plan.
//
// The state (lengths, block table, stack) changes in place, which a replayed graph needs; so everything that
// reads the old state and everything that writes the new one runs in ONE CTA with barriers between, and needs
// no counter in memory and no second launch. Only slots of long prompts are worth more CTAs: they depend on
// the new table alone, and a second kernel writes them.
#include <cstdint>

#include "../../include/dimmer_kv.h"
#include "dkv_ptx.cuh"
#include "dkv_serving.h"

namespace dkv {
namespace {

constexpr int kPage = DKV_PAGE_TOKENS;
constexpr int kPlanThreads = 1024;
constexpr int kBatch = 4;
constexpr int kMaxSeq = 8192;           // conversations of one table (offsets held in shared memory)
constexpr int64_t kSlotsInPlan = 8192;  // slots that the plan's CTA writes itself

__host__ __device__ __forceinline__ int pages_of(int tokens) { return (tokens + kPage - 1) / kPage; }

// Inclusive sum over the CTA's threads; `total` gets the sum of all. scratch: one int per warp.
__device__ __forceinline__ int cta_scan(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < n_warps; ++w) {
    const int s = scratch[w];
    if (w < warp) before += s;
    total += s;
  }
  return x + before;
}

// The slot of token `at` of a conversation whose blocks are `row`.
__device__ __forceinline__ int slot_of(const int32_t* row, int at) { return row[at / kPage] * kPage + at % kPage; }

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const dkv_page_args a, int slots_here) {
  __shared__ int offset[kMaxSeq];
  __shared__ int scratch[kPlanThreads / 32];
  const int tid = threadIdx.x;
  const int64_t capacity = static_cast<int64_t>(a.max_blocks) * kPage;
  const int n_free = a.n_free[0];
  bool bad = tid == 0 && status_at_entry(a.status) != 0;
  bool counts_bad = false;
  int64_t taken = 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int base = 0; base < a.n_seq; base += kPlanThreads) {
    const int s = base + tid;
    int take = 0;
    if (s < a.n_seq) {
      const int len = a.lengths[s], add = a.counts[s];
      if (len < 0 || add < 0 || add > a.q_len || static_cast<int64_t>(len) + add > capacity)
        counts_bad = true;
      else
        take = pages_of(len + add) - pages_of(len);
    }
    int total;
    const int incl = cta_scan(take, scratch, total);
    if (s < a.n_seq) offset[s] = static_cast<int>(taken) + incl - take;
    taken += total;
  }
  const bool no_pages = n_free < 0 || n_free > a.n_pages || taken > n_free;
  const bool fail_counts = __syncthreads_or(counts_bad) != 0;
  if (__syncthreads_or(bad) || fail_counts || no_pages) {
    if (tid == 0) record_error(a.status, kSitePages + (fail_counts ? kErrCounts : kErrNoPages));
    // the slots are -1 all the same: nothing that reads them finds another token's place
    const int64_t n = static_cast<int64_t>(a.n_seq) * a.q_len;
    for (int64_t e = tid; e < n; e += kPlanThreads) a.slots[e] = -1;
    return;
  }
  const int lane = tid & 31, warp = tid >> 5;
  for (int s = warp; s < a.n_seq; s += kPlanThreads / 32) {
    const int len = a.lengths[s];
    const int have = pages_of(len), need = pages_of(len + a.counts[s]);
    int* row = a.blocks + static_cast<int64_t>(s) * a.max_blocks;
    const int32_t* from = a.free_pages + n_free - 1 - offset[s] + have;  // page j is from[-j]
    for (int j = have + lane; j < need; j += 32 * kBatch) {
      int page[kBatch];  // kBatch loads under way at a time
#pragma unroll
      for (int k = 0; k < kBatch; ++k) page[k] = j + 32 * k < need ? __ldg(from - (j + 32 * k)) : 0;
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (j + 32 * k < need) row[j + 32 * k] = page[k];
    }
    if (lane == 0) a.starts[s] = len;
  }
  __syncthreads();
  if (slots_here) {
    const int n = a.n_seq * a.q_len;
    for (int e = tid; e < n; e += kPlanThreads) {
      const int s = e / a.q_len, i = e - s * a.q_len;
      a.slots[e] = i < a.counts[s] ? slot_of(a.blocks + static_cast<int64_t>(s) * a.max_blocks, a.starts[s] + i) : -1;
    }
  }
  for (int s = tid; s < a.n_seq; s += kPlanThreads) a.lengths[s] = a.starts[s] + a.counts[s];
  if (tid == 0) a.n_free[0] = n_free - static_cast<int>(taken);
}

// Slots of tokens starts[s] .. starts[s] + counts[s] - 1: a CTA takes kSlotTile rows of one conversation, a thread four.
// The table is read only. `planned`: the plan that ran before (this launch begins under its end) has checked the counts;
// a failed one left the status word set and every slot -1.
constexpr int kSlotThreads = 256, kSlotTile = 4 * kSlotThreads;
__global__ void __launch_bounds__(kSlotThreads) page_slots_kernel(const dkv_page_args a, int planned) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tiles = (a.q_len + kSlotTile - 1) / kSlotTile;
  const int s = blockIdx.x / tiles, i0 = (blockIdx.x - s * tiles) * kSlotTile + threadIdx.x * 4;
  const bool failed = status_at_entry(a.status) != 0;
  if (i0 >= a.q_len || (failed && planned)) return;
  const int start = a.starts[s], count = a.counts[s], len = a.lengths[s];
  const int32_t* row = a.blocks + static_cast<int64_t>(s) * a.max_blocks;
  int32_t* out = a.slots + static_cast<int64_t>(s) * a.q_len + i0;
  const int n = min(4, a.q_len - i0);
  if (!failed && count > i0 && (start < 0 || start > len || min(count, i0 + n) > len - start)) {
    record_error(a.status, kSitePages + kErrCounts);
    for (int k = 0; k < n; ++k) out[k] = -1;
    return;
  }
  int slot[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) slot[k] = !failed && k < n && i0 + k < count ? slot_of(row, start + i0 + k) : -1;
  if (n == 4 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    *reinterpret_cast<int4*>(out) = make_int4(slot[0], slot[1], slot[2], slot[3]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) out[k] = slot[k];
  }
}

__global__ void __launch_bounds__(kPlanThreads) page_trim_kernel(const dkv_page_args a) {
  __shared__ int offset[kMaxSeq];
  __shared__ int scratch[kPlanThreads / 32];
  const int tid = threadIdx.x;
  const int n_free = a.n_free[0];
  const int64_t capacity = static_cast<int64_t>(a.max_blocks) * kPage;
  bool bad = tid == 0 && status_at_entry(a.status) != 0;
  bool counts_bad = false;
  int64_t released = 0;
  for (int base = 0; base < a.n_seq; base += kPlanThreads) {
    const int s = base + tid;
    int drop = 0;
    if (s < a.n_seq) {
      const int len = a.lengths[s], keep = a.counts[s];
      if (len < 0 || len > capacity || keep < 0)
        counts_bad = true;
      else
        drop = pages_of(len) - pages_of(min(len, keep));
    }
    int total;
    const int incl = cta_scan(drop, scratch, total);
    if (s < a.n_seq) offset[s] = static_cast<int>(released) + incl - drop;
    released += total;
  }
  const bool fail = __syncthreads_or(counts_bad) != 0 || n_free < 0 || released + n_free > a.n_pages;
  if (__syncthreads_or(bad) || fail) {
    if (tid == 0) record_error(a.status, kSitePages + kErrCounts);
    return;
  }
  const int lane = tid & 31, warp = tid >> 5;
  const int top = n_free + static_cast<int>(released) - 1;
  for (int s = warp; s < a.n_seq; s += kPlanThreads / 32) {
    const int len = a.lengths[s], kept = min(len, a.counts[s]);
    const int first = pages_of(kept), have = pages_of(len);
    int* row = a.blocks + static_cast<int64_t>(s) * a.max_blocks;
    int32_t* to = a.free_pages + top - offset[s] + first;  // block j goes to to[-j]
    for (int j = first + lane; j < have; j += 32 * kBatch) {
      int page[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) page[k] = j + 32 * k < have ? row[j + 32 * k] : 0;
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (j + 32 * k < have) {
          to[-(j + 32 * k)] = page[k];
          row[j + 32 * k] = -1;
        }
    }
    __syncwarp();
    if (lane == 0) {
      a.lengths[s] = kept;
      a.starts[s] = kept;
    }
  }
  if (tid == 0) a.n_free[0] = top + 1;
}

int check_pages(const dkv_page_args* a) {
  if (a == nullptr || a->blocks == nullptr || a->lengths == nullptr || a->starts == nullptr || a->counts == nullptr ||
      a->status == nullptr || a->n_seq < 0 || a->max_blocks < 1)
    return DKV_ERR_ARGS;
  if (a->n_seq > kMaxSeq) return DKV_ERR_CONFIG;
  if (static_cast<int64_t>(a->max_blocks) * kPage > INT32_MAX) return DKV_ERR_CONFIG;
  return DKV_OK;
}

int check_pool(const dkv_page_args* a) {
  if (a->free_pages == nullptr || a->n_free == nullptr || a->n_pages < 1) return DKV_ERR_ARGS;
  if (static_cast<int64_t>(a->n_pages) * kPage > INT32_MAX) return DKV_ERR_CONFIG;
  return DKV_OK;
}

int launch_slots(const dkv_page_args& a, int planned, cudaStream_t stream) {
  const int64_t ctas = static_cast<int64_t>(a.n_seq) * ((a.q_len + kSlotTile - 1) / kSlotTile);
  if (ctas > INT32_MAX) return DKV_ERR_CONFIG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSlotThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = planned ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, page_slots_kernel, a, planned) == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

}  // namespace
}  // namespace dkv

extern "C" {

int dkv_page_plan(const dkv_page_args* a, void* stream) {
  int rc = dkv::check_pages(a);
  if (rc == DKV_OK) rc = dkv::check_pool(a);
  if (rc != DKV_OK) return rc;
  if (a->q_len < 0 || (a->slots == nullptr && a->q_len > 0)) return DKV_ERR_ARGS;
  if (a->n_seq == 0) return DKV_OK;
  const int64_t n = static_cast<int64_t>(a->n_seq) * a->q_len;
  const int here = n <= dkv::kSlotsInPlan;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  dkv::page_plan_kernel<<<1, dkv::kPlanThreads, 0, st>>>(*a, here);
  if (cudaGetLastError() != cudaSuccess) return DKV_ERR_CUDA;
  return here ? DKV_OK : dkv::launch_slots(*a, 1, st);
}

int dkv_page_trim(const dkv_page_args* a, void* stream) {
  int rc = dkv::check_pages(a);
  if (rc == DKV_OK) rc = dkv::check_pool(a);
  if (rc != DKV_OK) return rc;
  if (a->n_seq == 0) return DKV_OK;
  dkv::page_trim_kernel<<<1, dkv::kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(*a);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

int dkv_page_slots(const dkv_page_args* a, void* stream) {
  const int rc = dkv::check_pages(a);
  if (rc != DKV_OK) return rc;
  if (a->q_len < 0 || (a->slots == nullptr && a->q_len > 0)) return DKV_ERR_ARGS;
  if (a->n_seq == 0 || a->q_len == 0) return DKV_OK;
  return dkv::launch_slots(*a, 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
