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

namespace dkv {
namespace {

constexpr int kPage = DKV_PAGE_TOKENS;
constexpr int kPlanThreads = 1024;
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

__device__ __forceinline__ void write_slots(const dkv_page_args& a, const int* starts, int64_t first, int64_t step) {
  const int64_t n = static_cast<int64_t>(a.n_seq) * a.q_len;
  for (int64_t e = first; e < n; e += step) {
    const int s = static_cast<int>(e / a.q_len), i = static_cast<int>(e - static_cast<int64_t>(s) * a.q_len);
    int slot = -1;
    if (i < a.counts[s]) {
      const int at = starts[s] + i;
      slot = a.blocks[static_cast<int64_t>(s) * a.max_blocks + at / kPage] * kPage + at % kPage;
    }
    a.slots[e] = slot;
  }
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const dkv_page_args a, int slots_here) {
  __shared__ int offset[kMaxSeq];
  __shared__ int scratch[kPlanThreads / 32];
  const int tid = threadIdx.x;
  const int64_t capacity = static_cast<int64_t>(a.max_blocks) * kPage;
  const int n_free = a.n_free[0];
  bool bad = tid == 0 && status_at_entry(a.status) != 0;
  bool counts_bad = false;
  int64_t taken = 0;
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
    for (int j = have + lane; j < need; j += 32) row[j] = a.free_pages[n_free - 1 - (offset[s] + j - have)];
    if (lane == 0) a.starts[s] = len;
  }
  __syncthreads();
  if (slots_here) write_slots(a, a.starts, tid, kPlanThreads);
  for (int s = tid; s < a.n_seq; s += kPlanThreads) a.lengths[s] = a.starts[s] + a.counts[s];
  if (tid == 0) a.n_free[0] = n_free - static_cast<int>(taken);
}

// Slots of tokens starts[s] .. starts[s] + counts[s] - 1. The table is read only: any number of CTAs. `checked`:
// the plan that ran before has checked the counts (a failed one left the status word set).
__global__ void __launch_bounds__(256) page_slots_kernel(const dkv_page_args a, int planned) {
  if (status_at_entry(a.status) != 0) {
    if (planned) return;  // the plan wrote -1
    const int64_t n = static_cast<int64_t>(a.n_seq) * a.q_len;
    for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += 256ll * gridDim.x) a.slots[e] = -1;
    return;
  }
  const int64_t n = static_cast<int64_t>(a.n_seq) * a.q_len;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += 256ll * gridDim.x) {
    const int s = static_cast<int>(e / a.q_len), i = static_cast<int>(e - static_cast<int64_t>(s) * a.q_len);
    int slot = -1;
    if (i < a.counts[s]) {
      const int at = a.starts[s] + i;
      if (at < 0 || at >= a.lengths[s]) {
        record_error(a.status, kSitePages + kErrCounts);
      } else {
        slot = a.blocks[static_cast<int64_t>(s) * a.max_blocks + at / kPage] * kPage + at % kPage;
      }
    }
    a.slots[e] = slot;
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
    for (int j = first + lane; j < have; j += 32) {
      a.free_pages[top - (offset[s] + j - first)] = row[j];
      row[j] = -1;
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

int slots_grid(int64_t n) {
  const int64_t g = (n + 1023) / 1024;
  return static_cast<int>(g < 1 ? 1 : (g > 148 * 8 ? 148 * 8 : g));
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
  if (!here) dkv::page_slots_kernel<<<dkv::slots_grid(n), 256, 0, st>>>(*a, 1);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
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
  const int64_t n = static_cast<int64_t>(a->n_seq) * a->q_len;
  if (n == 0) return DKV_OK;
  dkv::page_slots_kernel<<<dkv::slots_grid(n), 256, 0, static_cast<cudaStream_t>(stream)>>>(*a, 0);
  return cudaGetLastError() == cudaSuccess ? DKV_OK : DKV_ERR_CUDA;
}

}  // extern "C"
