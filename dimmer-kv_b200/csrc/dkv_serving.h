// dkv_serving.h — status codes of the block tables, the paged 4-bit cache and the logit rules, beside those that
// dkv_ptx.cuh has for every kernel.
#pragma once

namespace dkv {

enum ServingError : int {
  kErrNoPages = 111,       // fewer free pages than the plan needs
  kErrCounts = 112,        // a token count or a length out of its range
  kErrCellRange = 113,     // a key or value that no 4-bit cell holds (not finite, or beyond 2^15)
  kErrHistory = 114,       // no room for a token in a history
};
// Added to the code, as dkv_ptx.cuh's sites are.
constexpr int kSiteQ4Attend = 7000;    // q4_decode_kernel, q4_prefill_kernel
constexpr int kSiteQ4Rows = 8000;      // q4_append_kernel, q4_read_kernel
constexpr int kSitePages = 9000;       // page_plan_kernel, page_trim_kernel, page_slots_kernel

}  // namespace dkv
