// The plan of an append (include/imba_b200.h, imba_append_plan): a step's rows
// by the pages they go to.
#pragma once

#include "cache8.cuh"

namespace imba {

constexpr int kTok = IMBA_PAGE_TOKENS;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxPairs = 64;  // of a head: d_qk <= 128
constexpr int kMaxAxes = 8;
constexpr float kLargest = 3.19014718988379809496e38f;  // 1.875 2^127

// Plan layout (int32 words): [0] number of pages, then from word 64 the hash
// table's keys [cap], the rows of each key's page [cap][16], and the list of
// occupied table positions [num_rows].
constexpr int kPlanHead = 64;
constexpr int kMostRows = 1 << 28;  // of a step: plan_cap is an int32
inline int plan_cap(int32_t n) {
  int cap = 64;
  while (cap < 2 * (int64_t)n) cap *= 2;
  return cap;
}
struct PlanView {
  int* count;
  int* keys;
  int* rows;
  int* list;
  int cap;
};
inline PlanView plan_view(void* plan, int32_t n) {
  PlanView v;
  v.cap = plan_cap(n);
  v.count = static_cast<int*>(plan);
  v.keys = v.count + kPlanHead;
  v.rows = v.keys + v.cap;
  v.list = v.rows + (size_t)v.cap * kTok;
  return v;
}

// k_tile, v_tile: elements from rows 16 i to rows 16 (i + 1) of k and v, 0
// when rows are evenly apart.
template <typename T>
imba_status_t launch_append(const imba_cache_desc& c, const imba_pool_desc& pool, const imba_append_desc& d,
                            void* plan, cudaStream_t s, int64_t k_tile = 0, int64_t v_tile = 0);
// The plan of `slots` in `plan` (imba_append_plan_bytes(num_rows) of device memory).
cudaError_t launch_append_plan(int64_t num_slots, int32_t num_rows, const int32_t* slots, void* plan, int32_t* status,
                               cudaStream_t s);

}  // namespace imba
