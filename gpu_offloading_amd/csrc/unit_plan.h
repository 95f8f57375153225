// Work lists of the kernels whose workgroups each run a list of units: one
// record of kUnitInts int32 per (item, KV head), entry 0 the KV head and entry 6
// the unit's tiles, behind a table of the workgroups' (first unit, units).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <functional>
#include <queue>
#include <utility>
#include <vector>

namespace kvc {

constexpr int kUnitInts = 8;

inline int64_t unit_table_ints(int64_t workgroups) { return (2 * workgroups + 3) / 4 * 4; }

// `rec`: n records, one per item, the same for every KV head but entry 0.
//
// Units (item, KV head) in the order a grid of (items, heads) workgroups would
// be dispatched: head-major, items longest first (short units fill the gaps at
// the end).  The hardware hands workgroup w to XCD w % 8 and each XCD's next
// workgroup to its first free CU; the plan replays that list scheduling with
// each unit's cost taken as its tiles + 2, assigning unit d to a workgroup of
// XCD d % 8, so that the units of one request and head run side by side on one
// XCD and share its L2.
inline void write_unit_plan(const std::vector<int32_t>& rec, int64_t n, int hkv, int64_t W,
                            int32_t* plan_host) {
  std::vector<int64_t> order(n);
  for (int64_t i = 0; i < n; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int64_t x, int64_t y) {
    return rec[x * kUnitInts + 6] > rec[y * kUnitInts + 6];
  });
  const int64_t units = n * hkv;
  const int groups = (W % 8 == 0) ? 8 : 1;
  std::vector<std::vector<int64_t>> lists(W);
  typedef std::pair<int64_t, int64_t> Slot;  // (load, workgroup)
  std::vector<std::priority_queue<Slot, std::vector<Slot>, std::greater<Slot>>> free_at(groups);
  for (int64_t b = 0; b < W; ++b) free_at[b % groups].push(Slot(0, b));
  for (int64_t d = 0; d < units; ++d) {
    auto& q = free_at[d % groups];
    const Slot sl = q.top();
    q.pop();
    lists[sl.second].push_back(d);
    q.push(Slot(sl.first + rec[order[d % n] * kUnitInts + 6] + 2, sl.second));
  }
  const int64_t table = unit_table_ints(W);
  std::fill_n(plan_host, table, 0);
  int64_t next = 0;
  for (int64_t b = 0; b < W; ++b) {
    plan_host[2 * b] = int32_t(next);
    plan_host[2 * b + 1] = int32_t(lists[b].size());
    for (const int64_t d : lists[b]) {
      int32_t* dst = plan_host + table + next * kUnitInts;
      std::copy_n(rec.data() + order[d % n] * kUnitInts, kUnitInts, dst);
      dst[0] = int32_t(d / n);  // the KV head
      ++next;
    }
  }
}

}  // namespace kvc
