// bn_qk_plan.hpp -- launches of the norms of single heads, by sizes alone (plain C++).
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bn {
namespace {

constexpr int kMostRows = 8, kJoinedRows = 16;  // rows of a workgroup at once; of backward's where one adds all sums

// Forward's rows of a workgroup: more of them share the wait for their positions and angles, fewer start
// sooner and end evenly.  In bf16, 1, 4 and 8 rows, us: 2047 and 2048 rows of 10 heads of 64 3.7, 3.5, 3.9, 8192
// 10.0, 6.7, 7.1; of 10 heads of 16 3.2, 2.7, 2.7 and 7.1, 3.7, 3.4; of 36 heads of 64 6.1, 7.0, 8.7 and 16.8, 15.6,
// 16.1, 16384 34.3, 35.6, 33.9; of 40 heads of 128 8192 38.1, 36.4, 40.2.  (Long rows alone would have 4 from some
// 6000 rows on.)
inline int rows_at_once(int n_rows) { return n_rows >= 8192 ? 8 : n_rows >= 2048 ? 4 : 1; }

// Backward's launch: its workgroups, their rows at once, whether the last of them adds their sums.
// It does for small calls, to which a second launch adds more on the host than they take (300 fp32
// rows of 32 and 4 heads of 64 called one behind the other 15.0 -> 12.1 us; in a graph, where it
// costs little, 8.1 -> 9.0).  Arrivals are counted one by one and one compute unit reads the sums,
// so there are at most 128 workgroups and 64 KB of sums (512 bf16 rows in a graph 9.6 us, with 256
// workgroups 11.8), and a workgroup has at most kJoinedWork elements (777 fp32 rows of heads of
// 128, which have more, 18.6, now 14.8; 33 bf16 rows of 124 heads of 256, two a workgroup, 15.3 in a graph, now 10.8).
constexpr size_t kArriveBytes = 256;  // (16 are used: the sums keep their lines: 16384 bf16 rows 51.2 -> 50.1 us)
constexpr int kBackGroups = 1024, kJoinedGroups = 128, kJoinedWork = 32768;
struct BackPlan {
  int rows, groups;
  bool joins;
};
inline BackPlan plan_back(int n_rows, int heads, int head_dim) {
  BackPlan d;
  const int most = std::min(kJoinedGroups, 8192 / head_dim);
  const int64_t joined = ((int64_t)n_rows + most - 1) / most;  // rows of a workgroup if they join
  d.joins = n_rows > 0 && joined <= kJoinedRows && joined * heads * head_dim <= kJoinedWork;
  d.rows = d.joins ? (int)joined : std::max(1, std::min(n_rows / 256, kMostRows));
  d.groups = std::min((n_rows + d.rows - 1) / d.rows, kBackGroups);
  return d;
}

}  // namespace
}  // namespace bn
