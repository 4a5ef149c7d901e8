// bn_q8_plan.hpp -- the 8-bit cache's choices of kernels, by sizes alone (plain C++).
#pragma once

#include <cstdint>

#include "bn_paged_plan.hpp"

namespace bn {
namespace {

// Whether a decode's rows go past the caches' keeping: where no other workgroup reads their lines.
// Of pages whose rows of a KV head lie one behind the other none does (64 caches of 4096 keys 29.9 us,
// else 33.1; three of 34763 to 131072 34.8, 38.5; 64 of 512..4096 23.6, 23.1); of token-major pages two
// heads' rows share a line (64 caches of 4096 35.3 us, else 38.4; of 512..4096 24.2, 27.9; 33.4 on XCDs of their own); and blocks of more than one of query heads (more than 16 a KV
// head) read all rows once each (64 caches of 4096 keys, 2 KV heads of 32 query heads each, 21.9 us,
// else 23.3; 64 of 512..4096, 4 of 32, 30.7, 32.6; of 1 of 32 18.2, 18.0).
inline bool decode_reads_once(int64_t row_stride, int hblocks) { return row_stride == HD && hblocks == 1; }

// Codes are turned into bf16 once a tile and workgroup, so that units of 256 rows pay
// at fewer rows than in a cache of bf16: with 32 and 4 heads the pipelined kernel takes, and
// units of 128, for 4 x 1024 rows (1028 units) 36.4 us and 35.3, 3 x 1500 (1128) 48.1 and 47.8,
// 2 x 2500 (1252) 74.3 and 77.3, 5200 (1304) 166 and 189, 6 prompts of 600..1100 behind 2000
// keys 121 and 128, 7 of 165..1500 behind up to 700 83 and 87.
constexpr int kPipeFrom = 1200;

inline PrefillPlan plan_q8(int dtype, int n_seq, int n_rows, int n_heads, int n_kv_heads, int cap, bool most = false) {
  return plan_prefill(dtype, n_seq, n_rows, n_heads, n_kv_heads, cap, most, kPipeFrom);
}

}  // namespace
}  // namespace bn
