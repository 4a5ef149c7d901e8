// bn_q8_plan.hpp -- the 8-bit cache's choices of kernels, by sizes alone (plain C++).
#pragma once

#include <cstdint>

#include "bn_paged_plan.hpp"

namespace bn {
namespace {

// Whether a decode's rows go past the caches' keeping: where no other workgroup reads their lines.
// Of pages whose rows of a KV head lie one behind the other none does (64 caches of 4096 keys 27.9 us,
// else 31.5); of token-major pages two heads' rows share a line (64 caches of 512..4096 23.9 us, else
// 26.1; 33.4 on XCDs of their own); and blocks of more than one of query heads (more than 16 a KV
// head) read all rows once each (64 caches of 4096 keys, 2 KV heads of 32 query heads each, 21.9 us,
// else 23.3; 64 of 512..4096, 4 of 32, 30.7, 32.6; of 1 of 32 18.2, 18.0).
inline bool decode_reads_once(int64_t row_stride, int hblocks) { return row_stride == HD && hblocks == 1; }

}  // namespace
}  // namespace bn
