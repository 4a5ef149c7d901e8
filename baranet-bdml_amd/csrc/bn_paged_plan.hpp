// bn_paged_plan.hpp -- the paged calls' parameters, and how a ragged prefill's
// work is divided: the host's choice of kernel, launch and records, and the
// search by which every workgroup finds its piece from the lengths.  Plain C++
// but for the lanes' operations: whoever includes it has wave_scan, wave_min,
// wave_total and the wave builtins, so that a CPU build can run 64 lanes of it.
#pragma once

#include <algorithm>
#include <cstdint>

#include "bn_hip.h"

namespace bn {
namespace {

constexpr int HD = 64;
constexpr int kRec = HD + 2;  // floats of a record's row: acc[64], m (log2 units), l

// The cache as the kernels see it.  Offsets in elements.
struct Paged {
  const void *k, *v;
  const int32_t *table, *lens;
  int64_t page_stride, head_stride, row_stride, table_stride;
  int batch, n_pages, shift, n_kv_heads;  // page_size = 1 << shift
  int cap;                                // keys a table row holds
};

struct AttnParams {
  Paged c;
  const void *q;
  void *o;
  const int32_t *starts;  // null: one row per sequence
  int64_t q_rs, o_rs;
  int n_rows, n_heads, group;
  float inv_group;  // 1 / group
  float cl;         // scale * log2(e)
  const int32_t *prefix_pages;
  int prefix_len;
};

// The rows of a (sequence, KV head) are its new tokens' query heads of the
// group, token by token (row r: token r / group, head r % group), so that any
// group fills the products' rows and a few tokens take few of them.  A unit is
// R = 32 * HW consecutive rows; its keys go in tiles of 32.
struct PrefillParams {
  AttnParams a;
  // Records.  Of a cut unit's part [slot][33][R] pairs of floats: the accumulators' pairs of
  // elements, row by row, then (reference, sum) -- through to memory 8 bytes a lane, which rows
  // of a record next to each other make whole lines (row by row they were not: the prefix of
  // 16387 keys for 200 sequences 112 us, its rows now 272 bytes apart through the caches).
  // Of a prefix's part [slot][R][kRow]: the same by rows, for the launch that adds them.
  float *ws;
  unsigned long long *arrive_end;  // two arrival words per slot below it
  unsigned long long tag;
  int slots;      // records that the workspace holds
  int parts_all;  // a part is at least 1 / parts_all of all the call's tiles
  int pieces;     // of a KV head, at most
  // not 0: the rows are the batch's, the keys those of prefix_pages, and every unit's are
  // cut into so many parts, whose records are left for the launch that adds them
  int prefix_parts;
};
struct Piece {
  int b, g, unit, part, parts;  // part of parts of the unit's keys
  int row0, rows;               // the sequence's rows of the tensors
  int last;                     // keys the sequence's last row sees, before the table's clamp
  int slot;                     // record of the unit's first part (parts > 1)
  int tok0, rem0;               // the unit's first row: token, head of the group
};
// Row r of the unit (r < 256): its token and its head of the group.  rem0 + r is
// below group + 256, where the product with 1 / group errs by less than half of that.
__device__ __forceinline__ int token_of(const Piece &w, float inv_group, int group, int r, int &head) {
  const int x = w.rem0 + r, q = (int)(((float)x + 0.5f) * inv_group);
  head = x - q * group;
  return w.tok0 + q;
}
__device__ __forceinline__ void first_row(Piece &w, int row, int group) {
  w.tok0 = __builtin_amdgcn_readfirstlane((int)((uint32_t)row / (uint32_t)group));
  w.rem0 = row - w.tok0 * group;
}
// Part `part` of `parts` of n: first and end.
__device__ __forceinline__ void part_of(int n, const Piece &w, int &from, int &to) {
  from = 0;
  to = n;
  if (w.parts > 1) {
    const int q = __builtin_amdgcn_readfirstlane((int)((uint32_t)n / (uint32_t)w.parts)), r = n - q * w.parts;
    from = w.part * q + min(w.part, r);
    to = from + q + (w.part < r);
  }
}
constexpr int kPartMin = 24;  // tiles of a part at least (128 rows behind 8064 keys 28 us, with parts of 16 tiles 51: records)
constexpr int kRow = HD + 4;  // floats of a prefix record's row

// Which piece of work is workgroup L's.  A call's units differ in length (the
// diagonal, and the sequences themselves): a unit whose keys are more than
// twice a 1024th part of all the call's tiles is cut into parts, as many as
// its sequence's longest unit has such shares, so that no compute unit is left
// with a long one at the end; sequences of no such unit are not cut.  XCDs: a
// KV head's units go to 8 / n_kv_heads of them, whose L2s then hold its keys.
// Every wave finds its piece itself from the lengths.  False: none.
template <int R>
__device__ __forceinline__ bool find_piece(const PrefillParams &p, int block, Piece &w) {
  const Paged &c = p.a.c;
  const int lane = threadIdx.x & 63, hkv = c.n_kv_heads, G = p.a.group;
  int idx;
  if (hkv <= 8 && (8 % hkv) == 0) {
    const int x = block & 7;
    int j = block >> 3;  // a compute unit that got a long piece of one round gets a short one of the next
    if ((j & 32) && !p.prefix_parts) j = (j & ~31) + 31 - (j & 31);
    w.g = x % hkv;
    idx = j * (8 / hkv) + x / hkv;
  } else {
    w.g = block % hkv;
    idx = block / hkv;
  }
  if (p.prefix_parts) {
    w.b = w.row0 = 0;
    w.rows = c.batch;
    w.last = p.a.prefix_len;
    w.parts = p.prefix_parts;
    w.unit = idx / w.parts;
    w.part = idx - w.unit * w.parts;
    w.slot = w.unit * w.parts * hkv + w.g;
    first_row(w, w.unit * R, G);
    return w.unit * R < w.rows * G;
  }
  struct Seq {
    int row0, rows, last, units, steps;  // steps: tiles of its longest unit
    float weight;                        // tiles of all its units, about
  };
  auto seq = [&](int b) __attribute__((always_inline)) {
    Seq s;
    const int bb = min(b, c.batch - 1), s0 = p.a.starts[bb], s1 = p.a.starts[bb + 1];
    s.row0 = min(max(s0, 0), p.a.n_rows);
    s.rows = min(max(s1, s.row0), p.a.n_rows) - s.row0;
    s.last = max(c.lens[bb], 0) - s1 + s.row0 + s.rows;  // (s1 is past the tensors' rows: not its last)
    if (b >= c.batch) s.rows = 0;
    s.units = (s.rows * G + R - 1) / R;
    auto tiles = [&](int n) { return (min(max(n, 0), c.cap) + 31) >> 5; };
    s.steps = tiles(s.last);
    const int first = tiles(s.last - s.rows + min(s.rows, (R + G - 1) / G));
    s.weight = (float)s.units * (0.5f * (float)(s.steps + first) + 1.f);
    return s;
  };
  const int n = c.batch, per = (n + 63) >> 6;
  Seq mine = seq(lane * per);
  float total = lane * per < n ? mine.weight : 0.f;
  for (int i = 1; i < per; ++i) total += lane * per + i < n ? seq(lane * per + i).weight : 0.f;
  total = wave_total(total);
  const int share = max((int)min(total * (float)hkv / (float)p.parts_all, 536870912.f), kPartMin);
  // (a division only where it can come to 2 or more)
  auto parts_of = [&](const Seq &s) { return s.steps < 2 * share ? 1 : (int)((uint32_t)s.steps / (uint32_t)share); };
  auto count = [&](const Seq &s, bool in, int &all, int &cut) __attribute__((always_inline)) {
    const int parts = parts_of(s), k = in ? s.units * parts : 0;
    all = min(all + k, p.pieces + 1);
    cut = min(cut + (parts > 1 ? k : 0), p.pieces + 1);
  };
  int all = 0, cut = 0;
  count(mine, lane * per < n, all, cut);
  for (int i = 1; i < per; ++i) count(seq(lane * per + i), lane * per + i < n, all, cut);
  int up = wave_scan(all), up_cut = wave_scan(cut);
  // (row_starts that decrease can count more pieces than the launch has: then none is
  // done, so that no count of a unit's parts is left unfinished in the workspace; a lane
  // counts no further than one too many, and 64 of those are below 2^32)
  const uint32_t total_pieces = (uint32_t)__builtin_amdgcn_readlane(up, 63);
  if ((uint32_t)idx >= total_pieces || total_pieces > (uint32_t)p.pieces) return false;
  int src, b, k, cuts;  // lane and number of the sequence, piece of it, pieces of cut sequences before it
  if (per == 1) {
    // The longest first over all sequences: from one unit to the one before it
    // the keys fall by the same R / group in every sequence, so that a sequence's
    // units take a run of levels, one each, from the level of its longest on.
    // (Levels only order the units, so lengths count up to the table's room and levels to
    // 2^28 here: neither a distance nor off + units, of at most 2^26 units, passes 32 bits.)
    const int parts = parts_of(mine), units = lane < n ? mine.units : 0;
    const int at = min(max(mine.last, 0), c.cap), top = -wave_min(units ? -at : 0);
    const int off = units ? (int)min((float)(top - at) * ((float)G * (1.f / R)), 268435456.f) : 0;
    auto pieces_above = [&](int level) __attribute__((always_inline)) {
      return __builtin_amdgcn_readlane(wave_scan(parts * min(max(level - off, 0), units)), 63);
    };
    int lo = 0, hi = -wave_min(-(off + units)), below = 0;  // pieces_above(lo) <= idx < pieces_above(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, n_mid = pieces_above(mid);
      if (n_mid <= idx) {
        lo = mid;
        below = n_mid;
      } else {
        hi = mid;
      }
    }
    const int here = off <= lo && lo < off + units ? parts : 0, to = wave_scan(here);
    src = __builtin_ctzll(__builtin_amdgcn_ballot_w64(to > idx - below));
    b = src;
    k = (lo - __builtin_amdgcn_readlane(off, src)) * __builtin_amdgcn_readlane(parts, src) + idx - below -
        __builtin_amdgcn_readlane(to - here, src);
    cuts = __builtin_amdgcn_readlane(up_cut - cut, src);
  } else {
    src = __builtin_ctzll(__builtin_amdgcn_ballot_w64(up > idx));
    int before = __builtin_amdgcn_readlane(up - all, src);
    cuts = __builtin_amdgcn_readlane(up_cut - cut, src);
    b = src * per;
    for (;;) {  // the sequence within the lane's run, 64 at a time
      mine = seq(b + lane);
      all = cut = 0;
      count(mine, b + lane < n, all, cut);
      up = wave_scan(all);
      up_cut = wave_scan(cut);
      const unsigned long long hit = __builtin_amdgcn_ballot_w64(before + up > idx);
      if (hit) {
        src = __builtin_ctzll(hit);
        before += __builtin_amdgcn_readlane(up - all, src);
        cuts += __builtin_amdgcn_readlane(up_cut - cut, src);
        b += src;
        break;
      }
      before += __builtin_amdgcn_readlane(up, 63);
      cuts += __builtin_amdgcn_readlane(up_cut, 63);
      b += 64;
    }
    k = idx - before;
  }
  w.b = b;
  w.row0 = __builtin_amdgcn_readlane(mine.row0, src);
  w.rows = __builtin_amdgcn_readlane(mine.rows, src);
  w.last = __builtin_amdgcn_readlane(mine.last, src);
  const int units = __builtin_amdgcn_readlane(mine.units, src), steps = __builtin_amdgcn_readlane(mine.steps, src);
  w.parts = steps < 2 * share ? 1 : __builtin_amdgcn_readfirstlane((int)((uint32_t)steps / (uint32_t)share));
  const int from_end =  // longest units first
      w.parts == 1 ? k : __builtin_amdgcn_readfirstlane((int)((uint32_t)k / (uint32_t)w.parts));
  w.unit = units - 1 - from_end;
  w.part = k - from_end * w.parts;
  w.slot = (cuts + from_end * w.parts) * hkv + w.g;  // parts of a unit: hkv slots apart
  first_row(w, w.unit * R, G);
  // (row_starts that decrease could count rows twice and pass the workspace)
  return w.parts == 1 || (int64_t)w.slot + (int64_t)(w.parts - 1) * hkv < p.slots;
}

// Which prefill kernel: by the units of 128 rows (32 in fp32) that the call has
// at most.  Few of them: the keys of a unit are split over more waves.  The
// pipelined kernel's units of 256 rows take longer to start and to fill the card:
// it is for many rows in sequences of 512 new ones or more (one prompt of 2048
// rows 42 us, units of 128 rows 37; of 4096 100 and 105; 64 prompts of 128 rows
// 54 and 28), or for long sequences, which the host knows only by what the
// table holds (behind 16384 keys 256 rows 95 -> 61 us, 2048 rows 319 -> 275;
// behind nothing 1024 rows 21 -> 30 where the table has room for 16384).  parts_all: one piece per compute unit, two of the
// pipelined kernel's (2048 rows of 16384 317 -> 275 us) unless that makes many
// records of few units (256 rows 61 -> 73).
struct PrefillPlan {
  int hw, kw;  // (hw 8: the pipelined kernel)
  int parts_all;
  int64_t pieces, groups, slots;  // pieces of a KV head, workgroups of the launch, records
  size_t records, words;   // bytes
};
// most: not this call's plan but one whose workspace does for any call of at
// most as many rows (with fewer rows a sequence the kernel may be another).
// pipe_from: the units of 128 rows from which the pipelined kernel is taken.
inline PrefillPlan plan_prefill(int dtype, int n_seq, int n_rows, int n_heads, int n_kv_heads, int cap, bool most = false,
                                int pipe_from = 2048) {
  PrefillPlan d;
  const int64_t rows = (int64_t)n_rows * (n_heads / n_kv_heads);  // of a KV head
  const int64_t u128 = (rows / 128 + 1) * n_kv_heads, u32 = (rows / 32 + 1) * n_kv_heads;
  const bool far = cap >= 16384 && u128 * cap >= 1 << 20, long_rows = n_rows / 512 >= n_seq;
  if (dtype == BN_F32) {
    d.hw = 1;
    d.kw = u32 <= 1024 ? 4 : 2;  // (one prompt of 512 rows 23 us, with 2 waves a unit 30; four of 300 39 and 31)
  } else if (far ? u128 < 1024 || long_rows || most : u128 >= pipe_from && (long_rows || most)) {
    d.hw = 8;
    d.kw = 1;
  } else if (u128 < 256) {
    d.hw = 1;  // (700 rows behind nothing 12.6 us, units of 128 rows 16.3; 256 x 3 behind 8192 93 and 106)
    // (256 rows behind 4096 29 us, with 4 waves 33; behind nothing 9.7 and 8.5; 300 behind 3700 43 and 37)
    d.kw = (rows + 31) / 32 * n_kv_heads <= 256 ? 8 : 4;
  } else {
    d.hw = 4;
    d.kw = u128 <= 768 ? 2 : 1;  // (2000 rows 37 us, with 1 wave a row block 48; 777 x 4 31 and 27)
  }
  d.parts_all = d.hw == 8 && (u128 >= 256 || most) ? 512 : 256;
  const int R = 32 * d.hw;
  const int64_t units = std::min((rows + R - 1) / R + n_seq, rows);  // of a KV head, over the sequences
  // a sequence of U units, the longest of s tiles, counts U * s / 2 tiles at least and is cut
  // into U * floor(s / share) pieces: at most 2 * total / share in all, where total is
  // below (share + 1) * parts_all / n_kv_heads and share at least kPartMin
  const int64_t most_parts = std::max(1, (cap / 32 + 1) / kPartMin);
  const int64_t cut =
      most_parts > 1 ? std::min<int64_t>(units * most_parts, (2 * d.parts_all + d.parts_all / 8) / n_kv_heads + 2) : 0;
  const int64_t pieces = d.pieces = units + cut;
  const int per = n_kv_heads <= 8 && 8 % n_kv_heads == 0 ? 8 / n_kv_heads : 1;
  // (whole rounds of 32 pieces an XCD, which are taken in reverse order every second time)
  d.groups = per > 1 || n_kv_heads == 8 || n_kv_heads == 1 ? ((pieces + per - 1) / per + 31) / 32 * 32 * per * n_kv_heads
                                                           : pieces * n_kv_heads;
  d.slots = cut * n_kv_heads;
  d.records = (size_t)d.slots * R * kRec * sizeof(float);
  d.words = (size_t)d.slots * 16 * d.hw;  // (16 are used: the words grow with the records)
  return d;
}

}  // namespace
}  // namespace bn
