// bn_paged_device.hpp -- what the paged caches' kernels share on the device: finding a row's
// sequence and its place in the pages, the rotation of a row's pieces, counting workgroups in
// at the end of cut work, and the prefill kernels' bodies.
#pragma once

#include <algorithm>
#include <atomic>

#include <cmath>

#include "bn_common.hpp"

namespace bn {
namespace {

// Sums of the lanes up to and with each lane, by moves inside a row of 16
// lanes, then of a row's last lane to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15 to rows 1 and 3
  return dpp_add<0x143, 0xc>(x);  // row_bcast 31 to rows 2 and 3
}

// The lanes' smallest value.
template <int CTRL>
__device__ __forceinline__ int dpp_min(int x) {
  return min(x, __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ int wave_min(int x) {
  x = dpp_min<0x140>(dpp_min<0x141>(dpp_min<0x4E>(dpp_min<0xB1>(x))));  // within a row of 16
  return min(min(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)),
             min(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
}
// The lanes' sum, the same in every wave.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_addf(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_total(float x) {
  x = dpp_addf<0x111, 0xf>(x);
  x = dpp_addf<0x112, 0xf>(x);
  x = dpp_addf<0x114, 0xf>(x);
  x = dpp_addf<0x118, 0xf>(x);
  x = dpp_addf<0x142, 0xa>(x);
  x = dpp_addf<0x143, 0xc>(x);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

}  // namespace
}  // namespace bn

#include "bn_paged_plan.hpp"

namespace bn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The sequence whose rows hold `row`: the last b with starts[b] <= row (-1:
// before the first or behind the last; starts null: one row each).
__device__ __forceinline__ int sequence_of(const int32_t *starts, int batch, int row) {
  if (!starts) return row < batch ? row : -1;
  if (row < starts[0] || row >= starts[batch]) return -1;
  int lo = 0, hi = batch;  // starts[lo] <= row < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Position of `row` (of sequence b) in its sequence.
__device__ __forceinline__ int position_of(const Paged &c, const int32_t *starts, int b, int row) {
  const int len = max(c.lens[b], 0);
  return starts ? len - starts[b + 1] + row : len - 1;
}

// Byte offset of eight rows from `key` on in their page: two 32 x 32 products.
struct PageRows {
  uint32_t page_bytes, row_bytes, slot_mask, n_pages;
  template <typename T>
  __device__ __forceinline__ static PageRows of(const Paged &c) {
    return PageRows{(uint32_t)(c.page_stride * sizeof(T)), (uint32_t)(c.row_stride * sizeof(T)), (1u << c.shift) - 1,
                    (uint32_t)c.n_pages};
  }
  __device__ __forceinline__ bool there(int id) const { return (uint32_t)id < n_pages; }
  __device__ __forceinline__ uint64_t at(int id, int key) const {  // (no page: page 0's rows)
    return (uint64_t)(there(id) ? (uint32_t)id : 0u) * page_bytes + (uint64_t)((uint32_t)key & slot_mask) * row_bytes;
  }
};
// How a pool holds its rows: a lane's 16 bytes of products' operands (piece) and two
// elements (pair) as they are loaded, and as they are used.  PlainPages: as they stand.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename E>
struct PlainPages {
  typedef E T;
  typedef u32x4 Raw;
  typedef float2 Pair;  // (fp32)
  static constexpr bool kScaled = false;
  // (kScaled: where the scales of KV head g's keys, or values, lie, and what a lane loads of them)
  __device__ __forceinline__ const uint8_t *scales(int, bool) const { return nullptr; }
  __device__ __forceinline__ int scale(const uint8_t *, const PageRows &, int, int) const { return 0; }
  __device__ __forceinline__ int scale_bits(int) const { return 0; }
  __device__ __forceinline__ u32x4 piece(Raw x, int) const { return x; }
  __device__ __forceinline__ float2 pair(Pair x, int) const { return x; }
  // element `lane` of a value's row, key k of page id
  __device__ __forceinline__ float value(const PageRows &rows, const char *Vg, int, int id, int k, int lane) const {
    return Elem<E>::load((const E *)(Vg + rows.at(id, k)) + lane);
  }
};
// table entries are read as scalars
typedef const __attribute__((address_space(4))) char *scalar_bytes;
typedef const __attribute__((address_space(4))) int32_t *scalar_ints;

// (cos, sin) of an angle in turns, reduced to an eighth of a turn before it is rounded to 32 bits.
__device__ __forceinline__ float2 cos_sin(double turns) {
  const double quarter = rint(4.0 * turns);
  float s, c;
  sincospif(2.f * (float)(turns - 0.25 * quarter), &s, &c);
  const int quadrant = (int)((int64_t)quarter & 3);
  const float cq = quadrant & 1 ? -s : c, sq = quadrant & 1 ? c : s;
  return quadrant & 2 ? make_float2(-cq, -sq) : make_float2(cq, sq);
}

// Rotates the pairs of a 16-byte piece; cs: (cos, sin) of its first pair on.
template <typename T>
__device__ __forceinline__ u32x4 rotate(u32x4 x, const float2 *cs);
template <>
__device__ __forceinline__ u32x4 rotate<float>(u32x4 x, const float2 *cs) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float a = __uint_as_float(x[2 * i]), b = __uint_as_float(x[2 * i + 1]);
    const float2 t = cs[i];
    y[2 * i] = __float_as_uint(a * t.x - b * t.y);
    y[2 * i + 1] = __float_as_uint(a * t.y + b * t.x);
  }
  return y;
}
template <>
__device__ __forceinline__ u32x4 rotate<bf16_t>(u32x4 x, const float2 *cs) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(x[i] << 16), b = __uint_as_float(x[i] & 0xffff0000u);
    const float2 t = cs[i];
    y[i] = (uint32_t)f32_to_bf16(a * t.x - b * t.y) | ((uint32_t)f32_to_bf16(a * t.y + b * t.x) << 16);
  }
  return y;
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bf16x4 lds_tr16(const bf16_t *p) {
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4 *)(__attribute__((address_space(3))) void *)p);
  return __builtin_bit_cast(bf16x4, r);
}
// The same of bytes: of eight rows, two lanes each, a lane gets one column.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 lds_tr8(const uint8_t *p) {
  const i32x2 r = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) i32x2 *)(__attribute__((address_space(3))) void *)p);
  return __builtin_bit_cast(u32x2, r);
}

// Counts the caller in as one of n on a pair of 64-bit words and says whether
// it is the last.  The first word holds kArrive between launches and counts up
// from it.  Anything else there (memory that nobody has counted in yet) sends
// every caller of the launch to the second word, where a count starts under
// the launch's tag.  A finished count leaves kArrive and 0, so neither fresh
// memory nor a replayed graph needs a clearing pass.
constexpr unsigned long long kArrive = 0x5bd1e995a93c71d4ull;
__device__ __forceinline__ bool arrive_last(unsigned long long *word, int n, unsigned long long tag) {
  unsigned long long old =
      __hip_atomic_fetch_add(word, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) - kArrive;
  bool last = old == (unsigned long long)(n - 1);
  if (old >= (unsigned long long)n) {
    old = __hip_atomic_load(word + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    while (old >> 16 != tag &&
           !__hip_atomic_compare_exchange_strong(word + 1, &old, tag << 16, __ATOMIC_RELAXED,
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) {
    }
    old = __hip_atomic_fetch_add(word + 1, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = (int)(old & 0xffff) == n - 1;
    if (last) __hip_atomic_store(word + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (last) __hip_atomic_store(word, kArrive, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last;
}

// Two floats through to memory, past the caches (another workgroup, on another
// XCD, reads them in the same launch), and back.
__device__ __forceinline__ void put2(float *p, float a, float b) {
  const unsigned long long v = (unsigned long long)__float_as_uint(a) | ((unsigned long long)__float_as_uint(b) << 32);
  __hip_atomic_store((unsigned long long *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__device__ __forceinline__ float2 get2(const float *p) {
  const unsigned long long v =
      __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// ----------------------------------------------------- decode, over pages
constexpr int kMaxRows = 16;   // query heads of a KV head that one workgroup serves
constexpr int kHold = HD + 4;  // floats of a part's row in LDS: a record's, 16-byte aligned
constexpr int kHoldRows = 160; // rows of LDS for the waves' parts of sequences
constexpr int kShareMin = 4;   // tiles of a share at least
constexpr int kMergeBatch = 16;  // records read at once

struct DecodeParams {
  AttnParams a;
  float *ws;                        // records: [bins][2][columns][rows][kRec]
  unsigned long long *arrive_end;   // two arrival words per (sequence, column) below it
  unsigned long long tag;           // the launch's 48-bit tag
  int bins, hblocks, columns, k0;   // k0: keys below it are not this kernel's
  // not null: nothing is added or written here.  A sequence that lies in one share leaves
  // its record in parts [batch][n_heads][kRec], a cut one its pieces' in ws, and either says
  // where in cuts [batch][columns]: its number of pieces << 16 | its first bin.
  float *parts;
  int *cuts;
};

// A tile of keys as a wave loads it: four 16-byte loads per lane of K and four
// of V, LPR lanes a row: whole rows, 1 KB of a head-major page an instruction
// (loads straight into the products' operands, 16 rows of 64 bytes an
// instruction, streamed a third slower).  P: pitch of a row in LDS, elements
// (144 and 272 bytes: the fragment reads below spread over the banks).
template <typename T> struct DecTile;
template <> struct DecTile<bf16_t> { static constexpr int TK = 32, LPR = 8, P = HD + 8; };
template <> struct DecTile<float> { static constexpr int TK = 16, LPR = 16, P = HD + 4; };

// The batch's tiles, sequences in order, are dealt in equal shares to the
// workgroups of a column (a KV head, or up to 16 of its query heads), so that
// any mix of lengths keeps every compute unit streaming to the end.  A
// workgroup's four waves take its share's tiles in turn, across the borders of
// sequences, with the loads of the next tiles and the table entries of the one
// after them in flight; no barrier between them.  A wave leaves its part of
// each sequence (running maximum, sum, accumulator) in LDS; when the share, or
// as many sequences as LDS has room for, are through, the workgroup adds the
// waves' parts.  A sequence that lies in one share is then written; of one cut
// between shares each workgroup leaves a record in the workspace and counts
// itself in, and the last to arrive adds the records, in the order of the keys,
// and writes the output: one launch, and the same bits whoever arrives last.
//
// Per tile, with the query heads as columns of the products:
//   S^T[key][head] = K . Q^T,  O^T[d][head] += V^T . P^T
// on v_mfma_f32_16x16x32_bf16 (bf16 probabilities, the products' operands: off by at most
// 2^-8 each; outputs 0.0023 off 64 bits in the mean, 0.0017 of it their own rounding)
// or v_mfma_f32_16x16x4_f32; a lane holds its 8 (4) keys' scores of one head,
// which are the second product's operand as they stand.  Bound by memory: 64
// caches of 512..4096 keys (32 and 4 heads) 33 us, 4.6 TB/s; three of 34763 to
// 131072 49 us, 5.1 TB/s, a copy's rate.  One of 640 fp32 keys 8.3 us: launch,
// lengths, table, keys and the merge's round trip, one after another.
template <typename T>
struct DecodeLds {
  T k[4][DecTile<T>::TK * DecTile<T>::P];
  T v[4][DecTile<T>::TK * DecTile<T>::P];
  float hold[kHoldRows * kHold];
  int last_in[2];
};
template <typename T, class Src = PlainPages<T>>
__device__ __forceinline__ void decode_body(const DecodeParams &p, DecodeLds<T> &lds, int block,
                                            const Src &src = Src{}) {
  using Ti = DecTile<T>;
  using E = typename Src::T;  // the pools' elements
  constexpr bool BF = sizeof(T) == 2;
  constexpr int TK = Ti::TK, LPR = Ti::LPR, RPI = 64 / LPR, VEC = HD / LPR, P = Ti::P;
  constexpr int NS = TK / 16;  // 16-key score tiles
  constexpr int NQ = BF ? 2 : 4;
  float *const hold = lds.hold;

  const Paged &c = p.a.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, grp = lane >> 4;
  const int bin = block / p.columns, col = block - bin * p.columns;
  const int g = col / p.hblocks, hb = col - g * p.hblocks;
  const int rows = min(kMaxRows, p.a.group - kMaxRows * hb), head0 = g * p.a.group + kMaxRows * hb;
  const int room = kHoldRows / (4 * rows);  // sequences that LDS has room for
  // the first tile begins at a multiple of the smallest page, so that eight rows
  // of a tile from a multiple of eight on lie in one page
  const int k0 = p.k0 & -8;
  auto clamp_len = [&](int n) { return max(min(n, c.cap), 0); };
  auto tiles_of = [&](int len) { return len > p.k0 ? (int)((uint32_t)(len - k0 + TK - 1) / TK) : 0; };

  // ---- the share: every wave scans the lengths for itself, a run of
  // `per` sequences a lane
  const int per = (c.batch + 63) >> 6;
  int own, some = 0;
  auto length_of = [&](int b) __attribute__((always_inline)) {
    const int n = c.lens[min(b, c.batch - 1)];
    return b < c.batch ? clamp_len(n) : 0;
  };
  if (per == 1) {
    some = length_of(lane);
    own = tiles_of(some);
  } else {
    own = 0;
    for (int i = 0; i < per; i += 8) {
      int n[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) n[j] = c.lens[min(lane * per + i + j, c.batch - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        own += i + j < per && lane * per + i + j < c.batch ? tiles_of(clamp_len(n[j])) : 0;
    }
  }
  const int upto = wave_scan(own);
  const int total = __builtin_amdgcn_readlane(upto, 63);
  const int share =
      __builtin_amdgcn_readfirstlane(max((int)((uint32_t)(total + p.bins - 1) / (uint32_t)p.bins), kShareMin));
  const int pos0 = (int)min((int64_t)bin * share, (int64_t)total), n_wg = min(share, total - pos0);

  struct Window {  // 64 lengths from sequence b0 on, one a lane
    int b0, len;
  };
  auto window = [&](int b) __attribute__((always_inline)) { return Window{b, length_of(b + lane)}; };
  struct Tile {
    int b, t, len, ord;  // tile t of sequence b of len keys, the share's ord-th sequence
  };
  // the sequence behind x's that has a tile (there is one)
  auto next_seq = [&](Tile x, Window &w) __attribute__((always_inline)) {
    int b = x.b + 1;
    for (;;) {
      if (b - w.b0 >= 64) w = window(b);
      const unsigned long long there = __builtin_amdgcn_ballot_w64(tiles_of(w.len) > 0) >> (b - w.b0);
      if (there) {
        b += __builtin_ctzll(there);
        return Tile{b, 0, __builtin_amdgcn_readlane(w.len, b - w.b0), x.ord + 1};
      }
      b = w.b0 + 64;
    }
  };
  auto skip = [&](Tile x, int by, Window &w) __attribute__((always_inline)) {
    x.t += by;
    for (int nt; x.t >= (nt = tiles_of(x.len));) {
      const int t = x.t - nt;
      x = next_seq(x, w);
      x.t = t;
    }
    return x;
  };

  // ---- loads: the RPI rows of a load instruction lie in one page, so that its
  // table entry and address are scalars and a lane's offset to them is fixed
  const int crow = lane / LPR, ccol = (lane % LPR) * VEC;
  const uint32_t off = (uint32_t)((crow * c.row_stride + ccol) * sizeof(E));
  const char *const Kg = (const char *)((const E *)c.k + g * c.head_stride);
  const char *const Vg = (const char *)((const E *)c.v + g * c.head_stride);
  const PageRows page_rows = PageRows::of<E>(c);
  const uint8_t *const sg = src.scales(g, lane & 1);  // (scaled: even lanes K's, odd ones V's; a tile lies in one block)
  // A tile's table entries are read as scalars: they come in their own order,
  // not behind the rows requested before them (as vector loads they held up
  // the next rows: 64 caches of 4096 keys 51 us).
  int ids[4];  // of rows RPI r .. of the tile to load next
  struct Rows {
    typename Src::Raw k[4], v[4];  // the lane's pieces of a tile
    int scale;                     // scaled: the byte of the tile's keys, or values
    int lo, hi;        // keys lo .. hi - 1 of the tile are the sequence's
    int pages;         // bit r: rows RPI r .. have memory (else page 0 is read)
  };
  auto load_ids = [&](const Tile &x) __attribute__((always_inline)) {
    const int b = __builtin_amdgcn_readfirstlane(x.b), key0 = k0 + TK * __builtin_amdgcn_readfirstlane(x.t);
    const int last = __builtin_amdgcn_readfirstlane(x.len) - 1;
    const scalar_bytes row = (scalar_bytes)(c.table + b * c.table_stride);
#pragma unroll
    for (int r = 0; r < 4; ++r) ids[r] = *(scalar_ints)(row + ((uint32_t)(min(key0 + RPI * r, last) >> c.shift) << 2));
  };
  uint64_t at[4];  // byte offsets of the rows
  int at_pages;   // bit r: those rows have memory (else page 0's are read)
  auto locate_rows = [&](const Tile &x) __attribute__((always_inline)) {
    const int key0 = k0 + TK * __builtin_amdgcn_readfirstlane(x.t);
    at_pages = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      at_pages |= page_rows.there(ids[r]) << r;
      at[r] = page_rows.at(ids[r], key0 + RPI * r);
    }
  };
  auto load_rows = [&](Rows &y, const Tile &x) __attribute__((always_inline)) {
    const int key0 = k0 + TK * x.t;
    y.lo = p.k0 - key0;
    y.hi = x.len - key0;
    y.pages = at_pages;
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // streamed once: non-temporal
      y.k[r] = __builtin_nontemporal_load((const typename Src::Raw *)(Kg + at[r] + off));
      y.v[r] = __builtin_nontemporal_load((const typename Src::Raw *)(Vg + at[r] + off));
    }
    if constexpr (Src::kScaled) y.scale = src.scale(sg, page_rows, ids[0], key0);
  };
  T *const kt = lds.k[wave], *const vt = lds.v[wave];
  auto put_rows = [&](u32x4 (&k)[4], u32x4 (&v)[4], const Rows &y, bool masked) __attribute__((always_inline)) {
    if (masked) {  // no key: zeros, whatever lies there (0 times an infinite value is none)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = crow + RPI * r;
        if (row < y.lo || row >= y.hi || !(y.pages >> r & 1)) k[r] = v[r] = u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) *(u32x4 *)(kt + (crow + RPI * r) * P + ccol) = k[r];
#pragma unroll
    for (int r = 0; r < 4; ++r) *(u32x4 *)(vt + (crow + RPI * r) * P + ccol) = v[r];
  };
  auto store_rows = [&](Rows &y, bool masked) __attribute__((always_inline)) {
    if constexpr (Src::kScaled) {
      const int bits = src.scale_bits(y.scale);
      u32x4 k[4], v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        k[r] = src.piece(y.k[r], __builtin_amdgcn_readlane(bits, 0));
        v[r] = src.piece(y.v[r], __builtin_amdgcn_readlane(bits, 1));
      }
      put_rows(k, v, y, masked);
    } else {
      put_rows(y.k, y.v, y, masked);
    }
  };
  // queries: lane holds head l16's elements 8 grp + 32 t .. +7 (bf16), 16 grp .. +15 (fp32)
  u32x4 q[NQ], qn[NQ];
  auto load_q = [&](int b) __attribute__((always_inline)) {
    const T *const qp = (const T *)p.a.q + b * p.a.q_rs + (head0 + min(l16, rows - 1)) * HD;
#pragma unroll
    for (int t = 0; t < NQ; ++t) qn[t] = *(const u32x4 *)(qp + (BF ? 8 * grp + 32 * t : 16 * grp + 4 * t));
  };

  // ---- a tile's arithmetic.  The probabilities are taken against a reference
  // that is the true running maximum only when it was last moved: it moves when
  // a key's weight against it passes 2^16 (or is NaN), which saves the maximum
  // over the lanes and the rescaling of the accumulator for most tiles.
  float mc = -INFINITY, l = 0.f;  // of head l16: reference, log2 units; this lane's keys' sum
  f32x4 o[4];
  const float cl = p.a.cl;
  auto compute = [&](bool masked, int lo, int hi, int pages) __attribute__((always_inline)) {
    f32x4 s[NS];
    if constexpr (BF) {
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const bf16_t *kp = kt + 8 * grp + (16 * u + l16) * P;
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8 *)kp, __builtin_bit_cast(bf16x8, q[0]),
                                                       f32x4{}, 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8 *)(kp + 32),
                                                       __builtin_bit_cast(bf16x8, q[1]), s[u], 0, 0, 0);
      }
    } else {
      const float *kp = kt + 16 * grp + l16 * P;
      f32x4 s2[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {  // four chains
        const f32x4 a = *(const f32x4 *)(kp + 4 * t), b = __builtin_bit_cast(f32x4, q[t]);
        s2[t] = f32x4{};
#pragma unroll
        for (int j = 0; j < 4; ++j) s2[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], s2[t], 0, 0, 0);
      }
      s[0] = (s2[0] + s2[1]) + (s2[2] + s2[3]);
    }
    // s[u][i]: key 16u + 4grp + i of the tile, head l16
    if (masked) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * u + 4 * grp + i;
          if (row < lo || row >= hi || !(pages >> (row / RPI) & 1)) s[u][i] = -INFINITY;
        }
    }
    float e[4 * NS], rs;
    auto weigh = [&](float ref) __attribute__((always_inline)) {
      rs = 0.f;
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[4 * u + i] = __builtin_amdgcn_exp2f(fmaf(s[u][i], cl, -ref));
          rs += e[4 * u + i];
        }
    };
    weigh(mc);  // (no key yet: mc is -inf, and the sum +inf or NaN)
    if (__builtin_amdgcn_ballot_w64(!(rs <= 65536.f)) != 0) {
      float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
      if constexpr (NS > 1) mx = fmaxf(mx, fmaxf(fmaxf(s[NS - 1][0], s[NS - 1][1]), fmaxf(s[NS - 1][2], s[NS - 1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(mc, mx * cl);
      const float ref = m_new == -INFINITY ? 0.f : m_new;  // no key above -inf yet: weights 0
      const float alpha = __builtin_amdgcn_exp2f(mc - ref);
      mc = m_new;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
      weigh(ref);
    }
    l += rs;
    if constexpr (BF) {
      bf16x8 pb;
#pragma unroll
      for (int i = 0; i < 8; ++i) pb[i] = (__bf16)e[i];
      // V^T: slot j of lane (grp, l16) is V[key 16(j/4) + 4grp + j%4][16dt + l16]
      const bf16_t *vp = vt + (4 * grp + (l16 >> 2)) * P + 4 * (l16 & 3);
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const bf16x4 x = lds_tr16(vp + 16 * dt), y = lds_tr16(vp + 16 * P + 16 * dt);
        const bf16x8 a = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb, o[dt], 0, 0, 0);
      }
    } else {
      // k slot grp of step i is key 4grp + i; row r of product dt is d = 4r + dt
      f32x4 a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = *(const f32x4 *)(vt + (4 * grp + i) * P + 4 * l16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][dt], e[i], o[dt], 0, 0, 0);
    }
  };

  // ---- results: two elements of a head's row a thread
  auto write2 = [&](int b, int h, int d, float x, float y, float ref, float sum) __attribute__((always_inline)) {
    if (p.parts) {  // one part of the row: left for the launch that adds them
      float *const r = p.parts + ((int64_t)b * p.a.n_heads + head0 + h) * kRec;
      *(float2 *)(r + d) = make_float2(x, y);
      if (d == 0) *(float2 *)(r + HD) = make_float2(ref, sum);
      return;
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    T *const op = (T *)p.a.o + b * p.a.o_rs + (head0 + h) * HD + d;
    if constexpr (BF)
      *(uint32_t *)op = (uint32_t)f32_to_bf16(x * inv) | ((uint32_t)f32_to_bf16(y * inv) << 16);
    else
      *(float2 *)op = make_float2(x * inv, y * inv);
  };
  // row h of the record of a sequence's piece in bin `at` (a bin has two: the end
  // of a sequence begun before it, and the start of one, begun in bin0, that goes on)
  auto record = [&](int at, int bin0, int h) __attribute__((always_inline)) {
    return p.ws + ((((int64_t)at * 2 + (at == bin0)) * p.columns + col) * kMaxRows + h) * kRec;
  };
  // a cut sequence: its first bin and the number of its pieces, one a bin
  struct Cut {
    int b, bin0, pieces;
  };
  Cut cuts[2] = {{0, 0, 0}, {0, 0, 0}};  // one that began before the share, one that goes on

  if (n_wg > 0) {
    Tile x;       // the wave's tile (its loads are in flight)
    Window w;     // of the tiles to come
    Tile seg;     // the next sequence whose parts are to be added (its t: 0), ...
    Window sw;
    int first;    // ... and the position of its first tile
    {
      const int src = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > pos0));
      first = __builtin_amdgcn_readlane(upto - own, src);
      if (per == 1) {
        w = Window{0, some};
        seg = Tile{src, 0, __builtin_amdgcn_readlane(some, src), 0};
      } else {
        w = window(src * per);
        for (;;) {  // (one round unless a lane's run is longer than a window)
          const int t = tiles_of(w.len), up = wave_scan(t);
          const unsigned long long hit = __builtin_amdgcn_ballot_w64(first + up > pos0);
          if (hit) {
            const int i = __builtin_ctzll(hit);
            first += __builtin_amdgcn_readlane(up - t, i);
            seg = Tile{w.b0 + i, 0, __builtin_amdgcn_readlane(w.len, i), 0};
            break;
          }
          first += __builtin_amdgcn_readlane(up, 63);
          w = window(w.b0 + 64);
        }
      }
      sw = w;
    }
    const int n = n_wg > wave ? (n_wg - wave + 3) / 4 : 0;  // the wave's tiles
    Rows buf;
    Tile ahead[3];  // the wave's tiles i .. i + 2 (the last one again past the end)
    bool fresh = true;
    if (n > 0) {
      x = seg;
      x.t = pos0 - first;
      if (wave) x = skip(x, wave, w);
      load_q(x.b);
      load_ids(x);
      ahead[0] = x;
      ahead[1] = 1 < n ? skip(x, 4, w) : x;
      locate_rows(x);
      load_rows(buf, x);
      load_ids(ahead[1]);
      ahead[2] = 2 < n ? skip(ahead[1], 4, w) : ahead[1];
    }
    int i = 0, base = 0;  // base: the sequence in the first place of LDS
    auto step = [&]() __attribute__((always_inline)) {
      locate_rows(ahead[1]);
      const int lo = buf.lo, hi = buf.hi, pages = buf.pages;
      const bool masked = lo > 0 || hi < TK || pages != 15;
      // a wave's LDS instructions execute in order, so its tile needs no
      // barrier; wave_barrier keeps the compiler from moving them across
      __builtin_amdgcn_wave_barrier();
      store_rows(buf, masked);
      __builtin_amdgcn_wave_barrier();
      if (fresh) {
#pragma unroll
        for (int t = 0; t < NQ; ++t) q[t] = qn[t];
        mc = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32x4{};
      }
      x = ahead[0];
      const bool ends = i + 1 == n || ahead[1].b != x.b;
      if (i + 1 < n) {
        load_rows(buf, ahead[1]);
        if (ends) load_q(ahead[1].b);
        load_ids(ahead[2]);
        ahead[0] = ahead[1];
        ahead[1] = ahead[2];
        if (i + 3 < n) ahead[2] = skip(ahead[2], 4, w);
      }
      compute(masked, lo, hi, pages);
      if (ends) {
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (l16 < rows) {
          float *const h = hold + (((x.ord - base) * 4 + wave) * rows + l16) * kHold;
#pragma unroll
          for (int j = 0; j < 4; ++j)  // bf16: o[j] is d = 16j + 4grp ..; fp32: o[0..3][j] is d = 16grp + 4j ..
            *(f32x4 *)(h + (BF ? 16 * j + 4 * grp : 16 * grp + 4 * j)) =
                BF ? o[j] : f32x4{o[0][j], o[1][j], o[2][j], o[3][j]};
          if (grp == 0) *(float2 *)(h + HD) = make_float2(mc, l);
        }
      }
      fresh = ends;
      ++i;
    };
    for (;;) {
      while (i < n && ahead[0].ord < base + room) step();
      __syncthreads();
      bool more = true;
      for (int place = 0; more && place < room; ++place) {
        const int nt = tiles_of(seg.len), i0 = max(first - pos0, 0), i1 = min(first + nt - pos0, n_wg);
        const int bin0 = (int)((uint32_t)first / (uint32_t)share);
        const int pieces = (int)((uint32_t)(first + nt - 1) / (uint32_t)share) - bin0 + 1;
        if (p.parts) {
          if (tid == 0 && bin0 == bin) p.cuts[seg.b * p.columns + col] = pieces << 16 | bin0;
        } else if (pieces > 1) {
          cuts[bin0 == bin] = Cut{seg.b, bin0, pieces};
        }
        for (int k = tid; k < rows * (HD / 2); k += 256) {
          const int h = k / (HD / 2), d = 2 * (k % (HD / 2));
          const float *r = hold + (place * 4 * rows + h) * kHold;
          float2 ml[4];
          float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            ml[v] = make_float2(-INFINITY, 0.f);  // no tile of it
            if (((v - i0) & 3) < i1 - i0) ml[v] = *(const float2 *)(r + v * rows * kHold + HD);
            M = fmaxf(M, ml[v].x);
          }
          const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            if (((v - i0) & 3) >= i1 - i0) continue;
            const float f = __builtin_amdgcn_exp2f(ml[v].x - Mu);
            const float2 a = *(const float2 *)(r + v * rows * kHold + d);
            L = fmaf(ml[v].y, f, L);
            A0 = fmaf(a.x, f, A0);
            A1 = fmaf(a.y, f, A1);
          }
          if (pieces == 1) {
            write2(seg.b, h, d, A0, A1, M, L);
          } else {
            float *const to = record(bin, bin0, h);
            put2(to + d, A0, A1);
            if (d == 0) put2(to + HD, M, L);
          }
        }
        first += nt;
        more = first < pos0 + n_wg;
        if (more) seg = next_seq(seg, sw);
      }
      if (!more) break;
      __syncthreads();  // the places are free again
      base += room;
    }
    if (cuts[0].pieces | cuts[1].pieces) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the records' stores have reached memory
      __syncthreads();
      if (tid < 2) {
        const Cut u = tid ? cuts[1] : cuts[0];
        lds.last_in[tid] =
            u.pieces && arrive_last(p.arrive_end - 2 * ((int64_t)u.b * p.columns + col + 1), u.pieces, p.tag);
      }
      __syncthreads();
#pragma unroll 1
      for (int side = 0; side < 2; ++side) {
        if (!lds.last_in[side]) continue;
        const Cut u = side ? cuts[1] : cuts[0];
        for (int k = tid; k < rows * (HD / 2); k += 256) {
          const int h = k / (HD / 2), d = 2 * (k % (HD / 2));
          float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
          for (int n0 = 0; n0 < u.pieces; n0 += kMergeBatch) {
            float2 ml[kMergeBatch], a[kMergeBatch];
#pragma unroll
            for (int v = 0; v < kMergeBatch; ++v) {
              const float *const r = record(u.bin0 + min(n0 + v, u.pieces - 1), u.bin0, h);
              ml[v] = get2(r + HD);
              a[v] = get2(r + d);
            }
            float mx = M;
#pragma unroll
            for (int v = 0; v < kMergeBatch; ++v) mx = n0 + v < u.pieces ? fmaxf(mx, ml[v].x) : mx;
            const float mu = mx == -INFINITY ? 0.f : mx, fo = __builtin_amdgcn_exp2f(M - mu);
            L *= fo;
            A0 *= fo;
            A1 *= fo;
#pragma unroll
            for (int v = 0; v < kMergeBatch; ++v) {
              const bool in = n0 + v < u.pieces;  // (a record past the end is never multiplied: it may hold anything)
              const float f = __builtin_amdgcn_exp2f(ml[v].x - mu);
              L = in ? fmaf(ml[v].y, f, L) : L;
              A0 = in ? fmaf(a[v].x, f, A0) : A0;
              A1 = in ? fmaf(a[v].y, f, A1) : A1;
            }
            M = mx;
          }
          write2(u.b, h, d, A0, A1, M, L);
        }
      }
    }
  }
  // sequences without a key
  for (int b = bin; b < c.batch; b += p.bins)
    if (tiles_of(clamp_len(c.lens[b])) == 0)
      for (int k = tid; k < rows * (HD / 2); k += 256) {
        write2(b, k / (HD / 2), 2 * (k % (HD / 2)), 0.f, 0.f, -INFINITY, 0.f);
        if (k == 0 && p.parts) p.cuts[b * p.columns + col] = 1 << 16;
      }
}
// ------------------------------------------------- prefill, over pages
typedef float f32x16 __attribute__((ext_vector_type(16)));

// What the two prefill kernels share: the piece's keys, the rows' limits and
// the scalars of the pages.
struct PieceKeys {
  const int32_t *table;
  int t0, t1;  // its tiles
  int end;     // keys that some row of the unit sees
  int whole;   // keys that every row of the unit sees
  int shift;
  // The table entry of a key (lanes may ask for different ones).  A vector load
  // on purpose: it comes behind the rows requested before it, for which the tile
  // waits anyway, where a scalar load would be waited for with every LDS read.
  __device__ __forceinline__ int entry(int key) const { return table[(uint32_t)(min(key, end - 1) >> shift)]; }
};
template <int R>
__device__ __forceinline__ PieceKeys piece_keys(const PrefillParams &p, const Piece &w) {
  const Paged &c = p.a.c;
  PieceKeys k;
  if (p.prefix_parts) {
    k.end = p.a.prefix_len;
    k.whole = p.a.prefix_len;  // unless a sequence is shorter
    int h;
    const int to = min(token_of(w, p.a.inv_group, p.a.group, R - 1, h) + 1, w.rows);
    for (int t = w.tok0 + (int)(threadIdx.x & 63); t < to; t += 64) k.whole = min(k.whole, max(c.lens[t], 0));
    k.whole = wave_min(k.whole);
    k.table = p.a.prefix_pages;
  } else {
    int h;
    const int tokens = min(__builtin_amdgcn_readfirstlane(token_of(w, p.a.inv_group, p.a.group, R - 1, h)) + 1, w.rows);
    k.end = min(max(w.last - w.rows + tokens, 0), c.cap);
    k.whole = min(max(w.last - w.rows + w.tok0 + 1, 0), c.cap);
    k.table = c.table + w.b * c.table_stride;
  }
  k.end = __builtin_amdgcn_readfirstlane(k.end);
  k.whole = __builtin_amdgcn_readfirstlane(k.whole);
  part_of((k.end + 31) >> 5, w, k.t0, k.t1);
  k.shift = c.shift;
  return k;
}
// keys that token t of the piece's sequence sees
__device__ __forceinline__ int key_limit(const PrefillParams &p, const Piece &w, int t) {
  return p.prefix_parts ? min(max(p.a.c.lens[t], 0), p.a.prefix_len)
                        : min(max(w.last - w.rows + t + 1, 0), p.a.c.cap);
}
// A tile's row sums come from the matrix cores against a 0/1 selector, which
// multiplies a lane's row with 1 and the row 16 away with 0: not a row's own sum
// where that one's probabilities are NaN (its query, or a key that it alone of
// the two sees).  A sum that is NaN always leads into a fixup, and there the sums
// are formed from the lane's own probabilities.  (Choosing between the two there
// cost registers: 200 sequences behind 16387 keys 76 -> 89 us.)
__device__ __forceinline__ float own_sums(const bf16x8 (&pb)[2]) {
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pb[u][j], pb[u][j + 1]}, bf16x2{(__bf16)1.f, (__bf16)1.f}, sum, false);
  return sum + __shfl_xor(sum, 32, 64);
}
// Infinite and NaN values of keys that not every row of a workgroup sees: a row
// that does not see one weighs it with 0, and 0 times it is not 0.  They are
// staged as zeros (tame), and if there were any, add_odd() puts each, as it
// is, into the rows that see it when the tiles are through: nothing of this in
// the loop.  (A sum with one of them in it is infinite or NaN whatever its weight;
// of a weight of 0 the products of the tiles that all rows see make NaN, this leaves
// it infinite.)
template <typename T>
__device__ __forceinline__ bool tame(u32x4 &x) {  // true: there was one
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) {
      const bool lo = (x[j] & 0x7f80u) == 0x7f80u, hi = (x[j] & 0x7f800000u) == 0x7f800000u;
      x[j] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
      odd |= lo || hi;
    } else {
      const bool b = (x[j] & 0x7f800000u) == 0x7f800000u;
      x[j] = b ? 0u : x[j];
      odd |= b;
    }
  }
  return odd;
}
// o[n], n < N: the lane's rows' accumulators in the order that d_of(i) gives
// the elements of; limit[n]: keys that the rows see; keys from .. to - 1, whose
// values' elements value(page, key, lane) gives.
template <int N, class V, class D>
__device__ __forceinline__ void add_odd(const PieceKeys &keys, const PageRows &rows, V &&value, int from, int to,
                                        f32x16 (&o)[N][2], const int (&limit)[N], D &&d_of) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int k = from; k < to; ++k) {
    const int id = __builtin_amdgcn_readfirstlane(keys.entry(k));
    if (!rows.there(id)) continue;
    const float v = value(id, k, lane);
    unsigned long long odd = __builtin_amdgcn_ballot_w64(!(fabsf(v) < INFINITY));
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int d = __builtin_ctzll(odd);
      const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), d));
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (d_of(i) == d && k < limit[n]) o[n][i >> 4][i & 15] += x;
    }
  }
}

// The end of a piece, all its waves: `sum(row, d, ml)` gives NV consecutive
// elements of a row's accumulator and its (reference in log2 units, sum); a
// whole unit is written, of a cut one a record is left and the last part to
// arrive adds them, in the order of the keys, and writes.
template <typename T, int R, int THREADS, class F>
__device__ __forceinline__ void finish_piece(const PrefillParams &p, const Piece &kept, int *last_in, F &&sum) {
  const Piece w = kept;
  constexpr int TPR = THREADS / R, NV = HD / TPR;  // threads a row, elements a thread
  static_assert(THREADS % R == 0 && NV % 4 == 0, "whole quads");
  const int tid = threadIdx.x, row = tid / TPR, d0 = (tid % TPR) * NV;
  int h;
  const int t = token_of(w, p.a.inv_group, p.a.group, row, h);
  h += w.g * p.a.group;
  const bool there = t < w.rows;
  float acc[NV];
  float2 ml = sum(row, d0, acc);
  auto write = [&]() __attribute__((always_inline)) {
    if (!there) return;
    const float inv = ml.y > 0.f ? 1.0f / ml.y : 0.f;
    T *const op = (T *)p.a.o + (int64_t)(w.row0 + t) * p.a.o_rs + h * HD + d0;
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t lo = (uint32_t)f32_to_bf16(acc[i] * inv) | ((uint32_t)f32_to_bf16(acc[i + 1] * inv) << 16);
        const uint32_t hi = (uint32_t)f32_to_bf16(acc[i + 2] * inv) | ((uint32_t)f32_to_bf16(acc[i + 3] * inv) << 16);
        *(uint2 *)(op + i) = make_uint2(lo, hi);
      } else {
        *(float4 *)(op + i) = make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
      }
    }
  };
  if (w.parts == 1 && !p.prefix_parts) return write();
  if (p.prefix_parts) {
    if (!there) return;
    float *const r = p.ws + (((int64_t)w.slot + (int64_t)w.part * p.a.c.n_kv_heads) * R + row) * kRow;
#pragma unroll
    for (int i = 0; i < NV; i += 4) *(float4 *)(r + d0 + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    if (d0 == 0) *(float2 *)(r + HD) = ml;
    return;
  }
  const int64_t step = (int64_t)p.a.c.n_kv_heads * R * kRec;
  float *const first = p.ws + (int64_t)w.slot * R * kRec + 2 * row;  // pair k: 2 R k floats on
  if (there) {
    float *const r = first + w.part * step;
#pragma unroll
    for (int i = 0; i < NV; i += 2) put2(r + R * (d0 + i), acc[i], acc[i + 1]);
    if (d0 == 0) put2(r + R * HD, ml.x, ml.y);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the record has reached memory
  __syncthreads();
  if (tid == 0) *last_in = arrive_last(p.arrive_end - 2 * ((int64_t)w.slot + 1), w.parts, p.tag);
  __syncthreads();
  if (!*last_in || !there) return;
  ml = make_float2(-INFINITY, 0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  constexpr int MB = NV >= 32 ? 1 : 4;  // records read at once
  for (int n0 = 0; n0 < w.parts; n0 += MB) {
    float2 m2[MB], a[MB][NV / 2];
#pragma unroll
    for (int v = 0; v < MB; ++v) {
      const float *const r = first + min(n0 + v, w.parts - 1) * step;
      m2[v] = get2(r + R * HD);
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) a[v][i] = get2(r + R * (d0 + 2 * i));
    }
#pragma unroll
    for (int v = 0; v < MB; ++v) {
      const bool in = n0 + v < w.parts;
      const float mn = in ? fmaxf(ml.x, m2[v].x) : ml.x, mu = mn == -INFINITY ? 0.f : mn;
      const float fo = __builtin_amdgcn_exp2f(ml.x - mu), fn = __builtin_amdgcn_exp2f(m2[v].x - mu);
      auto add = [&](float s, float x) { return in ? fmaf(x, fn, s * fo) : s; };
      ml.y = add(ml.y, m2[v].y);
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        acc[2 * i] = add(acc[2 * i], a[v][i].x);
        acc[2 * i + 1] = add(acc[2 * i + 1], a[v][i].y);
      }
      ml.x = mn;
    }
  }
  write();
}

// bf16.  HW waves of 32 rows share each staged K/V tile, KW such parts take a
// piece's tiles in turn; their (m, l, O) meet in LDS.  Per wave and tile
//   S^T[key][row] = K . Q^T  (v_mfma_f32_32x32x16_bf16: 16 keys of one row a lane)
//   O^T[d][row] += V^T . P^T, whose operand is P^T as the scores left it
// (bf16 probabilities, the matrix cores' operands: off by at most 2^-8 each, in the row sum too, which the
// matrix cores form against a 0/1 selector).  Weights are taken against a
// reference that moves to the true maximum only when a tile's sum passes 2^16.
// <4,1>: 7 prompts of 165..1500 tokens 50 us (543 TFLOP/s), VALU 58% and LDS 52%
// busy, the rest the units' start and end; <1,4>: 256 rows each behind 2697, 5444
// and 8192 keys 62 us (565), the LDS port 99% busy, but units of 64 rows, with
// half its traffic and two waves a SIMD in place of three, took 6% longer.
constexpr float kSumLimit = 65536.f, kMoveLog2 = 8.f;
template <int HW, int KW>
struct PrefillLds {
  static constexpr int W = HW * KW;
  static constexpr int KP = HD + 8;   // K row pitch, elements (144 B: conflict-free b128 rows)
  static constexpr int VP = HD + 16;  // V row pitch (160 B: conflict-free transpose reads)
  static constexpr int KT = 32 * KP, VT = 32 * VP;
  static constexpr int NB = HW > 1 ? 2 : 1;        // tile buffers (HW == 1: a wave's tile is its own)
  static constexpr int OP = HD + 4, OT = 32 * OP;  // a wave's O at the end, floats
  static constexpr int RING = KW * NB * (KT + VT);
  bf16_t smem[RING > 2 * W * OT ? RING : 2 * W * OT];
  float red_m[W][32], red_l[W][32];
  unsigned char __attribute__((aligned(4))) chunk_ok[KW][2][4];
  int odd[W];
  Piece piece;  // kept here across the tiles, not in scalar registers
  int last_in;
};
template <int HW, int KW, class Src = PlainPages<bf16_t>>
__device__ __forceinline__ void prefill_bf16_body(const PrefillParams &p, PrefillLds<HW, KW> &lds, int block,
                                                  const Src &src = Src{}) {
  typedef typename Src::T T;
  using L = PrefillLds<HW, KW>;
  constexpr int W = L::W, R = 32 * HW, KP = L::KP, VP = L::VP, KT = L::KT, VT = L::VT, NB = L::NB;
  constexpr int OP = L::OP, OT = L::OT;
  bf16_t *const smem = lds.smem;
  auto &red_m = lds.red_m, &red_l = lds.red_l;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hw = wave % HW, kw = wave / HW;
  const int r32 = lane & 31, hf = lane >> 5;
  Piece w;
  if (!find_piece<R>(p, block, w)) return;
  if (tid == 0) lds.piece = w;
  const Paged &c = p.a.c;
  const PieceKeys keys = piece_keys<R>(p, w);
  const float cl = p.a.cl;
  const int ni = (keys.t1 - keys.t0 + KW - 1) / KW;  // steps: tile t0 + kw + KW*i each

  // this lane's row
  int head;
  const int tok = token_of(w, p.a.inv_group, p.a.group, 32 * hw + r32, head);
  const bool there = tok < w.rows;
  const int limit = there ? key_limit(p, w, tok) : keys.end;  // (0: a fix of its reference in every tile)
  const int all_see = wave_min(there ? limit : 0x7fffffff);  // keys that all the wave's rows see
  bf16x8 qreg[4];
  {
    const bf16_t *const qp = (const bf16_t *)p.a.q + (int64_t)(w.row0 + (there ? tok : 0)) * p.a.q_rs +
                             (w.g * p.a.group + (there ? head : 0)) * HD + 8 * hf;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      qreg[t] = *(const bf16x8 *)(qp + 16 * t);
      if (!there) qreg[t] = bf16x8{};
    }
  }

  // staging: the HW waves of a key part share its tile, NC chunks of 8 rows
  // each (16-byte piece lane % 8 of row lane / 8); a chunk's rows lie in one page
  constexpr int NC = 4 / HW;
  const int crow = lane >> 3, ccol = (lane & 7) * 8;
  const PageRows rows = PageRows::of<T>(c);
  const uint32_t off = crow * rows.row_bytes + ccol * sizeof(T);
  const char *const Kg = (const char *)((const T *)c.k + w.g * c.head_stride);
  const char *const Vg = (const char *)((const T *)c.v + w.g * c.head_stride);
  typename Src::Raw kr[NC], vr[NC];
  // lanes j and NC + j (mod 2 NC): the scales of chunk j's keys and values, of the tile loaded last
  int sc = 0;
  const uint8_t *const sg = src.scales(w.g, lane & NC);
  int entry = 0;  // lane j (mod NC): of chunk j of the tile to load next
  bool any_odd = false;
  int chunks_next = 0;  // bit j: the wave's chunk j of the tile loaded last has memory
  auto key_of = [&](int i) { return 32 * (keys.t0 + kw + KW * i); };
  auto load_ids = [&](int i) __attribute__((always_inline)) {
    entry = keys.entry(key_of(i) + 8 * (NC * hw + (lane & (NC - 1))));
  };
  auto gload = [&](int i) __attribute__((always_inline)) {
    uint32_t o32 = off;
    asm volatile("" : "+v"(o32));  // a scalar base and this offset, not a sum of pointers kept in registers
    // Four chunks: a lane forms its chunk's offset (in scalars, chunk by chunk, 60 instructions in
    // the wave's way: 256 rows behind 4096 keys 28.1 us where this takes 26.5).
    uint64_t mine = 0;
    if constexpr (NC > 1) {
      mine = rows.at(entry, key_of(i) + 8 * (NC * hw + (lane & (NC - 1))));
      chunks_next = (int)__builtin_amdgcn_ballot_w64(rows.there(entry)) & ((1 << NC) - 1);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      uint64_t at;
      if constexpr (NC > 1) {
        at = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, j) |
             (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(mine >> 32), j) << 32;
      } else {
        const int id = __builtin_amdgcn_readlane(entry, 0);
        chunks_next = rows.there(id);
        at = rows.at(id, key_of(i) + 8 * hw);
      }
      kr[j] = *(const typename Src::Raw *)(Kg + at + o32);
      vr[j] = *(const typename Src::Raw *)(Vg + at + o32);
    }
    if constexpr (Src::kScaled) sc = src.scale(sg, rows, entry, key_of(i) + 8 * (NC * hw + (lane & (NC - 1))));
  };
  // (HW > 1: the waves that share a tile tell each other of their chunks through LDS)
  auto lstore = [&](int i) __attribute__((always_inline)) {
    const int key0 = key_of(i), b = NB > 1 ? i & 1 : 0;
    bf16_t *const kd = smem + (kw * NB + b) * (KT + VT), *const vd = kd + KT;
    const int bits = src.scale_bits(sc);
    u32x4 vb[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) vb[j] = src.piece(vr[j], __builtin_amdgcn_readlane(bits, NC + j));
    if (key0 + 32 > keys.end || chunks_next != (1 << NC) - 1) {  // no key: zeros, whatever lies there
#pragma unroll
      for (int j = 0; j < NC; ++j)
        if (!(chunks_next >> j & 1) || key0 + 8 * (NC * hw + j) + crow >= keys.end) vb[j] = u32x4{0, 0, 0, 0};
    }
    if (key0 + 32 > keys.whole) {
      bool odd = false;
#pragma unroll
      for (int j = 0; j < NC; ++j) odd |= tame<bf16_t>(vb[j]);
      any_odd |= __builtin_amdgcn_ballot_w64(odd) != 0;
    }
#pragma unroll
    for (int j = 0; j < NC; ++j)
      *(u32x4 *)(kd + (8 * (NC * hw + j) + crow) * KP + ccol) = src.piece(kr[j], __builtin_amdgcn_readlane(bits, j));
#pragma unroll
    for (int j = 0; j < NC; ++j) *(u32x4 *)(vd + (8 * (NC * hw + j) + crow) * VP + ccol) = vb[j];
    if (HW > 1 && lane == 0) lds.chunk_ok[kw][b][hw] = (unsigned char)chunks_next;
  };

  float l = 0.f, mcv = -INFINITY;  // row sum; reference, log2 units
  f32x16 ow[1][2] = {{f32x16{}, f32x16{}}};
  f32x16 (&o)[2] = ow[0];
  const uint32_t rs_bits = (((lane & 15) >> 2) & 1) == ((lane >> 4) & 1) ? 0x3f803f80u : 0u;
  const int tr_off = (4 * hf + ((lane & 15) >> 2)) * VP + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  // p = exp2(s * cl - mc) as bf16 operands, and the tile's row sum over both half-waves
  auto exps = [&](const f32x16 &s, float mc, bf16x8 (&pb)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[u][j] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[8 * u + j], cl, -mc));
    uint32_t b = rs_bits;
    asm volatile("" : "+v"(b));  // keeps the selector from being hoisted out of the loop
    const bf16x8 sel = __builtin_bit_cast(bf16x8, u32x4{b, b, b, b});
    const f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sel, pb[0], f32x4{}, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(sel, pb[1], d, 0, 0, 0)[0];
  };
  auto fixup = [&](const f32x16 &s, bf16x8 (&pb)[2]) __attribute__((always_inline)) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mt = fmaxf(mcv, mx * cl);  // -inf while nothing is visible
    const bool move = mcv == -INFINITY || mt - mcv > kMoveLog2;
    const float m_new = move ? mt : mcv;
    const float mn = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(mcv - mn);
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    mcv = m_new;
    exps(s, mn, pb);
    return own_sums(pb);
  };

  if (ni > 0) {
    load_ids(0);
    gload(0);
    load_ids(1);
    if (NB > 1) lstore(0);
  }
  if constexpr (NB > 1) __syncthreads();
  for (int i = 0; i < ni; ++i) {
    int pages = chunks_next;  // bit r: rows 8r .. of this tile have memory
    if constexpr (NB == 1) {
      // the wave's own tile: its LDS instructions execute in order, the
      // barriers keep the compiler from moving them across
      __builtin_amdgcn_wave_barrier();
      lstore(i);
      __builtin_amdgcn_wave_barrier();
    }
    gload(i + 1);  // past the range: the last key's page again, not used
    load_ids(i + 2);
    const bf16_t *const kl = smem + (kw * NB + (NB > 1 ? i & 1 : 0)) * (KT + VT), *const vl = kl + KT;
    const int tile = keys.t0 + kw + KW * i, kb = 32 * tile;
    if constexpr (HW > 1) {
      const uint32_t ok = __builtin_amdgcn_readfirstlane(*(const uint32_t *)lds.chunk_ok[kw][i & 1]);
      pages = (ok & 1) | (ok >> 7 & 2) | (ok >> 14 & 4) | (ok >> 21 & 8);
    }
    if (tile < keys.t1) {  // wave-uniform
      f32x16 s = f32x16{};
#pragma unroll
      for (int u = 0; u < 4; ++u)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8 *)(kl + r32 * KP + 16 * u + 8 * hf), qreg[u], s,
                                                    0, 0, 0);
      // V^T fragments: key slot j of 16-key chunk u is key 16u + (j/4)*8 + 4hf + j%4
      bf16x8 va[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          const bf16x4 lo = lds_tr16(vl + 16 * u * VP + tr_off + 32 * dt);
          const bf16x4 hi = lds_tr16(vl + (16 * u + 8) * VP + tr_off + 32 * dt);
          va[u][dt] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
      if (kb + 32 > all_see || pages != 15) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = (e >> 2) * 8 + hf * 4 + (e & 3);
          if (kb + k >= limit || !(pages >> (e >> 2) & 1)) s[e] = -INFINITY;
        }
      }
      bf16x8 pb[2];
      float rs = 0.f;
      bool bad = i == 0;  // the first tile sets the reference
      if (!bad) {
        rs = exps(s, mcv, pb);
        bad = !(rs <= kSumLimit);  // NaN included
      }
      if (__builtin_amdgcn_ballot_w64(bad) != 0) rs = fixup(s, pb);
      l += rs;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[u][dt], pb[u], o[dt], 0, 0, 0);
    }
    if constexpr (NB > 1) {
      lstore(i + 1);
      __syncthreads();
    }
  }

  // every wave scales its O to the key parts' common maximum and writes it to
  // its own share of the LDS as [row][d]
  if (hf == 0) {
    red_m[wave][r32] = mcv;
    red_l[wave][r32] = l;
  }
  if (lane == 0) lds.odd[wave] = any_odd;
  __syncthreads();
  any_odd = false;
#pragma unroll
  for (int v = 0; v < W; ++v) any_odd |= lds.odd[v] != 0;
  float *const ot = (float *)smem;
  float M = red_m[hw][r32];
#pragma unroll
  for (int v = 1; v < KW; ++v) M = fmaxf(M, red_m[v * HW + hw][r32]);
  const float f = mcv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mcv - M);
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] *= f;
  if (any_odd && kw == 0) {
    const int limits[1] = {limit};
    const int g = lds.piece.g;
    add_odd(keys, rows, [&](int id, int k, int i) { return src.value(rows, Vg, g, id, k, i); },
            max(32 * keys.t0, keys.whole & -32), min(32 * keys.t1, keys.end), ow, limits,
            [&](int i) { return 32 * (i >> 4) + 8 * (i >> 2 & 3) + 4 * hf + (i & 3); });
  }
  {
    float *dst = ot + wave * OT + r32 * OP + 4 * hf;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi)
        *(float4 *)(dst + 32 * dt + 8 * gi) =
            make_float4(o[dt][4 * gi], o[dt][4 * gi + 1], o[dt][4 * gi + 2], o[dt][4 * gi + 3]);
  }
  __syncthreads();
  constexpr int NV = R / W;  // = 64 elements over the row's threads
  static_assert(NV * (64 * W / R) == HD, "a row's threads cover it");
  finish_piece<bf16_t, R, 64 * W>(p, lds.piece, &lds.last_in, [&](int row, int d0, float (&acc)[NV]) __attribute__((always_inline)) {
    const int hu = row / 32, r = row % 32;
    float Mr = red_m[hu][r];
#pragma unroll
    for (int v = 1; v < KW; ++v) Mr = fmaxf(Mr, red_m[v * HW + hu][r]);
    const float Mu = Mr == -INFINITY ? 0.f : Mr;
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < KW; ++v) sum += red_l[v * HW + hu][r] * __builtin_amdgcn_exp2f(red_m[v * HW + hu][r] - Mu);
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.f;
#pragma unroll
    for (int v = 0; v < KW; ++v)
#pragma unroll
      for (int i = 0; i < NV; i += 4) {
        const float4 x = *(const float4 *)(ot + (v * HW + hu) * OT + r * OP + d0 + i);
        acc[i] += x.x; acc[i + 1] += x.y; acc[i + 2] += x.z; acc[i + 3] += x.w;
      }
    return make_float2(Mr, sum);
  });
}
// bf16, calls of many rows: 256 rows a unit, two 32-row tiles a wave, so that
// every fragment read from LDS feeds two products, and a software pipeline over
// 32-key tiles: step t issues O += V^T P of tile t - 1 and the scores of tile
// t + 1 on the matrix cores among the exponentials of tile t.  Blocks of 64
// keys in two-deep K and V rings, one barrier a block.  A tile's row sums (from
// the matrix cores) are looked at one step later, when they are long there; only
// if one passes 2^16 does the tile run again from its scores, still at hand,
// against the true maximum.  Tiles that every row of the workgroup sees whole
// run a step without mask code.  8192 rows behind 8192 keys 836 us (829 to 855 from
// card to card), 986 TFLOP/s, 77% of what an 8192^3 library product reaches: VALU
// 61%, matrix cores 55% busy.
constexpr int kBK = 64;  // keys of a block
constexpr int kPipeR = 256;
struct PipeLds {
  static constexpr int KP = HD + 8;   // 144 B: conflict-free b128 fragment reads
  static constexpr int VP = HD + 32;  // 192 B: transpose reads of 8 rows x 64 B in two passes
  static constexpr int KBUF = kBK * KP, VBUF = kBK * VP;
  bf16_t k[2 * KBUF], v[2 * VBUF];
  unsigned char __attribute__((aligned(8))) chunk_ok[4][8];  // block (mod 4): its chunks of 8 rows that have memory
  int limit[kPipeR];  // keys that the rows see
  Piece piece;
  int odd[4], last_in;
};
template <class Src = PlainPages<bf16_t>>
__device__ __forceinline__ void prefill_pipe_body(const PrefillParams &p, PipeLds &lds, int block,
                                                  const Src &src = Src{}) {
  typedef typename Src::T T;
  typedef typename Src::Raw Raw;
  constexpr int RT = 2, R = kPipeR, KP = PipeLds::KP, VP = PipeLds::VP, KBUF = PipeLds::KBUF, VBUF = PipeLds::VBUF;
  bf16_t *const kring = lds.k, *const vring = lds.v;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, hf = lane >> 5;
  Piece w;
  if (!find_piece<R>(p, block, w)) return;
  if (tid == 0) lds.piece = w;
  const Paged &c = p.a.c;
  const float cl = p.a.cl;
  const PieceKeys keys = piece_keys<R>(p, w);  // (its t0, t1 are not used: blocks)
  const int end = keys.end;
  const int nb = (end + kBK - 1) / kBK;
  int blk0, nblk;
  part_of(nb, w, blk0, nblk);
  nblk -= blk0;
  const int first = blk0 * kBK;  // the piece's keys and tiles are counted from here

  // the first block with a page without memory (from it on, steps with masks)
  int gap = nblk + 1;
  for (int key = (first & -(1 << c.shift)) + (lane << c.shift); key < min(first + kBK * (nblk + 1), end); key += 64 << c.shift)
    if ((unsigned)keys.entry(key) >= (unsigned)c.n_pages) gap = min(gap, (key - first) / kBK);
  gap = max(wave_min(gap), 0);

  // this lane's rows: Q^T operands, and the keys that they see
  bf16x8 qreg[RT][4];
  int most = 0, least = 0x7fffffff;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int head;
    const int tok = token_of(w, p.a.inv_group, p.a.group, 32 * (RT * wave + rt) + r32, head);
    const bool there = tok < w.rows;
    // (no row there: as if it saw all, since one that sees nothing has its reference fixed in every step)
    const int limit = (there ? key_limit(p, w, tok) : end) - first;
    lds.limit[32 * (RT * wave + rt) + r32] = limit;  // (the steps with masks read them there)
    most = max(most, limit);
    if (there) least = min(least, limit);
    const bf16_t *const qp = (const bf16_t *)p.a.q + (int64_t)(w.row0 + (there ? tok : 0)) * p.a.q_rs +
                             (w.g * p.a.group + (there ? head : 0)) * HD + 8 * hf;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      qreg[rt][t] = *(const bf16x8 *)(qp + 16 * t);
      if (!there) qreg[rt][t] = bf16x8{};
    }
  }
  least = wave_min(least);
  const bool idle = least == 0x7fffffff;  // no row: the wave only loads for the others
  const int ntw = min((-wave_min(-most) + 31) >> 5, 2 * nblk);  // tiles that the wave's rows see

  // staging: 2 x 16 B per thread of a K block and of a V block, rows crow and
  // crow + 32: a wave's are the block's chunks `wave` and `wave + 4`
  const int crow = tid >> 3, ccol = (tid & 7) * 8;
  const PageRows rows = PageRows::of<T>(c);
  const uint32_t off = (lane >> 3) * rows.row_bytes + ccol * sizeof(T);
  const char *const Kg = (const char *)((const T *)c.k + w.g * c.head_stride);
  const char *const Vg = (const char *)((const T *)c.v + w.g * c.head_stride);
  Raw k0, k1, v0, v1;
  int sk = 0, sv = 0;  // lanes 0 and 1 (mod 2): the scales of the wave's chunks of the K and V blocks loaded last
  const uint8_t *const skg = src.scales(w.g, false), *const svg = src.scales(w.g, true);
  bool any_odd = false;
  int k_ok = 0, v_ok = 0;  // bit 0, 1: the chunk in k0 / k1 has memory, in v0 / v1
  // lanes 0 and 1: the table entries of the wave's chunks of a block
  auto entry_of = [&](int blk) __attribute__((always_inline)) {
    return keys.entry(first + kBK * blk + 8 * wave + 32 * (lane & 1));
  };
  int e_k = 0;             // of the K block to load next
  int id0 = 0, id1 = 0;    // of the K block loaded last
  // K block blk, whose entries stand in e_k
  auto gload_k = [&](int blk) __attribute__((always_inline)) {
    uint32_t o32 = off;
    asm volatile("" : "+v"(o32));  // a scalar base and this offset, not a sum of pointers kept in registers
    id0 = __builtin_amdgcn_readlane(e_k, 0);
    id1 = __builtin_amdgcn_readlane(e_k, 1);
    const int key = first + kBK * blk + 8 * wave;
    k_ok = rows.there(id0) | rows.there(id1) << 1;
    k0 = *(const Raw *)(Kg + rows.at(id0, key) + o32);
    k1 = *(const Raw *)(Kg + rows.at(id1, key + 32) + o32);
    if constexpr (Src::kScaled) sk = src.scale(skg, rows, lane & 1 ? id1 : id0, key + 32 * (lane & 1));
  };
  // V block blk, the K block loaded last
  auto gload_v = [&](int blk) __attribute__((always_inline)) {
    uint32_t o32 = off;
    asm volatile("" : "+v"(o32));
    const int key = first + kBK * blk + 8 * wave;
    v_ok = rows.there(id0) | rows.there(id1) << 1;
    v0 = *(const Raw *)(Vg + rows.at(id0, key) + o32);
    v1 = *(const Raw *)(Vg + rows.at(id1, key + 32) + o32);
    if constexpr (Src::kScaled) sv = src.scale(svg, rows, lane & 1 ? id1 : id0, key + 32 * (lane & 1));
  };
  auto lstore_k = [&](int blk) __attribute__((always_inline)) {
    bf16_t *ks = kring + (blk & 1) * KBUF;
    const int bits = src.scale_bits(sk);
    *(u32x4 *)(ks + crow * KP + ccol) = src.piece(k0, __builtin_amdgcn_readlane(bits, 0));
    *(u32x4 *)(ks + (crow + 32) * KP + ccol) = src.piece(k1, __builtin_amdgcn_readlane(bits, 1));
    if (lane < 2) lds.chunk_ok[blk & 3][wave + 4 * lane] = (unsigned char)(k_ok >> lane & 1);
  };
  auto lstore_v = [&](int blk) __attribute__((always_inline)) {
    bf16_t *vs = vring + (blk & 1) * VBUF;
    const int bits = src.scale_bits(sv);
    u32x4 x0 = src.piece(v0, __builtin_amdgcn_readlane(bits, 0)), x1 = src.piece(v1, __builtin_amdgcn_readlane(bits, 1));
    if (first + kBK * (blk + 1) > end || v_ok != 3) {  // no key: zeros, whatever lies there
      const int key = first + kBK * blk + crow;
      if (!(v_ok & 1) || key >= end) x0 = u32x4{0, 0, 0, 0};
      if (!(v_ok & 2) || key + 32 >= end) x1 = u32x4{0, 0, 0, 0};
    }
    if (first + kBK * (blk + 1) > keys.whole) {
      const bool odd0 = tame<bf16_t>(x0), odd1 = tame<bf16_t>(x1);
      any_odd |= __builtin_amdgcn_ballot_w64(odd0 || odd1) != 0;
    }
    *(u32x4 *)(vs + crow * VP + ccol) = x0;
    *(u32x4 *)(vs + (crow + 32) * VP + ccol) = x1;
  };

  float l[RT], mcv[RT];  // row sum; reference, log2 units
  f32x16 o[RT][2];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    mcv[rt] = -INFINITY;
    l[rt] = 0.f;
    o[rt][0] = f32x16{};
    o[rt][1] = f32x16{};
  }
  const uint32_t rs_bits = (((lane & 15) >> 2) & 1) == ((lane >> 4) & 1) ? 0x3f803f80u : 0u;
  const int tr_off = (4 * hf + ((lane & 15) >> 2)) * VP + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  auto kfrags = [&](const bf16_t *ks, bf16x8 (&ka)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 4; ++t) ka[t] = *(const bf16x8 *)(ks + r32 * KP + 16 * t + 8 * hf);
  };
  // V^T fragments: key slot j of 16-key chunk u is key 16u + (j/4)*8 + 4hf + j%4
  auto vfrags = [&](const bf16_t *vs, bf16x8 (&va)[2][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bf16_t *vsl = vs + 16 * u * VP + tr_off;
#pragma unroll
      for (int dt = 0; dt < 2; ++dt) {
        const bf16x4 lo = lds_tr16(vsl + 32 * dt);
        const bf16x4 hi = lds_tr16(vsl + 8 * VP + 32 * dt);
        va[u][dt] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      }
    }
  };
  auto scores = [&](const bf16x8 (&ka)[4], f32x16 (&s)[RT]) __attribute__((always_inline)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      s[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[0], qreg[rt][0], f32x16{}, 0, 0, 0);
#pragma unroll
      for (int t = 1; t < 4; ++t) s[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[t], qreg[rt][t], s[rt], 0, 0, 0);
    }
  };
  auto pv = [&](const bf16x8 (&va)[2][2], const bf16x8 (&pb)[RT][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          o[rt][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[u][dt], pb[rt][u], o[rt][dt], 0, 0, 0);
  };
  auto exps = [&](const f32x16 &s, float mc, bf16x8 (&pb)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) pb[u][j] = (__bf16)__builtin_amdgcn_exp2f(fmaf(s[8 * u + j], cl, -mc));
  };
  auto rowsum = [&](const bf16x8 (&pb)[2]) __attribute__((always_inline)) {
    uint32_t b = rs_bits;
    asm volatile("" : "+v"(b));  // keeps the selector from being hoisted out of the loop
    const bf16x8 sel = __builtin_bit_cast(bf16x8, u32x4{b, b, b, b});
    f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(sel, pb[0], f32x4{}, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(sel, pb[1], d, 0, 0, 0)[0];
  };
  // bit r: rows 8r .. of tile t have memory
  auto pages_of = [&](int t) __attribute__((always_inline)) {
    const uint32_t ok =
        __builtin_amdgcn_readfirstlane(*(const uint32_t *)&lds.chunk_ok[(t >> 1) & 3][4 * (t & 1)]);
    return (ok & 1) | (ok >> 7 & 2) | (ok >> 14 & 4) | (ok >> 21 & 8);
  };
  auto mask = [&](int t, uint32_t pages, f32x16 (&sc)[RT]) __attribute__((always_inline)) {
    const int kb = 32 * t;
    if (kb + 32 > least || pages != 15) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int limit = lds.limit[32 * (RT * wave + rt) + r32] - kb - 4 * hf;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((i >> 2) * 8 + (i & 3) >= limit || !(pages >> (i >> 2) & 1)) sc[rt][i] = -INFINITY;
      }
    }
  };
  auto fixup = [&](int rt, const f32x16 &s, bf16x8 (&pb)[2], float &rs) __attribute__((always_inline)) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mt = fmaxf(mcv[rt], mx * cl);  // -inf while nothing is visible
    const bool move = mcv[rt] == -INFINITY || mt - mcv[rt] > kMoveLog2;
    const float m_new = move ? mt : mcv[rt];
    const float mn = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(mcv[rt] - mn);
    l[rt] *= alpha;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[rt][dt][i] *= alpha;
    mcv[rt] = m_new;
    exps(s, mn, pb);
    rs = own_sums(pb);
  };
  auto step = [&](auto masked_tag, int t, const bf16_t *vs, const bf16_t *ks, f32x16 (&sc)[RT], f32x16 (&sn)[RT],
                  bf16x8 (&pp)[RT][2], bf16x8 (&pc)[RT][2], float (&rsp)[RT], float (&rsc)[RT])
      __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    {
      bool bad = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) bad = bad || !(rsp[rt] <= kSumLimit);  // NaN included
      if (__builtin_amdgcn_ballot_w64(bad) != 0) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) fixup(rt, sn[rt], pp[rt], rsp[rt]);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) l[rt] += rsp[rt];
    }
    if (!MASKED) {
    } else if (t >= ntw) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[rt][i] = -INFINITY;
    } else {
      mask(t, pages_of(t), sc);
    }
    bf16x8 va[2][2], ka[4];
    vfrags(vs, va);
    kfrags(ks, ka);
    pv(va, pp);
    scores(ka, sn);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) exps(sc[rt], mcv[rt], pc[rt]);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) rsc[rt] = rowsum(pc[rt]);
    __builtin_amdgcn_sched_group_barrier(0x100, 12, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
#pragma unroll
    for (int i = 0; i < 10 * RT; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
    }
  };

  f32x16 sa[RT], sb[RT];
  bf16x8 pa[RT][2], pbb[RT][2];
  float rsa[RT], rsb[RT];
  if (nblk > 0) {
    // entries of the first three blocks in one load, then their rows in one round trip
    const int e = keys.entry(first + kBK * (lane >> 1) + 8 * wave + 32 * (lane & 1));
    e_k = e;
    gload_k(0);
    gload_v(0);
    const Raw ka = k0, kb = k1, va = v0, vb = v1;
    const int ok0 = k_ok, sk0 = sk, sv0 = sv;
    e_k = __shfl(e, 2 + (lane & 1), 64);
    gload_k(1);
    gload_v(1);
    const Raw kc = k0, kd = k1, vc = v0, vd = v1;
    const int ok1 = k_ok, sk1 = sk, sv1 = sv;
    e_k = __shfl(e, 4 + (lane & 1), 64);
    gload_k(2);
    const Raw ke = k0, kf = k1;
    const int ok2 = k_ok, sk2 = sk;
    e_k = entry_of(3);
    k0 = ka; k1 = kb; v0 = va; v1 = vb;
    k_ok = v_ok = ok0;
    sk = sk0; sv = sv0;
    lstore_k(0);
    lstore_v(0);
    k0 = kc; k1 = kd; v0 = vc; v1 = vd;
    k_ok = v_ok = ok1;
    sk = sk1; sv = sv1;
    lstore_k(1);
    k0 = ke; k1 = kf;
    k_ok = ok2;
    sk = sk2;
  }
  __syncthreads();
  if (nblk > 0) {  // step 0: scores of tiles 0 and 1, softmax of tile 0 against its true maximum
    bf16x8 ka[4];
    kfrags(kring, ka);
    scores(ka, sa);
    kfrags(kring + 32 * KP, ka);
    scores(ka, sb);
    mask(0, pages_of(0), sa);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) fixup(rt, sa[rt], pa[rt], rsa[rt]);
  }
  __syncthreads();  // iteration 0 stores K_2 where step 0 read K_0
  // iteration j: steps 2j+1 and 2j+2, which read only V_j and K_{j+1}; it
  // stores K_{j+2} and V_{j+1} where K_j and V_{j-1} were, last read one
  // iteration before: one barrier a block
  const int t_safe = min(least, kBK * nblk) >> 5;
  const int j_safe = min(min(nblk, max(0, (t_safe - 1) / 2)), max(gap - 1, 0));
  auto stage = [&](int j) __attribute__((always_inline)) {
    lstore_k(j + 2);
    lstore_v(j + 1);
    gload_v(j + 2);
    gload_k(j + 3);  // (past the end: the last key's page again)
    e_k = entry_of(j + 4);
    __syncthreads();
  };
  auto iteration = [&](auto masked_tag, int j) __attribute__((always_inline)) {
    const bf16_t *vc = vring + (j & 1) * VBUF;
    const bf16_t *kn = kring + ((j + 1) & 1) * KBUF;
    step(masked_tag, 2 * j + 1, vc, kn, sb, sa, pa, pbb, rsa, rsb);
    step(masked_tag, 2 * j + 2, vc + 32 * VP, kn + 32 * KP, sa, sb, pbb, pa, rsb, rsa);
    stage(j);
  };
  int j = 0;
  if (idle)
    for (; j < nblk; ++j) stage(j);
  for (; j < j_safe; ++j) iteration(std::false_type{}, j);
  for (; j < nblk; ++j) iteration(std::true_type{}, j);

  if (lane == 0) lds.odd[wave] = any_odd;
  __syncthreads();
  if (lds.odd[0] | lds.odd[1] | lds.odd[2] | lds.odd[3]) {
    const int *const limit = lds.limit + 32 * RT * wave + r32;
    const int limits[RT] = {limit[0] + first, limit[32] + first};
    const int g = lds.piece.g;
    add_odd(keys, rows, [&](int id, int k, int i) { return src.value(rows, Vg, g, id, k, i); },
            max(first, keys.whole & -kBK), min(first + kBK * nblk, end), o, limits,
            [&](int i) { return 32 * (i >> 4) + 8 * (i >> 2 & 3) + 4 * hf + (i & 3); });
  }
  // ---- results: lane holds row (rt, r32)'s elements 32 dt + 8 gi + 4 hf .. +3
  const Piece f = lds.piece;
  auto write = [&](int t, int h, int rt, float sum) __attribute__((always_inline)) {
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    bf16_t *const op = (bf16_t *)p.a.o + (int64_t)(f.row0 + t) * p.a.o_rs + h * HD;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int gi = 0; gi < 4; ++gi) {
        const f32x16 &x = o[rt][dt];
        const uint32_t lo = (uint32_t)f32_to_bf16(x[4 * gi] * inv) | ((uint32_t)f32_to_bf16(x[4 * gi + 1] * inv) << 16);
        const uint32_t hi = (uint32_t)f32_to_bf16(x[4 * gi + 2] * inv) | ((uint32_t)f32_to_bf16(x[4 * gi + 3] * inv) << 16);
        *(uint2 *)(op + 32 * dt + 8 * gi + 4 * hf) = make_uint2(lo, hi);
      }
  };
  const int64_t rec_step = (int64_t)c.n_kv_heads * R * kRec;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int h;
    const int row = 32 * (RT * wave + rt) + r32, t = token_of(f, p.a.inv_group, p.a.group, row, h);
    if (t >= f.rows) continue;
    h += f.g * p.a.group;
    if (f.parts == 1 && !p.prefix_parts) {
      write(t, h, rt, l[rt]);
    } else {
      if (p.prefix_parts) {
        float *const r = p.ws + (((int64_t)f.slot + (int64_t)f.part * c.n_kv_heads) * R + row) * kRow;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const f32x16 &x = o[rt][i >> 2];
          const int e = 4 * (i & 3);
          *(float4 *)(r + 32 * (i >> 2) + 8 * (i & 3) + 4 * hf) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
        }
        if (hf == 0) *(float2 *)(r + HD) = make_float2(mcv[rt], l[rt]);
        continue;
      }
      float *const r = p.ws + (int64_t)f.slot * R * kRec + 2 * row + f.part * rec_step;
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int i = 0; i < 16; i += 2)
          put2(r + R * (32 * dt + 8 * (i >> 2) + 4 * hf + (i & 3)), o[rt][dt][i], o[rt][dt][i + 1]);
      if (hf == 0) put2(r + R * HD, mcv[rt], l[rt]);
    }
  }
  if (f.parts == 1 || p.prefix_parts) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the records have reached memory
  __syncthreads();
  if (tid == 0) lds.last_in = arrive_last(p.arrive_end - 2 * ((int64_t)f.slot + 1), f.parts, p.tag);
  __syncthreads();
  if (!lds.last_in) return;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int h;
    const int row = 32 * (RT * wave + rt) + r32, t = token_of(f, p.a.inv_group, p.a.group, row, h);
    if (t >= f.rows) continue;
    h += f.g * p.a.group;
    const float *const r0 = p.ws + (int64_t)f.slot * R * kRec + 2 * row;
    float M = -INFINITY, L = 0.f;
    o[rt][0] = o[rt][1] = f32x16{};
    constexpr int MB = 2;  // records on their way together
    for (int n0 = 0; n0 < f.parts; n0 += MB) {
      float2 ml[MB], x[MB][16];
#pragma unroll
      for (int v = 0; v < MB; ++v) {
        const float *const r = r0 + min(n0 + v, f.parts - 1) * rec_step;
        ml[v] = get2(r + R * HD);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[v][i] = get2(r + R * (32 * (i >> 3) + 8 * ((i >> 1) & 3) + 4 * hf + 2 * (i & 1)));
      }
#pragma unroll
      for (int v = 0; v < MB; ++v) {
        if (n0 + v >= f.parts) break;
        const float mn = fmaxf(M, ml[v].x), mu = mn == -INFINITY ? 0.f : mn;
        const float fo = __builtin_amdgcn_exp2f(M - mu), fn = __builtin_amdgcn_exp2f(ml[v].x - mu);
        L = fmaf(ml[v].y, fn, L * fo);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[rt][i >> 3][2 * (i & 7)] = fmaf(x[v][i].x, fn, o[rt][i >> 3][2 * (i & 7)] * fo);
          o[rt][i >> 3][2 * (i & 7) + 1] = fmaf(x[v][i].y, fn, o[rt][i >> 3][2 * (i & 7) + 1] * fo);
        }
        M = mn;
      }
    }
    write(t, h, rt, L);
  }
}

// fp32, v_mfma_f32_32x32x2f32: matrix-core time is all that counts.  32 rows a
// unit, its tiles dealt to KW waves, no barrier before the merge: a wave
// stages its own K tile in LDS one tile ahead (rows of 272 B) and reads V
// straight from the pages as the second product's operand (two adjacent d of
// one key row a lane), requested before the scores' products, which cover it.
// 1636 and 1492 rows behind 435 and 539 (20 heads) 212 us, 96 TFLOP/s; 512 rows
// 20.6 us (52), matrix cores 39% busy: units of unequal length, 6 us of start.
template <int KW>
struct PrefillLdsF32 {
  float smem[KW * 32 * (HD + 4)];
  float red_m[KW][32], red_l[KW][32];
  int odd[KW];
  Piece piece;
  int last_in;
};
template <int KW, class Src = PlainPages<float>>
__device__ __forceinline__ void prefill_f32_body(const PrefillParams &p, PrefillLdsF32<KW> &lds, int block,
                                                 const Src &src = Src{}) {
  typedef typename Src::T T;
  constexpr int R = 32, KP = HD + 4;  // K row and O row pitch, floats
  constexpr int TILE = 32 * KP;
  float *const smem = lds.smem;
  auto &red_m = lds.red_m, &red_l = lds.red_l;

  const int tid = threadIdx.x, lane = tid & 63;
  const int kw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, hf = lane >> 5;
  Piece w;
  if (!find_piece<R>(p, block, w)) return;
  if (tid == 0) lds.piece = w;
  const Paged &c = p.a.c;
  const PieceKeys keys = piece_keys<R>(p, w);
  const float cl = p.a.cl;
  float *const kl = smem + kw * TILE;
  int head;
  const int tok = token_of(w, p.a.inv_group, p.a.group, r32, head);
  const bool there = tok < w.rows;
  const int limit = there ? key_limit(p, w, tok) : keys.end;

  const PageRows rows = PageRows::of<T>(c);
  const uint32_t row_bytes = rows.row_bytes;
  const uint32_t koff = (lane >> 4) * row_bytes + (lane & 15) * (4 * sizeof(T));  // 4 rows a load
  const uint32_t voff = 4 * hf * row_bytes + r32 * (2 * sizeof(T));
  const char *const Kg = (const char *)((const T *)c.k + w.g * c.head_stride);
  const char *const Vg = (const char *)((const T *)c.v + w.g * c.head_stride);
  typename Src::Raw kr[8];
  // scaled: lanes r and 4 + r (mod 8): the byte of rows 8r .. of K, of V, of the tile to load next
  int sc = 0;
  const uint8_t *const sg = src.scales(w.g, lane & 4);
  int entry = 0;  // lane r (mod 4): of rows 8r .. of the tile to load next
  uint64_t at[4], vat[4];  // byte offsets of rows 8r .. of the tile to load next, of this tile
  int pages = 0, pages_next = 0;
  auto load_ids = [&](int t) __attribute__((always_inline)) { entry = keys.entry(32 * t + 8 * (lane & 3)); };
  auto gload_k = [&](int t) __attribute__((always_inline)) {
    pages_next = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int id = __builtin_amdgcn_readlane(entry, r);
      pages_next |= rows.there(id) << r;
      at[r] = rows.at(id, 32 * t + 8 * r);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        kr[2 * r + j] = *(const typename Src::Raw *)(Kg + at[r] + (uint64_t)(j * 4u) * row_bytes + koff);
    }
    if constexpr (Src::kScaled) sc = src.scale(sg, rows, entry, 32 * t + 8 * (lane & 3));
  };
  float qreg[32];  // k slot (hf, t) of the score product is d = 32 hf + t
  {
    const float *const qp = (const float *)p.a.q + (int64_t)(w.row0 + (there ? tok : 0)) * p.a.q_rs +
                            (w.g * p.a.group + (there ? head : 0)) * HD + 32 * hf;
#pragma unroll
    for (int t = 0; t < 32; t += 4) {
      const float4 x = *(const float4 *)(qp + t);
      qreg[t] = x.x; qreg[t + 1] = x.y; qreg[t + 2] = x.z; qreg[t + 3] = x.w;
    }
  }
  float mc = -INFINITY, l = 0.f;
  f32x16 ow[1][2] = {{f32x16{}, f32x16{}}};  // ow[0][j] row i is d = 2i + j
  f32x16 (&o)[2] = ow[0];
  bool any_odd = false;
  int t = keys.t0 + kw;
  if (t < keys.t1) {
    load_ids(t);
    gload_k(t);
    load_ids(t + KW);
  }
  for (; t < keys.t1; t += KW) {
    pages = pages_next;
#pragma unroll
    for (int r = 0; r < 4; ++r) vat[r] = at[r];
    const int bits = src.scale_bits(sc);
    // the wave's own tile: its LDS instructions execute in order
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *(u32x4 *)(kl + (4 * j + (lane >> 4)) * KP + (lane & 15) * 4) =
          src.piece(kr[j], __builtin_amdgcn_readlane(bits, j >> 1));
    __builtin_amdgcn_wave_barrier();
    // this tile's V: key slot (hf, i) of the second product is key 8(i/4) + 4hf + i%4
    typename Src::Pair vp[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      vp[i] = *(const typename Src::Pair *)(Vg + vat[i >> 2] + (uint64_t)(i & 3u) * row_bytes + voff);
    gload_k(t + KW);  // past the range: the last key's page again, not used
    load_ids(t + 2 * KW);
    f32x16 s = f32x16{};
    const float *krow = kl + r32 * KP + 32 * hf;
#pragma unroll
    for (int u = 0; u < 32; u += 4) {
      const float4 a = *(const float4 *)(krow + u);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, qreg[u], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, qreg[u + 1], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, qreg[u + 2], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, qreg[u + 3], s, 0, 0, 0);
    }
    float2 vr[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) vr[i] = src.pair(vp[i], __builtin_amdgcn_readlane(bits, 4 + (i >> 2)));
    const int kb = 32 * t;
    if (kb + 32 > keys.whole || pages != 15) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = (i >> 2) * 8 + hf * 4 + (i & 3);
        const bool page = pages >> (i >> 2) & 1;
        if (kb + k >= limit || !page) s[i] = -INFINITY;
        if (kb + k >= keys.end || !page) vr[i] = make_float2(0.f, 0.f);  // no key: whatever lies there
        const bool bx = !(fabsf(vr[i].x) < INFINITY), by = !(fabsf(vr[i].y) < INFINITY);
        vr[i] = make_float2(bx ? 0.f : vr[i].x, by ? 0.f : vr[i].y);
        odd |= bx || by;
      }
      any_odd |= __builtin_amdgcn_ballot_w64(odd) != 0;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float m_new = fmaxf(mc, mx * cl);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(mc - ref);
    float rs = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], cl, -ref));
      rs += s[i];
    }
    l = l * alpha + rs;  // per half-wave; the halves are summed at the end
    mc = m_new;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[j][i] *= alpha;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[i].x, s[i], o[0], 0, 0, 0);
      o[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[i].y, s[i], o[1], 0, 0, 0);
    }
  }

  l += __shfl_xor(l, 32, 64);
  if (hf == 0) {
    red_m[kw][r32] = mc;
    red_l[kw][r32] = l;
  }
  if (lane == 0) lds.odd[kw] = any_odd;
  __syncthreads();
  any_odd = false;
#pragma unroll
  for (int v = 0; v < KW; ++v) any_odd |= lds.odd[v] != 0;
  float M = red_m[0][r32];
#pragma unroll
  for (int v = 1; v < KW; ++v) M = fmaxf(M, red_m[v][r32]);
  const float f = mc == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - M);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[j][i] *= f;
  if (any_odd && kw == 0) {
    const int limits[1] = {limit};
    const int g = lds.piece.g;
    add_odd(keys, rows, [&](int id, int k, int i) { return src.value(rows, Vg, g, id, k, i); },
            max(32 * keys.t0, keys.whole & -32), min(32 * keys.t1, keys.end), ow, limits,
            [&](int i) { return 2 * (8 * (i >> 2 & 3) + 4 * hf + (i & 3)) + (i >> 4); });
  }
#pragma unroll
  for (int gi = 0; gi < 4; ++gi) {
    float *dst = kl + r32 * KP + 2 * (8 * gi + 4 * hf);
    *(float4 *)dst = make_float4(o[0][4 * gi], o[1][4 * gi], o[0][4 * gi + 1], o[1][4 * gi + 1]);
    *(float4 *)(dst + 4) = make_float4(o[0][4 * gi + 2], o[1][4 * gi + 2], o[0][4 * gi + 3], o[1][4 * gi + 3]);
  }
  __syncthreads();
  constexpr int NV = HD / (2 * KW);
  finish_piece<float, R, 64 * KW>(p, lds.piece, &lds.last_in, [&](int row, int d0, float (&acc)[NV]) __attribute__((always_inline)) {
    float Mr = red_m[0][row];
#pragma unroll
    for (int v = 1; v < KW; ++v) Mr = fmaxf(Mr, red_m[v][row]);
    const float Mu = Mr == -INFINITY ? 0.f : Mr;
    float L = 0.f;
#pragma unroll
    for (int v = 0; v < KW; ++v) L += red_l[v][row] * __builtin_amdgcn_exp2f(red_m[v][row] - Mu);
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i += 4)
#pragma unroll
      for (int v = 0; v < KW; ++v) {
        const float4 x = *(const float4 *)(smem + v * TILE + row * KP + d0 + i);
        acc[i] += x.x; acc[i + 1] += x.y; acc[i + 2] += x.z; acc[i + 3] += x.w;
      }
    return make_float2(Mr, L);
  });
}

}  // namespace
}  // namespace bn
