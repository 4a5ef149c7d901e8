// bn_paged.hip -- paged KV cache: appending rows with their rotation, and the
// attention of one or many query rows per sequence over the pages.
//
// The reference keeps no cache (llama_model.py:135-141 recomputes the prefix);
// the rows computed here are those of its causal softmax (op_softmax.cuh:
// 89-99): the query at position pos sees keys 0 .. pos of its sequence, query
// head h reads KV head h / (n_heads / n_kv_heads) (llama_layers.hpp:159-163).
// Rotation as op_rope.cuh:55-99: adjacent pairs, angle pos * theta^(-2p/64).
//
// What lies in a page is found through the sequence's table, read on the
// device: every table entry is checked against n_pages before it is an
// address, and keys are counted up to what the table can hold, so that no
// contents of those arrays lead outside the pools.  (Positions are counted from
// the length as it stands.)
#include <atomic>

#include "bn_paged_device.hpp"
#include "bn_paged_host.hpp"

namespace bn {

// A launch's 48-bit tag: a mixed counter (SplitMix64's finaliser), so that no
// plausible memory contents look like this launch's arrivals.
unsigned long long next_tag() {
  static std::atomic<uint64_t> launches{0};
  uint64_t z = (launches.fetch_add(1) + 1) * 0x9e3779b97f4a7c15ull + 0x517cc1b727220a95ull;
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  return (z ^ (z >> 31)) >> 16 | 1;
}

namespace {

// ------------------------------------------------------------------ append
struct AppendParams {
  Paged c;
  const void *k, *v, *q;
  void *qo;
  const int32_t *starts;
  int64_t k_rs, v_rs, q_rs, qo_rs;
  int n_heads;          // 0 without q
  int turn;             // rotate
  double f[HD / 2];     // turns per position of each pair: theta^(-2p/64) / (2 pi)
};

// A row per workgroup.  32 threads form the pairs' cosines and sines: the
// angle in turns and in 64 bits, reduced to an eighth of a turn before it is
// rounded to 32 (at position 2^20 a 32-bit angle would be off by 0.06 rad).
// All take the row's 16-byte pieces, Q heads, K heads, V heads, consecutive
// threads on consecutive pieces, the first kBatch of a thread on their way
// while the angles are formed.  Bound by memory: 16384 bf16 rows of 32 + 2 * 4
// heads 33 us, 5.0 TB/s read and written, as fast as a copy; 16 rows 3.5 us, a
// launch and the chain row -> sequence -> position -> page.  (Eight rows a
// workgroup, a piece of a thread at a time: 41 us, and 1250 fp32 rows 13.7
// where this takes 8.3; one, three or four pieces a thread: the same to 6% more.)
constexpr int kBatch = 4;
template <typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  constexpr int PIECES = HD * sizeof(T) / 16;  // per head
  constexpr int VEC = 16 / sizeof(T);
  __shared__ float2 cs[HD / 2];
  __shared__ int64_t place;  // element offset of the row's slot in KV head 0 (-1: none)
  __shared__ int owner;      // the row's sequence (-1: padding)
  const int tid = threadIdx.x, row = blockIdx.x, stride = blockDim.x;
  const int hkv = p.c.n_kv_heads, kv0 = p.n_heads, v0 = kv0 + hkv, pieces = (v0 + hkv) * PIECES;
  const T *const Q = (const T *)p.q + row * p.q_rs, *const K = (const T *)p.k + row * p.k_rs,
          *const V = (const T *)p.v + row * p.v_rs;
  u32x4 x[kBatch];
  auto load = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int i = first + n * stride, h = i / PIECES, e = (i % PIECES) * VEC;
      if (i < pieces) x[n] = *(const u32x4 *)((h < kv0 ? Q + h * HD : h < v0 ? K + (h - kv0) * HD : V + (h - v0) * HD) + e);
    }
  };
  load(tid);
  if (tid < HD / 2) {
    const int b = sequence_of(p.starts, p.c.batch, row);
    const int pos = b < 0 ? 0 : position_of(p.c, p.starts, b, row);
    if (tid == 0) {
      int64_t at = -1;
      if (b >= 0 && pos >= 0 && pos < p.c.cap) {
        const int page = p.c.table[b * p.c.table_stride + (pos >> p.c.shift)];
        if ((unsigned)page < (unsigned)p.c.n_pages)
          at = page * p.c.page_stride + (pos & ((1 << p.c.shift) - 1)) * p.c.row_stride;
      }
      place = at;
      owner = b;
    }
    cs[tid] = cos_sin((double)pos * p.f[tid]);
  }
  __syncthreads();
  if (owner < 0) return;
  const int64_t at = place;
  T *const Kd = (T *)p.c.k + at, *const Vd = (T *)p.c.v + at;
  T *const Qo = (T *)p.qo + row * p.qo_rs;
  for (int first = tid; first < pieces; first += kBatch * stride) {
    if (first != tid) load(first);
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const int i = first + n * stride, h = i / PIECES, e = (i % PIECES) * VEC;
      if (i >= pieces) break;
      if (p.turn && h < v0) x[n] = rotate<T>(x[n], &cs[e / 2]);
      if (h < kv0) *(u32x4 *)(Qo + h * HD + e) = x[n];
      else if (at >= 0)
        *(u32x4 *)((h < v0 ? Kd + (h - kv0) * p.c.head_stride : Vd + (h - v0) * p.c.head_stride) + e) = x[n];
    }
  }
}

// ----------------------------------------------------- decode, over pages
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
template <typename T>
__device__ __forceinline__ void decode_body(const DecodeParams &p, DecodeLds<T> &lds, int block) {
  using Ti = DecTile<T>;
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
  const uint32_t off = (uint32_t)((crow * c.row_stride + ccol) * sizeof(T));
  const char *const Kg = (const char *)((const T *)c.k + g * c.head_stride);
  const char *const Vg = (const char *)((const T *)c.v + g * c.head_stride);
  const PageRows page_rows = PageRows::of<T>(c);
  // A tile's table entries are read as scalars: they come in their own order,
  // not behind the rows requested before them (as vector loads they held up
  // the next rows: 64 caches of 4096 keys 51 us).
  int ids[4];  // of rows RPI r .. of the tile to load next
  struct Rows {
    u32x4 k[4], v[4];  // the lane's pieces of a tile
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
      y.k[r] = __builtin_nontemporal_load((const u32x4 *)(Kg + at[r] + off));
      y.v[r] = __builtin_nontemporal_load((const u32x4 *)(Vg + at[r] + off));
    }
  };
  T *const kt = lds.k[wave], *const vt = lds.v[wave];
  auto store_rows = [&](Rows &y, bool masked) __attribute__((always_inline)) {
    if (masked) {  // no key: zeros, whatever lies there (0 times an infinite value is none)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = crow + RPI * r;
        if (row < y.lo || row >= y.hi || !(y.pages >> r & 1)) y.k[r] = y.v[r] = u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) *(u32x4 *)(kt + (crow + RPI * r) * P + ccol) = y.k[r];
#pragma unroll
    for (int r = 0; r < 4; ++r) *(u32x4 *)(vt + (crow + RPI * r) * P + ccol) = y.v[r];
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
template <typename T>
__global__ __launch_bounds__(256) void paged_decode_kernel(DecodeParams p) {
  __shared__ __attribute__((aligned(16))) DecodeLds<T> lds;
  decode_body<T>(p, lds, blockIdx.x);
}

// ------------------------------------------------- prefill, over pages
template <int HW, int KW, int OCC>
__global__ __launch_bounds__(64 * HW * KW, OCC) void paged_prefill_bf16_kernel(PrefillParams p) {
  __shared__ __attribute__((aligned(16))) PrefillLds<HW, KW> lds;
  prefill_bf16_body<HW, KW>(p, lds, blockIdx.x);
}

__global__ __launch_bounds__(256, 2) void paged_prefill_pipe_kernel(PrefillParams p) {
  __shared__ __attribute__((aligned(16))) PipeLds lds;
  prefill_pipe_body(p, lds, blockIdx.x);
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
template <int KW>
__device__ __forceinline__ void prefill_f32_body(const PrefillParams &p, PrefillLdsF32<KW> &lds, int block) {
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

  const PageRows rows = PageRows::of<float>(c);
  const uint32_t row_bytes = rows.row_bytes;
  const uint32_t koff = (lane >> 4) * row_bytes + (lane & 15) * 16;  // 4 rows of 256 bytes a load
  const uint32_t voff = 4 * hf * row_bytes + r32 * 8;
  const char *const Kg = (const char *)((const float *)c.k + w.g * c.head_stride);
  const char *const Vg = (const char *)((const float *)c.v + w.g * c.head_stride);
  u32x4 kr[8];
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
      for (int j = 0; j < 2; ++j) kr[2 * r + j] = *(const u32x4 *)(Kg + at[r] + (uint64_t)(j * 4u) * row_bytes + koff);
    }
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
    // the wave's own tile: its LDS instructions execute in order
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 8; ++j) *(u32x4 *)(kl + (4 * j + (lane >> 4)) * KP + (lane & 15) * 4) = kr[j];
    __builtin_amdgcn_wave_barrier();
    // this tile's V: key slot (hf, i) of the second product is key 8(i/4) + 4hf + i%4
    float2 vr[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      vr[i] = *(const float2 *)(Vg + vat[i >> 2] + (uint64_t)(i & 3u) * row_bytes + voff);
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
    add_odd(keys, rows, [&](int id, int k, int i) { return Elem<float>::load((const float *)(Vg + rows.at(id, k)) + i); },
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
template <int KW>
__global__ __launch_bounds__(64 * KW, 2) void paged_prefill_f32_kernel(PrefillParams p) {
  __shared__ __attribute__((aligned(16))) PrefillLdsF32<KW> lds;
  prefill_f32_body<KW>(p, lds, blockIdx.x);
}

// ------------------------------------------------- decode, a shared prefix
// One launch for the common keys and the sequences' own: workgroups of the
// prefill kernel over the batch's rows and the prefix (its keys are read once
// for 32 or 256 rows, and computed at matrix-core rates), and workgroups of
// the decode kernel over the keys behind it, eight of one kind and eight of
// the other in turn while both last, so that a compute unit has some of each:
// the one kind waits for memory, the other for the matrix cores.  Both leave
// records, which a second launch adds, a row's two elements a thread.  200
// sequences of up to 1000 keys behind 16387 76 us, 364 TFLOP/s: one prefix
// workgroup a compute unit, 18 MB of records; 64 behind 2048 16.3 us, two
// launches and their round trips.
struct SharedParams {
  DecodeParams d;
  PrefillParams f;
  int n_dec, n_pre;  // workgroups (multiples of 8 but for the last of a kind)
};
__device__ __forceinline__ bool shared_block(const SharedParams &p, int &block) {  // true: prefix
  const int q = blockIdx.x >> 3, x = blockIdx.x & 7;
  const int d8 = (p.n_dec + 7) >> 3, f8 = (p.n_pre + 7) >> 3, both = min(d8, f8);
  bool prefix = d8 < f8;
  if (q < 2 * both) {
    prefix = q & 1;
    block = (q >> 1) * 8 + x;
  } else {
    block = (q - both) * 8 + x;
  }
  return prefix;
}
template <int HW, int KW>
__global__ __launch_bounds__(256, 2) void paged_shared_bf16_kernel(SharedParams p) {
  static_assert(HW * KW == 4, "256 threads");
  union Lds {
    DecodeLds<bf16_t> d;
    PrefillLds<HW, KW> f;
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  int block;
  if (shared_block(p, block)) {
    if (block < p.n_pre) prefill_bf16_body<HW, KW>(p.f, lds.f, block);
  } else if (block < p.n_dec) {
    decode_body<bf16_t>(p.d, lds.d, block);
  }
}
__global__ __launch_bounds__(256, 2) void paged_shared_pipe_kernel(SharedParams p) {
  union Lds {
    DecodeLds<bf16_t> d;
    PipeLds f;
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  int block;
  if (shared_block(p, block)) {
    if (block < p.n_pre) prefill_pipe_body(p.f, lds.f, block);
  } else if (block < p.n_dec) {
    decode_body<bf16_t>(p.d, lds.d, block);
  }
}
__global__ __launch_bounds__(256, 2) void paged_shared_f32_kernel(SharedParams p) {
  union Lds {
    DecodeLds<float> d;
    PrefillLdsF32<4> f;
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  int block;
  if (shared_block(p, block)) {
    if (block < p.n_pre) prefill_f32_body<4>(p.f, lds.f, block);
  } else if (block < p.n_dec) {
    decode_body<float>(p.d, lds.d, block);
  }
}

// The records of a row, the prefix's parts and then its own keys' pieces: two
// elements a thread.
struct RowSum {
  float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
  // records rec(0) .. rec(n - 1), eight at a time
  template <class F>
  __device__ __forceinline__ void add(int n, int d, F &&rec) {
    constexpr int N = 8;
    for (int n0 = 0; n0 < n; n0 += N) {
      float2 ml[N], y[N];
#pragma unroll
      for (int v = 0; v < N; ++v) {
        const float *const q = rec(min(n0 + v, n - 1));
        ml[v] = *(const float2 *)(q + HD);
        y[v] = *(const float2 *)(q + d);
      }
      float mx = M;
#pragma unroll
      for (int v = 0; v < N; ++v) mx = n0 + v < n ? fmaxf(mx, ml[v].x) : mx;
      const float mu = mx == -INFINITY ? 0.f : mx, fo = __builtin_amdgcn_exp2f(M - mu);
      L *= fo;
      A0 *= fo;
      A1 *= fo;
#pragma unroll
      for (int v = 0; v < N; ++v) {
        const bool in = n0 + v < n;
        const float f = __builtin_amdgcn_exp2f(ml[v].x - mu);
        L = in ? fmaf(ml[v].y, f, L) : L;
        A0 = in ? fmaf(y[v].x, f, A0) : A0;
        A1 = in ? fmaf(y[v].y, f, A1) : A1;
      }
      M = mx;
    }
  }
};
template <typename T>
__global__ __launch_bounds__(256) void paged_shared_add_kernel(SharedParams p, int R) {
  const AttnParams &a = p.d.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int d = 2 * (int)(i % (HD / 2)), h = (int)(i / (HD / 2) % a.n_heads), b = (int)(i / (HD / 2) / a.n_heads);
  if (b >= a.c.batch) return;
  const int g = h / a.group, hg = h - g * a.group, col = g * p.d.hblocks + hg / kMaxRows, row = hg % kMaxRows;
  const int cut = p.d.cuts[b * p.d.columns + col], bin0 = min(cut & 0xffff, p.d.bins - 1);
  const int pieces = min(max(cut >> 16, 1), p.d.bins - bin0);
  const int fr = b * a.group + hg, unit = fr / R, parts = p.f.prefix_parts;
  const float *const r = p.f.ws + (((int64_t)unit * parts * a.c.n_kv_heads + g) * R + (fr - unit * R)) * kRow;
  const int64_t step = (int64_t)a.c.n_kv_heads * R * kRow;
  RowSum s;
  s.add(parts, d, [&](int n) { return r + n * step; });
  s.add(pieces, d, [&](int n) {
    return pieces == 1 ? p.d.parts + ((int64_t)b * a.n_heads + h) * kRec
                       : p.d.ws + ((((int64_t)(bin0 + n) * 2 + (n == 0)) * p.d.columns + col) * kMaxRows + row) * kRec;
  });
  const float inv = s.L > 0.f ? 1.0f / s.L : 0.f;
  T *const op = (T *)a.o + b * a.o_rs + h * HD + d;
  if constexpr (sizeof(T) == 2)
    *(uint32_t *)op = (uint32_t)f32_to_bf16(s.A0 * inv) | ((uint32_t)f32_to_bf16(s.A1 * inv) << 16);
  else
    *(float2 *)op = make_float2(s.A0 * inv, s.A1 * inv);
}

// ---------------------------------------------------------------- the host
int launch_decode(const AttnParams &a, int dtype, void *ws, hipStream_t s) {
  const DecodePlan d = plan_decode(a.c.batch, a.n_heads, a.c.n_kv_heads);
  DecodeParams p;
  p.a = a;
  p.ws = (float *)ws;
  p.arrive_end = (unsigned long long *)((char *)ws + d.records + d.words);
  p.tag = next_tag();
  p.bins = d.bins; p.hblocks = d.hblocks; p.columns = d.columns;
  p.k0 = 0;
  p.parts = nullptr;
  p.cuts = nullptr;
  const dim3 grid((unsigned)(d.bins * d.columns)), block(256);
  if (dtype == BN_BF16) hipLaunchKernelGGL(paged_decode_kernel<bf16_t>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(paged_decode_kernel<float>, grid, block, 0, s, p);
  BN_LAUNCH_CHECK();
  return BN_OK;
}

int launch_prefill(const AttnParams &a, int dtype, void *ws, hipStream_t s) {
  const PrefillPlan d = plan_prefill(dtype, a.c.batch, a.n_rows, a.n_heads, a.c.n_kv_heads, a.c.cap);
  PrefillParams p;
  p.a = a;
  p.ws = (float *)ws;
  p.arrive_end = (unsigned long long *)((char *)ws + d.records + d.words);
  p.tag = next_tag();
  p.slots = (int)d.slots;
  p.parts_all = d.parts_all;
  p.pieces = (int)d.pieces;
  p.prefix_parts = 0;
  const dim3 grid((unsigned)d.groups);
  if (dtype == BN_F32) {
    if (d.kw == 4) hipLaunchKernelGGL(paged_prefill_f32_kernel<4>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(paged_prefill_f32_kernel<2>, grid, dim3(128), 0, s, p);
  } else if (d.hw == 8) {
    hipLaunchKernelGGL(paged_prefill_pipe_kernel, grid, dim3(256), 0, s, p);
  } else if (d.hw == 4) {
    if (d.kw == 2) hipLaunchKernelGGL((paged_prefill_bf16_kernel<4, 2, 4>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((paged_prefill_bf16_kernel<4, 1, 4>), grid, dim3(256), 0, s, p);
  } else if (d.kw == 8) {
    hipLaunchKernelGGL((paged_prefill_bf16_kernel<1, 8, 2>), grid, dim3(512), 0, s, p);
  } else {
    hipLaunchKernelGGL((paged_prefill_bf16_kernel<1, 4, 3>), grid, dim3(256), 0, s, p);
  }
  BN_LAUNCH_CHECK();
  return BN_OK;
}

// The shared-prefix call: units of R rows, the prefix's tiles of each in
// `parts`, about two workgroups a compute unit.
struct SharedPlan {
  DecodePlan d;
  int hw, parts;
  int64_t n_pre;
  size_t own, cuts, records;  // bytes: the sequences' own parts and where they are, the prefix's parts
};
SharedPlan plan_shared(int dtype, int batch, int n_heads, int n_kv_heads, int prefix_len) {
  SharedPlan s;
  s.d = plan_decode(batch, n_heads, n_kv_heads);
  const int64_t rows = (int64_t)batch * (n_heads / n_kv_heads);
  // units of 256 rows (the pipelined kernel) once there is work enough to fill the card with them:
  // 64 sequences of 32 heads behind 16384 keys 37 us, with units of 32 rows 42; 100 behind 8192 35
  // and 41; but 64 behind 8192 29 and 27, 16 behind 65536 49 and 44
  const int64_t work = rows * n_kv_heads * prefix_len;
  s.hw = dtype == BN_BF16 && rows * n_kv_heads >= 1024 && work >= 3 << 23 ? 8 : 1;
  const int R = 32 * s.hw, steps = (prefix_len + 31) / 32;
  const int64_t units = (rows + R - 1) / R;
  // pieces: one per compute unit, of 8 tiles at least; two of the large kernel's if they keep 32
  // tiles each (1024 rows behind 16384 keys 80 -> 74 us, behind 4096 42 -> 37 with one;
  // 256 rows behind 2048, 32 rows a piece: 21.9 us with two, 17.5 with one)
  int64_t parts = 512 / (units * n_kv_heads);
  if (s.hw == 1 || parts < 1 || steps / parts < 32) parts = 256 / (units * n_kv_heads);
  s.parts = (int)std::max<int64_t>(1, std::min<int64_t>(parts, steps / 8));
  const int per = n_kv_heads <= 8 && 8 % n_kv_heads == 0 ? 8 / n_kv_heads : 1;
  s.n_pre = (units * s.parts + per - 1) / per * per * n_kv_heads;
  s.own = ((size_t)batch * n_heads * kRec * sizeof(float) + 15) / 16 * 16;
  s.cuts = ((size_t)batch * s.d.columns * sizeof(int) + 15) / 16 * 16;
  s.records = (size_t)units * s.parts * n_kv_heads * R * kRow * sizeof(float);
  return s;
}

int launch_shared(const AttnParams &a, int dtype, void *ws, hipStream_t s) {
  const SharedPlan m = plan_shared(dtype, a.c.batch, a.n_heads, a.c.n_kv_heads, a.prefix_len);
  char *at = (char *)ws;
  SharedParams p;
  p.d.a = p.f.a = a;
  p.d.ws = (float *)at;
  p.d.arrive_end = (unsigned long long *)(at + m.d.records + m.d.words);
  p.d.tag = p.f.tag = next_tag();
  p.d.bins = m.d.bins; p.d.hblocks = m.d.hblocks; p.d.columns = m.d.columns;
  p.d.k0 = a.prefix_len;
  p.d.parts = (float *)(at + m.d.records + m.d.words);
  p.f.ws = (float *)(at + m.d.records + m.d.words + m.own);
  p.d.cuts = (int *)(at + m.d.records + m.d.words + m.own + m.records);
  p.f.arrive_end = nullptr;
  p.f.slots = 0;
  p.f.prefix_parts = m.parts;
  p.n_dec = m.d.bins * m.d.columns;
  p.n_pre = (int)m.n_pre;
  const dim3 grid((unsigned)(((p.n_dec + 7) / 8 + (m.n_pre + 7) / 8) * 8)), block(256);
  if (dtype == BN_F32) hipLaunchKernelGGL(paged_shared_f32_kernel, grid, block, 0, s, p);
  else if (m.hw == 8) hipLaunchKernelGGL(paged_shared_pipe_kernel, grid, block, 0, s, p);
  else hipLaunchKernelGGL((paged_shared_bf16_kernel<1, 4>), grid, block, 0, s, p);
  BN_LAUNCH_CHECK();
  const int64_t pairs = (int64_t)a.c.batch * a.n_heads * (HD / 2);
  const dim3 add((unsigned)((pairs + 255) / 256));
  if (dtype == BN_F32) hipLaunchKernelGGL(paged_shared_add_kernel<float>, add, block, 0, s, p, 32 * m.hw);
  else hipLaunchKernelGGL(paged_shared_add_kernel<bf16_t>, add, block, 0, s, p, 32 * m.hw);
  BN_LAUNCH_CHECK();
  return BN_OK;
}

// The threads of a call's launches, which the runtime counts in 32 bits.
int check_launch(const std::string &op, int dtype, int batch, const int32_t *starts, int n_rows, int n_heads,
                 int n_kv_heads, int cap, int prefix_len) {
  int64_t threads = 0;
  if (prefix_len > 0) {
    const SharedPlan m = plan_shared(dtype, batch, n_heads, n_kv_heads, prefix_len);
    threads = std::max((m.d.bins * m.d.columns + m.n_pre + 16) * 256, (int64_t)batch * n_heads * (HD / 2) + 256);
  } else if (starts) {
    threads = prefill_threads(dtype, batch, n_rows, n_heads, n_kv_heads, cap);
  }
  if (threads >= (int64_t)1 << 32)
    return fail(BN_ERR_UNSUPPORTED, op + ": too many rows and sequences for one launch (2^32 threads)");
  return BN_OK;
}

int attention(const char *name, const bn_paged_kv *kv, const void *q, void *o, const int32_t *starts,
              int n_rows, int n_heads, int64_t q_rs, int64_t o_rs, float scale,
              const int32_t *prefix_pages, int prefix_len, void *workspace, size_t workspace_bytes,
              void *stream) {
  const std::string op = name;
  AttnParams p;
  int st = check_cache(op, kv, &p.c);
  if (st || (st = check_heads(op, n_heads, kv->n_kv_heads, n_rows)) ||
      (st = check_starts(op, starts, n_rows, kv->batch)))
    return st;
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(BN_ERR_INVALID_ARG, op + ": scale must be positive and finite");
  if (prefix_len < 0 || prefix_len > (1 << 30))
    return fail(BN_ERR_SHAPE, op + ": prefix length must be in [0, 2^30]");
  if (n_rows == 0 || kv->batch == 0) return BN_OK;
  if ((st = check_rows(op, "q", q, n_rows, n_heads, q_rs, kv->dtype)) ||
      (st = check_rows(op, "o", o, n_rows, n_heads, o_rs, kv->dtype)))
    return st;
  if (prefix_len > 0 && !prefix_pages) return fail(BN_ERR_INVALID_ARG, op + ": prefix_pages is NULL");
  if ((uintptr_t)prefix_pages & 3u)
    return fail(BN_ERR_UNSUPPORTED, op + ": prefix_pages must be 4-byte aligned");
  p.prefix_len = std::min(prefix_len, p.c.cap);
  if ((st = check_launch(op, kv->dtype, kv->batch, starts, n_rows, n_heads, kv->n_kv_heads, p.c.cap, p.prefix_len)))
    return st;
  const size_t need = bn_paged_workspace_size(kv, n_heads, n_rows, prefix_len);
  if (workspace && workspace_bytes < need)
    return fail(BN_ERR_INVALID_ARG, op + ": workspace of " + std::to_string(workspace_bytes) +
                                        " bytes, need " + std::to_string(need));
  if (workspace && !aligned16(workspace))
    return fail(BN_ERR_UNSUPPORTED, op + ": workspace must be 16-byte aligned");
  DeviceScope scope;
  if ((st = scope.enter(op, kv->seq_lens))) return st;
  p.q = q; p.o = o; p.starts = starts;
  p.q_rs = q_rs; p.o_rs = o_rs;
  p.n_rows = n_rows; p.n_heads = n_heads; p.group = n_heads / kv->n_kv_heads;
  p.inv_group = 1.0f / (float)p.group;
  p.cl = scale * kLog2e;
  p.prefix_pages = prefix_pages;
  Workspace ws;
  if ((st = ws.take(workspace, need, stream))) return st;
  hipStream_t s = as_stream(stream);
  return ws.release(p.prefix_len > 0 ? launch_shared(p, kv->dtype, ws.p, s)
                    : starts         ? launch_prefill(p, kv->dtype, ws.p, s)
                                     : launch_decode(p, kv->dtype, ws.p, s));
}

}  // namespace
}  // namespace bn

using namespace bn;

extern "C" {

int bn_paged_append(const bn_paged_kv *cache, const void *k, const void *v, const void *q, void *q_out,
                    const int32_t *row_starts, int n_rows, int n_heads, int64_t k_row_stride,
                    int64_t v_row_stride, int64_t q_row_stride, int64_t q_out_row_stride, float theta,
                    void *stream) {
  const std::string op = "Paged append";
  AppendParams p;
  int st = check_cache(op, cache, &p.c);
  if (st || (st = check_starts(op, row_starts, n_rows, cache->batch))) return st;
  if (!q != !q_out) return fail(BN_ERR_INVALID_ARG, op + ": q and q_out must be given together");
  if (q && (st = check_heads(op, n_heads, cache->n_kv_heads, n_rows))) return st;
  if (n_rows > (1 << 23)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^23 rows");
  if (!(theta >= 0.f) || !std::isfinite(theta))
    return fail(BN_ERR_INVALID_ARG, op + ": theta must be positive and finite, or 0 for no rotation");
  if (n_rows == 0 || cache->batch == 0) return BN_OK;
  if ((st = check_rows(op, "k", k, n_rows, cache->n_kv_heads, k_row_stride, cache->dtype)) ||
      (st = check_rows(op, "v", v, n_rows, cache->n_kv_heads, v_row_stride, cache->dtype)) ||
      (q && ((st = check_rows(op, "q", q, n_rows, n_heads, q_row_stride, cache->dtype)) ||
             (st = check_rows(op, "q_out", q_out, n_rows, n_heads, q_out_row_stride, cache->dtype)))))
    return st;
  if (q == q_out && q && q_row_stride != q_out_row_stride)
    return fail(BN_ERR_INVALID_ARG, op + ": q_out in q's place must have its row stride");
  DeviceScope scope;
  if ((st = scope.enter(op, cache->seq_lens))) return st;
  p.k = k; p.v = v; p.q = q; p.qo = q_out; p.starts = row_starts;
  p.k_rs = k_row_stride; p.v_rs = v_row_stride; p.q_rs = q_row_stride; p.qo_rs = q_out_row_stride;
  p.n_heads = q ? n_heads : 0;
  p.turn = theta > 0.f;
  for (int i = 0; i < HD / 2; ++i)
    p.f[i] = theta > 0.f ? std::pow((double)theta, -2.0 * i / HD) / (2.0 * M_PI) : 0.0;
  hipStream_t s = as_stream(stream);
  const int pieces = (p.n_heads + 2 * cache->n_kv_heads) * HD * (cache->dtype == BN_BF16 ? 2 : 4) / 16;
  const dim3 grid(n_rows), block(std::min(256, (pieces + 127) / 128 * 64));
  if (cache->dtype == BN_BF16) hipLaunchKernelGGL(paged_append_kernel<bf16_t>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(paged_append_kernel<float>, grid, block, 0, s, p);
  BN_LAUNCH_CHECK();
  return BN_OK;
}

size_t bn_paged_workspace_size(const bn_paged_kv *cache, int n_heads, int n_rows, int prefix_len) {
  Paged c;
  if (n_rows <= 0 || prefix_len < 0 || !cache || check_cache("", cache, &c) || cache->batch == 0 ||
      check_heads("", n_heads, cache->n_kv_heads, n_rows))
    return 0;
  const DecodePlan d = plan_decode(cache->batch, n_heads, cache->n_kv_heads);
  const PrefillPlan f = plan_prefill(cache->dtype, cache->batch, n_rows, n_heads, cache->n_kv_heads, c.cap, true);
  size_t need = std::max(d.records + d.words, f.records + f.words);
  if (prefix_len > 0) {
    const SharedPlan s = plan_shared(cache->dtype, cache->batch, n_heads, cache->n_kv_heads, std::min(prefix_len, c.cap));
    need = std::max(need, s.d.records + s.d.words + s.own + s.records + s.cuts);
  }
  return need;
}

int bn_paged_decode(const bn_paged_kv *cache, const void *q, void *o, int n_heads, int64_t q_row_stride,
                    int64_t o_row_stride, float scale, void *workspace, size_t workspace_bytes,
                    void *stream) {
  return attention("Paged decode", cache, q, o, nullptr, cache ? cache->batch : 0, n_heads, q_row_stride,
                   o_row_stride, scale, nullptr, 0, workspace, workspace_bytes, stream);
}

int bn_paged_prefill(const bn_paged_kv *cache, const void *q, void *o, const int32_t *row_starts,
                     int n_rows, int n_heads, int64_t q_row_stride, int64_t o_row_stride, float scale,
                     void *workspace, size_t workspace_bytes, void *stream) {
  return attention("Paged prefill", cache, q, o, row_starts, n_rows, n_heads, q_row_stride, o_row_stride,
                   scale, nullptr, 0, workspace, workspace_bytes, stream);
}

int bn_paged_decode_shared(const bn_paged_kv *cache, const void *q, void *o, int n_heads,
                           int64_t q_row_stride, int64_t o_row_stride, float scale,
                           const int32_t *prefix_pages, int prefix_len, void *workspace,
                           size_t workspace_bytes, void *stream) {
  return attention("Paged decode (shared prefix)", cache, q, o, nullptr, cache ? cache->batch : 0, n_heads,
                   q_row_stride, o_row_stride, scale, prefix_pages, prefix_len, workspace,
                   workspace_bytes, stream);
}

}  // extern "C"
