// bn_paged_q8.hip -- the paged KV cache in 8 bits: e4m3 codes under a power of
// two for every 16 keys of a page and KV head.  Appending (norms, rotation,
// rounding), reading back, and the attention over the pages.
//
// A float's e4m3 code has its relative precision, 2^-4, wherever the scale puts
// it above 2^-6, so nothing is gained by a finer scale than a power of two; and
// with that every value is a bf16 number, a scale that grows leaves older codes'
// values as they are (but for those that become subnormal), and the attention's
// kernels are those of the bf16 cache behind the conversion.
#include "bn_head_rows.hpp"
#include "bn_paged_host.hpp"
#include "bn_q8_plan.hpp"

namespace bn {
namespace {

constexpr int kBlock = BN_Q8_BLOCK;
constexpr int kLow = 10, kHigh = 247;  // scale bytes

// The cache as the kernels see it.
struct Q8 {
  Paged c;  // strides of the codes, in bytes
  uint8_t *ks, *vs;
  int64_t scale_page, scale_head;
};

// 2^(byte - 127)
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((uint32_t)min(max(byte, kLow), kHigh) << 23); }
// Codes 2 HALF and 2 HALF + 1 of four, as values.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <bool HALF>
__device__ __forceinline__ f32x2 two_values(uint32_t codes, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, HALF);
}
__device__ __forceinline__ Eight values(u32x2 codes, float scale) {
  Eight y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = two_values<false>(codes[i], scale), b = two_values<true>(codes[i], scale);
    y.x[4 * i] = a[0]; y.x[4 * i + 1] = a[1]; y.x[4 * i + 2] = b[0]; y.x[4 * i + 3] = b[1];
  }
  return y;
}
// The smallest scale byte with which |x| up to amax (finite) is at most 448.
__device__ __forceinline__ int byte_of(float amax) {
  const uint32_t u = __float_as_uint(amax);
  // amax = 1.m 2^(E - 127) <= 1.75 2^8 2^n: n = E - 127 - 8, one more where 1.m is above 1.75
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return min(max(e, kLow), kHigh);
}
__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
// Eight codes of x under the scale of a byte.
__device__ __forceinline__ u32x2 codes_of(const Eight &x, int byte) {
  const float inverse = __uint_as_float((uint32_t)(254 - byte) << 23), most = byte == kHigh ? 240.f : 448.f;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = fminf(fmaxf(x.x[i] * inverse, -most), most);
    y[i] = fabsf(x.x[i]) < INFINITY ? s : NAN;
  }
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    r[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], w, true);
  }
  return r;
}

// ------------------------------------------------------ a call's units of work
// A unit: the rows of a call that fall into one block of a sequence, so that one
// workgroup sees all of a block that the call writes.
struct Unit {
  int row0, rows;  // of the tensors; rows <= 16
  int b;
  int64_t pos0;    // position of row0
};
// Sequence b's units have numbers from (starts[b] - starts[0]) / 16 + 2 b on, of
// which n rows never need more than n / 16 + 2: the sequence is found by a search
// among 64 at a time, and numbers without a unit are left out.  False: none.
__device__ __forceinline__ bool find_unit(const Paged &c, const int32_t *starts, int n_rows, int number, Unit &u) {
  if (!starts) {
    u.b = u.row0 = number;
    u.rows = 1;
    u.pos0 = (int64_t)max(c.lens[number], 0) - 1;
    return true;
  }
  const int lane = threadIdx.x & 63;
  auto start = [&](int b) { return min(max(starts[b], 0), n_rows); };
  const int s0 = start(0);
  auto first_of = [&](int b) { return ((start(b) - s0) >> 4) + 2 * b; };
  int lo = 0, hi = c.batch;  // first_of(lo) <= number, and number < first_of(hi) unless it is past all
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6, at = lo + step * lane;
    const unsigned long long below =
        __builtin_amdgcn_ballot_w64(at < hi && first_of(min(at, c.batch)) <= number);
    const int n = __builtin_popcountll(below);
    if (n == 0) return false;  // (starts that decrease)
    lo = lo + step * (n - 1);
    hi = min(hi, lo + step);
  }
  const int j = number - first_of(lo);
  const int from = start(lo), to = start(lo + 1);
  if (j < 0 || to <= from) return false;
  // (starts[lo + 1] may lie past the tensors' rows)
  const int64_t p0 = (int64_t)max(c.lens[lo], 0) - starts[lo + 1] + from, end = p0 + (to - from);
  const int64_t block0 = ((p0 >> 4) + j) * kBlock;
  if (block0 >= end) return false;
  const int64_t p = block0 > p0 ? block0 : p0, q = block0 + kBlock < end ? block0 + kBlock : end;
  u.b = lo;
  u.row0 = from + (int)(p - p0);
  u.rows = (int)(q - p);
  u.pos0 = p;
  return true;
}
int64_t count_units(const int32_t *starts, int n_rows, int batch) {
  return starts ? (int64_t)n_rows / kBlock + 2 * (int64_t)batch : batch;
}

// Where a unit's rows lie: byte offsets of its first slot and of its block's scale
// in KV head 0 (-1: the block has no memory).
struct Place {
  int64_t codes, scale;
  int slot;  // of the first row in its block
};
__device__ __forceinline__ Place place_of(const Q8 &q, const Unit &u) {
  Place p{-1, -1, (int)(u.pos0 & (kBlock - 1))};
  // (a block lies within the table or outside it as a whole)
  if (u.pos0 < 0 || u.pos0 >= q.c.cap) return p;
  const int pos = (int)u.pos0, page = q.c.table[u.b * q.c.table_stride + (pos >> q.c.shift)];
  if ((unsigned)page >= (unsigned)q.c.n_pages) return p;
  const int in_page = pos & ((1 << q.c.shift) - 1);
  p.codes = page * q.c.page_stride + in_page * q.c.row_stride;
  p.scale = page * q.scale_page + (in_page >> 4);
  return p;
}

// ------------------------------------------------------------------ append
struct Q8AppendParams {
  Q8 s;
  const void *k, *v, *q, *wq, *wk;
  void *qo;
  const int32_t *starts;
  int64_t k_rs, v_rs, q_rs, qo_rs;
  int n_rows, n_heads, turn;  // n_heads: 0 without q
  float eps;
  double f[HD / 2];  // turns per position of each pair
};

// A unit a workgroup.  Its rows' angles once, while the first pieces of queries and
// the first task's rows are on their way; then its waves take the block's KV heads, K
// and V, in turn, 16 rows of 64 elements in two pieces of eight a lane: norm,
// rotation, the block's largest element, the scale, the codes.  The queries' pieces go
// to all threads.  Bound by memory, VALU 68% busy: 4 x 2048 rows of 32 and 4 heads 19.4 us
// under the profiler, 4.1 TB/s; 64 rows 5.2, launch and the chain row -> length -> table ->
// scale.  (Four waves, every row loaded when its turn comes: 24 and 6.)
constexpr int kAppendThreads = 512, kPieces = 4;
template <typename T>
__global__ __launch_bounds__(kAppendThreads) void paged_q8_append_kernel(Q8AppendParams p) {
  __shared__ float2 cs[kBlock][HD / 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Paged &c = p.s.c;
  Unit u;
  if (!find_unit(c, p.starts, p.n_rows, blockIdx.x, u)) return;
  const int e = lane % 8 * 8, per = p.n_heads * 8, total = u.rows * per, tasks = 2 * c.n_kv_heads;
  Walk at_q(tid, kAppendThreads, max(per, 1));
  Raw8<T> qx[kPieces];
  int q_row[kPieces], q_at[kPieces];
  auto load_q = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      if (first + kAppendThreads * n >= total) break;
      q_row[n] = at_q.row;
      q_at[n] = at_q.rest * 8;
      at_q.step();
      qx[n].load((const T *)p.q + (int64_t)(u.row0 + q_row[n]) * p.q_rs + q_at[n]);
    }
  };
  Raw8<T> kx[2];
  auto load_kv = [&](int task) __attribute__((always_inline)) {
    const bool is_v = task >= c.n_kv_heads;
    const T *const x = (is_v ? (const T *)p.v : (const T *)p.k) + (task - (is_v ? c.n_kv_heads : 0)) * HD + e;
#pragma unroll
    for (int n = 0; n < 2; ++n)
      if (lane / 8 + 8 * n < u.rows) kx[n].load(x + (int64_t)(u.row0 + lane / 8 + 8 * n) * (is_v ? p.v_rs : p.k_rs));
  };
  if (wave < tasks) load_kv(wave);
  load_q(tid);
  const Place at = place_of(p.s, u);
  if (p.turn) {
    for (int i = tid; i < u.rows * (HD / 2); i += kAppendThreads)
      cs[i / (HD / 2)][i % (HD / 2)] = cos_sin((double)(u.pos0 + i / (HD / 2)) * p.f[i % (HD / 2)]);
    __syncthreads();
  }
  auto normed = [&](Eight &x, const void *w) __attribute__((always_inline)) {
    const float r = head_rms<8>(x, p.eps);
    Raw8<T> wr;
    wr.load((const T *)w + e);
    const Eight y = wr.floats();
#pragma unroll
    for (int j = 0; j < 8; ++j) x.x[j] *= r * y.x[j];
  };
  if (at.codes >= 0) {
    for (int task = wave; task < tasks; task += kAppendThreads / 64) {
      if (task != wave) load_kv(task);
      const bool is_v = task >= c.n_kv_heads;
      const int g = is_v ? task - c.n_kv_heads : task;
      uint8_t *const codes = (uint8_t *)(is_v ? c.v : c.k) + at.codes + g * c.head_stride;
      uint8_t *const scale = (is_v ? p.s.vs : p.s.ks) + at.scale + g * p.s.scale_head;
      const int before = at.slot > 0 ? min(max((int)*scale, kLow), kHigh) : 0;  // of older rows in the block
      Eight x[2];
      float amax = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int row = lane / 8 + 8 * n;
        if (row < u.rows) {
          x[n] = kx[n].floats();
          if (!is_v) {
            if (p.wk) normed(x[n], p.wk);
            if (p.turn) turn8(x[n], &cs[row][e / 2]);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_size(x[n].x[j]));
        }
      }
      int byte = byte_of(wave_max(amax));
      if (at.slot > 0 && byte > before) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int back = lane / 8 + 8 * n - at.slot;  // rows before the first: negative
          if (back >= 0) continue;
          u32x2 *const row = (u32x2 *)(codes + back * c.row_stride + e);
          *row = codes_of(values(*row, scale_of(before)), byte);
        }
      }
      byte = max(byte, before);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int row = lane / 8 + 8 * n;
        if (row < u.rows) *(u32x2 *)(codes + row * c.row_stride + e) = codes_of(x[n], byte);
      }
      if (lane == 0) *scale = (uint8_t)byte;
    }
  }
  for (int first = tid; first < total; first += kAppendThreads * kPieces) {
    if (first != tid) load_q(first);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      if (first + kAppendThreads * n >= total) break;
      Eight x = qx[n].floats();
      if (p.wq) normed(x, p.wq);
      if (p.turn) turn8(x, &cs[q_row[n]][e / 2]);
      store8((T *)p.qo + (int64_t)(u.row0 + q_row[n]) * p.qo_rs + q_at[n], x);
    }
  }
}

// -------------------------------------------------------------------- read
struct Q8ReadParams {
  Q8 s;
  void *k, *v;
  const int32_t *starts;
  int64_t k_rs, v_rs;
  int n_rows;
};
// A unit a workgroup, its waves the block's KV heads, K and V, in turn.  Bound by memory: 55782 and 65536
// keys of 4 heads 38 us, 4.9 TB/s read and written, a copy's rate.  NT: codes and rows past the caches'
// keeping, for rows that the memory-side cache (256 MB) would not hold long: 131 MB of them 44.3 -> 40.0
// us, and a sum of keys and values behind it 73.1 -> 72.0 with them; of 65 MB 23.4 -> 22.4, but with that
// sum 37.8 -> 39.9.
template <typename T, bool NT>
__global__ __launch_bounds__(256) void paged_q8_read_kernel(Q8ReadParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Paged &c = p.s.c;
  Unit u;
  if (!find_unit(c, p.starts, p.n_rows, blockIdx.x, u)) return;
  const Place at = place_of(p.s, u);
  const int e = lane % 8 * 8;
  for (int task = wave; task < 2 * c.n_kv_heads; task += 4) {
    const bool is_v = task >= c.n_kv_heads;
    const int g = is_v ? task - c.n_kv_heads : task;
    T *const out = (T *)(is_v ? p.v : p.k);
    if (!out) continue;
    const uint8_t *const codes = (const uint8_t *)(is_v ? c.v : c.k) + at.codes + g * c.head_stride;
    const float scale = at.codes < 0 ? 0.f : scale_of((is_v ? p.s.vs : p.s.ks)[at.scale + g * p.s.scale_head]);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = lane / 8 + 8 * n;
      if (row >= u.rows) continue;
      Eight x{};
      const u32x2 *const from = (const u32x2 *)(codes + row * c.row_stride + e);
      if (at.codes >= 0) x = values(NT ? __builtin_nontemporal_load(from) : *from, scale);
      store8<T, NT>(out + (int64_t)(u.row0 + row) * (is_v ? p.v_rs : p.k_rs) + g * HD + e, x);
    }
  }
}

// --------------------------------------------------------------- attention
// The other caches' kernels over codes: eight elements become bf16 in four
// instructions, their scale an operand, where the bf16 cache's are stored to LDS
// (prefill) or where the products' operands are read from it (decode); and four
// elements fp32 in two for queries in fp32.
struct E4m3Scales {
  typedef uint8_t T;
  static constexpr bool kScaled = true;
  const uint8_t *ks, *vs;
  int64_t page, head;
  __device__ __forceinline__ const uint8_t *scales(int g, bool values) const { return (values ? vs : ks) + g * head; }
  // the byte of the block of key k of page id (no page: page 0's)
  __device__ __forceinline__ int scale(const uint8_t *base, const PageRows &rows, int id, int k) const {
    return base[(rows.there(id) ? id : 0) * page + ((k & rows.slot_mask) >> 4)];
  }
  __device__ __forceinline__ int scale_bits(int byte) const { return min(max(byte, kLow), kHigh) << 23; }
  __device__ __forceinline__ float value(const PageRows &rows, const char *Vg, int g, int id, int k, int lane) const {
    const uint8_t code = ((const uint8_t *)Vg + rows.at(id, k))[lane];
    return two_values<false>(code, scale_of(scale(scales(g, true), rows, id, k)))[0];
  }
};
struct E4m3Pages : E4m3Scales {  // as bf16
  typedef u32x2 Raw;
  __device__ __forceinline__ u32x4 bf16(uint32_t lo, uint32_t hi, float scale) const {
    u32x4 y;
    y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return y;
  }
  __device__ __forceinline__ u32x4 piece(Raw x, int bits) const { return bf16(x[0], x[1], __builtin_bit_cast(float, bits)); }
};
struct E4m3PagesF32 : E4m3Scales {  // as fp32
  typedef uint32_t Raw;
  typedef uint16_t Pair;
  __device__ __forceinline__ u32x4 piece(Raw x, int bits) const {
    const float scale = __builtin_bit_cast(float, bits);
    const f32x2 a = two_values<false>(x, scale), b = two_values<true>(x, scale);
    return u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
  }
  __device__ __forceinline__ float2 pair(Pair x, int bits) const {
    const f32x2 a = two_values<false>(x, __builtin_bit_cast(float, bits));
    return make_float2(a[0], a[1]);
  }
};

// ------------------------------------------------------------------ decode
// The batch's tiles of 64 keys, sequences in order, are dealt in equal shares to the
// workgroups of a column (a KV head, or up to 16 of its query heads).  A
// workgroup finds the sequences of its share by a scan of the lengths, one thread a
// run of them, and lists them in LDS; its eight waves take a run of the listed tiles
// each, with the next tile's rows on their way, leave their parts of each sequence
// (reference, sum, accumulator) in LDS and add them up; then the next list, if the
// share has more sequences than LDS holds parts of.  A sequence cut between shares
// leaves records, which the last of its pieces to arrive adds, in the order of the keys.
// What lies where -- page offsets, scales -- a wave looks up for 64 of its tiles at
// once, a tile a lane, so that a step has only to read it from there: with lookups and
// the walk over sequences in every step (650 instructions a tile, four waves) the
// instructions bounded the kernel, 31.9 us for 64 caches of 512..4096 keys.
//
// Per tile, with the query heads as columns of the products, as the bf16 cache's:
//   S^T[key][head] = K . Q^T,  O^T[d][head] += V^T . P^T   (v_mfma_f32_16x16x32_bf16)
// K's operand is sixteen codes of a row and V's a transposing read's column of
// eight rows, both converted (exactly) where they are used, the scale an operand.  A
// score tile's rows are keys 4 (u % 2) + 8 (row / 4) + row % 4 of its 32, so that a
// lane's scores of two tiles are those of eight keys in a row, V's operand's order.
//
// Bound by memory, and for small calls by the chain lengths -> list -> table -> rows ->
// parts -> records: 64 caches of 4096 keys (32 and 4 heads) 29.9 us, 4.5 TB/s; of 512..4096
// 22.5, 3.5 TB/s, of which 6 are that chain and 3 the records; three of 34763 to 131072 34.8,
// three of 5003 to 131072 30, 4.2 TB/s; one of 640 9.4.  Four waves and two tiles each in flight,
// before the probabilities were two values: 31.5 and 41.8 us for the second and third.  (Matrix cores 8
// to 11%, VALU 37 to 39%, LDS 25 to 29% busy.)
constexpr int kWaves = 8, kTile = 64;
constexpr int kListed = 32;                  // sequences of a list
constexpr int kHoldParts = 256;              // rows of LDS for the waves' parts of sequences
constexpr int kPitch = HD + 16;              // bytes of a row in LDS: b128 reads of 16 rows spread over the banks
constexpr int kRows16 = 16 * kPitch + 64;    // sixteen rows, and 64 bytes so that rows 16 apart do too
constexpr int kHoldRow = HD + 4;             // floats of a part's row: a record's, 16-byte aligned
constexpr int kShareLeast = 8;               // tiles of a share at least: one a wave (1 cache of 16384 keys 13.8 us, with 4 tiles 17.6)
constexpr int kMerged = 16;                  // records read at once
struct Q8DecodeLds {
  uint8_t k[kWaves][4 * kRows16], v[kWaves][4 * kRows16];
  float hold[kHoldParts * kHoldRow];
  int list_b[kListed], list_first[kListed], list_len[kListed];  // sequence, position of its first tile, keys
  int sums[2][kWaves], rank0, last_in[2];
};

// ONCE: rows past the caches' keeping (decode_reads_once).
template <bool ONCE>
__global__ __launch_bounds__(64 * kWaves) void paged_q8_decode_kernel(DecodeParams p, E4m3Pages src) {
  __shared__ __attribute__((aligned(16))) Q8DecodeLds lds;
  const Paged &c = p.a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, grp = lane >> 4;
  // A share's columns go to one XCD (workgroups are dealt to the eight in turn): they read the same
  // table entries, and of token-major pages the same 128-byte lines.
  int bin, col;
  if ((p.bins & 7) == 0) {
    const int j = blockIdx.x >> 3, r = (int)((uint32_t)j / (uint32_t)p.columns);
    col = j - r * p.columns;
    bin = 8 * r + (blockIdx.x & 7);
  } else {
    bin = blockIdx.x / p.columns;
    col = blockIdx.x - bin * p.columns;
  }
  const int g = col / p.hblocks, hb = col - g * p.hblocks;
  const int rows = min(kMaxRows, p.a.group - kMaxRows * hb), head0 = g * p.a.group + kMaxRows * hb;

  // ---- the share
  auto tiles_of = [](int len) { return (int)((uint32_t)(len + kTile - 1) / kTile); };
  const int per = (c.batch + 64 * kWaves - 1) / (64 * kWaves), from = min(tid * per, c.batch), to = min(from + per, c.batch);
  const int len0 = from < to ? c.lens[from] : 0;  // (the only one up to 512 sequences)
  auto keys_of = [&](int b) __attribute__((always_inline)) { return max(min(b == from ? len0 : c.lens[b], c.cap), 0); };
  int own = 0, some = 0;  // tiles of the thread's run of sequences; sequences of it that have any
#pragma unroll 8
  for (int b = from; b < to; ++b) {
    const int t = tiles_of(keys_of(b));
    own += t;
    some += t > 0;
  }
  int upto = wave_scan(own), rank = wave_scan(some);
  if (lane == 63) {
    lds.sums[0][wave] = upto;
    lds.sums[1][wave] = rank;
  }
  if (tid == 0) lds.rank0 = 0;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    const int t = lds.sums[0][v], r = lds.sums[1][v];
    total += t;
    upto += v < wave ? t : 0;
    rank += v < wave ? r : 0;
  }
  upto -= own;
  rank -= some;  // before the thread's run
  const int share =
      __builtin_amdgcn_readfirstlane(max((int)((uint32_t)(total + p.bins - 1) / (uint32_t)p.bins), kShareLeast));
  const int pos0 = (int)min((int64_t)bin * share, (int64_t)total), end = min(pos0 + share, total);

  auto write2 = [&](int b, int h, int d, float x, float y, float sum) __attribute__((always_inline)) {
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    *(uint32_t *)((bf16_t *)p.a.o + b * p.a.o_rs + (head0 + h) * HD + d) =
        (uint32_t)f32_to_bf16(x * inv) | ((uint32_t)f32_to_bf16(y * inv) << 16);
  };
  // row h of the record of a sequence's piece in bin `at` (a bin has two: the end
  // of a sequence begun before it, and the start of one, begun in bin0, that goes on)
  auto record = [&](int at, int bin0, int h) __attribute__((always_inline)) {
    return p.ws + ((((int64_t)at * 2 + (at == bin0)) * p.columns + col) * kMaxRows + h) * kRec;
  };
  const int pairs = (rows + 1) >> 1;  // results are formed two rows a wave
  auto by_pairs = [&](int u) __attribute__((always_inline)) {  // u / pairs (u up to 32 * 8, pairs up to 8)
    return (int)(((uint32_t)u * (uint32_t)(65536 / pairs + 1)) >> 16);
  };
  struct Cut {  // a sequence that is cut between shares: its first bin and its number of pieces, one a bin
    int b, bin0, pieces;
  };
  Cut cuts[2] = {{0, 0, 0}, {0, 0, 0}};  // one that began before the share, one that goes on

  if (pos0 < end) {
    // the first sequence's number among those that have tiles
    if (upto <= pos0 && pos0 < upto + own) {
      int at = upto, r = rank;
      for (int b = from; b < to; ++b) {
        const int t = tiles_of(keys_of(b));
        if (at + t > pos0) break;
        at += t;
        r += t > 0;
      }
      lds.rank0 = r;
    }
    const uint32_t off = (uint32_t)((lane >> 2) * c.row_stride + (lane & 3) * 16);
    const char *const Kg = (const char *)c.k + g * c.head_stride, *const Vg = (const char *)c.v + g * c.head_stride;
    const uint8_t *const ksg = src.scales(g, false), *const vsg = src.scales(g, true);
    const PageRows pages = PageRows::of<uint8_t>(c);
    uint8_t *const kt = lds.k[wave], *const vt = lds.v[wave];
    const float cl = p.a.cl;

    int at = pos0, listed = 0;                // the share's tiles and sequences that are through
    int wb = from, wfirst = upto, wrank = rank;  // the thread's first sequence that is not
    for (;;) {
      // ---- the list: the next sequences of the share
      if (tid < kListed) lds.list_b[tid] = -1;
      __syncthreads();
      if (upto < end && upto + own > at) {
        for (int t; wb < to && wfirst + (t = tiles_of(keys_of(wb))) <= at; ++wb) {
          wfirst += t;
          wrank += t > 0;
        }
        int first = wfirst, r = wrank - lds.rank0 - listed;
        for (int b = wb; b < to && first < end && r < kListed; ++b) {
          const int len = keys_of(b), t = tiles_of(len);
          if (t > 0) {
            lds.list_b[r] = b;
            lds.list_first[r] = first;
            lds.list_len[r] = len;
          }
          first += t;
          r += t > 0;
        }
      }
      __syncthreads();
      // lane l: the list's l-th sequence
      const int lb = lds.list_b[lane & (kListed - 1)], lfirst = lds.list_first[lane & (kListed - 1)],
                llen = lds.list_len[lane & (kListed - 1)];
      // A wave takes a run of the list's tiles, so that sequence l and wave w meet in a staircase: each of
      // their parts has place l + w, and LDS holds the parts of kHoldParts / rows - 7 sequences.
      const bool there = lane < min(kListed, kHoldParts / rows - (kWaves - 1)) && lb >= 0;
      const int lend = there ? lfirst + tiles_of(llen) : 0, lstop = min(lend, end);
      const int n_list = __builtin_popcountll(__builtin_amdgcn_ballot_w64(there));
      const int stop = __builtin_amdgcn_readlane(lstop, n_list - 1);
      const int run = (int)((uint32_t)(stop - at + kWaves - 1) / kWaves);
      const int lw0 = there ? (int)((uint32_t)(max(lfirst, at) - at) / (uint32_t)run) : 0;  // its first and last wave
      const int lw1 = there ? (int)((uint32_t)(lstop - 1 - at) / (uint32_t)run) : 0;

      // ---- the wave's tiles, looked up 64 at a time
      const int mine = at + wave * run, n = max(min(run, stop - mine), 0);
      uint32_t at_lo[4], at_hi[4];  // byte offset of rows 16 r ..
      uint32_t kscales, vscales;    // bytes of rows 16 r ..
      int info, first_keys;         // place in the list | bits 8 ..: rows 16 r .. have memory; keys of the tile
      auto look_up = [&](int i0) __attribute__((always_inline)) {
        const int pos = min(mine + i0 + lane, stop - 1);
        int place = 0;
        for (int l = 0; l < n_list - 1; ++l) place += pos >= __builtin_amdgcn_readlane(lstop, l);
        const int b = lds.list_b[place], len = lds.list_len[place], key0 = kTile * (pos - lds.list_first[place]);
        const int32_t *const table = c.table + b * c.table_stride;
        info = place;
        first_keys = min(len - key0, kTile);
        int id[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) id[r] = table[(uint32_t)min(key0 + 16 * r, len - 1) >> c.shift];
        kscales = vscales = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          info |= pages.there(id[r]) << (8 + r);
          const uint64_t x = pages.at(id[r], key0 + 16 * r);
          at_lo[r] = (uint32_t)x;
          at_hi[r] = (uint32_t)(x >> 32);
          kscales |= (uint32_t)min(max(src.scale(ksg, pages, id[r], key0 + 16 * r), kLow), kHigh) << (8 * r);
          vscales |= (uint32_t)min(max(src.scale(vsg, pages, id[r], key0 + 16 * r), kLow), kHigh) << (8 * r);
        }
      };
      struct Tile {  // in flight: its rows' pieces, 16 rows an instruction
        u32x4 k[4], v[4];
        int info, keys;
      } x;
      auto load = [&](int i) __attribute__((always_inline)) {
        const int j = i & 63;
        x.info = __builtin_amdgcn_readlane(info, j);
        x.keys = __builtin_amdgcn_readlane(first_keys, j);
        uint32_t o32 = off;
        asm volatile("" : "+v"(o32));  // a scalar base and this offset, not a sum of pointers kept in registers
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint64_t to_row = (uint32_t)__builtin_amdgcn_readlane(at_lo[r], j) |
                                  (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi[r], j) << 32;
          const u32x4 *const kp = (const u32x4 *)(Kg + to_row + o32), *const vp = (const u32x4 *)(Vg + to_row + o32);
          x.k[r] = ONCE ? __builtin_nontemporal_load(kp) : *kp;
          x.v[r] = ONCE ? __builtin_nontemporal_load(vp) : *vp;
        }
      };
      u32x4 q[2], qn[2];  // head l16's elements 16 grp .. + 15
      auto load_q = [&](int place) __attribute__((always_inline)) {
        const bf16_t *const qp = (const bf16_t *)p.a.q + (int64_t)__builtin_amdgcn_readlane(lb, place) * p.a.q_rs +
                                 (head0 + min(l16, rows - 1)) * HD + 16 * grp;
        qn[0] = *(const u32x4 *)qp;
        qn[1] = *(const u32x4 *)(qp + 8);
      };
      float mc = -INFINITY, sum = 0.f;  // of head l16: reference, log2 units; this lane's keys' sum
      f32x4 o[4];
      bool fresh = true;
      if (n > 0) {
        look_up(0);
        load(0);
        load_q(x.info & 255);
      }
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int place = x.info & 255, have = x.info >> 8 & 15, keys = x.keys;
        const uint32_t ks = __builtin_amdgcn_readlane(kscales, i & 63), vs = __builtin_amdgcn_readlane(vscales, i & 63);
        // a wave's LDS instructions execute in order, so its tile needs no
        // barrier; wave_barrier keeps the compiler from moving them across
        __builtin_amdgcn_wave_barrier();
        if (keys < kTile || have != 15) {  // no key: zeros, whatever lies there
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((lane >> 2) + 16 * r >= keys || !(have >> r & 1)) x.k[r] = x.v[r] = u32x4{0, 0, 0, 0};
        }
        {
          uint8_t *const kd = kt + (lane >> 2) * kPitch + (lane & 3) * 16, *const vd = vt + (lane >> 2) * kPitch + (lane & 3) * 16;
#pragma unroll
          for (int r = 0; r < 4; ++r) *(u32x4 *)(kd + r * kRows16) = x.k[r];
#pragma unroll
          for (int r = 0; r < 4; ++r) *(u32x4 *)(vd + r * kRows16) = x.v[r];
        }
        __builtin_amdgcn_wave_barrier();
        if (fresh) {
          q[0] = qn[0];
          q[1] = qn[1];
          mc = -INFINITY;
          sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = f32x4{};
        }
        bool ends = i + 1 == n;
        if (!ends) {
          if (((i + 1) & 63) == 0) look_up(i + 1);
          load(i + 1);
          ends = (x.info & 255) != place;
          if (ends) load_q(x.info & 255);
        }
        fresh = ends;
        // scores: s[u][j] of key 32 (u / 2) + 8 grp + 4 (u % 2) + j
        f32x4 s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int row = 8 * (l16 >> 2) + 4 * (u & 1) + (l16 & 3);  // of its 32; its sixteen: l16 / 8
          const u32x4 y = *(const u32x4 *)(kt + (u >> 1) * 2 * kRows16 + row * kPitch + (l16 >> 3) * 64 + 16 * grp);
          const float scale = __uint_as_float((ks >> (16 * (u >> 1) + (l16 & 8)) & 255u) << 23);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, src.bf16(y[0], y[1], scale)),
                                                         __builtin_bit_cast(bf16x8, q[0]), f32x4{}, 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, src.bf16(y[2], y[3], scale)),
                                                         __builtin_bit_cast(bf16x8, q[1]), s[u], 0, 0, 0);
        }
        if (keys < kTile || have != 15) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = 32 * (u >> 1) + 8 * grp + 4 * (u & 1) + j;
              if (key >= keys || !(have >> (key >> 4) & 1)) s[u][j] = -INFINITY;
            }
        }
        // The probabilities are taken against a reference that is the true running maximum only when it was
        // last moved: it moves when a lane's weights against it pass 2^16 in sum (or are NaN).  They enter the
        // products as two bf16 values each, the upper 16 bits and what is left of them (off by at most 2^-16
        // together; rounded to one, 3 caches of up to 131072 keys were 0.0024 off 64 bits, not 0.0017).
        float e[16], rs;
        auto weigh = [&](float ref) __attribute__((always_inline)) {
          rs = 0.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            e[j] = __builtin_amdgcn_exp2f(fmaf(s[j >> 2][j & 3], cl, -ref));
            rs += e[j];
          }
        };
        weigh(mc);  // (no key yet: mc is -inf, and the sum +inf or NaN)
        if (__builtin_amdgcn_ballot_w64(!(rs <= 65536.f)) != 0) {
          float mx = s[0][0];
#pragma unroll
          for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j >> 2][j & 3]);
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float m_new = fmaxf(mc, mx * cl);
          const float ref = m_new == -INFINITY ? 0.f : m_new;  // no key above -inf yet: weights 0
          const float alpha = __builtin_amdgcn_exp2f(mc - ref);
          mc = m_new;
          sum *= alpha;
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
          weigh(ref);
        }
        sum += rs;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 hi;
          bf16x8 lo;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const uint32_t x = __float_as_uint(e[8 * h + j]), y = __float_as_uint(e[8 * h + j + 1]);
            hi[j >> 1] = __builtin_amdgcn_perm(y, x, 0x07060302);
            lo[j] = (__bf16)(e[8 * h + j] - __uint_as_float(x & 0xffff0000u));
            lo[j + 1] = (__bf16)(e[8 * h + j + 1] - __uint_as_float(y & 0xffff0000u));
          }
          // V^T: slot j of lane (grp, l16) is V[key 32 h + 8 grp + j][16 dt + l16]
          const uint8_t *const vp = vt + h * 2 * kRows16 + (8 * grp + (l16 >> 1)) * kPitch + (grp >> 1) * 64 + 8 * (l16 & 1);
          const float scale = __uint_as_float((vs >> (16 * h + 8 * (grp >> 1)) & 255u) << 23);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            const u32x2 y = lds_tr8(vp + 16 * dt);
            const bf16x8 v = __builtin_bit_cast(bf16x8, src.bf16(y[0], y[1], scale));
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, hi), o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, lo, o[dt], 0, 0, 0);
          }
        }
        if (ends) {
          sum += __shfl_xor(sum, 16, 64);
          sum += __shfl_xor(sum, 32, 64);
          if (l16 < rows) {
            float *const h = lds.hold + ((place + wave) * rows + l16) * kHoldRow;
#pragma unroll
            for (int j = 0; j < 4; ++j) *(f32x4 *)(h + 16 * j + 4 * grp) = o[j];
            if (grp == 0) *(float2 *)(h + HD) = make_float2(mc, sum);
          }
        }
      }
      __syncthreads();

      // ---- the listed sequences' parts, added up: two rows a wave, two elements a lane
#pragma unroll 1
      for (int u = wave; u < n_list * pairs; u += kWaves) {
        const int place = by_pairs(u), h = 2 * (u - place * pairs) + (lane >> 5), d = 2 * (lane & 31);
        const int b = __builtin_amdgcn_readlane(lb, place), w0 = __builtin_amdgcn_readlane(lw0, place);
        const int parts = __builtin_amdgcn_readlane(lw1, place) - w0 + 1;
        const int first = __builtin_amdgcn_readlane(lfirst, place), last = __builtin_amdgcn_readlane(lend, place);
        if (h >= rows) continue;
        const float *const r = lds.hold + ((place + w0) * rows + h) * kHoldRow;
        float2 ml[kWaves], y[kWaves];
        float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
          const float *const e = r + min(v, parts - 1) * rows * kHoldRow;
          ml[v] = *(const float2 *)(e + HD);
          y[v] = *(const float2 *)(e + d);
        }
#pragma unroll
        for (int v = 0; v < kWaves; ++v) M = fmaxf(M, ml[v].x);
        const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
          const float f = __builtin_amdgcn_exp2f(ml[v].x - Mu);
          L = v < parts ? fmaf(ml[v].y, f, L) : L;
          A0 = v < parts ? fmaf(y[v].x, f, A0) : A0;
          A1 = v < parts ? fmaf(y[v].y, f, A1) : A1;
        }
        if (first >= pos0 && last <= end) {
          write2(b, h, d, A0, A1, L);
        } else {  // (cut: the only piece of it in this share)
          float *const to_rec = record(bin, first >= pos0 ? bin : -1, h);
          put2(to_rec + d, A0, A1);
          if (d == 0) put2(to_rec + HD, M, L);
        }
      }
      auto cut_of = [&](int place, Cut &u) __attribute__((always_inline)) {
        const int first = __builtin_amdgcn_readlane(lfirst, place), last = __builtin_amdgcn_readlane(lend, place);
        u.b = __builtin_amdgcn_readlane(lb, place);
        u.bin0 = (int)((uint32_t)first / (uint32_t)share);
        u.pieces = (int)((uint32_t)(last - 1) / (uint32_t)share) - u.bin0 + 1;
      };
      if (__builtin_amdgcn_readlane(lfirst, 0) < pos0 && at == pos0) cut_of(0, cuts[0]);
      if (__builtin_amdgcn_readlane(lend, n_list - 1) > end && __builtin_amdgcn_readlane(lfirst, n_list - 1) >= pos0)
        cut_of(n_list - 1, cuts[1]);
      if (stop >= end) break;
      __syncthreads();  // the list and the places are free again
      at = stop;
      listed += n_list;
    }

    // ---- cut sequences: the last of their pieces to arrive adds their records, in the order of the keys
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
        // Two rows a wave, two elements a lane; every groups-th record a group of waves, then the
        // groups' sums.  Only records that are there are asked for: past the caches a compute unit
        // gets some 64 bytes a few ns (16 a lane always, 8 us behind the last arrival).
        const int part = by_pairs(wave), groups = by_pairs(kWaves);
        const int h = 2 * (wave - part * pairs) + (lane >> 5), d = 2 * (lane & 31);
        if (part < groups && h < rows) {
          float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll 1
          for (int n0 = part; n0 < u.pieces; n0 += kMerged * groups) {
            float2 ml[kMerged], y[kMerged];
#pragma unroll
            for (int v = 0; v < kMerged; ++v) {
              ml[v] = make_float2(-INFINITY, 0.f);
              y[v] = make_float2(0.f, 0.f);
              if (n0 + v * groups < u.pieces) {
                const float *const r = record(u.bin0 + n0 + v * groups, u.bin0, h);
                ml[v] = get2(r + HD);
                y[v] = get2(r + d);
              }
            }
            float mx = M;
#pragma unroll
            for (int v = 0; v < kMerged; ++v) mx = fmaxf(mx, ml[v].x);
            const float mu = mx == -INFINITY ? 0.f : mx, fo = __builtin_amdgcn_exp2f(M - mu);
            L *= fo;
            A0 *= fo;
            A1 *= fo;
#pragma unroll
            for (int v = 0; v < kMerged; ++v) {
              const float f = __builtin_amdgcn_exp2f(ml[v].x - mu);
              L = fmaf(ml[v].y, f, L);
              A0 = fmaf(y[v].x, f, A0);
              A1 = fmaf(y[v].y, f, A1);
            }
            M = mx;
          }
          float *const r = lds.hold + (part * rows + h) * kHoldRow;
          *(float2 *)(r + d) = make_float2(A0, A1);
          if (d == 0) *(float2 *)(r + HD) = make_float2(M, L);
        }
        __syncthreads();
        if (part == 0 && h < rows) {
          float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
#pragma unroll 1
          for (int v = 0; v < groups; ++v) {
            const float *const r = lds.hold + (v * rows + h) * kHoldRow;
            const float2 ml = *(const float2 *)(r + HD), y = *(const float2 *)(r + d);
            const float mn = fmaxf(M, ml.x), mu = mn == -INFINITY ? 0.f : mn;
            const float fo = __builtin_amdgcn_exp2f(M - mu), fn = __builtin_amdgcn_exp2f(ml.x - mu);
            L = fmaf(ml.y, fn, L * fo);
            A0 = fmaf(y.x, fn, A0 * fo);
            A1 = fmaf(y.y, fn, A1 * fo);
            M = mn;
          }
          write2(u.b, h, d, A0, A1, L);
        }
        __syncthreads();
      }
    }
  }
  // sequences without a key
  for (int b = bin; b < c.batch; b += p.bins)
    if (c.lens[b] <= 0 || c.cap == 0)
      for (int k = tid; k < rows * (HD / 2); k += 64 * kWaves) write2(b, k / (HD / 2), 2 * (k % (HD / 2)), 0.f, 0.f, 0.f);
}
template <int HW, int KW, int OCC>
__global__ __launch_bounds__(64 * HW * KW, OCC) void paged_q8_prefill_kernel(PrefillParams p, E4m3Pages src) {
  __shared__ __attribute__((aligned(16))) PrefillLds<HW, KW> lds;
  prefill_bf16_body<HW, KW>(p, lds, blockIdx.x, src);
}
// Queries in fp32: the fp32 cache's kernels.  A prefill's time is mostly the matrix cores' fp32 rate (64%
// busy, VALU 20%): 8192 rows of 32 and 4 heads 2800 us, 98 TFLOP/s, 64% of an 8192^3 fp32 library
// product's rate; 2048 rows 215 us.  A decode's is not, nor memory's: its four waves walk 16 keys a step,
// one step's rows in flight (matrix cores 25%, VALU 15% busy, 60% of the waves' time waiting): 64
// caches of 512..4096 keys 73 us, 1.07 TB/s, where bf16 queries take 22.5; of 4096 115; one of 640 8.6.
__global__ __launch_bounds__(256) void paged_q8_decode_f32_kernel(DecodeParams p, E4m3PagesF32 src) {
  __shared__ __attribute__((aligned(16))) DecodeLds<float> lds;
  decode_body<float>(p, lds, blockIdx.x, src);
}
template <int KW>
__global__ __launch_bounds__(64 * KW, 2) void paged_q8_prefill_f32_kernel(PrefillParams p, E4m3PagesF32 src) {
  __shared__ __attribute__((aligned(16))) PrefillLdsF32<KW> lds;
  prefill_f32_body<KW>(p, lds, blockIdx.x, src);
}
__global__ __launch_bounds__(256, 2) void paged_q8_prefill_pipe_kernel(PrefillParams p, E4m3Pages src) {
  __shared__ __attribute__((aligned(16))) PipeLds lds;
  prefill_pipe_body(p, lds, blockIdx.x, src);
}

// ---------------------------------------------------------------- the host
int check_q8(const std::string &op, const bn_paged_q8 *kv, Q8 *s) {
  if (!kv) return fail(BN_ERR_INVALID_ARG, op + ": cache is NULL");
  const bn_paged_kv codes{kv->k, kv->v, kv->page_table, kv->seq_lens, kv->page_stride, kv->head_stride,
                          kv->row_stride, kv->table_stride, BN_BF16, kv->batch, kv->n_pages, kv->max_pages,
                          kv->page_size, kv->n_kv_heads, kv->head_dim};
  const int st = check_pool(op, &codes, 1, kBlock, &s->c);
  if (st || kv->batch == 0) return st;
  const int64_t most = (int64_t)1 << 40, blocks = kv->page_size / kBlock;
  if (kv->n_pages > 0 && (!kv->k_scale || !kv->v_scale))
    return fail(BN_ERR_INVALID_ARG, op + ": NULL pointer to scales in the cache");
  if ((kv->n_pages > 1 && kv->scale_page_stride < blocks) || (kv->n_kv_heads > 1 && kv->scale_head_stride < blocks) ||
      kv->scale_page_stride < 0 || kv->scale_head_stride < 0 || kv->scale_page_stride > most ||
      kv->scale_head_stride > most)
    return fail(BN_ERR_INVALID_ARG, op + ": scale strides must be at least a page's blocks");
  s->ks = (uint8_t *)kv->k_scale;
  s->vs = (uint8_t *)kv->v_scale;
  s->scale_page = kv->scale_page_stride;
  s->scale_head = kv->scale_head_stride;
  return BN_OK;
}

int launch_decode(const AttnParams &a, int dtype, const E4m3Scales &scales, void *ws, hipStream_t s) {
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
  const dim3 grid((unsigned)(d.bins * d.columns));
  if (dtype == BN_F32) hipLaunchKernelGGL(paged_q8_decode_f32_kernel, grid, dim3(256), 0, s, p, E4m3PagesF32{scales});
  else if (decode_reads_once(a.c.row_stride, d.hblocks)) hipLaunchKernelGGL(paged_q8_decode_kernel<true>, grid, dim3(64 * kWaves), 0, s, p, E4m3Pages{scales});
  else hipLaunchKernelGGL(paged_q8_decode_kernel<false>, grid, dim3(64 * kWaves), 0, s, p, E4m3Pages{scales});
  BN_LAUNCH_CHECK();
  return BN_OK;
}

int launch_prefill(const AttnParams &a, int dtype, const E4m3Scales &scales, void *ws, hipStream_t s) {
  const PrefillPlan d = plan_q8(dtype, a.c.batch, a.n_rows, a.n_heads, a.c.n_kv_heads, a.c.cap);
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
  const E4m3Pages src{scales};
  const E4m3PagesF32 src32{scales};
  if (dtype == BN_F32) {
    if (d.kw == 4) hipLaunchKernelGGL(paged_q8_prefill_f32_kernel<4>, grid, dim3(256), 0, s, p, src32);
    else hipLaunchKernelGGL(paged_q8_prefill_f32_kernel<2>, grid, dim3(128), 0, s, p, src32);
  } else if (d.hw == 8) {
    hipLaunchKernelGGL(paged_q8_prefill_pipe_kernel, grid, dim3(256), 0, s, p, src);
  } else if (d.hw == 4) {
    if (d.kw == 2) hipLaunchKernelGGL((paged_q8_prefill_kernel<4, 2, 4>), grid, dim3(512), 0, s, p, src);
    else hipLaunchKernelGGL((paged_q8_prefill_kernel<4, 1, 4>), grid, dim3(256), 0, s, p, src);
  } else if (d.kw == 8) {
    hipLaunchKernelGGL((paged_q8_prefill_kernel<1, 8, 2>), grid, dim3(512), 0, s, p, src);
  } else {
    hipLaunchKernelGGL((paged_q8_prefill_kernel<1, 4, 3>), grid, dim3(256), 0, s, p, src);
  }
  BN_LAUNCH_CHECK();
  return BN_OK;
}

int attention_q8(const char *name, const bn_paged_q8 *kv, int dtype, const void *q, void *o, const int32_t *starts,
                 int n_rows, int n_heads, int64_t q_rs, int64_t o_rs, float scale, void *workspace,
                 size_t workspace_bytes, void *stream) {
  const std::string op = name;
  Q8 c;
  AttnParams p;
  int st = check_q8(op, kv, &c);
  if (st || (st = check_heads(op, n_heads, kv->n_kv_heads, n_rows)) ||
      (st = check_starts(op, starts, n_rows, kv->batch)))
    return st;
  if (dtype != BN_F32 && dtype != BN_BF16) return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(BN_ERR_INVALID_ARG, op + ": scale must be positive and finite");
  if (n_rows == 0 || kv->batch == 0) return BN_OK;
  if ((st = check_rows(op, "q", q, n_rows, n_heads, q_rs, dtype)) ||
      (st = check_rows(op, "o", o, n_rows, n_heads, o_rs, dtype)))
    return st;
  if (starts && prefill_threads(plan_q8(dtype, kv->batch, n_rows, n_heads, kv->n_kv_heads, c.c.cap)) >= (int64_t)1 << 32)
    return fail(BN_ERR_UNSUPPORTED, op + ": too many rows and sequences for one launch (2^32 threads)");
  const size_t need = bn_paged_q8_workspace_size(kv, n_heads, n_rows);
  if (workspace && workspace_bytes < need)
    return fail(BN_ERR_INVALID_ARG, op + ": workspace of " + std::to_string(workspace_bytes) +
                                        " bytes, need " + std::to_string(need));
  if (workspace && !aligned16(workspace))
    return fail(BN_ERR_UNSUPPORTED, op + ": workspace must be 16-byte aligned");
  DeviceScope scope;
  if ((st = scope.enter(op, kv->seq_lens))) return st;
  p.c = c.c;
  p.q = q; p.o = o; p.starts = starts;
  p.q_rs = q_rs; p.o_rs = o_rs;
  p.n_rows = n_rows; p.n_heads = n_heads; p.group = n_heads / kv->n_kv_heads;
  p.inv_group = 1.0f / (float)p.group;
  p.cl = scale * kLog2e;
  p.prefix_pages = nullptr;
  p.prefix_len = 0;
  const E4m3Scales scales{c.ks, c.vs, c.scale_page, c.scale_head};
  Workspace ws;
  if ((st = ws.take(workspace, need, stream))) return st;
  hipStream_t s = as_stream(stream);
  return ws.release(starts ? launch_prefill(p, dtype, scales, ws.p, s) : launch_decode(p, dtype, scales, ws.p, s));
}

}  // namespace
}  // namespace bn

using namespace bn;

extern "C" {

int bn_paged_q8_append(const bn_paged_q8 *cache, int dtype, const void *k, const void *v, const void *q,
                       void *q_out, const int32_t *row_starts, int n_rows, int n_heads, int64_t k_row_stride,
                       int64_t v_row_stride, int64_t q_row_stride, int64_t q_out_row_stride, float theta,
                       const void *q_weight, const void *k_weight, float eps, void *stream) {
  const std::string op = "Paged Q8 append";
  Q8AppendParams p;
  int st = check_q8(op, cache, &p.s);
  if (st || (st = check_starts(op, row_starts, n_rows, cache->batch))) return st;
  if (dtype != BN_F32 && dtype != BN_BF16) return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  if (!q != !q_out) return fail(BN_ERR_INVALID_ARG, op + ": q and q_out must be given together");
  if (q_weight && !q) return fail(BN_ERR_INVALID_ARG, op + ": q_weight without q");
  if (q && (st = check_heads(op, n_heads, cache->n_kv_heads, n_rows))) return st;
  if (n_rows > (1 << 23)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^23 rows");
  if (!(theta >= 0.f) || !std::isfinite(theta))
    return fail(BN_ERR_INVALID_ARG, op + ": theta must be positive and finite, or 0 for no rotation");
  if ((q_weight || k_weight) && (!(eps >= 0.f) || !std::isfinite(eps)))
    return fail(BN_ERR_INVALID_ARG, op + ": eps must be finite and not negative");
  if (!aligned16(q_weight) || !aligned16(k_weight))
    return fail(BN_ERR_UNSUPPORTED, op + ": weights must be 16-byte aligned");
  if (n_rows == 0 || cache->batch == 0) return BN_OK;
  if ((st = check_rows(op, "k", k, n_rows, cache->n_kv_heads, k_row_stride, dtype)) ||
      (st = check_rows(op, "v", v, n_rows, cache->n_kv_heads, v_row_stride, dtype)) ||
      (q && ((st = check_rows(op, "q", q, n_rows, n_heads, q_row_stride, dtype)) ||
             (st = check_rows(op, "q_out", q_out, n_rows, n_heads, q_out_row_stride, dtype)))))
    return st;
  if (q == q_out && q && q_row_stride != q_out_row_stride)
    return fail(BN_ERR_INVALID_ARG, op + ": q_out in q's place must have its row stride");
  DeviceScope scope;
  if ((st = scope.enter(op, cache->seq_lens))) return st;
  p.k = k; p.v = v; p.q = q; p.qo = q_out; p.wq = q_weight; p.wk = k_weight; p.starts = row_starts;
  p.k_rs = k_row_stride; p.v_rs = v_row_stride; p.q_rs = q_row_stride; p.qo_rs = q_out_row_stride;
  p.n_rows = n_rows;
  p.n_heads = q ? n_heads : 0;
  p.turn = theta > 0.f;
  p.eps = eps;
  fill_turns(p.f, HD, theta);
  hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)count_units(row_starts, n_rows, cache->batch)), block(kAppendThreads);
  if (dtype == BN_BF16) hipLaunchKernelGGL(paged_q8_append_kernel<bf16_t>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(paged_q8_append_kernel<float>, grid, block, 0, s, p);
  BN_LAUNCH_CHECK();
  return BN_OK;
}

int bn_paged_q8_read(const bn_paged_q8 *cache, int dtype, void *k, void *v, const int32_t *row_starts, int n_rows,
                     int64_t k_row_stride, int64_t v_row_stride, void *stream) {
  const std::string op = "Paged Q8 read";
  Q8ReadParams p;
  int st = check_q8(op, cache, &p.s);
  if (st || (st = check_starts(op, row_starts, n_rows, cache->batch))) return st;
  if (dtype != BN_F32 && dtype != BN_BF16) return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  if (n_rows > (1 << 23)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^23 rows");
  if (n_rows == 0 || cache->batch == 0) return BN_OK;
  if (!k && !v) return fail(BN_ERR_INVALID_ARG, op + ": k and v are NULL");
  if ((k && (st = check_rows(op, "k", k, n_rows, cache->n_kv_heads, k_row_stride, dtype))) ||
      (v && (st = check_rows(op, "v", v, n_rows, cache->n_kv_heads, v_row_stride, dtype))))
    return st;
  DeviceScope scope;
  if ((st = scope.enter(op, cache->seq_lens))) return st;
  p.k = k; p.v = v; p.starts = row_starts;
  p.k_rs = k_row_stride; p.v_rs = v_row_stride;
  p.n_rows = n_rows;
  hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)count_units(row_starts, n_rows, cache->batch)), block(256);
  const int64_t bytes = (int64_t)n_rows * cache->n_kv_heads * HD * (dtype == BN_BF16 ? 2 : 4) * (!!k + !!v);
  if (bytes > (3 << 25)) {
    if (dtype == BN_BF16) hipLaunchKernelGGL((paged_q8_read_kernel<bf16_t, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_q8_read_kernel<float, true>), grid, block, 0, s, p);
  } else {
    if (dtype == BN_BF16) hipLaunchKernelGGL((paged_q8_read_kernel<bf16_t, false>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_q8_read_kernel<float, false>), grid, block, 0, s, p);
  }
  BN_LAUNCH_CHECK();
  return BN_OK;
}

size_t bn_paged_q8_workspace_size(const bn_paged_q8 *cache, int n_heads, int n_rows) {
  Q8 s;
  if (n_rows <= 0 || !cache || check_q8("", cache, &s) || cache->batch == 0 ||
      check_heads("", n_heads, cache->n_kv_heads, n_rows))
    return 0;
  const DecodePlan d = plan_decode(cache->batch, n_heads, cache->n_kv_heads);
  size_t need = d.records + d.words;  // (for either type)
  for (int dtype : {BN_F32, BN_BF16}) {
    const PrefillPlan f = plan_q8(dtype, cache->batch, n_rows, n_heads, cache->n_kv_heads, s.c.cap, true);
    need = std::max(need, f.records + f.words);
  }
  return need;
}

int bn_paged_q8_decode(const bn_paged_q8 *cache, int dtype, const void *q, void *o, int n_heads,
                       int64_t q_row_stride, int64_t o_row_stride, float scale, void *workspace,
                       size_t workspace_bytes, void *stream) {
  return attention_q8("Paged Q8 decode", cache, dtype, q, o, nullptr, cache ? cache->batch : 0, n_heads, q_row_stride,
                      o_row_stride, scale, workspace, workspace_bytes, stream);
}

int bn_paged_q8_prefill(const bn_paged_q8 *cache, int dtype, const void *q, void *o, const int32_t *row_starts,
                        int n_rows, int n_heads, int64_t q_row_stride, int64_t o_row_stride, float scale,
                        void *workspace, size_t workspace_bytes, void *stream) {
  return attention_q8("Paged Q8 prefill", cache, dtype, q, o, row_starts, n_rows, n_heads, q_row_stride, o_row_stride,
                      scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
