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
    threads = prefill_threads(plan_prefill(dtype, batch, n_rows, n_heads, n_kv_heads, cap));
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
