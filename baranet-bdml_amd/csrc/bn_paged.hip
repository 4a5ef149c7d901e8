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
// address, and lengths are clamped to what the table can hold, so that no
// contents of those arrays lead outside the pools.
#include <algorithm>
#include <cmath>

#include "bn_common.hpp"

namespace bn {
namespace {

constexpr int HD = 64;
constexpr float kLog2e = 1.4426950408889634f;

// The cache as the kernels see it.  Offsets in elements.
struct Paged {
  const void *k, *v;
  const int32_t *table, *lens;
  int64_t page_stride, head_stride, row_stride, table_stride;
  int batch, n_pages, max_pages, shift, n_kv_heads;  // page_size = 1 << shift
  int cap;                                           // keys a table row holds
};

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

// ------------------------------------------------------------------ append
struct AppendParams {
  Paged c;
  const void *k, *v, *q;
  void *qo;
  const int32_t *starts;
  int64_t k_rs, v_rs, q_rs, qo_rs;
  int n_rows, n_heads;  // n_heads: 0 without q
  int turn;             // rotate
  double f[HD / 2];     // turns per position of each pair: theta^(-2p/64) / (2 pi)
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

// RB rows per workgroup of 256 threads.  First a (row, pair) per thread: the
// row's place and the pair's cosine and sine, into LDS.  The angle is formed
// in turns and in 64 bits and reduced to an eighth of a turn before it is
// rounded to 32: at position 2^20 a 32-bit angle would be off by 0.06 rad.
// Then the rows' 16-byte pieces, Q heads, K heads, V heads, consecutive
// threads on consecutive pieces, 256 / RB threads a row.
template <typename T, int RB>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  constexpr int PIECES = HD * sizeof(T) / 16;  // per head
  constexpr int VEC = 16 / sizeof(T);
  constexpr int TPR = 256 / RB;
  __shared__ float2 cs[RB][HD / 2];
  __shared__ int64_t place[RB];  // element offset of the row's slot in KV head 0 (-1: none)
  __shared__ int owner[RB];      // the row's sequence (-1: padding)
  const int tid = threadIdx.x;
  const int row0 = blockIdx.x * RB;
  if (tid < RB * (HD / 2)) {
    const int r = tid / (HD / 2), pair = tid % (HD / 2);
    const int row = row0 + r;
    const int b = row < p.n_rows ? sequence_of(p.starts, p.c.batch, row) : -1;
    const int pos = b < 0 ? 0 : position_of(p.c, p.starts, b, row);
    if (pair == 0) {
      int64_t at = -1;
      if (b >= 0 && pos >= 0 && pos < p.c.cap) {
        const int page = p.c.table[b * p.c.table_stride + (pos >> p.c.shift)];
        if ((unsigned)page < (unsigned)p.c.n_pages)
          at = page * p.c.page_stride + (pos & ((1 << p.c.shift) - 1)) * p.c.row_stride;
      }
      place[r] = at;
      owner[r] = b;
    }
    const double turns = (double)pos * p.f[pair];
    const double quarter = rint(4.0 * turns);
    float s, c;
    sincospif(2.f * (float)(turns - 0.25 * quarter), &s, &c);
    const int quadrant = (int)((int64_t)quarter & 3);
    const float cq = quadrant & 1 ? -s : c, sq = quadrant & 1 ? c : s;
    cs[r][pair] = quadrant & 2 ? make_float2(-cq, -sq) : make_float2(cq, sq);
  }
  __syncthreads();
  const int r = tid / TPR, row = row0 + r;
  if (row >= p.n_rows || owner[r] < 0) return;
  const int64_t at = place[r];
  const int hkv = p.c.n_kv_heads, kv0 = p.n_heads, v0 = kv0 + hkv, pieces = (v0 + hkv) * PIECES;
  T *const Kd = (T *)p.c.k + at, *const Vd = (T *)p.c.v + at;
  const T *const Q = (const T *)p.q + row * p.q_rs, *const K = (const T *)p.k + row * p.k_rs,
          *const V = (const T *)p.v + row * p.v_rs;
  T *const Qo = (T *)p.qo + row * p.qo_rs;
  for (int i = tid % TPR; i < pieces; i += TPR) {
    const int h = i / PIECES, e = (i % PIECES) * VEC;
    if (h < kv0) {
      u32x4 x = *(const u32x4 *)(Q + h * HD + e);
      if (p.turn) x = rotate<T>(x, &cs[r][e / 2]);
      *(u32x4 *)(Qo + h * HD + e) = x;
    } else if (at >= 0 && h < v0) {
      u32x4 x = *(const u32x4 *)(K + (h - kv0) * HD + e);
      if (p.turn) x = rotate<T>(x, &cs[r][e / 2]);
      *(u32x4 *)(Kd + (h - kv0) * p.c.head_stride + e) = x;
    } else if (at >= 0) {
      *(u32x4 *)(Vd + (h - v0) * p.c.head_stride + e) = *(const u32x4 *)(V + (h - v0) * HD + e);
    }
  }
}

// --------------------------------------------------------------- attention
struct AttnParams {
  Paged c;
  const void *q;
  void *o;
  const int32_t *starts;  // null: one row per sequence
  int64_t q_rs, o_rs;
  int n_rows, n_heads, group;
  float cl;  // scale * log2(e)
  const int32_t *prefix_pages;
  int prefix_len;
};

// One wave per (row, query head), lane = element of the head: every key's
// dot product is a wave sum.
template <typename T>
__global__ __launch_bounds__(64) void paged_rows_kernel(AttnParams p) {
  const int lane = threadIdx.x, row = blockIdx.x, h = blockIdx.y, g = h / p.group;
  const int b = sequence_of(p.starts, p.c.batch, row);
  if (b < 0) return;
  const int end = min(position_of(p.c, p.starts, b, row) + 1, p.c.cap);
  const float q = Elem<T>::load((const T *)p.q + row * p.q_rs + h * HD + lane) * p.cl;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int j = 0; j < end; ++j) {
    const int page = j < p.prefix_len ? p.prefix_pages[j >> p.c.shift]
                                      : p.c.table[b * p.c.table_stride + (j >> p.c.shift)];
    if ((unsigned)page >= (unsigned)p.c.n_pages) continue;
    const int64_t at = page * p.c.page_stride + g * p.c.head_stride +
                       (j & ((1 << p.c.shift) - 1)) * p.c.row_stride + lane;
    const float s = wave_sum(q * Elem<T>::load((const T *)p.c.k + at));
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
    const float a = __builtin_amdgcn_exp2f(m - mu), e = __builtin_amdgcn_exp2f(s - mu);
    l = l * a + e;
    acc = fmaf(e, Elem<T>::load((const T *)p.c.v + at), acc * a);
    m = mn;
  }
  Elem<T>::store((T *)p.o + row * p.o_rs + h * HD + lane, l > 0.f ? acc / l : 0.f);
}

// ---------------------------------------------------------------- the host
bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// Sizes, strides and pointers of a cache; on success *c is the kernels' form.
int check_cache(const std::string &op, const bn_paged_kv *kv, Paged *c) {
  if (!kv) return fail(BN_ERR_INVALID_ARG, op + ": cache is NULL");
  if (kv->dtype != BN_F32 && kv->dtype != BN_BF16)
    return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  if (kv->batch < 0 || kv->n_pages < 0 || kv->max_pages < 0)
    return fail(BN_ERR_SHAPE, op + ": negative batch or number of pages");
  if (kv->n_kv_heads <= 0) return fail(BN_ERR_SHAPE, op + ": num_kv_heads must be positive");
  if (kv->head_dim != HD) return fail(BN_ERR_UNSUPPORTED, op + ": head_dim must be 64");
  if (kv->page_size <= 0 || (kv->page_size & (kv->page_size - 1)))
    return fail(BN_ERR_UNSUPPORTED, op + ": page_size must be a power of two");
  if ((int64_t)kv->max_pages * kv->page_size > (1 << 30))
    return fail(BN_ERR_UNSUPPORTED, op + ": max_pages * page_size must be at most 2^30 keys");
  if (kv->batch == 0) return BN_OK;
  if (kv->batch > (1 << 20)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^20 sequences");
  const int64_t vec = kv->dtype == BN_BF16 ? 8 : 4, most = (int64_t)1 << 40;
  for (int64_t s : {kv->page_stride, kv->head_stride, kv->row_stride})
    if (s < HD || s % vec || s > most)
      return fail(BN_ERR_INVALID_ARG, op + ": cache strides must be multiples of " + std::to_string(vec) +
                                          " elements (16 bytes), at least head_dim");
  if (kv->batch > 1 && (kv->table_stride < kv->max_pages || kv->table_stride > most))
    return fail(BN_ERR_SHAPE, op + ": page table rows overlap");
  if (!kv->seq_lens || (kv->max_pages > 0 && !kv->page_table) || (kv->n_pages > 0 && (!kv->k || !kv->v)))
    return fail(BN_ERR_INVALID_ARG, op + ": NULL pointer in the cache");
  if (!aligned16(kv->k) || !aligned16(kv->v))
    return fail(BN_ERR_UNSUPPORTED, op + ": pools must be 16-byte aligned");
  if (((uintptr_t)kv->page_table | (uintptr_t)kv->seq_lens) & 3u)
    return fail(BN_ERR_UNSUPPORTED, op + ": page table and lengths must be 4-byte aligned");
  c->k = kv->k; c->v = kv->v; c->table = kv->page_table; c->lens = kv->seq_lens;
  c->page_stride = kv->page_stride; c->head_stride = kv->head_stride; c->row_stride = kv->row_stride;
  c->table_stride = kv->table_stride;
  c->batch = kv->batch; c->n_pages = kv->n_pages; c->max_pages = kv->max_pages;
  c->shift = __builtin_ctz((unsigned)kv->page_size);
  c->n_kv_heads = kv->n_kv_heads;
  c->cap = kv->max_pages * kv->page_size;
  return BN_OK;
}

// A [n_rows, heads, 64] tensor with a row stride.
int check_rows(const std::string &op, const char *name, const void *t, int n_rows, int64_t heads,
               int64_t row_stride, int dtype) {
  if (n_rows == 0) return BN_OK;
  if (!t) return fail(BN_ERR_INVALID_ARG, op + ": " + name + " is NULL");
  if (row_stride < heads * HD)
    return fail(BN_ERR_SHAPE, op + ": " + name + " row stride smaller than heads*head_dim");
  if (!aligned16(t) || row_stride % (dtype == BN_BF16 ? 8 : 4) || row_stride > ((int64_t)1 << 40))
    return fail(BN_ERR_UNSUPPORTED, op + ": " + name +
                                        " must be 16-byte aligned, its row stride a multiple of 16 bytes");
  return BN_OK;
}

int check_starts(const std::string &op, const int32_t *row_starts, int n_rows, int batch) {
  if (n_rows < 0) return fail(BN_ERR_SHAPE, op + ": negative number of rows");
  if (!row_starts && n_rows != batch)
    return fail(BN_ERR_SHAPE, op + ": without row_starts there is one row per sequence");
  if ((uintptr_t)row_starts & 3u) return fail(BN_ERR_UNSUPPORTED, op + ": row_starts must be 4-byte aligned");
  return BN_OK;
}

int check_heads(const std::string &op, int n_heads, int n_kv_heads) {
  if (n_heads <= 0 || n_heads % n_kv_heads != 0)
    return fail(BN_ERR_SHAPE, op + ": num_heads must be a positive multiple of num_kv_heads");
  if (n_heads > 65535) return fail(BN_ERR_UNSUPPORTED, op + ": more than 65535 heads");
  return BN_OK;
}

// The library's device, made the calling thread's current one for the call,
// whatever was current before (another library may have changed it).
class DeviceScope {
  int before_ = -1;

 public:
  int enter(const std::string &op, const void *memory) {
    int st = ensure_device();
    if (st) return st;
    const int lib = library_device();
    int cur = lib;
    BN_HIP_TRY(hipGetDevice(&cur));
    if (cur != lib) {
      BN_HIP_TRY(hipSetDevice(lib));
      before_ = cur;
    }
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, memory) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
      (void)hipGetLastError();
      return fail(BN_ERR_NOT_DEVICE, op + ": only GPU implementation available");
    }
    if (a.type == hipMemoryTypeDevice && a.device != lib)
      return fail(BN_ERR_INVALID_ARG, op + ": the cache is on device " + std::to_string(a.device) +
                                          ", the library on device " + std::to_string(lib));
    return BN_OK;
  }
  ~DeviceScope() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
};

int attention(const char *name, const bn_paged_kv *kv, const void *q, void *o, const int32_t *starts,
              int n_rows, int n_heads, int64_t q_rs, int64_t o_rs, float scale,
              const int32_t *prefix_pages, int prefix_len, void *workspace, size_t workspace_bytes,
              void *stream) {
  const std::string op = name;
  AttnParams p;
  int st = check_cache(op, kv, &p.c);
  if (st || (st = check_heads(op, n_heads, kv->n_kv_heads)) ||
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
  p.cl = scale * kLog2e;
  p.prefix_pages = prefix_pages; p.prefix_len = prefix_len;
  const dim3 grid(n_rows, n_heads);
  if (kv->dtype == BN_BF16)
    hipLaunchKernelGGL(paged_rows_kernel<bf16_t>, grid, dim3(64), 0, as_stream(stream), p);
  else
    hipLaunchKernelGGL(paged_rows_kernel<float>, grid, dim3(64), 0, as_stream(stream), p);
  BN_LAUNCH_CHECK();
  return BN_OK;
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
  if (q && (st = check_heads(op, n_heads, cache->n_kv_heads))) return st;
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
  p.n_rows = n_rows; p.n_heads = q ? n_heads : 0;
  p.turn = theta > 0.f;
  for (int i = 0; i < HD / 2; ++i)
    p.f[i] = theta > 0.f ? std::pow((double)theta, -2.0 * i / HD) / (2.0 * M_PI) : 0.0;
  hipStream_t s = as_stream(stream);
  const bool few = n_rows < 1024;
  const dim3 grid(few ? n_rows : (n_rows + 7) / 8), block(256);
  if (cache->dtype == BN_BF16) {
    if (few) hipLaunchKernelGGL((paged_append_kernel<bf16_t, 1>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_append_kernel<bf16_t, 8>), grid, block, 0, s, p);
  } else {
    if (few) hipLaunchKernelGGL((paged_append_kernel<float, 1>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_append_kernel<float, 8>), grid, block, 0, s, p);
  }
  BN_LAUNCH_CHECK();
  return BN_OK;
}

size_t bn_paged_workspace_size(const bn_paged_kv *cache, int n_heads, int n_rows, int prefix_len) {
  (void)cache; (void)n_heads; (void)n_rows; (void)prefix_len;
  return 0;
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
