// bn_paged_host.hpp -- what the paged caches' calls share on the host: checks of sizes, strides and
// pointers, the device of a call, its workspace and its launch's tag.
#pragma once

#include <algorithm>
#include <cmath>
#include <string>

#include "bn_common.hpp"
#include "bn_paged_device.hpp"

namespace bn {

// A launch's 48-bit tag: no plausible memory contents look like this launch's arrivals.
unsigned long long next_tag();

namespace {

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

// Sizes, strides and pointers of a cache whose elements have `bytes` bytes and whose
// pages hold at least `least` keys; on success *c is the kernels' form.
inline int check_pool(const std::string &op, const bn_paged_kv *kv, int bytes, int least, Paged *c) {
  if (kv->batch < 0 || kv->n_pages < 0 || kv->max_pages < 0)
    return fail(BN_ERR_SHAPE, op + ": negative batch or number of pages");
  if (kv->n_kv_heads <= 0) return fail(BN_ERR_SHAPE, op + ": num_kv_heads must be positive");
  if (kv->n_kv_heads > 65535) return fail(BN_ERR_UNSUPPORTED, op + ": more than 65535 KV heads");
  if (kv->head_dim != HD) return fail(BN_ERR_UNSUPPORTED, op + ": head_dim must be 64");
  if (kv->page_size < least || kv->page_size > (1 << 20) || (kv->page_size & (kv->page_size - 1)))
    return fail(BN_ERR_UNSUPPORTED, op + ": page_size must be a power of two, at least " + std::to_string(least) +
                                        " and at most 2^20");
  const int64_t keys = (int64_t)kv->max_pages * kv->page_size;
  if (keys > (1 << 30))
    return fail(BN_ERR_UNSUPPORTED, op + ": max_pages * page_size must be at most 2^30 keys");
  if (kv->batch == 0) return BN_OK;
  if (kv->batch > (1 << 20)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^20 sequences");
  if (kv->batch * keys > ((int64_t)1 << 34))  // tiles of 16 keys are counted in 32 bits
    return fail(BN_ERR_UNSUPPORTED, op + ": batch * max_pages * page_size must be at most 2^34 keys");
  // (a load's rows are reached through 32-bit byte offsets, pages by 32 x 32-bit products)
  if (kv->row_stride > (1 << 24) || kv->page_stride >= (1 << 30))
    return fail(BN_ERR_UNSUPPORTED,
                op + ": cache row stride must be at most 2^24 elements, page stride below 2^30");
  const int64_t vec = 16 / bytes, most = (int64_t)1 << 40;
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
  c->batch = kv->batch; c->n_pages = kv->n_pages;
  c->shift = __builtin_ctz((unsigned)kv->page_size);
  c->n_kv_heads = kv->n_kv_heads;
  c->cap = kv->n_pages > 0 ? (int)keys : 0;  // without a page there is no key
  return BN_OK;
}
inline int check_cache(const std::string &op, const bn_paged_kv *kv, Paged *c) {
  if (!kv) return fail(BN_ERR_INVALID_ARG, op + ": cache is NULL");
  if (kv->dtype != BN_F32 && kv->dtype != BN_BF16)
    return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  return check_pool(op, kv, kv->dtype == BN_BF16 ? 2 : 4, 8, c);
}

// A [n_rows, heads, head_dim] tensor with a row stride.
inline int check_rows(const std::string &op, const char *name, const void *t, int n_rows, int64_t heads,
                      int64_t row_stride, int dtype, int head_dim = HD) {
  if (n_rows == 0) return BN_OK;
  if (!t) return fail(BN_ERR_INVALID_ARG, op + ": " + name + " is NULL");
  if (row_stride < heads * head_dim)
    return fail(BN_ERR_SHAPE, op + ": " + name + " row stride smaller than heads*head_dim");
  if (!aligned16(t) || row_stride % (dtype == BN_BF16 ? 8 : 4) || row_stride > ((int64_t)1 << 40))
    return fail(BN_ERR_UNSUPPORTED, op + ": " + name +
                                        " must be 16-byte aligned, its row stride a multiple of 16 bytes");
  return BN_OK;
}

inline int check_starts(const std::string &op, const int32_t *row_starts, int n_rows, int batch) {
  if (n_rows < 0) return fail(BN_ERR_SHAPE, op + ": negative number of rows");
  if (!row_starts && n_rows != batch)
    return fail(BN_ERR_SHAPE, op + ": without row_starts there is one row per sequence");
  if ((uintptr_t)row_starts & 3u) return fail(BN_ERR_UNSUPPORTED, op + ": row_starts must be 4-byte aligned");
  return BN_OK;
}

inline int check_heads(const std::string &op, int n_heads, int n_kv_heads, int n_rows) {
  if (n_heads <= 0 || n_heads % n_kv_heads != 0)
    return fail(BN_ERR_SHAPE, op + ": num_heads must be a positive multiple of num_kv_heads");
  if (n_heads > 65535) return fail(BN_ERR_UNSUPPORTED, op + ": more than 65535 heads");
  if ((int64_t)n_rows * n_heads > (1 << 30))
    return fail(BN_ERR_UNSUPPORTED, op + ": n_rows * num_heads must be at most 2^30");
  return BN_OK;
}

// The library's device, made the calling thread's current one for the call,
// whatever was current before (another library may have changed it).
class DeviceScope {
  int before_ = -1;

 public:
  int enter(const std::string &op, const void *memory, const char *what = "the cache") {
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
      return fail(BN_ERR_INVALID_ARG, op + ": " + what + " is on device " + std::to_string(a.device) +
                                          ", the library on device " + std::to_string(lib));
    return BN_OK;
  }
  ~DeviceScope() {
    if (before_ >= 0) (void)hipSetDevice(before_);
  }
};
// A call's workspace: the caller's, or one from the pool until the end of the call's work.
class Workspace {
  void *own_ = nullptr, *stream_ = nullptr;

 public:
  void *p = nullptr;
  int take(void *given, size_t need, void *stream) {
    p = given;
    if (p || need == 0) return BN_OK;
    const int st = bn_alloc(&own_, need, stream);
    stream_ = stream;
    p = own_;
    return st;
  }
  int release(int st) {
    if (own_) {
      const int st2 = bn_free(own_, stream_);
      own_ = nullptr;
      if (st == BN_OK) st = st2;
    }
    return st;
  }
};

// The decode kernel's launch: a workgroup per share and column, one per compute
// unit in all (two: 64 caches of 4096 keys 45.8 -> 49.0 us, of 512..4096 34.6 ->
// 35.7; 256 of 300 21.4 -> 18.8).
constexpr int kDecGroups = 256;
struct DecodePlan {
  int hblocks, columns, bins;
  size_t records, words;  // bytes
};
inline DecodePlan plan_decode(int batch, int n_heads, int n_kv_heads) {
  DecodePlan d;
  d.hblocks = (n_heads / n_kv_heads + kMaxRows - 1) / kMaxRows;
  d.columns = d.hblocks * n_kv_heads;
  d.bins = std::max(1, kDecGroups / d.columns);
  d.records = d.bins == 1 ? 0 : (size_t)d.bins * 2 * d.columns * kMaxRows * kRec * sizeof(float);
  d.words = d.bins == 1 ? 0 : (size_t)batch * d.columns * 16;
  return d;
}

// The threads of a prefill's launch, which the runtime counts in 32 bits.
inline int64_t prefill_threads(const PrefillPlan &d) {
  return d.groups * (d.hw == 8 ? 256 : 64 * d.hw * d.kw);
}

}  // namespace
}  // namespace bn
