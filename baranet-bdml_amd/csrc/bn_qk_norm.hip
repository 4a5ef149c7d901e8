// bn_qk_norm.hip -- RMSNorm of every head of queries and keys with the rotation
// by the row's position in the same pass, and its backward pass.
//
// The reference norms whole rows (op_rmsnorm.cuh:8-53) and turns heads
// (op_rope.cuh:55-99); here the norm is a head's own.  With r = 1 / sqrt(mean(x^2)
// + eps) and R the rotation by the row's position:
//   y = R (w * x r)
//   g = R^T dy,  dx = r (w g) - x r^3 / D * sum_d(w g x),  dw = sum_{rows, heads} g x r.
// Everything between load and store is fp32; a head's sums are formed by its 2 to
// 32 lanes, the weights' gradients per lane, then per workgroup, then over the
// workgroups in the order of their numbers.
#include <algorithm>

#include "bn_head_rows.hpp"
#include "bn_paged_host.hpp"
#include "bn_qk_plan.hpp"

namespace bn {
namespace {

constexpr int kMaxHeadDim = 256;
struct QkParams {
  const void *q, *k, *wq, *wk, *gq, *gk;  // gq, gk: gradients of the outputs (backward)
  void *qo, *ko;                          // outputs (backward: gradients of q and k)
  const int32_t *positions;
  int64_t q_rs, k_rs, gq_rs, gk_rs, qo_rs, ko_rs;
  int n_rows, n_heads, n_kv_heads, rows, turn;  // rows: of a workgroup at once
  int64_t offset;
  float eps;
  float *parts;                           // backward: [workgroups][2][D] sums
  float *dwq, *dwk;                       // the weights' gradients
  unsigned long long *arrive, tag;
};
template <int D>
struct Turns {  // per position, of each pair (a launch takes 0.35 us less with D = 64's 256 bytes than with D = 256's)
  double f[D / 2];
};

// The pairs' cosines and sines of the rows that a workgroup has at once.
template <int D>
__device__ __forceinline__ void angles(const QkParams &p, const Turns<D> &t, float2 (*cs)[D / 2], int row0, int rows) {
  if (!p.turn) return;
  for (int i = threadIdx.x; i < rows * (D / 2); i += blockDim.x) {
    const int r = i / (D / 2), row = row0 + r;
    const int64_t pos = (p.positions ? (int64_t)p.positions[row] : (int64_t)row) + p.offset;
    cs[r][i % (D / 2)] = cos_sin((double)pos * t.f[i % (D / 2)]);
  }
}

// `rows` rows a workgroup: their angles once, then their heads' pieces of eight
// elements, four of a thread on their way at once, the first of them while the
// angles are formed.  Bound by memory, VALU 87% busy: 8192 bf16 rows of 32 and 4 heads
// 15.6 us, 4.8 TB/s, a large copy's rate (a copy of as many bytes, all of which the memory-side cache
// holds, 12.3); as fp32 37, 4.1 TB/s; 16 rows 3.1, a launch.  (Stores past the caches' keeping: 16384
// rows 35 -> 25 us, but the attention that reads them takes as much longer.)
constexpr int kPieces = 4;
template <typename T, int D>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkParams p, Turns<D> t) {
  constexpr int LANES = D / 8;
  __shared__ float2 cs[kMostRows][D / 2];
  const int tid = threadIdx.x, row0 = blockIdx.x * p.rows, rows = min(p.rows, p.n_rows - row0);
  const int per = (p.n_heads + p.n_kv_heads) * LANES, total = rows * per;
  Walk at(tid, 256, per);
  struct Piece8 {
    int row, head, e;  // row of the workgroup, head (keys' behind the queries'), element
    Raw8<T> raw;
  } x[kPieces];
  auto load = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      if (first + 256 * n >= total) break;
      x[n].row = at.row;
      x[n].head = at.rest / LANES;
      x[n].e = at.rest % LANES * 8;
      at.step();
      const int64_t row = row0 + x[n].row;
      x[n].raw.load(x[n].head < p.n_heads ? (const T *)p.q + row * p.q_rs + x[n].head * D + x[n].e
                                          : (const T *)p.k + row * p.k_rs + (x[n].head - p.n_heads) * D + x[n].e);
    }
  };
  load(tid);
  angles<D>(p, t, cs, row0, rows);
  __syncthreads();
  for (int first = tid; first < total; first += 256 * kPieces) {
    if (first != tid) load(first);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      if (first + 256 * n >= total) break;
      const bool is_q = x[n].head < p.n_heads;
      Eight v = x[n].raw.floats();
      const float r = head_rms<LANES>(v, p.eps);
      Raw8<T> wr;
      wr.load((const T *)(is_q ? p.wq : p.wk) + x[n].e);
      const Eight w = wr.floats();
#pragma unroll
      for (int j = 0; j < 8; ++j) v.x[j] *= r * w.x[j];
      if (p.turn) turn8(v, &cs[x[n].row][x[n].e / 2]);
      const int64_t row = row0 + x[n].row;
      store8(is_q ? (T *)p.qo + row * p.qo_rs + x[n].head * D + x[n].e
                  : (T *)p.ko + row * p.ko_rs + (x[n].head - p.n_heads) * D + x[n].e,
             v);
    }
  }
}

constexpr int kPairs = 2;  // pieces of rows and gradients of a thread on their way at once
// A workgroup takes every gridDim.x-th group of `rows` rows.  A thread's pieces lie at
// one place of their heads, so it adds up eight elements of each weight's
// gradient in registers; a workgroup's sums go to the workspace, and the last workgroup to
// arrive (JOINS), or another launch, adds them.  Bound by memory: 16384 bf16 rows of 32 and 4 heads
// 46 us, 4.9 TB/s (59 with one piece at once), and 4 for the sums' launch; 1504 fp32 rows 14.7
// with their sums.
template <typename T, int D, int THREADS, bool JOINS>
__global__ __launch_bounds__(THREADS) void qk_norm_rope_backward_kernel(QkParams p, Turns<D> t) {
  constexpr int LANES = D / 8;
  __shared__ float2 cs[JOINS ? kJoinedRows : kMostRows][D / 2];
  constexpr int STEP = THREADS / D, N = 16;  // (of the sums behind the rows)
  __shared__ union {
    float of_wave[THREADS / 64][2][D], of_groups[STEP][2 * D];
  } sums;
  __shared__ bool last;
  const int tid = threadIdx.x, lane = tid & 63, e = tid % LANES * 8;
  Eight dw[2] = {};
  for (int64_t at = (int64_t)blockIdx.x * p.rows; at < p.n_rows; at += (int64_t)gridDim.x * p.rows) {
    const int row0 = (int)at, rows = min(p.rows, p.n_rows - row0);
    __syncthreads();  // the angles before are no longer read
    angles<D>(p, t, cs, row0, rows);
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int heads = side ? p.n_kv_heads : p.n_heads, per = heads * LANES, total = rows * per;
      const T *const x = (const T *)(side ? p.k : p.q), *const dy = (const T *)(side ? p.gk : p.gq);
      T *const dx = (T *)(side ? p.ko : p.qo);
      const int64_t x_rs = side ? p.k_rs : p.q_rs, dy_rs = side ? p.gk_rs : p.gq_rs, dx_rs = side ? p.ko_rs : p.qo_rs;
      if (total == 0) continue;
      Raw8<T> wr;
      wr.load((const T *)(side ? p.wk : p.wq) + e);
      const Eight w = wr.floats();
      Walk at(tid, THREADS, per);
      for (int first = tid; first < total; first += THREADS * kPairs) {
        Raw8<T> xr[kPairs], gr[kPairs];
        int row[kPairs], to[kPairs];
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
          if (first + THREADS * n >= total) break;
          row[n] = at.row;
          to[n] = at.rest / LANES * D + e;
          at.step();
          xr[n].load(x + (row0 + row[n]) * x_rs + to[n]);
          gr[n].load(dy + (row0 + row[n]) * dy_rs + to[n]);
        }
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
          if (first + THREADS * n >= total) break;
          const Eight v = xr[n].floats();
          Eight g = gr[n].floats();
          if (p.turn) turn8(g, &cs[row[n]][e / 2], true);
          const float r = head_rms<LANES>(v, p.eps);
          float dot = 0.f;
          Eight y;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float u = v.x[j] * r;  // the normed element
            dw[side].x[j] = fmaf(g.x[j], u, dw[side].x[j]);
            g.x[j] *= w.x[j];
            dot = fmaf(g.x[j], u, dot);
            y.x[j] = u;
          }
          dot = head_sum<LANES>(dot) * (1.0f / D);
#pragma unroll
          for (int j = 0; j < 8; ++j) y.x[j] = r * (g.x[j] - y.x[j] * dot);
          store8(dx + (row0 + row[n]) * dx_rs + to[n], y);
        }
      }
    }
  }
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = dw[side].x[j];
#pragma unroll
      for (int m = LANES; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
      if (lane < LANES) sums.of_wave[tid >> 6][side][e + j] = s;
    }
  __syncthreads();
  float *const part = p.parts + (int64_t)blockIdx.x * 2 * D;
  for (int i = 2 * tid; i < 2 * D; i += 2 * THREADS) {
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      s.x += sums.of_wave[w][i / D][i % D];
      s.y += sums.of_wave[w][i / D][i % D + 1];
    }
    if (JOINS) put2(part + i, s.x, s.y);
    else *(float2 *)(part + i) = s;
  }
  if constexpr (!JOINS) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums' stores have reached memory
  __syncthreads();
  if (tid == 0) last = arrive_last(p.arrive, (int)gridDim.x, p.tag);
  __syncthreads();
  if (!last) return;
  // The last workgroup to arrive: two elements a thread, of every STEP-th workgroup's sums.
  const int at2 = tid % D * 2, n = (int)gridDim.x;
  float2 s = make_float2(0.f, 0.f);
  for (int i0 = tid / D; i0 < n; i0 += STEP * N) {
    float2 x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i0 + STEP * j < n ? get2(p.parts + (int64_t)(i0 + STEP * j) * 2 * D + at2) : make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      s.x += x[j].x;
      s.y += x[j].y;
    }
  }
  *(float2 *)&sums.of_groups[tid / D][at2] = s;
  __syncthreads();
  for (int i = tid; i < 2 * D; i += THREADS) {
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < STEP; ++j) y += sums.of_groups[j][i];
    if (i < D) p.dwq[i] = y;
    else if (p.dwk) p.dwk[i - D] = y;
  }
}

// The workgroups' sums, added: eight elements a workgroup, 32 threads an element.
__global__ __launch_bounds__(256) void qk_norm_rope_weights_kernel(const float *parts, int n, int d, float *dwq,
                                                                   float *dwk) {
  constexpr int N = 16;  // on their way at once
  __shared__ float sums[4][8];
  const int tid = threadIdx.x, e = blockIdx.x * 8 + (tid & 7);
  float s = 0.f;
  for (int i0 = tid >> 3; i0 < n; i0 += 32 * N) {
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = i0 + 32 * j < n ? parts[(int64_t)(i0 + 32 * j) * 2 * d + e] : 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += x[j];
  }
#pragma unroll
  for (int m = 8; m < 64; m <<= 1) s += __shfl_xor(s, m, 64);
  if ((tid & 63) < 8) sums[tid >> 6][tid & 7] = s;
  __syncthreads();
  if (tid >= 8) return;
  s = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  if (e < d) dwq[e] = s;
  else if (dwk) dwk[e - d] = s;
}

int check_qk(const std::string &op, int dtype, const void *q, const void *k, const void *wq, const void *wk,
             int n_rows, int n_heads, int n_kv_heads, int head_dim, float eps, float theta) {
  if (dtype != BN_F32 && dtype != BN_BF16) return fail(BN_ERR_UNSUPPORTED, op + ": dtype must be F32 or BF16");
  if (n_rows < 0) return fail(BN_ERR_SHAPE, op + ": negative number of rows");
  if (n_rows > (1 << 23)) return fail(BN_ERR_UNSUPPORTED, op + ": more than 2^23 rows");
  if (n_heads <= 0) return fail(BN_ERR_SHAPE, op + ": num_heads must be positive");
  if (n_kv_heads < 0) return fail(BN_ERR_SHAPE, op + ": negative num_kv_heads");
  if (n_heads > 65535 || n_kv_heads > 65535) return fail(BN_ERR_UNSUPPORTED, op + ": more than 65535 heads");
  if (head_dim < 16 || head_dim > kMaxHeadDim || (head_dim & (head_dim - 1)))
    return fail(BN_ERR_UNSUPPORTED, op + ": head_dim must be 16, 32, 64, 128 or 256");
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(BN_ERR_INVALID_ARG, op + ": eps must be finite and not negative");
  if (!(theta >= 0.f) || !std::isfinite(theta))
    return fail(BN_ERR_INVALID_ARG, op + ": theta must be positive and finite, or 0 for no rotation");
  if (n_rows > 0 && ((n_kv_heads > 0) != (k != nullptr)))
    return fail(BN_ERR_INVALID_ARG, op + ": k and num_kv_heads must be given together");
  if (!wq || (n_kv_heads > 0 && !wk)) return fail(BN_ERR_INVALID_ARG, op + ": weight is NULL");
  if (!aligned16(wq) || !aligned16(wk)) return fail(BN_ERR_UNSUPPORTED, op + ": weights must be 16-byte aligned");
  return BN_OK;
}

// K<T, D, ...> for the dtype and head dimension
#define BN_QK_LAUNCH_D(K, D, grid, block, s, p, ...)                                                 \
  do {                                                                                               \
    Turns<D> t;                                                                                      \
    fill_turns(t.f, D, theta);                                                                       \
    if (dtype == BN_BF16) hipLaunchKernelGGL((K<bf16_t, D, ##__VA_ARGS__>), grid, dim3(block), 0, s, p, t); \
    else hipLaunchKernelGGL((K<float, D, ##__VA_ARGS__>), grid, dim3(block), 0, s, p, t);            \
  } while (0)
#define BN_QK_LAUNCH(K, grid, block, s, p, ...)                                          \
  do {                                                                                   \
    if (head_dim == 16) BN_QK_LAUNCH_D(K, 16, grid, block, s, p, ##__VA_ARGS__);         \
    else if (head_dim == 32) BN_QK_LAUNCH_D(K, 32, grid, block, s, p, ##__VA_ARGS__);    \
    else if (head_dim == 64) BN_QK_LAUNCH_D(K, 64, grid, block, s, p, ##__VA_ARGS__);    \
    else if (head_dim == 128) BN_QK_LAUNCH_D(K, 128, grid, block, s, p, ##__VA_ARGS__);  \
    else BN_QK_LAUNCH_D(K, 256, grid, block, s, p, ##__VA_ARGS__);                       \
  } while (0)

}  // namespace
}  // namespace bn

using namespace bn;

extern "C" {

int bn_qk_norm_rope(int dtype, const void *q, const void *k, const void *q_weight, const void *k_weight,
                    void *q_out, void *k_out, const int32_t *positions, int n_rows, int n_heads, int n_kv_heads,
                    int head_dim, int64_t q_row_stride, int64_t k_row_stride, int64_t q_out_row_stride,
                    int64_t k_out_row_stride, int position_offset, float eps, float theta, void *stream) {
  const std::string op = "QK norm";
  int st = check_qk(op, dtype, q, k, q_weight, k_weight, n_rows, n_heads, n_kv_heads, head_dim, eps, theta);
  if (st) return st;
  if (n_rows == 0) return BN_OK;
  if ((st = check_rows(op, "q", q, n_rows, n_heads, q_row_stride, dtype, head_dim)) ||
      (st = check_rows(op, "q_out", q_out, n_rows, n_heads, q_out_row_stride, dtype, head_dim)) ||
      (k && ((st = check_rows(op, "k", k, n_rows, n_kv_heads, k_row_stride, dtype, head_dim)) ||
             (st = check_rows(op, "k_out", k_out, n_rows, n_kv_heads, k_out_row_stride, dtype, head_dim)))))
    return st;
  if ((q == q_out && q_row_stride != q_out_row_stride) || (k && k == k_out && k_row_stride != k_out_row_stride))
    return fail(BN_ERR_INVALID_ARG, op + ": an output in its input's place must have its row stride");
  if ((uintptr_t)positions & 3u) return fail(BN_ERR_UNSUPPORTED, op + ": positions must be 4-byte aligned");
  DeviceScope scope;
  if ((st = scope.enter(op, q, "q"))) return st;
  QkParams p{};
  p.q = q; p.k = k; p.wq = q_weight; p.wk = k_weight; p.qo = q_out; p.ko = k_out;
  p.positions = positions;
  p.q_rs = q_row_stride; p.k_rs = k_row_stride; p.qo_rs = q_out_row_stride; p.ko_rs = k_out_row_stride;
  p.n_rows = n_rows; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
  p.rows = rows_at_once(n_rows);
  p.turn = theta > 0.f;
  p.offset = position_offset;
  p.eps = eps;
  const dim3 grid((unsigned)((n_rows + p.rows - 1) / p.rows));
  BN_QK_LAUNCH(qk_norm_rope_kernel, grid, 256, as_stream(stream), p);
  BN_LAUNCH_CHECK();
  return BN_OK;
}

size_t bn_qk_norm_rope_backward_workspace_size(int n_rows, int n_heads, int n_kv_heads, int head_dim) {
  const float w = 0.f;
  if (check_qk("", BN_F32, &w, n_kv_heads > 0 ? &w : nullptr, (const void *)16, (const void *)16, n_rows, n_heads, n_kv_heads,
               head_dim, 0.f, 0.f))
    return 0;
  return kArriveBytes + (size_t)std::min(n_rows, kBackGroups) * 2 * head_dim * sizeof(float);  // (does for fewer rows)
}

int bn_qk_norm_rope_backward(int dtype, const void *q, const void *k, const void *q_weight, const void *k_weight,
                             const void *dq_out, const void *dk_out, void *dq, void *dk, float *dq_weight,
                             float *dk_weight, const int32_t *positions, int n_rows, int n_heads, int n_kv_heads,
                             int head_dim, int64_t q_row_stride, int64_t k_row_stride, int64_t dq_out_row_stride,
                             int64_t dk_out_row_stride, int64_t dq_row_stride, int64_t dk_row_stride,
                             int position_offset, float eps, float theta, void *workspace, size_t workspace_bytes,
                             void *stream) {
  const std::string op = "QK norm backward";
  int st = check_qk(op, dtype, q, k, q_weight, k_weight, n_rows, n_heads, n_kv_heads, head_dim, eps, theta);
  if (st) return st;
  if (!dq_weight || (n_kv_heads > 0 && !dk_weight))
    return fail(BN_ERR_INVALID_ARG, op + ": gradient of a weight is NULL");
  if (((uintptr_t)dq_weight | (uintptr_t)dk_weight) & 3u)
    return fail(BN_ERR_UNSUPPORTED, op + ": gradients of the weights must be 4-byte aligned");
  if (n_rows > 0 &&
      ((st = check_rows(op, "q", q, n_rows, n_heads, q_row_stride, dtype, head_dim)) ||
       (st = check_rows(op, "dq_out", dq_out, n_rows, n_heads, dq_out_row_stride, dtype, head_dim)) ||
       (st = check_rows(op, "dq", dq, n_rows, n_heads, dq_row_stride, dtype, head_dim)) ||
       (k && ((st = check_rows(op, "k", k, n_rows, n_kv_heads, k_row_stride, dtype, head_dim)) ||
              (st = check_rows(op, "dk_out", dk_out, n_rows, n_kv_heads, dk_out_row_stride, dtype, head_dim)) ||
              (st = check_rows(op, "dk", dk, n_rows, n_kv_heads, dk_row_stride, dtype, head_dim))))))
    return st;
  if (n_rows > 0 && ((dq == q && dq_row_stride != q_row_stride) || (dq == dq_out && dq_row_stride != dq_out_row_stride) ||
                     (k && ((dk == k && dk_row_stride != k_row_stride) || (dk == dk_out && dk_row_stride != dk_out_row_stride)))))
    return fail(BN_ERR_INVALID_ARG, op + ": an output in an input's place must have its row stride");
  if ((uintptr_t)positions & 3u) return fail(BN_ERR_UNSUPPORTED, op + ": positions must be 4-byte aligned");
  const size_t need = bn_qk_norm_rope_backward_workspace_size(n_rows, n_heads, n_kv_heads, head_dim);
  if (workspace && workspace_bytes < need)
    return fail(BN_ERR_INVALID_ARG, op + ": workspace of " + std::to_string(workspace_bytes) + " bytes, need " +
                                        std::to_string(need));
  if (workspace && !aligned16(workspace))
    return fail(BN_ERR_UNSUPPORTED, op + ": workspace must be 16-byte aligned");
  DeviceScope scope;
  if ((st = scope.enter(op, q_weight, "q_weight"))) return st;
  QkParams p{};
  p.q = q; p.k = k; p.wq = q_weight; p.wk = k_weight; p.gq = dq_out; p.gk = dk_out; p.qo = dq; p.ko = dk;
  p.positions = positions;
  p.q_rs = q_row_stride; p.k_rs = k_row_stride; p.gq_rs = dq_out_row_stride; p.gk_rs = dk_out_row_stride;
  p.qo_rs = dq_row_stride; p.ko_rs = dk_row_stride;
  p.n_rows = n_rows; p.n_heads = n_heads; p.n_kv_heads = n_kv_heads;
  const BackPlan d = plan_back(n_rows, n_heads + n_kv_heads, head_dim);
  p.rows = d.rows;
  p.turn = theta > 0.f;
  p.offset = position_offset;
  p.eps = eps;
  Workspace ws;
  if ((st = ws.take(workspace, need, stream))) return st;
  p.arrive = (unsigned long long *)ws.p;
  p.parts = (float *)((char *)ws.p + kArriveBytes);
  p.dwq = dq_weight; p.dwk = dk_weight;
  p.tag = next_tag();
  hipStream_t s = as_stream(stream);
  auto launch = [&]() -> int {
    if (d.groups > 0) {
      // (512 threads for bf16 in few workgroups for a compute unit: 2048 rows 13.9 -> 12.6 us, of heads
      // of 256 38.4 -> 29.1; 16384 rows 49.6 -> 52.4; 777 of heads of 256 in fp32 24.3 -> 27.3)
      const dim3 grid((unsigned)d.groups);
      if (d.joins) BN_QK_LAUNCH(qk_norm_rope_backward_kernel, grid, 512, s, p, 512, true);
      else if (dtype == BN_BF16 && d.groups <= kBackGroups / 2) BN_QK_LAUNCH(qk_norm_rope_backward_kernel, grid, 512, s, p, 512, false);
      else BN_QK_LAUNCH(qk_norm_rope_backward_kernel, grid, 256, s, p, 256, false);
      BN_LAUNCH_CHECK();
    }
    if (d.joins) return BN_OK;
    hipLaunchKernelGGL(qk_norm_rope_weights_kernel, dim3((unsigned)(2 * head_dim / 8)), dim3(256), 0, s, p.parts, d.groups,
                       head_dim, dq_weight, dk_weight);
    BN_LAUNCH_CHECK();
    return BN_OK;
  };
  return ws.release(launch());
}

}  // extern "C"
