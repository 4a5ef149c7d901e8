// bn_head_rows.hpp -- rows of heads, eight consecutive elements a lane, a head's
// lanes next to each other: what kernels that norm or turn single heads share.
#pragma once

#include "bn_paged_device.hpp"

namespace bn {
namespace {

struct Eight {
  float x[8];
};
template <typename T>
struct Raw8 {  // as loaded
  u32x4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r[i] = ((const u32x4 *)p)[i];
  }
  __device__ __forceinline__ Eight floats() const {
    Eight y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        y.x[2 * i] = __uint_as_float(r[0][i] << 16);
        y.x[2 * i + 1] = __uint_as_float(r[0][i] & 0xffff0000u);
      } else {
        y.x[i] = __uint_as_float(r[0][i]);
        y.x[4 + i] = __uint_as_float(r[sizeof(T) / 2 - 1][i]);
      }
    }
    return y;
  }
};
template <typename T, bool NT = false>  // NT: past the caches' keeping
__device__ __forceinline__ void store8(T *p, const Eight &y) {
  u32x4 r[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      r[0][i] = (uint32_t)f32_to_bf16(y.x[2 * i]) | ((uint32_t)f32_to_bf16(y.x[2 * i + 1]) << 16);
    } else {
      r[0][i] = __float_as_uint(y.x[i]);
      r[sizeof(T) / 2 - 1][i] = __float_as_uint(y.x[4 + i]);
    }
  }
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    if constexpr (NT) __builtin_nontemporal_store(r[i], (u32x4 *)p + i);
    else ((u32x4 *)p)[i] = r[i];
  }
}

// The sum over the LANES lanes of a head (a power of two up to 32), in each of them.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (LANES >= 2) v = dpp_addf<0xB1, 0xf>(v);   // the neighbour's
  if constexpr (LANES >= 4) v = dpp_addf<0x4E, 0xf>(v);   // the other pair's of four
  if constexpr (LANES >= 8) v = dpp_addf<0x141, 0xf>(v);  // the other four's of eight
  if constexpr (LANES >= 16) v = dpp_addf<0x140, 0xf>(v);  // the other eight's of sixteen
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}

// 1 / sqrt(mean(x^2) + eps) of a head of 8 LANES elements.
template <int LANES>
__device__ __forceinline__ float head_rms(const Eight &v, float eps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(v.x[i], v.x[i], s);
  return rsqrtf(fmaf(head_sum<LANES>(s), 1.0f / (8 * LANES), eps));
}

// The four pairs turned by their angles (back: by the negative ones).
__device__ __forceinline__ void turn8(Eight &v, const float2 *cs, bool back = false) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = cs[i];
    const float s = back ? -t.y : t.y, a = v.x[2 * i], b = v.x[2 * i + 1];
    v.x[2 * i] = a * t.x - b * s;
    v.x[2 * i + 1] = a * s + b * t.x;
  }
}

// Thread tid's way through rows of `per` pieces each, every `by`-th piece, without a division a piece.
struct Walk {
  int row, rest, per, rows_by, rest_by;
  __device__ __forceinline__ Walk(int tid, int by, int per_) : per(per_) {
    row = (int)((uint32_t)tid / (uint32_t)per);
    rest = tid - row * per;
    rows_by = __builtin_amdgcn_readfirstlane((int)((uint32_t)by / (uint32_t)per));
    rest_by = by - rows_by * per;
  }
  __device__ __forceinline__ void step() {
    row += rows_by;
    rest += rest_by;
    if (rest >= per) {
      rest -= per;
      ++row;
    }
  }
};

// f[i] = theta^(-2i/head_dim) / (2 pi): turns per position of each pair (theta 0: none).
inline void fill_turns(double *f, int head_dim, float theta) {
  const int n = head_dim / 2;
  double low[8];  // (a power of eight pairs and one within: a few roundings instead of a pow a pair)
  for (int i = 0; i < 8 && i < n; ++i) low[i] = theta > 0.f ? std::pow((double)theta, -2.0 * i / head_dim) : 0.0;
  for (int i = 0; i < n; i += 8) {
    const double high = theta > 0.f ? std::pow((double)theta, -2.0 * i / head_dim) / (2.0 * M_PI) : 0.0;
    for (int j = 0; j < 8; ++j) f[i + j] = high * low[j];
  }
}

}  // namespace
}  // namespace bn
