// What the forward and the backward of the residual norm share (residual_norm_fwd.hip has the
// formulas).
#pragma once

#include <algorithm>
#include <type_traits>

#include "bevk_launch.h"

namespace bevk {
namespace rnorm {

// Sums over the TPR neighbouring threads that have a row, in each of them; the same order for all.
// More than a wave: through s (2 * THREADS / 64 * 2 floats, of which a call uses one half and the next
// the other, so one barrier is enough).
template <int TPR, int THREADS, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float *s, int &turn) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    auto turned = [&](float v, auto ctrl) __attribute__((always_inline)) {
      return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                                       decltype(ctrl)::value, 0xf, 0xf, false));
    };
    float v = x[k];
    v = turned(v, std::integral_constant<int, 0x128>());  // row_ror 8, 4, 2, 1
    v = turned(v, std::integral_constant<int, 0x124>());
    v = turned(v, std::integral_constant<int, 0x122>());
    v = turned(v, std::integral_constant<int, 0x121>());
    if constexpr (TPR >= 32) v += __shfl_xor(v, 16, kWave);
    if constexpr (TPR >= 64) v += __shfl_xor(v, 32, kWave);
    x[k] = v;
  }
  if constexpr (TPR > 64) {
    static_assert(N <= 2, "s");
    constexpr int W = TPR / 64, ALL = THREADS / 64;
    float *d = s + turn * ALL * 2;
    turn ^= 1;
    const int wave = threadIdx.x / 64, first = wave / W * W;
    if (threadIdx.x % 64 == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) d[wave * N + k] = x[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float v = d[first * N + k];
#pragma unroll
      for (int w = 1; w < W; ++w) v += d[(first + w) * N + k];
      x[k] = v;
    }
  }
}

// The stream's value, in the forward and again in the backward: the same bits.
__device__ __forceinline__ float block_value(float x, float mean, float rstd, float w, float b) {
  return __builtin_fmaf((x - mean) * rstd, w, b);
}
__device__ __forceinline__ float stream_value(float p, float scale, float gate, float residual) {
  return __builtin_fmaf(scale * gate, p, residual);
}

template <typename T, int V>
__device__ __forceinline__ void load_row(const T *p, float (&x)[V]) {
  const Vec<T, V> y = load_vec<T, V>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) x[e] = (float)y.v[e];
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T *p, const float (&x)[V]) {
  Vec<T, V> y;
#pragma unroll
  for (int e = 0; e < V; ++e) y.v[e] = static_cast<T>(x[e]);
  store_vec<T, V>(p, y);
}
// A parameter in T or (wide) fp32, `none` where there is none.
template <typename T, int V>
__device__ __forceinline__ void load_param(const void *p, bool wide, int64_t at, float none, float (&x)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = none;
  } else if (sizeof(T) == 4 || wide) {
    constexpr int W = V > 4 ? 4 : V;
#pragma unroll
    for (int k = 0; k < V; k += W) {
      const Vec<float, W> y = load_vec<float, W>(static_cast<const float *>(p) + at + k);
#pragma unroll
      for (int e = 0; e < W; ++e) x[k + e] = y.v[e];
    }
  } else {
    load_row<T, V>(static_cast<const T *>(p) + at, x);
  }
}

// A launch for a row of `vecs` vectors: f(threads a row, vectors a thread), or false where a row does
// not fit (2 vectors for each of 1,024 threads).
template <typename F> bool for_row(int64_t vecs, F f) {
  auto n = [](auto k) { return k; };
  using std::integral_constant;
  if (vecs <= 16) f(n(integral_constant<int, 16>()), n(integral_constant<int, 1>()));
  else if (vecs <= 32) f(n(integral_constant<int, 32>()), n(integral_constant<int, 1>()));
  else if (vecs <= 64) f(n(integral_constant<int, 64>()), n(integral_constant<int, 1>()));
  else if (vecs <= 128) f(n(integral_constant<int, 128>()), n(integral_constant<int, 1>()));
  else if (vecs <= 256) f(n(integral_constant<int, 256>()), n(integral_constant<int, 1>()));
  else if (vecs <= 512) f(n(integral_constant<int, 512>()), n(integral_constant<int, 1>()));
  else if (vecs <= 1024) f(n(integral_constant<int, 1024>()), n(integral_constant<int, 1>()));
  else if (vecs <= 2048) f(n(integral_constant<int, 1024>()), n(integral_constant<int, 2>()));
  else return false;
  return true;
}

constexpr int threads_of(int tpr) { return tpr > 256 ? tpr : 256; }

inline bool on_16(std::initializer_list<const void *> all) {
  for (const void *p : all)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

}  // namespace rnorm
}  // namespace bevk
