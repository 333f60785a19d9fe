// The norms between two blocks of a transformer (gfx950): a block's output through a norm of its own or
// none, times a gate and a scale onto the residual stream, and the next block's norm of that.
//
//   p = x, or (x - mean_x) rstd_x * bw + bb
//   h = residual + scale * gate * p
//   y = (h - mean) rstd * w + b            mean over a row's channels, rstd = 1 / sqrt(var + eps);
//                                          rms: no mean, rstd = 1 / sqrt(mean of squares + eps)
//
// A row stays in registers: one 16-byte vector a thread, TPR threads a row (16 of a wave up to a
// workgroup of 1,024; two vectors at the most), so that each input is read once and each output
// written once. The variance is taken about the mean, in a second sum over the registers: exact where
// the mean is far from zero. All sums fp32, in one order. y is computed from the unrounded h; the
// stream that is written is h rounded once.
// Rows that do not fit (more than 2,048 vectors) are read again for every sum (any_forward_kernel).
// Bound by memory: 40,000 x 256 bf16 61 MB in 11.5 us (5.3 TB/s), 34,800 x 512 fp16 with gate and stream 143 MB in
// 30 us (4.8), 16,384 x 2,048 bf16 with both norms 268 MB in 53 us (5.1, a copy's rate at that size); 300 x 256
// fp32 2.8 us, a launch.
#include "residual_norm.h"

namespace bevk {
namespace {
using namespace rnorm;

template <typename T, int V, int TPR, int L>
__global__ void __launch_bounds__(threads_of(TPR)) forward_kernel(const ResidualNormArgs a, const ResidualNormOut o,
                                                                  int64_t first) {
  constexpr int THREADS = threads_of(TPR), R = THREADS / TPR;
  __shared__ float s[2 * THREADS / 64 * 2];
  int turn = 0;
  const int j = threadIdx.x % TPR;
  const float inv = 1.f / (float)a.channels;
  const int64_t row = (first + blockIdx.x) * R + threadIdx.x / TPR;
  const bool there = row < a.rows;
  const int64_t at = row * a.channels;
  const T *x = static_cast<const T *>(a.x) + at, *res = static_cast<const T *>(a.residual) + at;
  float h[L][V], r[L][V];
  bool in[L];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const int c = (l * TPR + j) * V;
    in[l] = there && c < a.channels;
#pragma unroll
    for (int e = 0; e < V; ++e) h[l][e] = r[l][e] = 0.f;
    if (in[l]) {
      load_row<T, V>(x + c, h[l]);
      if (a.residual != nullptr) load_row<T, V>(res + c, r[l]);
    }
  }
  float *stats = o.stats == nullptr ? nullptr : o.stats + row * (a.block ? 4 : 2);
  // mean (0 for rms) and 1 / spread of h over the row; what is past its end is 0 and stays out of the variance
  auto moments = [&](float &mean, float &rstd, float *keep) __attribute__((always_inline)) {
    float t[1] = {0.f};
    if (!a.rms) {
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e) t[0] += h[l][e];
      row_sums<TPR, THREADS, 1>(t, s, turn);
    }
    mean = t[0] * inv;
    t[0] = 0.f;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = h[l][e] - mean;
        q = __builtin_fmaf(d, d, q);
      }
      t[0] += in[l] ? q : 0.f;
    }
    row_sums<TPR, THREADS, 1>(t, s, turn);
    // (the hardware's, right to a unit in the last place: a part in 2^23 of y, below the sums' own error)
    rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(t[0], inv, a.eps));
    if (keep != nullptr && there && j == 0) {
      keep[0] = mean;
      keep[1] = rstd;
    }
  };
  float mean, rstd;
  if (a.block) {
    moments(mean, rstd, stats == nullptr ? nullptr : stats + 2);
#pragma unroll
    for (int l = 0; l < L; ++l)
      if (in[l]) {
        const int c = (l * TPR + j) * V;
        float w[V], b[V];
        load_param<T, V>(a.block_weight, a.wide, c, 1.f, w);
        load_param<T, V>(a.block_bias, a.wide, c, 0.f, b);
#pragma unroll
        for (int e = 0; e < V; ++e) h[l][e] = block_value(h[l][e], mean, rstd, w[e], b[e]);
      }
  }
  const int64_t gate_at = a.set_rows > 0 ? row / a.set_rows * a.channels : 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
    if (in[l]) {
      const int c = (l * TPR + j) * V;
      float g[V];
      load_param<T, V>(a.gate, a.gate_wide, gate_at + c, 1.f, g);
#pragma unroll
      for (int e = 0; e < V; ++e) h[l][e] = stream_value(h[l][e], a.scale, g[e], r[l][e]);
      if (o.h != nullptr) store_row<T, V>(static_cast<T *>(o.h) + at + c, h[l]);
    }
  moments(mean, rstd, stats);
#pragma unroll
  for (int l = 0; l < L; ++l)
    if (in[l]) {
      const int c = (l * TPR + j) * V;
      float w[V], b[V];
      load_param<T, V>(a.weight, a.wide, c, 1.f, w);
      load_param<T, V>(a.bias, a.wide, c, 0.f, b);
#pragma unroll
      for (int e = 0; e < V; ++e) h[l][e] = __builtin_fmaf((h[l][e] - mean) * rstd, w[e], b[e]);
      store_row<T, V>(static_cast<T *>(o.y) + at + c, h[l]);
    }
}

// Any row length: a workgroup a row, each sum a pass over it.
template <typename T>
__global__ void __launch_bounds__(256) any_forward_kernel(const ResidualNormArgs a, const ResidualNormOut o,
                                                          int64_t first) {
  __shared__ float s[2 * 4 * 2];
  int turn = 0;
  const int64_t row = first + blockIdx.x, at = row * a.channels;
  const T *x = static_cast<const T *>(a.x) + at, *res = static_cast<const T *>(a.residual) + at;
  const int64_t gate_at = a.set_rows > 0 ? row / a.set_rows * a.channels : 0;
  float mean_x = 0.f, rstd_x = 1.f, mean, rstd;
  auto stream_at = [&](int c) __attribute__((always_inline)) {
    float p = (float)x[c];
    float w[1], b[1], g[1];
    if (a.block) {
      load_param<T, 1>(a.block_weight, a.wide, c, 1.f, w);
      load_param<T, 1>(a.block_bias, a.wide, c, 0.f, b);
      p = block_value(p, mean_x, rstd_x, w[0], b[0]);
    }
    load_param<T, 1>(a.gate, a.gate_wide, gate_at + c, 1.f, g);
    return stream_value(p, a.scale, g[0], a.residual != nullptr ? (float)res[c] : 0.f);
  };
  auto moments = [&](auto value, float &mean_of, float &rstd_of) __attribute__((always_inline)) {
    float m = 0.f;
    if (!a.rms) {
      float t[1] = {0.f};
      for (int c = threadIdx.x; c < a.channels; c += 256) t[0] += value(c);
      row_sums<256, 256, 1>(t, s, turn);
      m = t[0] / (float)a.channels;
    }
    float t[1] = {0.f};
    for (int c = threadIdx.x; c < a.channels; c += 256) {
      const float d = value(c) - m;
      t[0] = __builtin_fmaf(d, d, t[0]);
    }
    row_sums<256, 256, 1>(t, s, turn);
    mean_of = m;
    rstd_of = 1.f / sqrtf(t[0] / (float)a.channels + a.eps);
  };
  if (a.block) moments([&](int c) { return (float)x[c]; }, mean_x, rstd_x);
  moments(stream_at, mean, rstd);
  if (o.stats != nullptr && threadIdx.x == 0) {
    float *d = o.stats + row * (a.block ? 4 : 2);
    d[0] = mean;
    d[1] = rstd;
    if (a.block) {
      d[2] = mean_x;
      d[3] = rstd_x;
    }
  }
  for (int c = threadIdx.x; c < a.channels; c += 256) {
    const float h = stream_at(c);
    if (o.h != nullptr) static_cast<T *>(o.h)[at + c] = static_cast<T>(h);
    float w[1], b[1];
    load_param<T, 1>(a.weight, a.wide, c, 1.f, w);
    load_param<T, 1>(a.bias, a.wide, c, 0.f, b);
    static_cast<T *>(o.y)[at + c] = static_cast<T>(__builtin_fmaf((h - mean) * rstd, w[0], b[0]));
  }
}

template <typename T, int V>
hipError_t launch_v(const ResidualNormArgs &a, const ResidualNormOut &o, hipStream_t stream) {
  hipError_t e = hipSuccess;
  const bool fits = for_row((a.channels + V - 1) / V, [&](auto tpr, auto l) {
    constexpr int TPR = decltype(tpr)::value, L = decltype(l)::value, THREADS = threads_of(TPR);
    e = launch_in_parts((a.rows + THREADS / TPR - 1) / (THREADS / TPR), THREADS, [&](int64_t first, unsigned n) {
      hipLaunchKernelGGL((forward_kernel<T, V, TPR, L>), dim3(n), dim3(THREADS), 0, stream, a, o, first);
    });
  });
  if (fits) return e;
  return launch_in_parts(a.rows, 256, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((any_forward_kernel<T>), dim3(n), dim3(256), 0, stream, a, o, first);
  });
}
template <typename T> hipError_t launch_t(const ResidualNormArgs &a, const ResidualNormOut &o, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = a.channels % V == 0 && on_16({a.x, a.residual, a.weight, a.bias, a.gate, a.block_weight,
                                                   a.block_bias, o.y, o.h});
  return whole ? launch_v<T, V>(a, o, stream) : launch_v<T, 1>(a, o, stream);
}

}  // namespace

hipError_t launch_residual_norm_forward(int dtype, const ResidualNormArgs &a, const ResidualNormOut &o,
                                        hipStream_t stream) {
  switch (dtype) {
    case 0: return launch_t<float>(a, o, stream);
    case 1: return launch_t<f16>(a, o, stream);
    default: return launch_t<bf16>(a, o, stream);
  }
}

}  // namespace bevk
