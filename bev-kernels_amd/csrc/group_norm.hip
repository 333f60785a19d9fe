// Group normalization with an activation on channels-last maps, forward and backward (gfx950).
//
// x [N][P][C], C = G * per: each (image, group) of m = P * per values is brought to mean 0 and
// variance 1, then scaled and shifted by channel:
//   mean = sum x / m,  var = sum x^2 / m - mean^2,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) * rstd,  z = xh * w + b,  y = act(z)
// and, with gz = gy * act'(z):
//   gb = sum gz, gw = sum gz * xh over images and positions,
//   gx = rstd * (w * gz - (s1 + xh * s2) / m),  s1 = sum w * gz, s2 = sum w * gz * xh over the group.
//
// The sums of x and x^2 are held in fp64: then the squares need no second pass over x for their
// mean to be taken off first (var loses mean^2 / var * 2^-52), and the position where ReLU's
// derivative jumps is known to about 2^-50 (see Gate).
#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float to_f32(const void *p, int dtype, int64_t i, float none) {
  if (p == nullptr) return none;
  switch (dtype) {
    case 0: return static_cast<const float *>(p)[i];
    case 1: return (float)static_cast<const f16 *>(p)[i];
    default: return (float)static_cast<const bf16 *>(p)[i];
  }
}
__device__ __forceinline__ void from_f32(void *p, int dtype, int64_t i, float v) {
  switch (dtype) {
    case 0: static_cast<float *>(p)[i] = v; break;
    case 1: static_cast<f16 *>(p)[i] = static_cast<f16>(v); break;
    default: static_cast<bf16 *>(p)[i] = static_cast<bf16>(v); break;
  }
}

// Sum over a workgroup; every thread gets it.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A *s) {
  __syncthreads();
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_down(v, d, kWave);
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  A t = s[0];
  for (int k = 1; k < kThreads / kWave; ++k) t += s[k];
  return t;
}

__device__ __forceinline__ float act_of(float z, int act) {
  if (act == kActRelu) return z <= 0.f ? 0.f : z;  // NaN stays
  if (act == kActSilu) return z / (1.f + expf(-z));
  return z;
}

// x - mean with mean as two floats, so that a mean far from 0 costs no digits of the difference.
struct Mean2 {
  float h, l;
};
__device__ __forceinline__ Mean2 split_mean(double m) {
  const float h = (float)m;
  return {h, (float)(m - (double)h)};
}
__device__ __forceinline__ float centred(float x, Mean2 m) { return (x - m.h) - m.l; }

// Where a channel's z is above 0. z = 0 at x = mean - b / (rstd * w), and rounding z to 32 bits
// may put an element next to it on the wrong side, which moves its gradient by all of its size.
// So x itself is compared with the position, found in 64 bits and rounded towards -inf (x is a
// float: x > t as real numbers exactly if x > t rounded down).
struct Gate {
  float thr, sign;
};
__device__ __forceinline__ Gate make_gate(double mean, double rstd, float w, float b) {
  const double a = rstd * (double)w;
  if (a == 0.0) return {b > 0.f ? -INFINITY : INFINITY, 1.f};
  const double s = a < 0.0 ? -1.0 : 1.0, t = s * (mean - (double)b / a);
  float f = (float)t;
  if ((double)f > t) f = nextafterf(f, -INFINITY);
  return {f, (float)s};
}
__device__ __forceinline__ float gated(float gy, float x, Gate g) {
  return x * g.sign <= g.thr ? 0.f : gy;  // NaN passes, as in ReLU's own derivative
}

__device__ __forceinline__ float silu_grad(float gy, float z) {
  const float s = 1.f / (1.f + expf(-z));
  return gy * (s * (1.f + z * (1.f - s)));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) stats_kernel(const T *__restrict__ x, int64_t P, int C, int per,
                                                         double eps, double *__restrict__ stats) {
  __shared__ double s[kThreads / kWave];
  const int64_t n = blockIdx.y;
  const int g = blockIdx.x;
  double a = 0.0, q = 0.0;
  for (int64_t i = threadIdx.x; i < P * per; i += kThreads) {
    const double v = (double)x[(n * P + i / per) * C + (int64_t)g * per + i % per];
    a += v;
    q += v * v;
  }
  a = block_sum(a, s);
  q = block_sum(q, s);
  if (threadIdx.x == 0) {
    const double m = (double)(P * per), mean = a / m, var = q / m - mean * mean;
    stats[(n * gridDim.x + g) * 2] = mean;
    stats[(n * gridDim.x + g) * 2 + 1] = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T *__restrict__ x, int64_t total, int64_t P,
                                                           int C, int per, const void *w, const void *b,
                                                           int wd, int act,
                                                           const double *__restrict__ stats, T *__restrict__ y) {
  const int G = C / per;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int c = (int)(i % C);
    const int64_t n = i / C / P;
    const double *st = stats + (n * G + c / per) * 2;
    const float z = centred((float)x[i], split_mean(st[0])) * (float)st[1] * to_f32(w, wd, c, 1.f) +
                    to_f32(b, wd, c, 0.f);
    y[i] = static_cast<T>(act_of(z, act));
  }
}

// gz and xh of one element.
template <typename T>
__device__ __forceinline__ void grad_of(const T *gy, const T *x, int64_t i, const double *st, float w, float b,
                                        int act, float &gz, float &xh) {
  const float xv = (float)x[i];
  xh = centred(xv, split_mean(st[0])) * (float)st[1];
  gz = (float)gy[i];
  if (act == kActRelu) gz = gated(gz, xv, make_gate(st[0], st[1], w, b));
  if (act == kActSilu) gz = silu_grad(gz, xh * w + b);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) group_sums_kernel(const T *__restrict__ gy, const T *__restrict__ x,
                                                              int64_t P, int C, int per, const void *w,
                                                              const void *b, int wd, int act,
                                                              const double *__restrict__ stats,
                                                              double *__restrict__ sums) {
  __shared__ double s[kThreads / kWave];
  const int64_t n = blockIdx.y, at = n * gridDim.x + blockIdx.x;
  double a = 0.0, q = 0.0;
  for (int64_t k = threadIdx.x; k < P * per; k += kThreads) {
    const int c = (int)(blockIdx.x * per + k % per);
    float gz, xh;
    const float wv = to_f32(w, wd, c, 1.f);
    grad_of(gy, x, (n * P + k / per) * C + c, stats + at * 2, wv, to_f32(b, wd, c, 0.f), act, gz, xh);
    a += (double)(gz * wv);
    q += (double)(gz * wv * xh);
  }
  a = block_sum(a, s);
  q = block_sum(q, s);
  if (threadIdx.x == 0) {
    sums[at * 2] = a;
    sums[at * 2 + 1] = q;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) grad_x_kernel(const T *__restrict__ gy, const T *__restrict__ x,
                                                          int64_t total, int64_t P, int C, int per, const void *w,
                                                          const void *b, int wd, int act,
                                                          const double *__restrict__ stats,
                                                          const double *__restrict__ sums, T *__restrict__ gx) {
  const int G = C / per;
  const double m = (double)(P * per);
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int c = (int)(i % C);
    const int64_t at = i / C / P * G + c / per;
    float gz, xh;
    const float wv = to_f32(w, wd, c, 1.f);
    grad_of(gy, x, i, stats + at * 2, wv, to_f32(b, wd, c, 0.f), act, gz, xh);
    const float m1 = (float)(sums[at * 2] / m), m2 = (float)(sums[at * 2 + 1] / m);
    gx[i] = static_cast<T>((float)stats[at * 2 + 1] * (wv * gz - (m1 + xh * m2)));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) grad_params_kernel(const T *__restrict__ gy, const T *__restrict__ x,
                                                               int64_t N, int64_t P, int C, int per, const void *w,
                                                               const void *b, int wd, int act,
                                                               const double *__restrict__ stats, void *gw,
                                                               void *gb) {
  __shared__ double s[kThreads / kWave];
  const int c = blockIdx.x, G = C / per;
  double a = 0.0, q = 0.0;
  for (int64_t k = threadIdx.x; k < N * P; k += kThreads) {
    float gz, xh;
    grad_of(gy, x, k * C + c, stats + (k / P * G + c / per) * 2, to_f32(w, wd, c, 1.f), to_f32(b, wd, c, 0.f),
            act, gz, xh);
    a += (double)gz;
    q += (double)(gz * xh);
  }
  a = block_sum(a, s);
  q = block_sum(q, s);
  if (threadIdx.x == 0) {
    if (gb != nullptr) from_f32(gb, wd, c, (float)a);
    if (gw != nullptr) from_f32(gw, wd, c, (float)q);
  }
}

int grid_for(int64_t total) {
  const int64_t b = (total + kThreads - 1) / kThreads;
  return (int)(b < 4096 ? b : 4096);
}

template <typename T>
hipError_t forward(const GroupNormArgs &a, void *y, double *stats, hipStream_t stream) {
  const int per = a.channels / a.groups;
  const int64_t total = a.batch * a.pixels * a.channels;
  hipLaunchKernelGGL((stats_kernel<T>), dim3(a.groups, (unsigned)a.batch), dim3(kThreads), 0, stream,
                     static_cast<const T *>(a.x), a.pixels, a.channels, per, a.eps, stats);
  hipLaunchKernelGGL((forward_kernel<T>), dim3(grid_for(total)), dim3(kThreads), 0, stream,
                     static_cast<const T *>(a.x), total, a.pixels, a.channels, per, a.weight, a.bias,
                     a.param_dtype, a.act, stats, static_cast<T *>(y));
  return hipGetLastError();
}

template <typename T>
hipError_t backward(const GroupNormArgs &a, const void *grad_y, const double *stats, void *workspace, void *grad_x,
                    void *grad_w, void *grad_b, hipStream_t stream) {
  const int per = a.channels / a.groups;
  const int64_t total = a.batch * a.pixels * a.channels;
  double *sums = static_cast<double *>(workspace);
  const T *gy = static_cast<const T *>(grad_y), *x = static_cast<const T *>(a.x);
  if (grad_x != nullptr) {
    hipLaunchKernelGGL((group_sums_kernel<T>), dim3(a.groups, (unsigned)a.batch), dim3(kThreads), 0, stream, gy, x,
                       a.pixels, a.channels, per, a.weight, a.bias, a.param_dtype, a.act, stats, sums);
    hipLaunchKernelGGL((grad_x_kernel<T>), dim3(grid_for(total)), dim3(kThreads), 0, stream, gy, x, total,
                       a.pixels, a.channels, per, a.weight, a.bias, a.param_dtype, a.act, stats, sums,
                       static_cast<T *>(grad_x));
  }
  if (grad_w != nullptr || grad_b != nullptr)
    hipLaunchKernelGGL((grad_params_kernel<T>), dim3(a.channels), dim3(kThreads), 0, stream, gy, x, a.batch,
                       a.pixels, a.channels, per, a.weight, a.bias, a.param_dtype, a.act, stats, grad_w, grad_b);
  return hipGetLastError();
}

}  // namespace

int64_t group_norm_workspace_bytes(int dtype, bool backward, int64_t batch, int64_t pixels, int channels,
                                   int groups) {
  return backward ? batch * groups * 16 : 0;
}

hipError_t launch_group_norm_forward(int dtype, const GroupNormArgs &a, void *y, double *stats, void *workspace,
                                     hipStream_t stream) {
  switch (dtype) {
    case 0: return forward<float>(a, y, stats, stream);
    case 1: return forward<f16>(a, y, stats, stream);
    default: return forward<bf16>(a, y, stats, stream);
  }
}

hipError_t launch_group_norm_backward(int dtype, const GroupNormArgs &a, const void *grad_y, const double *stats,
                                      void *workspace, void *grad_x, void *grad_w, void *grad_b,
                                      hipStream_t stream) {
  switch (dtype) {
    case 0: return backward<float>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
    case 1: return backward<f16>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
    default: return backward<bf16>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
  }
}

}  // namespace bevk
