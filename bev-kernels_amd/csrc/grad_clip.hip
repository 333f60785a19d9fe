// The norm of many gradients together, and their clipping to a largest norm (gfx950).
//
//   norm = sqrt(sum g^2 over all tensors), by = min(1, max_norm / (norm + 1e-6)), out = by * g
//
// The squares are summed in fp64: no gradient that fp32 holds overflows or vanishes in them.
//
// The tensors' addresses go in as kernel arguments, up to kTensors of them a launch: nothing is
// copied to the device first, and a captured graph holds them itself. A tensor is cut into chunks
// of `per` values, a workgroup each; each leaves the sum of its squares in the workspace, and each
// workgroup of the second pass adds them all up again in one order, which saves a launch between.
#include <algorithm>

#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 96;   // 25 bytes each: 2.8 KB of the 4 KB of arguments
constexpr int kChunks = 1024;  // about that many for a large model

struct Table {
  const void *in[kTensors];
  void *out[kTensors];
  int64_t n[kTensors];
  int first[kTensors + 1];  // first chunk of each tensor in this launch
  unsigned char in_type[kTensors], out_type[kTensors];
  int count;
};

__device__ __forceinline__ double block_sum(double v, double *s) {
  __syncthreads();
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_down(v, d, kWave);
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  double t = s[0];
  for (int k = 1; k < kThreads / kWave; ++k) t += s[k];
  return t;
}

__device__ __forceinline__ int find_tensor(const Table &t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double squares(const T *p, int64_t n) {
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) {
    const double v = (double)(float)p[i];
    a += v * v;
  }
  return a;
}

__global__ void __launch_bounds__(kThreads) squares_kernel(const Table t, int64_t per, double *__restrict__ part) {
  __shared__ double s[kThreads / kWave];
  const int k = find_tensor(t, blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * per, n = min(per, t.n[k] - at);
  double a;
  switch (t.in_type[k]) {
    case 0: a = squares(static_cast<const float *>(t.in[k]) + at, n); break;
    case 1: a = squares(static_cast<const f16 *>(t.in[k]) + at, n); break;
    default: a = squares(static_cast<const bf16 *>(t.in[k]) + at, n); break;
  }
  a = block_sum(a, s);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

__device__ __forceinline__ double norm_of(const double *part, int parts, double *s) {
  double a = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) a += part[i];
  return sqrt(block_sum(a, s));
}

template <typename T, typename O>
__device__ __forceinline__ void scale(const T *p, O *out, int64_t n, float by) {
  for (int64_t i = threadIdx.x; i < n; i += kThreads) out[i] = static_cast<O>((float)p[i] * by);
}
template <typename T>
__device__ __forceinline__ void scale_to(const T *p, void *out, int type, int64_t at, int64_t n, float by) {
  switch (type) {
    case 0: scale(p + at, static_cast<float *>(out) + at, n, by); break;
    case 1: scale(p + at, static_cast<f16 *>(out) + at, n, by); break;
    default: scale(p + at, static_cast<bf16 *>(out) + at, n, by); break;
  }
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const Table t, int64_t per, const double *__restrict__ part,
                                                         int parts, double max_norm, float *__restrict__ norm_out) {
  __shared__ double s[kThreads / kWave];
  const double norm = norm_of(part, parts, s);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double q = max_norm / (norm + 1e-6);
  const float by = q >= 1.0 ? 1.f : (float)q;  // NaN stays
  const int k = find_tensor(t, blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * per, n = min(per, t.n[k] - at);
  switch (t.in_type[k]) {
    case 0: scale_to(static_cast<const float *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
    case 1: scale_to(static_cast<const f16 *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
    default: scale_to(static_cast<const bf16 *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
  }
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *__restrict__ part, int parts,
                                                        float *__restrict__ norm_out) {
  __shared__ double s[kThreads / kWave];
  const double norm = norm_of(part, parts, s);
  if (threadIdx.x == 0) *norm_out = (float)norm;
}

int64_t chunk_of(const GradList &g) {
  int64_t total = 0;
  for (int k = 0; k < g.count; ++k) total += g.n[k];
  return std::max<int64_t>(8192, (total / kChunks + 2047) / 2048 * 2048);
}

int64_t chunks_of(const GradList &g, int64_t per) {
  int64_t c = 0;
  for (int k = 0; k < g.count; ++k) c += (g.n[k] + per - 1) / per;
  return c;
}

// launch(table, chunks, chunks before it) for up to kTensors tensors with values at a time.
template <typename F>
hipError_t for_tables(const GradList &g, int64_t per, F launch) {
  int k = 0, before = 0;
  while (k < g.count) {
    Table t;
    t.count = 0;
    t.first[0] = 0;
    for (; k < g.count && t.count < kTensors; ++k) {
      if (g.n[k] == 0) continue;
      const int c = t.count++;
      t.in[c] = g.in[k];
      t.out[c] = g.out ? g.out[k] : nullptr;
      t.n[c] = g.n[k];
      t.in_type[c] = (unsigned char)g.in_type[k];
      t.out_type[c] = g.out ? (unsigned char)g.out_type[k] : 0;
      t.first[c + 1] = t.first[c] + (int)((g.n[k] + per - 1) / per);
    }
    if (t.count == 0) break;
    launch(t, t.first[t.count], before);
    before += t.first[t.count];
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace

int64_t clip_gradients_workspace_bytes(const GradList &g) { return chunks_of(g, chunk_of(g)) * 8; }

hipError_t launch_clip_gradients(const GradList &g, double max_norm, void *workspace, float *norm,
                                 hipStream_t stream) {
  const int64_t per = chunk_of(g);
  const int parts = (int)chunks_of(g, per);
  double *part = static_cast<double *>(workspace);
  hipError_t e = for_tables(g, per, [&](const Table &t, int chunks, int before) {
    hipLaunchKernelGGL(squares_kernel, dim3(chunks), dim3(kThreads), 0, stream, t, per, part + before);
  });
  if (e != hipSuccess) return e;
  if (g.out == nullptr || parts == 0) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, stream, part, parts, norm);
    return hipGetLastError();
  }
  return for_tables(g, per, [&](const Table &t, int chunks, int before) {
    hipLaunchKernelGGL(scale_kernel, dim3(chunks), dim3(kThreads), 0, stream, t, per, part, parts, max_norm,
                       before == 0 ? norm : nullptr);
  });
}

}  // namespace bevk
