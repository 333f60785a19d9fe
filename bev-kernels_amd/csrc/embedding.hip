// Embedding rows by index with a scale, and the gradient of the table (gfx950).
//
//   out[t] = scale * W[i_t], zeros where i_t is outside [0, rows) (a padded place)
//   gW[v]  = scale * sum over t with i_t = v of g[t], in the order of t, in fp32
#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;

template <typename T, typename I>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T *__restrict__ weight, int64_t rows, int dim,
                                                          const I *__restrict__ index, int64_t total, float scale,
                                                          T *__restrict__ out) {
  for (int64_t k = blockIdx.x * (int64_t)kThreads + threadIdx.x; k < total; k += (int64_t)gridDim.x * kThreads) {
    const int64_t v = (int64_t)index[k / dim];
    out[k] = v >= 0 && v < rows ? static_cast<T>((float)weight[v * dim + k % dim] * scale) : static_cast<T>(0.f);
  }
}

// One wave for a row of the table and 64 of its channels.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads) grad_kernel(const T *__restrict__ g, const I *__restrict__ index,
                                                        int64_t n, int64_t rows, int dim, float scale,
                                                        int64_t padding, T *__restrict__ gw) {
  const int pieces = (dim + 63) / 64, lane = threadIdx.x % kWave;
  for (int64_t u = blockIdx.x * (int64_t)(kThreads / kWave) + threadIdx.x / kWave; u < rows * pieces;
       u += (int64_t)gridDim.x * (kThreads / kWave)) {
    const int64_t v = u / pieces;
    const int c = (int)(u % pieces) * 64 + lane;
    float a = 0.f;
    for (int64_t t = 0; t < n && v != padding; t += 64) {
      uint64_t hit = __ballot(t + lane < n && (int64_t)index[t + lane < n ? t + lane : 0] == v);
      while (hit) {
        const int k = __builtin_ctzll(hit);
        hit &= hit - 1;
        if (c < dim) a += (float)g[(t + k) * dim + c];
      }
    }
    if (c < dim) gw[v * dim + c] = static_cast<T>(a * scale);
  }
}

int grid_for(int64_t threads) {
  const int64_t b = (threads + kThreads - 1) / kThreads;
  return (int)(b < 16384 ? b : 16384);
}

template <typename T, typename I>
hipError_t forward(const EmbeddingArgs &a, const void *weight, void *out, hipStream_t stream) {
  const int64_t total = a.n * a.dim;
  hipLaunchKernelGGL((lookup_kernel<T, I>), dim3(grid_for(total)), dim3(kThreads), 0, stream,
                     static_cast<const T *>(weight), a.rows, a.dim, static_cast<const I *>(a.index), total, a.scale,
                     static_cast<T *>(out));
  return hipGetLastError();
}

template <typename T, typename I>
hipError_t backward(const EmbeddingArgs &a, const void *grad_out, int64_t padding, void *grad_w,
                    hipStream_t stream) {
  hipLaunchKernelGGL((grad_kernel<T, I>), dim3(grid_for(a.rows * ((a.dim + 63) / 64) * kWave)), dim3(kThreads), 0,
                     stream, static_cast<const T *>(grad_out), static_cast<const I *>(a.index), a.n, a.rows, a.dim,
                     a.scale, padding, static_cast<T *>(grad_w));
  return hipGetLastError();
}

}  // namespace

int64_t embedding_backward_workspace_bytes(int dtype, int64_t n, int64_t rows, int dim) { return 0; }

hipError_t launch_embedding_forward(int dtype, const EmbeddingArgs &a, const void *weight, void *out,
                                    hipStream_t stream) {
  switch (dtype * 2 + (a.index64 ? 1 : 0)) {
    case 0: return forward<float, int32_t>(a, weight, out, stream);
    case 1: return forward<float, int64_t>(a, weight, out, stream);
    case 2: return forward<f16, int32_t>(a, weight, out, stream);
    case 3: return forward<f16, int64_t>(a, weight, out, stream);
    case 4: return forward<bf16, int32_t>(a, weight, out, stream);
    default: return forward<bf16, int64_t>(a, weight, out, stream);
  }
}

hipError_t launch_embedding_backward(int dtype, const EmbeddingArgs &a, const void *grad_out, int64_t padding,
                                     void *workspace, void *grad_w, hipStream_t stream) {
  switch (dtype * 2 + (a.index64 ? 1 : 0)) {
    case 0: return backward<float, int32_t>(a, grad_out, padding, grad_w, stream);
    case 1: return backward<float, int64_t>(a, grad_out, padding, grad_w, stream);
    case 2: return backward<f16, int32_t>(a, grad_out, padding, grad_w, stream);
    case 3: return backward<f16, int64_t>(a, grad_out, padding, grad_w, stream);
    case 4: return backward<bf16, int32_t>(a, grad_out, padding, grad_w, stream);
    default: return backward<bf16, int64_t>(a, grad_out, padding, grad_w, stream);
  }
}

}  // namespace bevk
