// Projections with everything behind them (gfx950): y = act(x W^T + bias) + residual, x [rows][K],
// W [N][K], and the gradients.
//
//   z = x W^T + bias,  y = act(z) + residual
//   gz = gy act'(z),  gx = gz W,  gW = gz^T x,  gbias = sum gz,  gresidual = gy
//
// Products of 16-bit types on the matrix cores with fp32 sums; bias, activation and residual in fp32 on the
// sums in registers, one rounding at the end. gz is rounded to the input's type, which is what the
// matrix cores read.
#include <algorithm>
#include <type_traits>

#include "bevk_launch.h"

namespace bevk {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

__device__ __forceinline__ floatx4 mfma16(int4v a, int4v b, floatx4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mfma16(int4v a, int4v b, floatx4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------------------

// The normal distribution below z, and its density. 16-bit types: erfc by Abramowitz and Stegun's
// 7.1.26, off by 1.5e-7 at the most (a rounding of the type is 4.9e-4 of the value), 14 instructions
// where erff takes 40 of a kernel that is bound by memory.
template <typename T> __device__ __forceinline__ void normal(float z, float &cdf, float &pdf) {
  const float e = __expf(-0.5f * z * z);
  pdf = 0.3989422804f * e;
  if constexpr (sizeof(T) == 4) {
    cdf = 0.5f * erfcf(-0.7071067812f * z);
  } else {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.7071067812f, __builtin_fabsf(z), 1.f));
    float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    q = __builtin_fmaf(t, q, 1.421413741f);
    q = __builtin_fmaf(t, q, -0.284496736f);
    q = __builtin_fmaf(t, q, 0.254829592f);
    const float tail = 0.5f * e * (t * q);
    cdf = z > 0.f ? 1.f - tail : tail;
  }
}
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
  if (act == kActRelu) return z > 0.f || z != z ? z : 0.f;
  if (act == kActSilu) return z / (1.f + __expf(-z));
  if (act == kActGelu) {
    float cdf, pdf;
    normal<T>(z, cdf, pdf);
    return z * cdf;
  }
  return z;
}
template <typename T> __device__ __forceinline__ float slope(float z, int act) {
  if (act == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kActSilu) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * __builtin_fmaf(z, 1.f - s, 1.f);
  }
  float cdf, pdf;
  normal<T>(z, cdf, pdf);
  return __builtin_fmaf(z, pdf, cdf);
}

// What is done with a sum. Tensors [M][N].
struct Epilogue {
  const void *bias, *residual;
  void *y, *z;  // z: or null
  bool bias_wide;
  int act;
  int N;
};

template <typename T> __device__ __forceinline__ float bias_at(const Epilogue &e, int n) {
  if (e.bias == nullptr) return 0.f;
  return e.bias_wide ? static_cast<const float *>(e.bias)[n] : (float)static_cast<const T *>(e.bias)[n];
}
template <typename T> __device__ __forceinline__ void finish(const Epilogue &e, int64_t m, int n, float v) {
  const int64_t at = m * e.N + n;
  v += bias_at<T>(e, n);
  if (e.z != nullptr) static_cast<T *>(e.z)[at] = static_cast<T>(v);
  v = activate<T>(v, e.act);
  if (e.residual != nullptr) v += (float)static_cast<const T *>(e.residual)[at];
  static_cast<T *>(e.y)[at] = static_cast<T>(v);
}

// ---------------------------------------------------------------------------------------
// Any sizes, strides and alignments: out[m][n] = sum_k a(m, k) b(n, k). A workgroup of four waves takes
// 64 x 64 values, 32 terms at a time through LDS (rows padded by 16 bytes: no two of 8 neighbouring
// rows' reads meet in a bank), elements loaded one by one. Few tiles of a long sum: the sum in parts,
// added up in order by finish_kernel.
// ---------------------------------------------------------------------------------------
template <typename T> struct Product {
  const T *a, *b;
  int64_t a_m, a_k, b_n, b_k;
  int64_t M, K, per;  // per: terms of a part, a multiple of 32
  float *part;        // [parts][M][N], or null for one part
  Epilogue e;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) any_kernel(const Product<T> p, int64_t first) {
  constexpr int P = 32 + 16 / (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) T sa[64][P], sb[64][P];
  const int N = p.e.N;
  const int64_t tn = (N + 63) / 64, tm = (p.M + 63) / 64, tile = first + blockIdx.x;
  const int64_t m0 = tile % tm * 64;
  const int n0 = (int)(tile / tm % tn) * 64, z = (int)(tile / tm / tn);
  const int64_t k0 = z * p.per, k1 = min(p.K, k0 + p.per);
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  // a thread's 8 elements of each tile: along k where that is dense, else of one row after another
  auto stage = [&](const T *src, int64_t by_row, int64_t by_k, int64_t row0, int64_t rows, int64_t k,
                   T (&s)[64][P]) __attribute__((always_inline)) {
    const bool along = by_k == 1;
    const int r = along ? tid / 4 : tid % 64, c = (along ? tid % 4 : tid / 64) * 8;
    const T *q = src + (row0 + r) * by_row;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t kk = k + c + e;
      s[r][c + e] = row0 + r < rows && kk < k1 ? q[kk * by_k] : static_cast<T>(0.f);
    }
  };
  floatx4 acc[2][2] = {};
  const int ra = wave / 2 * 32 + lane % 16, rb = wave % 2 * 32 + lane % 16, c = lane / 16 * 8;
  for (int64_t k = k0; k < k1; k += 32) {
    stage(p.a, p.a_m, p.a_k, m0, p.M, k, sa);
    stage(p.b, p.b_n, p.b_k, n0, N, k, sb);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const T *qa = &sa[ra + i * 16][c], *qb = &sb[rb + j * 16][c];
        if constexpr (sizeof(T) == 2) {
          acc[i][j] = mfma16(*reinterpret_cast<const int4v *>(qb), *reinterpret_cast<const int4v *>(qa), acc[i][j], T());
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(qb[e], qa[e], acc[i][j], 0, 0, 0);
        }
      }
    __syncthreads();
  }
  // a lane holds one m and four neighbouring n
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t m = m0 + ra + i * 16;
        const int n = n0 + wave % 2 * 32 + j * 16 + lane / 16 * 4 + e;
        if (m >= p.M || n >= N) continue;
        if (p.part != nullptr) p.part[(z * p.M + m) * N + n] = acc[i][j][e];
        else finish<T>(p.e, m, n, acc[i][j][e]);
      }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) finish_kernel(const Epilogue e, const float *__restrict__ part, int parts,
                                                          int64_t total, int64_t first) {
  const int64_t i = (first + blockIdx.x) * kThreads + threadIdx.x;
  if (i >= total) return;
  float v = 0.f;
#pragma unroll 4
  for (int q = 0; q < parts; ++q) v += part[q * total + i];
  finish<T>(e, i / e.N, (int)(i % e.N), v);
}

struct AnyPlan {
  int parts;
  int64_t per;
};
AnyPlan any_plan(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((M + 63) / 64) * ((N + 63) / 64), want = 4 * std::max(1, device_cus());
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({want / tiles, K / 256, 64}));
  AnyPlan pl;
  pl.per = ((K + parts - 1) / parts + 31) / 32 * 32;
  pl.parts = (int)((K + pl.per - 1) / pl.per);
  return pl;
}
int64_t any_bytes(int64_t M, int64_t N, int64_t K) {
  const AnyPlan pl = any_plan(M, N, K);
  return pl.parts > 1 ? pl.parts * M * N * 4 : 0;
}
template <typename T>
hipError_t launch_any(const T *a, int64_t a_m, int64_t a_k, const T *b, int64_t b_n, int64_t b_k, int64_t M, int64_t K,
                      const Epilogue &e, void *workspace, hipStream_t stream) {
  const AnyPlan pl = any_plan(M, e.N, K);
  Product<T> p{a, b, a_m, a_k, b_n, b_k, M, K, pl.per, pl.parts > 1 ? static_cast<float *>(workspace) : nullptr, e};
  const int64_t tiles = ((M + 63) / 64) * (((int64_t)e.N + 63) / 64) * pl.parts;
  hipError_t err = launch_in_parts(tiles, kThreads, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((any_kernel<T>), dim3(n), dim3(kThreads), 0, stream, p, first);
  });
  if (err != hipSuccess || pl.parts == 1) return err;
  const int64_t total = M * e.N;
  return launch_in_parts((total + kThreads - 1) / kThreads, kThreads, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((finish_kernel<T>), dim3(n), dim3(kThreads), 0, stream, e, p.part, pl.parts, total, first);
  });
}

// ---------------------------------------------------------------------------------------
// gz = gy act'(z) and its column sums: a workgroup takes a range of rows of up to 256 vectors of
// columns; each thread keeps its columns' sums, the workgroup adds up its rows side by side and
// total_kernel the workgroups, in order.
// ---------------------------------------------------------------------------------------
constexpr int kSumBlocks = 512;

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) grad_z_kernel(const T *__restrict__ gy, const T *__restrict__ z,
                                                          T *__restrict__ gz, int act, int64_t rows, int n, int per,
                                                          float *__restrict__ part) {
  __shared__ float s[kThreads][V + 1];
  const int lanes = kThreads / per, col = (blockIdx.y * per + threadIdx.x % per) * V, row = threadIdx.x / per;
  const int64_t r0 = rows * blockIdx.x / gridDim.x, r1 = rows * (blockIdx.x + 1) / gridDim.x;
  float a[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = 0.f;
  if (row < lanes && col < n) {
#pragma unroll 2
    for (int64_t r = r0 + row; r < r1; r += lanes) {
      const int64_t at = r * n + col;
      Vec<T, V> g = load_vec<T, V>(gy + at);
      if (act != kActNone) {
        const Vec<T, V> x = load_vec<T, V>(z + at);
#pragma unroll
        for (int e = 0; e < V; ++e) g.v[e] = static_cast<T>((float)g.v[e] * slope<T>((float)x.v[e], act));
        store_vec<T, V>(gz + at, g);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] += (float)g.v[e];
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) s[threadIdx.x][e] = a[e];
  __syncthreads();
  if ((int)threadIdx.x >= per || col >= n) return;
  for (int l = 1; l < lanes; ++l)
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] += s[threadIdx.x + l * per][e];
#pragma unroll
  for (int e = 0; e < V; ++e) part[(int64_t)blockIdx.x * n + col + e] = a[e];
}

// 16 columns: 64 threads add up every 64th part each, then in order.
template <typename O>
__global__ void __launch_bounds__(1024) total_kernel(const float *__restrict__ part, int parts, int n, O *__restrict__ out) {
  __shared__ float s[64][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
  float v = 0.f;
  if (c < n)
#pragma unroll 8
    for (int q = k; q < parts; q += 64) v += part[(int64_t)q * n + c];
  s[k][threadIdx.x % 16] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (k < half) s[k][threadIdx.x % 16] += s[k + half][threadIdx.x % 16];
    __syncthreads();
  }
  if (k == 0 && c < n) out[c] = static_cast<O>(s[0][threadIdx.x]);
}

int sum_blocks(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(kSumBlocks, rows / 16)); }

template <typename T, int V>
hipError_t launch_grad_z_v(const T *gy, const T *z, T *gz, int act, int64_t rows, int n, float *part, hipStream_t stream) {
  const int vecs = (n + V - 1) / V, per = std::min(vecs, kThreads);
  hipLaunchKernelGGL((grad_z_kernel<T, V>), dim3(sum_blocks(rows), (vecs + per - 1) / per), dim3(kThreads), 0, stream,
                     gy, z, gz, act, rows, n, per, part);
  return hipGetLastError();
}
bool on_16(std::initializer_list<const void *> all) {
  for (const void *p : all)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}
template <typename T>
hipError_t launch_grad_z(const T *gy, const T *z, T *gz, int act, int64_t rows, int n, float *part, void *grad_bias,
                         bool bias_wide, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  hipError_t e = n % V == 0 && on_16({gy, z, gz}) ? launch_grad_z_v<T, V>(gy, z, gz, act, rows, n, part, stream)
                                                  : launch_grad_z_v<T, 1>(gy, z, gz, act, rows, n, part, stream);
  if (e != hipSuccess || grad_bias == nullptr) return e;
  const dim3 grid((n + 15) / 16);
  if (bias_wide) hipLaunchKernelGGL((total_kernel<float>), grid, dim3(1024), 0, stream, part, sum_blocks(rows), n, static_cast<float *>(grad_bias));
  else hipLaunchKernelGGL((total_kernel<T>), grid, dim3(1024), 0, stream, part, sum_blocks(rows), n, static_cast<T *>(grad_bias));
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// What a call runs
// ---------------------------------------------------------------------------------------
int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

template <typename T>
hipError_t forward(const LinearArgs &a, const void *residual, void *y, void *z, void *workspace, hipStream_t stream) {
  const Epilogue e{a.bias, residual, y, z, a.bias_wide, a.act, a.N};
  return launch_any(static_cast<const T *>(a.x), a.K, 1, static_cast<const T *>(a.weight), a.K, 1, a.rows, a.K, e,
                    workspace, stream);
}

// Workspace of the backward: gz, the bias' parts, then what the products take.
struct BackWs {
  int64_t part, product, total;
};
BackWs back_ws(int dtype, const LinearArgs &a) {
  const int64_t size = dtype == 0 ? 4 : 2;
  BackWs w;
  w.part = a.act != kActNone ? up(a.rows * a.N * size) : 0;
  w.product = w.part + up((int64_t)kSumBlocks * a.N * 4);
  w.total = w.product + up(std::max(any_bytes(a.rows, a.K, a.N), any_bytes(a.N, a.K, a.rows)));
  return w;
}

template <typename T>
hipError_t backward(int dtype, const LinearArgs &a, const void *grad_y, const void *z, void *workspace, void *grad_x,
                    void *grad_w, void *grad_b, hipStream_t stream) {
  const BackWs ws = back_ws(dtype, a);
  char *base = static_cast<char *>(workspace);
  const T *gy = static_cast<const T *>(grad_y), *gz = gy;
  if (a.act != kActNone) gz = reinterpret_cast<T *>(base);
  if (a.act != kActNone || grad_b != nullptr)
    if (hipError_t e = launch_grad_z<T>(gy, static_cast<const T *>(z), const_cast<T *>(gz), a.act, a.rows, a.N,
                                        grad_b != nullptr ? reinterpret_cast<float *>(base + ws.part) : nullptr, grad_b,
                                        a.bias_wide, stream))
      return e;
  if (grad_x != nullptr) {
    const Epilogue e{nullptr, nullptr, grad_x, nullptr, false, kActNone, a.K};
    if (hipError_t err = launch_any<T>(gz, a.N, 1, static_cast<const T *>(a.weight), 1, a.K, a.rows, a.N, e,
                                       base + ws.product, stream))
      return err;
  }
  if (grad_w != nullptr) {
    const Epilogue e{nullptr, nullptr, grad_w, nullptr, false, kActNone, a.K};
    return launch_any<T>(gz, 1, a.N, static_cast<const T *>(a.x), 1, a.K, a.N, a.rows, e, base + ws.product, stream);
  }
  return hipSuccess;
}

}  // namespace

int64_t linear_forward_workspace_bytes(int dtype, const LinearArgs &a) { return any_bytes(a.rows, a.N, a.K); }

hipError_t launch_linear_forward(int dtype, const LinearArgs &a, const void *residual, void *y, void *z, void *workspace,
                                 hipStream_t stream) {
  switch (dtype) {
    case 0: return forward<float>(a, residual, y, z, workspace, stream);
    case 1: return forward<f16>(a, residual, y, z, workspace, stream);
    default: return forward<bf16>(a, residual, y, z, workspace, stream);
  }
}

int64_t linear_backward_workspace_bytes(int dtype, const LinearArgs &a) { return back_ws(dtype, a).total; }

hipError_t launch_linear_backward(int dtype, const LinearArgs &a, const void *grad_y, const void *z, void *workspace,
                                  void *grad_x, void *grad_w, void *grad_b, hipStream_t stream) {
  switch (dtype) {
    case 0: return backward<float>(dtype, a, grad_y, z, workspace, grad_x, grad_w, grad_b, stream);
    case 1: return backward<f16>(dtype, a, grad_y, z, workspace, grad_x, grad_w, grad_b, stream);
    default: return backward<bf16>(dtype, a, grad_y, z, workspace, grad_x, grad_w, grad_b, stream);
  }
}

}  // namespace bevk
