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
// Both passes are bound by memory (squares at two fp64 instructions a value stay behind the loads);
// the second takes the chunks in the opposite order, since what the first read last may still be
// in the last-level cache of 256 MB: the same tables from the last on, and each from its last chunk
// to its first (97 bf16 tensors of 30 MB, second pass: 21.4 us in the first pass' order of
// tensors, 19.8 us so; 109 M fp32 values: 141 and 139 us). Its own loads and stores leave that cache
// alone where inputs and outputs together do not fit (109 M fp32 values: first pass 115 -> 78 us
// without the last call's outputs to write back, second 152 -> 139 us; where they fit, the outputs
// stay there for the optimizer).
#include <algorithm>

#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 128;  // 30 bytes each: 3.8 KB of the 4 KB of arguments
constexpr int kChunks = 2048;  // about that many for a large model
constexpr int kUnroll = 4;     // vectors of a thread in flight
constexpr int kXcds = 8;

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

// The values [0, n) at p as a few single ones up to a 16-byte boundary, vectors, and the rest.
template <typename T> struct Span {
  static constexpr int V = 16 / sizeof(T);
  int64_t head, vecs, tail;  // tail: first value of the rest
  __device__ __forceinline__ Span(const T *p, int64_t n) {
    const int64_t off = reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T);
    head = min((V - off) % V, n);
    vecs = (n - head) / V;
    tail = head + vecs * V;
  }
};

template <typename T>
__device__ __forceinline__ double squares(const T *p, int64_t n) {
  const Span<T> s(p, n);
  double a = 0.0;
  auto add = [&](T x) __attribute__((always_inline)) {
    const double v = (double)(float)x;
    a += v * v;
  };
  if ((int64_t)threadIdx.x < s.head) add(p[threadIdx.x]);
  if (s.tail + threadIdx.x < n) add(p[s.tail + threadIdx.x]);
  const T *q = p + s.head;
  int64_t i = threadIdx.x;
  for (; i + (kUnroll - 1) * kThreads < s.vecs; i += kUnroll * kThreads) {
    Vec<T, Span<T>::V> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = load_vec<T, Span<T>::V>(q + (i + u * kThreads) * Span<T>::V);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < Span<T>::V; ++e) add(v[u].v[e]);
  }
  for (; i < s.vecs; i += kThreads) {
    const Vec<T, Span<T>::V> v = load_vec<T, Span<T>::V>(q + i * Span<T>::V);
#pragma unroll
    for (int e = 0; e < Span<T>::V; ++e) add(v.v[e]);
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

// N values of O in memory instructions of up to 16 bytes.
template <typename O, int N, bool STREAM>
__device__ __forceinline__ void store_pieces(O *p, const Vec<O, N> &x) {
  constexpr int W = sizeof(O) * N > 16 ? 16 / sizeof(O) : N;
#pragma unroll
  for (int k = 0; k < N; k += W) {
    Vec<O, W> y;
#pragma unroll
    for (int e = 0; e < W; ++e) y.v[e] = x.v[k + e];
    if constexpr (STREAM) store_vec_nt<O, W>(p + k, y); else store_vec<O, W>(p + k, y);
  }
}

template <bool STREAM, typename T, typename O>
__device__ __forceinline__ void scale(const T *p, O *out, int64_t n, float by) {
  constexpr int V = Span<T>::V;
  constexpr uintptr_t align = sizeof(O) * V > 16 ? 16 : sizeof(O) * V;
  const Span<T> s(p, n);
  auto one = [&](int64_t i) __attribute__((always_inline)) { out[i] = static_cast<O>((float)p[i] * by); };
  if (reinterpret_cast<uintptr_t>(out + s.head) % align != 0) {  // out starts elsewhere within a vector
    for (int64_t i = threadIdx.x; i < n; i += kThreads) one(i);
    return;
  }
  if ((int64_t)threadIdx.x < s.head) one(threadIdx.x);
  if (s.tail + threadIdx.x < n) one(s.tail + threadIdx.x);
  const T *q = p + s.head;
  O *o = out + s.head;
  for (int64_t i = threadIdx.x; i < s.vecs; i += kUnroll * kThreads) {
    Vec<T, V> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < s.vecs)
        v[u] = STREAM ? load_vec_nt<T, V>(q + (i + u * kThreads) * V) : load_vec<T, V>(q + (i + u * kThreads) * V);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i + u * kThreads < s.vecs) {
        Vec<O, V> x;
#pragma unroll
        for (int e = 0; e < V; ++e) x.v[e] = static_cast<O>((float)v[u].v[e] * by);
        store_pieces<O, V, STREAM>(o + (i + u * kThreads) * V, x);
      }
  }
}
template <bool STREAM, typename T>
__device__ __forceinline__ void scale_to(const T *p, void *out, int type, int64_t at, int64_t n, float by) {
  switch (type) {
    case 0: scale<STREAM>(p + at, static_cast<float *>(out) + at, n, by); break;
    case 1: scale<STREAM>(p + at, static_cast<f16 *>(out) + at, n, by); break;
    default: scale<STREAM>(p + at, static_cast<bf16 *>(out) + at, n, by); break;
  }
}

template <bool STREAM>
__global__ void __launch_bounds__(kThreads) scale_kernel(const Table t, int64_t per, const double *__restrict__ part,
                                                         int parts, double max_norm, float *__restrict__ norm_out) {
  __shared__ double s[kThreads / kWave];
  const double norm = norm_of(part, parts, s);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double q = max_norm / (norm + 1e-6);
  const float by = q >= 1.0 ? 1.f : (float)q;  // NaN stays
  const int chunks = t.first[t.count], up = (chunks + kXcds - 1) / kXcds * kXcds;
  const int chunk = up - kXcds - (int)blockIdx.x / kXcds * kXcds + (int)blockIdx.x % kXcds;  // on its XCD again
  if (chunk >= chunks) return;
  const int k = find_tensor(t, chunk);
  if (by == 1.f && t.in[k] == t.out[k]) return;  // its own values again
  const int64_t at = (int64_t)(chunk - t.first[k]) * per, n = min(per, t.n[k] - at);
  switch (t.in_type[k]) {
    case 0: scale_to<STREAM>(static_cast<const float *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
    case 1: scale_to<STREAM>(static_cast<const f16 *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
    default: scale_to<STREAM>(static_cast<const bf16 *>(t.in[k]), t.out[k], t.out_type[k], at, n, by); break;
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

// launch(table, chunks, chunks so far) for kTensors tensors with values at a time, and the rest: the
// same tables, in the order of the tensors, from the first table on or from the last.
template <typename F>
hipError_t for_tables(const GradList &g, int64_t per, bool back, F launch) {
  int left = 0;  // tensors with values
  for (int k = 0; k < g.count; ++k) left += g.n[k] > 0;
  int begin = 0, end = g.count, before = 0;
  while (left > 0) {
    const int size = back ? (left - 1) % kTensors + 1 : std::min(left, kTensors);
    if (back) {
      begin = end;
      for (int k = 0; k < size; k += g.n[begin] > 0) --begin;
    }
    Table t;
    t.count = 0;
    t.first[0] = 0;
    int i = begin;
    for (; t.count < size; ++i) {
      if (g.n[i] == 0) continue;
      const int c = t.count++;
      t.in[c] = g.in[i];
      t.out[c] = g.out ? g.out[i] : nullptr;
      t.n[c] = g.n[i];
      t.in_type[c] = (unsigned char)g.in_type[i];
      t.out_type[c] = g.out ? (unsigned char)g.out_type[i] : 0;
      t.first[c + 1] = t.first[c] + (int)((g.n[i] + per - 1) / per);
    }
    (back ? end : begin) = back ? begin : i;
    left -= size;
    launch(t, t.first[t.count], before);
    before += t.first[t.count];
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

constexpr int64_t kCached = 192 << 20;  // bytes of inputs and outputs

int64_t bytes_of(const GradList &g) {
  int64_t b = 0;
  for (int k = 0; k < g.count; ++k) b += g.n[k] * ((g.in_type[k] == 0 ? 4 : 2) + (g.out_type[k] == 0 ? 4 : 2));
  return b;
}

}  // namespace

int64_t clip_gradients_workspace_bytes(const GradList &g) { return chunks_of(g, chunk_of(g)) * 8; }

hipError_t launch_clip_gradients(const GradList &g, double max_norm, void *workspace, float *norm,
                                 hipStream_t stream) {
  const int64_t per = chunk_of(g);
  const int parts = (int)chunks_of(g, per);
  double *part = static_cast<double *>(workspace);
  hipError_t e = for_tables(g, per, false, [&](const Table &t, int chunks, int before) {
    hipLaunchKernelGGL(squares_kernel, dim3(chunks), dim3(kThreads), 0, stream, t, per, part + before);
  });
  if (e != hipSuccess) return e;
  if (g.out == nullptr || parts == 0) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, stream, part, parts, norm);
    return hipGetLastError();
  }
  const bool stream_by = bytes_of(g) > kCached;
  return for_tables(g, per, true, [&](const Table &t, int chunks, int before) {
    const auto kernel = stream_by ? scale_kernel<true> : scale_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((chunks + kXcds - 1) / kXcds * kXcds), dim3(kThreads), 0, stream, t, per, part, parts, max_norm,
                       before == 0 ? norm : nullptr);
  });
}

}  // namespace bevk
