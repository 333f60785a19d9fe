// An AdamW step over many tensors at once (gfx950), moments in 32 or in 8 bits.
//
//   t = t + 1,  g = min(1, max_norm / (norm + 1e-6)) g           (the factor where a norm is given)
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = (1 - lr decay) p - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps),  copy = p
//
// All in fp32 from values of whatever type, each result rounded once; t and what follows from it
// in fp64 by one thread of a launch before (step_kernel), so that t may advance in a replayed graph.
//
// 8 bits: kBlock values share a scale, the biased exponent of their largest (rounded up to three
// mantissa bits, so that no rounding passes it). A first moment is a sign, 4 exponent and 3 mantissa
// bits, a second moment 5 and 3 (it has no sign; its range of 2^31 is the square of the first's), the
// largest exponent meaning the scale's; code 0 is zero. A second moment that is not zero never
// becomes it (a parameter's step would have eps alone below it): below the range it is held at the
// smallest code, which makes a step smaller, never larger. A first moment below it is lost.
// Rounding to three mantissa bits is random: nearest would leave a second moment where it is until
// g^2 passes 60 times it (b2 = 0.999 changes it by less than half a step of 2^-4 otherwise), while
// random rounding is right on average and, as a step there is taken seldom, leaves a spread of a
// quarter of v. 20 random bits are added below the kept ones: 16 from a mixing of place, step and
// seed, and a half (fewer would bias 1,000 steps' sum: 2^-16 of a step each is 0.1% of v). Same
// seed, step and inputs: same results.
//
// Bound by memory: 15 M values with 32-bit moments 420 MB in 89 us from memory (4.7 TB/s, a copy's rate at that
// size 5.2), 69 us where the state is still in the last-level cache; 109 M with 8-bit moments, bf16 gradients and
// copies 1.75 GB in 390 us (4.5 TB/s); the codes' values as bf16 330 MB in 65 us. Non-temporal loads and stores:
// 92 for 96 us a call from memory, 89 for 69 from the cache, not kept.
#include <algorithm>

#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 64;   // 47 bytes each: 3.0 KB of the 4 KB of arguments
constexpr int kBlock = kAdamwBlock;
constexpr int kChunks = 4096;  // about that many for a large model

struct Table {
  void *p[kTensors], *copy[kTensors];
  const void *g[kTensors];
  int64_t n[kTensors], at[kTensors];  // values, and their place in the moments
  int first[kTensors + 1];            // first chunk of each tensor in this launch
  unsigned char p_type[kTensors], g_type[kTensors], c_type[kTensors];
  int count;
};

// What the step's launches share: written by step_kernel into the workspace.
struct Factors {
  float by, decay, size, root, b1, rest1, b2, rest2, eps;
  uint32_t key;
};

struct Moments {
  void *m, *v;
  unsigned char *m_scale, *v_scale;
};

// A bijection of 32 bits: odd multipliers (2^32 over the golden ratio, 2^31 times the root of 2)
// carry low bits up, the shifts carry high bits down.
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x *= 0x9E3779B1u;
  x = (x ^ (x >> 15)) * 0xB504F333u;
  x = (x ^ (x >> 13)) * 0x9E3779B1u;
  return x ^ (x >> 16);
}

struct StepArgs {
  int64_t *step;
  uint64_t seed;
  double lr, beta1, beta2, eps, decay, max_norm;
  const float *lr_at, *norm;
};

__global__ void __launch_bounds__(64) step_kernel(const StepArgs a, Factors *__restrict__ f) {
  if (threadIdx.x != 0) return;
  const int64_t t = *a.step + 1;
  *a.step = t;
  const double lr = a.lr_at != nullptr ? (double)*a.lr_at : a.lr;
  double by = 1.0;
  if (a.norm != nullptr) {
    const double q = a.max_norm / ((double)*a.norm + 1e-6);
    by = q >= 1.0 ? 1.0 : q;  // NaN stays
  }
  f->by = (float)by;
  f->decay = (float)(1.0 - lr * a.decay);
  f->size = (float)(lr / (1.0 - pow(a.beta1, (double)t)));
  f->root = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
  f->b1 = (float)a.beta1;
  f->rest1 = (float)(1.0 - a.beta1);
  f->b2 = (float)a.beta2;
  f->rest2 = (float)(1.0 - a.beta2);
  f->eps = (float)a.eps;
  f->key = mix(mix(mix(mix((uint32_t)a.seed) + (uint32_t)(a.seed >> 32)) + (uint32_t)t) + (uint32_t)((uint64_t)t >> 32));
}

__device__ __forceinline__ int find_tensor(const Table &t, int chunk) {
  int lo = 0, hi = t.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// V values at p, or the first `left` of them (the others 0).
template <typename T, int V>
__device__ __forceinline__ void load_values(const T *p, int64_t left, bool whole, float (&x)[V]) {
  if (whole && left >= V) {
    constexpr int W = sizeof(T) * V > 16 ? 16 / sizeof(T) : V;
#pragma unroll
    for (int k = 0; k < V; k += W) {
      const Vec<T, W> y = load_vec<T, W>(p + k);
#pragma unroll
      for (int e = 0; e < W; ++e) x[k + e] = (float)y.v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = e < left ? (float)p[e] : 0.f;
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T *p, int64_t left, bool whole, const float (&x)[V]) {
  if (whole && left >= V) {
    constexpr int W = sizeof(T) * V > 16 ? 16 / sizeof(T) : V;
#pragma unroll
    for (int k = 0; k < V; k += W) {
      Vec<T, W> y;
#pragma unroll
      for (int e = 0; e < W; ++e) y.v[e] = static_cast<T>(x[k + e]);
      store_vec<T, W>(p + k, y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = static_cast<T>(x[e]);
  }
}
template <int V>
__device__ __forceinline__ void load_as(const void *p, int type, int64_t i, int64_t left, bool whole, float (&x)[V]) {
  switch (type) {
    case 0: load_values<float, V>(static_cast<const float *>(p) + i, left, whole, x); break;
    case 1: load_values<f16, V>(static_cast<const f16 *>(p) + i, left, whole, x); break;
    default: load_values<bf16, V>(static_cast<const bf16 *>(p) + i, left, whole, x); break;
  }
}
template <int V>
__device__ __forceinline__ void store_as(void *p, int type, int64_t i, int64_t left, bool whole, const float (&x)[V]) {
  switch (type) {
    case 0: store_values<float, V>(static_cast<float *>(p) + i, left, whole, x); break;
    case 1: store_values<f16, V>(static_cast<f16 *>(p) + i, left, whole, x); break;
    default: store_values<bf16, V>(static_cast<bf16 *>(p) + i, left, whole, x); break;
  }
}

__device__ __forceinline__ bool on_16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The largest of a row of 16 lanes, in each of them.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false));  // row_ror 8
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false));
}

// TOP: the code's exponent that stands for the scale's; the code of 0 is 0.
template <int TOP> __device__ __forceinline__ float decode(uint32_t code, uint32_t scale) {
  const uint32_t q = code & (TOP * 8 + 7);
  return __builtin_bit_cast(float, q < 8 ? 0u : (q + ((scale - TOP) << 3)) << 20);
}
template <int TOP> __device__ __forceinline__ uint32_t scale_of(uint32_t largest) {
  return min(max((largest + 0xfffffu) >> 23, TOP + 1u), 255u);
}
// bits of a value >= 0
template <int TOP> __device__ __forceinline__ uint32_t encode(uint32_t bits, uint32_t random, uint32_t scale) {
  const int q = min((int)((bits + (random << 4) + 8) >> 20) - (int)((scale - TOP) << 3), TOP * 8 + 7);
  if (TOP == 31) return q < 8 ? (bits > 0 ? 8 : 0) : q;
  return q < 8 ? 0 : q;
}

template <int BITS>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const Table t, int64_t per, const Moments mo,
                                                         const Factors *__restrict__ fs) {
  constexpr int V = BITS == 8 ? 8 : 4;  // 8: a row of 16 lanes holds a block
  const Factors f = *fs;
  const int k = find_tensor(t, blockIdx.x);
  const int64_t from = (int64_t)((int)blockIdx.x - t.first[k]) * per, n = t.n[k];
  const int64_t to = min(from + per, (n + kBlock - 1) / kBlock * kBlock);
  const bool p_whole = on_16(t.p[k]), g_whole = on_16(t.g[k]), c_whole = on_16(t.copy[k]);
  for (int64_t i0 = from; i0 < to; i0 += kThreads * V) {
    const int64_t i = i0 + threadIdx.x * V, left = n - i, at = t.at[k] + i;
    const bool there = i < to;  // whole rows of lanes
    float p[V], g[V], m[V], v[V];
    uint32_t ms = 0, vs = 0;
    Vec<unsigned char, 8> mc, vc;
    load_as(t.p[k], t.p_type[k], i, there ? left : 0, p_whole, p);
    load_as(t.g[k], t.g_type[k], i, there ? left : 0, g_whole, g);
    if constexpr (BITS == 8) {
      if (there) {
        const unsigned char *pm = static_cast<const unsigned char *>(mo.m) + at, *pv = static_cast<const unsigned char *>(mo.v) + at;
        mc = load_vec<unsigned char, 8>(pm);
        vc = load_vec<unsigned char, 8>(pv);
        ms = mo.m_scale[at / kBlock];
        vs = mo.v_scale[at / kBlock];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t c = there && e < left ? mc.v[e] : 0;
        const float size = decode<15>(c, ms);
        m[e] = c >= 128 ? -size : size;
        v[e] = decode<31>(there && e < left ? vc.v[e] : 0, vs);
      }
    } else {
      load_values<float, V>(static_cast<const float *>(mo.m) + at, there ? left : 0, true, m);
      load_values<float, V>(static_cast<const float *>(mo.v) + at, there ? left : 0, true, v);
    }
    {
#pragma clang fp contract(off)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = g[e] * f.by;
        m[e] = __builtin_fmaf(x, f.rest1, m[e] * f.b1);
        v[e] = __builtin_fmaf(x * x, f.rest2, v[e] * f.b2);
        // the hardware's square root and reciprocal, each right to a unit in the last place of a step that
        // is small next to p; a small v 2^64 times as large, as that root takes no subnormals. Where root and eps are
        // both 0 (v has underflown; or eps is a subnormal, of which the reciprocal is Inf) there is no step
        const bool small = v[e] < 0x1p-96f;
        const float root = __builtin_amdgcn_sqrtf(small ? v[e] * 0x1p64f : v[e]) * (small ? 0x1p-32f : 1.f);
        const float den = __builtin_fmaf(root, f.root, f.eps);
        p[e] = __builtin_fmaf(-f.size, den < 0x1p-126f ? 0.f : m[e] * __builtin_amdgcn_rcpf(den), p[e] * f.decay);
      }
    }
    if (there) {
      store_as(t.p[k], t.p_type[k], i, left, p_whole, p);
      if (t.copy[k] != nullptr) store_as(t.copy[k], t.c_type[k], i, left, c_whole, p);
    }
    if constexpr (BITS == 8) {
      uint32_t mb[V], vb[V], ml = 0, vl = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        mb[e] = e < left ? __builtin_bit_cast(uint32_t, m[e]) & 0x7fffffffu : 0u;
        vb[e] = e < left ? __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu : 0u;
        ml = max(ml, mb[e]);
        vl = max(vl, vb[e]);
      }
      ms = scale_of<15>(row_max(ml));
      vs = scale_of<31>(row_max(vl));
      const uint32_t high = mix(f.key + (uint32_t)((uint64_t)at >> 32));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t r = mix((uint32_t)(at + e) + high);
        mc.v[e] = (unsigned char)(encode<15>(mb[e], r >> 16, ms) | (m[e] < 0.f ? 128u : 0u));
        vc.v[e] = (unsigned char)encode<31>(vb[e], r & 0xffffu, vs);
      }
      if (there) {
        unsigned char *pm = static_cast<unsigned char *>(mo.m) + at, *pv = static_cast<unsigned char *>(mo.v) + at;
        store_vec<unsigned char, 8>(pm, mc);
        store_vec<unsigned char, 8>(pv, vc);
        if (threadIdx.x % 16 == 0) {
          mo.m_scale[at / kBlock] = (unsigned char)ms;
          mo.v_scale[at / kBlock] = (unsigned char)vs;
        }
      }
    } else if (there) {
      store_values<float, V>(static_cast<float *>(mo.m) + at, left, true, m);
      store_values<float, V>(static_cast<float *>(mo.v) + at, left, true, v);
    }
  }
}

// The values that the codes of a moment stand for. n: a multiple of kBlock.
template <typename O, int TOP>
__global__ void __launch_bounds__(kThreads) moments_kernel(const unsigned char *__restrict__ codes,
                                                           const unsigned char *__restrict__ scale, int64_t n,
                                                           int64_t from, O *__restrict__ out) {
  const int64_t i = from + ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i >= n) return;
  const Vec<unsigned char, 8> c = load_vec<unsigned char, 8>(codes + i);
  const uint32_t s = scale[i / kBlock];
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float size = decode<TOP>(c.v[e], s);
    x[e] = TOP == 15 && c.v[e] >= 128 ? -size : size;
  }
  store_values<O, 8>(out + i, 8, true, x);
}

template <typename O>
hipError_t launch_moments(const unsigned char *codes, const unsigned char *scale, bool second, int64_t n, O *out,
                          hipStream_t stream) {
  return launch_in_parts((n / 8 + kThreads - 1) / kThreads, kThreads, [&](int64_t first, unsigned blocks) {
    const int64_t from = first * kThreads * 8;
    if (second) hipLaunchKernelGGL((moments_kernel<O, 31>), dim3(blocks), dim3(kThreads), 0, stream, codes, scale, n, from, out);
    else hipLaunchKernelGGL((moments_kernel<O, 15>), dim3(blocks), dim3(kThreads), 0, stream, codes, scale, n, from, out);
  });
}

}  // namespace

int64_t adamw_workspace_bytes() { return sizeof(Factors); }

hipError_t launch_adamw(const AdamwTensors &a, const AdamwMoments &mo, const AdamwStep &s, void *workspace,
                        hipStream_t stream) {
  Factors *f = static_cast<Factors *>(workspace);
  hipLaunchKernelGGL(step_kernel, dim3(1), dim3(64), 0, stream,
                     StepArgs{s.step, s.seed, s.lr, s.beta1, s.beta2, s.eps, s.decay, s.max_norm, s.lr_at, s.norm}, f);
  if (hipError_t e = hipGetLastError()) return e;
  int64_t total = 0;
  for (int k = 0; k < a.count; ++k) total += a.n[k];
  // whole rounds of a workgroup, and no more chunks than 2^31 / kThreads a launch
  const int64_t per = std::max<int64_t>(2048, (total / kChunks + 2047) / 2048 * 2048);
  const Moments m{mo.m, mo.v, mo.m_scale, mo.v_scale};
  int64_t at = 0;
  for (int k = 0; k < a.count;) {
    Table t;
    t.count = 0;
    t.first[0] = 0;
    for (; k < a.count && t.count < kTensors; ++k) {
      if (a.n[k] > 0) {
        const int c = t.count++;
        t.p[c] = a.p[k];
        t.g[c] = a.g[k];
        t.copy[c] = a.copy ? a.copy[k] : nullptr;
        t.n[c] = a.n[k];
        t.at[c] = at;
        t.p_type[c] = (unsigned char)a.p_type[k];
        t.g_type[c] = (unsigned char)a.g_type[k];
        t.c_type[c] = a.copy ? (unsigned char)a.copy_type[k] : 0;
        t.first[c + 1] = t.first[c] + (int)((a.n[k] + per - 1) / per);
      }
      at += (a.n[k] + kBlock - 1) / kBlock * kBlock;
    }
    if (t.count == 0) break;
    const dim3 grid(t.first[t.count]);
    hipLaunchKernelGGL((mo.bits == 8 ? adamw_kernel<8> : adamw_kernel<32>), grid, dim3(kThreads), 0, stream, t, per, m, f);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

hipError_t launch_adamw_moments(const unsigned char *codes, const unsigned char *scale, bool second, int64_t n,
                                int out_dtype, void *out, hipStream_t stream) {
  if (out_dtype == 0) return launch_moments(codes, scale, second, n, static_cast<float *>(out), stream);
  return launch_moments(codes, scale, second, n, static_cast<bf16 *>(out), stream);
}

}  // namespace bevk
