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
// derivative jumps is known to about 2^-50 (see Gate). At two fp64 instructions a value they
// stay behind the loads.
//
// Both directions are bound by memory and take two launches over the same tiles: sums, then values.
// A tile is a slab of 128 bytes of channels (whole cache lines) by a share of an image's positions,
// one workgroup. Between the launches only each tile's sums by group pass through memory, and each
// workgroup of the second adds up again those of its own slab's groups: a few KB, where a third
// launch between would cost 4 us and tiles of whole rows would read the sums of every group.
// The second launch takes the tiles in the opposite order (within the XCD that had them), so that
// what the first one read last is still in the caches. Six 58 x 100 x 256 maps in 16 bits (res4): 6
// and 9 us forward, 10 and 11 us backward; their 36 and 53 MB once take 5.5 and 8.2 us at the rate of
// a copy of that size.
#include <algorithm>

#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kXcds = 8;

// Lanes across a slab: 8 vectors of 16 bytes, or 64 single channels where rows or tensors are not
// aligned to vectors.
template <typename T, int V> struct Tile {
  static constexpr int kLanes = V > 1 ? 8 : 64;
  static constexpr int kSlab = kLanes * V;            // channels
  static constexpr int kRows = kThreads / kLanes;     // positions side by side
  // Positions of a thread loaded together, one such step ahead (res4 in 16 bits, when it was chosen,
  // 2 / 4 / 8 of them: 6.0 / 6.6 / 8.3 and 9.0 / 9.7 / 10.4 us forward, 9.9 / 10.3 / 11.6 and
  // 10.5 / 10.5 / 12.3 backward).
  static constexpr int kAhead = V > 1 ? 2 : 8;
};

struct Geo {
  int64_t pixels, each;  // positions of an image, and of a tile
  int channels, per;
  int slabs, splits;     // tiles of an image: slabs x splits
  int local;             // room for the groups of a slab
  int64_t tiles;
  int64_t first;         // workgroups in the launches before (launch_in_parts)
};

__device__ __forceinline__ float to_f32(const void *p, int dtype, int64_t i, float none) {
  if (p == nullptr) return none;
  switch (dtype) {
    case 0: return static_cast<const float *>(p)[i];
    case 1: return (float)static_cast<const f16 *>(p)[i];
    default: return (float)static_cast<const bf16 *>(p)[i];
  }
}
// V parameters from channel c on, of x's type or fp32: loaded together.
template <typename T, int V>
__device__ __forceinline__ void load_params(const void *p, int dtype, int c, float none, float *v) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (dtype == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = static_cast<const float *>(p)[c + e];
  } else {
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = static_cast<const T *>(p)[c + e];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)t[e];
  }
}
__device__ __forceinline__ void from_f32(void *p, int dtype, int64_t i, float v) {
  switch (dtype) {
    case 0: static_cast<float *>(p)[i] = v; break;
    case 1: static_cast<f16 *>(p)[i] = static_cast<f16>(v); break;
    default: static_cast<bf16 *>(p)[i] = static_cast<bf16>(v); break;
  }
}

// 1 / (1 + exp(-z)). The types of 16 bits do with the hardware's exp2 and reciprocal (2^-20 relative
// for |z| up to 10, where fp32's own functions have 2^-22): the second launch of six 116 x 200 x 256
// bf16 maps took 29.6 us with them and 34.8 us with fp32's (26.5 us now).
template <typename T> __device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __expf(-z));
}
template <> __device__ __forceinline__ float sigmoid<float>(float z) { return 1.f / (1.f + expf(-z)); }

template <typename T, int ACT> __device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == kActRelu) return z <= 0.f ? 0.f : z;  // NaN stays
  if constexpr (ACT == kActSilu) return z * sigmoid<T>(z);
  return z;
}

// x - mean with mean as two floats, so that a mean far from 0 costs no digits of the difference.
__device__ __forceinline__ float centred(float x, float high, float low) { return (x - high) - low; }

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

// What a channel's values are computed from: its group's mean and 1 / deviation, its own weight, and
// for ReLU its gate (thr, sign), for SiLU its bias.
struct Channel {
  float high, low, rstd, w, u, v;
};

// The constants of a thread's V channels, of one group (WHOLE) or not.
template <int V, bool WHOLE> struct Channels {
  static constexpr int E = WHOLE ? 1 : V;
  float high[E], low[E], rstd[E], w[V], u[V], v[V];
  __device__ __forceinline__ void read(const Channel *ch) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e < E) {
        high[e] = ch[e].high;
        low[e] = ch[e].low;
        rstd[e] = ch[e].rstd;
      }
      w[e] = ch[e].w;
      u[e] = ch[e].u;
      v[e] = ch[e].v;
    }
  }
  // gz and xh of one value of channel e
  template <typename T, int ACT>
  __device__ __forceinline__ void grad(int e, float gy, float x, float &gz, float &xh) const {
    const int k = WHOLE ? 0 : e;
    xh = centred(x, high[k], low[k]) * rstd[k];
    gz = gy;
    if constexpr (ACT == kActRelu) gz = x * v[e] <= u[e] ? 0.f : gy;  // NaN passes, as in ReLU's own derivative
    if constexpr (ACT == kActSilu) {
      const float z = xh * w[e] + u[e], s = sigmoid<T>(z);
      gz = gy * (s * (1.f + z * (1.f - s)));
    }
  }
};

// One tile's place. `back`: the tiles in reverse, each on the XCD (workgroup number modulo 8) that
// has it in the forward order.
struct Place {
  int64_t n, p0, p1;
  int slab, split;
};
__device__ __forceinline__ int64_t tile_of(const Geo &g, int64_t block, bool back) {
  return back ? (g.tiles + kXcds - 1) / kXcds * kXcds - kXcds - block / kXcds * kXcds + block % kXcds : block;
}
__device__ __forceinline__ Place place_of(const Geo &g, int64_t tile) {
  Place p;
  p.slab = (int)(tile % g.slabs);
  const int64_t r = tile / g.slabs;
  p.split = (int)(r % g.splits);
  p.n = r / g.splits;
  p.p0 = p.split * g.each;
  p.p1 = min(p.p0 + g.each, g.pixels);
  return p;
}

// Groups with channels in a slab.
template <int SLAB> __device__ __forceinline__ int first_group(const Geo &g, int slab) { return slab * SLAB / g.per; }
template <int SLAB> __device__ __forceinline__ int group_count(const Geo &g, int slab) {
  return (min(g.channels, (slab + 1) * SLAB) - 1) / g.per - first_group<SLAB>(g, slab) + 1;
}
template <int SLAB>
__device__ __forceinline__ int64_t part_at(const Geo &g, int64_t n, int slab, int split, int group) {
  return ((n * g.slabs + slab) * g.splits + split) * g.local + group - first_group<SLAB>(g, slab);
}

template <typename A> struct Pair {
  A a, b;
};

// The sums of a slab's groups over their tiles: thread k of the first ones returns group k's. 16-byte
// pairs of fp64, or of fp32 as the backward's first launch leaves them.
template <int SLAB, typename A>
__device__ __forceinline__ Pair<double> sum_parts(const Geo &g, int64_t n, int slab, const Pair<A> *part,
                                                  Pair<double> (*sums)[SLAB]) {
  static_assert(SLAB <= kWave, "a lane of each wave for every group");
  const int g0 = first_group<SLAB>(g, slab), count = group_count<SLAB>(g, slab);
  int wide = 1;
  while (wide < count) wide *= 2;
  const int k = threadIdx.x & (wide - 1), j = threadIdx.x / wide, step = kThreads / wide;
  Pair<double> t{0.0, 0.0};
  if (k < count) {
    const int group = g0 + k;
    for (int s = group * g.per / SLAB; s <= ((group + 1) * g.per - 1) / SLAB; ++s) {
      const Pair<A> *p = part + part_at<SLAB>(g, n, s, 0, group);
#pragma unroll 4
      for (int i = j; i < g.splits; i += step) {
        const Pair<A> v = p[(int64_t)i * g.local];
        t.a += (double)v.a;
        t.b += (double)v.b;
      }
    }
  }
  for (int d = wide; d < kWave; d *= 2) {
    t.a += __shfl_xor(t.a, d, kWave);
    t.b += __shfl_xor(t.b, d, kWave);
  }
  if ((int)threadIdx.x % kWave < count) sums[threadIdx.x / kWave][threadIdx.x % kWave] = t;
  __syncthreads();
  if ((int)threadIdx.x < count) {
    t = sums[0][threadIdx.x];
    for (int w = 1; w < kWaves; ++w) {
      t.a += sums[w][threadIdx.x].a;
      t.b += sums[w][threadIdx.x].b;
    }
  }
  return t;
}

// A thread's vectors of U positions of a tile, from position q on. They are loaded a step ahead of
// their use, the first ones before the workgroup adds up the sums it needs.
template <typename T, int V, int U> struct Rows {
  static constexpr int kRows = Tile<T, V>::kRows, kStep = kRows * U;
  Vec<T, V> v[U];
  __device__ __forceinline__ void load(const T *src, const Geo &g, const Place &p, int64_t q, int c) {
    const T *at = src + (p.n * g.pixels + q) * g.channels + c;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * kRows < p.p1 && c < g.channels) v[u] = load_vec<T, V>(at + (int64_t)u * kRows * g.channels);
  }
  __device__ __forceinline__ void store(T *dst, const Geo &g, const Place &p, int64_t q, int c) const {
    T *at = dst + (p.n * g.pixels + q) * g.channels + c;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q + u * kRows < p.p1) store_vec<T, V>(at + (int64_t)u * kRows * g.channels, v[u]);
  }
};

// ---------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------

// Sums of x and x^2 by group of one tile. WHOLE: a vector's channels are of one group.
template <typename T, int V, bool WHOLE>
__global__ void __launch_bounds__(kThreads) stats_kernel(const T *__restrict__ x, Geo g,
                                                         Pair<double> *__restrict__ part) {
  using TL = Tile<T, V>;
  using R = Rows<T, V, TL::kAhead>;
  constexpr int E = WHOLE ? 1 : V;  // sums of a thread
  __shared__ Pair<double> s[kWaves][TL::kLanes * E];
  const Place p = place_of(g, g.first + blockIdx.x);
  const int lane = threadIdx.x % TL::kLanes, wave = threadIdx.x / kWave;
  const int c = (p.slab * TL::kLanes + lane) * V;
  Pair<double> a[E];
#pragma unroll
  for (int e = 0; e < E; ++e) a[e] = {0.0, 0.0};
  int64_t q = p.p0 + threadIdx.x / TL::kLanes;
  R next;
  next.load(x, g, p, q, c);
  for (; q < p.p1 && c < g.channels; q += R::kStep) {
    const R v = next;
    next.load(x, g, p, q + R::kStep, c);
#pragma unroll
    for (int u = 0; u < TL::kAhead; ++u)
      if (q + u * TL::kRows < p.p1)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double t = (double)(float)v.v[u].v[e];
          a[WHOLE ? 0 : e].a += t;
          a[WHOLE ? 0 : e].b += t * t;
        }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    for (int d = TL::kLanes; d < kWave; d *= 2) {
      a[e].a += __shfl_xor(a[e].a, d, kWave);
      a[e].b += __shfl_xor(a[e].b, d, kWave);
    }
    if (threadIdx.x % kWave < TL::kLanes) s[wave][lane * E + e] = a[e];
  }
  __syncthreads();
  const int k = threadIdx.x;
  if (k < group_count<TL::kSlab>(g, p.slab)) {
    const int group = first_group<TL::kSlab>(g, p.slab) + k, c0 = p.slab * TL::kSlab;
    const int lo = max(group * g.per - c0, 0) / (V / E);
    const int hi = min(min((group + 1) * g.per, g.channels) - c0, TL::kSlab) / (V / E);
    Pair<double> t{0.0, 0.0};
    for (int w = 0; w < kWaves; ++w)
      for (int i = lo; i < hi; ++i) {
        t.a += s[w][i].a;
        t.b += s[w][i].b;
      }
    part[part_at<TL::kSlab>(g, p.n, p.slab, p.split, group)] = t;
  }
}

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kThreads) forward_kernel(const T *__restrict__ x, Geo g, GroupNormArgs args,
                                                           const Pair<double> *__restrict__ part,
                                                           Pair<double> *__restrict__ stats, T *__restrict__ y) {
  using TL = Tile<T, V>;
  using R = Rows<T, V, TL::kAhead>;
  constexpr int E = WHOLE ? 1 : V;  // groups of a thread
  __shared__ Pair<double> sums[kWaves][TL::kSlab];
  __shared__ float high_of[TL::kSlab], low_of[TL::kSlab], rstd_of[TL::kSlab];
  const int64_t tile = tile_of(g, g.first + blockIdx.x, true);
  if (tile >= g.tiles) return;
  const Place p = place_of(g, tile);
  const int c = (p.slab * TL::kLanes + threadIdx.x % TL::kLanes) * V;
  int64_t q = p.p0 + threadIdx.x / TL::kLanes;
  R next;
  next.load(x, g, p, q, c);
  float a[V], b[V];
  if (c < g.channels) {
    load_params<T, V>(args.weight, args.param_dtype, c, 1.f, a);
    load_params<T, V>(args.bias, args.param_dtype, c, 0.f, b);
  }
  const Pair<double> t = sum_parts<TL::kSlab>(g, p.n, p.slab, part, sums);
  const int g0 = first_group<TL::kSlab>(g, p.slab);
  if ((int)threadIdx.x < group_count<TL::kSlab>(g, p.slab)) {
    const double m = (double)g.pixels * g.per, mean = t.a / m, var = t.b / m - mean * mean;
    const Pair<double> st{mean, 1.0 / sqrt((var < 0.0 ? 0.0 : var) + args.eps)};
    high_of[threadIdx.x] = (float)mean;
    low_of[threadIdx.x] = (float)(mean - (double)(float)mean);
    rstd_of[threadIdx.x] = (float)st.b;
    const int group = g0 + threadIdx.x;
    if (stats != nullptr && p.split == 0 && group * g.per / TL::kSlab == p.slab) stats[p.n * args.groups + group] = st;
  }
  __syncthreads();
  if (c >= g.channels) return;
  float high[E], low[E];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int k = (c + e) / g.per - g0;
    if (e < E) {
      high[e] = high_of[k];
      low[e] = low_of[k];
    }
    a[e] *= rstd_of[k];
  }
  for (; q < p.p1; q += R::kStep) {
    R v = next;
    next.load(x, g, p, q + R::kStep, c);
#pragma unroll
    for (int u = 0; u < TL::kAhead; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = centred((float)v.v[u].v[e], high[WHOLE ? 0 : e], low[WHOLE ? 0 : e]);
        v.v[u].v[e] = static_cast<T>(act_of<T, ACT>(d * a[e] + b[e]));
      }
    v.store(y, g, p, q, c);
  }
}

// Small maps whose groups each lie in one slab: a workgroup keeps a whole slab of an image in
// registers, and one launch does both. Up to 1,024 positions in fp32, where 1 / 6 images of 1,000 x 256
// take 6.1 / 7.6 us against 6.7 / 9.4 us in two launches, and 512 in 16 bits, where the fp64 sums of
// twice the channels on few CUs cost more (500: 7.1 / 7.3 us against 7.0 / 8.1; 1,000: 9.4 / 9.9
// against 7.2 / 8.8).
constexpr int kSmallThreads = 1024;
template <typename T> constexpr int kSmallRows = sizeof(T) == 4 ? 8 : 4;
template <typename T, int V> constexpr int small_pixels() {
  return kSmallThreads / Tile<T, V>::kLanes * kSmallRows<T>;
}

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(const T *__restrict__ x, Geo g, GroupNormArgs args,
                                                              Pair<double> *__restrict__ stats, T *__restrict__ y) {
  using TL = Tile<T, V>;
  constexpr int E = WHOLE ? 1 : V, kAll = kSmallThreads / kWave, kAcross = kSmallThreads / TL::kLanes;
  __shared__ Pair<double> s[kAll][TL::kLanes * E];
  __shared__ float high_of[TL::kSlab], low_of[TL::kSlab], rstd_of[TL::kSlab];
  const int slab = blockIdx.x % g.slabs, lane = threadIdx.x % TL::kLanes, row = threadIdx.x / TL::kLanes;
  const int64_t n = blockIdx.x / g.slabs;
  const int c = (slab * TL::kLanes + lane) * V, pixels = (int)g.pixels;
  const int64_t at = (n * pixels + row) * g.channels + c;
  const bool in = c < g.channels;
  Vec<T, V> v[kSmallRows<T>];
#pragma unroll
  for (int u = 0; u < kSmallRows<T>; ++u)
    if (in && row + u * kAcross < pixels) v[u] = load_vec<T, V>(x + at + (int64_t)u * kAcross * g.channels);
  float a[V], b[V];
  if (in) {
    load_params<T, V>(args.weight, args.param_dtype, c, 1.f, a);
    load_params<T, V>(args.bias, args.param_dtype, c, 0.f, b);
  }
  Pair<double> t[E];
#pragma unroll
  for (int e = 0; e < E; ++e) t[e] = {0.0, 0.0};
#pragma unroll
  for (int u = 0; u < kSmallRows<T>; ++u)
    if (in && row + u * kAcross < pixels)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double d = (double)(float)v[u].v[e];
        t[WHOLE ? 0 : e].a += d;
        t[WHOLE ? 0 : e].b += d * d;
      }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    for (int d = TL::kLanes; d < kWave; d *= 2) {
      t[e].a += __shfl_xor(t[e].a, d, kWave);
      t[e].b += __shfl_xor(t[e].b, d, kWave);
    }
    if (threadIdx.x % kWave < TL::kLanes) s[threadIdx.x / kWave][lane * E + e] = t[e];
  }
  __syncthreads();
  // A wave for each group in turn: its units of all waves.
  const int g0 = first_group<TL::kSlab>(g, slab), count = group_count<TL::kSlab>(g, slab), units = g.per * E / V;
  for (int k = threadIdx.x / kWave; k < count; k += kAll) {
    const int first = ((g0 + k) * g.per - slab * TL::kSlab) * E / V;
    Pair<double> m{0.0, 0.0};
    for (int i = threadIdx.x % kWave; i < units * kAll; i += kWave) {
      m.a += s[i % kAll][first + i / kAll].a;
      m.b += s[i % kAll][first + i / kAll].b;
    }
    for (int d = kWave / 2; d >= 1; d /= 2) {
      m.a += __shfl_xor(m.a, d, kWave);
      m.b += __shfl_xor(m.b, d, kWave);
    }
    if (threadIdx.x % kWave == 0) {
      const double num = (double)g.pixels * g.per, mean = m.a / num, var = m.b / num - mean * mean;
      const Pair<double> st{mean, 1.0 / sqrt((var < 0.0 ? 0.0 : var) + args.eps)};
      high_of[k] = (float)mean;
      low_of[k] = (float)(mean - (double)(float)mean);
      rstd_of[k] = (float)st.b;
      if (stats != nullptr) stats[n * args.groups + g0 + k] = st;
    }
  }
  __syncthreads();
  if (!in) return;
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] *= rstd_of[(c + e) / g.per - g0];
#pragma unroll
  for (int u = 0; u < kSmallRows<T>; ++u)
    if (row + u * kAcross < pixels) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int k = (c + (WHOLE ? 0 : e)) / g.per - g0;
        v[u].v[e] = static_cast<T>(act_of<T, ACT>(centred((float)v[u].v[e], high_of[k], low_of[k]) * a[e] + b[e]));
      }
      store_vec<T, V>(y + at + (int64_t)u * kAcross * g.channels, v[u]);
    }
}

// ---------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------

// The slab's channels from the forward's statistics.
template <typename T, int V, int ACT>
__device__ __forceinline__ void load_channels(const Geo &g, const GroupNormArgs &args, const Place &p,
                                              const Pair<double> *stats, Channel *ch) {
  using TL = Tile<T, V>;
  const int c = p.slab * TL::kSlab + threadIdx.x;
  if ((int)threadIdx.x < TL::kSlab && c < g.channels) {
    const Pair<double> st = stats[p.n * args.groups + c / g.per];
    Channel r;
    r.high = (float)st.a;
    r.low = (float)(st.a - (double)r.high);
    r.rstd = (float)st.b;
    r.w = to_f32(args.weight, args.param_dtype, c, 1.f);
    r.u = to_f32(args.bias, args.param_dtype, c, 0.f);
    r.v = 0.f;
    if constexpr (ACT == kActRelu) {
      const Gate gate = make_gate(st.a, st.b, r.w, r.u);
      r.u = gate.thr;
      r.v = gate.sign;
    }
    ch[threadIdx.x] = r;
  }
  __syncthreads();
}

// Sums of gz and gz * xh of one tile, by channel for the parameters and, times w, by group for gx.
template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(const T *__restrict__ gy, const T *__restrict__ x, Geo g,
                                                             GroupNormArgs args,
                                                             const Pair<double> *__restrict__ stats,
                                                             Pair<float> *__restrict__ by_group,
                                                             Pair<float> *__restrict__ by_channel) {
  using TL = Tile<T, V>;
  using R = Rows<T, V, TL::kAhead>;
  __shared__ Channel ch[TL::kSlab];
  __shared__ Pair<float> s[kWaves][TL::kSlab];
  const Place p = place_of(g, g.first + blockIdx.x);
  const int lane = threadIdx.x % TL::kLanes, wave = threadIdx.x / kWave;
  const int c = (p.slab * TL::kLanes + lane) * V;
  int64_t q = p.p0 + threadIdx.x / TL::kLanes;
  R next_x, next_d;
  next_x.load(x, g, p, q, c);
  next_d.load(gy, g, p, q, c);
  load_channels<T, V, ACT>(g, args, p, stats, ch);
  Pair<float> a[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = {0.f, 0.f};
  if (c < g.channels) {
    Channels<V, WHOLE> k;
    k.read(ch + lane * V);
    for (; q < p.p1; q += R::kStep) {
      const R v = next_x, d = next_d;
      next_x.load(x, g, p, q + R::kStep, c);
      next_d.load(gy, g, p, q + R::kStep, c);
#pragma unroll
      for (int u = 0; u < TL::kAhead; ++u)
        if (q + u * TL::kRows < p.p1)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float gz, xh;
            k.template grad<T, ACT>(e, (float)d.v[u].v[e], (float)v.v[u].v[e], gz, xh);
            a[e].a += gz;
            a[e].b += gz * xh;
          }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    for (int d = TL::kLanes; d < kWave; d *= 2) {
      a[e].a += __shfl_xor(a[e].a, d, kWave);
      a[e].b += __shfl_xor(a[e].b, d, kWave);
    }
    if (threadIdx.x % kWave < TL::kLanes) s[wave][lane * V + e] = a[e];
  }
  __syncthreads();
  const int k = threadIdx.x, c0 = p.slab * TL::kSlab;
  if (k < TL::kSlab && c0 + k < g.channels) {
    Pair<float> t = s[0][k];
    for (int w = 1; w < kWaves; ++w) {
      t.a += s[w][k].a;
      t.b += s[w][k].b;
    }
    by_channel[(p.n * g.splits + p.split) * g.channels + c0 + k] = t;
    s[0][k] = {t.a * ch[k].w, t.b * ch[k].w};
  }
  __syncthreads();
  if (k < group_count<TL::kSlab>(g, p.slab)) {
    const int group = first_group<TL::kSlab>(g, p.slab) + k;
    const int lo = max(group * g.per - c0, 0), hi = min(min((group + 1) * g.per, g.channels) - c0, TL::kSlab);
    Pair<double> t{0.0, 0.0};
    for (int i = lo; i < hi; ++i) {
      t.a += (double)s[0][i].a;
      t.b += (double)s[0][i].b;
    }
    by_group[part_at<TL::kSlab>(g, p.n, p.slab, p.split, group)] = {(float)t.a, (float)t.b};
  }
}

// gw and gb of 32 channels: all tiles' sums of them.
constexpr int kParamLanes = 32;
__device__ __forceinline__ void param_grads(const Geo &g, const GroupNormArgs &args, int block,
                                            const Pair<float> *by_channel, void *grad_w, void *grad_b,
                                            Pair<double> *sums) {
  const int lane = threadIdx.x % kParamLanes, c = block * kParamLanes + lane;
  const int64_t rows = args.batch * g.splits;
  Pair<double> t{0.0, 0.0};
  if (c < g.channels)
#pragma unroll 4
    for (int64_t r = threadIdx.x / kParamLanes; r < rows; r += kThreads / kParamLanes) {
      const Pair<float> v = by_channel[r * g.channels + c];
      t.a += (double)v.a;
      t.b += (double)v.b;
    }
  sums[threadIdx.x] = t;
  __syncthreads();
  if ((int)threadIdx.x < kParamLanes && c < g.channels) {
    for (int k = lane + kParamLanes; k < kThreads; k += kParamLanes) {
      t.a += sums[k].a;
      t.b += sums[k].b;
    }
    if (grad_b != nullptr) from_f32(grad_b, args.param_dtype, c, (float)t.a);
    if (grad_w != nullptr) from_f32(grad_w, args.param_dtype, c, (float)t.b);
  }
}

template <typename T, int V, bool WHOLE, int ACT>
__global__ void __launch_bounds__(kThreads) grad_x_kernel(const T *__restrict__ gy, const T *__restrict__ x, Geo g,
                                                          GroupNormArgs args, int param_blocks,
                                                          const Pair<double> *__restrict__ stats,
                                                          const Pair<float> *__restrict__ by_group,
                                                          const Pair<float> *__restrict__ by_channel,
                                                          T *__restrict__ gx, void *grad_w, void *grad_b) {
  using TL = Tile<T, V>;
  using R = Rows<T, V, TL::kAhead>;
  constexpr int E = WHOLE ? 1 : V;
  __shared__ union {
    Pair<double> by_group[kWaves][TL::kSlab], by_channel[kThreads];
  } sums;
  __shared__ Pair<float> means[TL::kSlab];
  __shared__ Channel ch[TL::kSlab];
  const int64_t block = g.first + blockIdx.x;
  if (block < param_blocks) {
    param_grads(g, args, (int)block, by_channel, grad_w, grad_b, sums.by_channel);
    return;
  }
  const int64_t tile = tile_of(g, block - param_blocks, true);
  if (tile >= g.tiles || gx == nullptr) return;
  const Place p = place_of(g, tile);
  const int lane = threadIdx.x % TL::kLanes, g0 = first_group<TL::kSlab>(g, p.slab);
  const int c = (p.slab * TL::kLanes + lane) * V;
  int64_t q = p.p0 + threadIdx.x / TL::kLanes;
  R next_x, next_d;
  next_x.load(x, g, p, q, c);
  next_d.load(gy, g, p, q, c);
  load_channels<T, V, ACT>(g, args, p, stats, ch);
  const Pair<double> t = sum_parts<TL::kSlab>(g, p.n, p.slab, by_group, sums.by_group);
  if ((int)threadIdx.x < group_count<TL::kSlab>(g, p.slab)) {
    const double m = (double)g.pixels * g.per;
    means[threadIdx.x] = {(float)(t.a / m), (float)(t.b / m)};
  }
  __syncthreads();
  if (c >= g.channels) return;
  Channels<V, WHOLE> k;
  k.read(ch + lane * V);
  Pair<float> mean[E];
#pragma unroll
  for (int e = 0; e < E; ++e) mean[e] = means[(c + e) / g.per - g0];
  for (; q < p.p1; q += R::kStep) {
    R v = next_x;
    const R d = next_d;
    next_x.load(x, g, p, q + R::kStep, c);
    next_d.load(gy, g, p, q + R::kStep, c);
#pragma unroll
    for (int u = 0; u < TL::kAhead; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float gz, xh;
        k.template grad<T, ACT>(e, (float)d.v[u].v[e], (float)v.v[u].v[e], gz, xh);
        const Pair<float> m = mean[WHOLE ? 0 : e];
        v.v[u].v[e] = static_cast<T>(k.rstd[WHOLE ? 0 : e] * (k.w[e] * gz - (m.a + xh * m.b)));
      }
    v.store(gx, g, p, q, c);
  }
}

// ---------------------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------------------

constexpr int kTiles = 512;  // about: two workgroups on each of 256 CUs

Geo make_geo(int64_t batch, int64_t pixels, int channels, int groups, int slab, int rows) {
  Geo g;
  g.pixels = pixels;
  g.channels = channels;
  g.per = channels / groups;
  g.slabs = (channels + slab - 1) / slab;
  g.local = std::min(groups, (slab - 1) / g.per + 2);
  const int64_t rounds = (pixels + rows - 1) / rows;  // a tile has whole rounds of its positions side by side
  // and at most 64 of them: the fp32 sums of a thread
  const int64_t want = std::max<int64_t>(kTiles / std::max<int64_t>(1, batch * g.slabs), (rounds + 63) / 64);
  g.each = std::max<int64_t>(1, (rounds + want - 1) / want) * rows;
  g.splits = (int)((pixels + g.each - 1) / g.each);
  g.tiles = batch * g.slabs * g.splits;
  g.first = 0;
  return g;
}

template <typename T, int V> Geo geo_of(const GroupNormArgs &a) {
  return make_geo(a.batch, a.pixels, a.channels, a.groups, Tile<T, V>::kSlab, Tile<T, V>::kRows);
}

int64_t by_group_pairs(const Geo &g) { return g.tiles * g.local; }
int64_t by_channel_pairs(const Geo &g, int64_t batch) { return batch * g.splits * g.channels; }

// Vectors of 16 bytes where each row and tensor begins on them.
template <typename T> bool vectors(const GroupNormArgs &a, const void *p, const void *q, const void *r) {
  const uintptr_t all = (uintptr_t)((int64_t)a.channels * sizeof(T)) | reinterpret_cast<uintptr_t>(p) |
                        reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(r);
  return all % 16 == 0;
}

// One launch: up to small_pixels() positions, no group in two slabs, and no more workgroups
// than a launch takes.
template <typename T, int V> bool small(const GroupNormArgs &a) {
  constexpr int kSlab = Tile<T, V>::kSlab;
  const int per = a.channels / a.groups;
  const int64_t workgroups = a.batch * ((a.channels + kSlab - 1) / kSlab);
  return a.pixels <= small_pixels<T, V>() && (a.channels <= kSlab || kSlab % per == 0) &&
         workgroups * kSmallThreads < 1LL << 32;
}

// f(whether a vector's channels are of one group, the activation) as constants.
template <int V, typename F> hipError_t with_kinds(const Geo &g, int act, F f) {
  auto with_act = [&](auto whole) -> hipError_t {
    switch (act) {
      case kActRelu: return f(whole, std::integral_constant<int, kActRelu>());
      case kActSilu: return f(whole, std::integral_constant<int, kActSilu>());
      default: return f(whole, std::integral_constant<int, kActNone>());
    }
  };
  if constexpr (V == 1) {
    return with_act(std::true_type());
  } else if (g.per % V == 0) {
    return with_act(std::true_type());
  } else {
    return with_act(std::false_type());
  }
}

int64_t back_grid(const Geo &g) { return (g.tiles + kXcds - 1) / kXcds * kXcds; }

// f(geometry, workgroups) for `blocks` workgroups of kThreads.
template <typename F> hipError_t in_parts(Geo g, int64_t blocks, F f) {
  return launch_in_parts(blocks, kThreads, [&](int64_t first, unsigned count) {
    g.first = first;
    f(g, count);
  });
}

template <typename T, int V>
hipError_t forward(const GroupNormArgs &a, void *y, double *stats, void *workspace, hipStream_t stream) {
  const Geo geo = geo_of<T, V>(a);
  const T *x = static_cast<const T *>(a.x);
  Pair<double> *part = static_cast<Pair<double> *>(workspace), *st = reinterpret_cast<Pair<double> *>(stats);
  return with_kinds<V>(geo, a.act, [&](auto whole, auto act) {
    constexpr bool W = decltype(whole)::value;
    constexpr int A = decltype(act)::value;
    if (small<T, V>(a)) {
      hipLaunchKernelGGL((small_kernel<T, V, W, A>), dim3((unsigned)(a.batch * geo.slabs)), dim3(kSmallThreads), 0,
                         stream, x, geo, a, st, static_cast<T *>(y));
      return hipGetLastError();
    }
    const hipError_t e = in_parts(geo, geo.tiles, [&](const Geo &g, unsigned count) {
      hipLaunchKernelGGL((stats_kernel<T, V, W>), dim3(count), dim3(kThreads), 0, stream, x, g, part);
    });
    if (e != hipSuccess) return e;
    return in_parts(geo, back_grid(geo), [&](const Geo &g, unsigned count) {
      hipLaunchKernelGGL((forward_kernel<T, V, W, A>), dim3(count), dim3(kThreads), 0, stream, x, g, a, part, st,
                         static_cast<T *>(y));
    });
  });
}

template <typename T, int V>
hipError_t backward(const GroupNormArgs &a, const void *grad_y, const double *stats, void *workspace, void *grad_x,
                    void *grad_w, void *grad_b, hipStream_t stream) {
  const Geo geo = geo_of<T, V>(a);
  const T *gy = static_cast<const T *>(grad_y), *x = static_cast<const T *>(a.x);
  const Pair<double> *st = reinterpret_cast<const Pair<double> *>(stats);
  Pair<float> *by_group = static_cast<Pair<float> *>(workspace), *by_channel = by_group + by_group_pairs(geo);
  // a multiple of the XCDs, so that the tiles behind them begin on the first (those past the channels
  // do nothing)
  const int params = grad_w || grad_b ? (a.channels + kParamLanes * kXcds - 1) / (kParamLanes * kXcds) * kXcds : 0;
  return with_kinds<V>(geo, a.act, [&](auto whole, auto act) {
    constexpr bool W = decltype(whole)::value;
    constexpr int A = decltype(act)::value;
    const hipError_t e = in_parts(geo, geo.tiles, [&](const Geo &g, unsigned count) {
      hipLaunchKernelGGL((grad_sums_kernel<T, V, W, A>), dim3(count), dim3(kThreads), 0, stream, gy, x, g, a, st,
                         by_group, by_channel);
    });
    if (e != hipSuccess) return e;
    return in_parts(geo, params + (grad_x ? back_grid(geo) : 0), [&](const Geo &g, unsigned count) {
      hipLaunchKernelGGL((grad_x_kernel<T, V, W, A>), dim3(count), dim3(kThreads), 0, stream, gy, x, g, a, params, st,
                         by_group, by_channel, static_cast<T *>(grad_x), grad_w, grad_b);
    });
  });
}

template <typename T, int V> int64_t workspace_bytes(const GroupNormArgs &a, bool backward) {
  const Geo g = geo_of<T, V>(a);
  if (backward) return (by_group_pairs(g) + by_channel_pairs(g, a.batch)) * (int64_t)sizeof(Pair<float>);
  return small<T, V>(a) ? 0 : by_group_pairs(g) * (int64_t)sizeof(Pair<double>);
}

template <typename T>
hipError_t forward_t(const GroupNormArgs &a, void *y, double *stats, void *ws, hipStream_t stream) {
  if (vectors<T>(a, a.x, y, y)) return forward<T, 16 / sizeof(T)>(a, y, stats, ws, stream);
  return forward<T, 1>(a, y, stats, ws, stream);
}
template <typename T>
hipError_t backward_t(const GroupNormArgs &a, const void *gy, const double *stats, void *ws, void *gx, void *gw,
                      void *gb, hipStream_t stream) {
  if (vectors<T>(a, a.x, gy, gx)) return backward<T, 16 / sizeof(T)>(a, gy, stats, ws, gx, gw, gb, stream);
  return backward<T, 1>(a, gy, stats, ws, gx, gw, gb, stream);
}

}  // namespace

int64_t group_norm_workspace_bytes(int dtype, bool backward, int64_t batch, int64_t pixels, int channels,
                                   int groups, bool aligned) {
  GroupNormArgs a{};
  a.batch = batch; a.pixels = pixels; a.channels = channels; a.groups = groups;
  aligned = aligned && (int64_t)channels * (dtype == 0 ? 4 : 2) % 16 == 0;
  if (dtype == 0) return aligned ? workspace_bytes<float, 4>(a, backward) : workspace_bytes<float, 1>(a, backward);
  return aligned ? workspace_bytes<f16, 8>(a, backward) : workspace_bytes<f16, 1>(a, backward);
}

hipError_t launch_group_norm_forward(int dtype, const GroupNormArgs &a, void *y, double *stats, void *workspace,
                                     hipStream_t stream) {
  switch (dtype) {
    case 0: return forward_t<float>(a, y, stats, workspace, stream);
    case 1: return forward_t<f16>(a, y, stats, workspace, stream);
    default: return forward_t<bf16>(a, y, stats, workspace, stream);
  }
}

hipError_t launch_group_norm_backward(int dtype, const GroupNormArgs &a, const void *grad_y, const double *stats,
                                      void *workspace, void *grad_x, void *grad_w, void *grad_b,
                                      hipStream_t stream) {
  switch (dtype) {
    case 0: return backward_t<float>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
    case 1: return backward_t<f16>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
    default: return backward_t<bf16>(a, grad_y, stats, workspace, grad_x, grad_w, grad_b, stream);
  }
}

}  // namespace bevk
