// Projections with everything behind them (gfx950): y = act(x W^T + bias) + residual, x [rows][K],
// W [N][K], and the gradients.
//
//   z = x W^T + bias,  y = act(z) + residual,  slope = act'(z)
//   gz = gy slope,  gx = gz W,  gW = gz^T x,  gbias = sum gz,  gresidual = gy
//
// Products of 16-bit types on the matrix cores with fp32 sums; bias, activation and residual in fp32 on the
// sums in registers, one rounding at the end. The forward keeps the slope, as wide as the input, where the
// backward needs it, which then has no exp to take (gz of 40,000 x 512 gelu bf16 in one value: 46 us from z,
// 24 from the slope). gz of 16-bit types is kept as two values of the type, what the first leaves in the second: the
// matrix cores read 16 bits, and one value's rounding would be as large an error of gx and gW as their own.
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

// 16 bytes of a row of each operand: 8 terms of 16 bits in one product, 4 of fp32 in four (each takes one
// of every lane's, the same of both operands: the terms' order does not matter).
template <typename T> __device__ __forceinline__ floatx4 multiply16(int4v a, int4v b, floatx4 c) {
  if constexpr (sizeof(T) == 2) {
    return mfma16(a, b, c, T());
  } else {
    const floatx4 af = __builtin_bit_cast(floatx4, a), bf = __builtin_bit_cast(floatx4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[e], bf[e], c, 0, 0, 0);
    return c;
  }
}

// ---------------------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------------------

// The normal distribution below z, and its density. 16-bit types: below -|z| it is exp(-z^2 / 2) t Q(t) with t = 1 / (1 +
// p |z|), which is nowhere 0 and flat where z is large; Q of degree 6 and p by linear programming over 3,001
// places for the least largest error, of 7e-8 in all or 3e-5 of the value, whichever is less. Q itself is off by 6e-8 at most
// and by 2.5e-5 of the value, however small (half a step of fp16 is 4.9e-4 of it), in 16 instructions where
// erfcf takes 40 of a kernel that is bound by memory. fp32: z^2 and z / sqrt(2) are taken in two pieces, since their
// rounding alone is z^2 / 2 and z^2 half steps of the result, and exp is the exact one.
template <typename T> __device__ __forceinline__ void normal(float z, float &cdf, float &pdf) {
  if constexpr (sizeof(T) == 4) {
    const float q = z * z, e = expf(-0.5f * q);
    const float rest = __builtin_fmaf(z, z, -q);  // (NaN where q is Inf, and e 0)
    pdf = e > 0.f ? 0.3989422804f * __builtin_fmaf(-0.5f * rest, e, e) : 0.3989422804f * e;
    // erfc(y + d) = erfc(y) - 2 / sqrt(pi) exp(-y^2) d
    constexpr float kHigh = 0.707106769f, kLow = 1.21016175e-8f;  // 1 / sqrt(2)
    const float y = -kHigh * z, d = -__builtin_fmaf(kLow, z, __builtin_fmaf(kHigh, z, y));
    cdf = 0.5f * erfcf(y);
    if (e > 0.f) cdf = __builtin_fmaf(-0.5641895835f * e, d, cdf);
  } else {
    const float e = __expf(-0.5f * z * z);
    pdf = 0.3989422804f * e;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.361881793f, __builtin_fabsf(z), 1.f));
    float q = __builtin_fmaf(t, 0.0427341759f, -0.160822466f);
    q = __builtin_fmaf(t, q, 0.148689866f);
    q = __builtin_fmaf(t, q, 0.0493161306f);
    q = __builtin_fmaf(t, q, 0.131715715f);
    q = __builtin_fmaf(t, q, 0.143993139f);
    q = __builtin_fmaf(t, q, 0.144373551f);
    const float tail = e * (t * q);
    cdf = z > 0.f ? 1.f - tail : tail;
  }
}
// act(z), and its derivative.
template <typename T> __device__ __forceinline__ float activate(float z, int act, float &slope) {
  if (act == kActRelu) {
    slope = z <= 0.f ? 0.f : 1.f;  // (a NaN goes through, both ways)
    return z <= 0.f ? 0.f : z;
  }
  if (act == kActSilu) {
    if constexpr (sizeof(T) == 4) {  // s and 1 - s, each to its own last places
      const float e = expf(-__builtin_fabsf(z)), high = 1.f / (1.f + e), low = e * high;
      const float s = z < 0.f ? low : high;
      slope = s * __builtin_fmaf(z, z < 0.f ? high : low, 1.f);
      return z * s;
    }
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));  // (16 bits: off by |z| ulps of fp32)
    slope = s * __builtin_fmaf(z, 1.f - s, 1.f);
    return z * s;
  }
  if (act == kActGelu) {
    float cdf, pdf;
    normal<T>(z, cdf, pdf);
    slope = __builtin_fmaf(z, pdf, cdf);
    return z * cdf;
  }
  slope = 1.f;
  return z;
}

// A slope as the forward keeps it for the backward: fp32 as it is, ReLU's 0 or 1; in 16 bits those of SiLU and
// GELU, between -0.13 and 1.13, as whole numbers: half a step is 2^-16, where rounding to the type would
// add an error of the size that gz's own rounding has.
constexpr uint16_t kSlopeNan = 65535;
template <typename T, int ACT> __device__ __forceinline__ T keep_slope(float s) {
  if constexpr (sizeof(T) == 4 || ACT == kActRelu) return static_cast<T>(s);
  else return __builtin_bit_cast(T, s == s ? (uint16_t)__builtin_rintf(__builtin_fmaf(s, 32768.f, 8192.f)) : kSlopeNan);
}
template <typename T> __device__ __forceinline__ float kept_slope(T v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else {
    const uint16_t u = __builtin_bit_cast(uint16_t, v);
    return u == kSlopeNan ? __builtin_nanf("") : __builtin_fmaf((float)u, 1.f / 32768.f, -0.25f);
  }
}
template <typename T> __device__ __forceinline__ T keep_slope(float s, int act) {
  return act == kActRelu ? keep_slope<T, kActRelu>(s) : keep_slope<T, kActGelu>(s);
}

// f(the activation as a type): a kernel for each, whose code has that one alone.
template <typename F> void with_act(int act, F f) {
  switch (act) {
    case kActNone: f(std::integral_constant<int, kActNone>()); break;
    case kActRelu: f(std::integral_constant<int, kActRelu>()); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>()); break;
    default: f(std::integral_constant<int, kActGelu>()); break;
  }
}

// What is done with a sum. Tensors [M][N].
struct Epilogue {
  const void *bias, *residual;
  void *y, *slope;  // slope: act'(z), or null
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
  float s;
  v = activate<T>(v + bias_at<T>(e, n), e.act, s);
  if (e.act != kActNone && e.slope != nullptr) static_cast<T *>(e.slope)[at] = keep_slope<T>(s, e.act);
  if (e.residual != nullptr) v += (float)static_cast<const T *>(e.residual)[at];
  static_cast<T *>(e.y)[at] = static_cast<T>(v);
}

// ---------------------------------------------------------------------------------------
// Any sizes, strides and alignments: out[m][n] = sum_k a(m, k) b(n, k). A workgroup of four waves takes
// 64 x 64 values, 32 terms at a time through LDS (rows padded by 16 bytes: no two of 8 neighbouring
// rows' reads meet in a bank). Eight neighbouring terms are loaded at once, from whatever address (114,075 x
// 1,001 x 64 fp16: 89 us, 2.7 TB/s; 393 one by one). Few tiles of a long sum: the sum in parts, added up
// in order by finish_kernel. Bound by the latency of its loads, which nothing else is under way beside.
// ---------------------------------------------------------------------------------------
template <typename A, typename B> struct Product {
  const A *a;
  const B *b;
  int64_t a_m, a_k, b_n, b_k;
  int64_t M, K, per;  // per: terms of a part, a multiple of 32
  float *part;        // [parts][M][N], or null for one part
  Epilogue e;
  int halves;         // 2: a is the sum of two, the second a_half behind
  int64_t a_half;
};

// Operands of two types (few rows' gz in fp32 by 16-bit values) meet in fp32. O: the output's type.
template <typename A, typename B, typename O>
__global__ void __launch_bounds__(kThreads) any_kernel(const Product<A, B> p, int64_t first) {
  using T = std::conditional_t<std::is_same_v<A, B>, A, float>;
  constexpr int P = 32 + 16 / (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) T sa[64][P], sb[64][P];
  const int N = p.e.N;
  const int64_t tn = (N + 63) / 64, tm = (p.M + 63) / 64, tile = first + blockIdx.x;
  const int64_t m0 = tile % tm * 64;
  const int n0 = (int)(tile / tm % tn) * 64, z = (int)(tile / tm / tn);
  const int64_t k0 = z * p.per, k1 = min(p.K, k0 + p.per);
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  // a thread's 8 elements of each tile: along k where that is dense, else of one row after another
  auto stage = [&](const auto *src, int64_t by_row, int64_t by_k, int64_t row0, int64_t rows, int64_t k,
                   T (&s)[64][P]) __attribute__((always_inline)) {
    using S = std::remove_cv_t<std::remove_pointer_t<decltype(src)>>;
    const bool along = by_k == 1;
    const int r = along ? tid / 4 : tid % 64, c = (along ? tid % 4 : tid / 64) * 8;
    const S *q = src + (row0 + r) * by_row;
    if (along && row0 + r < rows && k + c + 8 <= k1) {  // (loads of 16 bytes from any address)
      struct __attribute__((packed, aligned(sizeof(S)))) Any { S v[8]; };
      const Any v = *reinterpret_cast<const Any *>(q + k + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[r][c + e] = static_cast<T>(v.v[e]);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t kk = k + c + e;
      s[r][c + e] = row0 + r < rows && kk < k1 ? static_cast<T>(q[kk * by_k]) : static_cast<T>(0.f);
    }
  };
  floatx4 acc[2][2] = {};
  const int ra = wave / 2 * 32 + lane % 16, rb = wave % 2 * 32 + lane % 16, c = lane / 16 * 8;
  for (int half = 0; half < p.halves; ++half)
    for (int64_t k = k0; k < k1; k += 32) {
      stage(p.a + half * p.a_half, p.a_m, p.a_k, m0, p.M, k, sa);
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
        else finish<O>(p.e, m, n, acc[i][j][e]);
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
  const int64_t tiles = ((M + 63) / 64) * ((N + 63) / 64), cus = std::max(1, device_cus());
  // four workgroups a CU in parts of 256 terms or more, or one in shorter ones (300 x 1,001 x 64: 11 us, 18 in parts
  // of 256; 5,000 x 1,001 x 64: 24 us in 12 parts, 19 in 3)
  const int64_t long_parts = std::min(4 * cus / tiles, K / 256), short_parts = std::min(cus / tiles, K / 64);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(std::max(long_parts, short_parts), 64));
  AnyPlan pl;
  pl.per = ((K + parts - 1) / parts + 31) / 32 * 32;
  pl.parts = (int)((K + pl.per - 1) / pl.per);
  return pl;
}
int64_t any_bytes(int64_t M, int64_t N, int64_t K) {
  const AnyPlan pl = any_plan(M, N, K);
  return pl.parts > 1 ? pl.parts * M * N * 4 : 0;
}
template <typename O, typename A, typename B>
hipError_t launch_any(const A *a, int64_t a_m, int64_t a_k, const B *b, int64_t b_n, int64_t b_k, int64_t M, int64_t K,
                      const Epilogue &e, void *workspace, hipStream_t stream, int halves = 1, int64_t a_half = 0) {
  const AnyPlan pl = any_plan(M, e.N, K);
  Product<A, B> p{a, b, a_m, a_k, b_n, b_k, M, K, pl.per, pl.parts > 1 ? static_cast<float *>(workspace) : nullptr, e,
                  halves, a_half};
  const int64_t tiles = ((M + 63) / 64) * (((int64_t)e.N + 63) / 64) * pl.parts;
  hipError_t err = launch_in_parts(tiles, kThreads, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((any_kernel<A, B, O>), dim3(n), dim3(kThreads), 0, stream, p, first);
  });
  if (err != hipSuccess || pl.parts == 1) return err;
  const int64_t total = M * e.N;
  return launch_in_parts((total + kThreads - 1) / kThreads, kThreads, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((finish_kernel<O>), dim3(n), dim3(kThreads), 0, stream, e, p.part, pl.parts, total, first);
  });
}

// ---------------------------------------------------------------------------------------
// Products of tiles: both operands' rows dense, of a multiple of 16 bytes and on such boundaries. A workgroup
// of WM x WN waves takes BM x BN values, 128 bytes of a row (64 terms of 16 bits) at a time: they go straight from
// memory into LDS (8 rows an instruction), the next step's while this one multiplies, in products of 16 x 16
// (of 32 x 32: 245 us where these take 235) that go before the other waves' instructions. Tiles whose
// fragments of a whole step fit read them all before the first product (2,048 x 4,096 x 4,096: 65 us, 73 without).
// 8,192 x 2,048 x 8,192 bf16: 235 us, 1,170 TF; silu, 242. Bound there by what the loads into LDS cost beside the
// products (a quarter of them: 188 us); small ones by the latency of a step, 0.5 us. A row's eight 16-byte
// pieces lie in the order piece ^ (row / 2 % 8), so that 16 neighbouring rows' reads of one piece
// meet none of the 64 banks twice; the order is made by the address that a lane loads from, since it always
// writes where its number says. Rows past the end are the last row's again and are not stored; terms
// past K are zeros in both operands.
// ---------------------------------------------------------------------------------------
constexpr int kRowBytes = 128;  // of a row a step

// 16 bytes from `off` + `k` of the buffer for each lane, to `to` + 16 lane (`to` and k: the wave's).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, char *to, uint32_t off, uint32_t k) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass does not know the builtin, and would leave the kernel out)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)to, 16, off, k, 0, 0);
#endif
}

struct TileArgs {
  const void *a, *b;
  int64_t M;
  int K;
  Epilogue e;
  int64_t tm;
  int tn;
  int64_t per_xcd;
  bool wide;  // N * size a multiple of 16, tensors on 16-byte boundaries
};

// 16 bytes of a row, whose sums have the bias.
template <typename T, int ACT, int V>
__device__ __forceinline__ void finish16(const Epilogue &e, int64_t m, int n, float (&v)[V]) {
  const int64_t at = m * e.N + n;
  Vec<T, V> r;
  if (e.residual != nullptr) r = load_vec<T, V>(static_cast<const T *>(e.residual) + at);
  Vec<T, V> y;
  if (ACT != kActNone && e.slope != nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float s;
      v[k] = activate<T>(v[k], ACT, s);
      y.v[k] = keep_slope<T, ACT>(s);
    }
    store_vec<T, V>(static_cast<T *>(e.slope) + at, y);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float s;
      v[k] = activate<T>(v[k], ACT, s);
    }
  }
  if (e.residual != nullptr)
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] += (float)r.v[k];
#pragma unroll
  for (int k = 0; k < V; ++k) y.v[k] = static_cast<T>(v[k]);
  store_vec<T, V>(static_cast<T *>(e.y) + at, y);
}

// Tile number L of all: groups of 8 rows of tiles, in a group one column of tiles after another, so that
// the tiles that run on an XCD at a time share rows of both operands in its L2.
__device__ __forceinline__ void tile_at(int64_t L, int64_t tm, int tn, int64_t &i, int &j) {
  const int64_t group = L / (8 * (int64_t)tn), left = L - group * 8 * tn;
  const int rows = (int)min((int64_t)8, tm - group * 8);
  j = (int)(left / rows);
  i = group * 8 + left % rows;
}

template <typename T, int ACT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) tile_kernel(const TileArgs p, int64_t first) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, kBK = kRowBytes / (int)sizeof(T);
  constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // 8-row pieces that a wave loads a step
  static_assert(LA * 8 * WAVES == BM && LB * 8 * WAVES == BN && TM * 32 * WM == BM && TN * 32 * WN == BN, "tile");
  __shared__ __attribute__((aligned(1024))) char lds[2][(BM + BN) * kRowBytes];
  const int64_t block = first + blockIdx.x;
  const int64_t L = block % 8 * p.per_xcd + block / 8;
  if (L >= p.tm * p.tn) return;
  int64_t ti;
  int tj;
  tile_at(L, p.tm, p.tn, ti, tj);
  const int64_t m0 = ti * BM;
  const int n0 = tj * BN, N = p.e.N, K = p.K;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  // a tile's rows are below 2^31 bytes apart (K at most 2^21)
  const int ma = (int)min((int64_t)BM, p.M - m0), nb = min(BN, N - n0);
  const uint32_t ld = (uint32_t)K * sizeof(T);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(static_cast<const char *>(p.a) + m0 * ld, ma * ld);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(static_cast<const char *>(p.b) + (int64_t)n0 * ld, nb * ld);
  const int piece[2] = {(lane % 8 ^ lane / 16) * 16, (lane % 8 ^ lane / 16 ^ 4) * 16};  // of even and odd groups of 8 rows
  uint32_t oa[LA], ob[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) oa[i] = min((wave * LA + i) * 8 + lane / 8, ma - 1) * ld + piece[(wave * LA + i) % 2];
#pragma unroll
  for (int i = 0; i < LB; ++i) ob[i] = min((wave * LB + i) * 8 + lane / 8, nb - 1) * ld + piece[(wave * LB + i) % 2];
  const int steps = K / kBK;

  auto load = [&](int step, char *to) __attribute__((always_inline)) {
    const uint32_t k = (uint32_t)step * kRowBytes;
    char *da = to + wave * LA * 1024, *db = to + BM * kRowBytes + wave * LB * 1024;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      load_to_lds(ra, da + i * 1024, oa[i], k);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      load_to_lds(rb, db + i * 1024, ob[i], k);
  };

  floatx4 acc[TM * 2][TN * 2] = {};
  const int wm = wave / WN, wn = wave % WN, row = lane % 16, half = lane / 16;
  auto multiply = [&](const char *from) __attribute__((always_inline)) {
    const char *fa = from + (wm * TM * 32 + row) * kRowBytes, *fb = from + (BM + wn * TN * 32 + row) * kRowBytes;
    int4v a[2][TM * 2], b[2][TN * 2];
    auto read = [&](int k) __attribute__((always_inline)) {
      const int at = ((k * 4 + half) ^ (row / 2 % 8)) * 16;
#pragma unroll
      for (int j = 0; j < TN * 2; ++j) b[k][j] = *reinterpret_cast<const int4v *>(fb + j * 16 * kRowBytes + at);
#pragma unroll
      for (int i = 0; i < TM * 2; ++i) a[k][i] = *reinterpret_cast<const int4v *>(fa + i * 16 * kRowBytes + at);
    };
    constexpr bool kAhead = TM * TN <= 4;  // both steps' fragments fit beside the sums
    if constexpr (kAhead) {
      read(0);
      read(1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (!kAhead) read(k);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < TM * 2; ++i)
#pragma unroll
        for (int j = 0; j < TN * 2; ++j) acc[i][j] = multiply16<T>(b[k][j], a[k][i], acc[i][j]);
      __builtin_amdgcn_s_setprio(0);
    }
  };

  int s = 0;
  if (steps > 0) load(0, lds[0]);
  for (; s + 1 < steps; s += 2) {
    __syncthreads();
    load(s + 1, lds[1]);
    multiply(lds[0]);
    __syncthreads();
    if (s + 2 < steps) load(s + 2, lds[0]);
    multiply(lds[1]);
  }
  if (s < steps) {
    __syncthreads();
    multiply(lds[0]);
  }
  if (K % kBK != 0) {  // the rest of the terms, through registers
    const uint32_t k = (uint32_t)steps * kRowBytes;
    const bool there[2] = {k + piece[0] < ld, k + piece[1] < ld};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const Vec<int, 4> v = buffer_load_vec<int, 4>(ra, there[(wave * LA + i) % 2] ? oa[i] + k : 0xffffffffu);
      *reinterpret_cast<Vec<int, 4> *>(lds[0] + (wave * LA + i) * 1024 + lane * 16) = v;
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const Vec<int, 4> v = buffer_load_vec<int, 4>(rb, there[(wave * LB + i) % 2] ? ob[i] + k : 0xffffffffu);
      *reinterpret_cast<Vec<int, 4> *>(lds[0] + BM * kRowBytes + (wave * LB + i) * 1024 + lane * 16) = v;
    }
    __syncthreads();
    multiply(lds[0]);
  }
  __syncthreads();

  // A lane holds one row and four times four neighbouring columns of each 32 x 32. Each wave turns 32 rows of
  // its own at a time in LDS, so that eight lanes store 128 neighbouring bytes of a row. LDS serves a wave's
  // instructions in order: what keeps the compiler from moving them past each other is turned() alone.
  auto turned = [] __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  };
  constexpr int V = 16 / sizeof(T), P = TN * 32 + 4, C = TN * 32 / V;  // floats of a row, and its pieces of V
  float *turn = reinterpret_cast<float *>(lds[0]) + wave * 32 * P;
  static_assert(WAVES * 32 * P * 4 <= (int)sizeof(lds), "turn");
  const int wn0 = n0 + wn * TN * 32;
  static_assert(64 % C == 0, "a lane's columns are the same in every row");
  float bias[V];
#pragma unroll
  for (int e = 0; e < V; ++e) bias[e] = p.wide && wn0 + lane % C * V < N ? bias_at<T>(p.e, wn0 + lane % C * V + e) : 0.f;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
      for (int j = 0; j < TN * 2; ++j)
        *reinterpret_cast<floatx4 *>(turn + (ii * 16 + row) * P + j * 16 + half * 4) = acc[i * 2 + ii][j];
    turned();
    const int64_t mi = m0 + wm * TM * 32 + i * 32;
    if (p.wide) {
#pragma unroll 2
      for (int c = lane; c < 32 * C; c += 64) {
        const int64_t m = mi + c / C;
        const int n = wn0 + c % C * V;
        float v[V];
#pragma unroll
        for (int h = 0; h < V; h += 4) {
          const Vec<float, 4> x = load_vec<float, 4>(turn + c / C * P + c % C * V + h);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[h + e] = x.v[e] + bias[h + e];
        }
        if (m < p.M && n < N) finish16<T, ACT>(p.e, m, n, v);
      }
    } else {
#pragma unroll 1
      for (int c = lane; c < 32 * TN * 32; c += 64) {
        const int64_t m = mi + c / (TN * 32);
        const int n = wn0 + c % (TN * 32);
        if (m < p.M && n < N) finish<T>(p.e, m, n, turn[c / (TN * 32) * P + c % (TN * 32)]);
      }
    }
    turned();
  }
}

// ---------------------------------------------------------------------------------------
// 16-bit products of many rows by a weight of few terms (K 256 or 512): bound by memory, where a tile of
// few steps waits for its first loads and its stores: 184,950 x 256 x 256 fp16 45 us, 4.2 TB/s (a copy of as
// much 6.0); 40,000 x 256 x 512 bf16 gelu with its slope 37 us (20 without either). A workgroup of eight waves a CU keeps NT
// columns of the weight in LDS (128 KB) for the whole launch; each wave takes R x 16 rows at a time, whose
// fragments it loads straight into registers, a whole 256 terms ahead, across the rows' ends.
// Rows of the weight lie in LDS so that a lane ends up with eight neighbouring columns: row 16 j + 4 g + e
// is column 32 (j / 2) + 8 g + 4 (j % 2) + e.
// ---------------------------------------------------------------------------------------
struct StreamArgs {
  const void *a, *b;
  int64_t M, strips;
  Epilogue e;
  int parts, shares;  // column parts, workgroups of each
};

// act(v) + residual of a few rows of the output, eight neighbouring values (16 bits) or four (fp32) at a byte offset
// that is past `bytes` where there are none. The residual is loaded ahead (RES).
template <typename T, bool RES> struct Rows {
  static constexpr int V = 16 / sizeof(T);
  __amdgpu_buffer_rsrc_t y, slope, residual;
  bool with_slope;
  __device__ __forceinline__ Rows(const Epilogue &e, int64_t row, uint32_t bytes) {
    const int64_t at = row * e.N;
    y = make_rsrc(static_cast<const T *>(e.y) + at, bytes);
    slope = make_rsrc(static_cast<const T *>(e.slope) + at, bytes);
    residual = make_rsrc(static_cast<const T *>(e.residual) + at, bytes);
    with_slope = e.slope != nullptr;
  }
  __device__ __forceinline__ Vec<T, V> ahead(uint32_t at) const { return buffer_load_vec<T, V>(residual, at); }
  template <int ACT> __device__ __forceinline__ void finish(uint32_t at, const Vec<T, V> &r, float (&v)[V]) const {
    Vec<T, V> o;
    if (ACT != kActNone && with_slope) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float s;
        v[k] = activate<T>(v[k], ACT, s);
        o.v[k] = keep_slope<T, ACT>(s);
      }
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(int4v, o), slope, at, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float s;
        v[k] = activate<T>(v[k], ACT, s);
      }
    }
    if constexpr (RES)
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] += (float)r.v[k];
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = static_cast<T>(v[k]);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(int4v, o), y, at, 0, 0);
  }
};

template <typename T, int ACT, bool RES, int K, int NT, int R>
__global__ void __launch_bounds__(512) stream_kernel(const StreamArgs p) {
  constexpr int J = NT / 16, G = J / 4, WAVES = 8;
  __shared__ __attribute__((aligned(1024))) char w[NT * K * 2];  // [K / 128][NT][128 terms]
  __shared__ __attribute__((aligned(16))) float bias[NT];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r16 = lane % 16, g = lane / 16, N = p.e.N;
  constexpr int ld = K * 2, BLOCKS = K / 256;
  // workgroups of one XCD (their number modulo 8) take the parts of one share of rows after another
  const int part = (int)(blockIdx.x / 8) % p.parts, share = (int)(blockIdx.x / 8) / p.parts * 8 + (int)blockIdx.x % 8;
  if (share >= p.shares) return;
  const int n0 = part * NT;
  const int64_t step = (int64_t)p.shares * WAVES;
  int64_t strip = (int64_t)share * WAVES + wave;
  const char *at[R];
  auto rows_of = [&](int64_t s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      at[i] = static_cast<const char *>(p.a) + min((s * R + i) * 16 + r16, p.M - 1) * ld + g * 16;
  };
  int4v a[4][R][2];  // 64 terms each
  auto load = [&](int c, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) a[c][i][h] = *reinterpret_cast<const int4v *>(at[i] + k * 512 + c * 128 + h * 64);
  };
  if (strip < p.strips) {
    rows_of(strip);
#pragma unroll
    for (int c = 0; c < 4; ++c) load(c, 0);
  }
  {
    // (a row's 16-byte pieces lie in the order piece ^ (row % 16): 16 rows' reads of one meet no bank twice)
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(static_cast<const char *>(p.b) + (int64_t)n0 * ld, min(NT, N - n0) * ld);
#pragma unroll 4
    for (int i = wave; i < K / 128 * (NT / 4); i += WAVES) {  // four rows of 256 bytes an instruction
      const int k = i / (NT / 4), r = i % (NT / 4) * 4 + lane / 16;
      const int n = r / 32 * 32 + r % 16 / 4 * 8 + r / 16 % 2 * 4 + r % 4;
      load_to_lds(rb, w + i * 1024, min(n, N - n0 - 1) * ld + (lane ^ r) % 16 * 16, k * 256);
    }
  }
  for (int n = threadIdx.x; n < NT; n += 64 * WAVES) bias[n] = n0 + n < N ? bias_at<T>(p.e, n0 + n) : 0.f;
  __syncthreads();
  if (strip >= p.strips) return;
  const char *from[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) from[h] = w + r16 * 256 + ((h * 4 + g) ^ r16) * 16;
  // four columns' fragments are read while the four before multiply
  int4v b[2][4];
  auto read = [&](int unit, int to) __attribute__((always_inline)) {
    const int q = unit % G, h = unit / G;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      b[to][j] = *reinterpret_cast<const int4v *>(from[h % 4] + (q * 4 + j) * 16 * 256 + h / 4 * NT * 256);
  };
  read(0, 0);
  for (; strip < p.strips; strip += step) {
    asm volatile("" ::: "memory");  // (the weight's reads stay in the loop: registers hold no 128 KB)
    // through buffers that end with the rows: nothing branches around the stores, so that the next rows' loads,
    // which are sent before them, can be waited for without them
    const int64_t row = strip * R * 16;
    const Rows<T, RES> out(p.e, row, (uint32_t)min(p.M - row, (int64_t)R * 16) * (uint32_t)N * 2);
    auto place = [&](int i, int j) __attribute__((always_inline)) {
      const int n = n0 + j * 16 + g * 8;
      return n < N ? (uint32_t)((i * 16 + r16) * N + n) * 2 : 0xffffff00u;
    };
    Vec<T, 8> ahead[RES ? R : 1][RES ? J / 2 : 1];
    if constexpr (RES)
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < J; j += 2) ahead[i][j / 2] = out.ahead(place(i, j));
    floatx4 acc[R][J];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < R; ++i)
        acc[i][j] = *reinterpret_cast<const floatx4 *>(bias + j / 2 * 32 + g * 8 + j % 2 * 4);
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
      if (k + 1 == BLOCKS) rows_of(min(strip + step, p.strips - 1));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < G; ++q) {
            const int unit = (c * 2 + h) * G + q;
            read((k * 8 * G + unit + 1) % (BLOCKS * 8 * G), (unit + 1) % 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int i = 0; i < R; ++i)
                acc[i][q * 4 + j] = mfma16(b[unit % 2][j], a[c][i][h], acc[i][q * 4 + j], T());
            __builtin_amdgcn_sched_barrier(0);
          }
        load(c, (k + 1) % BLOCKS);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < J; j += 2) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = acc[i][j][e];
          v[4 + e] = acc[i][j + 1][e];
        }
        out.template finish<ACT>(place(i, j), ahead[RES ? i : 0][RES ? j / 2 : 0], v);
      }
  }
}

template <typename T, int K, int NT, int R>
hipError_t launch_stream_of(StreamArgs p, hipStream_t stream) {
  p.strips = (p.M + R * 16 - 1) / (R * 16);
  p.parts = (p.e.N + NT - 1) / NT;
  const int cus = std::max(8, device_cus());
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(cus / p.parts, (p.strips + 7) / 8));
  with_act(p.e.act, [&](auto act) {
    const auto kernel = p.e.residual != nullptr ? stream_kernel<T, decltype(act)::value, true, K, NT, R>
                                                : stream_kernel<T, decltype(act)::value, false, K, NT, R>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.shares + 7) / 8 * 8 * p.parts)), dim3(512), 0, stream, p);
  });
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------
// Few rows (single tokens, a decoder's queries): the weight's bytes or the latency of a launch are the
// bound. A workgroup of WAVES waves takes NT x 16 columns of MT x 16 rows; the waves take 64 bytes of the rows in
// turn, which they load straight into the fragments, U loads ahead; their sums meet in LDS. fp32 runs on the
// fp32 matrix cores. 300 x 256 x 256 fp16 4.3 us, of which a launch that does nothing has about 2.5; 4 x 2,048 x
// 8,192 bf16 9.2 us (34 MB at 3.7 TB/s: 16 rows of 64 bytes a load are half the cache lines' width).
// ---------------------------------------------------------------------------------------
struct FewArgs {
  const void *a, *b;
  int64_t M;
  int K;
  Epilogue e;
  int64_t tm;
};

template <typename T, int MT, int NT, int WAVES, int U>
__global__ void __launch_bounds__(64 * WAVES) few_kernel(const FewArgs p, int64_t first) {
  __shared__ __attribute__((aligned(16))) float sum[WAVES][MT * 16][NT * 16 + 4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, r16 = lane % 16, g = lane / 16, N = p.e.N, K = p.K;
  const int64_t tile = first + blockIdx.x, m0 = tile % p.tm * (MT * 16);
  const int n0 = (int)(tile / p.tm) * (NT * 16);
  const uint32_t ld = (uint32_t)K * sizeof(T);  // (below 2^23 bytes)
  const int mt = (int)min((int64_t)MT * 16, p.M - m0), nt = min(NT * 16, N - n0);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(static_cast<const char *>(p.a) + m0 * ld, mt * ld);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(static_cast<const char *>(p.b) + (int64_t)n0 * ld, nt * ld);
  uint32_t oa[MT], ob[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) oa[i] = min(i * 16 + r16, mt - 1) * ld;
#pragma unroll
  for (int j = 0; j < NT; ++j) ob[j] = min(j * 16 + r16, nt - 1) * ld;
  floatx4 acc[MT][NT] = {};
  for (uint32_t k = wave * 64; k < ld; k += U * WAVES * 64) {  // bytes of a row; past its end a load gives zeros
    int4v w[U][NT], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = k + u * WAVES * 64 + g * 16;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        w[u][j] = __builtin_bit_cast(int4v, buffer_load_vec<int, 4>(rb, at < ld ? ob[j] + at : 0xffffffffu));
#pragma unroll
      for (int i = 0; i < MT; ++i)
        x[u][i] = __builtin_bit_cast(int4v, buffer_load_vec<int, 4>(ra, at < ld ? oa[i] + at : 0xffffffffu));
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = multiply16<T>(w[u][j], x[u][i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<floatx4 *>(&sum[wave][i * 16 + r16][j * 16 + g * 4]) = acc[i][j];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * NT * 256; i += 64 * WAVES) {
    const int row = i / (NT * 16), c = i % (NT * 16);
    float v = sum[0][row][c];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) v += sum[q][row][c];
    if (row < mt && c < nt) finish<T>(p.e, m0 + row, n0 + c, v);
  }
}

template <typename T, int MT, int NT, int WAVES, int U>
hipError_t launch_few_of(FewArgs p, hipStream_t stream) {
  p.tm = (p.M + MT * 16 - 1) / (MT * 16);
  return launch_in_parts(p.tm * ((p.e.N + NT * 16 - 1) / (NT * 16)), 64 * WAVES, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((few_kernel<T, MT, NT, WAVES, U>), dim3(n), dim3(64 * WAVES), 0, stream, p, first);
  });
}

bool on_16(std::initializer_list<const void *> all) {
  for (const void *p : all)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

bool rows_take(const void *a, const void *b, int64_t K, int size) {
  return K * size % 16 == 0 && K <= 1 << 21 && on_16({a, b});
}

template <typename T, int BM, int BN, int WM, int WN>
hipError_t launch_tile_of(TileArgs p, hipStream_t stream) {
  p.tm = (p.M + BM - 1) / BM;
  p.tn = (p.e.N + BN - 1) / BN;
  p.per_xcd = (p.tm * p.tn + 7) / 8;
  return launch_in_parts(p.per_xcd * 8, 64 * WM * WN, [&](int64_t first, unsigned n) {
    with_act(p.e.act, [&](auto act) {
      hipLaunchKernelGGL((tile_kernel<T, decltype(act)::value, BM, BN, WM, WN>), dim3(n), dim3(64 * WM * WN), 0, stream, p, first);
    });
  });
}
// Which kernel a product of dense rows takes. 16 bits, K 256 or 512 and enough rows for a few strips a
// wave: the streaming kernel (measured at 40,000 x 256 x 512, 184,950 x 256 x 256, 20,000 x 256 x 4,096
// and 184,950 x 512 x 256: 20.4, 43, 49 and 72 us, the fastest tile 24.5, 54, 76 and 80). Else the least of these
// estimates in us, fitted to some 200 shapes from 1 x 256 x 256 to 40,000 x 4,096 x 1,024, of whose
// measured times the choice is 0.2% off the fastest in the mean:
//   tiles   rounds over the CUs, each of steps of 128 bytes that take the longer of a step's latency and what the
//           tiles on a CU take at its full rate, and what a round's first loads and stores take
//   few     a CU's loads at 33 bytes a ns (each touches 16 rows' 64 bytes)
// fp32: 64 x 64 tiles alone (larger ones were the faster by 5% at the most, below where the split product wins).
enum Kind { kFew4, kFew8, kFew22, kFew42, kTile64, kTile64x128, kTile128, kTile256, kStream };
struct Shape {
  int bm, bn, on_cu;          // rows and columns, workgroups on a CU
  double first, step, latency;  // tiles: us of a round besides its steps, of a step of one tile at full rate, alone
};
constexpr Shape kShapes[kTile256 + 1] = {
    {16, 16, 0, 2.5, 0, 0},      {16, 16, 0, 2.6, 0, 0},      {32, 32, 0, 3.0, 0, 0},      {64, 32, 0, 3.5, 0, 0},
    {64, 64, 5, 3, 0.21, 0.49}, {64, 128, 3, 3.4, 0.32, 0.56}, {128, 128, 2, 5.9, 0.46, 0.62}, {256, 256, 1, 8, 1.51, 1.51}};

constexpr Shape kTile64F32 = {64, 64, 5, 2.3, 0.52, 0.35};

Kind plan(int size, int64_t M, int64_t N, int64_t K, bool wide, double *estimate = nullptr) {
  const int64_t cus = std::max(8, device_cus());
  // streamed rows: enough of them that the weight's way into LDS does not count, and not more parts of the
  // columns than workgroups on an XCD, whose L2 they read the rows from (10,000 x 256 x 8,192: 54 us streamed, 76 by
  // tiles; x 12,288: 128 and 109. 40,000 x 512 x 256: 20 and 26; 10,000 x 512 x 256: 11.0 and 10.4)
  if (size == 2 && wide && (K == 256 || K == 512)) {
    const int64_t parts = (N + 65536 / K - 1) / (65536 / K);
    if (parts * 8 <= cus && (M + 15) / 16 * parts >= cus * (K == 256 ? 12 : 24)) return kStream;
  }
  Kind best = kFew4;
  double best_t = 0;
  for (int k = kFew4; k <= (size == 2 ? kTile256 : kTile64); ++k) {
    const Shape &s = size == 4 && k == kTile64 ? kTile64F32 : kShapes[k];
    const int64_t n = (((M + s.bm - 1) / s.bm) * ((N + s.bn - 1) / s.bn) + cus - 1) / cus;  // workgroups of a CU
    double t;
    if (k <= kFew42) {
      const double steps = (double)((K * size + 63) / 64);  // (a wave has at least one batch of loads to wait for)
      t = s.first + (double)n * (s.bm + s.bn) * steps * 64 / 33e3 + (k == kFew4 ? 0.0125 : 0.007) * steps;
    } else {
      const int64_t full = n / s.on_cu, rest = n % s.on_cu;
      const double steps = (double)((K * size + kRowBytes - 1) / kRowBytes);
      t = full * (steps * std::max(s.latency, s.on_cu * s.step) + s.first) +
          (rest > 0 ? steps * std::max(s.latency, rest * s.step) + s.first : 0);
    }
    if (k == kFew4 || t < best_t) {
      best = (Kind)k;
      best_t = t;
    }
  }
  if (estimate != nullptr) *estimate = best_t;
  return best;
}

template <typename T>
hipError_t launch_rows(const T *a, const T *b, int64_t M, int64_t K, const Epilogue &e, hipStream_t stream) {
  const bool wide = e.N * sizeof(T) % 16 == 0 && on_16({e.residual, e.y, e.slope, e.bias});
  const Kind kind = plan(sizeof(T), M, e.N, K, wide);
  const FewArgs few{a, b, M, (int)K, e, 0};
  switch (kind) {
    case kFew4: return launch_few_of<T, 1, 1, 4, 8>(few, stream);
    case kFew8: return launch_few_of<T, 1, 1, 8, 8>(few, stream);
    case kFew22: return launch_few_of<T, 2, 2, 8, 4>(few, stream);
    case kFew42: return launch_few_of<T, 4, 2, 8, 4>(few, stream);
    default: break;
  }
  const TileArgs tile{a, b, M, (int)K, e, 0, 0, 0, wide};
  if (kind == kTile64) return launch_tile_of<T, 64, 64, 2, 2>(tile, stream);
  if constexpr (sizeof(T) == 2) {
    const StreamArgs rows{a, b, M, 0, e, 0, 0};
    switch (kind) {
      case kTile64x128: return launch_tile_of<T, 64, 128, 1, 4>(tile, stream);
      case kTile128: return launch_tile_of<T, 128, 128, 2, 2>(tile, stream);
      case kTile256: return launch_tile_of<T, 256, 256, 2, 4>(tile, stream);
      default: break;
    }
    return K == 256 ? launch_stream_of<T, 256, 256, 1>(rows, stream) : launch_stream_of<T, 512, 128, 1>(rows, stream);
  }
  return hipErrorInvalidValue;
}

// fp32 products of more than a few rows: the split product of dcn_f32.hip (three bf16 pieces an operand).
// It adds a residual or applies ReLU itself; other epilogues are a pass behind it.
bool split_takes(const void *a, const void *b, int64_t N, int64_t K, bool transposed) {
  return K % 32 == 0 && K <= 1 << 20 && (!transposed || (N % 16 == 0 && N <= 1 << 20)) &&
         f32_split_weight_bytes(N, K) < 1LL << 31 && on_16({a, b});  // (32-bit offsets, a grid's second size)
}
// Against the kernels that run on the fp32 matrix cores, by estimates of both (us) fitted to 166 shapes from 32 x 256 x 64
// to 10,000 x 2,048 x 256: the faster in nearly all, 1.3% off it in the mean. Cutting the weight is what few rows
// do not pay for: 2 x 2,048 x 8,192 18 us without and 62 with, 600 x 2,048 x 8,192 182 and 161.
bool split_pays(int64_t M, int64_t N, int64_t K) {
  double rows = 0;
  plan(4, M, N, K, false, &rows);
  return rows > 9.5 + 1.4e-6 * N * K + 4e-3 * K + 12.3e-9 * M * N * K;
}

// y = act(y) + residual, and slope (or null).
template <typename T>
__global__ void __launch_bounds__(kThreads) act_kernel(T *__restrict__ y, const T *__restrict__ residual,
                                                       T *__restrict__ slope, int act, int64_t total, bool wide, int64_t first) {
  constexpr int V = 16 / sizeof(T);
  const int64_t i = ((first + blockIdx.x) * kThreads + threadIdx.x) * V;
  if (i >= total) return;
  if (wide && i + V <= total) {
    Vec<T, V> v = load_vec<T, V>(y + i), r{}, d;
    if (residual != nullptr) r = load_vec<T, V>(residual + i);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s;
      v.v[e] = static_cast<T>(activate<T>((float)v.v[e], act, s) + (float)r.v[e]);
      d.v[e] = keep_slope<T>(s, act);
    }
    store_vec<T, V>(y + i, v);
    if (slope != nullptr) store_vec<T, V>(slope + i, d);
  } else {
    for (int64_t k = i; k < min(i + V, total); ++k) {
      float s;
      y[k] = static_cast<T>(activate<T>((float)y[k], act, s) + (residual != nullptr ? (float)residual[k] : 0.f));
      if (slope != nullptr) slope[k] = keep_slope<T>(s, act);
    }
  }
}

// The streaming kernel for fp32: K 256 or 512, N a multiple of 4. NB x 16 columns of the split weight (its three planes
// in the order of the fragments, 96 KB) stay in LDS, a wave takes 16 rows at a time, eight steps of 32 terms ahead,
// and cuts its fragments as they come. A strip that meets a value that is not finite (or rounds to Inf as a bf16) is
// computed again in plain fp32. 40,000 x 256 x 256 36 us and 44 with a residual (82 and 123 MB, six products of bf16
// for each of fp32: 31 GF at 880 TF): bound by the products and their operands' cutting.
struct SplitStreamArgs {
  const float *a;
  const void *w;  // split weight, then its flags
  int64_t M, strips;
  Epilogue e;
  int parts, shares;
};

template <int ACT, bool RES, int K>
__global__ void __launch_bounds__(512) split_stream_kernel(const SplitStreamArgs p) {
  constexpr int S = K / 32, NB = 32 / S, WAVES = 8, PIECE = 3 * 1024, BLOCK = S * PIECE;  // S steps; bytes of 16 columns
  __shared__ __attribute__((aligned(1024))) char w[NB * BLOCK];
  __shared__ __attribute__((aligned(16))) float bias[NB * 16];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int r16 = lane % 16, g = lane / 16, N = p.e.N;
  const int part = (int)(blockIdx.x / 8) % p.parts, share = (int)(blockIdx.x / 8) / p.parts * 8 + (int)blockIdx.x % 8;
  if (share >= p.shares) return;
  const int n0 = part * NB * 16, nb_total = (N + 15) / 16, nb = min(NB, nb_total - part * NB);
  const int64_t step = (int64_t)p.shares * WAVES;
  int64_t strip = (int64_t)share * WAVES + wave;
  const float *at;
  auto rows_of = [&](int64_t s) __attribute__((always_inline)) { at = p.a + min(s * 16 + r16, p.M - 1) * K + g * 8; };
  floatx4 a[8][2];
  auto load = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) a[k % 8][h] = *reinterpret_cast<const floatx4 *>(at + k * 32 + h * 4);
  };
  if (strip < p.strips) {
    rows_of(strip);
#pragma unroll
    for (int k = 0; k < 8; ++k) load(k);
  }
  {
    const char *from = static_cast<const char *>(p.w) + (int64_t)part * NB * BLOCK;
    const __amdgpu_buffer_rsrc_t rb = make_rsrc(from, nb * BLOCK);
#pragma unroll 4
    for (int i = wave; i < NB * BLOCK / 1024; i += WAVES)  // (columns past the last block: the first block's again)
      load_to_lds(rb, w + i * 1024, (i * 1024 < nb * BLOCK ? i * 1024 : i * 1024 % BLOCK) + lane * 16, 0);
  }
  for (int n = threadIdx.x; n < NB * 16; n += 64 * WAVES) bias[n] = n0 + n < N ? bias_at<float>(p.e, n0 + n) : 0.f;
  const uint32_t *flags = reinterpret_cast<const uint32_t *>(static_cast<const char *>(p.w) + (int64_t)nb_total * BLOCK) + part * NB * S;
  bool bad_weight = false;
  for (int i = threadIdx.x; i < nb * S; i += 64 * WAVES) bad_weight |= flags[i] != 0;
  bad_weight = __syncthreads_or(bad_weight);
  if (strip >= p.strips) return;
  // one block's three fragments are read while the block before multiplies
  int4v b[2][3];
  auto read = [&](int unit, int to) __attribute__((always_inline)) {
    const int j = unit % NB, k = unit / NB % S;
#pragma unroll
    for (int q = 0; q < 3; ++q)
      b[to][q] = *reinterpret_cast<const int4v *>(w + j * BLOCK + k * PIECE + q * 1024 + lane * 16);
  };
  read(0, 0);
  for (; strip < p.strips; strip += step) {
    asm volatile("" ::: "memory");  // (the weight's reads stay in the loop)
    const int64_t row = strip * 16;
    const Rows<float, RES> out(p.e, row, (uint32_t)min(p.M - row, (int64_t)16) * (uint32_t)N * 4);
    auto place = [&](int j) __attribute__((always_inline)) {
      const int n = n0 + j * 16 + g * 4;
      return n < N ? (uint32_t)(r16 * N + n) * 4 : 0xffffff00u;
    };
    Vec<float, 4> ahead[RES ? NB : 1];
    if constexpr (RES)
#pragma unroll
      for (int j = 0; j < NB; ++j) ahead[j] = out.ahead(place(j));
    floatx4 hi[NB] = {}, lo[NB] = {};
    float nf = 0.f;
#pragma unroll
    for (int k = 0; k < S; ++k) {
      int4v x[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Cut2 c = cut2(a[k % 8][e / 2][e % 2 * 2], a[k % 8][e / 2][e % 2 * 2 + 1]);
        x[0][e] = c.h; x[1][e] = c.m; x[2][e] = c.l;
        nf += c.nf;
      }
      if (k + 8 == S) rows_of(min(strip + step, p.strips - 1));
      load((k + 8) % S);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int unit = k * NB + j;
        read(unit + 1, (unit + 1) % 2);
        __builtin_amdgcn_sched_barrier(0);
        const int4v(&f)[3] = b[unit % 2];
        lo[j] = mfma16(f[0], x[2], lo[j], bf16());
        hi[j] = mfma16(f[0], x[0], hi[j], bf16());
        lo[j] = mfma16(f[2], x[0], lo[j], bf16());
        lo[j] = mfma16(f[1], x[1], lo[j], bf16());
        lo[j] = mfma16(f[0], x[1], lo[j], bf16());
        lo[j] = mfma16(f[1], x[0], lo[j], bf16());
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (__any(bad_weight || !(nf == nf))) {
      const float *xr = p.a + min(row + r16, p.M - 1) * K;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        floatx4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
          const char *blk = w + j * BLOCK + k / 32 * PIECE + k % 32 / 8 * 256 + k % 8 * 2 + g * 64;  // column 4 g
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float wv = 0.f;
#pragma unroll
            for (int q = 2; q >= 0; --q)
              wv += __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t *>(blk + q * 1024 + e * 16) << 16);
            v[e] = __builtin_fmaf(xr[k], wv, v[e]);
          }
        }
        hi[j] = v;
        lo[j] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const floatx4 c = *reinterpret_cast<const floatx4 *>(bias + j * 16 + g * 4);
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (hi[j][e] + lo[j][e]) + c[e];
      out.template finish<ACT>(place(j), ahead[RES ? j : 0], v);
    }
  }
}

template <int K> hipError_t launch_split_stream(SplitStreamArgs p, hipStream_t stream) {
  p.strips = (p.M + 15) / 16;
  p.parts = (p.e.N + 16384 / K - 1) / (16384 / K);
  const int cus = std::max(8, device_cus());
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(cus / p.parts, (p.strips + 7) / 8));
  with_act(p.e.act, [&](auto act) {
    const auto kernel = p.e.residual != nullptr ? split_stream_kernel<decltype(act)::value, true, K>
                                                : split_stream_kernel<decltype(act)::value, false, K>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.shares + 7) / 8 * 8 * p.parts)), dim3(512), 0, stream, p);
  });
  return hipGetLastError();
}

// act(x W^T + bias) + residual as Epilogue has them; workspace: f32_split_weight_bytes.
hipError_t launch_split(const float *x, const float *weight, bool transposed, int64_t M, int N, int K, const Epilogue &e,
                        void *workspace, hipStream_t stream) {
  hipError_t err = transposed ? launch_f32_split_weight(weight, K, N, 1, true, workspace, stream)
                              : launch_f32_split_weight(weight, N, K, 1, false, workspace, stream);
  if (err != hipSuccess) return err;
  // (K 512 without anything behind it: 89 us in the tiled kernel at 40,000 x 512 x 256, 94 streamed; with a residual
  // 111 and 99. More parts of columns than workgroups on an XCD read the rows too often: 10,000 x 256 x 2,048 68 us
  // streamed and 86 tiled, x 4,096 207 and 154)
  const bool few_parts = (N + 16384 / K - 1) / (16384 / K) * 8 <= std::max(8, device_cus());
  if ((K == 256 || (K == 512 && (e.residual != nullptr || e.act != kActNone))) && few_parts && N % 4 == 0 &&
      on_16({e.residual, e.y, e.slope})) {
    const SplitStreamArgs p{x, workspace, M, 0, e, 0, 0};
    return K == 256 ? launch_split_stream<256>(p, stream) : launch_split_stream<512>(p, stream);
  }
  const bool relu = e.act == kActRelu && e.residual == nullptr && e.slope == nullptr;
  const bool pass = e.act != kActNone && !relu;  // act(z) + residual in a pass of its own
  float *out = static_cast<float *>(e.y);
  const float *addend = pass ? nullptr : static_cast<const float *>(e.residual);
  const int64_t most = ((1LL << 31) - 4096) / ((int64_t)K * 4) / 16 * 16;  // rows below 2 GiB
  for (int64_t m = 0; m < M; m += most) {
    err = launch_f32_split(nullptr, N, (int)std::min(most, M - m), K, x + m * K, nullptr, 0, nullptr, workspace,
                           static_cast<const float *>(e.bias), out + m * N, stream, relu,
                           addend == nullptr ? nullptr : addend + m * N);
    if (err != hipSuccess) return err;
  }
  if (!pass) return hipSuccess;
  const int64_t total = M * N;
  return launch_in_parts((total + kThreads * 4 - 1) / (kThreads * 4), kThreads, [&](int64_t first, unsigned n) {
    hipLaunchKernelGGL((act_kernel<float>), dim3(n), dim3(kThreads), 0, stream, out, static_cast<const float *>(e.residual),
                       static_cast<float *>(e.slope), e.act, total, on_16({out, e.residual, e.slope}), first);
  });
}

// ---------------------------------------------------------------------------------------
// gz = gy slope and its column sums, bound by memory (40,000 x 512 bf16, gz in two values: 164 MB in 31 us, 5.2 TB/s): a workgroup
// takes a range of rows of up to 256 vectors of columns;
// each thread keeps its columns' sums, the workgroup adds up its rows side by side and turn_kernel the
// workgroups, in order; in the same launch it turns the weight for the gradient of x.
// ---------------------------------------------------------------------------------------
constexpr int kSumBlocks = 1024;

// v = first + second: the nearest value of T, kept finite where v is (a slope is up to 1.13, so gz may leave T's
// range), and the nearest to what it leaves (|second| at most half a step of first, its own error 2^-8 of that
// in bf16). NaN and Inf are the first's alone.
template <typename T> __device__ __forceinline__ void in_two(float v, T &first, T &second) {
  constexpr float kMost = std::is_same_v<T, f16> ? 65504.f : 3.38953139e38f;
  const bool finite = __builtin_fabsf(v) <= 3.402823466e38f;
  first = static_cast<T>(finite ? __builtin_amdgcn_fmed3f(v, -kMost, kMost) : v);
  second = static_cast<T>(finite ? v - (float)first : 0.f);
}

// PAIR: gz in two values, a row's first ones and then its second ones.
template <typename T, typename O, int V, bool PAIR>
__global__ void __launch_bounds__(kThreads) grad_z_kernel(const T *__restrict__ gy, const T *__restrict__ slope,
                                                          O *__restrict__ gz, int act, int64_t rows, int n, int per,
                                                          float *__restrict__ part) {
  __shared__ float s[kThreads][V + 1];
  const int lanes = kThreads / per, col = (blockIdx.x * per + threadIdx.x % per) * V, row = threadIdx.x / per;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float a[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = 0.f;
  if (row < lanes && col < n) {
#pragma unroll 4
    for (int64_t r = r0 + row; r < r1; r += lanes) {
      const int64_t at = r * n + col;
      const Vec<T, V> g = load_vec<T, V>(gy + at);
      float z[V];  // (the sums are those of gz before its rounding)
#pragma unroll
      for (int e = 0; e < V; ++e) z[e] = (float)g.v[e];
      if (act != kActNone) {
        const Vec<T, V> x = load_vec<T, V>(slope + at);
        Vec<O, V> out, rest;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (act == kActRelu) z[e] = (float)x.v[e] <= 0.f ? 0.f : z[e];  // (slope, or y)
          else z[e] *= kept_slope(x.v[e]);
          if constexpr (PAIR) in_two(z[e], out.v[e], rest.v[e]);
          else out.v[e] = static_cast<O>(z[e]);
        }
        O *to = gz + (PAIR ? at + r * n : at);
        store_vec<O, V>(to, out);
        if constexpr (PAIR) store_vec<O, V>(to + n, rest);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] += z[e];
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
  for (int e = 0; e < V; ++e) part[(int64_t)blockIdx.y * n + col + e] = a[e];
}

// The first `sums` workgroups: 16 columns each, 64 threads add up every 64th part, then in order. The others:
// 64 x 64 values of weight [rows][cols] into turned [cols][halves][rows].
struct TurnArgs {
  const float *part;
  int parts, n, sums;
  void *out;
  const void *weight;
  void *turned;
  int rows, cols, halves;
};
template <typename T, bool WIDE>
__global__ void __launch_bounds__(1024) turn_kernel(const TurnArgs p, int64_t first) {
  __shared__ float s[64][17];
  __shared__ T tile[64][65];
  const int64_t block = first + blockIdx.x;
  if (block < p.sums) {
    const int c = (int)block * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
    float v = 0.f;
    if (c < p.n)
#pragma unroll 8
      for (int q = k; q < p.parts; q += 64) v += p.part[(int64_t)q * p.n + c];
    s[k][threadIdx.x % 16] = v;
    __syncthreads();
    for (int half = 32; half > 0; half /= 2) {
      if (k < half) s[k][threadIdx.x % 16] += s[k + half][threadIdx.x % 16];
      __syncthreads();
    }
    if (k == 0 && c < p.n) {
      if (WIDE) static_cast<float *>(p.out)[c] = s[0][threadIdx.x];
      else static_cast<T *>(p.out)[c] = static_cast<T>(s[0][threadIdx.x]);
    }
    return;
  }
  const int across = (p.cols + 63) / 64;
  const int r0 = (int)((block - p.sums) / across) * 64, c0 = (int)((block - p.sums) % across) * 64, lane = threadIdx.x % 64;
  const T *w = static_cast<const T *>(p.weight);
  T *t = static_cast<T *>(p.turned);
#pragma unroll
  for (int i = threadIdx.x / 64; i < 64; i += 16)
    if (r0 + i < p.rows && c0 + lane < p.cols) tile[i][lane] = w[(int64_t)(r0 + i) * p.cols + c0 + lane];
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x / 64; i < 64; i += 16)
    if (c0 + i < p.cols && r0 + lane < p.rows)
      for (int h = 0; h < p.halves; ++h) t[((int64_t)(c0 + i) * p.halves + h) * p.rows + r0 + lane] = tile[lane][i];
}

// (a launch of many columns has workgroups enough: its grid and the parts' memory stay small)
int sum_blocks(int64_t rows, int n) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({kSumBlocks, rows / 16, (1 << 22) / n}));
}

template <int V, bool PAIR, typename T, typename O>
hipError_t launch_grad_z_v(const T *gy, const T *slope, O *gz, int act, int64_t rows, int n, float *part, hipStream_t stream) {
  const int vecs = (n + V - 1) / V, per = std::min(vecs, kThreads);
  hipLaunchKernelGGL((grad_z_kernel<T, O, V, PAIR>), dim3((vecs + per - 1) / per, sum_blocks(rows, n)), dim3(kThreads), 0, stream,
                     gy, slope, gz, act, rows, n, per, part);
  return hipGetLastError();
}
template <bool PAIR, typename T, typename O>
hipError_t launch_grad_z(const T *gy, const T *slope, O *gz, int act, int64_t rows, int n, float *part, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  return n % V == 0 && on_16({gy, slope, gz}) ? launch_grad_z_v<V, PAIR>(gy, slope, gz, act, rows, n, part, stream)
                                              : launch_grad_z_v<1, PAIR>(gy, slope, gz, act, rows, n, part, stream);
}
// The bias' gradient (or null for none) and, where `halves` is not 0, the weight turned, that many times side by side.
template <typename T>
hipError_t launch_turn(const float *part, int64_t rows, void *grad_bias, bool wide, const LinearArgs &a, int halves,
                       void *turned, hipStream_t stream) {
  const TurnArgs p{part, sum_blocks(rows, a.N), a.N, grad_bias != nullptr ? (a.N + 15) / 16 : 0, grad_bias, a.weight, turned, a.N, a.K, halves};
  const int64_t tiles = halves > 0 ? ((a.N + 63) / 64) * (int64_t)((a.K + 63) / 64) : 0;
  return launch_in_parts(p.sums + tiles, 1024, [&](int64_t first, unsigned n) {
    if (wide) hipLaunchKernelGGL((turn_kernel<T, true>), dim3(n), dim3(1024), 0, stream, p, first);
    else hipLaunchKernelGGL((turn_kernel<T, false>), dim3(n), dim3(1024), 0, stream, p, first);
  });
}

// ---------------------------------------------------------------------------------------
// What a call runs
// ---------------------------------------------------------------------------------------
int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

enum Route { kAny, kSplit, kRows };
template <typename T> Route route(const T *x, const T *weight, bool transposed, int64_t M, int64_t N, int64_t K) {
  if (sizeof(T) == 4 && split_takes(x, weight, N, K, transposed) && split_pays(M, N, K)) return kSplit;
  return rows_take(x, transposed ? nullptr : weight, K, sizeof(T)) ? kRows : kAny;
}
// What a product of rows x [M][halves][K] by weight [N][K] (transposed: [K][N]) needs, its operands on 16-byte boundaries
// or not.
int64_t product_bytes(int dtype, bool transposed, int64_t M, int64_t N, int64_t K, bool aligned, int halves = 1) {
  if (!aligned) return any_bytes(M, N, K);
  switch (dtype == 0 ? route<float>(nullptr, nullptr, transposed, M, N, K)
                     : route<f16>(nullptr, nullptr, transposed, M, N, K * halves)) {
    case kSplit: return f32_split_weight_bytes(N, K);
    case kRows: return transposed ? up(N * K * halves * (dtype == 0 ? 4 : 2)) : 0;
    default: return any_bytes(M, N, K);
  }
}
// transposed: of kRows the workspace holds the weight's transpose already (it is small next to the rows), for each
// of x's halves, whose sum is then one product of twice the terms
template <typename T>
hipError_t product(const T *x, const T *weight, bool transposed, int64_t M, int K, const Epilogue &e, void *workspace,
                   hipStream_t stream, int halves = 1) {
  switch (route(x, weight, transposed, M, e.N, K * halves)) {
    case kAny: return launch_any<T>(x, (int64_t)K * halves, 1, weight, transposed ? 1 : K, transposed ? e.N : 1, M, K, e, workspace,
                                    stream, halves, K);
    case kRows: return launch_rows(x, transposed ? static_cast<const T *>(workspace) : weight, M, K * halves, e, stream);
    default: break;
  }
  if constexpr (sizeof(T) == 4) return launch_split(x, weight, transposed, M, e.N, K, e, workspace, stream);
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t forward(const LinearArgs &a, const void *residual, void *y, void *slope, void *workspace, hipStream_t stream) {
  const Epilogue e{a.bias, residual, y, slope, a.bias_wide, a.act, a.N};
  return product(static_cast<const T *>(a.x), static_cast<const T *>(a.weight), false, a.rows, a.K, e, workspace, stream);
}

bool weight_grad_takes(int dtype, const LinearArgs &a) {
  const int64_t size = dtype == 0 ? 4 : 2, vec = 16 / size;
  const int64_t runs = a.N * (int64_t)((a.K + 63) / 64);  // workgroups that add up the parts
  return a.K % vec == 0 && a.N % vec == 0 && a.rows < 1LL << 30 && std::max(a.K, a.N) * size * 64 <= 1LL << 28 &&
         runs < 1 << 23;
}

// Few rows of 16 bits keep gz in fp32, and their products meet in fp32 (any_kernel), without the weight's turning.
// The whole backward of 4 x 2,048 x 8,192 takes 105 us, of 17 rows by the kernels for more 217; of 4 x 256 x 512 26
// and 23, which is why more rows than one product of 16 take the others.
constexpr int64_t kWideRows = 16;
bool keeps_wide(int dtype, const LinearArgs &a) { return dtype != 0 && a.act != kActNone && a.rows <= kWideRows; }
// More rows of 16 bits keep gz in two values where a slope has made it longer than gy (SiLU, GELU): rounded to one,
// gx and gW were off by two roundings (bf16 0.00235 relative, 0.00166 with two values, as from 64 bits).
// The backward of 40,000 x 256 x 512 takes 114 us where the rounded one took 89, of 8,192 x 2,048 x 8,192 1,313
// and 831 (the products have twice the terms); ReLU's gz has gy's bits and stays one value.
int halves_of(int dtype, const LinearArgs &a) {
  return dtype != 0 && (a.act == kActSilu || a.act == kActGelu) && !keeps_wide(dtype, a) ? 2 : 1;
}

// Workspace of the backward: gz, the bias' parts, then what the products take.
struct BackWs {
  int64_t part, product, total;
};
BackWs back_ws(int dtype, const LinearArgs &a) {
  const int64_t size = dtype == 0 ? 4 : 2;
  BackWs w;
  const int halves = halves_of(dtype, a);
  w.part = a.act != kActNone ? up(a.rows * a.N * (keeps_wide(dtype, a) ? 4 : size * halves)) : 0;
  w.product = w.part + up((int64_t)sum_blocks(a.rows, a.N) * a.N * 4);
  int64_t grad_w = any_bytes(a.N, a.K, a.rows);
  if (weight_grad_takes(dtype, a)) grad_w = std::max(grad_w, weight_grad_workspace_bytes(dtype, a.rows, a.K, 1, a.N, halves));
  for (bool aligned : {false, true}) grad_w = std::max(grad_w, product_bytes(dtype, true, a.rows, a.K, a.N, aligned, halves));
  w.total = w.product + up(grad_w);
  return w;
}

template <typename T>
hipError_t backward(int dtype, const LinearArgs &a, const void *grad_y, const void *slope, void *workspace, void *grad_x,
                    void *grad_w, void *grad_b, hipStream_t stream) {
  const BackWs ws = back_ws(dtype, a);
  char *base = static_cast<char *>(workspace);
  const T *gy = static_cast<const T *>(grad_y), *gz = gy, *x = static_cast<const T *>(a.x);
  const T *weight = static_cast<const T *>(a.weight);
  float *part = grad_b != nullptr ? reinterpret_cast<float *>(base + ws.part) : nullptr;
  if (keeps_wide(dtype, a)) {
    float *wide = reinterpret_cast<float *>(base);
    if (hipError_t e = launch_grad_z<false>(gy, static_cast<const T *>(slope), wide, a.act, a.rows, a.N, part, stream)) return e;
    if (hipError_t e = launch_turn<T>(part, a.rows, grad_b, a.bias_wide, a, 0, nullptr, stream)) return e;
    Epilogue e{nullptr, nullptr, grad_x, nullptr, false, kActNone, a.K};
    if (grad_x != nullptr)
      if (hipError_t err = launch_any<T>(wide, a.N, 1, weight, 1, a.K, a.rows, a.N, e, base + ws.product, stream)) return err;
    e.y = grad_w;
    if (grad_w == nullptr) return hipSuccess;
    return launch_any<T>(wide, 1, a.N, x, 1, a.K, a.N, a.rows, e, base + ws.product, stream);
  }
  const int halves = halves_of(dtype, a);
  if (a.act != kActNone) gz = reinterpret_cast<T *>(base);
  if (a.act != kActNone || grad_b != nullptr) {
    const T *s = static_cast<const T *>(slope);
    hipError_t e = hipErrorInvalidValue;
    if constexpr (sizeof(T) == 2)
      if (halves == 2) e = launch_grad_z<true>(gy, s, const_cast<T *>(gz), a.act, a.rows, a.N, part, stream);
    if (halves == 1) e = launch_grad_z<false>(gy, s, const_cast<T *>(gz), a.act, a.rows, a.N, part, stream);
    if (e != hipSuccess) return e;
  }
  const bool turn = grad_x != nullptr && route(gz, weight, true, a.rows, a.K, (int64_t)a.N * halves) == kRows;
  if (hipError_t e = launch_turn<T>(part, a.rows, grad_b, a.bias_wide, a, turn ? halves : 0, base + ws.product, stream)) return e;
  if (grad_x != nullptr) {
    const Epilogue e{nullptr, nullptr, grad_x, nullptr, false, kActNone, a.K};
    if (hipError_t err = product<T>(gz, weight, true, a.rows, a.N, e, base + ws.product, stream, halves)) return err;
  }
  if (grad_w == nullptr) return hipSuccess;
  if (weight_grad_takes(dtype, a) && on_16({gz, x}))
    return launch_weight_grad(dtype, x, gz, a.rows, a.K, 1, a.N, base + ws.product, dtype, grad_w, stream, halves);
  const Epilogue e{nullptr, nullptr, grad_w, nullptr, false, kActNone, a.K};
  return launch_any<T>(gz, 1, (int64_t)a.N * halves, x, 1, a.K, a.N, a.rows, e, base + ws.product, stream, halves, a.N);
}

}  // namespace

int64_t linear_forward_workspace_bytes(int dtype, const LinearArgs &a, bool aligned) {
  return product_bytes(dtype, false, a.rows, a.N, a.K, aligned);
}
bool linear_aligned(const LinearArgs &a) { return on_16({a.x, a.weight}); }

hipError_t launch_linear_forward(int dtype, const LinearArgs &a, const void *residual, void *y, void *slope, void *workspace,
                                 hipStream_t stream) {
  switch (dtype) {
    case 0: return forward<float>(a, residual, y, slope, workspace, stream);
    case 1: return forward<f16>(a, residual, y, slope, workspace, stream);
    default: return forward<bf16>(a, residual, y, slope, workspace, stream);
  }
}

int64_t linear_backward_workspace_bytes(int dtype, const LinearArgs &a) { return back_ws(dtype, a).total; }

hipError_t launch_linear_backward(int dtype, const LinearArgs &a, const void *grad_y, const void *slope, void *workspace,
                                  void *grad_x, void *grad_w, void *grad_b, hipStream_t stream) {
  switch (dtype) {
    case 0: return backward<float>(dtype, a, grad_y, slope, workspace, grad_x, grad_w, grad_b, stream);
    case 1: return backward<f16>(dtype, a, grad_y, slope, workspace, grad_x, grad_w, grad_b, stream);
    default: return backward<bf16>(dtype, a, grad_y, slope, workspace, grad_x, grad_w, grad_b, stream);
  }
}

}  // namespace bevk
