// The gradients of the residual norm (gfx950; residual_norm_fwd.hip has the formulas and names).
//
//   hh = (h - mean) rstd, t = gy w
//   gh = rstd (t - mean(t) - hh mean(t hh)) + gs          (rms: without mean(t)); the residual's too
//   gw = sum gy hh, gb = sum gy, ggate = scale sum gh p   over the rows (a set's rows)
//   gp = scale gate gh; without the block's norm the block's gradient gx = gp, else
//   gbw = sum gp ph, gbb = sum gp, u = gp bw, gx = rstd_x (u - mean(u) - ph mean(u ph))
//
// The row in registers as in the forward; h is computed again from x and the residual with the forward's means
// and spreads, to the same bits (read as it was written, rounded, it would be off by half a step of h where hh is
// small next to it, for as many bytes in most cases). A workgroup takes a range of rows and keeps its threads'
// part of the parameters' sums in registers; at its end (for the gate: at the end of a set) they are
// added over its rows in LDS and written to the workspace, and join_kernel adds up the workgroups' parts
// in order: no atomics, the same results on every run.
//
// Rows of more than 512 vectors of 16 bits or 1,024 of fp32 (4,096 channels) take two passes, rows_kernel and sums_kernel:
// 10 tensors read or written for 6, and no scratch memory. 4,096 x 8,192 bf16 with both norms 200 us (479 in one
// pass), 2,048 x 16,384 198 (796), without the block's norm 155 (211 and 488); 2,048 x 8,192 fp32 161 (371).
// Bound by memory and by what a thread can have in flight beside its sums (a row ahead, two or three waves a
// SIMD): 16,384 x 2,048 bf16 with both norms 336 MB in 80 us (4.2 TB/s; a workgroup a row and no prefetch
// 147 us), 34,800 x 512 fp16 178 MB in 38 us (4.7), and 5 to 6 us for the parts' sums.
#include "residual_norm.h"

namespace bevk {
namespace {
using namespace rnorm;

// Rows that take two passes: 1,024 threads have 128 registers each, and one with 8 values or more of every sum, parameter
// and tensor has no room for them (up to 524 of them went through scratch memory).
constexpr bool in_two_passes(int tpr, int values) { return tpr == 1024 && values >= 8; }

// Workgroups on the chip at a time: what a thread keeps leaves room for two or three waves a SIMD (four of 1,024 threads:
// 4,096 x 4,096 fp32 with both norms 96 us on all CUs, 114 on half of them).
constexpr int parts_at_most(int tpr) { return tpr <= 64 ? 768 : std::max(256, 512 * 256 / threads_of(tpr)); }

template <typename T, int V>
__device__ __forceinline__ void buffer_store(__amdgpu_buffer_rsrc_t r, uint32_t off, const Vec<T, V> &y) {
  typedef int int4v __attribute__((ext_vector_type(4)));
  if constexpr (sizeof(y) == 16) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(int4v, y), r, off, 0, 0);
  else if constexpr (sizeof(y) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, y), r, off, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, y), r, off, 0, 0);
}

// Workgroup k: `per` parts of a set (sets split), or whole sets (per == 1).
struct Split {
  int64_t sets, set_rows;
  int per, blocks;
};
Split split_of(const ResidualNormArgs &a, int rows_a_block, int64_t most_blocks) {
  Split s;
  s.set_rows = a.set_rows > 0 ? a.set_rows : a.rows;
  s.sets = a.rows / s.set_rows;
  const int64_t most = std::max<int64_t>(1, s.set_rows / (rows_a_block * 2));  // two rows a thread at least
  s.per = (int)std::max<int64_t>(1, std::min<int64_t>(most_blocks / std::min(s.sets, most_blocks), most));
  s.blocks = (int)(s.per > 1 ? s.sets * s.per : std::min(s.sets, most_blocks));
  return s;
}

// Parts in the workspace: [4][blocks][channels] of weight, bias, block weight, block bias (those that
// are wanted), then the gate's [sets][per][channels].
struct Parts {
  float *sum[4], *gate;
  float *means;  // two passes: [rows][2] mean(t) (rms: 0) and mean(t hh); or null where no sums are wanted
};

template <typename T, int V, int TPR, int L, bool BLOCK>
__global__ void __launch_bounds__(threads_of(TPR)) backward_kernel(const ResidualNormArgs a, const ResidualNormGrads g,
                                                                   const Split sp, const Parts parts) {
  constexpr int THREADS = threads_of(TPR), R = THREADS / TPR, N = BLOCK ? 5 : 3;
  __shared__ float s[2 * THREADS / 64 * 2];
  __shared__ float joined[R > 1 ? THREADS * L * V : 1];
  int turn = 0;
  const int j = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int64_t set0 = sp.per > 1 ? blockIdx.x / sp.per : sp.sets * blockIdx.x / sp.blocks;
  const int64_t set1 = sp.per > 1 ? set0 + 1 : sp.sets * (blockIdx.x + 1) / sp.blocks;
  const int part = sp.per > 1 ? blockIdx.x % sp.per : 0;
  float sum[N][L][V];  // gate, weight, bias, block weight, block bias
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int e = 0; e < V; ++e) sum[n][l][e] = 0.f;
  // Rows from r on through a buffer that ends with the part's rows or 2 GiB on, and at nothing where there is no
  // such tensor: past that a load gives zeros and a store does nothing. So nothing branches around them, and
  // the next row's loads stay in flight over this row's stores, which count as they do.
  auto left = [&](int64_t r, int64_t r1) __attribute__((always_inline)) {
    const int64_t bytes = (r1 - r) * a.channels * (int64_t)sizeof(T);
    return bytes < (int64_t)1 << 31 ? (uint32_t)bytes : 1u << 31;
  };
  uint32_t off[L];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const int c = (l * TPR + j) * V;
    off[l] = c < a.channels ? (uint32_t)(group * a.channels + c) * sizeof(T) : 0xffffff00u;
  }
  Vec<T, V> next[4][L];
  auto load = [&](int64_t r, int64_t r1) __attribute__((always_inline)) {
    const uint32_t bytes = left(r, r1);
    const void *from[4] = {g.grad_y, a.x, g.grad_h, a.residual};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const __amdgpu_buffer_rsrc_t b = make_rsrc(static_cast<const T *>(from[n]) + r * a.channels, from[n] != nullptr ? bytes : 0);
#pragma unroll
      for (int l = 0; l < L; ++l) {
        if constexpr (V == 1) next[n][l].v[0] = buffer_load_one<T>(b, off[l]);
        else next[n][l] = buffer_load_vec<T, V>(b, off[l]);
      }
    }
  };
  Vec<float, BLOCK ? 4 : 2> st_next;
  auto load_stats = [&](int64_t r) __attribute__((always_inline)) {  // of row r + group or, past the end, the last one
    st_next = load_vec<float, BLOCK ? 4 : 2>(g.stats + min(r + group, sp.sets * sp.set_rows - 1) * (BLOCK ? 4 : 2));
  };
  auto store = [&](void *to, int64_t r, uint32_t bytes, const float (&v)[L][V]) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t b = make_rsrc(static_cast<T *>(to) + r * a.channels, to != nullptr ? bytes : 0);
#pragma unroll
    for (int l = 0; l < L; ++l) {
      Vec<T, V> y;
#pragma unroll
      for (int e = 0; e < V; ++e) y.v[e] = static_cast<T>(v[l][e]);
      buffer_store(b, off[l], y);
    }
  };
  // the workgroup's sum of one parameter's parts, in the order of its rows
  auto write = [&](float (&x)[L][V], float *to) __attribute__((always_inline)) {
    if constexpr (R > 1) {
      __syncthreads();
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e) joined[(group * L + l) * TPR * V + j * V + e] = x[l][e];
      __syncthreads();
      for (int i = threadIdx.x; i < L * TPR * V; i += THREADS) {
        float v = joined[i];
#pragma unroll
        for (int k = 1; k < R; ++k) v += joined[k * L * TPR * V + i];
        if (i < a.channels) to[i] = v;
      }
    } else {
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const int c = (l * TPR + j) * V;
        if (c < a.channels)
#pragma unroll
          for (int e = 0; e < V; ++e) to[c + e] = x[l][e];
      }
    }
  };
  const float inv = 1.f / (float)a.channels;
  // the parameters stay in registers: read again for each row they came late, in the middle of its sums
  float w[L][V], gate[L][V], bw[BLOCK ? L : 1][V], bb[BLOCK ? L : 1][V];
#pragma unroll
  for (int l = 0; l < L; ++l) {
    const int c = (l * TPR + j) * V;
    if (c >= a.channels) continue;
    load_param<T, V>(a.weight, a.wide, c, 1.f, w[l]);
    if constexpr (BLOCK) {
      load_param<T, V>(a.block_weight, a.wide, c, 1.f, bw[l]);
      load_param<T, V>(a.block_bias, a.wide, c, 0.f, bb[l]);
    }
  }
  for (int64_t set = set0; set < set1; ++set) {
    const int64_t r0 = set * sp.set_rows + sp.set_rows * part / sp.per;
    const int64_t r1 = set * sp.set_rows + sp.set_rows * (part + 1) / sp.per;
    const int64_t gate_at = a.set_rows > 0 ? set * a.channels : 0;
#pragma unroll
    for (int l = 0; l < L; ++l)
      if ((l * TPR + j) * V < a.channels) load_param<T, V>(a.gate, a.gate_wide, gate_at + (l * TPR + j) * V, 1.f, gate[l]);
    load(r0, r1);
    load_stats(r0);
    for (int64_t r = r0; r < r1; r += R) {
      float gy[L][V], h[L][V], x[L][V], gs[L][V];
      bool in[L];
#pragma unroll
      for (int l = 0; l < L; ++l) {
        in[l] = r + group < r1 && (l * TPR + j) * V < a.channels;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          gy[l][e] = (float)next[0][l].v[e];
          x[l][e] = (float)next[1][l].v[e];
          gs[l][e] = (float)next[2][l].v[e];
          h[l][e] = (float)next[3][l].v[e];
        }
      }
      const uint32_t here = left(r, r1);
      load(min(r + R, r1), r1);
      const Vec<float, BLOCK ? 4 : 2> st = st_next;
      load_stats(min(r + R, r1 - 1));
      const float mean = st.v[0], rstd = st.v[1];
      float t[2] = {0.f, 0.f};
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (in[l]) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float p = x[l][e];
            if constexpr (BLOCK) {
              x[l][e] = (p - st.v[2]) * st.v[3];  // ph
              p = __builtin_fmaf(x[l][e], bw[l][e], bb[l][e]);
            }
            const float hh = (stream_value(p, a.scale, gate[l][e], h[l][e]) - mean) * rstd;
            sum[1][l][e] = __builtin_fmaf(gy[l][e], hh, sum[1][l][e]);
            sum[2][l][e] += gy[l][e];
            h[l][e] = hh;
            gy[l][e] *= w[l][e];
            t[0] += gy[l][e];
            t[1] = __builtin_fmaf(gy[l][e], hh, t[1]);
          }
        }
      row_sums<TPR, THREADS, 2>(t, s, turn);
      const float c1 = a.rms ? 0.f : t[0] * inv, c2 = t[1] * inv;
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e)
          gs[l][e] = __builtin_fmaf(rstd, gy[l][e] - c1 - h[l][e] * c2, gs[l][e]);  // gh
      t[0] = t[1] = 0.f;
      store(g.grad_residual, r, here, gs);
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (in[l]) {
          if constexpr (BLOCK) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float ph = x[l][e], gh = a.scale * gs[l][e], gp = gate[l][e] * gh;
              sum[0][l][e] = __builtin_fmaf(gh, __builtin_fmaf(ph, bw[l][e], bb[l][e]), sum[0][l][e]);
              sum[3][l][e] = __builtin_fmaf(gp, ph, sum[3][l][e]);
              sum[4][l][e] += gp;
              gs[l][e] = gp * bw[l][e];
              t[0] += gs[l][e];
              t[1] = __builtin_fmaf(gs[l][e], ph, t[1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float gh = a.scale * gs[l][e];
              sum[0][l][e] = __builtin_fmaf(gh, x[l][e], sum[0][l][e]);
              gs[l][e] = gate[l][e] * gh;
            }
          }
        }
      if constexpr (BLOCK) {
        row_sums<TPR, THREADS, 2>(t, s, turn);
        const float d1 = a.rms ? 0.f : t[0] * inv, d2 = t[1] * inv;
#pragma unroll
        for (int l = 0; l < L; ++l)
#pragma unroll
          for (int e = 0; e < V; ++e) gs[l][e] = st.v[3] * (gs[l][e] - d1 - x[l][e] * d2);
      }
      store(g.grad_x, r, here, gs);
    }
    if (parts.gate != nullptr) {
      write(sum[0], parts.gate + (set * sp.per + part) * a.channels);
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e) sum[0][l][e] = 0.f;
    }
  }
#pragma unroll
  for (int n = 1; n < N; ++n)
    if (parts.sum[n - 1] != nullptr) write(sum[n], parts.sum[n - 1] + (int64_t)blockIdx.x * a.channels);
}

// The first pass over long rows: the rows' own gradients. A workgroup takes a row at a time, whose four tensors stay in
// registers as they were loaded; what is computed from them is computed again behind each sum, with the parameters
// from the L2.
template <typename T, int V, int L, bool BLOCK>
__global__ void __launch_bounds__(1024) rows_kernel(const ResidualNormArgs a, const ResidualNormGrads g, float *means) {
  __shared__ float s[2 * 1024 / 64 * 2];
  int turn = 0;
  const int64_t r0 = a.rows * blockIdx.x / gridDim.x, r1 = a.rows * (blockIdx.x + 1) / gridDim.x;
  const float inv = 1.f / (float)a.channels;
  const uint32_t bytes = (uint32_t)a.channels * sizeof(T);
  uint32_t off[L];
#pragma unroll
  for (int l = 0; l < L; ++l) off[l] = (uint32_t)(l * 1024 + threadIdx.x) * V * sizeof(T);  // (past a row's end: nothing)
  typedef int int4v __attribute__((ext_vector_type(4)));
  int4v now[4][L], next[4][L];  // 16 bytes of the gradient of y, x, the gradient of the stream, the residual
  auto value = [&](int n, int l, int e) __attribute__((always_inline)) {
    return (float)__builtin_bit_cast(Vec<T, V>, now[n][l]).v[e];
  };
  auto load = [&](int64_t r) __attribute__((always_inline)) {
    const void *from[4] = {g.grad_y, a.x, g.grad_h, a.residual};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const __amdgpu_buffer_rsrc_t b = make_rsrc(static_cast<const T *>(from[n]) + r * a.channels, from[n] != nullptr ? bytes : 0);
#pragma unroll
      for (int l = 0; l < L; ++l) next[n][l] = __builtin_bit_cast(int4v, buffer_load_vec<T, V>(b, off[l]));
    }
  };
  constexpr bool AHEAD = L == 1;
  if constexpr (AHEAD) load(r0);
  for (int64_t r = r0; r < r1; ++r) {
    if constexpr (!AHEAD) load(r);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int l = 0; l < L; ++l) now[n][l] = next[n][l];
    if constexpr (AHEAD) load(min(r + 1, r1 - 1));
    const Vec<float, BLOCK ? 4 : 2> st = load_vec<float, BLOCK ? 4 : 2>(g.stats + r * (BLOCK ? 4 : 2));
    const int64_t gate_at = a.set_rows > 0 ? r / a.set_rows * a.channels : 0;
    // f(value, t = gy w, hh, ph, scale * gate, bw) for each value of vector l that there is
    auto each = [&](int l, auto f) __attribute__((always_inline)) {
      // (to the compiler new values, and parameters that may have changed: what it computes from them twice it would
      // keep, and that does not fit)
#pragma unroll
      for (int n = 0; n < 4; ++n) asm volatile("" : "+v"(now[n][l]));
      asm volatile("" ::: "memory");
      const int c = (l * 1024 + (int)threadIdx.x) * V;
      if (c >= a.channels) return;
      float w[V], gate[V], bw[V], bb[V];
      load_param<T, V>(a.weight, a.wide, c, 1.f, w);
      load_param<T, V>(a.gate, a.gate_wide, gate_at + c, 1.f, gate);
      if constexpr (BLOCK) {
        load_param<T, V>(a.block_weight, a.wide, c, 1.f, bw);
        load_param<T, V>(a.block_bias, a.wide, c, 0.f, bb);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float p = value(1, l, e), ph = 0.f;
        if constexpr (BLOCK) {
          ph = (p - st.v[2]) * st.v[3];
          p = __builtin_fmaf(ph, bw[e], bb[e]);
        }
        const float hh = (stream_value(p, a.scale, gate[e], value(3, l, e)) - st.v[0]) * st.v[1];
        f(e, value(0, l, e) * w[e], hh, ph, gate[e], BLOCK ? bw[e] : 1.f);
      }
    };
    auto store = [&](void *to, int l, const float (&v)[V]) __attribute__((always_inline)) {
      Vec<T, V> y;
#pragma unroll
      for (int e = 0; e < V; ++e) y.v[e] = static_cast<T>(v[e]);
      buffer_store(make_rsrc(static_cast<T *>(to) + r * a.channels, to != nullptr ? bytes : 0), off[l], y);
    };
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int l = 0; l < L; ++l)
      each(l, [&](int, float u, float hh, float, float, float) __attribute__((always_inline)) {
        t[0] += u;
        t[1] = __builtin_fmaf(u, hh, t[1]);
      });
    row_sums<1024, 1024, 2>(t, s, turn);
    const float c1 = a.rms ? 0.f : t[0] * inv, c2 = t[1] * inv;
    if (threadIdx.x == 0 && means != nullptr) {
      means[r * 2] = c1;
      means[r * 2 + 1] = c2;
    }
    auto grad_stream = [&](int l, int e, float u, float hh) __attribute__((always_inline)) {
      return __builtin_fmaf(st.v[1], u - c1 - hh * c2, value(2, l, e));
    };
    t[0] = t[1] = 0.f;
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float gr[V], gx[V];
      each(l, [&](int e, float u, float hh, float ph, float gate, float bw) __attribute__((always_inline)) {
        gr[e] = grad_stream(l, e, u, hh);
        gx[e] = gate * (a.scale * gr[e]);
        if constexpr (BLOCK) {
          const float v = gx[e] * bw;
          t[0] += v;
          t[1] = __builtin_fmaf(v, ph, t[1]);
        }
      });
      store(g.grad_residual, l, gr);
      if constexpr (!BLOCK) store(g.grad_x, l, gx);
    }
    if constexpr (BLOCK) {
      row_sums<1024, 1024, 2>(t, s, turn);
      const float d1 = a.rms ? 0.f : t[0] * inv, d2 = t[1] * inv;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        float gx[V];
        each(l, [&](int e, float u, float hh, float ph, float gate, float bw) __attribute__((always_inline)) {
          gx[e] = st.v[3] * (gate * (a.scale * grad_stream(l, e, u, hh)) * bw - d1 - ph * d2);
        });
        store(g.grad_x, l, gx);
      }
    }
  }
}

// The parameters' sums of long rows, in a second pass: a thread has V channels of a part's rows, one after another, with
// the means over each row that the first pass found. No sum over a row, so no wait between two of them.
template <typename T, int V, bool BLOCK>
__global__ void __launch_bounds__(256) sums_kernel(const ResidualNormArgs a, const ResidualNormGrads g, const Split sp,
                                                   const Parts parts) {
  const int c = (int)(blockIdx.y * 256 + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int64_t set0 = sp.per > 1 ? blockIdx.x / sp.per : sp.sets * blockIdx.x / sp.blocks;
  const int64_t set1 = sp.per > 1 ? set0 + 1 : sp.sets * (blockIdx.x + 1) / sp.blocks;
  const int part = sp.per > 1 ? blockIdx.x % sp.per : 0;
  const T *from[4] = {static_cast<const T *>(g.grad_y) + c, static_cast<const T *>(a.x) + c,
                      g.grad_h != nullptr ? static_cast<const T *>(g.grad_h) + c : nullptr,
                      a.residual != nullptr ? static_cast<const T *>(a.residual) + c : nullptr};
  constexpr int N = BLOCK ? 5 : 3, S = BLOCK ? 4 : 2;
  float sum[N][V], w[V], gate[V], bw[V], bb[V];  // gate, weight, bias, block weight, block bias
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int e = 0; e < V; ++e) sum[n][e] = 0.f;
  load_param<T, V>(a.weight, a.wide, c, 1.f, w);
  if constexpr (BLOCK) {
    load_param<T, V>(a.block_weight, a.wide, c, 1.f, bw);
    load_param<T, V>(a.block_bias, a.wide, c, 0.f, bb);
  }
  auto write = [&](const float (&v)[V], float *to) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < V; ++e) to[c + e] = v[e];
  };
  for (int64_t set = set0; set < set1; ++set) {
    const int64_t r0 = set * sp.set_rows + sp.set_rows * part / sp.per;
    const int64_t r1 = set * sp.set_rows + sp.set_rows * (part + 1) / sp.per;
    load_param<T, V>(a.gate, a.gate_wide, (a.set_rows > 0 ? set * a.channels : 0) + c, 1.f, gate);
    Vec<T, V> next[4];
    auto load = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        next[n] = from[n] != nullptr ? load_vec<T, V>(from[n] + r * a.channels) : Vec<T, V>{};
    };
    load(r0);
    for (int64_t r = r0; r < r1; ++r) {
      const Vec<float, S> st = load_vec<float, S>(g.stats + r * S);
      const Vec<float, 2> means = load_vec<float, 2>(parts.means + r * 2);
      Vec<T, V> now[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) now[n] = next[n];
      load(min(r + 1, r1 - 1));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gy = (float)now[0].v[e];
        float p = (float)now[1].v[e], ph = 0.f;
        if constexpr (BLOCK) {
          ph = (p - st.v[2]) * st.v[3];
          p = __builtin_fmaf(ph, bw[e], bb[e]);
        }
        const float hh = (stream_value(p, a.scale, gate[e], (float)now[3].v[e]) - st.v[0]) * st.v[1];
        const float gh = a.scale * __builtin_fmaf(st.v[1], gy * w[e] - means.v[0] - hh * means.v[1], (float)now[2].v[e]);
        sum[0][e] = __builtin_fmaf(gh, p, sum[0][e]);
        sum[1][e] = __builtin_fmaf(gy, hh, sum[1][e]);
        sum[2][e] += gy;
        if constexpr (BLOCK) {
          const float gp = gate[e] * gh;
          sum[3][e] = __builtin_fmaf(gp, ph, sum[3][e]);
          sum[4][e] += gp;
        }
      }
    }
    if (parts.gate != nullptr) {
      write(sum[0], parts.gate + (set * sp.per + part) * a.channels);
#pragma unroll
      for (int e = 0; e < V; ++e) sum[0][e] = 0.f;
    }
  }
#pragma unroll
  for (int n = 1; n < N; ++n)
    if (parts.sum[n - 1] != nullptr) write(sum[n], parts.sum[n - 1] + (int64_t)blockIdx.x * a.channels);
}

// Any row length: a workgroup a row at a time, each sum a pass over it; a thread adds its channels' parts
// up in the workspace.
template <typename T, bool BLOCK>
__global__ void __launch_bounds__(256) any_backward_kernel(const ResidualNormArgs a, const ResidualNormGrads g,
                                                           const Split sp, const Parts parts) {
  __shared__ float s[2 * 4 * 2];
  int turn = 0;
  const int64_t set0 = sp.per > 1 ? blockIdx.x / sp.per : sp.sets * blockIdx.x / sp.blocks;
  const int64_t set1 = sp.per > 1 ? set0 + 1 : sp.sets * (blockIdx.x + 1) / sp.blocks;
  const int part = sp.per > 1 ? blockIdx.x % sp.per : 0;
  const float inv = 1.f / (float)a.channels;
  const int64_t mine = (int64_t)blockIdx.x * a.channels;
  for (int n = 0; n < 4; ++n)
    if (parts.sum[n] != nullptr)
      for (int c = threadIdx.x; c < a.channels; c += 256) parts.sum[n][mine + c] = 0.f;
  for (int64_t set = set0; set < set1; ++set) {
    const int64_t r0 = set * sp.set_rows + sp.set_rows * part / sp.per;
    const int64_t r1 = set * sp.set_rows + sp.set_rows * (part + 1) / sp.per;
    const int64_t gate_at = a.set_rows > 0 ? set * a.channels : 0;
    float *gate_sum = parts.gate == nullptr ? nullptr : parts.gate + (set * sp.per + part) * a.channels;
    if (gate_sum != nullptr)
      for (int c = threadIdx.x; c < a.channels; c += 256) gate_sum[c] = 0.f;
    for (int64_t row = r0; row < r1; ++row) {
      const int64_t at = row * a.channels;
      const T *gy = static_cast<const T *>(g.grad_y) + at, *x = static_cast<const T *>(a.x) + at;
      const T *res = a.residual == nullptr ? nullptr : static_cast<const T *>(a.residual) + at;
      const T *gs = g.grad_h == nullptr ? nullptr : static_cast<const T *>(g.grad_h) + at;
      const float *st = g.stats + row * (BLOCK ? 4 : 2);
      const float mean = st[0], rstd = st[1], mean_x = BLOCK ? st[2] : 0.f, rstd_x = BLOCK ? st[3] : 1.f;
      float t[2] = {0.f, 0.f}, w[1], b[1], gate[1];
      auto normed = [&](int c) __attribute__((always_inline)) {  // hh
        float p = (float)x[c];
        if (BLOCK) {
          load_param<T, 1>(a.block_weight, a.wide, c, 1.f, w);
          load_param<T, 1>(a.block_bias, a.wide, c, 0.f, b);
          p = block_value(p, mean_x, rstd_x, w[0], b[0]);
        }
        load_param<T, 1>(a.gate, a.gate_wide, gate_at + c, 1.f, gate);
        return (stream_value(p, a.scale, gate[0], res != nullptr ? (float)res[c] : 0.f) - mean) * rstd;
      };
      for (int c = threadIdx.x; c < a.channels; c += 256) {
        const float hh = normed(c);
        load_param<T, 1>(a.weight, a.wide, c, 1.f, w);
        const float v = (float)gy[c] * w[0];
        t[0] += v;
        t[1] = __builtin_fmaf(v, hh, t[1]);
      }
      row_sums<256, 256, 2>(t, s, turn);
      const float c1 = a.rms ? 0.f : t[0] * inv, c2 = t[1] * inv;
      auto grad_stream = [&](int c, float hh) __attribute__((always_inline)) {
        load_param<T, 1>(a.weight, a.wide, c, 1.f, w);
        return __builtin_fmaf(rstd, (float)gy[c] * w[0] - c1 - hh * c2, gs != nullptr ? (float)gs[c] : 0.f);
      };
      auto grad_block = [&](int c, float gh) __attribute__((always_inline)) {
        load_param<T, 1>(a.gate, a.gate_wide, gate_at + c, 1.f, gate);
        return gate[0] * (a.scale * gh);
      };
      t[0] = t[1] = 0.f;
      if (BLOCK)
        for (int c = threadIdx.x; c < a.channels; c += 256) {
          const float hh = normed(c), gp = grad_block(c, grad_stream(c, hh));
          load_param<T, 1>(a.block_weight, a.wide, c, 1.f, w);
          const float ph = ((float)x[c] - mean_x) * rstd_x, u = gp * w[0];
          t[0] += u;
          t[1] = __builtin_fmaf(u, ph, t[1]);
        }
      if (BLOCK) row_sums<256, 256, 2>(t, s, turn);
      const float d1 = a.rms ? 0.f : t[0] * inv, d2 = t[1] * inv;
      for (int c = threadIdx.x; c < a.channels; c += 256) {
        const float hh = normed(c), dy = (float)gy[c];
        const float gh = grad_stream(c, hh), gp = grad_block(c, gh);
        if (parts.sum[0] != nullptr) parts.sum[0][mine + c] += dy * hh;
        if (parts.sum[1] != nullptr) parts.sum[1][mine + c] += dy;
        float p = (float)x[c], gx = gp;
        if (BLOCK) {
          const float ph = (p - mean_x) * rstd_x;
          load_param<T, 1>(a.block_weight, a.wide, c, 1.f, w);
          load_param<T, 1>(a.block_bias, a.wide, c, 0.f, b);
          p = __builtin_fmaf(ph, w[0], b[0]);
          if (parts.sum[2] != nullptr) parts.sum[2][mine + c] += gp * ph;
          if (parts.sum[3] != nullptr) parts.sum[3][mine + c] += gp;
          gx = rstd_x * (gp * w[0] - d1 - ph * d2);
        }
        if (gate_sum != nullptr) gate_sum[c] += a.scale * gh * p;
        if (g.grad_residual != nullptr) static_cast<T *>(g.grad_residual)[at + c] = static_cast<T>(gh);
        if (g.grad_x != nullptr) static_cast<T *>(g.grad_x)[at + c] = static_cast<T>(gx);
      }
    }
  }
}

struct Join {
  const float *from;
  void *to;
  int parts;      // to add up for each output row
  int64_t rows;   // output rows
  bool wide;
};
struct Joins {
  Join of[5];
  int count, channels;
};

// 16 channels of one output row: 64 threads add up every 64th part each, then in order.
template <typename T>
__global__ void __launch_bounds__(1024) join_kernel(const Joins all, int64_t first) {
  __shared__ float s[64][17];
  const int64_t tiles = (all.channels + 15) / 16, at = first + blockIdx.x;
  const int which = (int)min(at / tiles, (int64_t)all.count - 1);  // the last one may have several rows
  const Join &j = all.of[which];
  const int64_t row = at / tiles - which;
  const int c = (int)(at % tiles) * 16 + threadIdx.x % 16, k = threadIdx.x / 16;
  float v = 0.f;
  if (row < j.rows && c < all.channels) {
    const float *p = j.from + row * j.parts * all.channels + c;
#pragma unroll 8
    for (int q = k; q < j.parts; q += 64) v += p[(int64_t)q * all.channels];
  }
  s[k][threadIdx.x % 16] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (k < half) s[k][threadIdx.x % 16] += s[k + half][threadIdx.x % 16];
    __syncthreads();
  }
  if (k == 0 && row < j.rows && c < all.channels) {
    v = s[0][threadIdx.x];
    if (j.wide) static_cast<float *>(j.to)[row * all.channels + c] = v;
    else static_cast<T *>(j.to)[row * all.channels + c] = static_cast<T>(v);
  }
}

// The split of the sums for rows of vectors of v values, and whether they are a second pass.
struct Plan {
  Split split;
  bool two;
};
Plan plan(const ResidualNormArgs &a, int v) {
  int rows = 1;
  int64_t blocks = 1024;
  bool two = false;
  const int64_t vecs = (a.channels + v - 1) / v;
  for_row(vecs, [&](auto tpr, auto l) {
    constexpr int TPR = decltype(tpr)::value, L = decltype(l)::value;
    two = in_two_passes(TPR, v * L);
    rows = two ? 1 : threads_of(TPR) / TPR;
    blocks = two ? 512 / ((vecs + 255) / 256) : parts_at_most(TPR);  // (two workgroups of sums_kernel a CU)
  });
  return {split_of(a, rows, blocks), two};
}

template <typename T, int V, bool BLOCK>
hipError_t launch_v(const ResidualNormArgs &a, const ResidualNormGrads &g, const Split &sp, const Parts &parts,
                    hipStream_t stream) {
  const bool fits = for_row((a.channels + V - 1) / V, [&](auto tpr, auto l) {
    constexpr int TPR = decltype(tpr)::value, L = decltype(l)::value;
    if constexpr (in_two_passes(TPR, V * L)) {
      const int cus = std::max(1, device_cus());  // (a workgroup fills a CU)
      hipLaunchKernelGGL((rows_kernel<T, V, L, BLOCK>), dim3((unsigned)std::min<int64_t>(a.rows, cus)), dim3(1024), 0, stream,
                         a, g, parts.means);
      if (parts.means != nullptr)
        hipLaunchKernelGGL((sums_kernel<T, V, BLOCK>), dim3(sp.blocks, (unsigned)((a.channels / V + 255) / 256)), dim3(256), 0,
                           stream, a, g, sp, parts);
    } else {
      hipLaunchKernelGGL((backward_kernel<T, V, TPR, L, BLOCK>), dim3(sp.blocks), dim3(threads_of(TPR)), 0, stream, a,
                         g, sp, parts);
    }
  });
  if (!fits)
    hipLaunchKernelGGL((any_backward_kernel<T, BLOCK>), dim3(sp.blocks), dim3(256), 0, stream, a, g, sp, parts);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const ResidualNormArgs &a, const ResidualNormGrads &g, bool whole, void *workspace,
                    hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const Plan pl = plan(a, whole ? V : 1);
  const Split &sp = pl.split;
  float *ws = static_cast<float *>(workspace);
  Parts parts{};
  Joins joins{};
  joins.channels = a.channels;
  void *to[4] = {g.grad_weight, g.grad_bias, g.grad_block_weight, g.grad_block_bias};
  for (int n = 0; n < 4; ++n) {
    if (to[n] == nullptr) continue;
    parts.sum[n] = ws;
    joins.of[joins.count++] = Join{ws, to[n], sp.blocks, 1, a.wide};
    ws += (int64_t)sp.blocks * a.channels;
  }
  int64_t rows = joins.count;  // output rows of all
  if (g.grad_gate != nullptr) {
    parts.gate = ws;
    joins.of[joins.count++] = Join{ws, g.grad_gate, sp.per, sp.sets, a.gate_wide};
    rows += sp.sets;
    ws += sp.sets * sp.per * a.channels;
  }
  if (pl.two && joins.count > 0) parts.means = ws;
  hipError_t e;
  if (whole) e = a.block ? launch_v<T, V, true>(a, g, sp, parts, stream) : launch_v<T, V, false>(a, g, sp, parts, stream);
  else e = a.block ? launch_v<T, 1, true>(a, g, sp, parts, stream) : launch_v<T, 1, false>(a, g, sp, parts, stream);
  if (e != hipSuccess) return e;
  return launch_in_parts((a.channels + 15) / 16 * rows, 1024, [&](int64_t first, unsigned blocks) {
    hipLaunchKernelGGL((join_kernel<T>), dim3(blocks), dim3(1024), 0, stream, joins, first);
  });
}

bool whole_rows(int dtype, const ResidualNormArgs &a, const ResidualNormGrads &g) {
  return a.channels % (dtype == 0 ? 4 : 8) == 0 &&
         on_16({a.x, a.residual, a.weight, a.gate, a.block_weight, a.block_bias, g.grad_y, g.grad_h, g.grad_x, g.grad_residual});
}

}  // namespace

int64_t residual_norm_backward_workspace_bytes(int dtype, const ResidualNormArgs &a) {
  int64_t most = 0;  // for either alignment
  for (int v : {dtype == 0 ? 4 : 8, 1}) {
    const Plan pl = plan(a, v);
    most = std::max(most, (4 * (int64_t)pl.split.blocks + pl.split.sets * pl.split.per) * a.channels * 4 + (pl.two ? a.rows * 8 : 0));
  }
  return most;
}

hipError_t launch_residual_norm_backward(int dtype, const ResidualNormArgs &a, const ResidualNormGrads &g,
                                         void *workspace, hipStream_t stream) {
  const bool whole = whole_rows(dtype, a, g);
  switch (dtype) {
    case 0: return launch_t<float>(a, g, whole, workspace, stream);
    case 1: return launch_t<f16>(a, g, whole, workspace, stream);
    default: return launch_t<bf16>(a, g, whole, workspace, stream);
  }
}

}  // namespace bevk
