// Embedding rows by index with a scale, and the gradient of the table (gfx950).
//
//   out[t] = scale * W[i_t], zeros where i_t is outside [0, rows) (a padded place)
//   gW[v]  = scale * sum over t with i_t = v of g[t], in fp32 and in an order that does not change
//
// Both are bound by memory: a row read for a row written. The gradient's rows come sorted by index:
//   sort   one launch without a pass between workgroups: workgroup w of R (a power of two) owns the
//          rows v with v % R = w, so that frequent neighbours spread over workgroups, and reads all
//          indices, which cost it n * 8 bytes out of L2. It counts its rows' places, knows its part
//          of the sorted list from how many indices belong to workgroups before it, and writes
//          that part in the order of t.
//   sum    a group of lanes for each row of the table adds up its rows of g and writes the sum (or
//          zeros). Rows with more than kChunk places are left to workgroups for kChunk places of
//          the sorted list, which write partial sums, so that a row that many places share
//          does not hang on one group of lanes.
//   join   adds up the partial sums of those rows in the order of their chunks.
// 60,000 places of 40,000 rows of 256 fp16 (six cameras): sort 14.7 us, 8.5 of them reading the
// indices, sum 12, join 4; 16,384 tokens of 32,768 rows of 1,024 bf16, frequency as one over the
// rank: 8.6, 20 (4.9 TB/s) and 4. The lookup of 16,384 x 2,048 bf16 takes 17.6 us (5.1 TB/s).
#include <algorithm>

#include "bevk_launch.h"

namespace bevk {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRows = 512;  // counters of 16 waves: 32 KB
constexpr int kChunk = 32;      // (sums of the tokens above with 16 / 32 / 64: 21.6 / 20.8 / 23.4 us, cameras
                                // 12.5 / 12.0 / 11.7)

// N elements of T from memory aligned to them all together.
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T *p, float *v) {
  const Vec<T, N> x = load_vec<T, N>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (float)x.v[e];
}

// ---------------------------------------------------------------------------------------
// Lookup
// ---------------------------------------------------------------------------------------

// A workgroup takes kThreads * kUnroll vectors of the output in a row; the indices of a thread's
// vectors are all loaded before their rows, and those before any store.
constexpr int kUnroll = 4;
template <typename T, typename I, int N>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T *__restrict__ weight, int64_t rows,
                                                          uint32_t vecs, const I *__restrict__ index,
                                                          int64_t total, int64_t first, float scale,
                                                          T *__restrict__ out) {
  const int64_t base = (first + blockIdx.x) * (kThreads * kUnroll);
  const int64_t t0 = base / vecs;
  const uint32_t r0 = (uint32_t)(base - t0 * vecs);
  int64_t row[kUnroll];
  uint32_t col[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const uint32_t o = r0 + j * kThreads + threadIdx.x, t = o / vecs;
    col[j] = o - t * vecs;
    row[j] = base + j * kThreads + threadIdx.x < total ? (int64_t)index[t0 + t] : -1;
  }
  Vec<T, N> x[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    if (row[j] >= 0 && row[j] < rows) {
      x[j] = load_vec<T, N>(weight + (row[j] * vecs + col[j]) * N);
#pragma unroll
      for (int e = 0; e < N; ++e) x[j].v[e] = static_cast<T>((float)x[j].v[e] * scale);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[j].v[e] = static_cast<T>(0.f);
    }
  }
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    const int64_t k = base + j * kThreads + threadIdx.x;
    if (k < total) store_vec<T, N>(out + k * N, x[j]);
  }
}

// ---------------------------------------------------------------------------------------
// Gradient
// ---------------------------------------------------------------------------------------

// Places of the rows in the sorted list.
struct Sorted {
  int2 *span;    // [rows] first place and count
  int *order;    // [n] t of each place
  int *row;      // [n] row of each place
  int *valid;    // places in use
};

struct SortArgs {
  uint32_t n, rows, padding;  // padding: ~0 for none
  int log_r, per;             // rows v with v % R = w are a workgroup's; at most `per` of them
  uint32_t first;             // workgroups in the launches before (launch_in_parts)
};

// Lanes whose index is a row of this workgroup, or of one before it. An index is compared as unsigned
// numbers, so that negative ones are past the table too.
struct Owned {
  uint32_t row;
  bool mine, before;
};
template <bool PADDED, typename I>
__device__ __forceinline__ Owned owned(I index, const SortArgs &p, uint32_t w) {
  const uint32_t row = (uint32_t)index;
  bool there = row < p.rows;
  if constexpr (sizeof(I) == 8) there = there && (uint64_t)index >> 32 == 0;
  if constexpr (PADDED) there = there && row != p.padding;
  const uint32_t owner = row & ((1u << p.log_r) - 1);
  return {row, there && owner == w, there && owner < w};
}

// f(t of the wave's first lane, what its 64 indices are) over [begin, end), kScan times 64 of them
// loaded together and the rest by half of that; lanes past the end have no row.
constexpr int kScan = 8;
template <bool PADDED, typename I, typename F>
__device__ __forceinline__ void scan(const I *index, uint32_t begin, uint32_t end, const SortArgs &p, F f) {
  const uint32_t lane = threadIdx.x % kWave, w = p.first + blockIdx.x;
  uint32_t t = begin;
  const I *at = index + begin + lane;
  for (; t + kScan * kWave <= end; t += kScan * kWave, at += kScan * kWave) {
    I v[kScan];
#pragma unroll
    for (int j = 0; j < kScan; ++j) v[j] = at[j * kWave];
#pragma unroll
    for (int j = 0; j < kScan; ++j) f(t + j * kWave, owned<PADDED>(v[j], p, w));
  }
  for (; t < end; t += kScan / 2 * kWave) {
    I v[kScan / 2];
#pragma unroll
    for (int j = 0; j < kScan / 2; ++j) v[j] = index[min(t + j * kWave + lane, end - 1)];
#pragma unroll
    for (int j = 0; j < kScan / 2; ++j) {
      Owned o = owned<PADDED>(v[j], p, w);
      if (t + j * kWave + lane >= end) o.mine = o.before = false;
      f(t + j * kWave, o);
    }
  }
}

// Two passes over the indices' owners, one where no wave finds more than kKept of its workgroup's
// (n / (16 R) on average): those it keeps.
constexpr int kKept = 128;
template <typename I, bool PADDED>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const I *__restrict__ index, SortArgs p, Sorted out) {
  extern __shared__ int count[];  // [wave][per]
  __shared__ int before[kSortWaves], wave_sum[kSortWaves];
  __shared__ uint2 kept[kSortWaves][kKept];  // (t, row of the workgroup)
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, per = p.per;
  const uint32_t w = p.first + blockIdx.x;
  int *mine = count + wave * per;
  for (int i = threadIdx.x; i < kSortWaves * per; i += kSortThreads) count[i] = 0;
  __syncthreads();

  const uint32_t seg = (p.n + kSortThreads - 1) / kSortThreads * kWave;  // indices of a wave
  const uint32_t begin = min((uint32_t)wave * seg, p.n), end = min(begin + seg, p.n);
  const uint64_t lanes_before = (1ull << lane) - 1;
  int lower = 0;
  uint32_t found = 0;
  scan<PADDED>(index, begin, end, p, [&](uint32_t t, Owned o) __attribute__((always_inline)) {
    lower += o.before ? 1 : 0;
    const uint64_t own = __ballot(o.mine);
    if (own) {
      if (o.mine) {
        const uint32_t k = found + __popcll(own & lanes_before), r = o.row >> p.log_r;
        if (k < kKept) kept[wave][k] = make_uint2(t + lane, r);
        atomicAdd(&mine[r], 1);
      }
      found += __popcll(own);
    }
  });
  for (int d = kWave / 2; d >= 1; d /= 2) lower += __shfl_xor(lower, d, kWave);
  if (lane == 0) before[wave] = lower;
  __syncthreads();

  // First place of every row, and of every wave's part in it.
  const int i = threadIdx.x;
  int total = 0;
  if (i < per)
    for (int k = 0; k < kSortWaves; ++k) total += count[k * per + i];
  int sum = total;
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(sum, d, kWave);
    if (lane >= d) sum += up;
  }
  if (lane == kWave - 1) wave_sum[wave] = sum;
  __syncthreads();
  int at = sum - total;
  for (int k = 0; k < kSortWaves; ++k) {
    at += before[k];
    if (k < wave) at += wave_sum[k];
  }
  if (i < per) {
    const uint32_t v = ((uint32_t)i << p.log_r) | w;
    if (v < p.rows) out.span[v] = make_int2(at, total);
    int run = at;
    for (int k = 0; k < kSortWaves; ++k) {
      const int c = count[k * per + i];
      count[k * per + i] = run;
      run += c;
    }
  }
  if (w == (1u << p.log_r) - 1 && threadIdx.x == kSortThreads - 1) *out.valid = at + total;
  __syncthreads();

  // Places of up to 64 of the wave's indices, in their order: the lanes that have a lane's row are
  // found from the rows' bits.
  const int bits = 32 - __builtin_clz(per);
  auto place = [&](bool own, uint32_t t, uint32_t r) __attribute__((always_inline)) {
    uint64_t same = __ballot(own);
    for (int k = 0; k < bits; ++k) {
      const bool bit = r >> k & 1;
      const uint64_t set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    if (own) {
      const int rank = __popcll(same & lanes_before), k = mine[r] + rank;
      out.order[k] = (int)t;
      out.row[k] = (int)((r << p.log_r) | w);
      if (rank == 0) atomicAdd(&mine[r], __popcll(same));  // after all lanes have read it
    }
  };
  if (found <= kKept) {
    for (uint32_t k = 0; k < found; k += kWave) {
      const uint2 e = kept[wave][min(k + lane, kKept - 1u)];
      place(k + lane < found, e.x, e.y);
    }
  } else {
    scan<PADDED>(index, begin, end, p, [&](uint32_t t, Owned o) __attribute__((always_inline)) {
      place(o.mine, t + lane, o.row >> p.log_r);
    });
  }
}

// Sum and join give a group of `lanes` lanes (a power of two) one slice of a row: N channels each.
struct SumArgs {
  int64_t rows;
  int dim, lanes, slices, chunk_blocks, row_blocks;
  int first;  // workgroups in the launches before (launch_in_parts)
  float scale;
};

template <typename T, int N>
__device__ __forceinline__ void add_row(const T *g, int64_t at, float *a) {
  float v[N];
  load_f32<T, N>(g + at, v);
#pragma unroll
  for (int e = 0; e < N; ++e) a[e] += v[e];
}

template <typename T, int N>
__device__ __forceinline__ void write_row(T *gw, int64_t at, const float *a, float scale) {
  Vec<T, N> x;
#pragma unroll
  for (int e = 0; e < N; ++e) x.v[e] = static_cast<T>(a[e] * scale);
  store_vec<T, N>(gw + at, x);
}

// The two rows of more than kChunk places that a chunk of the sorted list can hold: one from the
// chunks before (places [0, head)) and one that goes on after it (places [tail, kChunk)).
struct Shared {
  int head, tail;
};
__device__ __forceinline__ Shared shared_rows(const Sorted &s, int chunk, int valid, int2 &span) {
  const int lane = threadIdx.x % kWave, place = chunk * kChunk + lane;
  span = make_int2(0, 0);
  if (lane < kChunk && place < valid) span = s.span[s.row[place]];
  const bool many = span.y > kChunk;
  return {(int)__popcll(__ballot(many && span.x < chunk * kChunk)),
          kChunk - (int)__popcll(__ballot(many && span.x >= chunk * kChunk))};
}

// a of the workgroup's groups of lanes added up in their order, into the first group's.
template <int N>
__device__ __forceinline__ void add_groups(float *a, float *s, int lanes) {
  __syncthreads();
#pragma unroll
  for (int e = 0; e < N; ++e) s[threadIdx.x * N + e] = a[e];
  __syncthreads();
  if ((int)threadIdx.x < lanes)
    for (int k = threadIdx.x + lanes; k < kThreads; k += lanes)
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] += s[k * N + e];
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) sum_kernel(const T *__restrict__ g, Sorted s, SumArgs p,
                                                       float *__restrict__ part, T *__restrict__ gw) {
  __shared__ float buf[kThreads * N];
  const int lane = threadIdx.x % p.lanes, group = threadIdx.x / p.lanes, groups = kThreads / p.lanes;
  const int block = p.first + (int)blockIdx.x;
  if (block < p.chunk_blocks) {
    const int chunk = block / p.slices, c = (block % p.slices * p.lanes + lane) * N;
    int2 span;
    const Shared sh = shared_rows(s, chunk, *s.valid, span);
    for (int side = 0; side < 2; ++side) {
      const int lo = side ? sh.tail : 0, hi = side ? kChunk : sh.head;
      if (lo >= hi) continue;
      float a[N] = {};
      if (c < p.dim)
#pragma unroll 4
        for (int k = lo + group; k < hi; k += groups)
          add_row<T, N>(g, (int64_t)s.order[chunk * kChunk + k] * p.dim + c, a);
      add_groups<N>(a, buf, p.lanes);
      if (group == 0 && c < p.dim)
#pragma unroll
        for (int e = 0; e < N; ++e) part[((int64_t)chunk * 2 + side) * p.dim + c + e] = a[e];
    }
    return;
  }
  const int64_t units = p.rows * p.slices;
  for (int64_t u = (int64_t)(block - p.chunk_blocks) * groups + group; u < units;
       u += (int64_t)p.row_blocks * groups) {
    const int64_t v = u / p.slices;
    const int c = ((int)(u - v * p.slices) * p.lanes + lane) * N;
    const int2 span = s.span != nullptr ? s.span[v] : make_int2(0, 0);
    if (c >= p.dim || span.y > kChunk) continue;
    float a[N] = {};
#pragma unroll 4
    for (int k = 0; k < span.y; ++k) add_row<T, N>(g, (int64_t)s.order[span.x + k] * p.dim + c, a);
    write_row<T, N>(gw, v * p.dim + c, a, p.scale);
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) join_kernel(Sorted s, SumArgs p, const float *__restrict__ part,
                                                        T *__restrict__ gw) {
  __shared__ float buf[kThreads * N];
  const int lane = threadIdx.x % p.lanes, group = threadIdx.x / p.lanes, groups = kThreads / p.lanes;
  const int block = p.first + (int)blockIdx.x;
  const int chunk = block / p.slices, c = (block % p.slices * p.lanes + lane) * N;
  int2 span;
  const Shared sh = shared_rows(s, chunk, *s.valid, span);
  if (sh.tail == kChunk) return;  // no such row begins here
  span.x = __builtin_amdgcn_readlane(span.x, kChunk - 1);
  span.y = __builtin_amdgcn_readlane(span.y, kChunk - 1);
  const int64_t v = s.row[span.x];
  const int more = (span.x + span.y - 1) / kChunk - chunk, each = (more + groups) / groups;
  float a[N] = {};
  if (c < p.dim)
#pragma unroll 4
    for (int k = group * each; k < min((group + 1) * each, more + 1); ++k)
      add_row<float, N>(part, ((int64_t)(chunk + k) * 2 + (k == 0 ? 1 : 0)) * p.dim + c, a);
  add_groups<N>(a, buf, p.lanes);
  if (group == 0 && c < p.dim) write_row<T, N>(gw, v * p.dim + c, a, p.scale);
}

int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

// Workspace: span, order, row, valid, then the partial sums.
struct Layout {
  int64_t order, row, valid, part, total;
  Layout(int64_t n, int64_t rows, int dim) {
    order = align256(rows * 8);
    row = order + align256(n * 4);
    valid = row + align256(n * 4);
    part = valid + 256;
    total = n == 0 ? 0 : part + (n > kChunk ? (n + kChunk - 1) / kChunk * 2 * dim * 4 : 0);
  }
};

// Channels a lane takes: 16 or 8 bytes of them where rows and tensors are aligned to that.
int lane_bytes(int64_t row_bytes, const void *a, const void *b) {
  const uintptr_t all = (uintptr_t)row_bytes | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : 0;
}

template <typename T, typename I, int N>
hipError_t forward_n(const EmbeddingArgs &a, const void *weight, void *out, hipStream_t stream) {
  const int64_t total = a.n * (a.dim / N), blocks = (total + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  return launch_in_parts(blocks, kThreads, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL((lookup_kernel<T, I, N>), dim3(count), dim3(kThreads), 0, stream,
                       static_cast<const T *>(weight), a.rows, (uint32_t)(a.dim / N),
                       static_cast<const I *>(a.index), total, first, a.scale, static_cast<T *>(out));
  });
}

template <typename T, typename I>
hipError_t forward(const EmbeddingArgs &a, const void *weight, void *out, hipStream_t stream) {
  switch (lane_bytes((int64_t)a.dim * sizeof(T), weight, out)) {
    case 16: return forward_n<T, I, 16 / sizeof(T)>(a, weight, out, stream);
    case 8: return forward_n<T, I, 8 / sizeof(T)>(a, weight, out, stream);
    default: return forward_n<T, I, 1>(a, weight, out, stream);
  }
}

template <typename T, int N>
hipError_t sums(const EmbeddingArgs &a, const void *grad_out, const Sorted &s, float *part, void *grad_w,
                hipStream_t stream) {
  SumArgs p;
  p.rows = a.rows; p.dim = a.dim; p.scale = a.scale;
  p.lanes = 1;
  while (p.lanes < kWave && p.lanes * N < a.dim) p.lanes *= 2;
  p.slices = (a.dim + p.lanes * N - 1) / (p.lanes * N);
  const int64_t chunks = a.n > kChunk ? (a.n + kChunk - 1) / kChunk * p.slices : 0;
  p.chunk_blocks = (int)chunks;  // below 2^30 with at most 2^40 values of grad_out
  p.row_blocks = (int)std::min<int64_t>(1 << 20, (a.rows * p.slices + kThreads / p.lanes - 1) /
                                                     (kThreads / p.lanes));
  const hipError_t e = launch_in_parts(chunks + p.row_blocks, kThreads, [&](int64_t first, unsigned count) {
    p.first = (int)first;
    hipLaunchKernelGGL((sum_kernel<T, N>), dim3(count), dim3(kThreads), 0, stream, static_cast<const T *>(grad_out),
                       s, p, part, static_cast<T *>(grad_w));
  });
  if (e != hipSuccess) return e;
  return launch_in_parts(chunks, kThreads, [&](int64_t first, unsigned count) {
    p.first = (int)first;
    hipLaunchKernelGGL((join_kernel<T, N>), dim3(count), dim3(kThreads), 0, stream, s, p, part,
                       static_cast<T *>(grad_w));
  });
}

template <typename T, typename I>
hipError_t backward(const EmbeddingArgs &a, const void *grad_out, int64_t padding, void *workspace, void *grad_w,
                    hipStream_t stream) {
  const Layout l(a.n, a.rows, a.dim);
  char *ws = static_cast<char *>(workspace);
  Sorted s{};
  if (a.n > 0) {
    s = {reinterpret_cast<int2 *>(ws), reinterpret_cast<int *>(ws + l.order), reinterpret_cast<int *>(ws + l.row),
         reinterpret_cast<int *>(ws + l.valid)};
    SortArgs p;
    p.n = (uint32_t)a.n; p.rows = (uint32_t)a.rows; p.padding = (uint32_t)padding;
    p.log_r = 8;  // 256 workgroups, or as many as have at most kSortRows rows each
    while ((a.rows - 1) >> p.log_r >= kSortRows) ++p.log_r;
    p.per = (int)((a.rows - 1) >> p.log_r) + 1;
    const auto sort = padding < 0 ? sort_kernel<I, false> : sort_kernel<I, true>;
    const hipError_t e = launch_in_parts(1 << p.log_r, kSortThreads, [&](int64_t first, unsigned count) {
      p.first = (uint32_t)first;
      hipLaunchKernelGGL(sort, dim3(count), dim3(kSortThreads), kSortWaves * p.per * 4, stream,
                         static_cast<const I *>(a.index), p, s);
    });
    if (e != hipSuccess) return e;
  }
  float *part = reinterpret_cast<float *>(ws + l.part);
  switch (lane_bytes((int64_t)a.dim * sizeof(T), grad_out, grad_w)) {
    case 16: return sums<T, 16 / sizeof(T)>(a, grad_out, s, part, grad_w, stream);
    case 8: return sums<T, 8 / sizeof(T)>(a, grad_out, s, part, grad_w, stream);
    default: return sums<T, 1>(a, grad_out, s, part, grad_w, stream);
  }
}

}  // namespace

int64_t embedding_backward_workspace_bytes(int64_t n, int64_t rows, int dim) { return Layout(n, rows, dim).total; }

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
    case 0: return backward<float, int32_t>(a, grad_out, padding, workspace, grad_w, stream);
    case 1: return backward<float, int64_t>(a, grad_out, padding, workspace, grad_w, stream);
    case 2: return backward<f16, int32_t>(a, grad_out, padding, workspace, grad_w, stream);
    case 3: return backward<f16, int64_t>(a, grad_out, padding, workspace, grad_w, stream);
    case 4: return backward<bf16, int32_t>(a, grad_out, padding, workspace, grad_w, stream);
    default: return backward<bf16, int64_t>(a, grad_out, padding, workspace, grad_w, stream);
  }
}

}  // namespace bevk
