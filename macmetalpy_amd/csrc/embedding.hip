// embedding.hip -- rows of a table by tokens, scaled, and the gradient.
//
//   out[i]  = scale * table[tok[i]]
//   grad[v] = scale * sum over i with tok[i] = v, in order of i, of g[i]
//
// A token outside [0, rows) is none: its output is zeros and it has no
// gradient, so ragged batches can be filled up with -1.  Sums are held in 32
// bits (64 for float64) and rounded once.
//
// Both are bound by memory.  The gradient sorts the tokens by their row without
// a sort's passes: every workgroup owns a range of rows and goes through all
// tokens twice, first counting those of its rows (and those of lower rows,
// which is where its part of the order begins), then placing them.  The
// tokens are read from the caches by all workgroups; they are few bytes
// against the gradient's rows.  A wave owns a contiguous part of the tokens and
// counters of its own, so that equal tokens keep their order and the sums
// their bits.
#include "mmp_nn.h"

#include <algorithm>

namespace {

using mmpn::Vec;
using mmpn::Wide;

constexpr int kBlock = 256;

// ------------------------------------------------------------------ lookup
// `lanes` threads a row (a power of two), a vector of V elements each and
// step.  A row's last vector ends with the row, so it may overlap the one
// before it, which writes the same values.
template <typename T, typename I, int V>
__global__ __launch_bounds__(kBlock) void k_embed(const I *__restrict__ tokens, long long n,
                                                  const T *__restrict__ table, long long rows,
                                                  long long stride, int dim, int lanes,
                                                  typename Wide<T>::type scale,
                                                  T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  const int per = kBlock / lanes;
  const long long i = (long long)blockIdx.x * per + threadIdx.x / lanes;
  if (i >= n) return;
  const long long tok = (long long)tokens[i];
  const bool there = tok >= 0 && tok < rows;
  const T *src = table + (there ? tok : 0) * stride;
  T *dst = out + i * dim;
  for (int c = (threadIdx.x & (lanes - 1)) * V; c < dim; c += lanes * V) {
    const int at = c + V > dim ? dim - V : c;
    Vec<T, V> v;
    if (there) {
      v = mmpn::load_vec<T, V>(src + at);
#pragma unroll
      for (int k = 0; k < V; ++k) v.e[k] = (T)((A)v.e[k] * scale);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) v.e[k] = (T)0;
    }
    mmpn::store_vec<T, V>(dst + at, v);
  }
}

// ---------------------------------------------------------------- grouping
constexpr int kGroupBlock = 1024, kGroupWaves = kGroupBlock / 64;
constexpr int kMaxBins = 1024;  // rows of a workgroup: 64 KiB of counters

// Workgroup b: rows [b * bins, (b + 1) * bins).  order: the tokens' positions
// by row, equal ones ascending; start[v]: where row v's positions begin, and
// start[rows] the number of tokens that have a row.
template <typename I>
__global__ __launch_bounds__(kGroupBlock) void k_group(const I *__restrict__ tokens, unsigned n,
                                                       long long rows, int bins,
                                                       unsigned *__restrict__ start,
                                                       unsigned *__restrict__ order) {
  extern __shared__ unsigned count[];  // [kGroupWaves][bins]
  __shared__ unsigned part[kGroupWaves];
  __shared__ unsigned lower;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long first = (long long)blockIdx.x * bins;
  const int own = (int)(rows - first < bins ? rows - first : bins);
  for (int k = tid; k < kGroupWaves * bins; k += kGroupBlock) count[k] = 0;
  if (tid == 0) lower = 0;
  __syncthreads();
  const unsigned per = (n + kGroupBlock - 1) / kGroupBlock * 64;  // tokens of a wave
  const unsigned from = wave * per < n ? wave * per : n;
  const unsigned to = n - from < per ? n : from + per;
  unsigned *mine = count + wave * bins;
  unsigned below = 0;
  for (unsigned p = from + lane; p < to; p += 64) {
    const long long t = (long long)tokens[p] - first;
    below += t < 0 && t + first >= 0;
    if (t >= 0 && t < own) atomicAdd(&mine[t], 1u);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) below += __shfl_xor(below, m, 64);
  if (lane == 0) atomicAdd(&lower, below);
  __syncthreads();
  // exclusive sums over the rows (a row a thread), and within a row over the waves
  unsigned total = 0;
  if (tid < own)
    for (int w = 0; w < kGroupWaves; ++w) total += count[w * bins + tid];
  unsigned incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  unsigned at = lower + incl - total;
  for (int w = 0; w < wave; ++w) at += part[w];
  if (tid < own) {
    start[first + tid] = at;
    if (first + tid == rows - 1) start[rows] = at + total;
    for (int w = 0; w < kGroupWaves; ++w) {
      const unsigned c = count[w * bins + tid];
      count[w * bins + tid] = at;
      at += c;
    }
  }
  __syncthreads();
  for (unsigned p0 = from; p0 < to; p0 += 64) {
    const unsigned p = p0 + lane;
    const long long t = p < to ? (long long)tokens[p] - first : -1;
    const bool here = t >= 0 && t < own;
    const int b = here ? (int)t : 0;
    unsigned long long left = __ballot(here);
    while (left) {  // one row a turn: its lanes take consecutive places
      const int lead = __ffsll((long long)left) - 1;
      const int row = __builtin_amdgcn_readlane(b, lead);
      const unsigned long long same = __ballot(here && b == row);
      if (here && b == row) {
        const unsigned base = mine[row];
        order[base + __popcll(same & ((1ull << lane) - 1))] = p;
        if (lane == lead) mine[row] = base + (unsigned)__popcll(same);
      }
      left &= ~same;
    }
  }
}

// ---------------------------------------------------------------- row sums
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void k_embed_grad(const T *__restrict__ grad, long long stride,
                                                       long long rows, int dim, int lanes,
                                                       typename Wide<T>::type scale,
                                                       const unsigned *__restrict__ start,
                                                       const unsigned *__restrict__ order,
                                                       T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  const int per = kBlock / lanes;
  const long long v = (long long)blockIdx.x * per + threadIdx.x / lanes;
  if (v >= rows) return;
  const unsigned from = start[v], to = start[v + 1];
  T *dst = out + v * dim;
  for (int c = (threadIdx.x & (lanes - 1)) * V; c < dim; c += lanes * V) {
    const int at = c + V > dim ? dim - V : c;
    A sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0;
    for (unsigned j = from; j < to; ++j) {
      const Vec<T, V> g = mmpn::load_vec<T, V>(grad + (long long)order[j] * stride + at);
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] += (A)g.e[k];
    }
    Vec<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.e[k] = (T)(sum[k] * scale);
    mmpn::store_vec<T, V>(dst + at, r);
  }
}

// Threads a row: enough for its vectors, a power of two up to the workgroup.
inline int row_lanes(int64_t dim, int vec) {
  int lanes = 1;
  while (lanes < kBlock && (int64_t)lanes * vec < dim) lanes <<= 1;
  return lanes;
}

// Temporaries from the library's stream-ordered pool, released on scope exit.
struct Temp {
  void *p = nullptr;
  ~Temp() {
    if (p) (void)mmp_free(p);
  }
  int get(size_t bytes) { return mmp_alloc(bytes ? bytes : 1, &p); }
};

constexpr int64_t kMost = 0x7fffffffLL;

}  // namespace

extern "C" int mmp_embedding(int dtype, int index_dtype, int64_t n, const void *tokens,
                             int64_t rows, int64_t dim, const void *table, int64_t row_stride,
                             double scale, void *out) {
  if (int st = mmpi::ensure_init()) return st;
  if (n < 0 || rows < 0 || dim < 0) return mmpi::fail(MMP_E_ARG, "mmp_embedding: negative extent");
  if (n == 0 || dim == 0) return MMP_OK;
  if (!tokens || !out || (rows > 0 && !table))
    return mmpi::fail(MMP_E_ARG, "mmp_embedding: null pointer");
  if (dim > kMost) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding: rows of 2^31 or more");
  MMP_DISPATCH_FLOAT(dtype, "mmp_embedding", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_embedding", {
      constexpr int V = 16 / sizeof(T);
      const int vec = dim >= V ? V : 1;
      const int lanes = row_lanes(dim, vec);
      const int64_t blocks = mmpi::ceil_div(n, kBlock / lanes);
      if (!mmpi::grid_fits(blocks, kBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding: too many tokens");
      auto kernel = vec == V ? k_embed<T, I, V> : k_embed<T, I, 1>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(),
                         (const I *)tokens, (long long)n, (const T *)table, (long long)rows,
                         (long long)row_stride, (int)dim, lanes, (typename Wide<T>::type)scale,
                         (T *)out);
      return mmpi::check_launch("mmp_embedding");
    })
  })
}

extern "C" int mmp_embedding_grad(int dtype, int index_dtype, int64_t n, const void *tokens,
                                  const void *grad, int64_t row_stride, int64_t rows, int64_t dim,
                                  double scale, void *out) {
  if (int st = mmpi::ensure_init()) return st;
  if (n < 0 || rows < 0 || dim < 0)
    return mmpi::fail(MMP_E_ARG, "mmp_embedding_grad: negative extent");
  if (rows == 0 || dim == 0) return MMP_OK;
  if (!out || (n > 0 && (!tokens || !grad)))
    return mmpi::fail(MMP_E_ARG, "mmp_embedding_grad: null pointer");
  if (dim > kMost || n > kMost || rows > kMost)
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: 2^31 tokens, rows or columns, or more");
  Temp order, start;
  if (int st = order.get((size_t)n * 4)) return st;
  if (int st = start.get((size_t)(rows + 1) * 4)) return st;
  const int64_t cus = mmpi::cu_count();
  int64_t bins = mmpi::ceil_div(rows, cus);
  bins = bins < 16 ? 16 : bins > kMaxBins ? kMaxBins : bins;
  MMP_DISPATCH_FLOAT(dtype, "mmp_embedding_grad", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_embedding_grad", {
      constexpr int V = 16 / sizeof(T);
      hipLaunchKernelGGL((k_group<I>), dim3((unsigned)mmpi::ceil_div(rows, bins)),
                         dim3(kGroupBlock), (unsigned)(kGroupWaves * bins * 4), mmpi::stream(),
                         (const I *)tokens, (unsigned)n, (long long)rows, (int)bins,
                         (unsigned *)start.p, (unsigned *)order.p);
      if (int st = mmpi::check_launch("mmp_embedding_grad(group)")) return st;
      const int vec = dim >= V ? V : 1;
      const int lanes = row_lanes(dim, vec);
      const int64_t blocks = mmpi::ceil_div(rows, kBlock / lanes);
      if (!mmpi::grid_fits(blocks, kBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: too many rows");
      auto kernel = vec == V ? k_embed_grad<T, V> : k_embed_grad<T, 1>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(),
                         (const T *)grad, (long long)row_stride, (long long)rows, (int)dim, lanes,
                         (typename Wide<T>::type)scale, (const unsigned *)start.p,
                         (const unsigned *)order.p, (T *)out);
      return mmpi::check_launch("mmp_embedding_grad");
    })
  })
}
