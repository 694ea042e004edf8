// embedding.hip -- rows of a table by tokens, scaled, and the gradient.
//
//   out[i]  = scale * table[tok[i]]
//   grad[v] = scale * sum over i with tok[i] = v, in order of i, of g[i]
//
// A token outside [0, rows) is none: its output is zeros and it has no
// gradient, so ragged batches can be filled up with -1.  Sums are held in 32
// bits (64 for float64) and rounded once.
//
// Both are bound by memory.  The gradient first orders the tokens' positions by
// row, equal ones ascending, so that the sums keep their bits.  One pass of a
// radix sort splits them into at most 256 groups of neighbouring rows (tiles of the
// tokens count and then place their own, in order), and a workgroup orders a
// group's by row with counters in LDS.  More than 2^20 rows are too many for those:
// then every 8 bits of the row have a pass, from the lowest on.
//
// Then a few lanes sum a row's positions.  Words' frequencies are skewed: a row
// of more than kWindow positions is summed in windows of kWindow places of the
// order (a window holds the end of one such row and the beginning of another
// at most), and the row's workgroup adds up the windows' sums.
#include "mmp_nn.h"

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
constexpr int kDigits = 256, kMaxTiles = 256;
constexpr int kSplitWaves = kBlock / 64;

// A token's position and row.
struct Entry {
  unsigned row, at;
};
// What a pass reads: the tokens (row = -1 where they have none), or the
// entries of the pass before, whose number is on the device.
template <typename I> struct Tokens {
  const I *tokens;
  unsigned n, rows;
  __device__ __forceinline__ unsigned count() const { return n; }
  __device__ __forceinline__ bool get(unsigned i, Entry &e) const {
    const long long t = (long long)tokens[i];
    e = {(unsigned)t, i};
    return t >= 0 && t < (long long)rows;
  }
};
struct Entries {
  const Entry *entries;
  const unsigned *n;
  __device__ __forceinline__ unsigned count() const { return *n; }
  __device__ __forceinline__ bool get(unsigned i, Entry &e) const {
    e = entries[i];
    return true;
  }
};

__device__ __forceinline__ unsigned lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}
// The lanes of `among` whose low `bits` bits of d are this lane's.
__device__ __forceinline__ unsigned long long lanes_alike(unsigned long long among, unsigned d,
                                                          int bits) {
  for (int b = 0; b < bits; ++b) {
    const bool one = (d >> b) & 1;
    const unsigned long long m = __ballot(one);
    among &= one ? m : ~m;
  }
  return among;
}

// count[t][d]: entries of tile t with digit d = row >> shift & 255.
template <typename S>
__global__ __launch_bounds__(kBlock) void k_split_count(S src, unsigned tile_len, int shift,
                                                        unsigned *__restrict__ count) {
  __shared__ unsigned h[kDigits];
  h[threadIdx.x] = 0;
  __syncthreads();
  const unsigned n = src.count();
  const unsigned from = blockIdx.x * tile_len < n ? blockIdx.x * tile_len : n;
  const unsigned to = n - from < tile_len ? n : from + tile_len;
#pragma unroll 4
  for (unsigned i = from + threadIdx.x; i < to; i += kBlock) {
    Entry e;
    if (src.get(i, e)) atomicAdd(&h[e.row >> shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  count[blockIdx.x * kDigits + threadIdx.x] = h[threadIdx.x];
}

// Places the entries by digit, otherwise in order; first[d] is where digit d
// begins, and first[256] the number of all.  Every workgroup adds up the
// counts of the tiles before its own.
template <typename S>
__global__ __launch_bounds__(kBlock) void k_split(S src, unsigned tile_len, int shift,
                                                  const unsigned *__restrict__ count,
                                                  unsigned *__restrict__ first,
                                                  Entry *__restrict__ out) {
  __shared__ unsigned next[kSplitWaves][kDigits];
  __shared__ unsigned part[kSplitWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int w = 0; w < kSplitWaves; ++w) next[w][tid] = 0;
  const unsigned n = src.count();
  const unsigned quarter = tile_len / kSplitWaves, tile = blockIdx.x * tile_len;
  unsigned from = tile + wave * quarter;
  from = from < n ? from : n;
  const unsigned to = n - from < quarter ? n : from + quarter;
  unsigned before = 0, total = 0;
#pragma unroll 8
  for (unsigned t = 0; t < gridDim.x; ++t) {
    const unsigned c = count[t * kDigits + tid];
    before += t < blockIdx.x ? c : 0;
    total += c;
  }
  __syncthreads();
#pragma unroll 4
  for (unsigned i = from + lane; i < to; i += 64) {
    Entry e;
    if (src.get(i, e)) atomicAdd(&next[wave][e.row >> shift & (kDigits - 1)], 1u);
  }
  unsigned incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  unsigned at = incl - total;
  for (int w = 0; w < wave; ++w) at += part[w];
  if (blockIdx.x == 0) {
    first[tid] = at;
    if (tid == kDigits - 1) first[kDigits] = at + total;
  }
  at += before;
#pragma unroll
  for (int w = 0; w < kSplitWaves; ++w) {
    const unsigned c = next[w][tid];
    next[w][tid] = at;
    at += c;
  }
  __syncthreads();
  for (unsigned i0 = from; i0 < to; i0 += 64) {
    Entry e{0, 0};
    const bool there = i0 + lane < to && src.get(i0 + lane, e);
    const unsigned d = e.row >> shift & (kDigits - 1);
    const unsigned long long same = lanes_alike(__ballot(there), d, 8);
    const unsigned rank = lanes_below(same);
    if (there) {
      const unsigned base = next[wave][d];
      out[base + rank] = e;
      if (rank == 0) next[wave][d] = base + (unsigned)__popcll(same);
    }
  }
}

// Workgroup g orders group g, rows [g << bits, (g + 1) << bits), by row.
// order: the positions; start[v]: where row v's begin, start[rows] their number.
constexpr int kGroupBlock = 512, kGroupRows = 4096;
__global__ __launch_bounds__(kGroupBlock) void k_group(const Entry *__restrict__ entries,
                                                       const unsigned *__restrict__ first,
                                                       unsigned rows, int bits, int waves,
                                                       unsigned *__restrict__ start,
                                                       unsigned *__restrict__ order) {
  extern __shared__ unsigned next[];  // [waves][1 << bits]
  __shared__ unsigned part[kGroupBlock / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned bins = 1u << bits, row0 = blockIdx.x << bits;
  for (unsigned k = tid; k < waves * bins; k += kGroupBlock) next[k] = 0;
  const unsigned base = first[blockIdx.x], n = first[blockIdx.x + 1] - base;
  const unsigned per = (n + waves * 64 - 1) / (waves * 64) * 64;
  unsigned from = wave < waves ? wave * per : n;
  from = from < n ? from : n;
  const unsigned to = n - from < per ? n : from + per;
  unsigned *mine = next + wave * bins;
  __syncthreads();
#pragma unroll 4
  for (unsigned i = from + lane; i < to; i += 64)
    atomicAdd(&mine[entries[base + i].row - row0], 1u);
  __syncthreads();
  // exclusive sums over the rows, neighbouring ones a thread's, and within a
  // row over the waves
  const unsigned mult = (bins + kGroupBlock - 1) / kGroupBlock;
  unsigned total = 0;
  for (unsigned k = tid * mult; k < (tid + 1) * mult && k < bins; ++k)
    for (int w = 0; w < waves; ++w) total += next[w * bins + k];
  unsigned incl = total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  unsigned at = base + incl - total;
  for (int w = 0; w < wave; ++w) at += part[w];
  for (unsigned k = tid * mult; k < (tid + 1) * mult && k < bins; ++k) {
    if (row0 + k < rows) start[row0 + k] = at;
    for (int w = 0; w < waves; ++w) {
      const unsigned c = next[w * bins + k];
      next[w * bins + k] = at;
      at += c;
    }
    if (row0 + k == rows - 1) start[rows] = at;
  }
  __syncthreads();
  for (unsigned i0 = from; i0 < to; i0 += 64) {
    const bool there = i0 + lane < to;
    const Entry e = entries[base + (there ? i0 + lane : from)];
    const unsigned k = e.row - row0;
    const unsigned long long same = lanes_alike(__ballot(there), k, bits);
    const unsigned rank = lanes_below(same);
    if (there) {
      const unsigned o = mine[k];
      order[o + rank] = e.at;
      if (rank == 0) mine[k] = o + (unsigned)__popcll(same);
    }
  }
}

// From entries in the order of their rows: start and order as above.
__global__ __launch_bounds__(kBlock) void k_starts(const Entry *__restrict__ entries,
                                                   const unsigned *__restrict__ count,
                                                   unsigned rows, unsigned *__restrict__ start,
                                                   unsigned *__restrict__ order) {
  const unsigned i = blockIdx.x * kBlock + threadIdx.x, n = *count;
  if (i < n) order[i] = entries[i].at;
  if (i > rows) return;
  unsigned lo = 0, hi = n;  // the first entry of row i or a later one
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    if (entries[mid].row < i) lo = mid + 1;
    else hi = mid;
  }
  start[i] = lo;
}

// ---------------------------------------------------------------- row sums
constexpr int kWindow = 64;

// sum += the vectors at column `at` of the rows that `from` to `to` of the order
// name, one after another.  The next kLoads vectors are on their way while as
// many are added, and their places while those are.
template <typename T, int V, int kLoads, typename A>
__device__ __forceinline__ void add_rows(A (&sum)[V], const T *__restrict__ grad, long long stride,
                                         const unsigned *__restrict__ order, unsigned from,
                                         unsigned to, int at) {
  if (from >= to) return;
  unsigned id[kLoads];
  Vec<T, V> g[kLoads];
  auto places = [&](unsigned j) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) id[i] = order[j + i < to ? j + i : to - 1];
  };
  auto vectors = [&]() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      g[i] = mmpn::load_vec<T, V, true>(grad + (long long)id[i] * stride + at);
  };
  places(from);
  vectors();
  if (to - from > kLoads) places(from + kLoads);
  for (unsigned j = from; j < to; j += kLoads) {
    Vec<T, V> now[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) now[i] = g[i];
    if (j + kLoads < to) {
      vectors();
      if (to - j > 2 * kLoads) places(j + 2 * kLoads);
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (j + i < to) {
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += (A)now[i].e[k];
      }
  }
}

// Window w of the order: the sums of its pieces of rows of more than kWindow
// positions, part[2 w] of one that began before it and part[2 w + 1] of one
// that begins in it.
template <typename T, typename I, int V>
__global__ __launch_bounds__(kBlock) void k_window_sums(const I *__restrict__ tokens,
                                                        const T *__restrict__ grad, long long stride,
                                                        long long rows, int dim, int lanes,
                                                        unsigned windows,
                                                        const unsigned *__restrict__ start,
                                                        const unsigned *__restrict__ order,
                                                        typename Wide<T>::type *__restrict__ part) {
  typedef typename Wide<T>::type A;
  const unsigned w = blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes;
  const unsigned total = start[rows];
  if (w >= windows || w * (unsigned)kWindow >= total) return;
  const unsigned p0 = w * kWindow, p1 = total - p0 < kWindow ? total : p0 + kWindow;
#pragma unroll
  for (int piece = 0; piece < 2; ++piece) {
    const long long r = (long long)tokens[order[piece ? p1 - 1 : p0]];
    const unsigned from = start[r], to = start[r + 1];
    if (to - from <= kWindow || (from >= p0) != (piece == 1)) continue;
    for (int c = (threadIdx.x & (lanes - 1)) * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
      add_rows<T, V, 8, A>(sum, grad, stride, order, from > p0 ? from : p0, to < p1 ? to : p1, at);
      A *dst = part + (2ll * w + piece) * dim + at;
#pragma unroll
      for (int k = 0; k < V; ++k) dst[k] = sum[k];
    }
  }
}

// Rows of the gradient: kRows for `lanes` threads.  Those of up to kFirst
// positions, most of them, are read all at once (one after another they would
// wait for their order, then for their vectors), then the longer ones; one in
// windows is the whole workgroup's.
constexpr int kRows = 4, kFirst = 2;
template <typename T, int V>
__global__ __launch_bounds__(kBlock) void k_row_sums(
    const T *__restrict__ grad, long long stride, long long rows, int dim, int lanes,
    typename Wide<T>::type scale, const unsigned *__restrict__ start,
    const unsigned *__restrict__ order, const typename Wide<T>::type *__restrict__ part,
    T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  __shared__ A lds[kBlock * V];
  __shared__ int long_rows[kBlock * kRows], count;
  const int per = kBlock / lanes, g = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  const long long v0 = (long long)blockIdx.x * per * kRows;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const long long v = v0 + g * kRows;
  {
    unsigned edge[kRows + 1], id[kRows][kFirst];
#pragma unroll
    for (int r = 0; r <= kRows; ++r) edge[r] = start[v + r < rows ? v + r : rows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < kFirst; ++i)
        if (edge[r] + i < edge[r + 1]) id[r][i] = order[edge[r] + i];
    for (int c = lane * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      Vec<T, V> x[kRows][kFirst];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kFirst; ++i)
          if (edge[r] + i < edge[r + 1] && edge[r + 1] - edge[r] <= kFirst)
            x[r][i] = mmpn::load_vec<T, V, true>(grad + (long long)id[r][i] * stride + at);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        A sum[V];
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] = 0;
#pragma unroll
        for (int i = 0; i < kFirst; ++i)
          if (edge[r] + i < edge[r + 1]) {
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += (A)x[r][i].e[k];
          }
        Vec<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = (T)(sum[k] * scale);
        if (v + r < rows && edge[r + 1] - edge[r] <= kFirst)
          mmpn::store_vec<T, V, true>(out + (v + r) * dim + at, o);
      }
    }
  }
#pragma unroll 1
  for (int r = 0; r < kRows && v + r < rows; ++r) {
    const unsigned from = start[v + r], to = start[v + r + 1];
    if (to - from <= kFirst) continue;
    if (to - from > kWindow) {
      if (lane == 0) long_rows[atomicAdd(&count, 1)] = g * kRows + r;
      continue;
    }
    for (int c = lane * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
      add_rows<T, V, 4, A>(sum, grad, stride, order, from, to, at);
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.e[k] = (T)(sum[k] * scale);
      mmpn::store_vec<T, V, true>(out + (v + r) * dim + at, o);
    }
  }
  __syncthreads();
  const int n = count;
  for (int q = 0; q < n; ++q) {
    const long long v = v0 + long_rows[q];
    const unsigned w0 = start[v] / kWindow, w1 = (start[v + 1] - 1) / kWindow;
    for (int c0 = 0; c0 < dim; c0 += lanes * V) {
      const int c = c0 + lane * V, at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
      if (c < dim) {
#pragma unroll 4
        for (unsigned w = w0 + g; w <= w1; w += per) {
          const A *src = part + (2ll * w + (w == w0)) * dim + at;
#pragma unroll
          for (int k = 0; k < V; ++k) sum[k] += src[k];
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) lds[(g * lanes + lane) * V + k] = sum[k];
      __syncthreads();
      if (g == 0 && c < dim) {
        Vec<T, V> r;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          A s = 0;
          for (int o = 0; o < per; ++o) s += lds[(o * lanes + lane) * V + k];
          r.e[k] = (T)(s * scale);
        }
        mmpn::store_vec<T, V, true>(out + v * dim + at, r);
      }
      __syncthreads();
    }
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

// Orders the tokens' positions by row; ea, eb: room for n entries each.
template <typename I>
int order_tokens(unsigned n, const I *tokens, unsigned rows, Entry *ea, Entry *eb, unsigned *count,
                 unsigned *first, unsigned *start, unsigned *order) {
  // up to 256 tiles of at least 1024 tokens, which every workgroup of k_split
  // adds up
  unsigned tile = (unsigned)(mmpi::ceil_div(mmpi::ceil_div(n, kMaxTiles), 256) * 256);
  if (tile < 1024) tile = 1024;
  const unsigned tiles = n ? (unsigned)mmpi::ceil_div(n, tile) : 1;
  auto pass = [&](auto src, int shift, Entry *out) -> int {
    typedef decltype(src) S;
    hipLaunchKernelGGL((k_split_count<S>), dim3(tiles), dim3(kBlock), 0, mmpi::stream(), src, tile,
                       shift, count);
    if (int st = mmpi::check_launch("mmp_embedding_grad(count)")) return st;
    hipLaunchKernelGGL((k_split<S>), dim3(tiles), dim3(kBlock), 0, mmpi::stream(), src, tile,
                       shift, (const unsigned *)count, first, out);
    return mmpi::check_launch("mmp_embedding_grad(split)");
  };
  int bits = 0;
  while ((rows - 1) >> bits) ++bits;  // of a row
  if (rows <= (unsigned)kDigits * kGroupRows) {
    const int low = bits > 8 ? bits - 8 : 0;
    if (int st = pass(Tokens<I>{tokens, n, rows}, low, ea)) return st;
    const unsigned groups = ((rows - 1) >> low) + 1;
    const int waves = low > 11 ? 4 : 8;  // 64 KiB of counters at most
    hipLaunchKernelGGL(k_group, dim3(groups), dim3(kGroupBlock), (unsigned)(waves * 4) << low,
                       mmpi::stream(), (const Entry *)ea, (const unsigned *)first, rows, low, waves,
                       start, order);
    return mmpi::check_launch("mmp_embedding_grad(group)");
  }
  if (int st = pass(Tokens<I>{tokens, n, rows}, 0, ea)) return st;
  for (int shift = 8; shift < bits; shift += 8) {
    if (int st = pass(Entries{ea, first + kDigits}, shift, eb)) return st;
    Entry *t = ea;
    ea = eb;
    eb = t;
  }
  const unsigned most = n > rows + 1 ? n : rows + 1;
  hipLaunchKernelGGL(k_starts, dim3((unsigned)mmpi::ceil_div(most, kBlock)), dim3(kBlock), 0,
                     mmpi::stream(), (const Entry *)ea, (const unsigned *)(first + kDigits), rows,
                     start, order);
  return mmpi::check_launch("mmp_embedding_grad(starts)");
}

template <typename T, typename I>
int grad_impl(int64_t n, const I *tokens, const T *grad, int64_t stride, int64_t rows, int dim,
              double scale, T *out) {
  typedef typename Wide<T>::type A;
  constexpr int V = 16 / sizeof(T);
  Temp order, start, part, entries, counts;
  const bool twice = rows > (int64_t)kDigits * kGroupRows;
  if (int st = order.get((size_t)n * 4)) return st;
  if (int st = start.get((size_t)(rows + 1) * 4)) return st;
  if (int st = entries.get((size_t)n * sizeof(Entry) * (twice ? 2 : 1))) return st;
  if (int st = counts.get((size_t)(kMaxTiles * kDigits + kDigits + 1) * 4)) return st;
  unsigned *count = (unsigned *)counts.p;
  if (int st = order_tokens<I>((unsigned)n, tokens, (unsigned)rows, (Entry *)entries.p,
                               (Entry *)entries.p + n, count, count + kMaxTiles * kDigits,
                               (unsigned *)start.p, (unsigned *)order.p))
    return st;
  const int vec = dim >= V ? V : 1;
  const int lanes = row_lanes(dim, vec);
  const int64_t windows = mmpi::ceil_div(n, kWindow);
  const int64_t blocks = mmpi::ceil_div(rows, kBlock / lanes * kRows);
  const int64_t wblocks = mmpi::ceil_div(windows, kBlock / lanes);
  if (!mmpi::grid_fits(blocks, kBlock) || !mmpi::grid_fits(wblocks, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: too many rows or tokens");
  if (n > kWindow) {
    if (int st = part.get((size_t)windows * 2 * dim * sizeof(A))) return st;
    auto kernel = vec == V ? k_window_sums<T, I, V> : k_window_sums<T, I, 1>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wblocks), dim3(kBlock), 0, mmpi::stream(), tokens,
                       grad, (long long)stride, (long long)rows, dim, lanes, (unsigned)windows,
                       (const unsigned *)start.p, (const unsigned *)order.p, (A *)part.p);
    if (int st = mmpi::check_launch("mmp_embedding_grad(windows)")) return st;
  }
  auto kernel = vec == V ? k_row_sums<T, V> : k_row_sums<T, 1>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(), grad,
                     (long long)stride, (long long)rows, dim, lanes, (A)scale,
                     (const unsigned *)start.p, (const unsigned *)order.p, (const A *)part.p, out);
  return mmpi::check_launch("mmp_embedding_grad");
}

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
  MMP_DISPATCH_FLOAT(dtype, "mmp_embedding_grad", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_embedding_grad", {
      return grad_impl<T, I>(n, (const I *)tokens, (const T *)grad, row_stride, rows, (int)dim,
                             scale, (T *)out);
    })
  })
}
