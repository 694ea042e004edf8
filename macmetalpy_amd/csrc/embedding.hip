// embedding.hip -- rows of a table by tokens, scaled, and the gradient.
//
//   out[i]  = scale * table[tok[i]]
//   grad[v] = scale * sum over i with tok[i] = v of g[i]
//
// A token outside [0, rows) is none: its output is zeros and it has no
// gradient, so ragged batches can be filled up with -1.  Sums are held in 32
// bits (64 for float64), added in an order that follows from the tokens, the width
// and the type, not from timing, and rounded once.
//
// Both are bound by memory.  The gradient first brings the tokens' positions of
// each row together, ascending, so that the sums keep their bits.  One pass of a
// radix sort splits them by the low 8 bits of the row (tiles of the tokens
// count and then place their own, in order): low ones, because the frequent
// words of a vocabulary are neighbours, and one group of half the tokens would
// be one workgroup's.  That orders a group's by row with counters in LDS.  More
// than 2^20 rows are too many for those, and of more than 2^17 tokens a workgroup
// has too many: then every 8 bits of the row have a pass (8 columns; groups and
// passes, of 60,000 rows: 60,000 tokens 42 and 51 us, 131,072 52 and 58, 200,000 61
// and 67, 262,144 79 and 71, 524,288 118 and 94; of a million rows: 66 and 87, 87
// and 92, 109 and 102, 122 and 110, 186 and 136).
//
// Then a few lanes sum a row's positions.  Words' frequencies are skewed: a row
// of more than a window's positions is summed in windows of places of the
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
// before it, which writes the same values.  Written past the caches, which the
// table's frequent rows keep: 65,536 tokens of 50,021 x 2048 float32 145 us (152
// through them), 4.6 TB/s of 665 MB; 402,413 of 159 x 90 float16 16 us.
template <typename T, typename I, int V>
__global__ __launch_bounds__(kBlock) void k_embed(const I *__restrict__ tokens, long long n,
                                                  const T *__restrict__ table, long long rows,
                                                  long long stride, int dim, int lanes,
                                                  typename Wide<T>::type scale,
                                                  T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  const int per = kBlock / lanes;
  for (long long i = (long long)blockIdx.x * per + threadIdx.x / lanes; i < n;
       i += (long long)gridDim.x * per) {
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
      mmpn::store_vec<T, V, true>(dst + at, v);
    }
  }
}

// ---------------------------------------------------------------- grouping
using mmpi::kDigits;
constexpr int kMaxTiles = 256;
constexpr int kSplitBlock = 1024, kSplitWaves = kSplitBlock / 64;

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
// The lanes of `among` whose d, a number of `bits` bits, is this lane's: with a
// ballot on each bit, unless it is the same for all.
__device__ __forceinline__ unsigned long long lanes_alike(unsigned long long among, unsigned d,
                                                          int bits) {
  if (among == 0) return 0;
  const int lead = __ffsll((long long)among) - 1;
  if ((__ballot(d == (unsigned)__builtin_amdgcn_readlane((int)d, lead)) & among) == among)
    return among;
  for (int b0 = 0; b0 < bits; b0 += 4)  // bits above the number's are 0 for all
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int set = (int)(d << (31 - b0 - b)) >> 31;  // all ones or 0
      among &= ~(__ballot(set) ^ (unsigned long long)(long long)set);
    }
  return among;
}

// Between one lane's access to its wave's counters and another lane's.  A wave's
// LDS accesses run in their order, so this only keeps the compiler from moving
// them: no instruction.
__device__ __forceinline__ void lanes_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// counters[d] += 1 for every lane of `among`, in a wave's own counters.  Lanes with
// one d are counted together: as atomics they would queue (131,072 equal tokens
// 186 us in k_group).
__device__ __forceinline__ void tally(unsigned *counters, bool there, unsigned d, int bits) {
  const unsigned long long same = lanes_alike(__ballot(there), d, bits);
  if (there && lanes_below(same) == 0) counters[d] += (unsigned)__popcll(same);
  lanes_in_order();
}

// The place among the equal d that a lane's entry takes: counters[d], which goes up
// by the lanes that have it, and the rank among those.
__device__ __forceinline__ unsigned take_place(unsigned *counters, unsigned long long among, bool there,
                                               unsigned d, int bits) {
  const unsigned long long same = lanes_alike(among, d, bits);
  const unsigned rank = lanes_below(same);
  unsigned at = 0;
  if (there) at = counters[d];
  lanes_in_order();
  if (there && rank == 0) counters[d] = at + (unsigned)__popcll(same);
  lanes_in_order();
  return at + rank;
}

// count[t][d]: entries of tile t with digit d = row >> shift & 255.  131,072 tokens
// 5 us, and 6 in k_split: chains of loads and counters in 128 workgroups.
template <typename S>
__global__ __launch_bounds__(kSplitBlock) void k_split_count(S src, unsigned tile_len, int shift,
                                                             unsigned *__restrict__ count) {
  __shared__ unsigned h[kSplitWaves][kDigits];
  const int tid = threadIdx.x, wave = tid >> 6;
  for (int k = tid; k < kSplitWaves * kDigits; k += kSplitBlock) h[0][k] = 0;
  __syncthreads();
  const unsigned n = src.count();
  const unsigned from = blockIdx.x * tile_len < n ? blockIdx.x * tile_len : n;
  const unsigned to = n - from < tile_len ? n : from + tile_len;
  for (unsigned i0 = from; i0 < to; i0 += kSplitBlock) {
    Entry e{0, 0};
    const bool there = i0 + tid < to && src.get(i0 + tid, e);
    tally(h[wave], there, e.row >> shift & (kDigits - 1), 8);
  }
  __syncthreads();
  if (tid < kDigits) {
    unsigned c = 0;
    for (int w = 0; w < kSplitWaves; ++w) c += h[w][tid];
    count[blockIdx.x * kDigits + tid] = c;
  }
}

// Places the entries by digit, otherwise in order; first[d] is where digit d
// begins, and first[256] the number of all.  Every workgroup adds up the
// counts of the tiles before its own, four threads a digit; a single one has
// no others (count is NULL).
template <typename S>
__global__ __launch_bounds__(kSplitBlock) void k_split(S src, unsigned tile_len, int shift,
                                                       const unsigned *__restrict__ count,
                                                       unsigned *__restrict__ first,
                                                       Entry *__restrict__ out) {
  constexpr int kEach = kSplitBlock / kDigits;
  __shared__ unsigned next[kSplitWaves][kDigits];
  __shared__ unsigned sums[2][kEach][kDigits], part[kDigits / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int k = tid; k < kSplitWaves * kDigits; k += kSplitBlock) next[0][k] = 0;
  const unsigned n = src.count();
  const unsigned piece = tile_len / kSplitWaves;
  unsigned from = blockIdx.x * tile_len + wave * piece;
  from = from < n ? from : n;
  const unsigned to = n - from < piece ? n : from + piece;
  if (count) {
    const int d = tid & (kDigits - 1);
    unsigned before = 0, total = 0;
#pragma unroll 16
    for (unsigned t = tid / kDigits; t < gridDim.x; t += kEach) {
      const unsigned c = count[t * kDigits + d];
      before += t < blockIdx.x ? c : 0;
      total += c;
    }
    sums[0][tid / kDigits][d] = before;
    sums[1][tid / kDigits][d] = total;
  }
  __syncthreads();
  for (unsigned i0 = from; i0 < to; i0 += 64) {
    Entry e{0, 0};
    const bool there = i0 + lane < to && src.get(i0 + lane, e);
    tally(next[wave], there, e.row >> shift & (kDigits - 1), 8);
  }
  if (!count) __syncthreads();
  unsigned total = 0, incl = 0;
  if (tid < kDigits) {
    if (count)
      for (int k = 0; k < kEach; ++k) total += sums[1][k][tid];
    else
      for (int w = 0; w < kSplitWaves; ++w) total += next[w][tid];
    incl = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    if (lane == 63) part[wave] = incl;
  }
  __syncthreads();
  if (tid < kDigits) {
    unsigned at = incl - total;
    for (int w = 0; w < wave; ++w) at += part[w];
    if (blockIdx.x == 0) {
      first[tid] = at;
      if (tid == kDigits - 1) first[kDigits] = at + total;
    }
    if (count)
      for (int k = 0; k < kEach; ++k) at += sums[0][k][tid];
#pragma unroll
    for (int w = 0; w < kSplitWaves; ++w) {
      const unsigned c = next[w][tid];
      next[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  for (unsigned i0 = from; i0 < to; i0 += 64) {
    Entry e{0, 0};
    const bool there = i0 + lane < to && src.get(i0 + lane, e);
    const unsigned at =
        take_place(next[wave], __ballot(there), there, e.row >> shift & (kDigits - 1), 8);
    if (there) out[at] = e;
  }
}

// A row's positions in the order.
struct Span {
  unsigned from, to;
};

// Workgroup g orders group g, the rows v with v % 256 = g, by v / 256: order has
// the positions, span the rows' places in it.  S is Entry, where k_split has
// placed the group's at first[g], or the tokens' type: then every workgroup
// looks for its own among all n tokens, at most 64 * kKept a wave, and
// workgroup 0 writes first[256] (two launches less: 2000 tokens of 60,000 x 8
// 34 to 19 us, 16,000 45 to 32).
using mmpi::kGroupBlock;
using mmpi::kKept;
template <typename S>
__global__ __launch_bounds__(kGroupBlock) void k_group(const S *__restrict__ src, unsigned n,
                                                       unsigned *__restrict__ first,
                                                       unsigned rows, unsigned bins, int bits,
                                                       int waves, Span *__restrict__ span,
                                                       unsigned *__restrict__ order) {
  constexpr bool kSplit = __is_same(S, Entry);
  // [waves][bins], 64 KiB at most; with the others up to 192 bytes more, of a CU's 160 KiB
  extern __shared__ unsigned next[];
  __shared__ unsigned part[kGroupBlock / 64], low[kGroupBlock / 64], all[kGroupBlock / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (unsigned k = tid; k < waves * bins; k += kGroupBlock) next[k] = 0;
  unsigned base = 0;
  if constexpr (kSplit) {
    base = first[blockIdx.x];
    n = first[blockIdx.x + 1] - base;
  }
  const unsigned per = (n + waves * 64 - 1) / (waves * 64) * 64;
  unsigned from = wave < waves ? wave * per : n;
  from = from < n ? from : n;
  const unsigned to = n - from < per ? n : from + per;
  unsigned *mine = next + wave * bins;
  __syncthreads();
  // Up to kKept entries a lane stay in registers, with their places among the
  // wave's of their row: then the second time through has no chain of counters.
  constexpr int kLoads = 4;
  const bool kept = per <= 64 * kKept;
  Entry e[kKept];
  unsigned place[kKept];
  unsigned long long there[kKept];
  if (kept) {
    unsigned lower = 0, valid = 0;
#pragma unroll
    for (int l = 0; l < kKept; ++l) {
      const unsigned i = from + l * 64 + lane;
      e[l] = {0, 0};
      bool ok = i < to;
      if constexpr (kSplit) {
        if (ok) e[l] = src[base + i];
      } else {
        const long long t = ok ? (long long)src[i] : -1;
        e[l] = {(unsigned)t, i};
        ok = t >= 0 && t < (long long)rows;
        const unsigned d = e[l].row % kDigits;
        lower += (unsigned)__popcll(__ballot(ok && d < blockIdx.x));
        valid += (unsigned)__popcll(__ballot(ok));
        ok = ok && d == blockIdx.x;
      }
      there[l] = __ballot(ok);
    }
    if constexpr (!kSplit)
      if (lane == 0) {
        low[wave] = lower;
        all[wave] = valid;
      }
#pragma unroll
    for (int l = 0; l < kKept; ++l) {
      if (there[l] == 0) continue;
      place[l] = take_place(mine, there[l], there[l] >> lane & 1, e[l].row / kDigits, bits);
    }
  } else if constexpr (kSplit) {
    for (unsigned i0 = from; i0 < to; i0 += 64 * kLoads) {
      unsigned row[kLoads];
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const unsigned i = i0 + l * 64 + lane;
        row[l] = src[base + (i < to ? i : from)].row;
      }
#pragma unroll
      for (int l = 0; l < kLoads; ++l) tally(mine, i0 + l * 64 + lane < to, row[l] / kDigits, bits);
    }
  }
  __syncthreads();
  if constexpr (!kSplit) {
    unsigned valid = 0;
#pragma unroll
    for (int w = 0; w < kGroupBlock / 64; ++w) {
      base += low[w];
      valid += all[w];
    }
    if (blockIdx.x == 0 && tid == 0) first[kDigits] = valid;
  }
  // exclusive sums over the rows, neighbouring ones a thread's, and within a
  // row over the waves
  const unsigned mult = (bins + kGroupBlock - 1) / kGroupBlock;
  unsigned total = 0;
  constexpr int kMostWaves = kGroupBlock / 64;
  for (unsigned k = tid * mult; k < (tid + 1) * mult && k < bins; ++k)
#pragma unroll
    for (int w = 0; w < kMostWaves; ++w)
      if (w < waves) total += next[w * bins + k];
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
    const unsigned begin = at, v = k * kDigits + blockIdx.x;
    unsigned c[kMostWaves];
#pragma unroll
    for (int w = 0; w < kMostWaves; ++w) c[w] = w < waves ? next[w * bins + k] : 0;
#pragma unroll
    for (int w = 0; w < kMostWaves; ++w)
      if (w < waves) {
        next[w * bins + k] = at;
        at += c[w];
      }
    if (v < rows) span[v] = {begin, at};
  }
  __syncthreads();
  if (kept) {
#pragma unroll
    for (int l = 0; l < kKept; ++l)
      if (there[l] >> lane & 1) order[mine[e[l].row / kDigits] + place[l]] = e[l].at;
    return;
  }
  if constexpr (kSplit) {
    for (unsigned i0 = from; i0 < to; i0 += 64 * kLoads) {
      Entry x[kLoads];
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const unsigned i = i0 + l * 64 + lane;
        x[l] = src[base + (i < to ? i : from)];
      }
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const bool is = i0 + l * 64 + lane < to;
        const unsigned at = take_place(mine, __ballot(is), is, x[l].row / kDigits, bits);
        if (is) order[at] = x[l].at;
      }
    }
  }
}

// From entries in the order of their rows: the same.
__global__ __launch_bounds__(kBlock) void k_starts(const Entry *__restrict__ entries,
                                                   const unsigned *__restrict__ count,
                                                   unsigned rows, Span *__restrict__ span,
                                                   unsigned *__restrict__ order) {
  const unsigned i = blockIdx.x * kBlock + threadIdx.x, n = *count;
  if (i < n) order[i] = entries[i].at;
  if (i >= rows) return;
  auto begin_of = [&](unsigned row) {  // the first entry of a row or a later one
    unsigned lo = 0, hi = n;
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (entries[mid].row < row) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  span[i] = {begin_of(i), begin_of(i + 1)};
}

// ---------------------------------------------------------------- row sums
constexpr int kInFlight = 4;  // vectors of a thread that are added, and as many on their way

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

// Window w of the order: the sums of its pieces of rows of more than `window`
// positions, part[2 w] of one that began before it and part[2 w + 1] of one
// that begins in it; begins[w] is that row, or -1.
template <typename T, typename I, int V>
__device__ __forceinline__ void window_sums(const I *__restrict__ tokens, const T *__restrict__ grad,
                                            long long stride, unsigned total, int dim, int lanes,
                                            unsigned window, unsigned w,
                                            const Span *__restrict__ span,
                                            const unsigned *__restrict__ order,
                                            typename Wide<T>::type *__restrict__ part,
                                            int *__restrict__ begins) {
  typedef typename Wide<T>::type A;
  const unsigned p0 = w * window, p1 = total - p0 < window ? total : p0 + window;
#pragma unroll 1
  for (int piece = 0; piece < 2; ++piece) {
    const long long r = (long long)tokens[order[piece ? p1 - 1 : p0]];
    const unsigned from = span[r].from, to = span[r].to;
    const bool mine = to - from > window && (from >= p0) == (piece == 1);
    if (piece == 1 && (threadIdx.x & (lanes - 1)) == 0) begins[w] = mine ? (int)r : -1;
    if (!mine) continue;
    for (int c = (threadIdx.x & (lanes - 1)) * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
      add_rows<T, V, kInFlight, A>(sum, grad, stride, order, from > p0 ? from : p0,
                                   to < p1 ? to : p1, at);
      Vec<A, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.e[k] = sum[k];
      mmpn::store_vec<A, V>(part + (2ll * w + piece) * dim + at, o);
    }
  }
}

// A row of more than a window's positions that begins in the window, whole: the
// workgroup's `lanes` threads side by side have some of its columns, and their
// sums of parts of the row are added up in LDS.
using mmpi::kWholeLanes;
constexpr int kWholeChunks = 64;
template <typename T, typename I, int V>
__device__ __forceinline__ void whole_row(const I *__restrict__ tokens, const T *__restrict__ grad,
                                          long long stride, unsigned total, int dim, int lanes,
                                          typename Wide<T>::type scale, unsigned window,
                                          unsigned w, int chunk, int chunks,
                                          const Span *__restrict__ span,
                                          const unsigned *__restrict__ order, T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  __shared__ A lds[kBlock * V];
  const unsigned p0 = w * window;
  if (p0 >= total) return;
  const long long r = (long long)tokens[order[total - p0 < window ? total - 1 : p0 + window - 1]];
  const unsigned from = span[r].from, to = span[r].to;
  if (to - from <= window || from < p0) return;
  const int slots = kBlock / lanes, slot = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  const unsigned each = (to - from + slots - 1) / slots;
  const unsigned f0 = from + slot * each < to ? from + slot * each : to;
  const unsigned t0 = to - f0 < each ? to : f0 + each;
  for (long long c0 = (long long)chunk * lanes * V; c0 < dim; c0 += (long long)chunks * lanes * V) {
    const long long c = c0 + lane * V;
    A sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0;
    if (c < dim)
      add_rows<T, V, kInFlight, A>(sum, grad, stride, order, f0, t0, c + V > dim ? dim - V : (int)c);
#pragma unroll
    for (int k = 0; k < V; ++k) lds[threadIdx.x * V + k] = sum[k];
    __syncthreads();
    const int j = threadIdx.x;  // a column of the chunk
    const long long cj = c0 + j / V * V;
    if (j < lanes * V && cj < dim) {
      A s = 0;
      for (int o = 0; o < slots; ++o) s += lds[o * lanes * V + j];
      out[r * dim + (cj + V > dim ? dim - V : cj) + j % V] = (T)(s * scale);
    }
    __syncthreads();
  }
}

// The first `window_blocks` workgroups sum windows (the longest work starts
// first).  The others have kRows rows of the gradient for `lanes` threads: those
// of up to kFirst positions, most of them, are read all at once (one
// after another they would wait for their order, then for their vectors), then
// those of up to a window.  With WHOLE they are `chunks` workgroups a window, and
// sum the long rows themselves.  Bound by the reads of scattered rows: 131,072 x 1024
// float16 into 64,000 rows 88 us, 4.5 TB/s.  More vectors in flight (kInFlight 8)
// take registers, 16 us more there.
constexpr int kRows = 4, kFirst = 2;
template <typename T, typename I, int V, bool WHOLE>
__global__ __launch_bounds__(kBlock) void k_row_sums(
    const I *__restrict__ tokens, const T *__restrict__ grad, long long stride, long long rows,
    int dim, int lanes, typename Wide<T>::type scale, unsigned window, unsigned window_blocks,
    int chunks, const Span *__restrict__ span, const unsigned *__restrict__ count,
    const unsigned *__restrict__ order, typename Wide<T>::type *__restrict__ part,
    int *__restrict__ begins, T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  const int per = kBlock / lanes, g = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  if (blockIdx.x < window_blocks) {
    if constexpr (WHOLE) {
      whole_row<T, I, V>(tokens, grad, stride, *count, dim,
                         lanes < kWholeLanes ? lanes : kWholeLanes, scale, window,
                         blockIdx.x / chunks, blockIdx.x % chunks, chunks, span, order, out);
      return;
    }
    const unsigned w = blockIdx.x * per + g, total = *count;
    if ((unsigned long long)w * window < total)
      window_sums<T, I, V>(tokens, grad, stride, total, dim, lanes, window, w, span, order, part,
                              begins);
    return;
  }
  const long long v = ((long long)(blockIdx.x - window_blocks) * per + g) * kRows;
  {
    Span p[kRows];
    unsigned id[kRows][kFirst];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      p[r] = {0, window + 1};  // not one of these rows
      if (v + r < rows) p[r] = span[v + r];
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int i = 0; i < kFirst; ++i)
        if (p[r].from + i < p[r].to && p[r].to - p[r].from <= kFirst) id[r][i] = order[p[r].from + i];
    for (int c = lane * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      Vec<T, V> x[kRows][kFirst];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < kFirst; ++i)
          if (p[r].from + i < p[r].to && p[r].to - p[r].from <= kFirst)
            x[r][i] = mmpn::load_vec<T, V, true>(grad + (long long)id[r][i] * stride + at);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        A sum[V];
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] = 0;
#pragma unroll
        for (int i = 0; i < kFirst; ++i)
          if (p[r].from + i < p[r].to) {
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += (A)x[r][i].e[k];
          }
        Vec<T, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = (T)(sum[k] * scale);
        if (p[r].to - p[r].from <= kFirst)
          mmpn::store_vec<T, V, true>(out + (v + r) * dim + at, o);
      }
    }
  }
#pragma unroll 1
  for (int r = 0; r < kRows && v + r < rows; ++r) {
    const unsigned from = span[v + r].from, to = span[v + r].to;
    if (to - from <= kFirst || to - from > window) continue;
    for (int c = lane * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
      add_rows<T, V, kInFlight, A>(sum, grad, stride, order, from, to, at);
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.e[k] = (T)(sum[k] * scale);
      mmpn::store_vec<T, V, true>(out + (v + r) * dim + at, o);
    }
  }
}

// Few tokens, two a lane: every row looks for its own among them, and no order
// is made (whose four launches take 17 us, one 5).
constexpr int kFew = 128, kFewRows = 4;
template <typename T, typename I, int V>
__global__ __launch_bounds__(kBlock) void k_row_sums_few(const I *__restrict__ tokens, int n,
                                                         const T *__restrict__ grad,
                                                         long long stride, long long rows, int dim,
                                                         int lanes, typename Wide<T>::type scale,
                                                         T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  const int wl = threadIdx.x & 63, lane = threadIdx.x & (lanes - 1);
  const long long low = wl < n ? (long long)tokens[wl] : -1;
  const long long high = wl + 64 < n ? (long long)tokens[wl + 64] : -1;
  const int per = kBlock / lanes;
  const long long v0 = (long long)blockIdx.x * per * kFewRows;
  const int together = lanes < 64 ? 64 / lanes : 1;  // rows of a wave at once
#pragma unroll 1
  for (int r = 0; r < kFewRows; ++r) {
    const long long v = v0 + r * per + threadIdx.x / lanes;
    // the wave's first row of this turn, and the masks of each of its rows
    const long long first = v0 + r * per + (threadIdx.x & ~63) / lanes;
    unsigned long long mine[2] = {0, 0};
    for (int k = 0; k < together; ++k) {
      const unsigned long long a = __ballot(low == first + k), b = __ballot(high == first + k);
      if (v == first + k) {
        mine[0] = a;
        mine[1] = b;
      }
    }
    if (v >= rows) continue;
    for (int c = lane * V; c < dim; c += lanes * V) {
      const int at = c + V > dim ? dim - V : c;
      A sum[V];
#pragma unroll
      for (int k = 0; k < V; ++k) sum[k] = 0;
#pragma unroll
      for (int part = 0; part < 2; ++part)
        for (unsigned long long left = mine[part]; left;) {
          constexpr int kLoads = 8;
          Vec<T, V> x[kLoads];
          bool there[kLoads];
#pragma unroll
          for (int l = 0; l < kLoads; ++l) {
            there[l] = left != 0;
            if (there[l]) {
              const int i = __ffsll((long long)left) - 1 + part * 64;
              x[l] = mmpn::load_vec<T, V>(grad + (long long)i * stride + at);
            }
            left &= left - 1;
          }
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (there[l]) {
#pragma unroll
              for (int k = 0; k < V; ++k) sum[k] += (A)x[l].e[k];
            }
        }
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) o.e[k] = (T)(sum[k] * scale);
      mmpn::store_vec<T, V, true>(out + v * dim + at, o);
    }
  }
}

// The rows in windows, of those that begin in kLongWindows windows kLongCols
// columns a workgroup, whose threads add up windows in kLongParts parts.  Its rows
// come one after another: with 32 windows a workgroup 478 x 113 by 59,961 tokens
// take 4 us more.
constexpr int kLongWindows = 8, kLongCols = 64, kLongParts = 16;
template <typename T>
__global__ __launch_bounds__(kBlock) void k_long_rows(
    int dim, typename Wide<T>::type scale, unsigned window, const Span *__restrict__ span,
    const unsigned *__restrict__ count, const typename Wide<T>::type *__restrict__ part,
    const int *__restrict__ begins, T *__restrict__ out) {
  typedef typename Wide<T>::type A;
  constexpr int V = kLongCols * kLongParts / kBlock;  // columns of a thread
  __shared__ A lds[kLongParts][kLongCols];
  __shared__ unsigned long long there;
  __shared__ int row_of[kLongWindows];
  const int c = (threadIdx.x % (kLongCols / V)) * V, g = threadIdx.x / (kLongCols / V);
  const unsigned chunks = (dim + kLongCols - 1) / kLongCols;
  const unsigned first = blockIdx.x / chunks * kLongWindows;
  const int c0 = (int)(blockIdx.x % chunks) * kLongCols;
  if (threadIdx.x < 64) {
    const unsigned w = first + threadIdx.x;
    int v = -1;
    if (threadIdx.x < kLongWindows && (unsigned long long)w * window < *count) v = begins[w];
    const unsigned long long m = __ballot(v >= 0);
    if (v >= 0) row_of[threadIdx.x] = v;
    if (threadIdx.x == 0) there = m;
  }
  __syncthreads();
  for (unsigned long long left = there; left; left &= left - 1) {
    const long long v = row_of[__ffsll((long long)left) - 1];
    const unsigned w0 = span[v].from / window, w1 = (span[v].to - 1) / window;
    const unsigned each = (w1 - w0 + kLongParts) / kLongParts;
    const unsigned from = w0 + g * each, to = from + each < w1 + 1 ? from + each : w1 + 1;
    A sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0;
    if (c0 + c + V <= dim) {
#pragma unroll 8
      for (unsigned w = from; w < to; ++w) {
        const Vec<A, V> x = mmpn::load_vec<A, V>(part + (2ll * w + (w == w0)) * dim + c0 + c);
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += x.e[k];
      }
    } else {
      for (unsigned w = from; w < to; ++w)
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c0 + c + k < dim) sum[k] += part[(2ll * w + (w == w0)) * dim + c0 + c + k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) lds[g][c + k] = sum[k];
    __syncthreads();
    if (threadIdx.x < kLongCols && c0 + (int)threadIdx.x < dim) {
      A s = 0;
#pragma unroll
      for (int o = 0; o < kLongParts; ++o) s += lds[o][threadIdx.x];
      out[v * dim + c0 + threadIdx.x] = (T)(s * scale);
    }
    __syncthreads();
  }
}

// Threads a row: enough for its vectors, a power of two up to the workgroup.
inline int row_lanes(int64_t dim, int vec) {
  int lanes = 1;
  while (lanes < kBlock && (int64_t)lanes * vec < dim) lanes <<= 1;
  return lanes;
}

constexpr int64_t kMost = 0x7fff0000LL;  // room for a step past the end in 32 bits

// Orders the tokens' positions by row; ea, eb: room for n entries each.
template <typename I>
int order_tokens(unsigned n, const I *tokens, unsigned rows, Entry *ea, Entry *eb, unsigned *count,
                 unsigned *first, Span *span, unsigned *order) {
  // up to 256 tiles of at least 1024 tokens, which every workgroup of k_split
  // adds up
  const unsigned tile = (unsigned)(mmpi::ceil_div(mmpi::ceil_div(n, kMaxTiles), 1024) * 1024);
  const unsigned tiles = (unsigned)mmpi::ceil_div(n, tile);
  auto pass = [&](auto src, int shift, Entry *out) -> int {
    typedef decltype(src) S;
    if (tiles > 1) {
      hipLaunchKernelGGL((k_split_count<S>), dim3(tiles), dim3(kSplitBlock), 0, mmpi::stream(),
                         src, tile, shift, count);
      if (int st = mmpi::check_launch("mmp_embedding_grad(count)")) return st;
    }
    hipLaunchKernelGGL((k_split<S>), dim3(tiles), dim3(kSplitBlock), 0, mmpi::stream(), src,
                       tile, shift, tiles > 1 ? (const unsigned *)count : nullptr, first, out);
    return mmpi::check_launch("mmp_embedding_grad(split)");
  };
  if (mmpi::in_groups(n, rows)) {
    const unsigned bins = (unsigned)mmpi::group_bins(rows);
    int bits = 0;
    while ((bins - 1) >> bits) ++bits;
    const int waves = mmpi::group_waves(rows);
    const dim3 grid(rows < kDigits ? rows : kDigits);
    const unsigned lds = (unsigned)waves * bins * 4;
    if (mmpi::in_one_group_pass(n, rows)) {
      hipLaunchKernelGGL((k_group<I>), grid, dim3(kGroupBlock), lds, mmpi::stream(), tokens, n,
                         first, rows, bins, bits, waves, span, order);
    } else {
      if (int st = pass(Tokens<I>{tokens, n, rows}, 0, ea)) return st;
      hipLaunchKernelGGL((k_group<Entry>), grid, dim3(kGroupBlock), lds, mmpi::stream(),
                         (const Entry *)ea, n, first, rows, bins, bits, waves, span, order);
    }
    return mmpi::check_launch("mmp_embedding_grad(group)");
  }
  if (int st = pass(Tokens<I>{tokens, n, rows}, 0, ea)) return st;
  for (int p = 1; p < mmpi::row_passes(rows); ++p) {
    if (int st = pass(Entries{ea, first + kDigits}, 8 * p, eb)) return st;
    Entry *t = ea;
    ea = eb;
    eb = t;
  }
  const unsigned most = n > rows ? n : rows;
  hipLaunchKernelGGL(k_starts, dim3((unsigned)mmpi::ceil_div(most, kBlock)), dim3(kBlock), 0,
                     mmpi::stream(), (const Entry *)ea, (const unsigned *)(first + kDigits), rows,
                     span, order);
  return mmpi::check_launch("mmp_embedding_grad(starts)");
}

template <typename T, typename I>
int grad_impl(int64_t n, const I *tokens, const T *grad, int64_t stride, int64_t rows, int dim,
              double scale, T *out) {
  typedef typename Wide<T>::type A;
  constexpr int V = 16 / sizeof(T);
  const int vec = dim >= V ? V : 1;
  const int lanes = row_lanes(dim, vec);
  if (n <= kFew) {
    const int64_t blocks = mmpi::ceil_div(rows, kBlock / lanes * kFewRows);
    if (!mmpi::grid_fits(blocks, kBlock))
      return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: too many rows");
    auto kernel = vec == V ? k_row_sums_few<T, I, V> : k_row_sums_few<T, I, 1>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(), tokens,
                       (int)n, grad, (long long)stride, (long long)rows, dim, lanes, (A)scale, out);
    return mmpi::check_launch("mmp_embedding_grad(few)");
  }
  // One block for all: sums of windows, entries, places of rows, the order,
  // rows that begin in windows, counts of tiles, beginnings of groups.
  mmpn::Temp temp;
  size_t size = 0;
  auto place = [&](size_t bytes) {
    const size_t at = size;
    size += (bytes + 255) / 256 * 256;
    return at;
  };
  const bool whole = mmpi::long_rows_whole(n, rows, lanes);
  const unsigned window = (unsigned)mmpi::row_window(n, lanes, whole);
  const int64_t windows = mmpi::ceil_div(n, window);
  const size_t at_part = place(whole ? 0 : (size_t)windows * 2 * dim * sizeof(A));
  const size_t entry_lists = whole ? 0 : mmpi::in_groups(n, rows) ? 1 : 2;
  const size_t at_entries = place((size_t)n * sizeof(Entry) * entry_lists);
  const size_t at_span = place((size_t)rows * sizeof(Span));
  const size_t at_order = place((size_t)n * 4), at_begins = place((size_t)windows * 4);
  const size_t at_count = place(kMaxTiles * kDigits * 4), at_first = place((kDigits + 1) * 4);
  if (int st = temp.get(size, "mmp_embedding_grad")) return st;
  char *base = (char *)temp.p;
  A *part = (A *)(base + at_part);
  Entry *entries = (Entry *)(base + at_entries);
  Span *span = (Span *)(base + at_span);
  unsigned *order = (unsigned *)(base + at_order), *first = (unsigned *)(base + at_first);
  int *begins = (int *)(base + at_begins);
  if (int st = order_tokens<I>((unsigned)n, tokens, (unsigned)rows, entries, entries + n,
                               (unsigned *)(base + at_count), first, span, order))
    return st;
  int64_t chunks = 1, wblocks = mmpi::ceil_div(windows, kBlock / lanes);
  if (whole) {
    chunks = mmpi::ceil_div(dim, (int64_t)(lanes < kWholeLanes ? lanes : kWholeLanes) * vec);
    if (chunks > kWholeChunks) chunks = kWholeChunks;
    wblocks = windows * chunks;
  }
  const int64_t blocks = mmpi::ceil_div(rows, kBlock / lanes * kRows) + wblocks;
  if (!mmpi::grid_fits(blocks, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: too many rows or tokens");
  auto kernel = whole ? (vec == V ? k_row_sums<T, I, V, true> : k_row_sums<T, I, 1, true>)
                      : (vec == V ? k_row_sums<T, I, V, false> : k_row_sums<T, I, 1, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(), tokens, grad,
                     (long long)stride, (long long)rows, dim, lanes, (A)scale, window,
                     (unsigned)wblocks, (int)chunks, (const Span *)span, (const unsigned *)first + kDigits,
                     (const unsigned *)order, part, begins, out);
  if (int st = mmpi::check_launch("mmp_embedding_grad")) return st;
  if (whole) return MMP_OK;
  const int64_t lblocks = mmpi::ceil_div(windows, kLongWindows) * mmpi::ceil_div(dim, kLongCols);
  if (!mmpi::grid_fits(lblocks, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: too many tokens and columns");
  hipLaunchKernelGGL((k_long_rows<T>), dim3((unsigned)lblocks), dim3(kBlock), 0, mmpi::stream(),
                     dim, (A)scale, window, (const Span *)span, (const unsigned *)first + kDigits,
                     (const A *)part, (const int *)begins, out);
  return mmpi::check_launch("mmp_embedding_grad(long)");
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
  if (dim > kMost) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding: rows of 2^31 elements");
  MMP_DISPATCH_FLOAT(dtype, "mmp_embedding", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_embedding", {
      constexpr int V = 16 / sizeof(T);
      const int vec = dim >= V ? V : 1;
      const int lanes = row_lanes(dim, vec);
      int64_t blocks = mmpi::ceil_div(n, kBlock / lanes);
      if (blocks > 1 << 22) blocks = 1 << 22;  // then a workgroup takes several turns
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
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_embedding_grad: 2^31 tokens, rows or columns");
  MMP_DISPATCH_FLOAT(dtype, "mmp_embedding_grad", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_embedding_grad", {
      return grad_impl<T, I>(n, (const I *)tokens, (const T *)grad, row_stride, rows, (int)dim,
                             scale, (T *)out);
    })
  })
}
