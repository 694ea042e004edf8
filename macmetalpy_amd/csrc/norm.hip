// norm.hip -- the norm of many arrays together, and their scaling down to a
// limit.
//
//   norm = sqrt(sum over all arrays of squares),  out = x * min(1, limit / norm)
//
// Squares and sums are held in 64 bits: a float32 gradient's square can
// overflow 32.  The arrays are cut into chunks; a workgroup sums one, and the
// chunks' sums are added in their order by one workgroup (up to 1024 of them by
// every workgroup of the second pass, which saves a launch), so the norm's bits
// do not depend on timing.
//
// Bound by memory: the limit needs the norm first, so the arrays are read twice
// and written once.  600,000,011 float16 in 60 arrays 632 us, 5.7 TB/s over the three:
// 203 squares, 429 scaling, which goes backwards; 60,001 float32 in 40 arrays 4.4 and
// 4.2, two launches.
//
// A chunk is read and written by its own workgroup, so an array may be scaled in
// place, but memory that two of them share would be scaled once or twice, by
// timing.  The host refuses that.
#include <memory>
#include <new>

#include "mmp_nn.h"

namespace {

using mmpn::Vec;
using mmpn::Wide;

constexpr int kBlock = 256, kNormBlock = 1024;
constexpr int kArrays = 64;  // of one launch: they go in the kernel's arguments

struct Table {
  const void *in[kArrays];
  void *out[kArrays];
  long long n[kArrays];
  unsigned first[kArrays];  // the array's first chunk
  int count;
};

// The array that a chunk belongs to.
__device__ __forceinline__ int array_of(const Table &t, unsigned chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int BLOCK> __device__ __forceinline__ double block_sum(double s, double *lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  double r = 0;
#pragma unroll
  for (int w = 0; w < BLOCK / 64; ++w) r += lds[w];
  return r;
}

// The elements of a chunk that are before the first address that is a multiple
// of 16, then vectors of 16 bytes, then the rest.
template <typename T> struct Chunk {
  static constexpr int V = 16 / sizeof(T);
  const T *x;
  long long from, to;  // of the array
  long long head, vecs;
  int array;
  __device__ __forceinline__ Chunk(const Table &t, unsigned chunk, long long chunk_len) {
    array = array_of(t, chunk);
    from = (long long)(chunk - t.first[array]) * chunk_len;
    to = t.n[array] - from < chunk_len ? t.n[array] : from + chunk_len;
    x = (const T *)t.in[array] + from;
    const long long n = to - from;
    head = (long long)((16 - ((uintptr_t)x & 15)) & 15) / (long long)sizeof(T);
    head = head < n ? head : n;
    vecs = (n - head) / V;
  }
};

// A vector's squares.  float16's fit 32 bits without rounding; wider ones are
// widened first.
template <typename T> __device__ __forceinline__ double squares(const Vec<T, 16 / sizeof(T)> &v) {
  double s = 0;
#pragma unroll
  for (int k = 0; k < (int)(16 / sizeof(T)); ++k) {
    if constexpr (sizeof(T) == 2) s += (double)((float)v.e[k] * (float)v.e[k]);
    else s = __builtin_fma((double)v.e[k], (double)v.e[k], s);
  }
  return s;
}

constexpr int kLoads = 8;  // vectors of a thread in flight

template <typename T>
__global__ __launch_bounds__(kBlock) void k_squares(Table t, long long chunk_len,
                                                    double *__restrict__ part) {
  __shared__ double lds[kBlock / 64];
  const Chunk<T> c(t, blockIdx.x, chunk_len);
  const T *x = c.x + c.head;
  double s = 0;
  for (long long i0 = threadIdx.x; i0 < c.vecs; i0 += kLoads * kBlock) {
    Vec<T, Chunk<T>::V> v[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (i0 + l * kBlock < c.vecs)
        v[l] = mmpn::load_vec<T, Chunk<T>::V>(x + (i0 + l * kBlock) * Chunk<T>::V);
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (i0 + l * kBlock < c.vecs) s += squares<T>(v[l]);
  }
  // at most 7 elements before the vectors and 7 after them
  const long long rest = c.to - c.from - c.vecs * Chunk<T>::V;
  if (threadIdx.x < rest) {
    const double v = (double)c.x[threadIdx.x < c.head ? threadIdx.x : threadIdx.x + c.vecs * Chunk<T>::V];
    s = __builtin_fma(v, v, s);
  }
  s = block_sum<kBlock>(s, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the chunks' sums, in the same order wherever it is called.
template <int BLOCK> __device__ __forceinline__ double norm_of(const double *part, int n, double *lds) {
  double s = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += BLOCK) s += part[i];
  return sqrt(block_sum<BLOCK>(s, lds));
}
__device__ __forceinline__ void put_norm(void *norm, bool wide, double v) {
  if (wide) *(double *)norm = v;
  else *(float *)norm = (float)v;
}

template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void k_norm(const double *__restrict__ part, int n, bool wide,
                                                void *__restrict__ norm, double *__restrict__ full) {
  __shared__ double lds[BLOCK / 64];
  const double s = norm_of<BLOCK>(part, n, lds);
  if (threadIdx.x == 0) {
    put_norm(norm, wide, s);
    *full = s;
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_clip(Table t, long long chunk_len, double limit,
                                                 const double *__restrict__ part, int parts,
                                                 bool wide, void *__restrict__ norm) {
  typedef typename Wide<T>::type A;
  constexpr int V = Chunk<T>::V;
  // backwards: what was summed last is the likeliest to be in a cache
  const Chunk<T> c(t, gridDim.x - 1 - blockIdx.x, chunk_len);
  const T *x = c.x + c.head;
  T *y0 = (T *)t.out[c.array] + c.from, *y = y0 + c.head;
  // few sums: every workgroup adds them up by itself; else *part is the norm
  __shared__ double lds[kBlock / 64];
  const double n = parts ? norm_of<kBlock>(part, parts, lds) : *part;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) put_norm(norm, wide, n);
  // a norm that is NaN scales by NaN: a broken step shows
  const A by = (A)(n <= limit ? 1.0 : limit / n);
  if (by == 1 && y0 == c.x) return;  // in place, and nothing to change
  // A factor below the normal range has few bits or none, though its products
  // need not be below: large elements, a small limit.  Those are divided and
  // multiplied in 64 bits.  (float16 ones would all be 0.)
  if constexpr (sizeof(T) > 2) {
    if (limit > 0 && by < (A)(sizeof(T) == 4 ? 0x1p-126 : 0x1p-1022)) {
      for (long long i = threadIdx.x; i < c.to - c.from; i += kBlock)
        y0[i] = (T)((double)c.x[i] / n * limit);
      return;
    }
  }
  auto scaled = [&](const Vec<T, V> &v) {
    Vec<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.e[k] = (T)((A)v.e[k] * by);
    return r;
  };
  for (long long i0 = threadIdx.x; i0 < c.vecs; i0 += kLoads * kBlock) {
    Vec<T, V> v[kLoads];
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (i0 + l * kBlock < c.vecs) v[l] = mmpn::load_vec<T, V, true>(x + (i0 + l * kBlock) * V);
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (i0 + l * kBlock < c.vecs)
        mmpn::store_vec<T, V, true>(y + (i0 + l * kBlock) * V, scaled(v[l]));
  }
  const long long rest = c.to - c.from - c.vecs * V;
  if (threadIdx.x < rest) {
    const long long i = threadIdx.x < c.head ? threadIdx.x : threadIdx.x + c.vecs * V;
    y0[i] = (T)((A)c.x[i] * by);
  }
}

// Refuses outputs that share memory with another array's input or output, or
// with a part of their own input.
int check_outs(int64_t count, const int *dtypes, const int64_t *sizes, const void *const *arrays,
               void *const *outs) {
  std::unique_ptr<mmpi::Extent[]> extents(new (std::nothrow) mmpi::Extent[2 * count]);
  if (!extents) return mmpi::fail(MMP_E_OOM, "mmp_clip_norm: %lld arrays", (long long)count);
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    const unsigned long long in = (uintptr_t)arrays[i], out = (uintptr_t)outs[i];
    const unsigned long long bytes =
        (unsigned long long)sizes[i] * (dtypes[i] == MMP_F16 ? 2 : dtypes[i] == MMP_F32 ? 4 : 8);
    extents[n++] = {out, out + bytes, true};
    if (in != out) extents[n++] = {in, in + bytes, false};
  }
  if (mmpi::written_overlap(extents.get(), n))
    return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: an output overlaps another array");
  return MMP_OK;
}

}  // namespace

extern "C" int mmp_clip_norm(int64_t count, const int *dtypes, const int64_t *sizes,
                             const void *const *arrays, void *const *outs, double limit,
                             int norm_dtype, void *norm) {
  if (int st = mmpi::ensure_init()) return st;
  if (count < 0) return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: negative count");
  if (!norm || (count > 0 && (!dtypes || !sizes || !arrays)))
    return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: null pointer");
  if (outs && !(limit >= 0)) return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: limit %g", limit);
  if (norm_dtype != MMP_F32 && norm_dtype != MMP_F64)
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_clip_norm: norm dtype code %d", norm_dtype);
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0) return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: negative extent");
    if (dtypes[i] != MMP_F16 && dtypes[i] != MMP_F32 && dtypes[i] != MMP_F64)
      return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_clip_norm: dtype code %d is not floating", dtypes[i]);
    if (sizes[i] > 0 && (!arrays[i] || (outs && !outs[i])))
      return mmpi::fail(MMP_E_ARG, "mmp_clip_norm: null pointer");
    total += sizes[i];
  }
  if (outs && count > 0)
    if (int st = check_outs(count, dtypes, sizes, arrays, outs)) return st;
  // About 4096 chunks, of 4096 elements at least.
  int64_t chunk = mmpi::ceil_div(mmpi::ceil_div(total, 4096), 4096) * 4096;
  if (chunk == 0) chunk = 4096;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += mmpi::ceil_div(sizes[i], chunk);
  mmpn::Temp part;
  if (int st = part.get((size_t)(chunks + 1) * 8, "mmp_clip_norm")) return st;
  double *sums = (double *)part.p, *full = sums + chunks;
  const bool wide = norm_dtype == MMP_F64;
  if (chunks > 0x7fffffffLL) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_clip_norm: too many arrays");
  // Up to this many sums the second pass adds them up without a launch between.
  const bool few = chunks > 0 && chunks <= 1024 && outs;
  void *norm_left = norm;  // to be written by the second pass's first launch
  // Arrays of one type are launched together, up to kArrays of them.
  for (int pass = 0; pass < 2; ++pass) {
    int64_t done = 0;
    for (int dtype = MMP_F16; dtype <= MMP_F64; ++dtype) {
      Table t;
      int64_t of = 0;
      t.count = 0;
      auto launch = [&]() -> int {
        const dim3 grid((unsigned)of), block(kBlock);
        MMP_DISPATCH_FLOAT(dtype, "mmp_clip_norm", {
          if (pass == 0)
            hipLaunchKernelGGL((k_squares<T>), grid, block, 0, mmpi::stream(), t, (long long)chunk,
                               sums + done);
          else
            hipLaunchKernelGGL((k_clip<T>), grid, block, 0, mmpi::stream(), t, (long long)chunk,
                               limit, (const double *)(few ? sums : full), few ? (int)chunks : 0, wide,
                               few ? norm_left : nullptr);
          break;
        })
        if (pass == 1) norm_left = nullptr;
        done += of;
        of = 0;
        t.count = 0;
        return mmpi::check_launch("mmp_clip_norm");
      };
      for (int64_t i = 0; i < count; ++i) {
        if (dtypes[i] != dtype || sizes[i] == 0) continue;
        t.in[t.count] = arrays[i];
        t.out[t.count] = outs ? outs[i] : nullptr;
        t.n[t.count] = sizes[i];
        t.first[t.count] = (unsigned)of;
        of += mmpi::ceil_div(sizes[i], chunk);
        if (++t.count == kArrays)
          if (int st = launch()) return st;
      }
      if (t.count)
        if (int st = launch()) return st;
    }
    if (pass == 1) break;
    if (few) continue;
    if (chunks <= 1024)
      hipLaunchKernelGGL((k_norm<kBlock>), dim3(1), dim3(kBlock), 0, mmpi::stream(),
                         (const double *)sums, (int)chunks, wide, norm, full);
    else
      hipLaunchKernelGGL((k_norm<kNormBlock>), dim3(1), dim3(kNormBlock), 0, mmpi::stream(),
                         (const double *)sums, (int)chunks, wide, norm, full);
    if (int st = mmpi::check_launch("mmp_clip_norm(norm)")) return st;
    if (!outs) break;
  }
  return MMP_OK;
}
