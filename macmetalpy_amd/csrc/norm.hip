// norm.hip -- the norm of many arrays together, and their scaling down to a
// limit.
//
//   norm = sqrt(sum over all arrays of squares),  out = x * min(1, limit / norm)
//
// Squares and sums are held in 64 bits: a float32 gradient's square can
// overflow 32.  The arrays are cut into chunks; a workgroup sums one, and the
// chunks' sums are added in their order by one workgroup, so the norm's bits
// do not depend on timing.
#include "mmp_nn.h"

namespace {

using mmpn::Vec;
using mmpn::Wide;

constexpr int kBlock = 256;
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

__device__ __forceinline__ double block_sum(double s, double *lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) s += __shfl_xor(s, m, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  double r = 0;
#pragma unroll
  for (int w = 0; w < kBlock / 64; ++w) r += lds[w];
  return r;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_squares(Table t, long long chunk_len,
                                                    double *__restrict__ part) {
  __shared__ double lds[kBlock / 64];
  const int a = array_of(t, blockIdx.x);
  const long long from = (long long)(blockIdx.x - t.first[a]) * chunk_len;
  const long long to = t.n[a] - from < chunk_len ? t.n[a] : from + chunk_len;
  const T *x = (const T *)t.in[a];
  double s = 0;
  for (long long i = from + threadIdx.x; i < to; i += kBlock) {
    const double v = (double)x[i];
    s = __builtin_fma(v, v, s);
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename N>
__global__ __launch_bounds__(kBlock) void k_norm(const double *__restrict__ part, long long n,
                                                 N *__restrict__ norm, double *__restrict__ full) {
  __shared__ double lds[kBlock / 64];
  double s = 0;
  for (long long i = threadIdx.x; i < n; i += kBlock) s += part[i];
  s = sqrt(block_sum(s, lds));
  if (threadIdx.x == 0) {
    *norm = (N)s;
    *full = s;
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void k_clip(Table t, long long chunk_len, double limit,
                                                 const double *__restrict__ norm) {
  typedef typename Wide<T>::type A;
  const int a = array_of(t, blockIdx.x);
  const long long from = (long long)(blockIdx.x - t.first[a]) * chunk_len;
  const long long to = t.n[a] - from < chunk_len ? t.n[a] : from + chunk_len;
  const T *x = (const T *)t.in[a];
  T *y = (T *)t.out[a];
  const double n = *norm;
  // a norm that is NaN scales by NaN: a broken step shows
  const A by = (A)(n <= limit ? 1.0 : limit / n);
  for (long long i = from + threadIdx.x; i < to; i += kBlock) y[i] = (T)((A)x[i] * by);
}

struct Temp {
  void *p = nullptr;
  ~Temp() {
    if (p) (void)mmp_free(p);
  }
  int get(size_t bytes) { return mmp_alloc(bytes ? bytes : 1, &p); }
};

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
  int64_t chunk = mmpi::ceil_div(total, 4096);
  chunk = chunk < 4096 ? 4096 : mmpi::ceil_div(chunk, 1024) * 1024;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += mmpi::ceil_div(sizes[i], chunk);
  Temp part;
  if (int st = part.get((size_t)(chunks + 1) * 8)) return st;
  double *sums = (double *)part.p, *full = sums + chunks;
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
                               limit, (const double *)full);
          break;
        })
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
    if (norm_dtype == MMP_F32)
      hipLaunchKernelGGL((k_norm<float>), dim3(1), dim3(kBlock), 0, mmpi::stream(),
                         (const double *)sums, (long long)chunks, (float *)norm, full);
    else
      hipLaunchKernelGGL((k_norm<double>), dim3(1), dim3(kBlock), 0, mmpi::stream(),
                         (const double *)sums, (long long)chunks, (double *)norm, full);
    if (int st = mmpi::check_launch("mmp_clip_norm(norm)")) return st;
    if (!outs) break;
  }
  return MMP_OK;
}
