// loss.hip -- softmax cross entropy of rows of logits, and its gradient.
//
//   loss = log(sum exp(x)) - x_t        grad = w (softmax(x) - onehot(t))
//
// computed as m + log(sum exp(x - m)) with m the row's maximum.  A target
// outside [0, classes) is an ignored row: loss 0 and gradient 0, whatever its
// logits hold.  Statistics are held in 32 bits (64 for float64).  Logits of -inf
// are classes that cannot be: they add nothing and get no gradient.  A row
// that holds nothing else, or a logit of +inf, has no distribution and gives
// NaN.
#include "mmp_nn.h"

namespace {

using mmpn::Wide;

constexpr int kBlock = 256;

// A maximum and the sum of exponentials relative to it.
template <typename A> struct Stat {
  A m, s;
};
template <typename A> __device__ __forceinline__ Stat<A> join(Stat<A> a, Stat<A> b) {
  // the larger maximum, NaN if either is; of equal ones (also -inf, where the
  // difference would be NaN) both sums as they are
  const A m = a.m != a.m ? a.m : b.m != b.m ? b.m : a.m > b.m ? a.m : b.m;
  const A ea = a.m == m ? (A)1 : mmpn::exp_of(a.m - m);
  const A eb = b.m == m ? (A)1 : mmpn::exp_of(b.m - m);
  return {m, a.s * ea + b.s * eb};
}

template <typename T, typename I>
__global__ __launch_bounds__(kBlock) void k_loss(const T *__restrict__ logits, long long classes,
                                                 long long stride, const I *__restrict__ targets,
                                                 const typename Wide<T>::type *__restrict__ weight,
                                                 double scale,
                                                 typename Wide<T>::type *__restrict__ loss,
                                                 T *__restrict__ grad) {
  typedef typename Wide<T>::type A;
  __shared__ A sm[kBlock / 64], ss[kBlock / 64];
  const long long row = blockIdx.x;
  const long long t = (long long)targets[row];
  const T *x = logits + row * stride;
  T *g = grad ? grad + row * classes : nullptr;
  if (t < 0 || t >= classes) {
    if (threadIdx.x == 0) loss[row] = 0;
    if (g)
      for (long long c = threadIdx.x; c < classes; c += kBlock) g[c] = (T)0;
    return;
  }
  A m = -__builtin_inf();
  for (long long c = threadIdx.x; c < classes; c += kBlock) {
    const A v = (A)x[c];
    m = v > m || v != v ? v : m;
  }
  A s = 0;
  for (long long c = threadIdx.x; c < classes; c += kBlock) {
    const A v = (A)x[c];
    s += mmpn::exp_of(v - m);
  }
  Stat<A> st{m, m == -__builtin_inf() ? (A)0 : s};  // nothing but -inf: their differences are NaN
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) st = join(st, Stat<A>{__shfl_xor(st.m, d, 64), __shfl_xor(st.s, d, 64)});
  if ((threadIdx.x & 63) == 0) {
    sm[threadIdx.x >> 6] = st.m;
    ss[threadIdx.x >> 6] = st.s;
  }
  __syncthreads();
  st = {sm[0], ss[0]};
#pragma unroll
  for (int w = 1; w < kBlock / 64; ++w) st = join(st, Stat<A>{sm[w], ss[w]});
  if (threadIdx.x == 0) {
    if constexpr (sizeof(A) == 8) loss[row] = (st.m - (A)x[t]) + log(st.s);
    else loss[row] = (st.m - (A)x[t]) + logf(st.s);
  }
  if (!g) return;
  const A w = (A)scale * (weight ? weight[row] : (A)1), inv = (A)1 / st.s;
  for (long long c = threadIdx.x; c < classes; c += kBlock) {
    const A p = mmpn::exp_of((A)x[c] - st.m) * inv;
    g[c] = (T)((c == t ? p - 1 : p) * w);
  }
}

}  // namespace

extern "C" int mmp_cross_entropy(int dtype, int index_dtype, int64_t rows, int64_t classes,
                                 const void *logits, int64_t row_stride, const void *targets,
                                 const void *weight, double scale, void *loss, void *grad) {
  if (int st = mmpi::ensure_init()) return st;
  if (rows < 0 || classes < 0) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: negative extent");
  if (rows == 0) return MMP_OK;
  if (classes == 0) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: no classes");
  if (!logits || !targets || !loss) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: null pointer");
  if (!mmpi::grid_fits(rows, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: too many rows");
  MMP_DISPATCH_FLOAT(dtype, "mmp_cross_entropy", {
    MMP_DISPATCH_INDEX(index_dtype, "mmp_cross_entropy", {
      typedef typename Wide<T>::type A;
      hipLaunchKernelGGL((k_loss<T, I>), dim3((unsigned)rows), dim3(kBlock), 0, mmpi::stream(),
                         (const T *)logits, (long long)classes, (long long)row_stride,
                         (const I *)targets, (const A *)weight, scale, (A *)loss, (T *)grad);
      return mmpi::check_launch("mmp_cross_entropy");
    })
  })
}
