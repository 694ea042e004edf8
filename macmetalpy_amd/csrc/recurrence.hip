// recurrence.hip -- a gated linear recurrence over sequences, and its gradient.
//
// Per channel, with the state in 32 bits (64 for float64):
//   gates as logits g:   f = 1 / (1 + exp(-g));  h_t = f h_{t-1} + (1 - f) x_t
//   gates as factors a:  h_t = a_t h_{t-1} + x_t
// The gradient runs the same recurrence backwards on what a step passes to
// the one before it: with c_T the final state's gradient,
//   d_t = grad_t + c_{t+1},  c_t = f_t d_t
//   logits:   grad_g = d_t (h_{t-1} - x_t) f (1 - f),  grad_x = d_t (1 - f)
//   factors:  grad_a = d_t h_{t-1},                    grad_x = d_t
// and c_0 is the initial state's gradient.
#include "mmp_nn.h"

namespace {

using mmpn::Wide;

constexpr int kBlock = 256;

// Steps of a (batch, steps, dim) array: adjacent channels, any other strides.
template <typename T> struct Steps {
  const T *p;
  long long sb, st;
};

template <typename T, bool LOGITS>
__global__ __launch_bounds__(kBlock) void k_recur(long long batch, long long steps, long long dim,
                                                  Steps<T> gate, Steps<T> x,
                                                  const typename Wide<T>::type *__restrict__ initial,
                                                  T *__restrict__ h,
                                                  typename Wide<T>::type *__restrict__ final_) {
  typedef typename Wide<T>::type A;
  const long long i = (long long)blockIdx.x * kBlock + threadIdx.x;
  if (i >= batch * dim) return;
  const long long b = i / dim, c = i - b * dim;
  A s = initial ? initial[i] : 0;
  for (long long t = 0; t < steps; ++t) {
    const A g = (A)gate.p[b * gate.sb + t * gate.st + c], v = (A)x.p[b * x.sb + t * x.st + c];
    A f = g, u = v;
    if constexpr (LOGITS) {
      A r;
      mmpn::sigmoid_pair(g, f, r);
      u = r * v;
    }
    s = mmpn::fma_of(f, s, u);
    h[(b * steps + t) * dim + c] = (T)s;
  }
  final_[i] = s;
}

template <typename T, bool LOGITS>
__global__ __launch_bounds__(kBlock) void k_recur_grad(
    long long batch, long long steps, long long dim, Steps<T> grad, Steps<T> gate, Steps<T> x,
    Steps<T> h, const typename Wide<T>::type *__restrict__ initial,
    const typename Wide<T>::type *__restrict__ grad_final, T *__restrict__ grad_gate,
    T *__restrict__ grad_x, typename Wide<T>::type *__restrict__ grad_initial) {
  typedef typename Wide<T>::type A;
  const long long i = (long long)blockIdx.x * kBlock + threadIdx.x;
  if (i >= batch * dim) return;
  const long long b = i / dim, c = i - b * dim;
  A carry = grad_final ? grad_final[i] : 0;
  for (long long t = steps - 1; t >= 0; --t) {
    const A g = (A)gate.p[b * gate.sb + t * gate.st + c];
    const A before = t > 0 ? (A)h.p[b * h.sb + (t - 1) * h.st + c] : initial ? initial[i] : 0;
    const A d = (A)grad.p[b * grad.sb + t * grad.st + c] + carry;
    const long long o = (b * steps + t) * dim + c;
    if constexpr (LOGITS) {
      A f, u;
      mmpn::sigmoid_pair(g, f, u);
      const A v = (A)x.p[b * x.sb + t * x.st + c], du = d * u;
      grad_gate[o] = (T)(du * f * (before - v));
      grad_x[o] = (T)du;
      carry = f * d;
    } else {
      grad_gate[o] = (T)(d * before);
      grad_x[o] = (T)d;
      carry = g * d;
    }
  }
  grad_initial[i] = carry;
}

}  // namespace

extern "C" int mmp_recurrence(int dtype, int logits, int64_t batch, int64_t steps, int64_t dim,
                              const void *gate, int64_t gate_sb, int64_t gate_st, const void *x,
                              int64_t x_sb, int64_t x_st, const void *initial, void *h,
                              void *final_) {
  if (int st = mmpi::ensure_init()) return st;
  if (batch < 0 || steps < 0 || dim < 0)
    return mmpi::fail(MMP_E_ARG, "mmp_recurrence: negative extent");
  if (batch == 0 || dim == 0) return MMP_OK;
  if (!final_ || (steps > 0 && (!gate || !x || !h)))
    return mmpi::fail(MMP_E_ARG, "mmp_recurrence: null pointer");
  const int64_t blocks = mmpi::ceil_div(batch * dim, kBlock);
  if (!mmpi::grid_fits(blocks, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence: too many channels");
  MMP_DISPATCH_FLOAT(dtype, "mmp_recurrence", {
    typedef typename Wide<T>::type A;
    auto kernel = logits ? k_recur<T, true> : k_recur<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(),
                       (long long)batch, (long long)steps, (long long)dim,
                       Steps<T>{(const T *)gate, gate_sb, gate_st},
                       Steps<T>{(const T *)x, x_sb, x_st}, (const A *)initial, (T *)h, (A *)final_);
    return mmpi::check_launch("mmp_recurrence");
  })
}

extern "C" int mmp_recurrence_grad(int dtype, int logits, int64_t batch, int64_t steps, int64_t dim,
                                   const void *grad, int64_t grad_sb, int64_t grad_st,
                                   const void *gate, int64_t gate_sb, int64_t gate_st,
                                   const void *x, int64_t x_sb, int64_t x_st, const void *h,
                                   int64_t h_sb, int64_t h_st, const void *initial,
                                   const void *grad_final, void *grad_gate, void *grad_x,
                                   void *grad_initial) {
  if (int st = mmpi::ensure_init()) return st;
  if (batch < 0 || steps < 0 || dim < 0)
    return mmpi::fail(MMP_E_ARG, "mmp_recurrence_grad: negative extent");
  if (batch == 0 || dim == 0) return MMP_OK;
  if (!grad_initial || (steps > 0 && (!grad || !gate || !x || !h || !grad_gate || !grad_x)))
    return mmpi::fail(MMP_E_ARG, "mmp_recurrence_grad: null pointer");
  const int64_t blocks = mmpi::ceil_div(batch * dim, kBlock);
  if (!mmpi::grid_fits(blocks, kBlock))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence_grad: too many channels");
  MMP_DISPATCH_FLOAT(dtype, "mmp_recurrence_grad", {
    typedef typename Wide<T>::type A;
    auto kernel = logits ? k_recur_grad<T, true> : k_recur_grad<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), 0, mmpi::stream(),
                       (long long)batch, (long long)steps, (long long)dim,
                       Steps<T>{(const T *)grad, grad_sb, grad_st},
                       Steps<T>{(const T *)gate, gate_sb, gate_st},
                       Steps<T>{(const T *)x, x_sb, x_st}, Steps<T>{(const T *)h, h_sb, h_st},
                       (const A *)initial, (const A *)grad_final, (T *)grad_gate, (T *)grad_x,
                       (A *)grad_initial);
    return mmpi::check_launch("mmp_recurrence_grad");
  })
}
