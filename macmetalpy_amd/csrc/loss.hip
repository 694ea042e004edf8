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
//
// Bound by memory: the logits are read once and the gradient is written once,
// so a row whose gradient is wanted stays in registers between the two, from
// 8 threads of a wave with 4 vectors of 16 bytes each (256 float16 classes) to a
// workgroup of 1024 threads with 16 (131,072).  Longer rows are read again for
// their gradient, out of the last cache mostly.  The loss alone is one pass with a
// running maximum and sum.  Few long rows are cut into parts that their own
// workgroups sum, and joined by a second launch.
//
// Measured: 16,384 rows of 50,021 float16 with gradient 600 us, 5.5 TB/s; the loss
// alone of 2047 rows of 100,003 float32 131 us, 6.3 TB/s; 50 rows of 32,000 float16
// with gradient 8.5 us, a workgroup's chain of load, exponentials and store.
#include <iterator>
#include <utility>

#include "mmp_nn.h"

namespace {

using mmpn::Vec;
using mmpn::Wide;

template <typename T> constexpr int vec_of() { return 16 / sizeof(T); }

// exp(x - m) of an element.  The exponent's rounding grows with |x - m|, about
// 2^-24 of it; a float16 gradient has 11 bits of its own, so only wider ones correct
// it.  The loss takes that error weighted by the softmax, whose mean of m - x is at most
// log(classes) - log(sum): under the rounding of the loss itself (64 rows of 50,021
// normal logits times 0.5, 2.5 and 6: 17, 21 and 32 units of 2^-24 off at most, corrected
// or not).  Corrected, 16,384 rows of 50,021 with gradient take 715 us for 600.
template <typename T, typename A> __device__ __forceinline__ A exp_diff(A x, A m) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f((x - m) * 1.44269502f);
  else return mmpn::exp_of(x - m);
}

__device__ __forceinline__ float max_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float log_of(float x) { return logf(x); }
__device__ __forceinline__ double log_of(double x) { return log(x); }

// A maximum and the sum of exponentials relative to it.
template <typename A> struct Stat {
  A m, s;
};
// Of equal maxima (also -inf, where the difference would be NaN) both sums as
// they are.  A NaN is in the sum, so the maxima may leave it out.
template <typename A> __device__ __forceinline__ Stat<A> join(Stat<A> a, Stat<A> b) {
  const A m = max_of(a.m, b.m);
  const A ea = a.m == m ? (A)1 : mmpn::exp_of(a.m - m);
  const A eb = b.m == m ? (A)1 : mmpn::exp_of(b.m - m);
  return {m, a.s * ea + b.s * eb};
}

// A row as vectors of 16 bytes at addresses that are multiples of 16: the first
// may begin before the row and the last end after it (inside the same 16
// bytes, so inside the allocation); what is not the row's counts as -inf.
template <typename T> struct Row {
  static constexpr int V = vec_of<T>();
  const T *base;
  int head, classes, vecs;
  __device__ __forceinline__ Row(const T *x, int n)
      : head((int)(((uintptr_t)x & 15) / sizeof(T))), classes(n) {
    base = x - head;
    vecs = (int)(((long long)head + n + V - 1) / V);
  }
  typedef typename Vec<T, V>::Words Words;
  // vector v with what is outside of the row replaced; v < vecs
  template <bool STREAM> __device__ __forceinline__ Words load(int v) const {
    Words w = mmpn::words_of<T, V>(mmpn::load_vec<T, V, STREAM>(base + (long long)v * V));
    if (v == 0 || v == vecs - 1) {
      const Words fill = nothing();
      const int first = head - v * V;  // the row's first element, as one of this vector
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned keep = 0;
#pragma unroll
        for (int q = 0; q < (sizeof(T) == 2 ? 2 : 1); ++q) {
          const int k = (j * 4 + q * 2) / (int)sizeof(T);
          if ((unsigned)(k - first) < (unsigned)classes) keep |= sizeof(T) == 2 ? 0xffffu << (16 * q) : 0xffffffffu;
        }
        w[j] = (w[j] & keep) | (fill[j] & ~keep);
      }
    }
    return w;
  }
  static __device__ __forceinline__ Words nothing() {
    Vec<T, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.e[k] = (T)-__builtin_inff();
    return mmpn::words_of<T, V>(r);
  }
  // vector v of the row g of the gradient
  __device__ __forceinline__ void store(T *g, int v, const Vec<T, V> &r) const {
    const int first = head - v * V;
    T *p = g - first;
    if (v == 0 || v == vecs - 1) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if ((unsigned)(k - first) < (unsigned)classes) p[k] = r.e[k];
    } else {
      mmpn::store_vec<T, V, true>(p, r);
    }
  }
};

// The gradient of a vector; `at` is the target's place in it, if it is there.
template <typename T, typename A>
__device__ __forceinline__ Vec<T, vec_of<T>()> grad_of(
    typename Vec<T, vec_of<T>()>::Words words, A m, A by, A w, long long at) {
  const Vec<T, vec_of<T>()> x = mmpn::elements_of<T, vec_of<T>()>(words);
  Vec<T, vec_of<T>()> g;
#pragma unroll
  for (int k = 0; k < vec_of<T>(); ++k) g.e[k] = (T)(exp_diff<T, A>((A)x.e[k], m) * by);
  if (at >= 0 && at < vec_of<T>()) {
#pragma unroll
    for (int k = 0; k < vec_of<T>(); ++k)
      if (k == at) g.e[k] = (T)(exp_diff<T, A>((A)x.e[k], m) * by - w);
  }
  return g;
}

// What a call works on.
template <typename T> struct Loss {
  typedef typename Wide<T>::type A;
  const T *logits;
  long long rows, stride;
  int classes, wide;  // wide: targets of 64 bits
  const void *targets;
  const A *weight;
  double scale;
  A *loss;
  T *grad;
  __device__ __forceinline__ long long target(long long r) const {
    return wide ? ((const long long *)targets)[r] : (long long)((const int *)targets)[r];
  }
  __device__ __forceinline__ bool counts(long long t) const { return t >= 0 && t < classes; }
  __device__ __forceinline__ A factor(long long r) const {
    return (A)scale * (weight ? weight[r] : (A)1);
  }
  // log(sum exp(x)) - x_t
  __device__ __forceinline__ A value(long long r, long long t, A m, A s) const {
    return log_of(s) + (m - (A)logits[r * stride + t]);
  }
};

// Over the L threads of a row: lanes of a wave, or all of the workgroup.
template <int L, typename A, typename F> __device__ __forceinline__ A over_row(A v, A *lds, F f) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d, 64));
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < L / 64; ++w) v = f(v, lds[w]);
  }
  return v;
}

template <int L> constexpr int block_of() { return L < 256 ? 256 : L; }

template <typename T>
__device__ __forceinline__ void zero_row(T *g, int classes, int lane, int lanes) {
  for (int c = lane; c < classes; c += lanes) g[c] = (T)0;
}

// Loss and gradient of rows of up to L * K - 1 vectors, held in registers.
template <typename T, int L, int K>
__global__ __launch_bounds__(block_of<L>(), L >= 512 ? 4 : 1) void k_loss_held(Loss<T> p) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), kRows = block_of<L>() / L;
  __shared__ A lm[L > 64 ? L / 64 : 1], ls[L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x % L;
  const long long r = (long long)blockIdx.x * kRows + threadIdx.x / L;
  if (r >= p.rows) return;
  const long long t = p.target(r);
  T *g = p.grad + r * p.classes;
  if (!p.counts(t)) {
    if (lane == 0) p.loss[r] = 0;
    zero_row(g, p.classes, lane, L);
    return;
  }
  const Row<T> row(p.logits + r * p.stride, p.classes);
  typename Row<T>::Words x[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int v = i * L + lane;
    x[i] = row.nothing();
    if (v < row.vecs) x[i] = row.template load<true>(v);
  }
  A m = -__builtin_inf();
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const Vec<T, V> e = mmpn::elements_of<T, V>(x[i]);
#pragma unroll
    for (int k = 0; k < V; ++k) m = max_of(m, (A)e.e[k]);
  }
  m = over_row<L>(m, lm, [](A a, A b) { return max_of(a, b); });
  A s = 0;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    mmpn::forget(x[i]);
    const Vec<T, V> e = mmpn::elements_of<T, V>(x[i]);
    A part = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) part += exp_diff<T, A>((A)e.e[k], m);
    s += part;
  }
  s = over_row<L>(s, ls, [](A a, A b) { return a + b; });
  if (lane == 0) p.loss[r] = p.value(r, t, m, s);
  const A w = p.factor(r), by = w / s;
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int v = i * L + lane;
    mmpn::forget(x[i]);
    if (v < row.vecs)
      row.store(g, v, grad_of<T, A>(x[i], m, by, w, t + row.head - (long long)v * V));
  }
}

// A thread's part of a row: vectors `from` to `to` in steps of `step`, a
// running maximum and sum over kTogether of them at a time.
constexpr int kTogether = 4;
template <bool STREAM, typename T, typename A>
__device__ __forceinline__ Stat<A> pass(const Row<T> &row, int from, int to, int step) {
  constexpr int V = vec_of<T>();
  Stat<A> st{-__builtin_inf(), 0};
  for (int v0 = from; v0 < to; v0 += kTogether * step) {
    typename Row<T>::Words x[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int v = v0 + i * step;
      x[i] = row.nothing();
      if (v < to) x[i] = row.template load<STREAM>(v);
    }
    A m = st.m;
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const Vec<T, V> e = mmpn::elements_of<T, V>(x[i]);
#pragma unroll
      for (int k = 0; k < V; ++k) m = max_of(m, (A)e.e[k]);
    }
    // nothing but -inf so far: differences to 0 instead, which add nothing
    const A ref = m == -__builtin_inf() ? (A)0 : m;
    A s = st.s * mmpn::exp_of(st.m - ref);
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const Vec<T, V> e = mmpn::elements_of<T, V>(x[i]);
      A part = 0;
#pragma unroll
      for (int k = 0; k < V; ++k) part += exp_diff<T, A>((A)e.e[k], ref);
      s += part;
    }
    st = {m, s};
  }
  return st;
}

template <int L, typename A> __device__ __forceinline__ Stat<A> join_row(Stat<A> st, Stat<A> *lds) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d > 0; d >>= 1)
    st = join(st, Stat<A>{__shfl_xor(st.m, d, 64), __shfl_xor(st.s, d, 64)});
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = st;
    __syncthreads();
    st = lds[0];
#pragma unroll
    for (int w = 1; w < L / 64; ++w) st = join(st, lds[w]);
  }
  return st;
}

// Rows of any length: the loss, and the gradient by reading the row again.
template <typename T, int L, bool GRAD>
__global__ __launch_bounds__(block_of<L>()) void k_loss_pass(Loss<T> p) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>(), kRows = block_of<L>() / L;
  __shared__ Stat<A> lds[L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x % L;
  const long long r = (long long)blockIdx.x * kRows + threadIdx.x / L;
  if (r >= p.rows) return;
  const long long t = p.target(r);
  T *g = GRAD ? p.grad + r * p.classes : nullptr;
  if (!p.counts(t)) {
    if (lane == 0) p.loss[r] = 0;
    if constexpr (GRAD) zero_row(g, p.classes, lane, L);
    return;
  }
  const Row<T> row(p.logits + r * p.stride, p.classes);
  Stat<A> st = pass<!GRAD, T, A>(row, lane, row.vecs, L);
  st = join_row<L>(st, lds);
  if (lane == 0) p.loss[r] = p.value(r, t, st.m, st.s);
  if constexpr (GRAD) {
    const A w = p.factor(r), by = w / st.s;
    // the end of the row was read last, so it is the likeliest to be near
    for (int v = lane + (row.vecs - 1 - lane) / L * L; v >= 0; v -= L)
      row.store(g, v, grad_of<T, A>(row.template load<true>(v), st.m, by, w,
                                    t + row.head - (long long)v * V));
  }
}

// Few long rows: `parts` workgroups a row, each with its statistics in `part`,
// then as many again that join them.
constexpr int kPartBlock = 256;
template <typename T>
__global__ __launch_bounds__(kPartBlock) void k_loss_part(Loss<T> p, int parts,
                                                          Stat<typename Wide<T>::type> *part) {
  typedef typename Wide<T>::type A;
  __shared__ Stat<A> lds[kPartBlock / 64];
  const long long r = blockIdx.x / parts;
  const int q = (int)(blockIdx.x - r * parts);
  if (!p.counts(p.target(r))) return;
  const Row<T> row(p.logits + r * p.stride, p.classes);
  const int per = (row.vecs + parts - 1) / parts;
  const int from = q * per, to = from + per < row.vecs ? from + per : row.vecs;
  Stat<A> st = pass<false, T, A>(row, from + threadIdx.x, to, kPartBlock);
  st = join_row<kPartBlock>(st, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = st;
}
template <typename T, bool GRAD>
__global__ __launch_bounds__(kPartBlock) void k_loss_join(Loss<T> p, int parts,
                                                          const Stat<typename Wide<T>::type> *part) {
  typedef typename Wide<T>::type A;
  constexpr int V = vec_of<T>();
  const long long r = GRAD ? blockIdx.x / parts : blockIdx.x;
  const int q = GRAD ? (int)(blockIdx.x - r * parts) : 0;
  const long long t = p.target(r);
  const bool counts = p.counts(t);
  // every wave joins the row's parts for itself
  Stat<A> st{-__builtin_inf(), 0};
  if (counts)
    for (int i = threadIdx.x & 63; i < parts; i += 64) st = join(st, part[r * parts + i]);
  st = join_row<64>(st, (Stat<A> *)nullptr);
  if (q == 0 && threadIdx.x == 0) p.loss[r] = counts ? p.value(r, t, st.m, st.s) : (A)0;
  if constexpr (GRAD) {
    const Row<T> row(p.logits + r * p.stride, p.classes);
    const int per = (row.vecs + parts - 1) / parts;
    const int from = q * per, to = from + per < row.vecs ? from + per : row.vecs;
    T *g = p.grad + r * p.classes;
    const A w = p.factor(r), by = w / st.s;
    for (int v = from + threadIdx.x; v < to; v += kPartBlock) {
      Vec<T, V> o;
      if (counts) {
        o = grad_of<T, A>(row.template load<false>(v), st.m, by, w,
                          t + row.head - (long long)v * V);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) o.e[k] = (T)0;
      }
      row.store(g, v, o);
    }
  }
}

template <typename T, int L, int K> int launch_held(const Loss<T> &p) {
  const int64_t blocks = mmpi::ceil_div(p.rows, block_of<L>() / L);
  if (!mmpi::grid_fits(blocks, block_of<L>()))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: too many rows");
  hipLaunchKernelGGL((k_loss_held<T, L, K>), dim3((unsigned)blocks), dim3(block_of<L>()), 0, mmpi::stream(), p);
  return mmpi::check_launch("mmp_cross_entropy(held)");
}
template <typename T, int L, bool GRAD> int launch_pass(const Loss<T> &p) {
  const int64_t blocks = mmpi::ceil_div(p.rows, block_of<L>() / L);
  if (!mmpi::grid_fits(blocks, block_of<L>()))
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: too many rows");
  hipLaunchKernelGGL((k_loss_pass<T, L, GRAD>), dim3((unsigned)blocks), dim3(block_of<L>()), 0,
                     mmpi::stream(), p);
  return mmpi::check_launch("mmp_cross_entropy(pass)");
}

// The layouts of mmp_plan.h, by their numbers.
template <typename T, size_t... I>
int launch_held_of(const Loss<T> &p, const mmpi::LossPlan &plan, std::index_sequence<I...>) {
  using mmpi::kLossHeld;
  int st = MMP_OK;
  const bool found =
      ((plan.lanes == kLossHeld[I].lanes && plan.held == kLossHeld[I].held &&
        ((st = launch_held<T, kLossHeld[I].lanes, kLossHeld[I].held>(p)), true)) || ...);
  return found ? st : mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: no layout");
}
template <typename T, size_t... I>
int launch_pass_of(const Loss<T> &p, const mmpi::LossPlan &plan, std::index_sequence<I...>) {
  using mmpi::kLossPass;
  int st = MMP_OK;
  const bool found = ((plan.lanes == kLossPass[I].lanes &&
                       ((st = launch_pass<T, kLossPass[I].lanes, false>(p)), true)) || ...);
  return found ? st : mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: no layout");
}

template <typename T> int loss_impl(const Loss<T> &p) {
  typedef typename Wide<T>::type A;
  // Whether the stream is captured is asked only where it matters.
  auto plan_of = [&](bool may_split) {
    return mmpi::loss_plan(p.grad != nullptr, sizeof(T), p.rows, p.classes, mmpi::cu_count(), may_split);
  };
  mmpi::LossPlan plan = plan_of(true);
  if (plan.parts && mmpn::capturing()) plan = plan_of(false);
  if (const int parts = plan.parts) {
    mmpn::Temp part;
    if (int st = part.get((size_t)(p.rows * parts) * sizeof(Stat<A>), "mmp_cross_entropy")) return st;
    hipLaunchKernelGGL((k_loss_part<T>), dim3((unsigned)(p.rows * parts)), dim3(kPartBlock), 0,
                       mmpi::stream(), p, parts, (Stat<A> *)part.p);
    if (int st = mmpi::check_launch("mmp_cross_entropy(part)")) return st;
    if (p.grad)
      hipLaunchKernelGGL((k_loss_join<T, true>), dim3((unsigned)(p.rows * parts)),
                         dim3(kPartBlock), 0, mmpi::stream(), p, parts, (const Stat<A> *)part.p);
    else
      hipLaunchKernelGGL((k_loss_join<T, false>), dim3((unsigned)p.rows), dim3(kPartBlock), 0,
                         mmpi::stream(), p, parts, (const Stat<A> *)part.p);
    return mmpi::check_launch("mmp_cross_entropy(join)");
  }
  if (plan.held)
    return launch_held_of(p, plan, std::make_index_sequence<std::size(mmpi::kLossHeld)>());
  if (p.grad) return launch_pass<T, mmpi::kLossAgainLanes, true>(p);
  return launch_pass_of(p, plan, std::make_index_sequence<std::size(mmpi::kLossPass)>());
}

constexpr int64_t kMost = 0x7fff0000LL;  // room for a step past the end in 32 bits

}  // namespace

extern "C" int mmp_cross_entropy(int dtype, int index_dtype, int64_t rows, int64_t classes,
                                 const void *logits, int64_t row_stride, const void *targets,
                                 const void *weight, double scale, void *loss, void *grad) {
  if (int st = mmpi::ensure_init()) return st;
  if (rows < 0 || classes < 0) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: negative extent");
  if (rows == 0) return MMP_OK;
  if (classes == 0) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: no classes");
  if (!logits || !targets || !loss) return mmpi::fail(MMP_E_ARG, "mmp_cross_entropy: null pointer");
  if (index_dtype != MMP_I32 && index_dtype != MMP_I64)
    return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: index dtype code %d", index_dtype);
  if (classes > kMost) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_cross_entropy: 2^31 classes");
  MMP_DISPATCH_FLOAT(dtype, "mmp_cross_entropy", {
    typedef typename Wide<T>::type A;
    return loss_impl<T>(Loss<T>{(const T *)logits, (long long)rows, (long long)row_stride,
                                (int)classes, index_dtype == MMP_I64, targets, (const A *)weight,
                                scale, (A *)loss, (T *)grad});
  })
}
