// mmp_nn.h -- what the operators of sequence models share: vectors of a few
// elements at any address, and the exponentials that they need.
#pragma once
#include "mmp_ops.h"
#include "mmp_internal.h"

namespace mmpn {

// The type that sums and states are held in: 32 bits for float16 and float32,
// 64 for float64.
template <typename T> struct Wide { typedef float type; };
template <> struct Wide<double> { typedef double type; };

// N adjacent elements, moved by one instruction (or by two or four of 16
// bytes).  The address need only be a multiple of the element's size: rows of
// odd lengths start anywhere, and the device's vector loads and stores take any
// address.
template <typename T, int N> struct Vec {
  typedef unsigned int Words __attribute__((ext_vector_type(sizeof(T) * N >= 4 ? sizeof(T) * N / 4 : 1)));
  T e[N];
};

template <typename T, int N, bool STREAM = false>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p) {
  Vec<T, N> r;
  if constexpr (sizeof(T) * N >= 4) {
    typedef typename Vec<T, N>::Words W;
    typedef W U __attribute__((aligned(sizeof(T))));
    W w;
    if constexpr (STREAM) w = __builtin_nontemporal_load(reinterpret_cast<const U *>(p));
    else w = *reinterpret_cast<const U *>(p);
    __builtin_memcpy(&r, &w, sizeof(r));
  } else {
    for (int i = 0; i < N; ++i) r.e[i] = p[i];
  }
  return r;
}

template <typename T, int N, bool STREAM = false>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, N> &v) {
  if constexpr (sizeof(T) * N >= 4) {
    typedef typename Vec<T, N>::Words W;
    typedef W U __attribute__((aligned(sizeof(T))));
    W w;
    __builtin_memcpy(&w, &v, sizeof(v));
    if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<U *>(p));
    else *reinterpret_cast<U *>(p) = w;
  } else {
    for (int i = 0; i < N; ++i) p[i] = v.e[i];
  }
}

// Vectors that are kept for a while are kept as words: as elements, a float16
// vector that passes a branch takes a register for each of its halves.
template <typename T, int N> __device__ __forceinline__ typename Vec<T, N>::Words words_of(const Vec<T, N> &v) {
  if constexpr (sizeof(T) * N < 4) {
    typename Vec<T, N>::Words w = 0;
    __builtin_memcpy(&w, &v, sizeof(v));
    return w;
  } else {
    return __builtin_bit_cast(typename Vec<T, N>::Words, v);
  }
}
template <typename T, int N> __device__ __forceinline__ Vec<T, N> elements_of(typename Vec<T, N>::Words w) {
  if constexpr (sizeof(T) * N < 4) {
    Vec<T, N> v;
    __builtin_memcpy(&v, &w, sizeof(v));
    return v;
  } else {
    return __builtin_bit_cast(Vec<T, N>, w);
  }
}

// Words that the compiler takes for others from here on, so that it works out
// again what it made of them before, where that is used again, instead of
// keeping all of it (widened values first of all) in registers in between.
template <typename W> __device__ __forceinline__ void forget(W &w) {
#pragma unroll
  for (unsigned k = 0; k < sizeof(W) / 4; ++k) {
    unsigned u = w[k];
    asm volatile("" : "+v"(u));
    w[k] = u;
  }
}

// exp(x) of x <= 0 or NaN in 32 bits: 2^(x log2 e) by the hardware's
// exponential.  The product's rounding error, which grows with |x|, is carried
// over to the result, so the relative error stays at a few units of the last
// place.  Below the normal range the result is 0; so it is for x < -126, where
// x is cut off because -inf has no product to correct.
__device__ __forceinline__ float exp_of(float x) {
  const float l2e = 1.44269502f, l2e_lo = 1.92596303e-8f;  // log2 e in two parts
  x = x < -126.0f ? -126.0f : x;
  const float t = x * l2e;
  const float r = __builtin_fmaf(x, l2e_lo, __builtin_fmaf(x, l2e, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(e, r * 0.693147182f, e);
}
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return __builtin_fma(a, b, c); }

// f = 1 / (1 + exp(-g)) and u = 1 - f = 1 / (1 + exp(g)), each to its own
// last places: the exponential's argument is never positive, so neither
// overflows, and u keeps its digits where f is near 1.  g was rounded to a T: the
// 11 bits of a float16 move exp(g) by a thousand times what the two corrections
// below do, so there they are left out.  In units of 2^-24: f or u is off by up to 16
// for |g| up to 20 (6 with them), by a factor that is the same in every step and does
// not add up; what does, f + u - 1, holds a state of 1 within 2.0 / (1 - f) for every
// float16 gate from -4 to 6 (1.96 with them).  They cost (us a call, on one set of
// inputs), forwards, 16 x 2048 x 2048 88 to 99, 253 x 170 x 1390 71 to 85, backwards 144 to
// 153.
template <typename T, typename A> __device__ __forceinline__ void sigmoid_pair(A g, A &f, A &u) {
  const A x = g < 0 ? g : -g;
  A e, r;
  if constexpr (sizeof(T) == 2) {
    e = __builtin_amdgcn_exp2f(x * 1.44269502f);
    r = __builtin_amdgcn_rcpf(1 + e);
  } else if constexpr (sizeof(T) == 4) {
    // The hardware's reciprocal is within a unit of the last place; the same
    // error in every step would add up along a sequence, so one more step of
    // Newton's iteration.
    e = exp_of(x);
    const A d = 1 + e;
    r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  } else {
    e = exp_of(x);
    r = 1 / (1 + e);
  }
  const A s = e * r;
  f = g < 0 ? s : r;
  u = g < 0 ? r : s;
}

// Whether the library's stream is being captured into a graph.  Its replays
// outlive the call: memory of the pool is another array's by then, and a tag
// fixed at capture time no longer tells a replay's words from the ones before.
inline bool capturing() {
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(mmpi::stream(), &s) == hipSuccess) return s != hipStreamCaptureStatusNone;
  (void)hipGetLastError();
  return true;
}
inline int refuse_capture(const char *what) {
  return mmpi::fail(MMP_E_UNSUPPORTED, "%s: takes scratch memory, so it cannot be captured", what);
}

// Memory of the library's stream-ordered pool for the length of a call.
struct Temp {
  void *p = nullptr;
  ~Temp() {
    if (p) (void)mmp_free(p);
  }
  int get(size_t bytes, const char *what) {
    if (capturing()) return refuse_capture(what);
    return mmp_alloc(bytes ? bytes : 1, &p);
  }
};

}  // namespace mmpn

// Dispatch a floating dtype code onto a C++ type `T`.
#define MMP_DISPATCH_FLOAT(dtype, what, ...)                                  \
  switch (dtype) {                                                            \
    case MMP_F16: { typedef mmp_half T; __VA_ARGS__ }                         \
    case MMP_F32: { typedef float T; __VA_ARGS__ }                            \
    case MMP_F64: { typedef double T; __VA_ARGS__ }                           \
    default:                                                                  \
      return mmpi::fail(MMP_E_UNSUPPORTED, what ": dtype code %d is not floating", \
                        (int)(dtype));                                        \
  }
// Dispatch an index dtype code (MMP_I32, MMP_I64) onto a C++ type `I`.
#define MMP_DISPATCH_INDEX(dtype, what, ...)                                  \
  switch (dtype) {                                                            \
    case MMP_I32: { typedef mmp_i32 I; __VA_ARGS__ }                          \
    case MMP_I64: { typedef mmp_i64 I; __VA_ARGS__ }                          \
    default:                                                                  \
      return mmpi::fail(MMP_E_UNSUPPORTED, what ": index dtype code %d", (int)(dtype)); \
  }
