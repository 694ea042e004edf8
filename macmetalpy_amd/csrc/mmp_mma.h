// mmp_mma.h -- 16 x 16 tiles of products on the matrix cores, for operands that
// come from LDS or from the accumulators of the product before.
//
// A lane (fr = lane % 16, g = lane / 16) has one row of the left operand, or one
// column of the right one, and of an accumulator tile the column fr and the rows
// row(g, r), r < 4.  The order of a product's k is free as long as both operands
// agree, so the k that a lane feeds is chosen to be row(g, .): then a tile of
// accumulators is a right operand as it is, without a move between lanes.
// Swapping the operands gives the transposed tile, in which a lane has one row
// and the columns row(g, .).
#pragma once
#include "mmp_nn.h"

namespace mmpx {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef double d4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));

template <typename T> struct Mma;

// v_mfma_f32_16x16x32_f16: two tiles of accumulators make one operand.
template <> struct Mma<mmp_half> {
  typedef float A;
  typedef f4 Acc;
  typedef h8 Frag;
  static constexpr int K = 32, E = 8, PAD = 8;
  static constexpr bool SPLIT = true;
  static __device__ __forceinline__ int row(int g, int r) { return 4 * g + r; }
  static __device__ __forceinline__ Acc mul(Frag a, Frag b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  // k along the rows of `m`: row first + fr, k from k0 on
  static __device__ __forceinline__ Frag rows(const mmp_half *m, int ld, int first, int k0, int lane) {
    const mmp_half *p = m + (first + (lane & 15)) * ld + k0 + 4 * (lane >> 4);
    const s4 lo = *reinterpret_cast<const s4 *>(p), hi = *reinterpret_cast<const s4 *>(p + 16);
    return __builtin_bit_cast(h8, (s8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
  // k along the columns of `m`: column first + fr.  A transposing read gives
  // element j of lane 4 a + b of a group of 16 element b of what lane a + 4 j addresses.
  static __device__ __forceinline__ Frag cols(const mmp_half *m, int ld, int k0, int first, int lane) {
    const int q = lane & 15;
    const mmp_half *p = m + (k0 + 4 * (lane >> 4) + (q >> 2)) * ld + first + 4 * (q & 3);
    typedef __attribute__((address_space(3))) s4 L;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(p + 16 * ld));
    return __builtin_bit_cast(h8, (s8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
};

// Four v_mfma_f32_16x16x4f32.
template <> struct Mma<float> {
  typedef float A;
  typedef f4 Acc;
  typedef f4 Frag;
  static constexpr int K = 16, E = 4, PAD = 4;
  static constexpr bool SPLIT = false;
  static __device__ __forceinline__ int row(int g, int r) { return 4 * g + r; }
  static __device__ __forceinline__ Acc mul(Frag a, Frag b, Acc c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag rows(const float *m, int ld, int first, int k0, int lane) {
    return *reinterpret_cast<const f4 *>(m + (first + (lane & 15)) * ld + k0 + 4 * (lane >> 4));
  }
  static __device__ __forceinline__ Frag cols(const float *m, int ld, int k0, int first, int lane) {
    const float *p = m + (k0 + 4 * (lane >> 4)) * ld + first + (lane & 15);
    return Frag{p[0], p[ld], p[2 * ld], p[3 * ld]};
  }
};

// Four v_mfma_f64_16x16x4f64, whose accumulators have rows g + 4 r.
template <> struct Mma<double> {
  typedef double A;
  typedef d4 Acc;
  typedef d4 Frag;
  static constexpr int K = 16, E = 4, PAD = 2;
  static constexpr bool SPLIT = false;
  static __device__ __forceinline__ int row(int g, int r) { return g + 4 * r; }
  static __device__ __forceinline__ Acc mul(Frag a, Frag b, Acc c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f64_16x16x4f64(a[t], b[t], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag rows(const double *m, int ld, int first, int k0, int lane) {
    const double *p = m + (first + (lane & 15)) * ld + k0 + (lane >> 4);
    return Frag{p[0], p[4], p[8], p[12]};
  }
  static __device__ __forceinline__ Frag cols(const double *m, int ld, int k0, int first, int lane) {
    const double *p = m + (k0 + (lane >> 4)) * ld + first + (lane & 15);
    return Frag{p[0], p[4 * ld], p[8 * ld], p[12 * ld]};
  }
};

// A value in 32 bits as two float16 operands, the value rounded and what that
// left: 22 bits, and a product of two such values but for the product of their
// small parts.  Other types hold their values as they are.
//
// The rounded value is made opaque before its rest is worked out: the compiler
// may round a product to float16 in one step where it is stored and in two, by way
// of 32 bits, where the rest needs it, and about one in 2^13 values then differs by a
// unit that the rest does not hold.
template <typename T> struct Two {
  typename Mma<T>::Frag hi, lo;
};
template <typename W> __device__ __forceinline__ void settle(W &w) {
  static_assert(sizeof(W) % 4 == 0, "");
  unsigned u[sizeof(W) / 4];
  __builtin_memcpy(u, &w, sizeof(W));
#pragma unroll
  for (unsigned i = 0; i < sizeof(W) / 4; ++i) asm volatile("" : "+v"(u[i]));
  __builtin_memcpy(&w, u, sizeof(W));
}
template <typename T> __device__ __forceinline__ Two<T> two_of(const typename Mma<T>::A (&v)[Mma<T>::E]) {
  Two<T> f;
#pragma unroll
  for (int e = 0; e < Mma<T>::E; ++e) f.hi[e] = (T)v[e];
  f.lo = f.hi;
  if constexpr (Mma<T>::SPLIT) {
    settle(f.hi);
#pragma unroll
    for (int e = 0; e < Mma<T>::E; ++e) f.lo[e] = (T)(v[e] - (float)f.hi[e]);
  }
  return f;
}
// Tiles [first, first + K / 16) of accumulators as an operand, each value times `by`.
template <typename T, int N>
__device__ __forceinline__ Two<T> operand(const typename Mma<T>::Acc (&acc)[N], int first) {
  typename Mma<T>::A v[Mma<T>::E];
#pragma unroll
  for (int e = 0; e < Mma<T>::E; ++e) v[e] = acc[first + (e >> 2)][e & 3];
  return two_of<T>(v);
}
// a (b.hi + b.lo) and (a.hi + a.lo)(b.hi + b.lo) but for a.lo b.lo.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Acc mul_two(typename Mma<T>::Frag a, const Two<T> &b, typename Mma<T>::Acc c) {
  if constexpr (Mma<T>::SPLIT) c = Mma<T>::mul(a, b.lo, c);
  return Mma<T>::mul(a, b.hi, c);
}
template <typename T>
__device__ __forceinline__ typename Mma<T>::Acc mul_twos(const Two<T> &a, const Two<T> &b, typename Mma<T>::Acc c) {
  if constexpr (Mma<T>::SPLIT) {
    c = Mma<T>::mul(a.lo, b.hi, c);
    c = Mma<T>::mul(a.hi, b.lo, c);
  }
  return Mma<T>::mul(a.hi, b.hi, c);
}
// The transposed product's.
template <typename T>
__device__ __forceinline__ typename Mma<T>::Acc two_mul(const Two<T> &a, typename Mma<T>::Frag b, typename Mma<T>::Acc c) {
  if constexpr (Mma<T>::SPLIT) c = Mma<T>::mul(a.lo, b, c);
  return Mma<T>::mul(a.hi, b, c);
}

}  // namespace mmpx
