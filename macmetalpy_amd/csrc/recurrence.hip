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
//
// Bound by memory: 3 arrays forwards, 6 (5 with factors) backwards.  Each is
// read or written once.  n steps together are one step h -> A h + B, with A
// the product of their factors and B what they make of h = 0, so time is cut
// into tiles: a workgroup loads its steps of some channels into registers, each
// thread joins the few steps of its own, the workgroup joins its threads'
// (A, B) in LDS, and the tile's state before its first step comes from the tiles
// before it by look-back; then each thread runs its steps from its state and
// writes.  With few steps, or sequences enough to fill the device with a thread
// for a few channels, a thread goes through the steps instead.
//
// Measured, float16: 16 x 2048 x 2048 backwards 144 us, 5.6 TB/s, forwards 82, 4.9; one
// sequence of 65,536 x 1024 104 us, 3.9 TB/s: its tiles wait for each other, and
// only two workgroups a CU have room for what they hold meanwhile.
//
// Look-back: a tile publishes (A, B) and, as soon as it knows it, the state
// after its last step.  It reads the kLook tiles before it until one of them
// has that state and all after it have (A, B), and goes through those in
// order, state = A state + B: the same operations whichever tile had its state
// first, so the results' bits do not depend on timing.  Nothing promises that
// an earlier tile's workgroup has started, so the wait is bounded: after
// kPolls reads a tile goes back as far as it must and joins the steps of the
// tiles that are missing itself.
#include "mmp_nn.h"

namespace {

using mmpn::Vec;
using mmpn::Wide;

constexpr int kBlock = mmpi::kRecurBlock;
constexpr int kLook = 4;                 // tiles that look-back reads at once
constexpr int kPolls = 256;
// Per SIMD: two workgroups a CU, so 128 registers.  float64's gradient from logits
// keeps 20 to 52 more in scratch (16 x 2048 x 512 153 us, 5.3 TB/s; from factors 114, 5.9).
constexpr int kWaves = 4;

// How a workgroup lies on its tile: `lanes` threads side by side on a step with
// vectors of `bytes`, kBlock / lanes of them one after another in time, `steps`
// steps each.
template <int LANES, int BYTES, int STEPS> struct Layout {
  static constexpr int lanes = LANES, steps = STEPS, slices = kBlock / LANES;
  static constexpr int tile = slices * STEPS;  // steps of a workgroup
  template <typename T> static constexpr int vec() { return BYTES / (int)sizeof(T); }
  template <typename T> static constexpr int channels() { return LANES * vec<T>(); }
};
template <const mmpi::RecurLayout &L> using LayoutOf = Layout<L.lanes, L.bytes, L.steps>;
typedef LayoutOf<mmpi::kForwardFew> ForwardFew;
typedef LayoutOf<mmpi::kForwardLong> ForwardLong;
template <typename T>
using ForwardWide = Layout<mmpi::kForwardWide.lanes, mmpi::forward_wide(sizeof(T)).bytes,
                           mmpi::kForwardWide.steps>;
typedef LayoutOf<mmpi::kForwardBrief> ForwardBrief;
typedef LayoutOf<mmpi::kBackwardFew> BackwardFew;
typedef LayoutOf<mmpi::kBackwardLong> BackwardLong;
typedef LayoutOf<mmpi::kBackwardWide> BackwardWide;
using mmpi::kShortBytes;

// Steps of a (batch, steps, dim) array: adjacent channels, any other strides.
template <typename T> struct Steps {
  const T *p;
  long long sb, st;
};

// A tile's descriptor holds 2 wide values per channel, each 32 bits of them in
// a word with a tag above: generation << 2 | state, 1 for (A, B), 2 for the
// state after the tile.  Words are written and read with relaxed atomics
// and taken only where all tags of a channel agree and are this call's, so
// they are never cleared and need no fence.  The replays of a graph would all
// have the tag of its capture and take the states of the replay before, so a
// call of more than one tile refuses to be captured.
struct Look {
  unsigned long long *desc;
  unsigned gen;       // this call's
  unsigned read_gen;  // the one that readers take (another one to force the slow way)
  long long polls;
};
template <typename A> constexpr int words_of() { return (int)sizeof(A) / 2; }

template <typename A, int CH>
__device__ __forceinline__ void publish(const Look &lk, long long tile, int ch, unsigned state, A a,
                                        A b) {
  constexpr int NW = words_of<A>();
  unsigned w[NW];
  const A v[2] = {a, b};
  __builtin_memcpy(w, v, sizeof(v));
  const unsigned long long tag = (unsigned long long)(lk.gen << 2 | state) << 32;
#pragma unroll
  for (int k = 0; k < NW; ++k)
    __hip_atomic_store(lk.desc + (tile * NW + k) * CH + ch, tag | w[k], __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

// The state of tile's descriptor for a channel: 0 (not there), 1 or 2.
template <typename A> struct Desc {
  unsigned long long w[words_of<A>()];
};
template <typename A, int CH>
__device__ __forceinline__ Desc<A> read_desc(const Look &lk, long long tile, int ch) {
  Desc<A> d;
#pragma unroll
  for (int k = 0; k < words_of<A>(); ++k)
    d.w[k] = __hip_atomic_load(lk.desc + (tile * words_of<A>() + k) * CH + ch, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
  return d;
}
template <typename A>
__device__ __forceinline__ unsigned parse(const Look &lk, const Desc<A> &d, A &a, A &b) {
  const unsigned tag = (unsigned)(d.w[0] >> 32);
  bool same = (tag >> 2) == lk.read_gen;
  unsigned w[words_of<A>()];
#pragma unroll
  for (int k = 0; k < words_of<A>(); ++k) {
    same = same && (unsigned)(d.w[k] >> 32) == tag;
    w[k] = (unsigned)d.w[k];
  }
  A v[2];
  __builtin_memcpy(v, w, sizeof(v));
  a = v[0];
  b = v[1];
  return same ? tag & 3u : 0u;
}

// The state before tile t of a sequence whose tiles' descriptors begin at
// `base`; a wave, a channel a lane (`on`: the lane has one).  own(j, a, b)
// joins the steps of tile j.
template <typename A, int CH, int W, typename Own>
__device__ A look_back(const Look &lk, long long base, long long t, int ch, bool on, A initial,
                       Own own) {
  for (long long poll = 0; poll < lk.polls; ++poll) {
    Desc<A> d[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const long long j = t - 1 - k < 0 ? 0 : t - 1 - k;
      d[k] = read_desc<A, CH>(lk, base + j, ch);
    }
    A h = 0;
    bool ok = !on;
#pragma unroll
    for (int k = W - 1; k >= 0; --k) {
      A a, b;
      const unsigned st = parse(lk, d[k], a, b);
      if (t - 1 - k < 0) {
        h = initial;
        ok = true;
      } else if (st == 2) {
        h = a;
        ok = true;
      } else if (st == 1) {
        h = mmpn::fma_of(a, h, b);
      } else {
        ok = !on;
      }
    }
    if (__ballot(!ok) == 0) return h;
    __builtin_amdgcn_s_sleep(1);
  }
  // Back to a tile that every channel knows the state after, or to the first.
  A h = initial, a, b;
  long long j = t - 1;
  for (; j >= 0; --j) {
    const unsigned st = parse(lk, read_desc<A, CH>(lk, base + j, ch), a, b);
    if (__ballot(on && st != 2) == 0) {
      h = a;
      break;
    }
  }
  for (++j; j < t; ++j) {
    const unsigned st = parse(lk, read_desc<A, CH>(lk, base + j, ch), a, b);
    if (__ballot(on && st == 0) != 0) {
      A a2, b2;
      own(j, a2, b2);
      if (st == 0) {
        a = a2;
        b = b2;
      }
    }
    h = st == 2 ? a : mmpn::fma_of(a, h, b);
  }
  return h;
}

// One step's factor and addend.
template <typename T, bool LOGITS, typename A>
__device__ __forceinline__ void factor(A g, A x, A &f, A &u) {
  if constexpr (LOGITS) {
    A r;
    mmpn::sigmoid_pair<T>(g, f, r);
    u = r * x;
  } else {
    f = g;
    u = x;
  }
}

// `count` of V adjacent elements (all of them, but at a row's end), zeros else.
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_some(const T *p, int count) {
  if (count >= V) return mmpn::load_vec<T, V>(p);
  Vec<T, V> v;
#pragma unroll
  for (int k = 0; k < V; ++k) v.e[k] = k < count ? p[k] : (T)0;
  return v;
}
template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ typename Vec<T, V>::Words load_words(const T *p) {
  return mmpn::words_of<T, V>(mmpn::load_vec<T, V, STREAM>(p));
}
// Past the caches: 64 x 500 x 1024 float16 39 us, through them 46.
template <typename T, int V>
__device__ __forceinline__ void store_some(T *p, const Vec<T, V> &v, int count) {
  if (count >= V) {
    mmpn::store_vec<T, V, true>(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < count) p[k] = v.e[k];
  }
}

// The channel of a workgroup's column: a row's last vector ends with it (where it
// is a vector's length at least), so that every vector is read and written
// whole.  Some of its channels may be the vector before's too, with the same results.
template <int V> __device__ __forceinline__ int channel_of(int column, int dim) {
  const int first = column / V * V;
  return (first + V > dim ? (dim > V ? dim - V : 0) : first) + column % V;
}

// Where a workgroup is: `groups` sequences times channel groups, and in each
// `tiles` tiles.  Early tiles have the low workgroup ids, which start first.
struct Place {
  long long seq, base;
  int group;     // of channels
  long long t;   // tile of the sequence
};
__device__ __forceinline__ Place place(long long tiles, long long groups, int cgroups) {
  Place p;
  p.t = blockIdx.x / groups;
  const long long g = blockIdx.x - p.t * groups;
  p.seq = g / cgroups;
  p.group = (int)(g - p.seq * cgroups);
  p.base = g * tiles;
  return p;
}

// Joins the slices' (A, B), which sa and sb hold: each becomes that of all
// slices before it, and the tile's is returned.  A channel a lane.
template <typename A, int CH, int SLICES>
__device__ __forceinline__ void join_slices(A *sa, A *sb, int ch, A &ta, A &tb) {
  A pa = 1, pb = 0;
#pragma unroll 8
  for (int s = 0; s < SLICES; ++s) {
    const A a = sa[s * CH + ch], b = sb[s * CH + ch];
    sa[s * CH + ch] = pa;
    sb[s * CH + ch] = pb;
    pb = mmpn::fma_of(a, pb, b);
    pa = a * pa;
  }
  ta = pa;
  tb = pb;
}

template <typename T, bool LOGITS, typename L, bool STREAM>
__global__ __launch_bounds__(kBlock, kWaves) void k_recur_tiles(
    long long steps, int dim, long long tiles, long long groups, int cgroups, Steps<T> gate,
    Steps<T> x, const typename Wide<T>::type *__restrict__ initial, T *__restrict__ h,
    typename Wide<T>::type *__restrict__ final_, Look lk) {
  typedef typename Wide<T>::type A;
  constexpr int V = L::template vec<T>(), CH = L::template channels<T>();
  constexpr int kSteps = L::steps, kSlices = L::slices, kTile = L::tile;
  __shared__ A sa[kSlices * CH], sb[kSlices * CH], sh[CH];
  const Place pl = place(tiles, groups, cgroups);
  const int tid = threadIdx.x, c = (tid & (L::lanes - 1)) * V, s = tid / L::lanes;
  const int ch = channel_of<V>(pl.group * CH + c, dim);  // the thread's first channel
  const int count = pl.group * CH + c < dim ? dim - ch : 0;
  const long long t0 = pl.t * kTile + s * kSteps;
  const T *pg = gate.p + pl.seq * gate.sb + t0 * gate.st + ch;
  const T *px = x.p + pl.seq * x.sb + t0 * x.st + ch;
  A f[kSteps][V], u[kSteps][V];
  {
    typename Vec<T, V>::Words g[kSteps], v[kSteps];
    if (count >= V && t0 < steps) {  // steps past the end read the last, and are not used
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        g[i] = load_words<T, V, STREAM>(pg);
        v[i] = load_words<T, V, STREAM>(px);
        pg += t0 + i + 1 < steps ? gate.st : 0;
        px += t0 + i + 1 < steps ? x.st : 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int n = t0 + i < steps ? count : 0;
        g[i] = mmpn::words_of<T, V>(load_some<T, V>(pg + i * gate.st, n));
        v[i] = mmpn::words_of<T, V>(load_some<T, V>(px + i * x.st, n));
      }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const Vec<T, V> gi = mmpn::elements_of<T, V>(g[i]), vi = mmpn::elements_of<T, V>(v[i]);
#pragma unroll
      for (int k = 0; k < V; ++k) factor<T, LOGITS>((A)gi.e[k], (A)vi.e[k], f[i][k], u[i][k]);
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    A a = 1, b = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      a = f[i][k] * a;
      b = mmpn::fma_of(f[i][k], b, u[i][k]);
    }
    sa[s * CH + c + k] = a;
    sb[s * CH + c + k] = b;
  }
  __syncthreads();
  if (tid < (CH < 64 ? 64 : CH)) {
    const int my = tid < CH ? tid : CH - 1;
    const int chan = channel_of<V>(pl.group * CH + my, dim);
    const bool on = tid < CH && pl.group * CH + my / V * V < dim && chan < dim;
    const long long at = pl.seq * dim + chan;
    A a, b;
    if (tid < CH) join_slices<A, CH, kSlices>(sa, sb, tid, a, b);
    A state = on && initial ? initial[at] : (A)0;
    if (tiles > 1) {
      if (on && pl.t > 0 && pl.t + 1 < tiles) publish<A, CH>(lk, pl.base + pl.t, my, 1, a, b);
      if (pl.t > 0)
        state = look_back<A, CH, kLook>(
            lk, pl.base, pl.t, my, on, state, [&](long long j, A &ja, A &jb) {
              ja = 1;
              jb = 0;
              if (!on) return;
              const T *qg = gate.p + pl.seq * gate.sb + j * kTile * gate.st + chan;
              const T *qx = x.p + pl.seq * x.sb + j * kTile * x.st + chan;
              for (int w = 0; w < kSlices; ++w) {
                A wa = 1, wb = 0;
                for (int i = 0; i < kSteps; ++i) {
                  const long long r = w * kSteps + i;
                  A ff, uu;
                  factor<T, LOGITS>((A)qg[r * gate.st], (A)qx[r * x.st], ff, uu);
                  wa = ff * wa;
                  wb = mmpn::fma_of(ff, wb, uu);
                }
                jb = mmpn::fma_of(wa, jb, wb);
                ja = wa * ja;
              }
            });
      if (on && pl.t + 1 < tiles)
        publish<A, CH>(lk, pl.base + pl.t, my, 2, mmpn::fma_of(a, state, b), (A)0);
    }
    if (tid < CH) sh[tid] = state;
  }
  __syncthreads();
  A st[V];
#pragma unroll
  for (int k = 0; k < V; ++k)
    st[k] = mmpn::fma_of(sa[s * CH + c + k], sh[c + k], sb[s * CH + c + k]);
  T *ph = h + (pl.seq * steps + t0) * dim + ch;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (t0 + i >= steps) break;
    Vec<T, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      st[k] = mmpn::fma_of(f[i][k], st[k], u[i][k]);
      o.e[k] = (T)st[k];
    }
    store_some<T, V>(ph + (long long)i * dim, o, count);
  }
  if (t0 < steps && t0 + kSteps >= steps)
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < count) final_[pl.seq * dim + ch + k] = st[k];
}

// Backwards: tile 0 holds the last steps, a thread's first step is its latest.
template <typename T, bool LOGITS, typename L, bool STREAM>
__global__ __launch_bounds__(kBlock, kWaves) void k_recur_grad_tiles(
    long long steps, int dim, long long tiles, long long groups, int cgroups, Steps<T> grad,
    Steps<T> gate, Steps<T> x, Steps<T> h, const typename Wide<T>::type *__restrict__ initial,
    const typename Wide<T>::type *__restrict__ grad_final, T *__restrict__ grad_gate,
    T *__restrict__ grad_x, typename Wide<T>::type *__restrict__ grad_initial, Look lk) {
  typedef typename Wide<T>::type A;
  constexpr int V = L::template vec<T>(), CH = L::template channels<T>();
  constexpr int kSteps = L::steps, kSlices = L::slices, kTile = L::tile;
  __shared__ A sa[kSlices * CH], sb[kSlices * CH], sh[CH];
  const Place pl = place(tiles, groups, cgroups);
  const int tid = threadIdx.x, c = (tid & (L::lanes - 1)) * V, s = tid / L::lanes;
  const int ch = channel_of<V>(pl.group * CH + c, dim);
  const int count = pl.group * CH + c < dim ? dim - ch : 0;
  const long long t0 = steps - 1 - (pl.t * kTile + s * kSteps);  // the thread's latest step
  const T *pd = grad.p + pl.seq * grad.sb + t0 * grad.st + ch;
  const T *pg = gate.p + pl.seq * gate.sb + t0 * gate.st + ch;
  const T *px = x.p + pl.seq * x.sb + t0 * x.st + ch;
  const T *ph = h.p + pl.seq * h.sb + (t0 - 1) * h.st + ch;
  typedef typename Vec<T, V>::Words Words;
  Words wg[kSteps], wd[kSteps], wx[kSteps], wh[kSteps];
  if (count >= V && t0 >= 0) {  // steps before the first read it, and are not used
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      wg[i] = load_words<T, V, STREAM>(pg);
      wd[i] = load_words<T, V, STREAM>(pd);
      pg -= t0 > i ? gate.st : 0;
      pd -= t0 > i ? grad.st : 0;
    }
    if (t0 == 0) ph += h.st;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if constexpr (LOGITS) wx[i] = load_words<T, V, STREAM>(px);
      wh[i] = load_words<T, V, STREAM>(ph);
      px -= t0 > i ? x.st : 0;
      ph -= t0 > i + 1 ? h.st : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int n = t0 >= i ? count : 0;
      wg[i] = mmpn::words_of<T, V>(load_some<T, V>(pg - i * gate.st, n));
      wd[i] = mmpn::words_of<T, V>(load_some<T, V>(pd - i * grad.st, n));
      if constexpr (LOGITS) wx[i] = mmpn::words_of<T, V>(load_some<T, V>(px - i * x.st, n));
      wh[i] = mmpn::words_of<T, V>(load_some<T, V>(ph - i * h.st, t0 > i ? count : 0));
    }
  }
  A pa[V], pb[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    pa[k] = 1;
    pb[k] = 0;
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const Vec<T, V> g = mmpn::elements_of<T, V>(wg[i]), d = mmpn::elements_of<T, V>(wd[i]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      A f, u;
      factor<T, LOGITS>((A)g.e[k], (A)0, f, u);
      pa[k] = f * pa[k];
      pb[k] = f * ((A)d.e[k] + pb[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    sa[s * CH + c + k] = pa[k];
    sb[s * CH + c + k] = pb[k];
  }
  __syncthreads();
  if (tid < (CH < 64 ? 64 : CH)) {
    const int my = tid < CH ? tid : CH - 1;
    const int chan = channel_of<V>(pl.group * CH + my, dim);
    const bool on = tid < CH && pl.group * CH + my / V * V < dim && chan < dim;
    const long long at = pl.seq * dim + chan;
    A a, b;
    if (tid < CH) join_slices<A, CH, kSlices>(sa, sb, tid, a, b);
    A state = on && grad_final ? grad_final[at] : (A)0;
    if (tiles > 1) {
      if (on && pl.t > 0 && pl.t + 1 < tiles) publish<A, CH>(lk, pl.base + pl.t, my, 1, a, b);
      if (pl.t > 0)
        state = look_back<A, CH, kLook>(
            lk, pl.base, pl.t, my, on, state, [&](long long j, A &ja, A &jb) {
              ja = 1;
              jb = 0;
              if (!on) return;
              const long long q = steps - 1 - j * kTile;
              const T *qd = grad.p + pl.seq * grad.sb + q * grad.st + chan;
              const T *qg = gate.p + pl.seq * gate.sb + q * gate.st + chan;
              for (int w = 0; w < kSlices; ++w) {
                A wa = 1, wb = 0;
                for (int i = 0; i < kSteps; ++i) {
                  const long long r = w * kSteps + i;
                  A ff, uu;
                  factor<T, LOGITS>((A)qg[-r * gate.st], (A)0, ff, uu);
                  wa = ff * wa;
                  wb = ff * ((A)qd[-r * grad.st] + wb);
                }
                jb = mmpn::fma_of(wa, jb, wb);
                ja = wa * ja;
              }
            });
      if (on && pl.t + 1 < tiles)
        publish<A, CH>(lk, pl.base + pl.t, my, 2, mmpn::fma_of(a, state, b), (A)0);
    }
    if (tid < CH) sh[tid] = state;
  }
  __syncthreads();
  A carry[V];
#pragma unroll
  for (int k = 0; k < V; ++k)
    carry[k] = mmpn::fma_of(sa[s * CH + c + k], sh[c + k], sb[s * CH + c + k]);
  const long long o0 = (pl.seq * steps + t0) * dim + ch;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (t0 < i) break;
    mmpn::forget(wg[i]);
    mmpn::forget(wd[i]);
    const Vec<T, V> g = mmpn::elements_of<T, V>(wg[i]), d = mmpn::elements_of<T, V>(wd[i]);
    const Vec<T, V> before = mmpn::elements_of<T, V>(wh[i]);
    Vec<T, V> v, og, ox;
    if constexpr (LOGITS) v = mmpn::elements_of<T, V>(wx[i]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      A hb = (A)before.e[k];
      if (t0 == i) hb = initial && k < count ? initial[pl.seq * dim + ch + k] : (A)0;
      const A dd = (A)d.e[k] + carry[k];
      if constexpr (LOGITS) {
        A f, u;
        mmpn::sigmoid_pair<T>((A)g.e[k], f, u);
        const A du = dd * u;
        og.e[k] = (T)(du * f * (hb - (A)v.e[k]));
        ox.e[k] = (T)du;
        carry[k] = f * dd;
      } else {
        og.e[k] = (T)(dd * hb);
        ox.e[k] = (T)dd;
        carry[k] = (A)g.e[k] * dd;
      }
    }
    store_some<T, V>(grad_gate + o0 - (long long)i * dim, og, count);
    store_some<T, V>(grad_x + o0 - (long long)i * dim, ox, count);
  }
  if (t0 >= 0 && t0 < kSteps)
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < count) grad_initial[pl.seq * dim + ch + k] = carry[k];
}

// A thread per V channels goes through the steps, with the next kAhead on their
// way.  They are kept as words: float16 elements would be unpacked, and so waited
// for, before those on hand are used (64 x 500 x 1024 544 us instead of 121).  One
// step of 200 x 2048 float16 4 us, 253 x 170 x 1390 92 us, 3.9 TB/s.  Backwards, one step
// of 200 x 2048 4.2 us (float64 6.5), 16 steps 16 (48).
constexpr int kShortBlock = 256, kAhead = 4, kAheadGrad = 2;
template <typename T, bool LOGITS, int V>
__global__ __launch_bounds__(kShortBlock) void k_recur_short(
    long long n, long long steps, int dim, int vecs, Steps<T> gate, Steps<T> x,
    const typename Wide<T>::type *__restrict__ initial, T *__restrict__ h,
    typename Wide<T>::type *__restrict__ final_) {
  typedef typename Wide<T>::type A;
  const long long i = (long long)blockIdx.x * kShortBlock + threadIdx.x;
  if (i >= n) return;
  const long long b = i / vecs;
  // a row's last vector ends with it: some of its channels may be the vector
  // before's too, with the same results
  int c = (int)(i - b * vecs) * V;
  c = c + V > dim ? dim - V : c;
  Vec<A, V> s;
  if (initial) {
    s = mmpn::load_vec<A, V>(initial + b * dim + c);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) s.e[k] = 0;
  }
  const T *pg = gate.p + b * gate.sb + c, *px = x.p + b * x.sb + c;
  T *ph = h + b * steps * dim + c;
  typedef typename Vec<T, V>::Words Words;
  Words g[kAhead], v[kAhead];
  auto load = [&](long long t0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (t0 + j < steps) {
        g[j] = load_words<T, V>(pg + (t0 + j) * gate.st);
        v[j] = load_words<T, V>(px + (t0 + j) * x.st);
      }
  };
  load(0);
  for (long long t0 = 0; t0 < steps; t0 += kAhead) {
    Words gn[kAhead], vn[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      gn[j] = g[j];
      vn[j] = v[j];
    }
    load(t0 + kAhead);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (t0 + j >= steps) break;
      const Vec<T, V> gj = mmpn::elements_of<T, V>(gn[j]), vj = mmpn::elements_of<T, V>(vn[j]);
      Vec<T, V> o;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A f, u;
        factor<T, LOGITS>((A)gj.e[k], (A)vj.e[k], f, u);
        s.e[k] = mmpn::fma_of(f, s.e[k], u);
        o.e[k] = (T)s.e[k];
      }
      mmpn::store_vec<T, V, true>(ph + (t0 + j) * dim, o);
    }
  }
  mmpn::store_vec<A, V>(final_ + b * dim + c, s);
}

template <typename T, bool LOGITS, int V>
__global__ __launch_bounds__(kShortBlock) void k_recur_grad_short(
    long long n, long long steps, int dim, int vecs, Steps<T> grad, Steps<T> gate, Steps<T> x,
    Steps<T> h, const typename Wide<T>::type *__restrict__ initial,
    const typename Wide<T>::type *__restrict__ grad_final, T *__restrict__ grad_gate,
    T *__restrict__ grad_x, typename Wide<T>::type *__restrict__ grad_initial) {
  typedef typename Wide<T>::type A;
  const long long i = (long long)blockIdx.x * kShortBlock + threadIdx.x;
  if (i >= n) return;
  const long long b = i / vecs;
  // a row's last vector ends with it: some of its channels may be the vector
  // before's too, with the same results
  int c = (int)(i - b * vecs) * V;
  c = c + V > dim ? dim - V : c;
  Vec<A, V> carry;
  if (grad_final) {
    carry = mmpn::load_vec<A, V>(grad_final + b * dim + c);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) carry.e[k] = 0;
  }
  const T *pd = grad.p + b * grad.sb + c, *pg = gate.p + b * gate.sb + c;
  const T *px = x.p + b * x.sb + c, *ph = h.p + b * h.sb + c;
  typedef typename Vec<T, V>::Words Words;
  Words d[kAheadGrad], g[kAheadGrad], v[kAheadGrad], p[kAheadGrad];
  auto load = [&](long long t0) {  // t0 and the steps before it
#pragma unroll
    for (int j = 0; j < kAheadGrad; ++j) {
      const long long t = t0 - j;
      if (t < 0) break;
      d[j] = load_words<T, V>(pd + t * grad.st);
      g[j] = load_words<T, V>(pg + t * gate.st);
      if constexpr (LOGITS) v[j] = load_words<T, V>(px + t * x.st);
      if (t > 0) p[j] = load_words<T, V>(ph + (t - 1) * h.st);
    }
  };
  load(steps - 1);
  for (long long t0 = steps - 1; t0 >= 0; t0 -= kAheadGrad) {
    Words dn[kAheadGrad], gn[kAheadGrad], vn[kAheadGrad], pn[kAheadGrad];
#pragma unroll
    for (int j = 0; j < kAheadGrad; ++j) {
      dn[j] = d[j];
      gn[j] = g[j];
      if constexpr (LOGITS) vn[j] = v[j];
      pn[j] = p[j];
    }
    load(t0 - kAheadGrad);
#pragma unroll
    for (int j = 0; j < kAheadGrad; ++j) {
      const long long t = t0 - j;
      if (t < 0) break;
      const Vec<T, V> dj = mmpn::elements_of<T, V>(dn[j]), gj = mmpn::elements_of<T, V>(gn[j]);
      const Vec<T, V> pj = mmpn::elements_of<T, V>(pn[j]);
      Vec<T, V> vj, og, ox;
      if constexpr (LOGITS) vj = mmpn::elements_of<T, V>(vn[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A hb = (A)pj.e[k];
        if (t == 0) hb = initial ? initial[b * dim + c + k] : (A)0;
        const A dd = (A)dj.e[k] + carry.e[k];
        if constexpr (LOGITS) {
          A f, u;
          mmpn::sigmoid_pair<T>((A)gj.e[k], f, u);
          const A du = dd * u;
          og.e[k] = (T)(du * f * (hb - (A)vj.e[k]));
          ox.e[k] = (T)du;
          carry.e[k] = f * dd;
        } else {
          og.e[k] = (T)(dd * hb);
          ox.e[k] = (T)dd;
          carry.e[k] = (A)gj.e[k] * dd;
        }
      }
      const long long o = (b * steps + t) * dim + c;
      mmpn::store_vec<T, V, true>(grad_gate + o, og);
      mmpn::store_vec<T, V, true>(grad_x + o, ox);
    }
  }
  mmpn::store_vec<A, V>(grad_initial + b * dim + c, carry);
}

// The tiles of a call, and their descriptors.
struct Plan {
  int64_t tiles, groups;
  int cgroups;
};
template <typename T, typename L> Plan plan(int64_t batch, int64_t steps, int64_t dim) {
  Plan p;
  p.tiles = mmpi::ceil_div(steps, L::tile);
  p.cgroups = (int)mmpi::ceil_div(dim, L::template channels<T>());
  p.groups = batch * p.cgroups;
  return p;
}
template <typename T, typename L> int look_of(const Plan &p, const char *what, Look *lk) {
  typedef typename Wide<T>::type A;
  *lk = Look{nullptr, 0, 0, 0};
  if (p.tiles == 1) return MMP_OK;
  if (mmpn::capturing()) return mmpn::refuse_capture(what);
  int st = MMP_OK;
  lk->desc = (unsigned long long *)mmpi::scratch(
      mmpi::SCRATCH_RECUR_TILES,
      8ull * words_of<A>() * L::template channels<T>() * p.tiles * p.groups, &st);
  if (st) return st;
  const mmpi::WaitParams w = mmpi::wait_params();
  lk->gen = mmpi::next_generation();
  lk->read_gen = (lk->gen + w.tag_offset) & 0x3fffffffu;
  lk->polls = w.tag_offset ? 1 : kPolls;
  return MMP_OK;
}

constexpr int64_t kMost = 0x7fff0000LL;  // room for a group past the end in 32 bits

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
  if (dim > kMost) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence: 2^31 channels");
  MMP_DISPATCH_FLOAT(dtype, "mmp_recurrence", {
    typedef typename Wide<T>::type A;
    const Steps<T> sg{(const T *)gate, gate_sb, gate_st}, sx{(const T *)x, x_sb, x_st};
    constexpr int kVec = kShortBytes / sizeof(T);
    const int vec = dim >= kVec ? kVec : 1;
    const int64_t vecs = mmpi::ceil_div(dim, vec), n = batch * vecs;
    const mmpi::RecurForm form = mmpi::recur_form(sizeof(T), batch, steps, dim);
    if (form == mmpi::kRecurThreads) {
      const int64_t blocks = mmpi::ceil_div(n, kShortBlock);
      if (!mmpi::grid_fits(blocks, kShortBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence: too many channels");
      auto kernel = vec == kVec
                        ? (logits ? k_recur_short<T, true, kVec> : k_recur_short<T, false, kVec>)
                        : (logits ? k_recur_short<T, true, 1> : k_recur_short<T, false, 1>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kShortBlock), 0, mmpi::stream(),
                         (long long)n, (long long)steps, (int)dim, (int)vecs, sg, sx,
                         (const A *)initial, (T *)h, (A *)final_);
      return mmpi::check_launch("mmp_recurrence(short)");
    }
    auto launch = [&](auto layout) -> int {
      typedef decltype(layout) L;
      const Plan p = plan<T, L>(batch, steps, dim);
      if (!mmpi::grid_fits(p.groups * p.tiles, kBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence: too many tiles");
      std::lock_guard<std::mutex> lock(mmpi::launch_mutex());
      Look lk;
      if (int st = look_of<T, L>(p, "mmp_recurrence", &lk)) return st;
      auto kernel = mmpi::recur_past_caches(3, sizeof(T), batch, steps, dim)
                        ? (logits ? k_recur_tiles<T, true, L, true>
                                  : k_recur_tiles<T, false, L, true>)
                        : (logits ? k_recur_tiles<T, true, L, false>
                                  : k_recur_tiles<T, false, L, false>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(p.groups * p.tiles)), dim3(kBlock), 0,
                         mmpi::stream(), (long long)steps, (int)dim, (long long)p.tiles,
                         (long long)p.groups, p.cgroups, sg, sx, (const A *)initial, (T *)h,
                         (A *)final_, lk);
      return mmpi::check_launch("mmp_recurrence");
    };
    switch (form) {
      case mmpi::kRecurBrief: return launch(ForwardBrief());
      case mmpi::kRecurWide: return launch(ForwardWide<T>());
      case mmpi::kRecurFew: return launch(ForwardFew());
      default: return launch(ForwardLong());
    }
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
  if (dim > kMost) return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence_grad: 2^31 channels");
  MMP_DISPATCH_FLOAT(dtype, "mmp_recurrence_grad", {
    typedef typename Wide<T>::type A;
    const Steps<T> sd{(const T *)grad, grad_sb, grad_st}, sg{(const T *)gate, gate_sb, gate_st};
    const Steps<T> sx{(const T *)x, x_sb, x_st}, sh{(const T *)h, h_sb, h_st};
    const mmpi::RecurForm form = mmpi::recur_grad_form(sizeof(T), batch, steps, dim);
    if (form == mmpi::kRecurThreads) {
      constexpr int kVec = kShortBytes / sizeof(T);
      const int vec = dim >= kVec ? kVec : 1;
      const int64_t vecs = mmpi::ceil_div(dim, vec), n = batch * vecs;
      const int64_t blocks = mmpi::ceil_div(n, kShortBlock);
      if (!mmpi::grid_fits(blocks, kShortBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence_grad: too many channels");
      auto kernel = vec == kVec
                        ? (logits ? k_recur_grad_short<T, true, kVec> : k_recur_grad_short<T, false, kVec>)
                        : (logits ? k_recur_grad_short<T, true, 1> : k_recur_grad_short<T, false, 1>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kShortBlock), 0, mmpi::stream(),
                         (long long)n, (long long)steps, (int)dim, (int)vecs, sd, sg, sx, sh,
                         (const A *)initial, (const A *)grad_final, (T *)grad_gate, (T *)grad_x,
                         (A *)grad_initial);
      return mmpi::check_launch("mmp_recurrence_grad(short)");
    }
    auto launch = [&](auto layout) -> int {
      typedef decltype(layout) L;
      const Plan p = plan<T, L>(batch, steps, dim);
      if (!mmpi::grid_fits(p.groups * p.tiles, kBlock))
        return mmpi::fail(MMP_E_UNSUPPORTED, "mmp_recurrence_grad: too many tiles");
      std::lock_guard<std::mutex> lock(mmpi::launch_mutex());
      Look lk;
      if (int st = look_of<T, L>(p, "mmp_recurrence_grad", &lk)) return st;
      auto kernel = mmpi::recur_past_caches(logits ? 6 : 5, sizeof(T), batch, steps, dim)
                        ? (logits ? k_recur_grad_tiles<T, true, L, true>
                                  : k_recur_grad_tiles<T, false, L, true>)
                        : (logits ? k_recur_grad_tiles<T, true, L, false>
                                  : k_recur_grad_tiles<T, false, L, false>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(p.groups * p.tiles)), dim3(kBlock), 0,
                         mmpi::stream(), (long long)steps, (int)dim, (long long)p.tiles,
                         (long long)p.groups, p.cgroups, sd, sg, sx, sh, (const A *)initial,
                         (const A *)grad_final, (T *)grad_gate, (T *)grad_x, (A *)grad_initial,
                         lk);
      return mmpi::check_launch("mmp_recurrence_grad");
    };
    switch (form) {
      case mmpi::kRecurWide: return launch(BackwardWide());
      case mmpi::kRecurFew: return launch(BackwardFew());
      default: return launch(BackwardLong());
    }
  })
}
