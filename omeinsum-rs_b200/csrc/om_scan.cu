// Gated linear recurrence h_t = a_t h_{t-1} + b_t and its backward pass
//     S_t = a_t (dh_t + S_{t+1}),   G_t = dh_t + S_{t+1}.
//
// A step is the map s -> P s + Q with (P, Q) = (a, b) (backward: (a, a dh)), and
// maps compose, so time can be cut into chunks that run side by side:
//   map_kernel    composes the steps of each chunk, and of the consecutive
//                 chunks of a block together;
//   step_kernel   joins the maps before its chunk to the state that enters it
//                 and takes the chunk's steps one by one, writing the results.
// A warp has 32 lanes of 8 bytes of channels (one channel where rows are not
// 8-byte aligned or channels are not contiguous) and a chunk's steps; the next
// steps are under way while some are in use, and the state is in registers, so
// nothing but the maps passes through shared memory. Sums are formed in one
// order whatever the timing. Where the channels alone fill the card, a sequence
// is one chunk and map_kernel does not run.
//
// step_kernel moves 3 arrays (forward) or 5 to 6 (backward) per element, map_kernel 2
// more. Long sequences are bound by HBM: 65537 x 1032 bf16 map_kernel 270 MB in 45 to
// 47 us (5.8 to 6.0 TB/s), step_kernel 406 MB in 65 to 68 us (6.0 to 6.2). Shorter ones are not: the four
// launches of 4 x 4096 x 2048 bf16 sigmoid with the backward pass, 31 to 63 us each and
// 168 together, have DRAM busy for 50 to 70 %, and its 604 MB need 92 us at the card's
// copy rate; what is left is the ramps, the latency of the chunks' joined maps and,
// for sigmoid gates, an exponential and a reciprocal per element and kernel (150 us
// with linear gates). (One pass over tiles in shared memory that looked back at one
// another read everything once, but spent its time on the tiles' bookkeeping: 217
// us.)
//
// The backward pass takes h_{t-1} as the forward returned it, so in 16 bits dgate
// carries that rounding beside its own (relative to 64 bits 2.3e-3 against 1.7e-3
// with linear gates in bf16, 1.8e-3 with sigmoid gates): a 32-bit copy would be 4
// more bytes written and read per element, forward and backward.
#include <algorithm>

#include "om_convert.cuh"

namespace om {
namespace {

struct ScanArgs {
  int64_t D, T, B;
  const void* gate;
  int64_t gd, gt, gb;
  const void* x;
  int64_t xd, xt, xb;
  const void* h0;
  const int32_t* lengths;
  void* h;
  int64_t hd, ht, hb;
  void* h_last;
  // backward only
  const void* dh;
  int64_t ed, et, eb;
  const void* dh_last;
  void* dgate;
  int64_t pd, pt, pb;
  void* dx;
  int64_t qd, qt, qb;
  void* dh0;
};

// Warps of a block and blocks of an SM, by the bytes of a row that a lane has.
// 16 warps of 8-byte rows keep twice eight steps in registers (32 with half as
// many under way are up to 20 % slower), in blocks of four, which share out
// evenly; narrower rows do better in blocks of eight (7 x 1531 x 1001 f32 with
// the backward pass: 106 us, in blocks of four 121).
constexpr int warps_of(int lane_bytes) { return lane_bytes == 8 ? 4 : 8; }
constexpr int blocks_of(int lane_bytes) { return lane_bytes == 8 ? 4 : lane_bytes == 4 ? 3 : 2; }

struct ChunkArgs {
  int64_t groups;   // of VEC channels, a lane's
  int64_t pitch;    // channels of all columns of 32 lanes
  int columns;
  int warps_t;      // warps of a block that take consecutive chunks of one column
  int chunks;       // of a sequence
  int64_t steps;    // of a chunk
  int narrow;       // channel numbers fit 32 bits
  void* maps;       // [chunk][channel] pairs (P, Q)
  void* joined;     // [block of chunks][channel]
  void* start;      // [channel] the caller's state, which h_last may overwrite
};

// ---- arithmetic on the channels of a lane ------------------------------------------
// Two f32 channels share one instruction (the f32x2 forms of sm_100); one alone
// and f64 take the plain ones.

template <typename S, int N>
struct Pack;
template <>
struct Pack<float, 2> {
  float2 v;
  __device__ __forceinline__ float get(int i) const { return i ? v.y : v.x; }
  __device__ __forceinline__ void set(int i, float s) { (i ? v.y : v.x) = s; }
  static __device__ __forceinline__ Pack all(float s) { return Pack{make_float2(s, s)}; }
};
template <typename S>
struct Pack<S, 1> {
  S v;
  __device__ __forceinline__ S get(int) const { return v; }
  __device__ __forceinline__ void set(int, S s) { v = s; }
  static __device__ __forceinline__ Pack all(S s) { return Pack{s}; }
};
using Two = Pack<float, 2>;

__device__ __forceinline__ uint64_t bits_of(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ Two of_bits(uint64_t r) {
  Two p;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(p.v.x), "=f"(p.v.y) : "l"(r));
  return p;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a.v)), "l"(bits_of(b.v)));
  return of_bits(r);
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a.v)), "l"(bits_of(b.v)));
  return of_bits(r);
}
__device__ __forceinline__ Two mad(Two a, Two b, Two c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(bits_of(a.v)), "l"(bits_of(b.v)), "l"(bits_of(c.v)));
  return of_bits(r);
}
template <typename S>
__device__ __forceinline__ Pack<S, 1> operator*(Pack<S, 1> a, Pack<S, 1> b) {
  return Pack<S, 1>{a.v * b.v};
}
template <typename S>
__device__ __forceinline__ Pack<S, 1> operator+(Pack<S, 1> a, Pack<S, 1> b) {
  return Pack<S, 1>{a.v + b.v};
}
template <typename S>
__device__ __forceinline__ Pack<S, 1> mad(Pack<S, 1> a, Pack<S, 1> b, Pack<S, 1> c) {
  return Pack<S, 1>{fma(a.v, b.v, c.v)};
}

// a = sigmoid(g) and 1 - a without cancellation. f32: an exponential formed as
// a power of two and an approximate reciprocal, together below 24 half steps
// for |g| <= 16 (most of it the rounding of the exponent); values below f32's
// normal numbers become zero.
__device__ __forceinline__ float power_of_two(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void sigmoid_pair(Two g, Two* a, Two* keep) {
  const Two t = g * Two::all(-1.4426950408889634f);
  const Two e{make_float2(power_of_two(t.v.x), power_of_two(t.v.y))};
  const Two d = e + Two::all(1.f);
  const Two r{make_float2(inverse(d.v.x), inverse(d.v.y))};
  const Two small = e * r, large = mad(r, Two::all(-1.f), Two::all(1.f));
  keep->v.x = e.v.x > 1.f ? large.v.x : small.v.x;  // e may be infinite, r is then 0
  keep->v.y = e.v.y > 1.f ? large.v.y : small.v.y;
  *a = r;
}
__device__ __forceinline__ void sigmoid_pair(Pack<float, 1> g, Pack<float, 1>* a,
                                             Pack<float, 1>* keep) {
  const float e = power_of_two(g.v * -1.4426950408889634f), r = inverse(e + 1.f);
  keep->v = e > 1.f ? 1.f - r : e * r;
  a->v = r;
}
__device__ __forceinline__ void sigmoid_pair(Pack<double, 1> g, Pack<double, 1>* a,
                                             Pack<double, 1>* keep) {
  const double e = exp(-fabs(g.v)), r = 1 / (1 + e);
  a->v = g.v >= 0 ? r : e * r;
  keep->v = g.v >= 0 ? e * r : r;
  if (g.v != g.v) a->v = keep->v = g.v;
}

// ---- a lane's channels of one step ----------------------------------------------------

// V channels as they lie in memory
template <int BYTES>
struct Raw;
template <>
struct Raw<2> {
  using Type = uint16_t;
};
template <>
struct Raw<4> {
  using Type = uint32_t;
};
template <>
struct Raw<8> {
  using Type = uint2;
};

template <typename T, int V>
struct Lane {
  using S = typename Elem<T>::State;
  static constexpr int W = sizeof(S) == 4 && V % 2 == 0 ? 2 : 1;  // channels of a pack
  static constexpr int N = V / W;
  using K = Pack<S, W>;
  using R = typename Raw<sizeof(T) * V>::Type;
  K v[N];
  static __device__ __forceinline__ Lane of(R r) {
    Lane l;
    if constexpr (V == 1) {
      T t;
      memcpy(&t, &r, sizeof(T));
      l.v[0].v = Elem<T>::load(t);
    } else if constexpr (sizeof(T) == 4) {
      l.v[0].v = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
    } else {
      l.v[0] = two(r.x);
      l.v[1] = two(r.y);
    }
    return l;
  }
  __device__ __forceinline__ R raw() const {
    R r;
    if constexpr (V == 1) {
      const T t = Elem<T>::store(v[0].v);
      memcpy(&r, &t, sizeof(T));
    } else if constexpr (sizeof(T) == 4) {
      r = make_uint2(__float_as_uint(v[0].v.x), __float_as_uint(v[0].v.y));
    } else {
      r = make_uint2(pack2(v[0].v.x, v[0].v.y, T()), pack2(v[1].v.x, v[1].v.y, T()));
    }
    return r;
  }
  static __device__ __forceinline__ Two two(uint32_t u) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return Two{make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u))};
    } else {
      __half2 h;
      memcpy(&h, &u, 4);
      return Two{__half22float2(h)};
    }
  }
  __device__ __forceinline__ S get(int i) const { return v[i / W].get(i % W); }
  __device__ __forceinline__ void set(int i, S s) { v[i / W].set(i % W, s); }
};

template <typename S>
struct alignas(2 * sizeof(S)) Pair {
  S p, q;
};

// The map of V channels
template <typename T, int V>
struct Map {
  using S = typename Elem<T>::State;
  using L = Lane<T, V>;
  L p, q;
  static __device__ __forceinline__ Map identity() {
    Map m;
#pragma unroll
    for (int i = 0; i < L::N; ++i) m.p.v[i] = L::K::all(S(1)), m.q.v[i] = L::K::all(S(0));
    return m;
  }
  __device__ __forceinline__ void then(const Map& m) {
    q = m.at(q);
#pragma unroll
    for (int i = 0; i < L::N; ++i) p.v[i] = m.p.v[i] * p.v[i];
  }
  // A state of zero leaves q, also where gates above one let p overflow (what
  // is not a number in a step is in q already).
  __device__ __forceinline__ L at(const L& s) const {
    L r;
#pragma unroll
    for (int i = 0; i < L::N; ++i) r.v[i] = mad(p.v[i], s.v[i], q.v[i]);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (s.get(i) == S(0)) r.set(i, q.get(i));
    return r;
  }
  __device__ __forceinline__ void put(Pair<S>* to) const {
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = Pair<S>{p.get(i), q.get(i)};
  }
  static __device__ __forceinline__ Map take(const Pair<S>* from) {
    Map m;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const Pair<S> w = from[i];
      m.p.set(i, w.p);
      m.q.set(i, w.q);
    }
    return m;
  }
};

// Where a lane's channels are, and which steps of its chunk exist
struct Place {
  int64_t c0, b, d;   // first channel, its batch and place in the row
  int64_t t0, t1;     // the chunk
  int64_t end;        // steps before it exist (t1 at most, t0 at least)
  bool live;          // the lane has channels, and the chunk is one
  int order;          // chunk in the order in which states pass
  int col;
};
template <typename T, int V, bool BWD>
__device__ __forceinline__ Place place_of(const ScanArgs& p, const ChunkArgs& a, int col, int order) {
  Place r;
  const int lane = threadIdx.x & 31;
  r.col = col;
  r.order = order;
  const int64_t g = (int64_t)col * 32 + lane;
  r.c0 = g * V;
  r.live = col < a.columns && g < a.groups && order < a.chunks;
  const int64_t c = r.live ? r.c0 : 0;
  r.b = a.narrow ? (int64_t)((uint32_t)c / (uint32_t)p.D) : c / p.D;
  r.d = c - r.b * p.D;
  const int64_t k = BWD ? a.chunks - 1 - order : order;
  r.t0 = k * a.steps;
  r.t1 = min(r.t0 + a.steps, p.T);
  r.end = r.t1;
  if (p.lengths && r.live) r.end = max(r.t0, min((int64_t)p.lengths[r.b], r.t1));
  return r;
}

template <typename T, int V>
__device__ __forceinline__ typename Lane<T, V>::R fetch(const T* p) {
  using R = typename Lane<T, V>::R;
  return __ldg(reinterpret_cast<const R*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void keep(T* p, const Lane<T, V>& l) {
  *reinterpret_cast<typename Lane<T, V>::R*>(p) = l.raw();
}

// NA arrays' rows of a lane, in order: U rows are in use while the next U are
// under way. start() asks for the first ones.
template <typename T, int V, int NA, int U>
struct Stream {
  using R = typename Lane<T, V>::R;
  const T* p[NA];     // the next row
  int64_t step[NA];   // elements between rows
  int64_t n;          // rows
  int64_t asked = 0;
  R a[U][NA];

  __device__ __forceinline__ void ask(R (&r)[U][NA]) {
    if (asked + U <= n) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < NA; ++k) r[u][k] = fetch<T, V>(p[k] + u * step[k]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (asked + u < n) {
#pragma unroll
          for (int k = 0; k < NA; ++k) r[u][k] = fetch<T, V>(p[k] + u * step[k]);
        }
    }
    asked += U;
#pragma unroll
    for (int k = 0; k < NA; ++k) p[k] += U * step[k];
  }
  __device__ __forceinline__ void start() { ask(a); }
  template <typename F>
  __device__ __forceinline__ void use(const R (&r)[U][NA], int64_t i, F& f) {
    if (i + U <= n) {
#pragma unroll
      for (int u = 0; u < U; ++u) f(r[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < n) f(r[u]);
    }
  }
  // f(a row of each array), n times
  template <typename F>
  __device__ __forceinline__ void run(F f) {
    R b[U][NA];
    for (int64_t i = 0; i < n; i += 2 * U) {
      ask(b);
      use(a, i, f);
      if (i + U >= n) break;
      ask(a);
      use(b, i + U, f);
    }
  }
};

template <typename S>
__device__ __forceinline__ bool finite(S s) {
  return fabs(s) < S(INFINITY);
}

// ---- the maps of the chunks -------------------------------------------------------------

template <typename T, int V, bool SIG, bool BWD>
__device__ __forceinline__ void compose(Map<T, V>& m, Lane<T, V> g, Lane<T, V> x) {
  using L = Lane<T, V>;
#pragma unroll
  for (int i = 0; i < L::N; ++i) {
    typename L::K f = g.v[i], b = x.v[i];
    if constexpr (SIG) {
      typename L::K keep;
      sigmoid_pair(f, &f, &keep);
      if constexpr (!BWD) b = b * keep;
    }
    m.q.v[i] = BWD ? f * (b + m.q.v[i]) : mad(f, m.q.v[i], b);
    m.p.v[i] = f * m.p.v[i];
  }
}

template <typename T, int V, bool SIG, bool BWD>
__global__ void __launch_bounds__(warps_of(sizeof(T) * V) * 32, blocks_of(sizeof(T) * V)) map_kernel(const __grid_constant__ ScanArgs p,
                                                            const __grid_constant__ ChunkArgs a) {
  using S = typename Elem<T>::State;
  using L = Lane<T, V>;
  constexpr int WARPS = warps_of(sizeof(T) * V);
  __shared__ Pair<S> part[WARPS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wt = a.warps_t, team = warp / wt, tw = warp % wt;
  const int col = (int)(blockIdx.x % (unsigned)((a.columns + WARPS / wt - 1) / (WARPS / wt))) * (WARPS / wt) + team;
  const int block = (int)(blockIdx.x / (unsigned)((a.columns + WARPS / wt - 1) / (WARPS / wt)));
  const Place at = place_of<T, V, BWD>(p, a, col, block * wt + tw);
  Map<T, V> m = Map<T, V>::identity();
  // the last chunk's map is not needed
  if (at.live && at.order < a.chunks - 1) {
    const int64_t first = BWD ? at.end - 1 : at.t0;
    const int64_t xt = BWD ? p.et : p.xt;
    Stream<T, V, 2, 8> rows;
    rows.n = at.end - at.t0;
    rows.p[0] = (const T*)p.gate + at.b * p.gb + at.d * p.gd + first * p.gt;
    rows.p[1] = BWD ? (const T*)p.dh + at.b * p.eb + at.d * p.ed + first * xt
                    : (const T*)p.x + at.b * p.xb + at.d * p.xd + first * xt;
    rows.step[0] = BWD ? -p.gt : p.gt;
    rows.step[1] = BWD ? -xt : xt;
    rows.start();
    rows.run([&](const typename L::R (&r)[2]) { compose<T, V, SIG, BWD>(m, L::of(r[0]), L::of(r[1])); });
    m.put((Pair<S>*)a.maps + (int64_t)at.order * a.pitch + at.c0);
    const S* from = (const S*)(BWD ? p.dh_last : p.h0);
    if (at.order == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) ((S*)a.start)[at.c0 + i] = from ? from[at.c0 + i] : S(0);
    }
  }
  if (wt < WARPS) return;  // a block has no more chunks than the sequence
  m.put(&part[warp][lane * V]);
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += WARPS * 32) {
    S P = 1, Q = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const Pair<S> k = part[w][c];
      Q = Q == S(0) ? k.q : k.p * Q + k.q;  // as Map::at
      P = k.p * P;
    }
    ((Pair<S>*)a.joined)[(int64_t)block * a.pitch + (int64_t)col * 32 * V + c] = Pair<S>{P, Q};
  }
}

// ---- the steps ------------------------------------------------------------------------

// A chunk's steps: open() asks for the first rows, take() goes through them from
// the state s that enters and writes the results.
template <typename T, int V, bool SIG, bool BWD>
struct Steps {
  using S = typename Elem<T>::State;
  using L = Lane<T, V>;
  using K = typename L::K;
  using R = typename L::R;
  static constexpr int NA = BWD ? (SIG ? 4 : 3) : 2;
  Stream<T, V, NA, NA == 2 ? 8 : NA == 3 ? 4 : 3> rows;
  bool start;  // backward: step 0, which has no h before it, comes after the others
  const T *g, *x, *e;

  __device__ __forceinline__ void aim(const ScanArgs& p, const Place& at) {
    start = BWD && at.t0 == 0 && at.end > 0;
    g = (const T*)p.gate + at.b * p.gb + at.d * p.gd;
    x = (const T*)p.x + at.b * p.xb + at.d * p.xd;
    e = BWD ? (const T*)p.dh + at.b * p.eb + at.d * p.ed : nullptr;
    rows.n = at.live ? at.end - at.t0 - start : 0;
    if constexpr (!BWD) {
      rows.p[0] = g + at.t0 * p.gt, rows.step[0] = p.gt;
      rows.p[1] = x + at.t0 * p.xt, rows.step[1] = p.xt;
    } else {
      const int64_t t = at.end - 1;
      rows.p[0] = g + t * p.gt, rows.step[0] = -p.gt;
      rows.p[1] = e + t * p.et, rows.step[1] = -p.et;
      rows.p[2] = (const T*)p.h + at.b * p.hb + at.d * p.hd + (t - 1) * p.ht, rows.step[2] = -p.ht;
      if constexpr (SIG) rows.p[3] = x + t * p.xt, rows.step[3] = -p.xt;
    }
  }

  __device__ __forceinline__ void take(const ScanArgs& p, const ChunkArgs& a, const Place& at, L s) {
    L zero;
#pragma unroll
    for (int i = 0; i < V; ++i) zero.set(i, S(0));
    if constexpr (!BWD) {
      T* h = (T*)p.h + at.b * p.hb + at.d * p.hd + at.t0 * p.ht;
      rows.run([&](const R (&r)[2]) {
        const L f = L::of(r[0]), b = L::of(r[1]);
#pragma unroll
        for (int i = 0; i < L::N; ++i) {
          K fi = f.v[i], bi = b.v[i];
          if constexpr (SIG) {
            K rest;
            sigmoid_pair(fi, &fi, &rest);
            bi = bi * rest;
          }
          s.v[i] = mad(fi, s.v[i], bi);
        }
        keep<T, V>(h, s);
        h += p.ht;
      });
      for (int64_t t = at.end; t < at.t1; ++t, h += p.ht) keep<T, V>(h, zero);
    } else {
      T* dg = (T*)p.dgate + at.b * p.pb + at.d * p.pd + (at.t1 - 1) * p.pt;
      T* dx = (T*)p.dx + at.b * p.qb + at.d * p.qd + (at.t1 - 1) * p.qt;
      for (int64_t t = at.t1; t > at.end; --t, dg -= p.pt, dx -= p.qt)
        keep<T, V>(dg, zero), keep<T, V>(dx, zero);
      auto back = [&](R rg, R re, const L& before, R rx) {
        const L f = L::of(rg), d = L::of(re), v = L::of(rx);
        L og, ox;
#pragma unroll
        for (int i = 0; i < L::N; ++i) {
          K fi = f.v[i];
          const K total = d.v[i] + s.v[i];
          if constexpr (SIG) {
            K rest;
            sigmoid_pair(fi, &fi, &rest);
            ox.v[i] = total * rest;
            og.v[i] = mad(v.v[i], K::all(S(-1)), before.v[i]) * fi * ox.v[i];
          } else {
            ox.v[i] = total;
            og.v[i] = total * before.v[i];
          }
          s.v[i] = fi * total;
        }
        keep<T, V>(dg, og);
        keep<T, V>(dx, ox);
        dg -= p.pt;
        dx -= p.qt;
      };
      rows.run([&](const R (&r)[NA]) { back(r[0], r[1], L::of(r[2]), r[NA - 1]); });
      if (start) {
        L before;
#pragma unroll
        for (int i = 0; i < V; ++i) before.set(i, p.h0 ? ((const S*)p.h0)[at.c0 + i] : S(0));
        const R rg = fetch<T, V>(g);
        back(rg, fetch<T, V>(e), before, SIG ? fetch<T, V>(x) : rg);
      }
    }
    // the state that leaves the last chunk
    S* last = (S*)(BWD ? p.dh0 : p.h_last);
    if (last && at.order == a.chunks - 1) {
#pragma unroll
      for (int i = 0; i < V; ++i) last[at.c0 + i] = s.get(i);
    }
  }
};

// The chunk of a lane whose joined state is not finite in some channel. Where a
// group's product of gates overflows, its map gives infinity or NaN for states that
// the steps themselves keep finite (and NaN for an infinite state where it
// underflows); so such a channel's state is formed step by step from the caller's,
// as far as it is not NaN already. Out of line and to the chunk's end, so that the
// ordinary case keeps nothing for it (with the steps after it in the kernel, 7 x 1531
// x 1001 f32 took 95 us and not 89). Bound by the latency of one channel's loads: an
// infinity at the start of 65537 x 1032 bf16 takes 5.9 ms, finite inputs 0.12 ms.
template <typename T, int V, bool SIG, bool BWD>
__device__ __noinline__ void walk(const ScanArgs& p, const ChunkArgs& a, int col, int order,
                                  Lane<T, V> joined) {
  using S = typename Elem<T>::State;
  using L = Lane<T, V>;
  using R = typename L::R;
  constexpr int U = 8;  // steps under way
  const Place at = place_of<T, V, BWD>(p, a, col, order);
  const int64_t length = p.lengths ? max((int64_t)0, min((int64_t)p.lengths[at.b], p.T)) : p.T;
  const int64_t n = BWD ? length - at.t1 : min(length, at.t0), first = BWD ? length - 1 : 0;
  const int64_t gt = BWD ? -p.gt : p.gt, bt = BWD ? -p.et : p.xt;
  const T* g = (const T*)p.gate + at.b * p.gb + at.d * p.gd + first * p.gt;
  const T* b = BWD ? (const T*)p.dh + at.b * p.eb + at.d * p.ed + first * p.et
                   : (const T*)p.x + at.b * p.xb + at.d * p.xd + first * p.xt;
  L s;
#pragma unroll
  for (int i = 0; i < V; ++i) s.set(i, ((const S*)a.start)[at.c0 + i]);
  for (int64_t t = 0; t < n; t += U, g += U * gt, b += U * bt) {
    R rg[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < n) rg[u] = fetch<T, V>(g + u * gt), rb[u] = fetch<T, V>(b + u * bt);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u >= n) break;
      const L f = L::of(rg[u]), v = L::of(rb[u]);
#pragma unroll
      for (int i = 0; i < L::N; ++i) {
        typename L::K fi = f.v[i], bi = v.v[i], rest;
        if constexpr (SIG) {
          sigmoid_pair(fi, &fi, &rest);
          if constexpr (!BWD) bi = bi * rest;
        }
        s.v[i] = BWD ? fi * (bi + s.v[i]) : mad(fi, s.v[i], bi);
      }
    }
    bool gone = true;  // a NaN stays
#pragma unroll
    for (int i = 0; i < V; ++i) gone &= s.get(i) != s.get(i) || finite(joined.get(i));
    if (gone) break;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (!finite(joined.get(i))) joined.set(i, s.get(i));
  Steps<T, V, SIG, BWD> steps;
  steps.aim(p, at);
  steps.rows.start();
  steps.take(p, a, at, joined);
}

template <typename T, int V, bool SIG, bool BWD>
__global__ void __launch_bounds__(warps_of(sizeof(T) * V) * 32, blocks_of(sizeof(T) * V)) step_kernel(const __grid_constant__ ScanArgs p,
                                                             const __grid_constant__ ChunkArgs a) {
  using S = typename Elem<T>::State;
  using L = Lane<T, V>;
  constexpr int WARPS = warps_of(sizeof(T) * V);
  __shared__ Pair<S> part[WARPS][32 * V], chunk[WARPS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wt = a.warps_t, team = warp / wt, tw = warp % wt;
  const unsigned per = (unsigned)((a.columns + WARPS / wt - 1) / (WARPS / wt));
  const int blocks = (a.chunks + wt - 1) / wt;
  const int col = (int)(blockIdx.x % per) * (WARPS / wt) + team;
  const int block = blocks - 1 - (int)(blockIdx.x / per);  // the last chunks first
  const Place at = place_of<T, V, BWD>(p, a, col, block * wt + tw);

  // the state that enters: the caller's, through the maps of the blocks of
  // chunks before this one (shared out over the warps) and of the chunks
  // before this warp's
  Steps<T, V, SIG, BWD> steps;
  steps.aim(p, at);
  const S* from = (const S*)(a.chunks > 1 ? a.start : BWD ? p.dh_last : p.h0);
  L s;
#pragma unroll
  for (int i = 0; i < V; ++i) s.set(i, from && at.live ? from[at.c0 + i] : S(0));
  if (a.chunks > 1) {
    // this warp's own chunk's map goes to shared memory for the warps behind it
    Map<T, V> own = Map<T, V>::identity();
    if (at.live && at.order < a.chunks - 1) own = Map<T, V>::take((const Pair<S>*)a.maps + at.order * a.pitch + at.c0);
    Map<T, V> m = Map<T, V>::identity();
    if (wt == WARPS) {
      const Pair<S>* j = (const Pair<S>*)a.joined + ((int64_t)col * 32 + lane) * V;
      const int k1 = (int)((int64_t)block * (warp + 1) / WARPS);
#pragma unroll 4
      for (int k = (int)((int64_t)block * warp / WARPS); k < k1; ++k)
        m.then(Map<T, V>::take(j + k * a.pitch));
    }
    steps.rows.start();
    m.put(&part[warp][lane * V]);
    own.put(&chunk[warp][lane * V]);
    __syncthreads();
    if (wt == WARPS && block > 0) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s = Map<T, V>::take(&part[w][lane * V]).at(s);
    }
    for (int w = 0; w < tw; ++w) s = Map<T, V>::take(&chunk[team * wt + w][lane * V]).at(s);
    bool all = true;
#pragma unroll
    for (int i = 0; i < V; ++i) all &= finite(s.get(i));
    if (at.live && !all) {
      walk<T, V, SIG, BWD>(p, a, col, at.order, s);
      return;
    }
  } else {
    steps.rows.start();
  }
  if (at.live) steps.take(p, a, at, s);
}

// ---- host side ---------------------------------------------------------------------

// Whether every row can be read and written `bytes` at a time
bool aligned(const ScanArgs& p, int elem, int bytes, bool backward, bool need_x) {
  struct A {
    const void* ptr;
    int64_t d, t, b;
  };
  A arrays[6] = {{p.gate, p.gd, p.gt, p.gb}, {p.h, p.hd, p.ht, p.hb}};
  int n = 2;
  if (need_x) arrays[n++] = {p.x, p.xd, p.xt, p.xb};
  if (backward) {
    arrays[n++] = {p.dh, p.ed, p.et, p.eb};
    arrays[n++] = {p.dgate, p.pd, p.pt, p.pb};
    arrays[n++] = {p.dx, p.qd, p.qt, p.qb};
  }
  if (p.D * elem % bytes) return false;
  for (int i = 0; i < n; ++i)
    if (arrays[i].d != 1 || (uintptr_t)arrays[i].ptr % bytes || arrays[i].t * elem % bytes ||
        arrays[i].b * elem % bytes)
      return false;
  return true;
}

template <typename T, int V, bool SIG, bool BWD>
int launch_chunks(om_backend* be, const ScanArgs& p) {
  using S = typename Elem<T>::State;
  constexpr int WARPS = warps_of(sizeof(T) * V);
  ChunkArgs a{};
  a.groups = p.B * (p.D / V);
  const int64_t columns = (a.groups + 31) / 32;
  a.pitch = columns * 32 * V;
  a.narrow = a.groups * V < ((int64_t)1 << 32) && p.D < ((int64_t)1 << 32);
  // Four columns per SM run faster uncut, without the maps' second read (640
  // columns x 1024 steps bf16 with the backward pass: 305 us, cut 329; 512: cut
  // 252 us). Fewer are cut into as many chunks as one wave of the 16 warps that
  // an SM holds takes, whole blocks of them, of 16 steps at least (96 x 700: 50
  // us, in twice as many chunks 60). Narrow rows keep fewer bytes under way and
  // take twice the warps.
  const int64_t warps = (int64_t)be->num_sms * (V == 1 && sizeof(T) < 8 ? 32 : 16);
  int64_t chunks = 1;
  if (columns < 4 * be->num_sms) {
    chunks = warps / columns;
    if (chunks >= WARPS) chunks = chunks / WARPS * WARPS;
    else chunks = chunks >= 4 ? 4 : chunks >= 2 ? 2 : 1;
    chunks = std::max<int64_t>(1, std::min(chunks, p.T / 16));
  }
  a.steps = std::max<int64_t>(1, (p.T + chunks - 1) / chunks);
  if (chunks > 1) a.steps = (a.steps + 7) / 8 * 8;
  chunks = std::max<int64_t>(1, (p.T + a.steps - 1) / a.steps);
  a.warps_t = 1;
  while (a.warps_t < WARPS && a.warps_t < chunks) a.warps_t *= 2;
  const int64_t per = (columns + WARPS / a.warps_t - 1) / (WARPS / a.warps_t);
  const int64_t rows = (chunks + a.warps_t - 1) / a.warps_t, blocks = per * rows;
  if (blocks > 0x7fffffff || columns > 0x7fffff00)
    return set_error(OM_ERR_SHAPE, "gated_scan: too many channels and steps");
  a.columns = (int)columns;
  a.chunks = (int)chunks;
  Scratch ws;
  if (chunks > 1) {
    OM_TRY(ws.alloc(be, (size_t)(chunks + rows + 1) * a.pitch * sizeof(Pair<S>)));
    a.maps = ws.ptr;
    a.joined = (Pair<S>*)a.maps + chunks * a.pitch;
    a.start = (Pair<S>*)a.joined + rows * a.pitch;
    ProfScope prof(be, BWD ? "gated_scan_maps_backward" : "gated_scan_maps");
    map_kernel<T, V, SIG, BWD><<<(unsigned)blocks, WARPS * 32, 0, be->stream>>>(p, a);
    note_launch();
  }
  ProfScope prof(be, BWD ? "gated_scan_backward" : "gated_scan");
  step_kernel<T, V, SIG, BWD><<<(unsigned)blocks, WARPS * 32, 0, be->stream>>>(p, a);
  note_launch();
  return check_cuda(cudaGetLastError(), "gated_scan launch");
}

template <typename T, bool SIG, bool BWD>
int launch_scan(om_backend* be, const ScanArgs& p) {
  constexpr int V = 8 / sizeof(T);
  if constexpr (V > 1)
    if (aligned(p, sizeof(T), 8, BWD, SIG || !BWD)) return launch_chunks<T, V, SIG, BWD>(be, p);
  return launch_chunks<T, 1, SIG, BWD>(be, p);
}

template <typename T>
int launch_scan_kind(om_backend* be, om_gate kind, const ScanArgs& p, bool backward) {
  if (kind == OM_GATE_SIGMOID)
    return backward ? launch_scan<T, true, true>(be, p) : launch_scan<T, true, false>(be, p);
  return backward ? launch_scan<T, false, true>(be, p) : launch_scan<T, false, false>(be, p);
}

int dispatch_scan(om_backend* be, om_gate kind, om_dtype dtype, const ScanArgs& p, bool backward) {
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "gated_scan: device");
  switch (dtype) {
    case OM_F32: return launch_scan_kind<float>(be, kind, p, backward);
    case OM_F64: return launch_scan_kind<double>(be, kind, p, backward);
    case OM_BF16: return launch_scan_kind<__nv_bfloat16>(be, kind, p, backward);
    case OM_F16: return launch_scan_kind<__half>(be, kind, p, backward);
    default: return set_error(OM_ERR_UNSUPPORTED, "gated_scan: dtype must be f32, f64, bf16 or f16");
  }
}

int check_scan(const char* who, om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape) {
  const std::string w(who);
  if (!be || !shape) return set_error(OM_ERR_INVALID, w + ": null argument");
  if (kind != OM_GATE_LINEAR && kind != OM_GATE_SIGMOID)
    return set_error(OM_ERR_INVALID, w + ": unknown gate kind");
  if (dtype != OM_F32 && dtype != OM_F64 && !is_half(dtype))
    return set_error(OM_ERR_UNSUPPORTED, w + ": dtype must be f32, f64, bf16 or f16");
  for (int k = 0; k < 3; ++k)
    if (shape[k] < 0) return set_error(OM_ERR_SHAPE, w + ": negative extent");
  return OM_OK;
}

}  // namespace
}  // namespace om

using namespace om;

extern "C" int om_b200_gated_scan(om_backend* be, om_gate kind, om_dtype dtype,
                                  const int64_t* shape, const void* gate,
                                  const int64_t* strides_gate, const void* x,
                                  const int64_t* strides_x, const void* h0, const int32_t* lengths,
                                  void* h, const int64_t* strides_h, void* h_last) {
  OM_TRY(check_scan("om_b200_gated_scan", be, kind, dtype, shape));
  const bool steps = shape[0] && shape[1] && shape[2];
  if (steps && (!gate || !x || !h || !strides_gate || !strides_x || !strides_h))
    return set_error(OM_ERR_INVALID, "om_b200_gated_scan: null argument");
  if (shape[0] == 0 || shape[2] == 0) return OM_OK;
  ScanArgs p{};
  p.D = shape[0], p.T = shape[1], p.B = shape[2];
  if (steps) {
    p.gate = gate, p.gd = strides_gate[0], p.gt = strides_gate[1], p.gb = strides_gate[2];
    p.x = x, p.xd = strides_x[0], p.xt = strides_x[1], p.xb = strides_x[2];
    p.h = h, p.hd = strides_h[0], p.ht = strides_h[1], p.hb = strides_h[2];
  }
  p.h0 = h0, p.lengths = lengths, p.h_last = h_last;
  return dispatch_scan(be, kind, dtype, p, false);
}

extern "C" int om_b200_gated_scan_backward(
    om_backend* be, om_gate kind, om_dtype dtype, const int64_t* shape, const void* gate,
    const int64_t* strides_gate, const void* x, const int64_t* strides_x, const void* h,
    const int64_t* strides_h, const void* h0, const int32_t* lengths, const void* dh,
    const int64_t* strides_dh, const void* dh_last, void* dgate, const int64_t* strides_dgate,
    void* dx, const int64_t* strides_dx, void* dh0) {
  OM_TRY(check_scan("om_b200_gated_scan_backward", be, kind, dtype, shape));
  const bool steps = shape[0] && shape[1] && shape[2];
  const bool need_x = kind == OM_GATE_SIGMOID;
  if (steps && (!gate || !h || !dh || !dgate || !dx || !strides_gate || !strides_h || !strides_dh ||
                !strides_dgate || !strides_dx || (need_x && (!x || !strides_x))))
    return set_error(OM_ERR_INVALID, "om_b200_gated_scan_backward: null argument");
  if (shape[0] == 0 || shape[2] == 0) return OM_OK;
  ScanArgs p{};
  p.D = shape[0], p.T = shape[1], p.B = shape[2];
  if (steps) {
    p.gate = gate, p.gd = strides_gate[0], p.gt = strides_gate[1], p.gb = strides_gate[2];
    if (need_x) p.x = x, p.xd = strides_x[0], p.xt = strides_x[1], p.xb = strides_x[2];
    p.h = (void*)h, p.hd = strides_h[0], p.ht = strides_h[1], p.hb = strides_h[2];
    p.dh = dh, p.ed = strides_dh[0], p.et = strides_dh[1], p.eb = strides_dh[2];
    p.dgate = dgate, p.pd = strides_dgate[0], p.pt = strides_dgate[1], p.pb = strides_dgate[2];
    p.dx = dx, p.qd = strides_dx[0], p.qt = strides_dx[1], p.qb = strides_dx[2];
  }
  p.h0 = h0, p.lengths = lengths, p.dh_last = dh_last, p.dh0 = dh0;
  return dispatch_scan(be, kind, dtype, p, true);
}
