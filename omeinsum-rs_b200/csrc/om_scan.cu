// Gated linear recurrence h_t = a_t h_{t-1} + b_t and its backward pass
//     S_t = a_t (dh_t + S_{t+1}),   G_t = dh_t + S_{t+1},
// in one pass over the data: each element is read once and written once.
//
// A step is the map s -> P s + Q with (P, Q) = (a, b) (backward: (a, a dh)), and
// maps compose, so time can be cut. A tile is 256 bytes of channels (32 lanes
// of 8 bytes) by up to 128 steps, eight warps of 16 (backward: 8) each; it is copied to
// shared memory asynchronously and lives there until its results have taken
// its place. Each warp first composes its 16 steps (from shared memory), the
// block its eight warps, and, where a sequence has more than one tile, tiles
// find the state that enters them by looking back: 32 consecutive tiles of one
// column form a group; a tile composes the maps of its predecessors in the
// group with the state that left the group before, and the group's last tile
// passes the state on. So the serial chain has one link per 4096 (2048) steps, and
// every sum is formed in one order whatever the timing. Tiles are handed out by
// a counter, first tiles first, so whatever a tile waits for has started.
//
// Bound by HBM: 3 arrays (forward) or 5 to 6 (backward) per element; the two
// passes over shared memory cost instructions, not traffic, and leave six
// tiles (32 KiB each) per SM in flight, which hides the look-back.
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

constexpr int ROW = 256;       // bytes of channels in a tile
constexpr int WARPS = 8;       // of a block
constexpr int MAX_STEPS = 16;  // of a warp
constexpr int GROUP = 32;      // tiles that look back at one another
constexpr uint32_t POLL_LIMIT = 1u << 22;

struct TileArgs {
  int64_t channels;  // B * D
  int grain;         // bytes of a row that one copy moves
  int warps_t;       // warps along time; the block has 8 / warps_t columns
  int steps;         // of a warp
  int rows;          // steps of a tile
  int narrow;        // channel numbers fit 32 bits
  int columns;       // of 256 bytes
  int tiles;         // along time
  // looking back; null when a sequence is one tile
  uint32_t* ticket;
  uint32_t* flags;   // [tile][column]: warps that have put their part of the map into `maps`
  uint64_t* state;   // [group][channel of all columns][words]: 32 bits of the state and a set mark
  void* maps;        // [tile][channel of all columns] pairs (P, Q)
  uint32_t* err;
};

// ---- arithmetic on the channels of a lane ------------------------------------------
// Two f32 channels share one instruction (the f32x2 forms of sm_100); an f64
// channel stands alone.

template <typename S>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int N = 2;
  float2 v;
  __device__ __forceinline__ float get(int i) const { return i ? v.y : v.x; }
  __device__ __forceinline__ void set(int i, float s) { (i ? v.y : v.x) = s; }
};
template <>
struct Pack<double> {
  static constexpr int N = 1;
  double v;
  __device__ __forceinline__ double get(int) const { return v; }
  __device__ __forceinline__ void set(int, double s) { v = s; }
};

__device__ __forceinline__ uint64_t bits_of(float2 v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
  return r;
}
__device__ __forceinline__ Pack<float> of_bits(uint64_t r) {
  Pack<float> p;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(p.v.x), "=f"(p.v.y) : "l"(r));
  return p;
}
__device__ __forceinline__ Pack<float> fill(float s) { return Pack<float>{make_float2(s, s)}; }
__device__ __forceinline__ Pack<double> fill(double s) { return Pack<double>{s}; }
__device__ __forceinline__ Pack<float> operator*(Pack<float> a, Pack<float> b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a.v)), "l"(bits_of(b.v)));
  return of_bits(r);
}
__device__ __forceinline__ Pack<float> operator+(Pack<float> a, Pack<float> b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a.v)), "l"(bits_of(b.v)));
  return of_bits(r);
}
__device__ __forceinline__ Pack<float> mad(Pack<float> a, Pack<float> b, Pack<float> c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(bits_of(a.v)), "l"(bits_of(b.v)), "l"(bits_of(c.v)));
  return of_bits(r);
}
__device__ __forceinline__ Pack<double> operator*(Pack<double> a, Pack<double> b) {
  return Pack<double>{a.v * b.v};
}
__device__ __forceinline__ Pack<double> operator+(Pack<double> a, Pack<double> b) {
  return Pack<double>{a.v + b.v};
}
__device__ __forceinline__ Pack<double> mad(Pack<double> a, Pack<double> b, Pack<double> c) {
  return Pack<double>{fma(a.v, b.v, c.v)};
}

// a = sigmoid(g) and 1 - a without cancellation. f32: an exponential formed as
// a power of two and an approximate reciprocal, together below 24 half steps
// for |g| <= 16 (most of it the rounding of the exponent); values below f32's
// normal numbers become zero.
__device__ __forceinline__ void sigmoid_pair(Pack<float> g, Pack<float>* a, Pack<float>* keep) {
  const Pack<float> t = g * fill(-1.4426950408889634f);
  Pack<float> e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.v.x) : "f"(t.v.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.v.y) : "f"(t.v.y));
  const Pack<float> d = e + fill(1.f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v.x) : "f"(d.v.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v.y) : "f"(d.v.y));
  const Pack<float> small = e * r, large = mad(r, fill(-1.f), fill(1.f));
  keep->v.x = e.v.x > 1.f ? large.v.x : small.v.x;  // e may be infinite, r is then 0
  keep->v.y = e.v.y > 1.f ? large.v.y : small.v.y;
  *a = r;
}
__device__ __forceinline__ void sigmoid_pair(Pack<double> g, Pack<double>* a, Pack<double>* keep) {
  const double e = exp(-fabs(g.v)), r = 1 / (1 + e);
  a->v = g.v >= 0 ? r : e * r;
  keep->v = g.v >= 0 ? e * r : r;
  if (g.v != g.v) a->v = keep->v = g.v;
}

// 8 bytes of a row as packs, and back
template <typename T>
struct Lane {
  static constexpr int CHANNELS = 8 / sizeof(T);
  using P = Pack<typename Elem<T>::State>;
  static constexpr int PACKS = CHANNELS / P::N;
  P v[PACKS];
};
__device__ __forceinline__ void unpack(uint2 u, Lane<__nv_bfloat16>& l) {
  l.v[0].v = make_float2(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u));
  l.v[1].v = make_float2(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void unpack(uint2 u, Lane<__half>& l) {
  l.v[0].v = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  l.v[1].v = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
}
__device__ __forceinline__ void unpack(uint2 u, Lane<float>& l) {
  l.v[0].v = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
}
__device__ __forceinline__ void unpack(uint2 u, Lane<double>& l) {
  l.v[0].v = __hiloint2double((int)u.y, (int)u.x);
}
__device__ __forceinline__ uint2 repack(const Lane<__nv_bfloat16>& l) {
  return make_uint2(pack2(l.v[0].v.x, l.v[0].v.y, __nv_bfloat16()),
                    pack2(l.v[1].v.x, l.v[1].v.y, __nv_bfloat16()));
}
__device__ __forceinline__ uint2 repack(const Lane<__half>& l) {
  return make_uint2(pack2(l.v[0].v.x, l.v[0].v.y, __half()), pack2(l.v[1].v.x, l.v[1].v.y, __half()));
}
__device__ __forceinline__ uint2 repack(const Lane<float>& l) {
  return make_uint2(__float_as_uint(l.v[0].v.x), __float_as_uint(l.v[0].v.y));
}
__device__ __forceinline__ uint2 repack(const Lane<double>& l) {
  return make_uint2((uint32_t)__double2loint(l.v[0].v), (uint32_t)__double2hiint(l.v[0].v));
}
template <typename T>
__device__ __forceinline__ Lane<T> lane_load(const char* row, int lane) {
  Lane<T> r;
  unpack(*reinterpret_cast<const uint2*>(row + lane * 8), r);
  return r;
}
template <typename T>
__device__ __forceinline__ void lane_store(char* row, int lane, const Lane<T>& r) {
  *reinterpret_cast<uint2*>(row + lane * 8) = repack(r);
}

// ---- data of a tile --------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_at(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(shared_at(dst)), "l"(src), "n"(N)
               : "memory");
}
__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_at(dst)), "l"(src)
               : "memory");
}

// One array's view: byte strides
struct View {
  const char* ptr;
  int64_t d, t, b;
};

// Where piece p (of `grain` bytes) of a row of column `col` lies
struct Piece {
  int64_t b, d;
  bool in;
};
__device__ __forceinline__ Piece piece_at(const TileArgs& a, int64_t D, int elem, int col, int p) {
  const int64_t c = ((int64_t)col * (ROW / a.grain) + p) * (a.grain / elem);
  Piece r;
  r.in = c < a.channels;
  r.b = a.narrow ? (int64_t)((uint32_t)c / (uint32_t)D) : c / D;
  r.d = c - r.b * D;
  return r;
}

// f(shared place, global place) for rows r0, r0 + step, ... < r1 of a piece
template <typename F>
__device__ __forceinline__ void each_row(const View& v, const Piece& at, char* to, int64_t t0,
                                         int r0, int r1, int step, F f) {
  const char* g = v.ptr + at.b * v.b + at.d * v.d + (t0 + r0) * v.t;
  char* s = to + r0 * ROW;
  const int64_t skip = step * v.t;
#pragma unroll 4
  for (int r = r0; r < r1; r += step, g += skip, s += step * ROW) f(s, g);
}

// Rows [r0, r1) of a tile, the pieces of a row shared out over `tn` threads.
// `once`: this thread's only piece, where a row has at most 32 of them.
template <typename F>
__device__ __forceinline__ void each_piece(const TileArgs& a, int64_t D, int elem, const View& v,
                                           const Piece& once, char* tile, int col, int64_t t0,
                                           int r0, int r1, int tt, int tn, F f) {
  const int per_row = ROW / a.grain;
  if (per_row <= 32) {
    const int p = tt & (per_row - 1);
    if (once.in) each_row(v, once, tile + p * a.grain, t0, r0 + tt / per_row, r1, tn / per_row, f);
    return;
  }
  const int lanes = min(per_row, tn);
  for (int p = tt % lanes; p < per_row; p += lanes) {
    const Piece at = piece_at(a, D, elem, col, p);
    if (!at.in) break;
    each_row(v, at, tile + p * a.grain, t0, r0 + tt / lanes, r1, tn / lanes, f);
  }
}

__device__ __forceinline__ void load_rows(const TileArgs& a, int64_t D, int elem, const View& v,
                                          const Piece& once, char* tile, int col, int64_t t0,
                                          int r0, int r1, int tt, int tn) {
  if (a.grain == 16)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, tt, tn,
               [](char* s, const char* g) { copy_async16(s, g); });
  else if (a.grain == 8)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, tt, tn,
               [](char* s, const char* g) { copy_async<8>(s, g); });
  else if (a.grain == 4)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, tt, tn,
               [](char* s, const char* g) { copy_async<4>(s, g); });
  else
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, tt, tn,
               [](char* s, const char* g) { *(uint16_t*)s = *(const uint16_t*)g; });
}

__device__ __forceinline__ void store_rows_of(const TileArgs& a, int64_t D, int elem, const View& v,
                                              const Piece& once, char* tile, int col, int64_t t0,
                                              int r0, int r1, int lane) {
  if (a.grain == 16)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, lane, 32,
               [](char* s, const char* g) { *(uint4*)g = *(const uint4*)s; });
  else if (a.grain == 8)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, lane, 32,
               [](char* s, const char* g) { *(uint2*)g = *(const uint2*)s; });
  else if (a.grain == 4)
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, lane, 32,
               [](char* s, const char* g) { *(uint32_t*)g = *(const uint32_t*)s; });
  else
    each_piece(a, D, elem, v, once, tile, col, t0, r0, r1, lane, 32,
               [](char* s, const char* g) { *(uint16_t*)g = *(const uint16_t*)s; });
}

// ---- looking back ------------------------------------------------------------------

__device__ __forceinline__ uint32_t load_flag(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t load_word(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(uint64_t* p, uint64_t v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

// Polls until `ready`; gives up when the limit or another block's error says so
template <typename F>
__device__ __forceinline__ void poll(uint32_t* err, F ready) {
  for (uint32_t i = 0; i < POLL_LIMIT; ++i) {
    if (ready()) return;
    if ((i & 255) == 255 && load_flag(err)) return;
  }
  atomicOr(err, 1u);
}

template <typename S>
struct alignas(2 * sizeof(S)) Pair {
  S p, q;
};
__device__ __forceinline__ Pair<float> load_pair(const Pair<float>* m) {
  const float2 v = __ldcg(reinterpret_cast<const float2*>(m));
  return Pair<float>{v.x, v.y};
}
__device__ __forceinline__ Pair<double> load_pair(const Pair<double>* m) {
  const double2 v = __ldcg(reinterpret_cast<const double2*>(m));
  return Pair<double>{v.x, v.y};
}

// The state that entered from the group before, one word per 32 bits
template <typename S>
__device__ __forceinline__ S read_state(const uint64_t* w, uint32_t* err) {
  constexpr int NW = sizeof(S) / 4;
  uint64_t v[NW];
  poll(err, [&] {
    bool all = true;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      v[i] = load_word(w + i);
      all = all && (v[i] >> 32);
    }
    return all;
  });
  uint32_t bits[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) bits[i] = (uint32_t)v[i];
  S s;
  memcpy(&s, bits, sizeof(S));
  return s;
}
template <typename S>
__device__ __forceinline__ void write_state(uint64_t* w, S s) {
  constexpr int NW = sizeof(S) / 4;
  uint32_t bits[NW];
  memcpy(bits, &s, sizeof(S));
#pragma unroll
  for (int i = 0; i < NW; ++i) store_word(w + i, (1ull << 32) | bits[i]);
}

// ---- the kernel --------------------------------------------------------------------

template <typename T, bool SIG, bool BWD>
__global__ void __launch_bounds__(WARPS * 32) scan_kernel(const __grid_constant__ ScanArgs p,
                                                          const __grid_constant__ TileArgs a) {
  using S = typename Elem<T>::State;
  using L = Lane<T>;
  using K = Pack<S>;
  constexpr int N = L::CHANNELS, NP = L::PACKS, W = K::N;
  constexpr int ARRAYS = BWD ? (SIG ? 4 : 3) : 2;  // gate, x or dh, h, x
  constexpr int E = sizeof(T);
  extern __shared__ __align__(16) char smem[];
  constexpr int C = 32 * N;                    // channels of a column
  constexpr int SLICES = WARPS * 32 / C;       // threads per channel
  __shared__ __align__(16) S part_p[WARPS][C];
  __shared__ __align__(16) S part_q[WARPS][C];
  __shared__ Pair<S> back[SLICES][C];
  __shared__ uint32_t ticket;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wt = a.warps_t, team = warp / wt, tw = warp % wt;  // teams of warps per column
  // (tile along time, column); backward starts at the end of time
  int tile = 0, col;
  if (a.ticket) {
    if (threadIdx.x == 0) ticket = atomicAdd(a.ticket, 1u);
    __syncthreads();
    tile = (int)(ticket / (uint32_t)a.columns);
    col = (int)(ticket - (uint32_t)tile * (uint32_t)a.columns);
  } else {
    col = (int)blockIdx.x * (WARPS / wt) + team;
  }
  const int order = tile;  // place in the chain
  if (BWD) tile = a.tiles - 1 - tile;
  const bool live = col < a.columns;
  const int64_t t0 = (int64_t)tile * a.rows;
  char* gate = smem + (size_t)team * ARRAYS * a.rows * ROW;
  char* second = gate + a.rows * ROW;    // x, or dh
  char* before = second + a.rows * ROW;  // h, a step late (backward)
  char* xrow = before + a.rows * ROW;    // x (backward, sigmoid)

  const int have = (int)min((int64_t)a.rows, p.T - t0);  // steps of the tile that exist
  const Piece once = piece_at(a, p.D, E, col, lane & min(31, ROW / a.grain - 1));
  if (live) {
    const int tt = threadIdx.x - team * wt * 32, tn = wt * 32;
    load_rows(a, p.D, E, View{(const char*)p.gate, p.gd * E, p.gt * E, p.gb * E}, once, gate, col,
              t0, 0, have, tt, tn);
    if constexpr (!BWD) {
      load_rows(a, p.D, E, View{(const char*)p.x, p.xd * E, p.xt * E, p.xb * E}, once, second, col,
                t0, 0, have, tt, tn);
    } else {
      load_rows(a, p.D, E, View{(const char*)p.dh, p.ed * E, p.et * E, p.eb * E}, once, second, col,
                t0, 0, have, tt, tn);
      // step 0 has no h before it
      load_rows(a, p.D, E, View{(const char*)p.h - p.ht * E, p.hd * E, p.ht * E, p.hb * E}, once,
                before, col, t0, t0 == 0, have, tt, tn);
      if constexpr (SIG)
        load_rows(a, p.D, E, View{(const char*)p.x, p.xd * E, p.xt * E, p.xb * E}, once, xrow, col,
                  t0, 0, have, tt, tn);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");

  // this lane's channels and where their sequences end in the tile
  const int64_t c0 = ((int64_t)col * 32 + lane) * N;
  int end[N];
  bool full = true;  // every step of this warp's rows exists in every lane
  const int r0 = min(tw * a.steps, a.rows), r1 = min(r0 + a.steps, a.rows);
#pragma unroll
  for (int v = 0; v < N; ++v) {
    end[v] = 0;
    if (live && c0 + v < a.channels) {
      end[v] = have;
      if (p.lengths) {
        const int64_t n = p.lengths[a.narrow ? (int64_t)((uint32_t)(c0 + v) / (uint32_t)p.D) : (c0 + v) / p.D];
        end[v] = (int)max((int64_t)0, min(n - t0, (int64_t)have));
      }
    }
    full = full && end[v] >= r1;
  }
  full = __all_sync(0xffffffffu, full);

  // The state that enters the tile; the first group starts from the caller's.
  // It is read before this tile's map is published: the last tile, which may
  // overwrite it (h_last == h0), comes after every map of its group.
  const S* from = (const S*)(BWD ? p.dh_last : p.h0);
  K s[NP];
  S start = 0;
  if (!a.ticket) {
#pragma unroll
    for (int v = 0; v < N; ++v)
      s[v / W].set(v % W, from && live && c0 + v < a.channels ? from[c0 + v] : S(0));
  } else if (order < GROUP && from && threadIdx.x < C) {
    const int64_t c = (int64_t)col * C + threadIdx.x;
    if (c < a.channels) start = from[c];
  }

  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  if (wt > 1) {  // (all the warps of the block, where tiles look back)
    // the map of this warp's steps
    K P[NP], Q[NP];
#pragma unroll
    for (int v = 0; v < NP; ++v) P[v] = fill(S(1)), Q[v] = fill(S(0));
    auto compose = [&](int r, bool masked) {
      const L g = lane_load<T>(gate + r * ROW, lane), x = lane_load<T>(second + r * ROW, lane);
#pragma unroll
      for (int v = 0; v < NP; ++v) {
        K f = g.v[v], b = x.v[v];
        if constexpr (SIG) {
          K keep;
          sigmoid_pair(f, &f, &keep);
          if constexpr (!BWD) b = b * keep;
        }
        const K q = BWD ? f * (b + Q[v]) : mad(f, Q[v], b), pp = f * P[v];
        if (masked) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (r < end[v * W + w]) {
              Q[v].set(w, q.get(w));
              P[v].set(w, pp.get(w));
            }
        } else {
          Q[v] = q;
          P[v] = pp;
        }
      }
    };
    if (full) {
#pragma unroll 4
      for (int i = 0; i < r1 - r0; ++i) compose(BWD ? r1 - 1 - i : r0 + i, false);
    } else {
      for (int i = 0; i < r1 - r0; ++i) compose(BWD ? r1 - 1 - i : r0 + i, true);
    }
#pragma unroll
    for (int v = 0; v < NP; ++v) {
      *reinterpret_cast<K*>(&part_p[warp][lane * N + v * W]) = P[v];
      *reinterpret_cast<K*>(&part_q[warp][lane * N + v * W]) = Q[v];
    }
    __syncthreads();
    // From here a thread has one channel. Those of the first slice replace each
    // warp's map by that of the steps before it (which run forward from the
    // first warp, backward from the last) and keep the whole tile's.
    const int ch = threadIdx.x % C, slice = threadIdx.x / C;
    S TP = 1, TQ = 0;
    if (slice < WARPS / wt) {
      for (int i = 0; i < wt; ++i) {
        const int w = slice * wt + (BWD ? wt - 1 - i : i);
        const S mp = part_p[w][ch], mq = part_q[w][ch];
        part_p[w][ch] = TP;
        part_q[w][ch] = TQ;
        TQ = mp * TQ + mq;
        TP = mp * TP;
      }
    }
    if (a.ticket) {
      Pair<S>* maps = (Pair<S>*)a.maps + (int64_t)col * C + ch;
      const int group = order / GROUP, in_group = order % GROUP;
      const int64_t pitch = (int64_t)a.columns * C;
      if (slice == 0 && in_group < GROUP - 1 && order < a.tiles - 1) {
        maps[(int64_t)order * pitch] = Pair<S>{TP, TQ};
        __threadfence();
        // one mark per warp that wrote a part of the map
        __syncwarp();
        if (lane == 0)
          asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(
                           a.flags + (int64_t)order * a.columns + col)
                       : "memory");
      }
      // predecessors in the group, shared out over the slices
      const int i0 = slice * (GROUP / SLICES), i1 = min(i0 + GROUP / SLICES, in_group);
      S LP = 1, LQ = 0;
      if (i0 < i1) {
        if (lane < i1 - i0) {
          const uint32_t* f = a.flags + (int64_t)(group * GROUP + i0 + lane) * a.columns + col;
          poll(a.err, [&] { return load_flag(f) == C / 32; });
        }
        __syncwarp();
        const Pair<S>* m = maps + (int64_t)(group * GROUP) * pitch;
#pragma unroll 8
        for (int i = i0; i < i1; ++i) {
          const Pair<S> w = load_pair(m + i * pitch);
          LQ = w.p * LQ + w.q;
          LP = w.p * LP;
        }
      }
      back[slice][ch] = Pair<S>{LP, LQ};
      __syncthreads();
      if (slice == 0) {
        constexpr int NW = sizeof(S) / 4;
        const int64_t c = (int64_t)col * C + ch;
        uint64_t* w = a.state + ((int64_t)group * pitch + c) * NW;
        S in = group > 0 ? read_state<S>(w - pitch * NW, a.err) : start;
#pragma unroll
        for (int i = 0; i < SLICES; ++i) in = back[i][ch].p * in + back[i][ch].q;
        if (in_group == GROUP - 1 && order < a.tiles - 1) write_state<S>(w, TP * in + TQ);
        back[0][ch].p = in;
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < N; ++v) s[v / W].set(v % W, back[0][lane * N + v].p);
    } else {
      __syncthreads();
    }
#pragma unroll
    for (int v = 0; v < NP; ++v)
      s[v] = mad(*reinterpret_cast<const K*>(&part_p[warp][lane * N + v * W]), s[v],
                 *reinterpret_cast<const K*>(&part_q[warp][lane * N + v * W]));
  }
  if (!live) return;

  // the steps themselves; results take the place of what they came from
  auto step = [&](int r, bool masked) {
    const L g = lane_load<T>(gate + r * ROW, lane), x = lane_load<T>(second + r * ROW, lane);
    auto settle = [&](int v, K next, K& out) {  // behind the end: the state stays, results are 0
      if (!masked) {
        s[v] = next;
        return;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (r < end[v * W + w]) s[v].set(w, next.get(w));
        else out.set(w, S(0));
      }
    };
    if constexpr (!BWD) {
      L out;
#pragma unroll
      for (int v = 0; v < NP; ++v) {
        K f = g.v[v], b = x.v[v];
        if constexpr (SIG) {
          K keep;
          sigmoid_pair(f, &f, &keep);
          b = b * keep;
        }
        out.v[v] = mad(f, s[v], b);
        settle(v, out.v[v], out.v[v]);
      }
      lane_store<T>(second + r * ROW, lane, out);
    } else {
      L was = lane_load<T>(before + r * ROW, lane), xv{}, dg, dx;
      if constexpr (SIG) xv = lane_load<T>(xrow + r * ROW, lane);
      if (t0 + r == 0) {
#pragma unroll
        for (int v = 0; v < N; ++v)
          was.v[v / W].set(v % W, p.h0 && c0 + v < a.channels ? ((const S*)p.h0)[c0 + v] : S(0));
      }
#pragma unroll
      for (int v = 0; v < NP; ++v) {
        K f = g.v[v];
        const K total = x.v[v] + s[v];
        if constexpr (SIG) {
          K keep;
          sigmoid_pair(f, &f, &keep);
          dx.v[v] = total * keep;
          dg.v[v] = mad(xv.v[v], fill(S(-1)), was.v[v]) * f * dx.v[v];
        } else {
          dx.v[v] = total;
          dg.v[v] = total * was.v[v];
        }
        const K next = f * total;
        settle(v, next, dx.v[v]);
        if (masked) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (r >= end[v * W + w]) dg.v[v].set(w, S(0));
        }
      }
      lane_store<T>(gate + r * ROW, lane, dg);
      lane_store<T>(second + r * ROW, lane, dx);
    }
  };
  if (full) {
#pragma unroll 4
    for (int i = 0; i < r1 - r0; ++i) step(BWD ? r1 - 1 - i : r0 + i, false);
  } else {
    for (int i = 0; i < r1 - r0; ++i) step(BWD ? r1 - 1 - i : r0 + i, true);
  }
  __syncwarp();
  if (r0 < r1) {
    const int stop = min(r1, have);
    if constexpr (!BWD) {
      store_rows_of(a, p.D, E, View{(const char*)p.h, p.hd * E, p.ht * E, p.hb * E}, once, second,
                    col, t0, r0, stop, lane);
    } else {
      store_rows_of(a, p.D, E, View{(const char*)p.dgate, p.pd * E, p.pt * E, p.pb * E}, once, gate,
                    col, t0, r0, stop, lane);
      store_rows_of(a, p.D, E, View{(const char*)p.dx, p.qd * E, p.qt * E, p.qb * E}, once, second,
                    col, t0, r0, stop, lane);
    }
  }
  // the state that leaves the last tile
  S* last = (S*)(BWD ? p.dh0 : p.h_last);
  if (last && order == a.tiles - 1 && tw == (BWD ? 0 : wt - 1)) {
#pragma unroll
    for (int v = 0; v < N; ++v)
      if (c0 + v < a.channels) last[c0 + v] = s[v / W].get(v % W);
  }
}

// ---- host side ---------------------------------------------------------------------

// The bytes that one copy may move: the widest of 16, 8, 4 (2 for 16-bit
// types) that divides the rows and every address and stride
int grain_of(const ScanArgs& p, int elem, bool backward, bool need_x) {
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
  for (int g = 16; g > elem; g /= 2) {
    bool fits = p.D * elem % g == 0;
    for (int i = 0; i < n && fits; ++i)
      fits = (arrays[i].d == 1 || p.D == 1) && (uintptr_t)arrays[i].ptr % g == 0 &&
             arrays[i].t * elem % g == 0 && arrays[i].b * elem % g == 0;
    if (fits) return g;
  }
  return elem;
}

template <typename T, bool SIG, bool BWD>
int launch_scan(om_backend* be, const ScanArgs& p) {
  using S = typename Elem<T>::State;
  constexpr int ARRAYS = BWD ? (SIG ? 4 : 3) : 2;
  TileArgs a{};
  a.channels = p.D * p.B;
  a.grain = grain_of(p, sizeof(T), BWD, SIG || !BWD);
  const int64_t columns = (a.channels * (int64_t)sizeof(T) + ROW - 1) / ROW;
  a.narrow = a.channels < ((int64_t)1 << 32) && p.D < ((int64_t)1 << 32);
  // Up to 16 steps are one warp's work and eight columns share a block; longer
  // sequences take all eight warps, the backward pass with half the steps
  // each: its three or four arrays then leave three blocks on an SM.
  a.warps_t = p.T > MAX_STEPS ? WARPS : 1;
  a.steps = a.warps_t > 1 && BWD ? MAX_STEPS / 2 : MAX_STEPS;
  a.rows = (int)std::min<int64_t>(p.T, a.steps * a.warps_t);
  const int64_t tiles = p.T == 0 ? 1 : (p.T + a.rows - 1) / a.rows;
  const int64_t blocks = tiles > 1 ? tiles * columns : (columns + WARPS / a.warps_t - 1) / (WARPS / a.warps_t);
  if (blocks > 0x7fffffff || columns > 0x7ffffff0)
    return set_error(OM_ERR_SHAPE, "gated_scan: too many channels and steps");
  a.columns = (int)columns;
  a.tiles = (int)tiles;
  a.err = be->d_flags + 1;
  Scratch ws;
  if (tiles > 1) {
    const int64_t groups = (tiles + GROUP - 1) / GROUP;
    const size_t pitch = (size_t)columns * (ROW / sizeof(T));
    const size_t state = (size_t)groups * pitch * (sizeof(S) / 4) * 8;
    const size_t flags = ((size_t)blocks * 4 + 15) / 16 * 16;
    OM_TRY(ws.alloc(be, 16 + flags + state + (size_t)tiles * pitch * sizeof(Pair<S>)));
    char* at = (char*)ws.ptr;
    OM_CUDA(cudaMemsetAsync(at, 0, 16 + flags + state, be->stream), "gated_scan marks");
    a.ticket = (uint32_t*)at;
    a.flags = (uint32_t*)(at + 16);
    a.state = (uint64_t*)(at + 16 + flags);
    a.maps = at + 16 + flags + state;
  }
  const size_t smem = (size_t)(WARPS / a.warps_t) * ARRAYS * a.rows * ROW;
  auto kernel = scan_kernel<T, SIG, BWD>;
  if (smem > 40 * 1024)
    OM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
            "gated_scan");
  ProfScope prof(be, BWD ? "gated_scan_backward" : "gated_scan");
  kernel<<<(unsigned)blocks, WARPS * 32, smem, be->stream>>>(p, a);
  note_launch();
  return check_cuda(cudaGetLastError(), "gated_scan launch");
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
