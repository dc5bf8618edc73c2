// Softmax cross entropy of the logits z = x w^T over a vocabulary, and its
// gradients, without ever holding all logits:
//     lse_n = log sum_v exp(z_nv),  loss_n = lse_n - z_{n, target_n}
//     dz_nv = dloss_n (exp(z_nv - lse_n) - [v == target_n]),
//     dx = dz w,  dw = dz^T x.
// The forward keeps a maximum and a sum of exponentials per row and group of
// columns; the backward computes the logits a second time, a piece of the
// vocabulary at a time, writes dz of the piece once and multiplies it twice:
// 8 N D V operations, of which 6 are needed. Bound by the tensor cores, or,
// for few tokens, by reading w. Measured: 8192 x 4096 x 128000 bf16 with
// gradients 25.3 to 26.7 ms (34.4 TFLOP at 1.36 PFLOP/s, the card's power limit; writing
// the logits once and reading them three times would save 8.6 TFLOP and cost
// 4.2 GB held); 24 x 2048 x 32000 f16 forward 34 us, 20 of which w needs.
#include <algorithm>
#include <cfloat>

#include "om_convert.cuh"
#include "om_sm100.cuh"

namespace om {
namespace {

struct LossArgs {
  int64_t N, D, V;
  const void* x;
  int64_t xd, xn;
  const void* w;
  int64_t wd, wv;
  const void* targets;
  int target64;
};

__device__ __forceinline__ int64_t target_of(const void* t, int t64, int64_t n) {
  return t64 ? ((const int64_t*)t)[n] : (int64_t)((const int32_t*)t)[n];
}

// Which tokens carry no loss: those whose target lies outside the vocabulary. Their
// rows of dx are zero, and not 0 * w, which an infinite weight would make NaN.
// targets == null: all carry one.
struct Counted {
  const void* targets;
  int t64;
  int64_t vocab;
  __device__ __forceinline__ bool out(int64_t row) const {
    return targets && (uint64_t)target_of(targets, t64, row) >= (uint64_t)vocab;
  }
};

// a strided matrix as a row-major one, zero in rows whose target lies outside
// the vocabulary
template <typename S>
__global__ void masked_rows(const S* __restrict__ src, int64_t rows, int64_t cols, int64_t sr,
                            int64_t sc, S* __restrict__ dst, const void* targets, int t64,
                            int64_t vocab) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols, c = i - r * cols, t = target_of(targets, t64, r);
    dst[i] = t >= 0 && t < vocab ? src[r * sr + c * sc] : S(0);
  }
}

// a row-major matrix as a strided one
template <typename S>
__global__ void store_rows(const S* __restrict__ src, int64_t rows, int64_t cols, Counted counted,
                           S* __restrict__ dst, int64_t dr, int64_t dc) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols, c = i - r * cols;
    dst[r * dr + c * dc] = counted.out(r) ? S(0) : src[i];
  }
}

template <typename T>
__global__ void zero_rows(T* __restrict__ dst, int64_t rows, int64_t cols, int64_t dr, int64_t dc) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x)
    dst[i / cols * dr + i % cols * dc] = T(0.f);
}

template <typename S>
__global__ void add_into(S* __restrict__ acc, const S* __restrict__ v, int64_t n) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    acc[i] += v[i];
}

template <typename S>
__device__ __forceinline__ S lowest();
template <>
__device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ double lowest<double>() { return -INFINITY; }

// merges the sums (m, s) = (max, sum exp(. - max)) of two sets; a NaN maximum
// stays NaN, an empty set is (-inf, 0)
template <typename S>
__device__ __forceinline__ void merge(S& m, S& s, S m2, S s2) {
  const S top = m2 > m || m2 != m2 ? m2 : m;
  const S a = m == top ? s : s * exp(m - top);
  const S b = m2 == top ? s2 : s2 * exp(m2 - top);
  m = top;
  s = a + b;
}

// One block per row of a piece z [rows, cols]: maximum and sum of
// exponentials, merged into the row's running pair; the target's logit when
// it lies in the piece.  After the last piece the row's loss and lse.
template <typename S>
__global__ void piece_stats(const S* __restrict__ z, int64_t cols, int64_t v0, const void* targets,
                            int t64, int64_t vocab, S* run_m, S* run_s, S* hit, int first, int last,
                            S* loss, S* lse) {
  const int64_t row = blockIdx.x;
  const S* zr = z + row * cols;
  S m = lowest<S>(), s = 0;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) merge(m, s, zr[c], S(1));
  __shared__ S sm[32], ss[32];
  for (int o = 16; o; o >>= 1)
    merge(m, s, __shfl_down_sync(0xffffffffu, m, o), __shfl_down_sync(0xffffffffu, s, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m, ss[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) merge(m, s, sm[i], ss[i]);
  if (!first) {
    S pm = run_m[row], ps = run_s[row];
    merge(pm, ps, m, s);
    m = pm;
    s = ps;
  }
  run_m[row] = m;
  run_s[row] = s;
  const int64_t t = target_of(targets, t64, row);
  if (t >= v0 && t < v0 + cols) hit[row] = zr[t - v0];
  if (last) {
    const S total = m + log(s);
    lse[row] = total;
    loss[row] = t >= 0 && t < vocab ? total - hit[row] : S(0);
  }
}

// z becomes dz in place
template <typename S>
__global__ void piece_gradient(S* __restrict__ z, int64_t rows, int64_t cols, int64_t v0,
                               const void* targets, int t64, int64_t vocab,
                               const S* __restrict__ lse, const S* __restrict__ dloss) {
  const int64_t row = blockIdx.x;
  const int64_t t = target_of(targets, t64, row);
  const bool counts = t >= 0 && t < vocab;
  const S l = lse[row], g = counts ? dloss[row] : S(0);
  S* zr = z + row * cols;
  for (int64_t c = threadIdx.x; c < cols; c += blockDim.x)
    zr[c] = counts ? g * (exp(zr[c] - l) - (v0 + c == t ? S(1) : S(0))) : S(0);
}

Counted counted_of(const LossArgs& p) { return Counted{p.targets, p.target64, p.V}; }

unsigned flat_grid(om_backend* be, int64_t n) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, (int64_t)be->num_sms * 16));
}

template <typename S>
GemmArgs gemm(om_dtype dt, int64_t M, int64_t N, int64_t K, const void* a, int64_t am,
                 int64_t ak, const void* b, int64_t bk, int64_t bn, void* c, int64_t cm) {
  GemmArgs g{};
  g.alg = OM_STANDARD;
  g.dtype = dt;
  g.M = M, g.N = N, g.K = K, g.batch = 1;
  g.A = a, g.sam = am, g.sak = ak;
  g.B = b, g.sbk = bk, g.sbn = bn;
  g.C = c, g.scm = cm, g.scn = 1;
  return g;
}

// Vocabulary entries per piece: a piece's logits take at most 256 MiB, and the
// products' grids hold 65535 tiles of 64 columns
int64_t piece_size(int64_t N, int64_t V, size_t elem) {
  const int64_t fit = ((int64_t)256 << 20) / (int64_t)elem / std::max<int64_t>(N, 1) / 128 * 128;
  return std::min({V, std::max<int64_t>(128, fit), (int64_t)1 << 21});
}

// f64, and f32 in exact mode: pieces through the library's own products
template <typename S>
int loss_forward(om_backend* be, const LossArgs& p, S* loss, S* lse) {
  const om_dtype dt = sizeof(S) == 8 ? OM_F64 : OM_F32;
  const int64_t P = piece_size(p.N, p.V, sizeof(S));
  Scratch zs, stats;
  OM_TRY(zs.alloc(be, (size_t)p.N * P * sizeof(S)));
  OM_TRY(stats.alloc(be, (size_t)p.N * 3 * sizeof(S)));
  S* run = (S*)stats.ptr;
  for (int64_t v0 = 0; v0 < p.V; v0 += P) {
    const int64_t n = std::min(P, p.V - v0);
    const S* w = (const S*)p.w + v0 * p.wv;
    OM_TRY(launch_gemm(be, gemm<S>(dt, p.N, n, p.D, p.x, p.xn, p.xd, w, p.wd, p.wv, zs.ptr, n)));
    ProfScope prof(be, "loss_piece_stats");
    piece_stats<S><<<(unsigned)p.N, 256, 0, be->stream>>>(
        (const S*)zs.ptr, n, v0, p.targets, p.target64, p.V, run, run + p.N, run + 2 * p.N, v0 == 0,
        v0 + n == p.V, loss, lse);
    note_launch();
    OM_CUDA(cudaGetLastError(), "loss piece launch");
  }
  return OM_OK;
}

template <typename S>
int loss_backward(om_backend* be, const LossArgs& p, const S* lse, const S* dloss, S* dx,
                  int64_t dxd, int64_t dxn, S* dw, int64_t dwd, int64_t dwv) {
  const om_dtype dt = sizeof(S) == 8 ? OM_F64 : OM_F32;
  const int64_t P = piece_size(p.N, p.V, sizeof(S));
  const int64_t nx = p.N * p.D;
  if (p.N == 0) {  // no token: the weights' gradient is zero
    zero_rows<S><<<flat_grid(be, p.V * p.D), 256, 0, be->stream>>>(dw, p.V, p.D, dwv, dwd);
    note_launch();
    return check_cuda(cudaGetLastError(), "loss backward launch");
  }
  Scratch zs, xs, acc, part, dws;
  OM_TRY(zs.alloc(be, (size_t)p.N * P * sizeof(S)));
  OM_TRY(xs.alloc(be, (size_t)nx * sizeof(S)));
  OM_TRY(acc.alloc(be, (size_t)nx * sizeof(S)));
  if (P < p.V) OM_TRY(part.alloc(be, (size_t)nx * sizeof(S)));
  OM_TRY(dws.alloc(be, (size_t)P * p.D * sizeof(S)));
  // rows without a loss are zero here: whatever they hold reaches no gradient
  masked_rows<S><<<flat_grid(be, nx), 256, 0, be->stream>>>(
      (const S*)p.x, p.N, p.D, p.xn, p.xd, (S*)xs.ptr, p.targets, p.target64, p.V);
  note_launch();
  for (int64_t v0 = 0; v0 < p.V; v0 += P) {
    const int64_t n = std::min(P, p.V - v0);
    const S* w = (const S*)p.w + v0 * p.wv;
    OM_TRY(launch_gemm(be, gemm<S>(dt, p.N, n, p.D, xs.ptr, p.D, 1, w, p.wd, p.wv, zs.ptr, n)));
    piece_gradient<S><<<(unsigned)p.N, 256, 0, be->stream>>>((S*)zs.ptr, p.N, n, v0, p.targets,
                                                             p.target64, p.V, lse, dloss);
    note_launch();
    S* to = v0 ? (S*)part.ptr : (S*)acc.ptr;
    OM_TRY(launch_gemm(be, gemm<S>(dt, p.N, p.D, n, zs.ptr, n, 1, w, p.wv, p.wd, to, p.D)));
    if (v0) {
      add_into<S><<<flat_grid(be, nx), 256, 0, be->stream>>>((S*)acc.ptr, (const S*)part.ptr, nx);
      note_launch();
    }
    OM_TRY(launch_gemm(be, gemm<S>(dt, n, p.D, p.N, zs.ptr, 1, n, xs.ptr, p.D, 1, dws.ptr, p.D)));
    store_rows<S><<<flat_grid(be, n * p.D), 256, 0, be->stream>>>((const S*)dws.ptr, n, p.D, Counted{},
                                                                 dw + v0 * dwv, dwv, dwd);
    note_launch();
  }
  store_rows<S><<<flat_grid(be, nx), 256, 0, be->stream>>>((const S*)acc.ptr, p.N, p.D, counted_of(p), dx, dxn,
                                                            dxd);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss backward launch");
}

// ---- 16-bit types and f32 on the tensor cores ----------------------------------------

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What exponentials are taken relative to: the largest logit, kept finite. -inf
// then adds exp(-inf) = 0 where every logit so far is -inf (and not the NaN of
// -inf - -inf), an infinite maximum makes the sum infinite, NaN stays.
__device__ __forceinline__ float shift_of(float top) { return fminf(fmaxf(top, -FLT_MAX), FLT_MAX); }

// Maximum and sum of exponentials of a lane's columns of one row, and the
// target's logit.
struct StatsEpi {
  const void* targets;
  int t64;
  int64_t v0;    // vocabulary entry of column 0
  float2* part;  // [slot][rows]
  int64_t rows;
  float* hit;
  struct Row {
    float m, s;
    int64_t target;
  };
  int lent_bytes() const { return 0; }
  __device__ __forceinline__ Row begin(int m, bool in, int) const {
    return Row{-INFINITY, 0.f, in ? target_of(targets, t64, m) - v0 : -1};
  }
  __device__ __forceinline__ void columns(Row& row, int m, bool in, int n0, int N,
                                          const uint32_t (&r)[32], mma::Lent& lent) const {
    if (n0 >= N) return;
    const int n = N - n0;  // columns that exist
    float top = __uint_as_float(r[0]);
    if (n >= 32) {
#pragma unroll
      for (int c = 1; c < 32; ++c) top = fmaxf(top, __uint_as_float(r[c]));
    } else {
#pragma unroll
      for (int c = 1; c < 32; ++c)
        if (c < n) top = fmaxf(top, __uint_as_float(r[c]));
    }
    if (top > row.m) {
      row.s *= exp2_fast((row.m - top) * LOG2E);
      row.m = top;
    }
    const float base = shift_of(row.m);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (n >= 32) {
#pragma unroll
      for (int c = 0; c < 32; ++c) s[c & 3] += exp2_fast((__uint_as_float(r[c]) - base) * LOG2E);
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c < n) s[c & 3] += exp2_fast((__uint_as_float(r[c]) - base) * LOG2E);
    }
    row.s += (s[0] + s[1]) + (s[2] + s[3]);
    const int64_t at = row.target - n0;
    if (at >= 0 && at < 32 && at < n) {
      float z = 0.f;
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (at == c) z = __uint_as_float(r[c]);
      hit[m] = z;
    }
  }
  __device__ __forceinline__ void end(Row& row, int m, bool in, int slot) const {
    if (in) part[(int64_t)slot * rows + m] = make_float2(row.m, row.s);
  }
};

// Joins the slots of 8 rows per block, each of 32 threads of a row every 32nd
// slot; a row's threads are a stride of 8 apart, so that a slot's rows are read
// together. (32 rows by 8 threads left 4096 rows on 128 blocks of 50 dependent
// loads each: 36 us against 8.)
__global__ void __launch_bounds__(256) join_stats(const float2* __restrict__ part, int slots,
                                                  int64_t rows, const void* targets, int t64,
                                                  int64_t vocab, const float* hit, float* loss,
                                                  float* lse) {
  __shared__ float sm[32][9], ss[32][9];
  const int r = threadIdx.x & 7, k = threadIdx.x >> 3;
  const int64_t row = blockIdx.x * (int64_t)8 + r;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
    // eight slots at a time: one maximum, then their sums
    for (int i = k; i < slots; i += 256) {
      float2 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = i + 32 * u < slots ? part[(int64_t)(i + 32 * u) * rows + row] : make_float2(-INFINITY, 0.f);
      float top = v[0].x, sum = 0.f;
#pragma unroll
      for (int u = 1; u < 8; ++u) top = fmaxf(top, v[u].x);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        sum += v[u].y == 0.f ? 0.f : v[u].y * exp2_fast((v[u].x - shift_of(top)) * LOG2E);
      merge(m, s, top, sum);
    }
  }
  sm[k][r] = m;
  ss[k][r] = s;
  __syncthreads();
  // one warp per row now
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t mine = blockIdx.x * (int64_t)8 + w;
  m = sm[lane][w];
  s = ss[lane][w];
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  s = s == 0.f ? 0.f : s * exp2_fast((m - shift_of(top)) * LOG2E);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  m = top;
  if (lane || mine >= rows) return;
  const float total = m + logf(s);
  const int64_t t = target_of(targets, t64, mine);
  lse[mine] = total;
  loss[mine] = t >= 0 && t < vocab ? total - hit[mine] : 0.f;
}

// dz is rounded to 16 bits as dz / scale, scale = max |dloss| of the counted
// tokens over `top`, and the products' f32 sums are multiplied by it: where all
// tokens weigh the same, the one-hot part is a power of two and rounds to
// itself, while the rounding of dloss would be the same error in every term
// (measured on 4096 x 1024 x 50001: the gradients' error against 64 bits falls
// from 3.4e-3 to 1.7e-3, the f32 result's own rounding). top = 2^14 in f16 holds dz down to 2^-38 of the
// largest; bf16 needs no room and takes 1.
__global__ void gradient_scale(const float* __restrict__ dloss, const void* targets, int t64,
                               int64_t vocab, int64_t n, float top, float* scale) {
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t t = target_of(targets, t64, i);
    const float g = fabsf(dloss[i]);
    if (t >= 0 && t < vocab && g < INFINITY) m = fmaxf(m, g);  // one that is no number scales nothing
  }
  __shared__ float part[32];
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) m = fmaxf(m, part[i]);
  // a scale below f32's normal numbers would lose bits, none is needed at 0
  const float f = m / top;
  *scale = f >= FLT_MIN ? f : 1.f;
}

// 32 columns of a warp's rows, rounded to T, through TMA; m: this lane's row. A
// warp whose first row does not exist has none.
template <typename T>
__device__ __forceinline__ void store_half_box(mma::Lent& lent, const CUtensorMap* map,
                                               const float (&v)[32], int n0, int m, bool in) {
  if (!__shfl_sync(0xffffffffu, in, 0)) return;
  uint32_t u[16];
#pragma unroll
  for (int c = 0; c < 16; ++c) u[c] = pack2(v[2 * c], v[2 * c + 1], T());
  mma::store_box(lent, map, u, n0, m - (int)(threadIdx.x & 31));
}

// Whether 16-bit results go through store_box: sums of up to 8 slabs, whose tiles
// are bound by their stores (dw of 8 x 4096 x 128000 in bf16: 272 to 325 us, lanes
// storing their own rows 355 to 365). Longer ones hide their stores and need the stages that the boxes
// take (4096 x 1024 x 50001 with gradients: 1.4 % slower with boxes).
template <typename T>
int boxes(int64_t k, int vec) {
  return sizeof(T) == 2 && vec && k <= 512;
}

// The next of the three bf16 parts of an f32 number, as f32; what is left stays in
// v. x = x0 + x1 + x2 to 24 bits. x0 is cut at bf16's largest number, which f32's
// largest would round past. Infinity and NaN are the third part of 0, 0, x: in the
// products it meets the other operand's first part alone (A2 B0, A0 B2), where in
// the first it would meet zeros among the others' second and third parts.
__device__ __forceinline__ float next_part(float& v, bool third) {
  constexpr float LARGEST = 0x1.fep127f;
  const bool finite = fabsf(v) < INFINITY;
  if (third) return v;
  const float part = finite ? __bfloat162float(__float2bfloat16_rn(fminf(fmaxf(v, -LARGEST), LARGEST))) : 0.f;
  v -= part;
  return part;
}

// dz of a piece, rounded to T; the buffer's rows hold whole tiles. f32: as the
// three bf16 planes that the two products take.
template <typename T>
struct GradEpi {
  CUtensorMap map;  // of the piece of dz, where it is stored in boxes
  int boxed;
  const void* targets;
  int t64;
  int64_t vocab, v0;
  const float *lse, *dloss, *scale;
  void* dz;
  int64_t ld, plane;
  struct Row {
    float lse, g;
    int64_t target;  // within the piece
    bool counts;
  };
  int lent_bytes() const { return boxed ? 2 * mma::BOX_BYTES : 0; }
  __device__ __forceinline__ Row begin(int m, bool in, int) const {
    Row row{0.f, 0.f, -1, false};
    if (in) {
      const int64_t t = target_of(targets, t64, m);
      if (t >= 0 && t < vocab) {
        row.lse = lse[m];
        row.g = scale ? dloss[m] / *scale : dloss[m];
        row.target = t - v0;
        row.counts = true;
      }
    }
    return row;
  }
  __device__ __forceinline__ void columns(Row& row, int m, bool in, int n0, int N,
                                          const uint32_t (&r)[32], mma::Lent& lent) const {
    if (n0 >= N) return;
    float v[32];
#pragma unroll
    for (int c = 0; c < 32; ++c)
      v[c] = row.g * exp2_fast((__uint_as_float(r[c]) - row.lse) * LOG2E);
    const int64_t at = row.target - n0;
    if (at >= 0 && at < 32) {
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (at == c) v[c] = row.g * (exp2_fast((__uint_as_float(r[c]) - row.lse) * LOG2E) - 1.f);
    }
    if (!row.counts) {  // zero times an infinite weight made its logits NaN
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = 0.f;
    }
    if constexpr (sizeof(T) == 2) {
      if (boxed) store_half_box<T>(lent, &map, v, n0, m, in);
      else if (in) store_row((T*)dz + (int64_t)m * ld + n0, v, true);
    } else if (in) {
      __nv_bfloat16* to = (__nv_bfloat16*)dz + (int64_t)m * ld + n0;
#pragma unroll
      for (int z = 0; z < 3; ++z) {
        float part[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) part[c] = next_part(v[c], z == 2);
        store_row(to + z * plane, part, true);
      }
    }
  }
  __device__ __forceinline__ void end(Row&, int, bool, int) const {}
};

// Sums in f32 kept for later pieces or splits, or the finished result as T.
template <typename T>
struct OutEpi {
  CUtensorMap map;     // of `out`, where it is stored in boxes
  int boxed;
  T* out;
  int64_t dr, dc;
  int vec;             // row_stores of `out`
  const float* scale;  // null or gradient_scale's
  float* acc;          // [split][rows][acc_ld], whole tiles
  int64_t acc_ld, acc_split;
  int load, keep;      // add what acc holds; leave the sum there
  Counted counted;     // rows that are zero whatever their sums are (dx)
  struct Row {
    float f;
    float* acc;
    bool zero;
  };
  int lent_bytes() const {
    return keep ? 0 : !vec ? mma::TURN_BYTES : boxed ? 2 * mma::BOX_BYTES : 0;
  }
  __device__ __forceinline__ Row begin(int m, bool in, int split) const {
    return Row{scale ? *scale : 1.f,
               acc ? acc + (int64_t)split * acc_split + (int64_t)m * acc_ld : nullptr, in && counted.out(m)};
  }
  __device__ __forceinline__ void columns(Row& row, int m, bool in, int n0, int N,
                                          const uint32_t (&r)[32], mma::Lent& lent) const {
    if (n0 >= N) return;
    float v[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(r[c]);
    if (load && in) {
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 a = *reinterpret_cast<const float4*>(row.acc + n0 + c);
        v[c] += a.x, v[c + 1] += a.y, v[c + 2] += a.z, v[c + 3] += a.w;
      }
    }
    if (keep) {
      if (in) store_row(row.acc + n0, v, true);  // (whole tiles: 256-byte rows)
      return;
    }
#pragma unroll
    for (int c = 0; c < 32; ++c) v[c] *= row.f;
    if (row.zero) {
#pragma unroll
      for (int c = 0; c < 32; ++c) v[c] = 0.f;
    }
    const int lane = threadIdx.x & 31;
    if (!vec) {
      store_turned(lent.words, v, out + (int64_t)(m - lane) * dr + n0 * dc, dr, dc,
                   __popc(__ballot_sync(0xffffffffu, in)), N - n0);
    } else if (boxed) {
      if constexpr (sizeof(T) == 2) store_half_box<T>(lent, &map, v, n0, m, in);
    } else if (in) {
      T* to = out + (int64_t)m * dr;
      if (N - n0 >= 32) {
        store_row(to + n0, v, vec == 2);
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (n0 + c < N) to[n0 + c] = Elem<T>::store(v[c]);
      }
    }
  }
  __device__ __forceinline__ void end(Row&, int, bool, int) const {}
};

// out = scale * sum of the splits; bound by reading them
template <typename T>
__global__ void join_splits(const float* __restrict__ acc, int splits, int64_t acc_split,
                            int64_t acc_ld, int64_t rows, int64_t cols, const float* scale,
                            Counted counted, T* __restrict__ out, int64_t dr, int64_t dc) {
  const float f = scale ? *scale : 1.f;
  const int64_t total = rows * cols;
  const bool narrow = total < ((int64_t)1 << 32);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const RowItem at = row_item(i, cols, narrow);
    const int64_t r = at.row, c = at.item;
    const float* from = acc + r * acc_ld + c;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += __ldcg(from + k * acc_split);
    out[r * dr + c * dc] = Elem<T>::store(counted.out(r) ? 0.f : s * f);
  }
}

// A 16-bit matrix with rows at 16-byte aligned places, zero behind their end and
// where the target lies outside the vocabulary (targets given). A thread makes 8
// elements.
template <typename T>
__global__ void pack_rows(const T* __restrict__ src, int64_t rows, int64_t cols, int64_t sr,
                          int64_t sc, T* __restrict__ dst, int64_t ld, const void* targets, int t64,
                          int64_t vocab) {
  const int64_t per = ld / 8, total = rows * per;
  const bool narrow = total < ((int64_t)1 << 32);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const RowItem at = row_item(i, per, narrow);
    const int64_t c = at.item * 8;
    const int n = (int)min((int64_t)8, cols - c);
    uint4 o = make_uint4(0, 0, 0, 0);
    if (!targets || (uint64_t)target_of(targets, t64, at.row) < (uint64_t)vocab) {
      const T* from = src + at.row * sr + c * sc;
      if (sc == 1 && n == 8 && !((uintptr_t)from & 15)) {
        o = *reinterpret_cast<const uint4*>(from);
      } else if (sc == 1) {
        o = load_bytes(from, n * 2);
      } else {
        __align__(16) T v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < n ? from[k * sc] : T(0.f);
        o = *reinterpret_cast<const uint4*>(v);
      }
    }
    *reinterpret_cast<uint4*>(dst + i * 8) = o;
  }
}

// A matrix of f32 as three bf16 planes, the parts of next_part; zero as
// above. A thread makes 8 elements of each plane.
__global__ void split_rows(const float* __restrict__ src, int64_t rows, int64_t cols, int64_t sr,
                           int64_t sc, __nv_bfloat16* __restrict__ dst, int64_t ld, int64_t plane,
                           const void* targets, int t64, int64_t vocab) {
  const int64_t per = ld / 8, total = rows * per;
  const bool narrow = total < ((int64_t)1 << 32);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const RowItem at = row_item(i, per, narrow);
    const int64_t c = at.item * 8;
    const int n = (int)min((int64_t)8, cols - c);
    float v[8] = {};
    if (!targets || (uint64_t)target_of(targets, t64, at.row) < (uint64_t)vocab) {
      const float* from = src + at.row * sr + c * sc;
      if (sc == 1 && n == 8 && !((uintptr_t)from & 15)) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(from);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(from + 4);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < n) v[k] = from[k * sc];
      }
    }
#pragma unroll
    for (int z = 0; z < 3; ++z) {
      __align__(16) __nv_bfloat16 b[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) b[k] = __float2bfloat16_rn(next_part(v[k], z == 2));
      *reinterpret_cast<uint4*>(dst + z * plane + i * 8) = *reinterpret_cast<const uint4*>(b);
    }
  }
}

// What a copy of an operand takes: f32 is always split, 16-bit rows are copied
// where TMA cannot read them or rows without a loss must be zero
template <typename T>
size_t copy_bytes(const T* src, int64_t rows, int64_t cols, int64_t sr, int64_t sc, bool masked) {
  const int64_t ld = (cols + 7) / 8 * 8;
  if (sizeof(T) == 4) return (size_t)rows * ld * 6;
  const bool readable = (sc == 1 || cols == 1) && sr >= cols && mma::tma_readable(src, sr, 2);
  return readable && !masked ? 0 : (size_t)rows * ld * 2;
}
// The operand as the products take it, from `copy` (copy_bytes of it) or in place
template <typename T>
int operand(om_backend* be, const T* src, int64_t rows, int64_t cols, int64_t sr, int64_t sc,
            void* copy, mma::Matrix* out, const LossArgs* masked = nullptr) {
  if (!copy_bytes(src, rows, cols, sr, sc, masked != nullptr)) {
    *out = mma::Matrix{src, rows, cols, sr, 2};
    return OM_OK;
  }
  const int64_t ld = (cols + 7) / 8 * 8, plane = rows * ld, items = plane / 8;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, (int64_t)be->num_sms * 16));
  const void* targets = masked ? masked->targets : nullptr;
  const int t64 = masked ? masked->target64 : 0;
  const int64_t vocab = masked ? masked->V : 0;
  ProfScope prof(be, sizeof(T) == 4 ? "loss_split" : "loss_pack");
  if constexpr (sizeof(T) == 4)
    split_rows<<<grid, 256, 0, be->stream>>>(src, rows, cols, sr, sc, (__nv_bfloat16*)copy, ld, plane,
                                             targets, t64, vocab);
  else
    pack_rows<T><<<grid, 256, 0, be->stream>>>(src, rows, cols, sr, sc, (T*)copy, ld, targets, t64, vocab);
  note_launch();
  *out = mma::Matrix{copy, rows, cols, ld, 2, sizeof(T) == 4 ? plane : 0};
  return check_cuda(cudaGetLastError(), "loss operand launch");
}

// One allocation in parts of 256 bytes' alignment
struct Parts {
  size_t bytes = 0;
  size_t add(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

template <typename T, bool AMN, bool BMN, class Epi>
int product(om_backend* be, const char* name, const mma::Matrix& a, const mma::Matrix& b,
            mma::Tiling t, int splits, const Epi& epi) {
  constexpr bool P3 = sizeof(T) == 4, BF = !std::is_same<T, __half>::value;
  return mma::launch_product<false, P3, AMN, BMN>(be, name, a, b, BF, t, splits, epi);
}
template <typename T>
mma::Tiling tiles(const om_backend* be, int64_t M, int64_t N, bool odd = false) {
  return mma::tiling(be, M, N, 64, sizeof(T) == 4 ? 128 : 256, odd);
}
// rows [r0, r0 + n) of a K-major matrix
mma::Matrix rows_of(const mma::Matrix& m, int64_t r0, int64_t n) {
  mma::Matrix r = m;
  r.ptr = (const char*)m.ptr + r0 * m.ld * m.elem;
  r.rows = n;
  return r;
}
// the same memory with the roles of rows and k exchanged
mma::Matrix turned(const mma::Matrix& m) {
  mma::Matrix r = m;
  r.rows = m.k;
  r.k = m.rows;
  return r;
}

// Vocabulary entries whose f32 weights are split at a time (1 GiB of planes);
// 16-bit ones are read where they lie, or packed as a whole
template <typename T>
int64_t weight_rows(const LossArgs& p) {
  if (sizeof(T) == 2) return p.V;
  return std::min(p.V, std::max<int64_t>(256, ((int64_t)1 << 30) / (p.D * 6) / 256 * 256));
}

template <typename T>
int loss_forward_tc(om_backend* be, const LossArgs& p, float* loss, float* lse) {
  const T *px = (const T*)p.x, *pw = (const T*)p.w;
  const int64_t W = weight_rows<T>(p);
  const mma::Tiling t = tiles<T>(be, p.N, W, true);
  const int64_t slots = ((p.V + W - 1) / W) * ((W + t.bn - 1) / t.bn) * 2;
  Parts parts;
  const size_t ax = parts.add(copy_bytes(px, p.N, p.D, p.xn, p.xd, false));
  const size_t aw = parts.add(copy_bytes(pw, W, p.D, p.wv, p.wd, false));
  const size_t ap = parts.add((size_t)p.N * slots * 8), ah = parts.add((size_t)p.N * 4);
  Scratch ws;
  OM_TRY(ws.alloc(be, parts.bytes));
  char* at = (char*)ws.ptr;
  float2* part = (float2*)(at + ap);
  float* hit = (float*)(at + ah);
  mma::Matrix x, w;
  OM_TRY(operand(be, px, p.N, p.D, p.xn, p.xd, at + ax, &x));
  int64_t used = 0;
  for (int64_t v0 = 0; v0 < p.V; v0 += W) {
    const int64_t n = std::min(W, p.V - v0);
    OM_TRY(operand(be, pw + v0 * p.wv, n, p.D, p.wv, p.wd, at + aw, &w));
    const StatsEpi epi{p.targets, p.target64, v0, part + used * p.N, p.N, hit};
    OM_TRY((product<T, false, false>(be, "loss_logits", x, w, t, 1, epi)));
    used += (n + t.bn - 1) / t.bn * 2;
  }
  ProfScope prof(be, "loss_join_stats");
  join_stats<<<(unsigned)((p.N + 7) / 8), 256, 0, be->stream>>>(
      part, (int)used, p.N, p.targets, p.target64, p.V, hit, loss, lse);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss join launch");
}

template <typename T>
int loss_backward_tc(om_backend* be, const LossArgs& p, const float* lse, const float* dloss, T* dx,
                     int64_t dxd, int64_t dxn, T* dw, int64_t dwd, int64_t dwv) {
  constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
  if (p.N == 0) {
    zero_rows<T><<<flat_grid(be, p.V * p.D), 256, 0, be->stream>>>(dw, p.V, p.D, dwv, dwd);
    note_launch();
    return check_cuda(cudaGetLastError(), "loss backward launch");
  }
  // a piece's dz takes at most 512 MiB (f32: 1.5 GiB)
  const int64_t fit = ((int64_t)256 << 20) / p.N / 256 * 256;
  const int64_t P = std::min({(p.V + 255) / 256 * 256, std::max<int64_t>(256, fit),
                              (weight_rows<T>(p) + 255) / 256 * 256});
  // dx sums over the vocabulary. Its tiles are the widest that there are, and
  // where they leave SMs idle the sum is split, 16 slabs of 64 entries at least
  // to a split, which is worth its f32 sums (509 x 771 x 8191 f32: 80 us with
  // narrow tiles in two splits)
  const int most = PLANES == 3 ? 128 : 256;
  mma::Tiling tx{p.D > 128 ? most : p.D > 64 ? 128 : 64, 0};
  tx.pair = p.N > 128 && tx.bn >= 128;
  const int64_t rows = tx.pair ? 256 : 128;
  const int64_t txt = (p.N + rows - 1) / rows * ((p.D + tx.bn - 1) / tx.bn);
  const int64_t slots = tx.pair ? be->num_sms / 2 : be->num_sms;
  const int64_t least = (std::min(P, p.V) + 63) / 64;
  const int splits = (int)std::max<int64_t>(1, std::min<int64_t>({slots / txt, least / 16, 64}));
  const int64_t acc_ld = (p.D + tx.bn - 1) / tx.bn * tx.bn;
  const T *px = (const T*)p.x, *pw = (const T*)p.w;
  const int64_t W = PLANES == 3 ? std::min(P, p.V) : p.V;
  Parts parts;
  const size_t az = parts.add((size_t)p.N * P * 2 * PLANES);
  const size_t ax = parts.add(copy_bytes(px, p.N, p.D, p.xn, p.xd, true));
  const size_t aw = parts.add(copy_bytes(pw, W, p.D, p.wv, p.wd, false));
  const size_t as = parts.add(4);
  const size_t aa = parts.add(splits > 1 || P < p.V ? (size_t)splits * p.N * acc_ld * 4 : 0);
  Scratch ws;
  OM_TRY(ws.alloc(be, parts.bytes));
  char* at = (char*)ws.ptr;
  void* dzs = at + az;
  float* acc = (float*)(at + aa);
  float* scale = nullptr;
  // rows without a loss are zero here: whatever they hold reaches no gradient
  mma::Matrix x, w;
  OM_TRY(operand(be, px, p.N, p.D, p.xn, p.xd, at + ax, &x, &p));
  if (PLANES == 1) {
    OM_TRY(operand(be, pw, p.V, p.D, p.wv, p.wd, at + aw, &w));
    scale = (float*)(at + as);
    gradient_scale<<<1, 1024, 0, be->stream>>>(dloss, p.targets, p.target64, p.V, p.N,
                                               std::is_same<T, __half>::value ? 16384.f : 1.f, scale);
    note_launch();
  }
  const int vecx = row_stores(dx, dxn, dxd, sizeof(T)), vecw = row_stores(dw, dwv, dwd, sizeof(T));
  for (int64_t v0 = 0; v0 < p.V; v0 += P) {
    const int64_t n = std::min(P, p.V - v0);
    const bool last = v0 + n == p.V;
    mma::Matrix wp;
    if (PLANES == 1) wp = rows_of(w, v0, n);
    else OM_TRY(operand(be, pw + v0 * p.wv, n, p.D, p.wv, p.wd, at + aw, &wp));
    const mma::Matrix dz{dzs, p.N, n, P, 2, PLANES == 3 ? p.N * P : 0};
    GradEpi<T> ge{{}, boxes<T>(p.D, 1), p.targets, p.target64, p.V, v0, lse, dloss, scale, dzs, P, p.N * P};
    if (ge.boxed) OM_TRY(mma::encode_result(&ge.map, dzs, p.N, n, P));
    OM_TRY((product<T, false, false>(be, "loss_dlogits", x, wp, tiles<T>(be, p.N, n), 1, ge)));
    const int now = (int)std::min<int64_t>(splits, (n + 63) / 64);
    const OutEpi<T> xe{{}, 0, dx, dxn, dxd, vecx, scale, acc, acc_ld, p.N * acc_ld, v0 > 0, splits > 1 || !last,
                       counted_of(p)};
    OM_TRY((product<T, false, true>(be, "loss_dx", dz, turned(wp), tx, now, xe)));
    OutEpi<T> we{{}, boxes<T>(p.N, vecw), dw + v0 * dwv, dwv, dwd, vecw, scale, nullptr, 0, 0, 0, 0, Counted{}};
    if (we.boxed) OM_TRY(mma::encode_result(&we.map, dw + v0 * dwv, n, p.D, dwv));
    OM_TRY((product<T, true, true>(be, "loss_dw", turned(dz), turned(x), tiles<T>(be, n, p.D), 1, we)));
  }
  if (splits > 1) {
    ProfScope prof(be, "loss_join_splits");
    join_splits<T><<<flat_grid(be, p.N * p.D), 256, 0, be->stream>>>(
        acc, splits, p.N * acc_ld, acc_ld, p.N, p.D, scale, counted_of(p), dx, dxn, dxd);
    note_launch();
  }
  return check_cuda(cudaGetLastError(), "loss backward launch");
}

#include "om_loss_few.cuh"

int forward_f32(om_backend* be, const LossArgs& p, float* loss, float* lse) {
  if (few_tokens(p)) {
    if (p.N == 1) return few_forward<1>(be, few_args(p), p, loss, lse);
    if (p.N <= 4) return few_forward<4>(be, few_args(p), p, loss, lse);
    return few_forward<FEW>(be, few_args(p), p, loss, lse);
  }
  return be->f32_exact ? loss_forward<float>(be, p, loss, lse) : loss_forward_tc<float>(be, p, loss, lse);
}
int backward_f32(om_backend* be, const LossArgs& p, const float* lse, const float* dloss, float* dx,
                 int64_t dxd, int64_t dxn, float* dw, int64_t dwd, int64_t dwv) {
  if (p.N > 0 && few_tokens(p)) {
    if (p.N == 1) return few_backward<1>(be, few_args(p), p, lse, dloss, dx, dxd, dxn, dw, dwd, dwv);
    if (p.N <= 4) return few_backward<4>(be, few_args(p), p, lse, dloss, dx, dxd, dxn, dw, dwd, dwv);
    return few_backward<FEW>(be, few_args(p), p, lse, dloss, dx, dxd, dxn, dw, dwd, dwv);
  }
  return be->f32_exact ? loss_backward<float>(be, p, lse, dloss, dx, dxd, dxn, dw, dwd, dwv)
                       : loss_backward_tc<float>(be, p, lse, dloss, dx, dxd, dxn, dw, dwd, dwv);
}

int check_loss(const char* who, om_backend* be, om_dtype dtype, const int64_t* shape,
               om_dtype target_dtype) {
  const std::string w(who);
  if (!be || !shape) return set_error(OM_ERR_INVALID, w + ": null argument");
  if (dtype != OM_F32 && dtype != OM_F64 && !is_half(dtype))
    return set_error(OM_ERR_UNSUPPORTED, w + ": dtype must be f32, f64, bf16 or f16");
  if (target_dtype != OM_I32 && target_dtype != OM_I64)
    return set_error(OM_ERR_UNSUPPORTED, w + ": targets must be i32 or i64");
  for (int k = 0; k < 3; ++k)
    if (shape[k] < 0 || shape[k] > 0x7fffffff - 1024)
      return set_error(OM_ERR_SHAPE, w + ": extent out of range");
  if (shape[0] == 0 || shape[2] == 0)
    return set_error(OM_ERR_SHAPE, w + ": the width and the vocabulary must not be empty");
  return OM_OK;
}

}  // namespace
}  // namespace om

using namespace om;

extern "C" int om_b200_linear_cross_entropy(om_backend* be, om_dtype dtype, const int64_t* shape,
                                            const void* x, const int64_t* strides_x, const void* w,
                                            const int64_t* strides_w, om_dtype target_dtype,
                                            const void* targets, void* loss, void* lse) {
  OM_TRY(check_loss("om_b200_linear_cross_entropy", be, dtype, shape, target_dtype));
  if (shape[1] == 0) return OM_OK;
  if (!x || !strides_x || !w || !strides_w || !targets || !loss || !lse)
    return set_error(OM_ERR_INVALID, "om_b200_linear_cross_entropy: null argument");
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "linear_cross_entropy: device");
  const LossArgs p{shape[1], shape[0], shape[2], x, strides_x[0], strides_x[1], w, strides_w[0],
                   strides_w[1], targets, target_dtype == OM_I64};
  if (dtype == OM_F64) return loss_forward<double>(be, p, (double*)loss, (double*)lse);
  if (dtype == OM_BF16) return loss_forward_tc<__nv_bfloat16>(be, p, (float*)loss, (float*)lse);
  if (dtype == OM_F16) return loss_forward_tc<__half>(be, p, (float*)loss, (float*)lse);
  return forward_f32(be, p, (float*)loss, (float*)lse);
}

extern "C" int om_b200_linear_cross_entropy_backward(
    om_backend* be, om_dtype dtype, const int64_t* shape, const void* x, const int64_t* strides_x,
    const void* w, const int64_t* strides_w, om_dtype target_dtype, const void* targets,
    const void* lse, const void* dloss, void* dx, const int64_t* strides_dx, void* dw,
    const int64_t* strides_dw) {
  OM_TRY(check_loss("om_b200_linear_cross_entropy_backward", be, dtype, shape, target_dtype));
  if (!strides_w || !dw || !strides_dw || !w ||
      (shape[1] && (!x || !strides_x || !targets || !lse || !dloss || !dx || !strides_dx)))
    return set_error(OM_ERR_INVALID, "om_b200_linear_cross_entropy_backward: null argument");
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "linear_cross_entropy_backward: device");
  const int64_t zero[2] = {0, 0};
  if (shape[1] == 0) strides_x = strides_dx = zero;
  const LossArgs p{shape[1], shape[0], shape[2], x, strides_x[0], strides_x[1], w, strides_w[0],
                   strides_w[1], targets, target_dtype == OM_I64};
#define OM_LOSS_BWD(FN, T, S)                                                               \
  FN(be, p, (const S*)lse, (const S*)dloss, (T*)dx, strides_dx[0], strides_dx[1], \
                   (T*)dw, strides_dw[0], strides_dw[1])
  if (dtype == OM_F64) return OM_LOSS_BWD(loss_backward<double>, double, double);
  if (dtype == OM_BF16) return OM_LOSS_BWD(loss_backward_tc<__nv_bfloat16>, __nv_bfloat16, float);
  if (dtype == OM_F16) return OM_LOSS_BWD(loss_backward_tc<__half>, __half, float);
  return OM_LOSS_BWD(backward_f32, float, float);
#undef OM_LOSS_BWD
}
