// Softmax cross entropy of the logits z = x w^T over a vocabulary, and its
// gradients, without ever holding all logits:
//     lse_n = log sum_v exp(z_nv),  loss_n = lse_n - z_{n, target_n}
//     dz_nv = dloss_n (exp(z_nv - lse_n) - [v == target_n]),
//     dx = dz w,  dw = dz^T x.
// The vocabulary is walked in pieces; a piece's logits live in scratch memory
// until the next piece and are computed a second time by the backward pass.
#include <algorithm>

#include "om_convert.cuh"

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

// the element [r, c] of a strided matrix, into a row-major one of type S;
// rows whose target lies outside the vocabulary become zero when given
template <typename T, typename S>
__global__ void convert_rows(const T* __restrict__ src, int64_t rows, int64_t cols, int64_t sr,
                             int64_t sc, S* __restrict__ dst, const void* targets, int t64,
                             int64_t vocab) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols, c = i - r * cols;
    bool keep = true;
    if (targets) {
      const int64_t t = target_of(targets, t64, r);
      keep = t >= 0 && t < vocab;
    }
    dst[i] = keep ? (S)Elem<T>::load(src[r * sr + c * sc]) : S(0);
  }
}

// a row-major matrix of type S into a strided one of type T
template <typename T, typename S>
__global__ void store_rows(const S* __restrict__ src, int64_t rows, int64_t cols,
                           T* __restrict__ dst, int64_t dr, int64_t dc) {
  const int64_t total = rows * cols;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols, c = i - r * cols;
    dst[r * dr + c * dc] = Elem<T>::store(src[i]);
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

unsigned flat_grid(om_backend* be, int64_t n) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((n + 255) / 256, (int64_t)be->num_sms * 16));
}

template <typename S>
GemmArgs product(om_dtype dt, int64_t M, int64_t N, int64_t K, const void* a, int64_t am,
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

// Vocabulary entries per piece: a piece's logits take at most 256 MiB
int64_t piece_size(int64_t N, int64_t V, size_t elem) {
  const int64_t fit = ((int64_t)256 << 20) / (int64_t)elem / std::max<int64_t>(N, 1) / 128 * 128;
  return std::min(V, std::max<int64_t>(128, fit));
}

// f32 / f64: pieces through the library's own products
template <typename T>
int loss_forward(om_backend* be, const LossArgs& p, typename Elem<T>::State* loss,
                 typename Elem<T>::State* lse) {
  using S = typename Elem<T>::State;
  constexpr bool conv = !std::is_same<T, S>::value;
  const om_dtype dt = sizeof(S) == 8 ? OM_F64 : OM_F32;
  const int64_t P = piece_size(p.N, p.V, sizeof(S));
  Scratch zs, stats, xs, wsc;
  OM_TRY(zs.alloc(be, (size_t)p.N * P * sizeof(S)));
  OM_TRY(stats.alloc(be, (size_t)p.N * 3 * sizeof(S)));
  S* run = (S*)stats.ptr;
  const S* x = (const S*)p.x;
  int64_t xd = p.xd, xn = p.xn;
  if (conv) {
    OM_TRY(xs.alloc(be, (size_t)p.N * p.D * sizeof(S)));
    OM_TRY(wsc.alloc(be, (size_t)P * p.D * sizeof(S)));
    convert_rows<T, S><<<flat_grid(be, p.N * p.D), 256, 0, be->stream>>>(
        (const T*)p.x, p.N, p.D, p.xn, p.xd, (S*)xs.ptr, nullptr, 0, 0);
    note_launch();
    x = (const S*)xs.ptr, xd = 1, xn = p.D;
  }
  for (int64_t v0 = 0; v0 < p.V; v0 += P) {
    const int64_t n = std::min(P, p.V - v0);
    const T* wt = (const T*)p.w + v0 * p.wv;
    const S* w = (const S*)(const void*)wt;
    int64_t wd = p.wd, wv = p.wv;
    if (conv) {
      convert_rows<T, S><<<flat_grid(be, n * p.D), 256, 0, be->stream>>>(
          wt, n, p.D, p.wv, p.wd, (S*)wsc.ptr, nullptr, 0, 0);
      note_launch();
      w = (const S*)wsc.ptr, wd = 1, wv = p.D;
    }
    OM_TRY(launch_gemm(be, product<S>(dt, p.N, n, p.D, x, xn, xd, w, wd, wv, zs.ptr, n)));
    ProfScope prof(be, "loss_piece_stats");
    piece_stats<S><<<(unsigned)p.N, 256, 0, be->stream>>>(
        (const S*)zs.ptr, n, v0, p.targets, p.target64, p.V, run, run + p.N, run + 2 * p.N, v0 == 0,
        v0 + n == p.V, loss, lse);
    note_launch();
    OM_CUDA(cudaGetLastError(), "loss piece launch");
  }
  return OM_OK;
}

template <typename T>
int loss_backward(om_backend* be, const LossArgs& p, const typename Elem<T>::State* lse,
                  const typename Elem<T>::State* dloss, T* dx, int64_t dxd, int64_t dxn, T* dw,
                  int64_t dwd, int64_t dwv) {
  using S = typename Elem<T>::State;
  constexpr bool conv = !std::is_same<T, S>::value;
  const om_dtype dt = sizeof(S) == 8 ? OM_F64 : OM_F32;
  const int64_t P = piece_size(p.N, p.V, sizeof(S));
  const int64_t nx = p.N * p.D;
  if (p.N == 0) {  // no token: the weights' gradient is zero
    zero_rows<T><<<flat_grid(be, p.V * p.D), 256, 0, be->stream>>>(dw, p.V, p.D, dwv, dwd);
    note_launch();
    return check_cuda(cudaGetLastError(), "loss backward launch");
  }
  Scratch zs, xs, acc, part, wsc, dws;
  OM_TRY(zs.alloc(be, (size_t)p.N * P * sizeof(S)));
  OM_TRY(xs.alloc(be, (size_t)nx * sizeof(S)));
  OM_TRY(acc.alloc(be, (size_t)nx * sizeof(S)));
  if (P < p.V) OM_TRY(part.alloc(be, (size_t)nx * sizeof(S)));
  if (conv) OM_TRY(wsc.alloc(be, (size_t)P * p.D * sizeof(S)));
  OM_TRY(dws.alloc(be, (size_t)P * p.D * sizeof(S)));
  // rows without a loss are zero here: whatever they hold reaches no gradient
  convert_rows<T, S><<<flat_grid(be, nx), 256, 0, be->stream>>>(
      (const T*)p.x, p.N, p.D, p.xn, p.xd, (S*)xs.ptr, p.targets, p.target64, p.V);
  note_launch();
  for (int64_t v0 = 0; v0 < p.V; v0 += P) {
    const int64_t n = std::min(P, p.V - v0);
    const T* wt = (const T*)p.w + v0 * p.wv;
    const S* w = (const S*)(const void*)wt;
    int64_t wd = p.wd, wv = p.wv;
    if (conv) {
      convert_rows<T, S><<<flat_grid(be, n * p.D), 256, 0, be->stream>>>(
          wt, n, p.D, p.wv, p.wd, (S*)wsc.ptr, nullptr, 0, 0);
      note_launch();
      w = (const S*)wsc.ptr, wd = 1, wv = p.D;
    }
    OM_TRY(launch_gemm(be, product<S>(dt, p.N, n, p.D, xs.ptr, p.D, 1, w, wd, wv, zs.ptr, n)));
    piece_gradient<S><<<(unsigned)p.N, 256, 0, be->stream>>>((S*)zs.ptr, p.N, n, v0, p.targets,
                                                             p.target64, p.V, lse, dloss);
    note_launch();
    S* to = v0 ? (S*)part.ptr : (S*)acc.ptr;
    OM_TRY(launch_gemm(be, product<S>(dt, p.N, p.D, n, zs.ptr, n, 1, w, wv, wd, to, p.D)));
    if (v0) {
      add_into<S><<<flat_grid(be, nx), 256, 0, be->stream>>>((S*)acc.ptr, (const S*)part.ptr, nx);
      note_launch();
    }
    OM_TRY(launch_gemm(be, product<S>(dt, n, p.D, p.N, zs.ptr, 1, n, xs.ptr, p.D, 1, dws.ptr, p.D)));
    store_rows<T, S><<<flat_grid(be, n * p.D), 256, 0, be->stream>>>(
        (const S*)dws.ptr, n, p.D, dw + v0 * dwv, dwv, dwd);
    note_launch();
  }
  store_rows<T, S><<<flat_grid(be, nx), 256, 0, be->stream>>>((const S*)acc.ptr, p.N, p.D, dx, dxn,
                                                              dxd);
  note_launch();
  return check_cuda(cudaGetLastError(), "loss backward launch");
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
  if (dtype == OM_BF16) return loss_forward<__nv_bfloat16>(be, p, (float*)loss, (float*)lse);
  if (dtype == OM_F16) return loss_forward<__half>(be, p, (float*)loss, (float*)lse);
  return loss_forward<float>(be, p, (float*)loss, (float*)lse);
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
#define OM_LOSS_BWD(T, S)                                                                         \
  loss_backward<T>(be, p, (const S*)lse, (const S*)dloss, (T*)dx, strides_dx[0], strides_dx[1], \
                   (T*)dw, strides_dw[0], strides_dw[1])
  if (dtype == OM_F64) return OM_LOSS_BWD(double, double);
  if (dtype == OM_BF16) return OM_LOSS_BWD(__nv_bfloat16, float);
  if (dtype == OM_F16) return OM_LOSS_BWD(__half, float);
  return OM_LOSS_BWD(float, float);
#undef OM_LOSS_BWD
}
