// Matrix product in 8-bit integers with scales for each row and channel, and
// the quantiser of its rows.
#include <algorithm>

#include "om_convert.cuh"

namespace om {
namespace {

// the larger magnitude; a NaN on either side stays
__device__ __forceinline__ float max_abs(float m, float v) {
  v = fabsf(v);
  return v > m || v != v ? v : m;
}

// x / scale rounded to a whole number; an infinite scale leaves zero, as do
// NaN and infinite x
__device__ __forceinline__ int8_t quantized(float x, float scale) {
  const float r = rintf(__fdiv_rn(x, scale));
  return r != r ? (int8_t)0 : (int8_t)fminf(fmaxf(r, -127.f), 127.f);
}

__device__ __forceinline__ float block_max_abs(float m) {
  __shared__ float part[32];
  for (int o = 16; o; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = part[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) m = max_abs(m, part[i]);
  return m;
}

template <typename T>
__global__ void quantize_kernel(const T* __restrict__ x, int64_t K, int64_t xk, int64_t xm,
                                int8_t* __restrict__ q, int64_t qk, int64_t qm,
                                float* __restrict__ scale) {
  const int64_t row = blockIdx.x;
  const T* xr = x + row * xm;
  float m = 0.f;
  for (int64_t k = threadIdx.x; k < K; k += blockDim.x) m = max_abs(m, Elem<T>::load(xr[k * xk]));
  m = block_max_abs(m);
  const float s = __fdiv_rn(m, 127.f);
  if (threadIdx.x == 0) scale[row] = s;
  for (int64_t k = threadIdx.x; k < K; k += blockDim.x)
    q[row * qm + k * qk] = s > 0.f ? quantized(Elem<T>::load(xr[k * xk]), s) : (int8_t)0;
}

struct I8Args {
  int64_t M, N, K;
  const int8_t* q;
  int64_t qk, qm;
  const int8_t* w;
  int64_t wk, wn;
  const float *q_scale, *w_scale, *bias;
  void* y;
  int64_t yn, ym;
};

// 32 x 32 outputs per block of 256 threads, 32 k per step
template <typename T>
__global__ void matmul_i8_kernel(I8Args p, int64_t tiles_n) {
  __shared__ int8_t a[32][33], b[32][33];
  const int64_t m0 = blockIdx.x / tiles_n * 32, n0 = blockIdx.x % tiles_n * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  int acc[4] = {0, 0, 0, 0};
  for (int64_t k0 = 0; k0 < p.K; k0 += 32) {
    for (int i = ty; i < 32; i += 8) {
      const bool in = k0 + tx < p.K;
      a[i][tx] = in && m0 + i < p.M ? p.q[(m0 + i) * p.qm + (k0 + tx) * p.qk] : (int8_t)0;
      b[i][tx] = in && n0 + i < p.N ? p.w[(n0 + i) * p.wn + (k0 + tx) * p.wk] : (int8_t)0;
    }
    __syncthreads();
    for (int k = 0; k < 32; ++k)
      for (int i = 0; i < 4; ++i) acc[i] += (int)a[ty + 8 * i][k] * (int)b[tx][k];
    __syncthreads();
  }
  const int64_t n = n0 + tx;
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 8 * i;
    if (m >= p.M || n >= p.N) continue;
    float v = __fmul_rn(__fmul_rn((float)acc[i], p.q_scale[m]), p.w_scale[n]);
    if (p.bias) v = __fadd_rn(v, p.bias[n]);
    ((T*)p.y)[m * p.ym + n * p.yn] = Elem<T>::store(v);
  }
}

template <typename T>
int launch_quantize(om_backend* be, int64_t K, int64_t M, const void* x, const int64_t* sx, void* q,
                    int64_t qk, int64_t qm, float* scale) {
  ProfScope prof(be, "quantize_rows");
  quantize_kernel<T><<<(unsigned)M, 256, 0, be->stream>>>((const T*)x, K, sx[0], sx[1], (int8_t*)q,
                                                          qk, qm, scale);
  note_launch();
  return check_cuda(cudaGetLastError(), "quantize_rows launch");
}

int quantize(om_backend* be, om_dtype dtype, int64_t K, int64_t M, const void* x, const int64_t* sx,
             void* q, int64_t qk, int64_t qm, float* scale) {
  if (dtype == OM_BF16) return launch_quantize<__nv_bfloat16>(be, K, M, x, sx, q, qk, qm, scale);
  if (dtype == OM_F16) return launch_quantize<__half>(be, K, M, x, sx, q, qk, qm, scale);
  return launch_quantize<float>(be, K, M, x, sx, q, qk, qm, scale);
}

template <typename T>
int launch_matmul(om_backend* be, const I8Args& p) {
  const int64_t tm = (p.M + 31) / 32, tn = (p.N + 31) / 32;
  if (tm * tn > 0x7fffffff) return set_error(OM_ERR_SHAPE, "matmul_i8: too many tiles");
  ProfScope prof(be, "matmul_i8");
  matmul_i8_kernel<T><<<(unsigned)(tm * tn), 256, 0, be->stream>>>(p, tn);
  note_launch();
  return check_cuda(cudaGetLastError(), "matmul_i8 launch");
}

int matmul(om_backend* be, om_dtype dtype, const I8Args& p) {
  if (dtype == OM_BF16) return launch_matmul<__nv_bfloat16>(be, p);
  if (dtype == OM_F16) return launch_matmul<__half>(be, p);
  return launch_matmul<float>(be, p);
}

int check_i8(const char* who, om_backend* be, om_dtype dtype, const int64_t* shape, int ndim) {
  const std::string w(who);
  if (!be || !shape) return set_error(OM_ERR_INVALID, w + ": null argument");
  if (dtype != OM_F32 && !is_half(dtype))
    return set_error(OM_ERR_UNSUPPORTED, w + ": dtype must be f32, bf16 or f16");
  for (int k = 0; k < ndim; ++k)
    if (shape[k] < 0 || shape[k] > 0x7fffffff - 1024)
      return set_error(OM_ERR_SHAPE, w + ": extent out of range");
  // 128 * 128 * K (a caller's own q may hold -128) stays inside 32 bits
  if (ndim == 3 && shape[0] > 131071)
    return set_error(OM_ERR_SHAPE, w + ": more than 131071 products per sum");
  return OM_OK;
}

}  // namespace
}  // namespace om

using namespace om;

extern "C" int om_b200_quantize_rows(om_backend* be, om_dtype dtype, const int64_t* shape,
                                     const void* x, const int64_t* strides_x, void* q,
                                     const int64_t* strides_q, float* scale) {
  OM_TRY(check_i8("om_b200_quantize_rows", be, dtype, shape, 2));
  const int64_t K = shape[0], M = shape[1];
  if (M == 0) return OM_OK;
  if (!scale || (K && (!x || !strides_x || !q || !strides_q)))
    return set_error(OM_ERR_INVALID, "om_b200_quantize_rows: null argument");
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "quantize_rows: device");
  const int64_t none[2] = {0, 0};
  if (!K) strides_x = strides_q = none;
  return quantize(be, dtype, K, M, x, strides_x, q, strides_q[0], strides_q[1], scale);
}

extern "C" int om_b200_matmul_i8(om_backend* be, om_dtype dtype, const int64_t* shape,
                                 const void* q, const int64_t* strides_q, const float* q_scale,
                                 const void* w, const int64_t* strides_w, const float* w_scale,
                                 const float* bias, void* y, const int64_t* strides_y) {
  OM_TRY(check_i8("om_b200_matmul_i8", be, dtype, shape, 3));
  const int64_t K = shape[0], M = shape[1], N = shape[2];
  if (M == 0 || N == 0) return OM_OK;
  if (!q_scale || !w_scale || !y || !strides_y || (K && (!q || !strides_q || !w || !strides_w)))
    return set_error(OM_ERR_INVALID, "om_b200_matmul_i8: null argument");
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "matmul_i8: device");
  const int64_t none[2] = {0, 0};
  if (!K) strides_q = strides_w = none;
  const I8Args p{M, N, K, (const int8_t*)q, strides_q[0], strides_q[1], (const int8_t*)w,
                 strides_w[0], strides_w[1], q_scale, w_scale, bias, y, strides_y[0], strides_y[1]};
  return matmul(be, dtype, p);
}

extern "C" int om_b200_linear_i8(om_backend* be, om_dtype dtype, const int64_t* shape,
                                 const void* x, const int64_t* strides_x, const void* w,
                                 const int64_t* strides_w, const float* w_scale, const float* bias,
                                 void* y, const int64_t* strides_y) {
  OM_TRY(check_i8("om_b200_linear_i8", be, dtype, shape, 3));
  const int64_t K = shape[0], M = shape[1], N = shape[2];
  if (M == 0 || N == 0) return OM_OK;
  if (!w_scale || !y || !strides_y || (K && (!x || !strides_x || !w || !strides_w)))
    return set_error(OM_ERR_INVALID, "om_b200_linear_i8: null argument");
  DeviceGuard guard(be->device);
  OM_CUDA(guard.status, "linear_i8: device");
  const int64_t none[2] = {0, 0};
  if (!K) strides_x = strides_w = none;
  const int64_t Kp = (K + 15) / 16 * 16;
  Scratch ws;
  OM_TRY(ws.alloc(be, (size_t)M * (Kp + 4) + 16));
  float* scale = (float*)ws.ptr;
  int8_t* q = (int8_t*)ws.ptr + (M * 4 + 15) / 16 * 16;
  OM_TRY(quantize(be, dtype, K, M, x, strides_x, q, 1, Kp, scale));
  const I8Args p{M, N, K, q, 1, Kp, (const int8_t*)w, strides_w[0], strides_w[1], scale, w_scale,
                 bias, y, strides_y[0], strides_y[1]};
  return matmul(be, dtype, p);
}
