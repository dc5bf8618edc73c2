// Matrix product in 8-bit integers with scales for each row and channel, and
// the quantiser of its rows. Sums are 32-bit integers; the scales are applied in
// f32, in one order, and the result is rounded once, so every variant gives the
// same bits.
#include <algorithm>

#include "om_convert.cuh"
#include "om_sm100.cuh"

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

// Four values at once, as bytes. x * (1 / s) is off the quotient by less than
// 3e-5 where |x / s| <= 127, so the nearest whole number is the quotient's
// unless the product lies within 1e-4 of the middle of two; only then is the
// division made. Adding 1.5 * 2^23 rounds to a whole number, ties to even, and
// leaves it in the low byte. (Dividing every element took 71 us for
// 8192 x 4096 bf16.) `s` is a normal number here.
__device__ __forceinline__ uint32_t quantized4(const float (&x)[4], float s, float inv) {
  constexpr float MAGIC = 12582912.f;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = __fmaf_rn(x[i], inv, MAGIC);
    const float off = __fmaf_rn(x[i], inv, -__fsub_rn(t, MAGIC));
    b[i] = __float_as_uint(t);
    if (fabsf(off) > 0.4999f) b[i] = (uint32_t)(int)quantized(x[i], s);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// 8 elements, 16-byte aligned, as f32
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  __align__(16) T t[8];
#pragma unroll
  for (int b = 0; b < (int)sizeof(T) * 8; b += 16)
    *reinterpret_cast<uint4*>((char*)t + b) = __ldg(reinterpret_cast<const uint4*>((const char*)p + b));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Elem<T>::load(t[i]);
}

// the largest magnitude; magnitudes order like their bits, NaN above all
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// 8 elements quantised; whatever is not a normal scale takes the long way
__device__ __forceinline__ uint2 quantized8(const float (&v)[8], float s, float inv, bool normal) {
  if (normal) {
    const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
    return make_uint2(quantized4(lo, s, inv), quantized4(hi, s, inv));
  }
  uint32_t u[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (s > 0.f) u[i / 4] |= (uint32_t)(uint8_t)quantized(v[i], s) << (8 * (i % 4));
  return make_uint2(u[0], u[1]);
}
__device__ __forceinline__ bool normal_scale(float s) { return s > 1e-36f && s < 1e36f; }

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

// The same where a row is contiguous, 16-byte aligned and short enough for the
// block's registers: it is read once, 8 elements per thread and turn.
constexpr int TURNS = 8, QUANT_THREADS = 128;
template <typename T>
__device__ __forceinline__ void widen8(const uint4 (&raw)[sizeof(T) / 2], float (&v)[8]) {
  __align__(16) T t[8];
  memcpy(t, raw, sizeof(T) * 8);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Elem<T>::load(t[i]);
}
template <typename T, int N>
__global__ void __launch_bounds__(QUANT_THREADS) quantize_vec_kernel(const T* __restrict__ x, int K,
                                                                     int64_t xm, int8_t* __restrict__ q,
                                                                     int64_t qm, float* __restrict__ scale) {
  const int64_t row = blockIdx.x;
  const T* xr = x + row * xm;
  constexpr int W = sizeof(T) / 2;
  uint4 raw[N][W];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = (i * QUANT_THREADS + (int)threadIdx.x) * 8;
#pragma unroll
    for (int b = 0; b < W; ++b)
      raw[i][b] = k < K ? __ldcs(reinterpret_cast<const uint4*>(xr + k) + b) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[8];
    widen8<T>(raw[i], v);
    top = max_bits(top, v);
  }
  __shared__ uint32_t part[QUANT_THREADS / 32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QUANT_THREADS / 32; ++i) top = max(top, part[i]);
  const float s = __fdiv_rn(__uint_as_float(top), 127.f), inv = __fdiv_rn(1.f, s);
  const bool normal = normal_scale(s);
  if (threadIdx.x == 0) scale[row] = s;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = (i * QUANT_THREADS + (int)threadIdx.x) * 8;
    if (k >= K) break;
    float v[8];
    widen8<T>(raw[i], v);
    *reinterpret_cast<uint2*>(q + row * qm + k) = quantized8(v, s, inv, normal);
  }
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

__device__ __forceinline__ float scaled(int acc, float q_scale, float w_scale) {
  return __fmul_rn(__fmul_rn((float)acc, q_scale), w_scale);
}

// ---- many rows: tensor cores ---------------------------------------------------

template <typename T>
struct ScaleEpi {
  const float *q_scale, *w_scale, *bias;
  T* y;
  int64_t dr, dc;
  int vec;   // row_stores of y
  int wide;  // w_scale and bias can be read 16 bytes at a time
  struct Row {
    float s;
  };
  int lent_bytes() const { return vec ? 0 : mma::TURN_BYTES; }
  __device__ __forceinline__ Row begin(int m, bool in, int) const {
    return Row{in ? q_scale[m] : 0.f};
  }
  __device__ __forceinline__ void columns(Row& row, int m, bool in, int n0, int N,
                                          const uint32_t (&r)[32], mma::Lent& lent) const {
    if (n0 >= N) return;
    float v[32];
    if (wide && N - n0 >= 32) {
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 w = __ldg(reinterpret_cast<const float4*>(w_scale + n0 + c));
        v[c] = scaled((int)r[c], row.s, w.x);
        v[c + 1] = scaled((int)r[c + 1], row.s, w.y);
        v[c + 2] = scaled((int)r[c + 2], row.s, w.z);
        v[c + 3] = scaled((int)r[c + 3], row.s, w.w);
      }
      if (bias) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 b = __ldg(reinterpret_cast<const float4*>(bias + n0 + c));
          v[c] = __fadd_rn(v[c], b.x), v[c + 1] = __fadd_rn(v[c + 1], b.y);
          v[c + 2] = __fadd_rn(v[c + 2], b.z), v[c + 3] = __fadd_rn(v[c + 3], b.w);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        if (n0 + c >= N) break;
        v[c] = scaled((int)r[c], row.s, w_scale[n0 + c]);
        if (bias) v[c] = __fadd_rn(v[c], bias[n0 + c]);
      }
    }
    const int lane = threadIdx.x & 31;
    T* to = y + (int64_t)m * dr;
    if (!vec) {
      store_turned(lent.words, v, y + (int64_t)(m - lane) * dr + n0 * dc, dr, dc,
                   __popc(__ballot_sync(0xffffffffu, in)), N - n0);
    } else if (in) {
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

// Rows of 8-bit numbers at 16-byte aligned places, zero behind their end; a
// thread makes 16
__global__ void pack_i8(const int8_t* __restrict__ src, int64_t rows, int K, int64_t sr, int64_t sk,
                        int8_t* __restrict__ dst, int64_t ld) {
  const int64_t per = ld / 16, total = rows * per;
  const bool narrow = total < ((int64_t)1 << 32);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const RowItem at = row_item(i, per, narrow);
    const int c = (int)at.item * 16, n = min(16, K - c);
    const int8_t* from = src + at.row * sr + (int64_t)c * sk;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (sk == 1) {
      o = load_bytes(from, n);
    } else {
      __align__(16) int8_t b[16] = {};
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k < n) b[k] = from[k * sk];
      o = *reinterpret_cast<const uint4*>(b);
    }
    *reinterpret_cast<uint4*>(dst + i * 16) = o;
  }
}

// ---- few rows: the weights stream through the CUDA cores --------------------------

constexpr int TOKEN_ROWS = 8;
constexpr int TOKEN_SMEM = 160 * 1024;

// Up to eight rows, whose dot products grow with them: 7.1, 8.7, 12.0 and 19.4 us
// for 1, 2, 4 and 8 bf16 rows of 4096 through 4096 x 4096 from memory (floor 2.6
// us), where the tensor cores' product, which wastes most of its rows but none of the
// weights, takes 15 us for any of them with its quantiser and 11.7 without. See
// few_rows for where they cross.
// A block keeps the M <= MM rows of q in shared memory and walks its share of
// the channels, a warp per channel: 16 weights per lane and step, four
// products per instruction, one shuffle reduction per row. T: the type of y,
// and of x where the rows are quantised here (q == null): 8 / MM warps a row,
// while the first weights are already under way.
template <typename T, int MM>
__global__ void __launch_bounds__(256, 2) token_i8_kernel(I8Args p, const T* __restrict__ x, int64_t xk,
                                                       int64_t xm, int vec, int Kp) {
  extern __shared__ __align__(16) int8_t qs[];  // [MM][Kp]
  constexpr int AHEAD = 4;
  constexpr int SHARE = 8 / MM;  // warps per row
  __shared__ float scale[MM];
  __shared__ uint32_t part[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int M = (int)p.M, K = (int)p.K;
  const int64_t n0 = p.N * blockIdx.x / gridDim.x, n1 = p.N * (blockIdx.x + 1) / gridDim.x;
  auto weights = [&](const int8_t* wr, int k) {
    int4 w = make_int4(0, 0, 0, 0);
    if (k + 16 <= K) {
      w = __ldcs(reinterpret_cast<const int4*>(wr + k));
    } else if (k < K) {  // the row's end: nothing behind it is read
      __align__(16) int8_t tail[16] = {};
#pragma unroll
      for (int i = 0; i < 15; ++i)
        if (k + i < K) tail[i] = wr[k + i];
      w = *reinterpret_cast<const int4*>(tail);
    }
    return w;
  };
  int64_t n = n0 + warp;
  int4 ahead[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    ahead[i] = n < n1 ? weights(p.w + n * p.wn, lane * 16 + i * 512) : make_int4(0, 0, 0, 0);

  const int row = warp / SHARE, first = (warp % SHARE) * 32 + lane;  // of the row's threads
  if (p.q) {
    if (row < M) {
      for (int k = first; k < Kp; k += SHARE * 32)
        qs[row * Kp + k] = k < K ? p.q[row * p.qm + k * p.qk] : (int8_t)0;
      if (first == 0) scale[row] = p.q_scale[row];
    }
  } else {
    const T* xr = x + row * xm;
    uint32_t top = 0;
    if (row < M) {
      if (vec) {
#pragma unroll 2
        for (int k = first * 8; k < K; k += SHARE * 256) {
          float v[8];
          load8(xr + k, v);
          top = max_bits(top, v);
        }
      } else {
        for (int k = first; k < K; k += SHARE * 32)
          top = max(top, __float_as_uint(Elem<T>::load(xr[k * xk])) & 0x7fffffffu);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) part[warp] = top;
    __syncthreads();
    if (row < M) {
#pragma unroll
      for (int i = 0; i < SHARE; ++i) top = max(top, part[row * SHARE + i]);
      const float s = __fdiv_rn(__uint_as_float(top), 127.f), inv = __fdiv_rn(1.f, s);
      const bool normal = normal_scale(s);
      if (first == 0) scale[row] = s;
      if (vec) {
        for (int k = first * 8; k < Kp; k += SHARE * 256) {
          uint2 q = make_uint2(0, 0);
          if (k < K) {
            float v[8];
            load8(xr + k, v);
            q = quantized8(v, s, inv, normal);
          }
          *reinterpret_cast<uint2*>(qs + row * Kp + k) = q;
        }
      } else {
        for (int k = first; k < Kp; k += SHARE * 32)
          qs[row * Kp + k] = k < K && s > 0.f ? quantized(Elem<T>::load(xr[k * xk]), s) : (int8_t)0;
      }
    }
  }
  __syncthreads();

  for (; n < n1; n += 8) {
    const int8_t* wr = p.w + n * p.wn;
    int acc[MM];
#pragma unroll
    for (int m = 0; m < MM; ++m) acc[m] = 0;
    auto add = [&](const int4& w, int k) {
#pragma unroll
      for (int m = 0; m < MM; ++m) {
        if (m >= M) break;
        const int4 q = *reinterpret_cast<const int4*>(qs + m * Kp + k);
        acc[m] = __dp4a(w.x, q.x, acc[m]);
        acc[m] = __dp4a(w.y, q.y, acc[m]);
        acc[m] = __dp4a(w.z, q.z, acc[m]);
        acc[m] = __dp4a(w.w, q.w, acc[m]);
      }
    };
    // the next AHEAD steps' weights are always under way
    for (int k0 = lane * 16; k0 < Kp; k0 += AHEAD * 512) {
      int4 now[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) now[i] = ahead[i];
      int k1 = k0 + AHEAD * 512;
      const int8_t* next = wr;
      if (k1 >= Kp) {
        next = n + 8 < n1 ? wr + 8 * p.wn : nullptr;
        k1 = lane * 16;
      }
      if (next) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ahead[i] = weights(next, k1 + i * 512);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (k0 + i * 512 < Kp) add(now[i], k0 + i * 512);
    }
#pragma unroll
    for (int m = 0; m < MM; ++m) {
      if (m >= M) break;
      const int a = __reduce_add_sync(0xffffffffu, acc[m]);
      if (lane == m) {
        float v = scaled(a, scale[m], p.w_scale[n]);
        if (p.bias) v = __fadd_rn(v, p.bias[n]);
        ((T*)p.y)[m * p.ym + n * p.yn] = Elem<T>::store(v);
      }
    }
  }
}

template <typename T>
int launch_quantize(om_backend* be, int64_t K, int64_t M, const void* x, const int64_t* sx, void* q,
                    int64_t qk, int64_t qm, float* scale) {
  ProfScope prof(be, "quantize_rows");
  if (sx[0] == 1 && qk == 1 && K % 8 == 0 && K <= QUANT_THREADS * 8 * TURNS && !((uintptr_t)x & 15) &&
      sx[1] * (int64_t)sizeof(T) % 16 == 0 && !((uintptr_t)q & 7) && qm % 8 == 0) {
    // as many turns as the row needs, so that short rows take few registers
    auto kernel = K <= QUANT_THREADS * 8 ? quantize_vec_kernel<T, 1>
                  : K <= QUANT_THREADS * 16 ? quantize_vec_kernel<T, 2>
                  : K <= QUANT_THREADS * 32 ? quantize_vec_kernel<T, 4> : quantize_vec_kernel<T, TURNS>;
    kernel<<<(unsigned)M, QUANT_THREADS, 0, be->stream>>>((const T*)x, (int)K, sx[1], (int8_t*)q, qm, scale);
    note_launch();
    return check_cuda(cudaGetLastError(), "quantize_rows launch");
  }
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

// Whether the weights can be read in place 16 bytes at a time; else they are
// packed for the call.
int readable_i8(om_backend* be, const int8_t* src, int64_t rows, int64_t K, int64_t sr, int64_t sk,
                Scratch& copy, mma::Matrix* out) {
  *out = mma::Matrix{src, rows, K, sr, 1};
  if ((sk == 1 || K == 1) && sr >= K && mma::tma_readable(src, sr, 1)) return OM_OK;
  const int64_t ld = (K + 15) / 16 * 16;
  OM_TRY(copy.alloc(be, (size_t)rows * ld));
  const int64_t items = rows * (ld / 16);
  ProfScope prof(be, "pack_i8");
  pack_i8<<<(unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)be->num_sms * 16), 256, 0, be->stream>>>(
      src, rows, (int)K, sr, sk, (int8_t*)copy.ptr, ld);
  note_launch();
  *out = mma::Matrix{copy.ptr, rows, K, ld, 1};
  return check_cuda(cudaGetLastError(), "matmul_i8 pack launch");
}

template <typename T, int MM>
int launch_token_rows(om_backend* be, const I8Args& p, const T* x, int64_t xk, int64_t xm,
                      int64_t Kp) {
  const size_t smem = (size_t)p.M * Kp;
  if (smem > PLAIN_SHARED)
    OM_TRY(allow_shared(be, (const void*)token_i8_kernel<T, MM>, TOKEN_SMEM, "matmul_i8"));
  const int64_t blocks = std::min<int64_t>((p.N + 7) / 8, (int64_t)be->num_sms * 2);
  ProfScope prof(be, "matmul_i8_token");
  const int vec = x && xk == 1 && p.K % 8 == 0 && !((uintptr_t)x & 15) && xm * (int64_t)sizeof(T) % 16 == 0;
  token_i8_kernel<T, MM><<<(unsigned)blocks, 256, smem, be->stream>>>(p, x, xk, xm, vec, (int)Kp);
  note_launch();
  return check_cuda(cudaGetLastError(), "matmul_i8 launch");
}

// Whether the token kernel takes the rows: one always does, more where the products
// are at most 2^26, or 2^25 where the rows come quantised and the tensor cores need
// one launch instead of two. Measured, token kernel against tensor cores: quantising,
// 4 x 4096 x 4096 (2^26) 12.0 and 15.0 us, 4 x 2048 x 8200 11.0 and 11.9, 8 x 2048 x
// 4096 12.0 and 10.7, 6 x 4096 x 4096 17.2 and 15.1, 4 x 4096 x 12288 22 and 17.8;
// quantised, 2 x 4096 x 4096 (2^25) 9.3 and 11.7, 4 x 2048 x 2048 6.9 and 7.3, 4 x 2048
// x 4096 8.5 and 8.1, 3 x 4096 x 6000 15.3 and 12.8; one row of 4096 x 12288 13.5 and
// 14.2. (At the limit it depends on the shape: 8 x 4096 x 1024 quantised 13.6 and 11.1.)
bool few_rows(int64_t M, int64_t K, int64_t N, bool quantising) {
  return M <= TOKEN_ROWS && M * ((K + 15) / 16 * 16) <= TOKEN_SMEM &&
         (M == 1 || M * K * N <= (int64_t)1 << (quantising ? 26 : 25));
}

// p.q == null: the rows are x's, quantised within the kernel
template <typename T>
int launch_tokens(om_backend* be, I8Args p, const T* x, int64_t xk, int64_t xm) {
  Scratch copy;
  mma::Matrix w;
  OM_TRY(readable_i8(be, p.w, p.N, p.K, p.wn, p.wk, copy, &w));
  p.w = (const int8_t*)w.ptr;
  p.wn = w.ld;
  const int64_t Kp = (p.K + 15) / 16 * 16;
  if (p.M == 1) return launch_token_rows<T, 1>(be, p, x, xk, xm, Kp);
  if (p.M == 2) return launch_token_rows<T, 2>(be, p, x, xk, xm, Kp);
  if (p.M <= 4) return launch_token_rows<T, 4>(be, p, x, xk, xm, Kp);
  return launch_token_rows<T, 8>(be, p, x, xk, xm, Kp);
}

template <typename T>
int launch_matmul(om_backend* be, const I8Args& p) {
  if (few_rows(p.M, p.K, p.N, false)) return launch_tokens<T>(be, p, nullptr, 0, 0);
  Scratch qc, wc;
  mma::Matrix q, w;
  OM_TRY(readable_i8(be, p.q, p.M, p.K, p.qm, p.qk, qc, &q));
  OM_TRY(readable_i8(be, p.w, p.N, p.K, p.wn, p.wk, wc, &w));
  const ScaleEpi<T> epi{p.q_scale, p.w_scale, p.bias, (T*)p.y, p.ym, p.yn,
                        row_stores(p.y, p.ym, p.yn, sizeof(T)),
                        !(((uintptr_t)p.w_scale | (uintptr_t)p.bias) & 15)};
  const mma::Tiling t = mma::tiling(be, p.M, p.N, 32, 256, true);
  return mma::launch_product<true, false, false, false>(be, "matmul_i8", q, w, false, t, 1, epi);
}

int matmul(om_backend* be, om_dtype dtype, const I8Args& p) {
  if (p.K == 0) {  // nothing is summed: the token kernel's loop is empty
    I8Args one = p;
    for (int64_t m = 0; m < p.M; m += TOKEN_ROWS) {
      one.M = std::min<int64_t>(TOKEN_ROWS, p.M - m);
      one.q_scale = p.q_scale + m;
      one.q = (const int8_t*)p.q_scale;  // not read
      one.w = (const int8_t*)p.w_scale;
      one.wn = 16, one.wk = 1;
      one.y = (char*)p.y + m * p.ym * (dtype == OM_F32 ? 4 : 2);
      if (dtype == OM_BF16) OM_TRY((launch_token_rows<__nv_bfloat16, 8>(be, one, nullptr, 0, 0, 0)));
      else if (dtype == OM_F16) OM_TRY((launch_token_rows<__half, 8>(be, one, nullptr, 0, 0, 0)));
      else OM_TRY((launch_token_rows<float, 8>(be, one, nullptr, 0, 0, 0)));
    }
    return OM_OK;
  }
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
  if (K && few_rows(M, K, N, true)) {
    const I8Args p{M, N, K, nullptr, 0, 0, (const int8_t*)w, strides_w[0], strides_w[1], nullptr,
                   w_scale, bias, y, strides_y[0], strides_y[1]};
    if (dtype == OM_BF16)
      return launch_tokens(be, p, (const __nv_bfloat16*)x, strides_x[0], strides_x[1]);
    if (dtype == OM_F16) return launch_tokens(be, p, (const __half*)x, strides_x[0], strides_x[1]);
    return launch_tokens(be, p, (const float*)x, strides_x[0], strides_x[1]);
  }
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
