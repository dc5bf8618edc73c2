// Element types of the sequence-model operators and their conversion to and
// from the type they are computed in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "om_internal.h"

namespace om {

template <typename T>
struct Elem;  // State: the type sums and states of T are held in
template <>
struct Elem<float> {
  using State = float;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
};
template <>
struct Elem<double> {
  using State = double;
  static __device__ __forceinline__ double load(double v) { return v; }
  static __device__ __forceinline__ double store(double v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  using State = float;
  static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  using State = float;
  static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half store(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 32 values of a row as T. `wide`: dst is 32-byte aligned, and each store fills
// a sector of L2; else 16 bytes at a time.
__device__ __forceinline__ void store_sector(void* dst, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(u[0]),
               "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
__device__ __forceinline__ void store_sixteens(void* dst, const uint32_t (&u)[8]) {
  uint4* d = reinterpret_cast<uint4*>(dst);
  d[0] = make_uint4(u[0], u[1], u[2], u[3]);
  d[1] = make_uint4(u[4], u[5], u[6], u[7]);
}
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float (&v)[32], bool wide) {
  constexpr int PER = 32 / sizeof(T);  // values of a sector
#pragma unroll
  for (int c = 0; c < 32; c += PER) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(v[c + i]);
      else u[i] = pack2(v[c + 2 * i], v[c + 2 * i + 1], T());
    }
    if (wide) store_sector(dst + c, u);
    else store_sixteens(dst + c, u);
  }
}

// A warp's 32 x 32 results, lane by row, where rows cannot be written 16 bytes
// at a time: turned in shared memory (a word of padding per row), so that each
// store writes 32 neighbours of one row. rows: how many of the warp's 32 exist.
template <typename T>
__device__ __forceinline__ void store_turned(float* turn, const float (&v)[32], T* first, int64_t dr,
                                             int64_t dc, int rows, int cols) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 32; ++c) turn[lane * 33 + c] = v[c];
  __syncwarp();
  if (lane < cols) {
    T* to = first + lane * dc;
#pragma unroll 8
    for (int r = 0; r < rows; ++r, to += dr) *to = Elem<T>::store(turn[r * 33 + lane]);
  }
  __syncwarp();
}

// The `bytes` (16 at most) from `at` on, zero behind them, from the aligned words
// that hold them, shifted into place
__device__ __forceinline__ uint4 load_bytes(const void* at, int bytes) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)at & ~(uintptr_t)3);
  const int off = (int)((uintptr_t)at & 3);
  uint32_t v[5], o[4];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = i * 4 < bytes + off ? __ldg(w + i) : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = __funnelshift_r(v[i], v[i + 1], off * 8);
    const int keep = bytes - 4 * i;
    if (keep < 4) o[i] = keep <= 0 ? 0u : o[i] & ((1u << (8 * keep)) - 1u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Row and place of item i of rows of `per` items
struct RowItem {
  int64_t row;
  int64_t item;
};
__device__ __forceinline__ RowItem row_item(int64_t i, int64_t per, bool narrow) {
  const int64_t r = narrow ? (int64_t)((uint32_t)i / (uint32_t)per) : i / per;
  return RowItem{r, i - r * per};
}

// How a row-major result may be written: 2 = sectors of 32 bytes, 1 = 16 bytes,
// 0 = element by element
inline int row_stores(const void* ptr, int64_t row, int64_t col, int elem) {
  const uint64_t at = (uint64_t)(uintptr_t)ptr | (uint64_t)(row * elem);
  return col != 1 || row <= 0 || at % 16 ? 0 : at % 32 ? 1 : 2;
}

inline bool is_half(om_dtype dt) { return dt == OM_BF16 || dt == OM_F16; }

}  // namespace om
