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

// 32 values of a row as T, 16 bytes at a time
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 32; c += 8)
    *reinterpret_cast<uint4*>(dst + c) =
        make_uint4(pack2(v[c], v[c + 1], T()), pack2(v[c + 2], v[c + 3], T()),
                   pack2(v[c + 4], v[c + 5], T()), pack2(v[c + 6], v[c + 7], T()));
}
__device__ __forceinline__ void store_row(float* dst, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 32; c += 4)
    *reinterpret_cast<float4*>(dst + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
}

inline bool is_half(om_dtype dt) { return dt == OM_BF16 || dt == OM_F16; }

}  // namespace om
