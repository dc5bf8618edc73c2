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

inline bool is_half(om_dtype dt) { return dt == OM_BF16 || dt == OM_F16; }

}  // namespace om
