// Element types of the operators that take float32, bfloat16 or float16 rows:
// loads widen to float32, stores round once (to nearest even).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace mr {

inline int elt_bytes(int dtype) { return dtype == MR_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == MR_F32 || dtype == MR_BF16 || dtype == MR_F16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of a row: 4 float32 or 8 two-byte values.
template <typename T>
struct Vec16 {
  static constexpr int kN = 16 / int(sizeof(T));
  uint4 raw;
  __device__ __forceinline__ void get(float (&f)[kN]) const {
    if constexpr (sizeof(T) == 4) {
      f[0] = __uint_as_float(raw.x); f[1] = __uint_as_float(raw.y);
      f[2] = __uint_as_float(raw.z); f[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
          const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          f[2 * i] = p.x;
          f[2 * i + 1] = p.y;
        }
      }
    }
  }
  __device__ __forceinline__ void put(const float (&f)[kN]) {
    if constexpr (sizeof(T) == 4) {
      raw = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                       __float_as_uint(f[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&p);
        } else {
          const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
      }
      raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// Calls f with a value of the element type that `dtype` names.
template <typename F>
inline int with_dtype(int dtype, F f) {
  switch (dtype) {
    case MR_F32: return f(float());
    case MR_BF16: return f(__nv_bfloat16());
    case MR_F16: return f(__half());
    default: return MR_ERR_ARGUMENT;
  }
}

}  // namespace mr
