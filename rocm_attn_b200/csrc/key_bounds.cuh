// Vectors of kVec elements and their elementwise minimum and maximum, NaN where
// either is NaN: what page bounds are made of, for the kernels that keep them
// (kv_cache.cu, kv_pages.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

namespace ra {

namespace {

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
  T v[kVec];
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ __half min_nan(__half a, __half b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __half max_nan(__half a, __half b) { return __hmax_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 min_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmin_nan(a, b); }
__device__ __forceinline__ __nv_bfloat16 max_nan(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmax_nan(a, b); }

template <typename T, int kVec>
__device__ __forceinline__ void fold(Vec<T, kVec>& lo, Vec<T, kVec>& hi, const Vec<T, kVec>& a, const Vec<T, kVec>& b) {
  if constexpr (kVec % 2 == 0 && sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      T2 l, h, x, y;
      memcpy(&l, &lo.v[2 * i], 4);
      memcpy(&h, &hi.v[2 * i], 4);
      memcpy(&x, &a.v[2 * i], 4);
      memcpy(&y, &b.v[2 * i], 4);
      l = __hmin2_nan(l, x);
      h = __hmax2_nan(h, y);
      memcpy(&lo.v[2 * i], &l, 4);
      memcpy(&hi.v[2 * i], &h, 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      lo.v[i] = min_nan(lo.v[i], a.v[i]);
      hi.v[i] = max_nan(hi.v[i], b.v[i]);
    }
  }
}

}  // namespace

}  // namespace ra
