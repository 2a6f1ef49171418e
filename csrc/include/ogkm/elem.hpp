// Element types of the 16-bit kernels: 8-wide vectors and conversions to and
// from f32 (round to nearest even; gfx950 converts both types in hardware).
// Device code only.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ogkm {

template <typename T>
struct Vec {
  typedef T v8 __attribute__((ext_vector_type(8)));
  typedef T v4 __attribute__((ext_vector_type(4)));
  typedef T v2 __attribute__((ext_vector_type(2)));
};
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return (T)x;
}

}  // namespace ogkm
