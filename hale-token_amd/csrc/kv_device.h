// kv_device.h -- device helpers of the rotary and key/value cache kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "hale_device.h"

namespace hale {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // at any float's address

// A bf16 number: the upper half of an f32.
struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(Bf16 v) { return __uint_as_float((unsigned)v.bits << 16); }

// Rounded to nearest even; a NaN stays one.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) {
  asm volatile("" : "+v"(v));  // a rounded f32 first: no product is rounded straight to f16
  return (_Float16)v;
}
template <> __device__ __forceinline__ Bf16 from_f32<Bf16>(float v) {
  // by its bits: the attention's unit is compiled without comparisons of NaNs
  const unsigned u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return {(uint16_t)((u >> 16) | 0x40)};
  return {(uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16)};
}

// cos and sin, times factor, of the angle that position `pos` has at `turns`
// turns per position.
__device__ __forceinline__ void rope_angle(int pos, double turns, float factor, float* c, float* s) {
  const double t = (double)pos * turns;
  const float f = 2.0f * (float)(t - rint(t));  // half turns in [-1, 1]
  *c = cospif(f) * factor;
  *s = sinpif(f) * factor;
}

}  // namespace hale
