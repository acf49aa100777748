// Rows of fp32, bf16 and fp16 in groups of eight neighbours, and the 8-bit form of an activation checkpoint.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "row_tile.cuh"

namespace b200 {

// ---------------------------------------------------------------------------
// Eight neighbours of one row, as fp32.  VEC: one load of 32 (fp32) or 16 bytes on its own boundary; otherwise element
// by element, `step` apart, the last ones possibly beyond the row's end.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(h);
}
__device__ __forceinline__ float2 unpack_f16x2(uint32_t u) { return __half22float2(reinterpret_cast<const __half2&>(u)); }

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) return pack_f16x2(lo, hi);
  else return pack_bf16x2(lo, hi);
}
template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value) return unpack_f16x2(u);
  else return make_float2(bf16lo(u), bf16hi(u));
}

template <class T>
__device__ __forceinline__ void load_eight(const T* p, float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    ld_global_v8(p, x);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}
template <class T>
__device__ __forceinline__ void store_eight(T* p, const float (&x)[8]) {
  if constexpr (std::is_same<T, float>::value) st_global_v8(p, x);
  else
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// ---------------------------------------------------------------------------
// Checkpoints in 8 bits.  A group of 32 neighbours of a row shares the power of two 2^e, e = byte - 127 >= -127 the least
// with which its largest finite magnitude is at most 448 * 2^e; a value is kept as e4m3(x * 2^-e).  A power of two leaves
// the quotient exact, so the one rounding is the conversion's, and the same on any machine.  e4m3 has no infinity: infinities
// are kept as NaN, like NaN itself.
//
// A magnitude in the last 1/32 of its type's last binade rounds up to a power of two that the type does not have (fp16: 63488 and more
// to 65536).  What is finite comes back finite: as T's largest value, in every place that expands a checkpoint to T.
// ---------------------------------------------------------------------------
constexpr int kKeepGroup = 32;
template <class T>
constexpr float kLargest = std::is_same<T, __half>::value ? 65504.0f : std::is_same<T, float>::value ? 0x1.fffffep127f : 0x1.fep127f;
// The least power of two with which a kept value (448 at most) may be beyond that: 448 * 2^7 and 448 * 2^119 are not.  Only groups that
// reach it look at their values: the expansion's cost is one comparison for eight of them.
template <class T>
constexpr float kTopScale = std::is_same<T, __half>::value ? 0x1p8f : 0x1p120f;
template <class T>
__device__ __forceinline__ float no_larger(float x) {  // keeps NaN
  asm("min.NaN.f32 %0, %0, %1;\n\tmax.NaN.f32 %0, %0, %2;" : "+f"(x) : "f"(kLargest<T>), "f"(-kLargest<T>));
  return x;
}

// The largest finite magnitude of eight values, as its bits.  NaN never is the larger one of two.
__device__ __forceinline__ uint32_t largest_of(const float (&x)[8], bool& infinite) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
  infinite = m == INFINITY;
  if (infinite) {
    m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fabsf(x[e]) < INFINITY ? fmaxf(m, fabsf(x[e])) : m;
  }
  return __float_as_uint(m);
}
// The byte of a group whose largest magnitude has these bits: 1.m * 2^p is at most 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ uint32_t keep_byte(uint32_t largest) {
  const int e = int(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);
  return uint32_t(e > 0 ? e : 0);
}
__device__ __forceinline__ float keep_scale(uint32_t byte) {  // 2^e; byte 0 is the subnormal 2^-127
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ float keep_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

__device__ __forceinline__ uint32_t keep_pair(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float infinity_to_nan(float x) { return isinf(x) ? __uint_as_float(0x7fffffffu) : x; }
__device__ __forceinline__ uint2 keep_eight(const float (&x)[8], float inverse, bool infinite) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = keep_pair(x[2 * i] * inverse, x[2 * i + 1] * inverse);
  if (infinite) {  // the conversion would make them 448
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = keep_pair(infinity_to_nan(x[2 * i]) * inverse, infinity_to_nan(x[2 * i + 1]) * inverse);
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
__device__ __forceinline__ float2 kept_pair(uint32_t two) {  // e4m3 values are fp16 values
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}
// Eight kept values as fp32, none of them beyond T's largest.
template <class T>
__device__ __forceinline__ void kept_eight(uint2 u, float scale, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.x >> 16, u.y, u.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = kept_pair(w[i]);
    x[2 * i] = f.x * scale, x[2 * i + 1] = f.y * scale;
  }
  if (scale >= kTopScale<T>) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = no_larger<T>(x[e]);
  }
}

}  // namespace b200
