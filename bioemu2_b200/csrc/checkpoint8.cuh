// Activation checkpoints in 8 bits: written from and read back as rows of fp32, bf16 or fp16 (the form is in numeric8.cuh).
#pragma once
#include "numeric8.cuh"

namespace b200 {

struct KeepParams {
  const void* x;           // [rows][pitch], `cols` of each row
  long long pitch;         // elements
  uint8_t* values;         // [rows][cols] e4m3
  uint8_t* exponents;      // [rows][groups]
  void* out;               // [rows][cols], of the restored type
  long long rows;
  int cols, groups;        // groups = cols / 32, rounded up
};

// A thread takes eight neighbours, four threads a group; the byte is one shuffle maximum away.  Bound by memory: 1 + 1/32 bytes
// per element beside the activation's own.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) keep_kernel(KeepParams p) {
  pdl_wait();
  const long long total = p.rows * p.groups * 4;
  const long long stride = (long long)gridDim.x * blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  // whole warps stay in the loop: their lanes meet in the shuffles
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; (i & ~31ll) < total; i += stride) {
    const bool here = i < total;
    const long long group = here ? i >> 2 : 0;
    const long long row = group / p.groups;
    const int g = int(group - row * p.groups);
    const int c0 = g * kKeepGroup + int(i & 3) * 8;
    float v[8];
    if (VEC) {
      if (here && c0 < p.cols) {
        load_eight(x + row * p.pitch + c0, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = here && c0 + e < p.cols ? to_f32(x[row * p.pitch + c0 + e]) : 0.f;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) largest = max(largest, finite_magnitude(v[e]));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    const uint32_t byte = keep_byte(largest);
    const uint2 q = keep_eight(v, keep_inverse(byte));
    if (here) {
      if ((i & 3) == 0) p.exponents[group] = uint8_t(byte);
      uint8_t* dst = p.values + row * p.cols + c0;
      if (VEC) {
        if (c0 < p.cols) *reinterpret_cast<uint2*>(dst) = q;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e < p.cols) dst[e] = uint8_t((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
      }
    }
  }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(256) restore_kernel(KeepParams p) {
  pdl_wait();
  const long long total = p.rows * p.groups * 4;
  const long long stride = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    const long long group = i >> 2, row = group / p.groups;
    const int c0 = int(group - row * p.groups) * kKeepGroup + int(i & 3) * 8;
    if (c0 >= p.cols) continue;
    const float scale = keep_scale(p.exponents[group]);
    const uint8_t* src = p.values + row * p.cols + c0;
    T* out = static_cast<T*>(p.out) + row * p.cols + c0;
    uint2 q = make_uint2(0, 0);
    if (VEC) {
      q = *reinterpret_cast<const uint2*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < p.cols) (e < 4 ? q.x : q.y) |= uint32_t(src[e]) << (8 * (e & 3));
    }
    float v[8];
    kept_eight(q, scale, v);
    if (VEC) {
      store_eight(out, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < p.cols) out[e] = from_f32<T>(v[e]);
    }
  }
}

}  // namespace b200
