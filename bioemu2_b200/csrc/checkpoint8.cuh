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

// How the rows lie: one after the other in whole groups (an element is its number times eight away), or with a pitch or a shorter
// last group of their own, eight neighbours at a time or, where those are not on their boundary, one.
enum KeepRows : int { kKeepFlat = 0, kKeepVector = 1, kKeepScalar = 2 };

// Group i / 4 and the eight columns of it that are thread i's.
struct KeepPlace {
  long long row;
  int col;
};
__device__ __forceinline__ KeepPlace keep_place(long long i, int groups) {
  const long long group = i >> 2;
  long long row;
  if (group < (1ll << 32)) row = uint32_t(group) / uint32_t(groups);  // a 64-bit division takes as long as all the rest
  else row = group / groups;
  return {row, int(group - row * groups) * kKeepGroup + int(i & 3) * 8};
}

// A thread takes eight neighbours, four threads a group; the byte is two shuffles away.  Bound by memory, 1 + 1/32 bytes per element
// beside the activation's own: 262144 x 128 fp32 written in 24.1 us and read back in 25.0 (7.0 and 6.7 TB/s, part of it from the L2), 41209 x
// 512 bf16 in 13.9 and 15.0.  With a 64-bit division for the row and a test of each value for infinity instead of one for the eight:
// 29.8 and 26.2, 20.6 and 18.1.
template <class T, int ROWS>
__global__ void __launch_bounds__(256) keep_kernel(KeepParams p) {
  pdl_wait();
  const long long total = p.rows * p.groups * 4;
  const long long stride = (long long)gridDim.x * blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  // whole warps stay in the loop: their lanes meet in the shuffles
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; (i & ~31ll) < total; i += stride) {
    const bool here = i < total;
    KeepPlace at = {0, 0};
    if (ROWS != kKeepFlat) at = keep_place(here ? i : 0, p.groups);
    const bool some = here && (ROWS == kKeepFlat || at.col < p.cols);
    float v[8];
    if (ROWS != kKeepScalar) {
      if (some) {
        load_eight(x + (ROWS == kKeepFlat ? i * 8 : at.row * p.pitch + at.col), v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = here && at.col + e < p.cols ? to_f32(x[at.row * p.pitch + at.col + e]) : 0.f;
    }
    bool infinite;
    uint32_t largest = largest_of(v, infinite);
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    const uint32_t byte = keep_byte(largest);
    const uint2 q = keep_eight(v, keep_inverse(byte), infinite);
    if (here && (i & 3) == 0) p.exponents[i >> 2] = uint8_t(byte);
    if (some) {
      uint8_t* dst = p.values + (ROWS == kKeepFlat ? i * 8 : at.row * p.cols + at.col);
      if (ROWS != kKeepScalar) {
        *reinterpret_cast<uint2*>(dst) = q;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at.col + e < p.cols) dst[e] = uint8_t((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
      }
    }
  }
}

template <class T, int ROWS>
__global__ void __launch_bounds__(256) restore_kernel(KeepParams p) {
  pdl_wait();
  const long long total = p.rows * p.groups * 4;
  const long long stride = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += stride) {
    int left = 8;  // columns of the thread's eight that exist
    long long offset = i * 8;
    if (ROWS != kKeepFlat) {
      const KeepPlace at = keep_place(i, p.groups);
      left = p.cols - at.col;
      offset = at.row * p.cols + at.col;
      if (left <= 0) continue;
    }
    const float scale = keep_scale(p.exponents[i >> 2]);
    const uint8_t* src = p.values + offset;
    T* out = static_cast<T*>(p.out) + offset;
    uint2 q = make_uint2(0, 0);
    if (ROWS != kKeepScalar) {
      q = *reinterpret_cast<const uint2*>(src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) (e < 4 ? q.x : q.y) |= uint32_t(src[e]) << (8 * (e & 3));
    }
    float v[8];
    kept_eight<T>(q, scale, v);
    if (ROWS != kKeepScalar) {
      store_eight(out, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) out[e] = from_f32<T>(v[e]);
    }
  }
}

}  // namespace b200
