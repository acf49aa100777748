// LayerNorm of rows of 1 to 8192 columns, forward and backward, with the gradients of its parameters.
//
//   m = mean(x), r = (mean((x - m)^2) + eps)^(-1/2), n = (x - m) r, y = n w + b
//   dx = r (h - mean(h) - n mean(h n)) with h = dy w;  dw = sum over rows of dy n;  db = sum over rows of dy
//
// Bound by memory in both directions: a row is read once, stays in the registers of its L threads and leaves once.  w, b and
// the sums of dw and db belong to columns and so to threads; they stay in registers for all rows of a persistent CTA, and the next
// row is on its way while one is worked on.  Measured: forward of 262144 x 128 fp32 to bf16 34.4 us (5.9 TB/s of 6.5 that a copy
// reaches; 40.9 without the next row on its way), backward of 4099 x 4096 bf16 19 to 20 us (24 with a cold L2) and 5 to 8 for the sums over the
// 296 parts (9.7 MB of them).  Wide rows are bound by a row's chain (load, two sums over the CTA, store) at two CTAs of 256 threads an SM: with
// eight columns a thread and scalar arithmetic 42.5, sixteen and two-wide arithmetic 28.8, and 19 to 20 once a thread's sums went out sixteen
// bytes at a time instead of four.  Rows brought by bulk copies into a ring in shared memory, three to six ahead: no gain (31.6 for 28.8).
#pragma once
#include "numeric8.cuh"

namespace b200 {

constexpr int kLayerNormMaxCols = 8192;

struct LayerNormParams {
  const void* x;
  long long x_pitch;       // elements, like the other pitches
  const void* dy;          // backward
  long long dy_pitch;
  const float* w;          // may be null
  const float* b;          // may be null
  float* mean;             // [rows]; may be null (forward)
  float* rstd;
  void* out;               // y or dx, [rows][cols]
  uint8_t* values;         // x in 8 bits: forward writes it if not null, backward reads it in x's place
  uint8_t* exponents;
  float* partial;          // backward: [grid][2][cols]; may be null
  long long rows;
  int cols;
  float eps;
};

template <int L>
constexpr int kRowThreads = L > 32 ? L : 256;
// CTAs of an SM that the backward kernel's registers leave room for: 65536 / (threads x 80 or 128).
template <int L, int NV, bool VEC>
constexpr int kGradCtas = !VEC ? 1 : L <= 32 ? (NV == 1 ? 3 : 2) : (NV == 1 ? 768 : 512) / L;

// Sums of K values over the L threads of a row.  Beyond a warp the warps meet in shared memory, `turn` in two places by turns:
// one barrier a sum.
template <int L, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*meet)[2][32], int& turn) {
#pragma unroll
  for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (L > 32) {
    constexpr int W = L / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) meet[turn][k][threadIdx.x >> 5] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (W <= 8) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&meet[turn][k][i]);
          sum += (f.x + f.y) + (f.z + f.w);
        }
        v[k] = sum;
      } else {
        v[k] = meet[turn][k][lane & (W - 1)];
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      }
    }
    turn ^= 1;
  }
}

// Columns of thread t of a row: VEC takes eight neighbours per load; otherwise neighbours go to neighbouring threads, and 32 of
// them are a checkpoint's group.
template <int L, bool VEC>
__device__ __forceinline__ int row_column(int t, int i, int e) { return VEC ? (i * L + t) * 8 + e : (i * 8 + e) * L + t; }

// A thread's part of a row as it lies in memory, so that the next row can be on its way while this one is worked on.
template <class T, int NV, bool VEC>
struct RowBits {
  static constexpr bool kWide = std::is_same<T, float>::value;
  static constexpr int W = VEC ? (kWide ? 8 : 4) : 8;
  uint32_t u[NV][W];

  template <int L>
  __device__ __forceinline__ void load(const T* row, int t, int cols) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC) {
        const int c = row_column<L, VEC>(t, i, 0);
        if (c < cols) {
          if constexpr (kWide) {
            float f[8];
            ld_global_v8(row + c, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[i][e] = __float_as_uint(f[e]);
          } else {
            const uint4 q = *reinterpret_cast<const uint4*>(row + c);
            u[i][0] = q.x, u[i][1] = q.y, u[i][2] = q.z, u[i][3] = q.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) u[i][e] = 0u;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = row_column<L, VEC>(t, i, e);
          u[i][e] = c < cols ? __float_as_uint(to_f32(row[c])) : 0u;
        }
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) u[i][e] = 0u;
  }
  __device__ __forceinline__ void unpack(float (&v)[NV][8]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC && !kWide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack2<T>(u[i][e]);
          v[i][2 * e] = f.x, v[i][2 * e + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = __uint_as_float(u[i][e]);
      }
    }
  }
};

// The same of a checkpoint's row `r`, of an activation of type T.
template <class T, int NV, bool VEC>
struct KeptBits {
  uint32_t u[NV][VEC ? 2 : 8];
  float scale[NV][VEC ? 1 : 8];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < (VEC ? 2 : 8); ++e) u[i][e] = 0u;
#pragma unroll
      for (int e = 0; e < (VEC ? 1 : 8); ++e) scale[i][e] = 0.f;
    }
  }
  template <int L>
  __device__ __forceinline__ void load(const LayerNormParams& p, long long r, int t) {
    const int groups = (p.cols + kKeepGroup - 1) / kKeepGroup;
    const uint8_t* row = p.values + r * p.cols;
    const uint8_t* byte = p.exponents + r * groups;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC) {
        const int c = row_column<L, VEC>(t, i, 0);
        u[i][0] = u[i][1] = 0u, scale[i][0] = 0.f;
        if (c < p.cols) {
          const uint2 q = *reinterpret_cast<const uint2*>(row + c);
          u[i][0] = q.x, u[i][1] = q.y;
          scale[i][0] = keep_scale(byte[c / kKeepGroup]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = row_column<L, VEC>(t, i, e);
          u[i][e] = c < p.cols ? row[c] : 0u;
          scale[i][e] = c < p.cols ? keep_scale(byte[c / kKeepGroup]) : 0.f;
        }
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[NV][8]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC) {
        kept_eight<T>(make_uint2(u[i][0], u[i][1]), scale[i][0], v[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[i][e] = kept_pair(u[i][e]).x * scale[i][e];
          if (scale[i][e] >= kTopScale<T>) v[i][e] = no_larger<T>(v[i][e]);
        }
      }
    }
  }
};

template <class T, int L, int NV, bool VEC>
__device__ __forceinline__ void store_row(T* row, int t, int cols, const float (&v)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (VEC) {
      if (row_column<L, VEC>(t, i, 0) < cols) store_eight(row + row_column<L, VEC>(t, i, 0), v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_column<L, VEC>(t, i, e);
        if (c < cols) row[c] = from_f32<T>(v[i][e]);
      }
    }
  }
}

// Whole warps call this: rows that do not exist take part in the shuffles and store nothing.
template <int L, int NV, bool VEC>
__device__ __forceinline__ void keep_row(const LayerNormParams& p, long long r, bool here, int t, const float (&v)[NV][8]) {
  const int groups = (p.cols + kKeepGroup - 1) / kKeepGroup;
  uint8_t* row = p.values + r * p.cols;
  uint8_t* bytes = p.exponents + r * groups;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (VEC) {
      const int c = row_column<L, VEC>(t, i, 0);
      bool infinite;
      uint32_t largest = largest_of(v[i], infinite);
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
      largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
      const uint32_t byte = keep_byte(largest);
      if (here && c < p.cols) {
        *reinterpret_cast<uint2*>(row + c) = keep_eight(v[i], keep_inverse(byte), infinite);
        if ((t & 3) == 0) bytes[c / kKeepGroup] = uint8_t(byte);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_column<L, VEC>(t, i, e);
        const uint32_t size = __float_as_uint(fabsf(v[i][e]));
        const uint32_t byte = keep_byte(__reduce_max_sync(0xffffffffu, size < 0x7f800000u ? size : 0u));
        if (here && c < p.cols) {
          row[c] = uint8_t(keep_pair(infinity_to_nan(v[i][e]) * keep_inverse(byte), 0.f));
          if ((t & 31) == 0) bytes[c / kKeepGroup] = uint8_t(byte);
        }
      }
    }
  }
}

template <int L, int NV, bool VEC>
__device__ __forceinline__ void load_column_values(const float* w, int t, int cols, float otherwise, float (&v)[NV][8]) {
  const bool wide = VEC && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c0 = row_column<L, VEC>(t, i, 0);
    if (wide && w && c0 < cols) {
      const float4 lo = reinterpret_cast<const float4*>(w + c0)[0], hi = reinterpret_cast<const float4*>(w + c0)[1];
      v[i][0] = lo.x, v[i][1] = lo.y, v[i][2] = lo.z, v[i][3] = lo.w, v[i][4] = hi.x, v[i][5] = hi.y, v[i][6] = hi.z, v[i][7] = hi.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_column<L, VEC>(t, i, e);
        v[i][e] = w && c < cols ? w[c] : otherwise;
      }
    }
  }
}
// A thread's eight neighbouring fp32 values, on 16 bytes.
__device__ __forceinline__ void store_sums(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// The mean is taken twice: a first one in fp32, then that of the distances from it, which are exact where the row lies far from
// zero against its width; the second corrects mean, variance and the distances.
template <class TX, class TY, int L, int NV, bool VEC>
__global__ void __launch_bounds__(kRowThreads<L>) layer_norm_kernel(LayerNormParams p) {
  pdl_wait();
  __shared__ __align__(16) float meet[2][2][32];
  constexpr int RPB = kRowThreads<L> / L;  // rows a CTA has at a time
  const int t = threadIdx.x % L;
  int turn = 0;
  float w[NV][8], b[NV][8];
  load_column_values<L, NV, VEC>(p.w, t, p.cols, 1.f, w);
  load_column_values<L, NV, VEC>(p.b, t, p.cols, 0.f, b);
  const float inv = 1.0f / float(p.cols);
  RowBits<TX, NV, VEC> bits;
  const long long step = (long long)gridDim.x * RPB;
  const long long mine = (long long)blockIdx.x * RPB + threadIdx.x / L;
  const TX* next = static_cast<const TX*>(p.x) + mine * p.x_pitch;
  bits.clear();
  if (mine < p.rows) bits.template load<L>(next, t, p.cols);
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < p.rows; r0 += step) {  // whole warps: their lanes meet in the shuffles
    const long long r = r0 + threadIdx.x / L;
    const bool here = r < p.rows;
    float v[NV][8];
    bits.unpack(v);
    next += step * p.x_pitch;
    if (r + step < p.rows) bits.template load<L>(next, t, p.cols);
    if (p.values) keep_row<L, NV, VEC>(p, r, here, t, v);
    float s[4] = {0.f, 0.f, 0.f, 0.f};  // two sums, their odd columns apart
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 2) add_f32x2(s[0], s[1], v[i][e], v[i][e + 1]);
    float first[1] = {s[0] + s[1]};
    row_sums<L, 1>(first, meet, turn);
    first[0] *= inv;
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float shift = !VEC || row_column<L, VEC>(t, i, 0) < p.cols ? -first[0] : 0.f;  // columns that do not exist stay zero
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (VEC) {
          add_f32x2(v[i][e], v[i][e + 1], shift, shift);
        } else {
          v[i][e] = row_column<L, VEC>(t, i, e) < p.cols ? v[i][e] + shift : 0.f;
          v[i][e + 1] = row_column<L, VEC>(t, i, e + 1) < p.cols ? v[i][e + 1] + shift : 0.f;
        }
        add_f32x2(s[0], s[1], v[i][e], v[i][e + 1]);
        fma_f32x2(s[2], s[3], v[i][e], v[i][e + 1], v[i][e], v[i][e + 1], s[2], s[3]);
      }
    }
    float sums[2] = {s[0] + s[1], s[2] + s[3]};
    row_sums<L, 2>(sums, meet, turn);
    const float rest = sums[0] * inv;
    const float rstd = rsqrtf(fmaxf(fmaf(-rest, rest, sums[1] * inv), 0.f) + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        add_f32x2(v[i][e], v[i][e + 1], -rest, -rest);
        mul_f32x2(v[i][e], v[i][e + 1], rstd, rstd);
        fma_f32x2(v[i][e], v[i][e + 1], v[i][e], v[i][e + 1], w[i][e], w[i][e + 1], b[i][e], b[i][e + 1]);
      }
    if (here) {
      store_row<TY, L, NV, VEC>(static_cast<TY*>(p.out) + r * p.cols, t, p.cols, v);
      if (t == 0 && p.mean) {
        p.mean[r] = first[0] + rest;
        p.rstd[r] = rstd;
      }
    }
  }
}

// x is the saved tensor itself or its 8-bit checkpoint (KEPT).
template <class TX, class TY, bool KEPT, int L, int NV, bool VEC>
__global__ void __launch_bounds__(kRowThreads<L>, kGradCtas<L, NV, VEC>) layer_norm_grad_kernel(LayerNormParams p) {
  pdl_wait();
  __shared__ __align__(16) float meet[2][2][32];
  constexpr int THREADS = kRowThreads<L>, RPB = THREADS / L;
  const int t = threadIdx.x % L;
  int turn = 0;
  float w[NV][8], dw[NV][8], db[NV][8];
  load_column_values<L, NV, VEC>(p.w, t, p.cols, 1.f, w);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = db[i][e] = 0.f;
  const float inv = 1.0f / float(p.cols);
  RowBits<TY, NV, VEC> dy_bits;
  typename std::conditional<KEPT, KeptBits<TX, NV, VEC>, RowBits<TX, NV, VEC>>::type x_bits;
  float mean = 0.f, rstd = 0.f;
  const long long step = (long long)gridDim.x * RPB;
  const TY* next_dy = static_cast<const TY*>(p.dy) + ((long long)blockIdx.x * RPB + threadIdx.x / L) * p.dy_pitch;
  const TX* next_x = static_cast<const TX*>(p.x) + ((long long)blockIdx.x * RPB + threadIdx.x / L) * p.x_pitch;
  auto fetch = [&](long long r) {
    if (r < p.rows) {
      dy_bits.template load<L>(next_dy, t, p.cols);
      if constexpr (KEPT) x_bits.template load<L>(p, r, t);
      else x_bits.template load<L>(next_x, t, p.cols);
      mean = p.mean[r], rstd = p.rstd[r];
    } else {
      dy_bits.clear();  // adds nothing to any sum
    }
    next_dy += step * p.dy_pitch;
    next_x += step * p.x_pitch;
  };
  x_bits.clear();
  fetch((long long)blockIdx.x * RPB + threadIdx.x / L);
  for (long long r0 = (long long)blockIdx.x * RPB; r0 < p.rows; r0 += step) {
    const long long r = r0 + threadIdx.x / L;
    float x[NV][8], g[NV][8];
    x_bits.unpack(x);
    dy_bits.unpack(g);
    const float shift = -mean, factor = rstd;
    if (r0 + step < p.rows) fetch(r + step);
    float s[4] = {0.f, 0.f, 0.f, 0.f};  // of h and of h n, their odd columns apart; columns that do not exist have dy = 0
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        add_f32x2(x[i][e], x[i][e + 1], shift, shift);
        mul_f32x2(x[i][e], x[i][e + 1], factor, factor);
        fma_f32x2(dw[i][e], dw[i][e + 1], g[i][e], g[i][e + 1], x[i][e], x[i][e + 1], dw[i][e], dw[i][e + 1]);
        add_f32x2(db[i][e], db[i][e + 1], g[i][e], g[i][e + 1]);
        mul_f32x2(g[i][e], g[i][e + 1], w[i][e], w[i][e + 1]);
        add_f32x2(s[0], s[1], g[i][e], g[i][e + 1]);
        fma_f32x2(s[2], s[3], g[i][e], g[i][e + 1], x[i][e], x[i][e + 1], s[2], s[3]);
      }
    float sums[2] = {s[0] + s[1], s[2] + s[3]};
    row_sums<L, 2>(sums, meet, turn);
    const float a = -sums[0] * inv, c = -sums[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        add_f32x2(g[i][e], g[i][e + 1], a, a);
        fma_f32x2(x[i][e], x[i][e + 1], x[i][e], x[i][e + 1], c, c, g[i][e], g[i][e + 1]);
        mul_f32x2(x[i][e], x[i][e + 1], factor, factor);
      }
    if (r < p.rows && p.out) store_row<TX, L, NV, VEC>(static_cast<TX*>(p.out) + r * p.cols, t, p.cols, x);
  }
  if (!p.partial) return;
  float* mine = p.partial + (long long)blockIdx.x * 2 * p.cols;
  if constexpr (L > 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (VEC) {
        const int c = row_column<L, VEC>(t, i, 0);
        if (c < p.cols) store_sums(mine + c, dw[i]), store_sums(mine + p.cols + c, db[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = row_column<L, VEC>(t, i, e);
          if (c < p.cols) mine[c] = dw[i][e], mine[p.cols + c] = db[i][e];
        }
      }
    }
  } else {
    // The rows that the CTA's warps have had, added up in a fixed order.
    __shared__ float sums[THREADS / 32][L * NV * 8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float(&v)[NV][8] = half ? db : dw;
#pragma unroll
      for (int o = 16; o >= L; o >>= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] += __shfl_xor_sync(0xffffffffu, v[i][e], o);
      if ((threadIdx.x & 31) < L) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) sums[threadIdx.x >> 5][row_column<L, VEC>(t, i, e)] = v[i][e];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < p.cols; c += THREADS) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < THREADS / 32; ++k) s += sums[k][c];
        mine[half * p.cols + c] = s;
      }
      __syncthreads();
    }
  }
}

// out[c] = sum over the parts of partial[part][c], for the concatenation of up to two outputs: the gradients' last step.  V (4, or 1
// for odd widths) neighbouring columns a thread; a CTA has `across` threads side by side, the others take the parts in turn, and the
// order goes by the sizes alone.
struct PartSumParams {
  const float* partial;    // [parts][width]
  int parts, across;
  long long width, split;  // columns from `split` on go to the second output
  void* out[2];            // either may be null
  int dtype[2];
};

template <int V>
__global__ void __launch_bounds__(256) part_sum_kernel(PartSumParams p) {
  pdl_wait();
  __shared__ float sums[256][V];
  const int x = threadIdx.x % p.across, y = threadIdx.x / p.across, down = 256 / p.across;
  const long long c = ((long long)blockIdx.x * p.across + x) * V;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (c < p.width) {
#pragma unroll 8
    for (int k = y; k < p.parts; k += down) {
      if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p.partial + k * p.width + c);
        s[0] += f.x, s[1] += f.y, s[2] += f.z, s[3] += f.w;
      } else {
        s[0] += p.partial[k * p.width + c];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sums[threadIdx.x][e] = s[e];
  for (int half = down / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (y < half) {
#pragma unroll
      for (int e = 0; e < V; ++e) sums[threadIdx.x][e] += sums[threadIdx.x + half * p.across][e];
    }
  }
  if (y || c >= p.width) return;
  const int which = c >= p.split;  // a multiple of V
  const long long at = c - which * p.split;
  if (!p.out[which]) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float v = sums[threadIdx.x][e];
    if (p.dtype[which] == B200_DTYPE_F32) static_cast<float*>(p.out[which])[at + e] = v;
    else if (p.dtype[which] == B200_DTYPE_BF16) static_cast<__nv_bfloat16*>(p.out[which])[at + e] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p.out[which])[at + e] = __float2half_rn(v);
  }
}

}  // namespace b200
