// The linear layer y = act(x w^T + b) + residual and the products of its backward pass, bf16 or fp16 operands with fp32
// accumulation in tensor memory:
//
//   forward   y  [rows][n] = x [rows][k] . w [n][k]^T     both operands have the contraction along their rows (K-major)
//   backward  dx [rows][k] = d [rows][n] . w [n][k]       w has it across them (MN-major)
//             dw [n][k]    = d [rows][n]^T . x [rows][k]  so have both
//
// with d = dy act'(a), a the value before the activation.  d is made in fp32 and rounded to the operands' type for the two products, whose
// instruction takes both operands in one 16-bit type; db is summed before that.  Against 64 bits dx and dw are then off by 0.0023 of their
// norm in bf16 and 0.00029 in fp16, where the one rounding of the output leaves 0.0017 and 0.00021 (two independent roundings: the
// square root of two).  d as a sum of two 16-bit terms would keep that and double the products and d's shared memory.
//
// The shared-memory descriptors take either order, so nothing is transposed on the way.  Persistent kernel, one CTA per SM, 128 x BN tiles:
//   warp 0       TMA producer, K slabs of 64 through a ring in shared memory
//   warp 1       MMA issuer, two accumulators in tensor memory
//   warps 2..17  epilogue: four groups of four warps, which take the tile's 32-column pieces in turn; a warp stages its 32 rows of
//                a piece in a set of its own and sends them off by TMA without meeting the other warps.  (Two groups with
//                64-column pieces: the forward pass of 147456 rows 128 -> 512, silu and saved value, 97 us, two warps a scheduler
//                that wait for their own instructions, 1.4 a clock.)
// Measured: forward of 147456 rows 128 -> 512 with silu and the saved value 70 us (340 MB, 4.8 TB/s; the epilogue's chain: tensor memory,
// activation, staging, stores), of 41209 rows 512 -> 128 with an fp32 residual 18 to 20 us (27 with the residual read by the lanes, a row
// each); dx of 8192 rows 4096 -> 1024 67 us and dw 65 us (1.0 PFLOP/s; the tensor pipe is 49 % active: a 128 x 256 tile writes and
// reads 96 KB of shared memory for every 512 clocks of products, and that takes 768).
#pragma once
#include "numeric8.cuh"

namespace b200 {

enum LinearAct : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

struct LinearParams {
  int m, n;                // rows and columns of the output
  int tiles_m, tiles_n;
  int k_blocks;            // the contraction in blocks of 64, rounded up (TMA fills the rest with zeros)
  int splits;              // parts of the contraction, each with an output plane of its own
  int stages;              // of the operand ring
  int sets, set_bytes;     // staging sets of an epilogue warp (1 or 2): the output's piece, 2 or 4 KB, and behind it the saved value's
  uint32_t idesc;
  int act;
  int out_f32;             // type of the output (and of the residual); otherwise that of the operands
  int save;                // store the value before the activation too: 1 as the operands' type, 2 as fp32
  const float* bias;       // [n]; may be null
  int residual;            // add the tiles of the residual's map
  const uint8_t* values;   // KEPT: b's rows in 8 bits, [k][n], and their exponents
  const uint8_t* exponents;
  int k;                   // length of the contraction
};

// ---------------------------------------------------------------------------
// Activations and their slopes
// ---------------------------------------------------------------------------
// Both by the hardware's exponential and reciprocal (2^-22 of their values), two values at a time: an epilogue or a gradient pass of
// two operands has about fifteen instructions an element before the issue slots, not the memory, bound it (silu by expf and a
// division: the gradient of 147456 x 512 values 110 us, 4.1 TB/s), and two special-function operations an element before that pipe
// does, so two values share a reciprocal.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluTanhQ = 0.044715f;

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x and 1 / y by one reciprocal, for values of 1 to 2^63 each.
__device__ __forceinline__ void rcp_two(float& x, float& y) {
  const float r = rcp_approx(x * y), t = x;
  x = r * y;
  y = r * t;
}
// sigmoid of the two values whose product with -log2(e) is given.  The exponent is kept below 60, which leaves a sigmoid of 2^-60 for
// what lies beyond; a NaN gives a number here, so that it stays with its own element, and comes back with the factor a.  That
// factor is kept to 41.5 where its product with the rest is nothing (silu below, all slopes on both sides): 41.5 x 2^-60 for a
// value of any size, and no infinity times zero.
__device__ __forceinline__ float at_least(float a) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(-41.5f));
  return y;
}
__device__ __forceinline__ float within(float a) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(at_least(a)), "f"(41.5f));
  return y;
}
__device__ __forceinline__ void sigmoid_two(float& x0, float& x1) {
  x0 = exp2_approx(fminf(x0, 60.0f)), x1 = exp2_approx(fminf(x1, 60.0f));
  add_f32x2(x0, x1, 1.0f, 1.0f);
  rcp_two(x0, x1);
}

// The normal distribution's Phi(a) and phi(a).  Phi(-|a|) = poly(t) exp(-a^2 / 2) / 2 with t = 1 / (1 + p |a| / sqrt(2)): the
// rational approximation 7.1.26 of M. Abramowitz and I. Stegun, "Handbook of Mathematical Functions" (C. Hastings, 1955), off by 0.75e-7
// at most.  It shares its exponential with phi.
__device__ __forceinline__ void normal_cdf_two(float a0, float a1, float& c0, float& c1, float& f0, float& f1) {
  float t0 = fminf(fabsf(a0), 64.0f), t1 = fminf(fabsf(a1), 64.0f);
  fma_f32x2(t0, t1, t0, t1, 0.3275911f * 0.70710678118654752f, 0.3275911f * 0.70710678118654752f, 1.0f, 1.0f);
  rcp_two(t0, t1);
  mul_f32x2(f0 = a0, f1 = a1, a0, a1);
  mul_f32x2(f0, f1, -0.5f * kLog2e, -0.5f * kLog2e);
  f0 = exp2_approx(f0), f1 = exp2_approx(f1);
  float q0, q1;
  fma_f32x2(q0, q1, t0, t1, 1.061405429f, 1.061405429f, -1.453152027f, -1.453152027f);
  fma_f32x2(q0, q1, t0, t1, q0, q1, 1.421413741f, 1.421413741f);
  fma_f32x2(q0, q1, t0, t1, q0, q1, -0.284496736f, -0.284496736f);
  fma_f32x2(q0, q1, t0, t1, q0, q1, 0.254829592f, 0.254829592f);
  mul_f32x2(t0, t1, f0, f1);
  mul_f32x2(t0, t1, 0.5f, 0.5f);
  mul_f32x2(q0, q1, t0, t1);
  c0 = a0 < 0.f ? q0 : 1.0f - q0;
  c1 = a1 < 0.f ? q1 : 1.0f - q1;
  mul_f32x2(f0, f1, 0.3989422804014327f, 0.3989422804014327f);
}
// The argument of gelu_tanh's sigmoid times -log2(e).
__device__ __forceinline__ void gelu_tanh_argument(float a0, float a1, float& x0, float& x1) {
  constexpr float c = -2.0f * kLog2e * kGeluTanhC;
  x0 = a0, x1 = a1;
  mul_f32x2(x0, x1, a0, a1);
  fma_f32x2(x0, x1, x0, x1, c * kGeluTanhQ, c * kGeluTanhQ, c, c);
  mul_f32x2(x0, x1, a0, a1);
}

template <int ACT>
__device__ __forceinline__ void activate_two(float& a0, float& a1) {
  if constexpr (ACT == kActRelu) {
    a0 = a0 < 0.f ? 0.f : a0, a1 = a1 < 0.f ? 0.f : a1;  // keeps NaN
  } else if constexpr (ACT == kActGelu) {
    float c0, c1, f0, f1;
    normal_cdf_two(a0, a1, c0, c1, f0, f1);
    a0 = at_least(a0), a1 = at_least(a1);
    mul_f32x2(a0, a1, c0, c1);
  } else if constexpr (ACT != kActNone) {
    float x0 = a0, x1 = a1;
    if constexpr (ACT == kActGeluTanh) gelu_tanh_argument(a0, a1, x0, x1);
    else mul_f32x2(x0, x1, -kLog2e, -kLog2e);
    sigmoid_two(x0, x1);
    a0 = at_least(a0), a1 = at_least(a1);
    mul_f32x2(a0, a1, x0, x1);
  }
}
template <int ACT>
__device__ __forceinline__ void activate_all(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) activate_two<ACT>(v[i], v[i + 1]);
}

// d0, d1 times the slopes at a0, a1.
template <int ACT>
__device__ __forceinline__ void times_slope(float a0, float a1, float& d0, float& d1) {
  if constexpr (ACT == kActRelu) {
    d0 *= a0 > 0.f ? 1.f : a0 <= 0.f ? 0.f : a0, d1 *= a1 > 0.f ? 1.f : a1 <= 0.f ? 0.f : a1;  // NaN stays
  } else if constexpr (ACT == kActGelu) {
    float c0, c1, f0, f1;
    normal_cdf_two(a0, a1, c0, c1, f0, f1);
    fma_f32x2(c0, c1, within(a0), within(a1), f0, f1, c0, c1);
    mul_f32x2(d0, d1, c0, c1);
  } else if constexpr (ACT != kActNone) {
    a0 = within(a0), a1 = within(a1);
    float s0 = a0, s1 = a1, t0 = a0, t1 = a1, u0, u1;
    if constexpr (ACT == kActGeluTanh) gelu_tanh_argument(a0, a1, s0, s1);
    else mul_f32x2(s0, s1, -kLog2e, -kLog2e);
    sigmoid_two(s0, s1);
    mul_f32x2(t0, t1, s0, s1);                            // a s
    fma_f32x2(u0, u1, s0, s1, -1.0f, -1.0f, 1.0f, 1.0f);  // 1 - s
    mul_f32x2(t0, t1, u0, u1);
    if constexpr (ACT == kActGeluTanh) {
      constexpr float c = 2.0f * kGeluTanhC;
      mul_f32x2(u0 = a0, u1 = a1, a0, a1);
      fma_f32x2(u0, u1, u0, u1, 3.0f * c * kGeluTanhQ, 3.0f * c * kGeluTanhQ, c, c);
      fma_f32x2(s0, s1, t0, t1, u0, u1, s0, s1);
    } else {
      add_f32x2(s0, s1, t0, t1);
    }
    mul_f32x2(d0, d1, s0, s1);
  }
}
template <int ACT, int R>
__device__ __forceinline__ void slope_pairs(const float (&a)[R][8], float (&d)[R][8]) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < 8; e += 2) times_slope<ACT>(a[r][e], a[r][e + 1], d[r][e], d[r][e + 1]);
}

// Eight neighbours of fp32 or of T, on 16 bytes either way.
template <class T>
__device__ __forceinline__ void load_eight_of(const void* p, int f32, long long at, float (&x)[8]) {
  if (f32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 lo = s[0], hi = s[1];
    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
  } else {
    load_eight(static_cast<const T*>(p) + at, x);
  }
}

// Byte offset of 16-byte chunk `chunk` (0..3) of row `row` in a 64B-swizzled tile of 64-byte rows.
__device__ __forceinline__ uint32_t sw64_offset(uint32_t row, uint32_t chunk) { return row * 64u + ((chunk ^ ((row >> 1) & 3u)) << 4); }

// 32 values of a lane's row of a staging piece: 64 bytes of T or 128 of fp32, as TMA wants them.
template <class T>
__device__ __forceinline__ void stage_piece(uint8_t* s, int row, int f32, const float (&v)[32]) {
  if (f32) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4*>(s + sw128_offset(row, q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4*>(s + sw64_offset(row, q)) = make_uint4(pack2<T>(v[8 * q], v[8 * q + 1]), pack2<T>(v[8 * q + 2], v[8 * q + 3]),
                                                                    pack2<T>(v[8 * q + 4], v[8 * q + 5]), pack2<T>(v[8 * q + 6], v[8 * q + 7]));
  }
}
template <class T>
__device__ __forceinline__ void add_piece(const uint8_t* s, int row, int f32, float (&v)[32]) {
  if (f32) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 f = *reinterpret_cast<const float4*>(s + sw128_offset(row, q));
      add_f32x2(v[4 * q], v[4 * q + 1], f.x, f.y);
      add_f32x2(v[4 * q + 2], v[4 * q + 3], f.z, f.w);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 u = *reinterpret_cast<const uint4*>(s + sw64_offset(row, q));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<T>(w[e]);
        add_f32x2(v[8 * q + 2 * e], v[8 * q + 2 * e + 1], f.x, f.y);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------
template <int BN>
struct LinearCfg {
  static constexpr uint32_t A_BYTES = 128 * 64 * 2, B_BYTES = BN * 64 * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int EPILOGUE_WARPS = 16, THREADS = 64 + 32 * EPILOGUE_WARPS, MAX_STAGES = 8;
  static constexpr uint32_t HEAD_BYTES = 1024 + EPILOGUE_WARPS * 128;  // barriers, and a piece's bias for each epilogue warp
  static constexpr uint32_t smem_bytes(int stages, uint32_t staging) { return HEAD_BYTES + stages * STAGE_BYTES + EPILOGUE_WARPS * staging + 1024; }
};

// KEPT: b is an 8-bit checkpoint (of an operand across its rows); the epilogue's warps, which would wait for the products, expand its
// slabs into the ring.  (Expanded into memory first: 41209 rows, dw of 512 x 128, 15 us for that and as much again for the product.)
template <class T, bool A_MN, bool B_MN, int BN, bool KEPT>
__global__ void __launch_bounds__(LinearCfg<BN>::THREADS, 1)
linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmSave,
              const __grid_constant__ CUtensorMap tmResidual, LinearParams p) {
  using Cfg = LinearCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + Cfg::MAX_STAGES;
  uint64_t* acc_full = empty + Cfg::MAX_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* residual_full = acc_empty + 2;  // of each epilogue warp's two sets of staging tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(residual_full + 2 * Cfg::EPILOGUE_WARPS);
  uint8_t* ring = smem + Cfg::HEAD_BYTES;
  uint8_t* staging = ring + p.stages * Cfg::STAGE_BYTES;

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const int tiles = p.tiles_m * p.tiles_n;
  const int items = tiles * p.splits;
  auto first_block = [&](int split) { return int((long long)p.k_blocks * split / p.splits); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], KEPT ? 1 + Cfg::EPILOGUE_WARPS : 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 32 * Cfg::EPILOGUE_WARPS);
    }
    if (p.residual)
      for (int i = 0; i < 2 * Cfg::EPILOGUE_WARPS; ++i) mbar_init(&residual_full[i], 1);
    fence_mbar_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmY);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int split = item / tiles, tile = item - split * tiles;
        const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
        const int last = first_block(split + 1);
        for (int kb = first_block(split); kb < last; ++kb) {
          mbar_wait(&empty[stage], phase ^ 1, 90);
          uint8_t* sa = ring + stage * Cfg::STAGE_BYTES;
          uint8_t* sb = sa + Cfg::A_BYTES;
          mbar_arrive_expect_tx(&full[stage], KEPT ? Cfg::A_BYTES : Cfg::STAGE_BYTES);
          if constexpr (A_MN) {
            tma_load_2d(sa, &tmA, &full[stage], tm * 128, kb * 64);
            tma_load_2d(sa + 8192, &tmA, &full[stage], tm * 128 + 64, kb * 64);
          } else {
            tma_load_2d(sa, &tmA, &full[stage], kb * 64, tm * 128);
          }
          if constexpr (KEPT) {
          } else if constexpr (B_MN) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) tma_load_2d(sb + j * 8192, &tmB, &full[stage], tn * BN + j * 64, kb * 64);
          } else {
            tma_load_2d(sb, &tmB, &full[stage], kb * 64, tn * BN);
          }
          if (++stage == p.stages) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // An MN-major operand is 64-element columns of 64 k rows (8 KB each): a K step of 16 is 2048 bytes on, the next 64 elements
    // 8192.  A K-major one has 128-byte rows of 64 k: a step is 32 bytes on.
    const bool leader = elect_one();
    int stage = 0, it = 0;
    uint32_t phase = 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x, ++it) {
      const int split = item / tiles, acc = it & 1;
      const int begin = first_block(split), last = first_block(split + 1);
      mbar_wait(&acc_empty[acc], ((it >> 1) & 1) ^ 1, 91);
      tc_fence_after_sync();
      const uint32_t d_tmem = tmem_base + acc * BN;
      for (int kb = begin; kb < last; ++kb) {
        mbar_wait(&full[stage], phase, 92);
        tc_fence_after_sync();
        const uint32_t sa = smem_u32(ring + stage * Cfg::STAGE_BYTES);
        const uint32_t a_lo = desc_lo(sa, A_MN ? 8192 : 16), b_lo = desc_lo(sa + Cfg::A_BYTES, B_MN ? 8192 : 16);
        if (leader) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16_ss2(d_tmem, a_lo + k * (A_MN ? 128 : 2), kDescHiSw128, b_lo + k * (B_MN ? 128 : 2), kDescHiSw128, p.idesc,
                          kb != begin || k != 0);
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == p.stages) stage = 0, phase ^= 1;
      }
      if (leader) umma_commit(&acc_full[acc]);
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3;  // tensor-memory lanes this warp may read: 32 * quarter ..
    const int group = (warp - 2) >> 2;
    constexpr int PIECES = BN / 32;
    constexpr int ROUNDS = (PIECES + 3) / 4;  // pieces of a group
    float* bias = reinterpret_cast<float*>(smem + 1024) + (warp - 2) * 32;
    uint8_t* mine = staging + (warp - 2) * p.sets * p.set_bytes;
    uint64_t* arrived = residual_full + (warp - 2) * 2;
    const uint32_t piece_bytes = p.out_f32 ? 4096 : 2048;
    int it = 0, set = 0;
    uint32_t residual_phase = 0;  // bit s: parity of set s
    // A piece's stores are one bulk group.  The residual comes into the output's place in a set: of two sets while the piece before is
    // worked on, of one when that piece has left.
    auto fetch_residual = [&](int s, int item, int piece) {
      if (lane == 0 && item < items) {
        tma_store_wait_read0();  // the piece before this one has left the set
        const int tile = item % tiles, tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
        mbar_arrive_expect_tx(&arrived[s], piece_bytes);
        tma_load_2d(mine + s * p.set_bytes, &tmResidual, &arrived[s], tn * BN + piece * 32, tm * 128 + quarter * 32);
      }
      __syncwarp();
    };
    if (p.residual && group < PIECES) fetch_residual(0, blockIdx.x, group);
    // KEPT: vectors of eight of a slab of 64 rows, those of the next slabs on their way
    constexpr int VECTORS = KEPT ? 64 * BN / 8 / (32 * Cfg::EPILOGUE_WARPS) : 1, AHEAD = KEPT ? (BN == 256 ? 2 : 4) : 1;
    uint2 kept[AHEAD][VECTORS];
    uint32_t byte[AHEAD][VECTORS];
    int stage = 0;
    uint32_t phase = 0;
    auto fetch_kept = [&](int a, int kb, int tn) {
      const int groups = (p.n + kKeepGroup - 1) / kKeepGroup;
#pragma unroll
      for (int j = 0; j < VECTORS; ++j) {
        const int v = (warp - 2) * 32 + lane + j * 32 * Cfg::EPILOGUE_WARPS;
        const long long row = (long long)kb * 64 + v / (BN / 8);
        const int col = tn * BN + v % (BN / 8) * 8;
        kept[a][j] = make_uint2(0, 0), byte[a][j] = 0;
        if (row < p.k && col < p.n) {
          kept[a][j] = *reinterpret_cast<const uint2*>(p.values + row * p.n + col);
          byte[a][j] = p.exponents[row * groups + col / kKeepGroup];
        }
      }
    };
    for (int item = blockIdx.x; item < items; item += gridDim.x, ++it) {
      const int split = item / tiles, tile = item - split * tiles;
      const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
      const int acc = it & 1;
      const int row0 = tm * 128 + quarter * 32;
      if constexpr (KEPT) {
        const int begin = first_block(split), last = first_block(split + 1);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) fetch_kept(a, begin + a, tn);  // slabs of the next part too: they exist, or are zeros
        for (int kb = begin; kb < last; kb += AHEAD) {
#pragma unroll
          for (int a = 0; a < AHEAD; ++a) {
            if (kb + a >= last) break;
            mbar_wait(&empty[stage], phase ^ 1, 95);
            uint8_t* sb = ring + stage * Cfg::STAGE_BYTES + Cfg::A_BYTES;
#pragma unroll
            for (int j = 0; j < VECTORS; ++j) {
              const int v = (warp - 2) * 32 + lane + j * 32 * Cfg::EPILOGUE_WARPS;
              const int c8 = v % (BN / 8);
              float f[8];
              kept_eight<T>(kept[a][j], keep_scale(byte[a][j]), f);
              *reinterpret_cast<uint4*>(sb + (c8 >> 3) * 8192 + sw128_offset(v / (BN / 8), c8 & 7)) =
                  make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
            }
            fetch_kept(a, kb + a + AHEAD, tn);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
            if (++stage == p.stages) stage = 0, phase ^= 1;
          }
        }
      }
      float bias_next[ROUNDS];  // of the group's pieces, column `lane` of each: on its way while the product is waited for
      if (p.bias) {
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
          const int col = tn * BN + (group + 4 * i) * 32 + lane;
          bias_next[i] = col < p.n && group + 4 * i < PIECES ? p.bias[col] : 0.f;
        }
      }
      mbar_wait(&acc_full[acc], (it >> 1) & 1, 93);
      tc_fence_after_sync();
      if (group >= PIECES) {
        tc_fence_before_sync();
        mbar_arrive(&acc_empty[acc]);
        continue;
      }
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int piece = group + 4 * i;
        const int col0 = tn * BN + piece * 32;
        const bool more = i + 1 < ROUNDS;
        const int next_item = more ? item : item + int(gridDim.x), next_piece = more ? piece + 4 : group;
        float v[32];
        tmem_ld_32x32_f(tmem_addr(tmem_base, quarter * 32, acc * BN + piece * 32), v);
        if (p.bias) {
          __syncwarp();
          bias[lane] = bias_next[i];
          __syncwarp();
        }
        uint8_t* s_y = mine + set * p.set_bytes;
        uint8_t* s_save = s_y + piece_bytes;
        if (!p.residual) {
          if (lane == 0) {  // the stores that last used this set have read it
            if (p.sets == 2) tma_store_wait_read1();
            else tma_store_wait_read0();
          }
          __syncwarp();
        } else {
          if (p.sets == 2) fetch_residual(set ^ 1, next_item, next_piece);
          mbar_wait(&arrived[set], (residual_phase >> set) & 1, 94);
          residual_phase ^= 1u << set;
        }
        tmem_ld_wait();
        if (!more) {
          tc_fence_before_sync();
          mbar_arrive(&acc_empty[acc]);
        }
        if (p.bias) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 f = *reinterpret_cast<const float4*>(bias + q * 4);
            add_f32x2(v[4 * q], v[4 * q + 1], f.x, f.y);
            add_f32x2(v[4 * q + 2], v[4 * q + 3], f.z, f.w);
          }
        }
        if (p.save) stage_piece<T>(s_save, lane, p.save == 2, v);
        if (p.act == kActRelu) activate_all<kActRelu>(v);
        else if (p.act == kActGelu) activate_all<kActGelu>(v);
        else if (p.act == kActGeluTanh) activate_all<kActGeluTanh>(v);
        else if (p.act == kActSilu) activate_all<kActSilu>(v);
        if (p.residual) add_piece<T>(s_y, lane, p.out_f32, v);
        stage_piece<T>(s_y, lane, p.out_f32, v);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (col0 < p.n && row0 < p.m) {
            tma_store_3d(&tmY, s_y, col0, row0, split);
            if (p.save) tma_store_3d(&tmSave, s_save, col0, row0, 0);
          }
          tma_store_commit();  // an empty group too: the waits count groups
        }
        if (p.sets == 2) set ^= 1;
        else if (p.residual) fetch_residual(0, next_item, next_piece);
      }
    }
    if (lane == 0) tma_store_wait0();
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// ---------------------------------------------------------------------------
// d = dy act'(a) as the products' operand, and the sums of its columns (db) before it is rounded to it.
// A CTA has 256 columns at most and every gridDim.y-th run of rows; a thread eight columns.
// ---------------------------------------------------------------------------
struct LinearSlopeParams {
  const void* dy;          // [rows][dy_pitch], of T or fp32
  long long dy_pitch;
  int dy_f32;
  const void* a;           // [rows][a_pitch], of T or fp32; null without an activation
  long long a_pitch;
  int a_f32;
  void* d;                 // [rows][n], of T; null: sums only
  float* partial;          // [gridDim.y][n]; may be null
  long long rows;
  int n;
};

// Two rows of a thread are on their way at a time.
template <class T, int ACT>
__global__ void __launch_bounds__(256, 4) linear_slope_kernel(LinearSlopeParams p) {
  pdl_wait();
  __shared__ float sums[8][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * 256 + lane * 8;
  float total[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) total[e] = 0.f;
  if (c0 < p.n) {
    const long long step = (long long)gridDim.y * 8;
    for (long long r = (long long)blockIdx.y * 8 + warp; r < p.rows; r += 2 * step) {
      const bool second = r + step < p.rows;
      float d[2][8], a[2][8];
      load_eight_of<T>(p.dy, p.dy_f32, r * p.dy_pitch + c0, d[0]);
      if (ACT != kActNone) load_eight_of<T>(p.a, p.a_f32, r * p.a_pitch + c0, a[0]);
      if (second) {
        load_eight_of<T>(p.dy, p.dy_f32, (r + step) * p.dy_pitch + c0, d[1]);
        if (ACT != kActNone) load_eight_of<T>(p.a, p.a_f32, (r + step) * p.a_pitch + c0, a[1]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k && !second) break;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          times_slope<ACT>(a[k][e], a[k][e + 1], d[k][e], d[k][e + 1]);
          add_f32x2(total[e], total[e + 1], d[k][e], d[k][e + 1]);
        }
        if (p.d) store_eight(static_cast<T*>(p.d) + (r + k * step) * p.n + c0, d[k]);
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = total[e];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < p.n) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
    p.partial[(long long)blockIdx.y * p.n + c] = s;
  }
}

}  // namespace b200
