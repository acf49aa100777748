// The linear layer y = act(x w^T + b) + residual and the products of its backward pass, bf16 or fp16 operands with fp32
// accumulation in tensor memory:
//
//   forward   y  [rows][n] = x [rows][k] . w [n][k]^T     both operands have the contraction along their rows (K-major)
//   backward  dx [rows][k] = d [rows][n] . w [n][k]       w has it across them (MN-major)
//             dw [n][k]    = d [rows][n]^T . x [rows][k]  so have both
//
// with d = dy act'(a), a the value before the activation.  The shared-memory descriptors take either order, so nothing is
// transposed on the way.  Persistent kernel, one CTA per SM, 128 x BN tiles:
//   warp 0       TMA producer, K slabs of 64 through a ring in shared memory
//   warp 1       MMA issuer, two accumulators in tensor memory
//   warps 2..17  epilogue: four groups of four warps, which take the tile's 32-column pieces in turn; a warp stages its 32 rows of
//                a piece in a set of its own and sends them off by TMA without meeting the other warps.  (Two groups with
//                64-column pieces: the forward pass of 147456 rows 128 -> 512, silu and saved value, 97 us, two warps a scheduler
//                that wait for their own instructions, 1.4 a clock.)
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
};

// ---------------------------------------------------------------------------
// Activations and their slopes
// ---------------------------------------------------------------------------
// Both by the hardware's exponential and reciprocal (2^-22 of their values): an epilogue or a gradient pass of two operands has
// about fifteen instructions an element before the issue slots, not the memory, bound it (silu by expf and a division: the
// gradient of 147456 x 512 values 110 us, 4.1 TB/s).
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluTanhQ = 0.044715f;

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid_ex2(float x) { return rcp_approx(1.0f + exp2_approx(-kLog2e * x)); }

// The normal distribution's Phi(a) and phi(a).  Phi(-|a|) = poly(t) exp(-a^2 / 2) / 2 with t = 1 / (1 + p |a| / sqrt(2)): the
// rational approximation 7.1.26 of M. Abramowitz and I. Stegun, "Handbook of Mathematical Functions" (C. Hastings, 1955), off by 0.75e-7
// at most.  It shares its exponential with phi.
__device__ __forceinline__ float normal_cdf(float a, float& density) {
  const float t = rcp_approx(fmaf(0.3275911f * 0.70710678118654752f, fabsf(a), 1.0f));
  const float e = exp2_approx(-0.5f * kLog2e * a * a);
  float q = fmaf(t, 1.061405429f, -1.453152027f);
  q = fmaf(t, q, 1.421413741f);
  q = fmaf(t, q, -0.284496736f);
  q = fmaf(t, q, 0.254829592f);
  q *= 0.5f * e * t;
  density = 0.3989422804014327f * e;
  return a < 0.f ? q : 1.0f - q;
}

template <int ACT>
__device__ __forceinline__ float activate(float a) {
  if constexpr (ACT == kActRelu) return a < 0.f ? 0.f : a;  // keeps NaN
  else if constexpr (ACT == kActGelu) {
    float density;
    return a * normal_cdf(a, density);
  } else if constexpr (ACT == kActGeluTanh) return a * sigmoid_ex2(2.0f * kGeluTanhC * a * fmaf(kGeluTanhQ, a * a, 1.0f));
  else if constexpr (ACT == kActSilu) return a * sigmoid_ex2(a);
  else return a;
}

template <int ACT>
__device__ __forceinline__ float slope(float a) {
  if constexpr (ACT == kActRelu) return a > 0.f ? 1.f : a <= 0.f ? 0.f : a;  // NaN stays
  else if constexpr (ACT == kActGelu) {
    float density;
    const float below = normal_cdf(a, density);
    return fmaf(a, density, below);
  } else if constexpr (ACT == kActGeluTanh) {
    const float s = sigmoid_ex2(2.0f * kGeluTanhC * a * fmaf(kGeluTanhQ, a * a, 1.0f));
    return fmaf(a * s * (1.0f - s), 2.0f * kGeluTanhC * fmaf(3.0f * kGeluTanhQ, a * a, 1.0f), s);
  } else if constexpr (ACT == kActSilu) {
    const float s = sigmoid_ex2(a);
    return fmaf(a * s, 1.0f - s, s);
  } else return 1.0f;
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

// Two values at a time where the arithmetic around the exponential and the reciprocal has two-wide instructions.
template <int ACT>
__device__ __forceinline__ void activate_all(float (&v)[32]) {
  if constexpr (ACT == kActSilu || ACT == kActGeluTanh) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float x0 = v[i], x1 = v[i + 1];
      if constexpr (ACT == kActGeluTanh) {
        mul_f32x2(x0, x1, x0, x1);
        fma_f32x2(x0, x1, x0, x1, -2.0f * kLog2e * kGeluTanhC * kGeluTanhQ, -2.0f * kLog2e * kGeluTanhC * kGeluTanhQ,
                  -2.0f * kLog2e * kGeluTanhC, -2.0f * kLog2e * kGeluTanhC);
        mul_f32x2(x0, x1, v[i], v[i + 1]);
      } else {
        mul_f32x2(x0, x1, -kLog2e, -kLog2e);
      }
      x0 = exp2_approx(x0), x1 = exp2_approx(x1);
      add_f32x2(x0, x1, 1.0f, 1.0f);
      mul_f32x2(v[i], v[i + 1], rcp_approx(x0), rcp_approx(x1));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = activate<ACT>(v[i]);
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

template <class T, bool A_MN, bool B_MN, int BN>
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
      mbar_init(&full[s], 1);
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
          mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
          if constexpr (A_MN) {
            tma_load_2d(sa, &tmA, &full[stage], tm * 128, kb * 64);
            tma_load_2d(sa + 8192, &tmA, &full[stage], tm * 128 + 64, kb * 64);
          } else {
            tma_load_2d(sa, &tmA, &full[stage], kb * 64, tm * 128);
          }
          if constexpr (B_MN) {
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
    for (int item = blockIdx.x; item < items; item += gridDim.x, ++it) {
      const int split = item / tiles, tile = item - split * tiles;
      const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
      const int acc = it & 1;
      const int row0 = tm * 128 + quarter * 32;
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
  int n, act;
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
        for (int e = 0; e < 8; ++e) {
          if (ACT != kActNone) d[k][e] *= slope<ACT>(a[k][e]);
          total[e] += d[k][e];
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
