// The whole backward pass of a linear layer in one pass over its rows, for layers whose dw fits into the tensor memory of one or two
// CTAs (n <= 512, k <= 256 or 128):
//
//   d = dy act'(a),  dx = d w,  dw = d^T x,  db = column sums of d
//
// As separate kernels d is written once and read twice, which is most of what a layer of few columns and many rows moves
// (147456 rows, 128 -> 512: 831 MB against 378).  d is rounded to the operands' 16 bits for both products, as in linear.cuh, and not for
// db.  Here a CTA or a pair of them walks over tiles of 128 rows; d lives in shared memory
// only, 128 columns ("a chunk") at a time, in the layout that serves both products: 64-column atoms of 128 rows x 128 bytes,
// swizzled, are K-major for dx (contraction along a row) and MN-major for dw (contraction across the rows).  dw stays in tensor
// memory for all tiles: two buffers of dx and the chunks of dw, each KC columns of k wide.  Where k is wider, two CTAs take KC columns
// each; both need all of d, so each makes half of the tile's rows and copies them to the other.
//   warp 0        TMA: w once, x tile by tile
//   warp 1        MMA issuer
//   warps 2..17   d: one or two groups of warps, each with one or two chunks in turn, so that while one chunk is sent and multiplied the
//                 next is made, and a thread's columns and their sums for db are the same in all tiles; the next two rows of a
//                 thread on their way.  Then the dx of the tile before: tensor memory -> staging -> TMA store, a 32 x 32 piece a
//                 warp; at the end dw and db to the CTA's part
// Bound by the warps that make d (silu: 130 instructions for eight values of a thread, and their dependences): 147456 rows, 128 -> 512, 106
// to 110 us and 14 for the sums over the parts, against 158 to 168 as separate kernels.  What else was tried there: each CTA of the pair making
// all of d 178 us; d written to the other CTA by its threads' stores, 16 bytes each, 212 to 247 (the copies are 8 KB each); eight
// warps 192; one chunk a group, whose warps wait while it is sent 121; the rows of the next tile prefetched into the L2 112; four CTAs for
// wider layers, 100000 rows 512 -> 128 with x in 8 bits 148 against 114 as separate kernels then were.
#pragma once
#include "linear.cuh"

namespace b200 {

struct LinearGradParams {
  const void* dy;
  long long dy_pitch;
  const void* a;               // of T; null without an activation
  long long a_pitch;
  const uint8_t* values;       // x in 8 bits; null: x by TMA
  const uint8_t* exponents;
  float* dw;                   // [workers][n][k]
  float* db;                   // [CTAs][n]; may be null
  long long rows;
  int n, k;
  int chunks, kc, splits;      // of n in 128s; columns of k a CTA takes, CTAs of a cluster: 1 or 2
  int groups, group_warps;     // that make d: one of sixteen or two of eight
  int tiles, workers;          // row tiles; clusters
  int slots, x_slots;
  int act;
  uint32_t idesc_dx, idesc_dw;
};

constexpr int kGradWarps = 16;                       // that make d
constexpr int kGradThreads = 32 * (2 + kGradWarps);
constexpr uint32_t kGradHead = 1024, kGradChunkBytes = 128 * 128 * 2;

__host__ __device__ inline uint32_t linear_grad_smem(int chunks, int kc, int slots, int x_slots) {
  return kGradHead + uint32_t(chunks) * kc * 256 + uint32_t(slots) * kGradChunkBytes + uint32_t(x_slots) * kc * 256 + kc / 32 * 4 * 2048 + 1024;
}

// ---------------------------------------------------------------------------
// Cluster: shared memory of the other CTA, and barriers it arrives at
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_address(uint32_t smem, uint32_t cta) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(cta));
  return a;
}
// A block of this CTA's shared memory to another's, whose barrier counts its bytes.
__device__ __forceinline__ void cluster_copy(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Wait for arrivals from the whole cluster, bounded like mbar_wait.
__device__ __forceinline__ bool cluster_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void cluster_wait(uint64_t* bar, uint32_t parity, int site) {
  if (cluster_try_wait(bar, parity)) return;
  mbar_wait_slow(bar, parity, site);  // bounded; the look below is the one that acquires
  cluster_try_wait(bar, parity);
}
// One arrival at the same barrier of every CTA in the mask once the MMAs issued so far have completed.
__device__ __forceinline__ void umma_commit_cluster(uint64_t* bar, uint16_t mask) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"(mask)
               : "memory");
}

template <class T, bool DY_F32, bool ACT, bool KEPT>
__global__ void __launch_bounds__(kGradThreads, 1)
linear_grad_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmDx,
                   LinearGradParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* d_full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* d_empty = d_full + 4;
  uint64_t* x_full = d_empty + 4;
  uint64_t* x_empty = x_full + 2;
  uint64_t* dx_full = x_empty + 2;
  uint64_t* dx_empty = dx_full + 2;
  uint64_t* w_full = dx_empty + 2;
  uint64_t* dw_full = w_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dw_full + 1);
  const uint32_t w_bytes = uint32_t(p.chunks) * p.kc * 256, x_bytes = uint32_t(p.kc) * 256;
  uint8_t* w_s = smem + kGradHead;                   // [kc / 64][chunks * 128 rows of n][128 B]
  uint8_t* d_s = w_s + w_bytes;                      // [slots][2 atoms][128 rows][128 B]
  uint8_t* x_s = d_s + p.slots * kGradChunkBytes;    // [x_slots][kc / 64][128 rows][128 B]
  uint8_t* staging = x_s + p.x_slots * x_bytes;      // [kc / 32 * 4 warps][2 KB]

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const int split = blockIdx.x % p.splits, worker = blockIdx.x / p.splits;  // split: the CTA's rank in its cluster
  const int k0 = split * p.kc;
  const int atoms = p.kc / 64;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&d_full[s], 1);
      mbar_init(&d_empty[s], p.splits);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&x_full[s], KEPT ? 32 * kGradWarps : 1);
      mbar_init(&x_empty[s], 1);
      mbar_init(&dx_full[s], 1);
      mbar_init(&dx_empty[s], 4 * p.kc);
    }
    mbar_init(w_full, 1);
    mbar_init(dw_full, 1);
    fence_mbar_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmDx);
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before_sync();
  if (p.splits == 2) cluster_sync();                 // the other's barriers are there
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;             // [2][kc] columns of dx, then [chunks][kc] of dw
  const uint32_t dw_col = 2 * p.kc;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      mbar_arrive_expect_tx(w_full, w_bytes);
      for (int a = 0; a < atoms; ++a)
        for (int c = 0; c < p.chunks; ++c)
          tma_load_2d(w_s + (a * p.chunks + c) * 16384, &tmW, w_full, k0 + a * 64, c * 128);
      if (!KEPT) {
        int i = 0;
        for (int tile = worker; tile < p.tiles; tile += p.workers, ++i) {
          const int s = i % p.x_slots;
          mbar_wait(&x_empty[s], ((i / p.x_slots) & 1) ^ 1, 100);
          mbar_arrive_expect_tx(&x_full[s], x_bytes);
          for (int a = 0; a < atoms; ++a) tma_load_2d(x_s + s * x_bytes + a * 16384, &tmX, &x_full[s], k0 + a * 64, tile * 128);
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    mbar_wait(w_full, 0, 101);
    int i = 0, slot = 0;
    uint32_t phase = 0;
    const uint32_t w_lbo = uint32_t(p.chunks) * 16384;
    for (int tile = worker; tile < p.tiles; tile += p.workers, ++i) {
      const int xs = i % p.x_slots, ds = i & 1;
      mbar_wait(&x_full[xs], (i / p.x_slots) & 1, 102);
      mbar_wait(&dx_empty[ds], ((i >> 1) & 1) ^ 1, 103);
      const uint32_t x_lo = desc_lo(smem_u32(x_s + xs * x_bytes), 16384);
      for (int c = 0; c < p.chunks; ++c) {
        mbar_wait(&d_full[slot], phase, 104);
        tc_fence_after_sync();
        const uint32_t d_addr = smem_u32(d_s + slot * kGradChunkBytes);
        const uint32_t d_k = desc_lo(d_addr), d_mn = desc_lo(d_addr, 16384);
        const uint32_t w_lo = desc_lo(smem_u32(w_s + c * 16384), w_lbo);
        if (leader) {
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 columns of d at a time: atom k / 4
            umma_bf16_ss2(tmem_base + ds * p.kc, d_k + (k >> 2) * 1024 + (k & 3) * 2, kDescHiSw128, w_lo + k * 128, kDescHiSw128, p.idesc_dx,
                          c != 0 || k != 0);
#pragma unroll
          for (int k = 0; k < 8; ++k)  // 16 rows at a time
            umma_bf16_ss2(tmem_base + dw_col + c * p.kc, d_mn + k * 128, kDescHiSw128, x_lo + k * 128, kDescHiSw128, p.idesc_dw,
                          i != 0 || k != 0);
          if (p.splits == 2) umma_commit_cluster(&d_empty[slot], 3);
          else umma_commit(&d_empty[slot]);
        }
        __syncwarp();
        if (++slot == p.slots) slot = 0, phase ^= 1;
      }
      if (leader) {
        umma_commit(&dx_full[ds]);
        umma_commit(&x_empty[xs]);
      }
      __syncwarp();
    }
    if (leader) umma_commit(dw_full);
    __syncwarp();
    // The other CTA's commits arrive here on their own time, and the last ones release slots that nobody waits for any more.  With both
    // CTAs' arrivals of every slot's last use in hand, none is on its way to a CTA that has left behind the cluster's barrier below.
    if (p.splits == 2) {
      for (int s = 0; s < p.slots; ++s) {
        const int uses = (i * p.chunks - s + p.slots - 1) / p.slots;  // chunks s, s + slots, ... of the cluster's
        if (uses > 0) cluster_wait(&d_empty[s], (uses - 1) & 1, 109);
      }
    }
  } else {
    const int w = warp - 2, quarter = warp & 3;  // tensor-memory lanes 32 * quarter ..
    const int piece = w >> 2;
    const int g = w / p.group_warps;                                // its chunks are g and g + groups
    const int turns = g + p.groups < p.chunks ? 2 : 1;
    const int col = (lane & 15) * 8, row_in = (w % p.group_warps) * 2 + (lane >> 4);
    const int step = 2 * p.group_warps;                             // rows of the group's warps at a time
    const int steps = 128 / p.splits / step;                        // a chunk's rows of this CTA take; even
    const int first = split * (128 / p.splits) + row_in;
    float total[2][8];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) total[j][e] = 0.f;
    // Two rows of the thread are on their way: row `ahead_row`, its step and the group's turn.
    uint4 dy0[2], dy1[DY_F32 ? 2 : 1], av[ACT ? 2 : 1];
    constexpr int kDySize = DY_F32 ? 4 : 2;
    const uint8_t* dy_at = static_cast<const uint8_t*>(p.dy) + (g * 128 + col) * kDySize;
    const uint8_t* a_at = static_cast<const uint8_t*>(p.a) + (g * 128 + col) * 2;
    const uint32_t dy_pitch = uint32_t(p.dy_pitch * kDySize), a_pitch = uint32_t(p.a_pitch * 2);
    uint32_t ahead_row = uint32_t(worker) * 128 + first;
    int ahead = 0, ahead_turn = 0;
    auto fetch = [&](int v) {
      const int c = (g + ahead_turn * p.groups) * 128 + col;
      if (c < p.n && ahead_row < uint32_t(p.rows)) {
        const uint4* src = reinterpret_cast<const uint4*>(dy_at + uint64_t(ahead_row) * dy_pitch + ahead_turn * p.groups * 128 * kDySize);
        dy0[v] = src[0];
        if (DY_F32) dy1[v] = src[1];
        if (ACT) av[v] = *reinterpret_cast<const uint4*>(a_at + uint64_t(ahead_row) * a_pitch + ahead_turn * p.groups * 256);
      } else {
        dy0[v] = make_uint4(0, 0, 0, 0);
        if (DY_F32) dy1[v] = make_uint4(0, 0, 0, 0);
        if (ACT) av[v] = make_uint4(0, 0, 0, 0);
      }
      ahead_row += step;
      if (v == 1 && (ahead += 2) == steps) {
        ahead = 0;
        ahead_row -= steps * step;
        if (++ahead_turn >= turns) ahead_turn = 0, ahead_row += p.workers * 128;
      }
    };
    // x of a tile from its 8 bits: KC / 8 threads a row, KC / 32 rows a thread, those of the next tile on their way too.
    const int x_lanes = p.kc / 8, x_rows = 32 * kGradWarps / x_lanes;
    const int x_col = ((w * 32 + lane) % x_lanes) * 8, x_row = (w * 32 + lane) / x_lanes;
    const int x_groups = (p.k + kKeepGroup - 1) / kKeepGroup;
    uint2 xq[4];
    uint32_t x_byte;  // a byte each
    auto fetch_x = [&](int tile) {
      x_byte = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int rl = x_row + j * x_rows;
        const long long r = (long long)tile * 128 + rl;
        xq[j] = make_uint2(0, 0);
        if (rl < 128 && r < p.rows && k0 + x_col < p.k) {
          xq[j] = *reinterpret_cast<const uint2*>(p.values + r * p.k + k0 + x_col);
          x_byte |= uint32_t(p.exponents[r * x_groups + (k0 + x_col) / kKeepGroup]) << (8 * j);
        }
      }
    };
    auto put_x = [&](int i, int tile) {
      const int xs = i % p.x_slots;
      uint8_t* dst = x_s + xs * x_bytes + (x_col >> 6) * 16384;
      mbar_wait(&x_empty[xs], ((i / p.x_slots) & 1) ^ 1, 106);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int rl = x_row + j * x_rows;
        float f[8];
        kept_eight<T>(xq[j], keep_scale((x_byte >> (8 * j)) & 0xffu), f);
        if (rl < 128)
          *reinterpret_cast<uint4*>(dst + sw128_offset(rl, (x_col >> 3) & 7)) =
              make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
      }
      fence_proxy_async_smem();
      mbar_arrive(&x_full[xs]);
      fetch_x(tile + p.workers);
    };
    // The dx of the cluster's tile i, this warp's piece of it.
    auto drain = [&](int i) {
      if (piece >= p.kc / 32) return;
      mbar_wait(&dx_full[i & 1], (i >> 1) & 1, 105);
      tc_fence_after_sync();
      float v[32];
      tmem_ld_32x32_f(tmem_addr(tmem_base, quarter * 32, (i & 1) * p.kc + piece * 32), v);
      if (lane == 0) tma_store_wait_read0();  // the store before has read the staging tile
      __syncwarp();
      tmem_ld_wait();
      tc_fence_before_sync();
      mbar_arrive(&dx_empty[i & 1]);
      uint8_t* out = staging + (piece * 4 + quarter) * 2048;
      stage_piece<T>(out, lane, 0, v);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        const int col = k0 + piece * 32, row = (worker + i * p.workers) * 128 + quarter * 32;
        if (col < p.k && row < p.rows) tma_store_2d(&tmDx, out, col, row);
        tma_store_commit();
      }
    };
    const int mine = worker < p.tiles ? (p.tiles - 1 - worker) / p.workers + 1 : 0;  // tiles of the cluster
    if (KEPT) fetch_x(worker);
#pragma unroll
    for (int v = 0; v < 2; ++v) fetch(v);
    for (int i = 0; i < mine; ++i) {
      if (KEPT) put_x(i, worker + i * p.workers);
#pragma unroll
      for (int turn = 0; turn < 2; ++turn) {
        if (turn >= turns) break;
        const int number = i * p.chunks + g + turn * p.groups, slot = number % p.slots;
        cluster_wait(&d_empty[slot], ((number / p.slots) & 1) ^ 1, 107);
        const uint32_t dst = smem_u32(d_s + slot * kGradChunkBytes + (col >> 6) * 16384);
#pragma unroll 1
        for (int s = 0; s < steps; s += 2) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float d[1][8], a[1][8];
            const uint32_t q0[4] = {dy0[v].x, dy0[v].y, dy0[v].z, dy0[v].w};
            if constexpr (DY_F32) {
              const uint32_t q1[4] = {dy1[v].x, dy1[v].y, dy1[v].z, dy1[v].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) d[0][e] = __uint_as_float(q0[e]), d[0][4 + e] = __uint_as_float(q1[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(q0[e]);
                d[0][2 * e] = f.x, d[0][2 * e + 1] = f.y;
              }
            }
            if constexpr (ACT) {
              const uint32_t qa[4] = {av[v].x, av[v].y, av[v].z, av[v].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<T>(qa[e]);
                a[0][2 * e] = f.x, a[0][2 * e + 1] = f.y;
              }
            }
            fetch(v);
            if constexpr (ACT) {
              if (p.act == kActSilu) slope_pairs<kActSilu>(a, d);
              else if (p.act == kActGelu) slope_pairs<kActGelu>(a, d);
              else if (p.act == kActGeluTanh) slope_pairs<kActGeluTanh>(a, d);
              else slope_pairs<kActRelu>(a, d);
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2) add_f32x2(total[turn][e], total[turn][e + 1], d[0][e], d[0][e + 1]);
            const uint4 q = make_uint4(pack2<T>(d[0][0], d[0][1]), pack2<T>(d[0][2], d[0][3]), pack2<T>(d[0][4], d[0][5]), pack2<T>(d[0][6], d[0][7]));
            const uint32_t at = dst + sw128_offset(first + (s + v) * step, lane & 7);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
          }
        }
        // the group's rows are in place: one thread sends them to the other CTA
        fence_proxy_async_smem();
        named_bar_sync(2 + g, 32 * p.group_warps);
        if (w % p.group_warps == 0 && lane == 0) {
          const uint32_t share = 128 / p.splits * 128, from = smem_u32(d_s + slot * kGradChunkBytes) + split * share;
          const uint32_t bar = smem_u32(&d_full[slot]);
          mbar_arrive_expect_tx(&d_full[slot], (p.splits - 1) * 2 * share);
          if (p.splits == 2) {
            const int cta = split ^ 1;
            cluster_copy(cluster_address(from, cta), from, share, cluster_address(bar, cta));
            cluster_copy(cluster_address(from + 16384, cta), from + 16384, share, cluster_address(bar, cta));
          }
        }
      }
      if (i > 0) drain(i - 1);
    }
    if (mine > 0) drain(mine - 1);
    if (lane == 0) tma_store_wait0();
    mbar_wait(dw_full, 0, 108);
    tc_fence_after_sync();
    if (p.db) {  // the rows' sums of the warps, in their order, where dx was staged (chunks may still be on their way to the other CTA)
      float* sums = reinterpret_cast<float*>(staging);  // [warps of a group][chunks * 128]: 8, 16, 12 or 16 KB of 16 at least
      named_bar_sync(1, 32 * kGradWarps);               // every warp's stores have read it
      const int width = p.chunks * 128;
#pragma unroll
      for (int turn = 0; turn < 2; ++turn)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          total[turn][e] += __shfl_xor_sync(0xffffffffu, total[turn][e], 16);
          if (lane < 16 && turn < turns) sums[(w % p.group_warps) * width + (g + turn * p.groups) * 128 + col + e] = total[turn][e];
        }
      named_bar_sync(1, 32 * kGradWarps);
      for (int t = w * 32 + lane; t < p.n; t += 32 * kGradWarps) {
        float s = 0.f;
        for (int j = 0; j < p.group_warps; ++j) s += sums[j * width + t];
        p.db[(long long)blockIdx.x * p.n + t] = s;
      }
    }
    const int pieces = p.chunks * (p.kc / 32);
    for (int j = piece; j < pieces; j += kGradWarps / 4) {
      const int chunk = j / (p.kc / 32), kcol = k0 + (j - chunk * (p.kc / 32)) * 32;
      const int row = chunk * 128 + quarter * 32 + lane;
      float v[32];
      tmem_ld_32x32_f(tmem_addr(tmem_base, quarter * 32, dw_col + j * 32), v);
      tmem_ld_wait();
      if (row < p.n) {
        float* out = p.dw + ((long long)worker * p.n + row) * p.k + kcol;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float f[8] = {v[8 * q], v[8 * q + 1], v[8 * q + 2], v[8 * q + 3], v[8 * q + 4], v[8 * q + 5], v[8 * q + 6], v[8 * q + 7]};
          if (kcol + q * 8 < p.k) st_global_v8(out + q * 8, f);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if (p.splits == 2) cluster_sync();  // no CTA leaves while the other may still arrive at its barriers
  else __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

}  // namespace b200
