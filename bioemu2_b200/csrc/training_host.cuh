// Launches of the training operators: LayerNorm forward and backward, 8-bit checkpoints, the linear layer forward and backward.
#pragma once
#include "host_util.cuh"
#include "checkpoint8.cuh"
#include "layer_norm.cuh"
#include "linear_grad.cuh"

namespace b200 {

static bool training_dtype(int d) { return d == B200_DTYPE_BF16 || d == B200_DTYPE_F32 || d == B200_DTYPE_F16; }
static size_t dtype_bytes(int d) { return d == B200_DTYPE_F32 ? 4 : 2; }
// Eight neighbours of a row in one access: 32 bytes of fp32, 16 of the shorter types.
static bool eight_aligned(const void* p, int64_t pitch, int dtype) { return aligned(p, dtype_bytes(dtype) * 8) && pitch % 8 == 0; }

template <class F>
static int with_dtype(int dtype, F f) {
  if (dtype == B200_DTYPE_F32) return f(float());
  if (dtype == B200_DTYPE_BF16) return f(__nv_bfloat16());
  return f(__half());
}

// ---------------------------------------------------------------------------
// Checkpoints
// ---------------------------------------------------------------------------
static int launch_keep(const KeepParams& p, int dtype, bool write, cudaStream_t st) {
  if (p.rows == 0) return B200_OK;
  const bool vec = p.cols % 8 == 0 && aligned(p.values, 8) && (write ? eight_aligned(p.x, p.pitch, dtype) : eight_aligned(p.out, p.cols, dtype));
  const bool flat = vec && p.cols % kKeepGroup == 0 && (!write || p.pitch == p.cols || p.rows == 1);
  const int64_t threads = p.rows * p.groups * 4;
  const int64_t cap = int64_t(sm_count()) * 64;
  const int64_t need = (threads + 255) / 256;
  const int grid = int(need < cap ? need : cap);
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto go = [&](auto rows) -> int {
      if (write) B200_LAUNCH((keep_kernel<T, rows()>), grid, 256, 0, st, p);
      else B200_LAUNCH((restore_kernel<T, rows()>), grid, 256, 0, st, p);
      return B200_OK;
    };
    if (flat) return go(std::integral_constant<int, kKeepFlat>());
    if (vec) return go(std::integral_constant<int, kKeepVector>());
    return go(std::integral_constant<int, kKeepScalar>());
  });
}

// ---------------------------------------------------------------------------
// LayerNorm
// ---------------------------------------------------------------------------
// Threads a row is given, and how many rows' CTAs an SM is given: what the row needs at eight columns a thread.  f(L, NV, VEC).
template <class F>
static int with_row_shape(int cols, bool vec, F f) {
  using std::integral_constant;
#define B200_ROW(L, NV, VEC) return f(integral_constant<int, L>(), integral_constant<int, NV>(), integral_constant<bool, VEC>())
  if (vec) {
    if (cols <= 64) B200_ROW(8, 1, true);
    if (cols <= 128) B200_ROW(16, 1, true);
    if (cols <= 256) B200_ROW(32, 1, true);
    if (cols <= 512) B200_ROW(32, 2, true);
    if (cols <= 1024) B200_ROW(128, 1, true);
    if (cols <= 2048) B200_ROW(128, 2, true);
    if (cols <= 4096) B200_ROW(256, 2, true);
    B200_ROW(512, 2, true);
  }
  if (cols <= 256) B200_ROW(32, 1, false);
  if (cols <= 2048) B200_ROW(128, 2, false);
  B200_ROW(512, 2, false);
#undef B200_ROW
}

// CTAs of the backward pass, each of which leaves a row of sums of dw and db.
static int64_t layer_norm_parts(int64_t rows, int cols, bool vec) {
  int rpb = 1;
  int ctas = 1;
  with_row_shape(cols, vec, [&](auto L, auto NV, auto VEC) -> int {
    rpb = kRowThreads<L()> / L(), ctas = kGradCtas<L(), NV(), VEC()>;
    return 0;
  });
  const int64_t need = (rows + rpb - 1) / rpb, cap = int64_t(sm_count()) * ctas;
  return need < cap ? need : cap;
}

// Sums over `parts` rows of `width` columns; the columns from `split` on go to out1.
static int launch_part_sum(const float* partial, int64_t parts, int64_t width, int64_t split, void* out0, int dtype0, void* out1, int dtype1,
                           cudaStream_t st) {
  const int v = width % 4 == 0 && split % 4 == 0 ? 4 : 1;
  // threads that share a column: more of them while there are parts for four each and threads for half of the device, as long as a
  // CTA still reads whole lines of wide rows (74 parts of 65536 columns: 16 threads; with 32 the backward pass around it takes 125 to 126 us
  // for 121, with 8 the same.  296 parts of 8192: 32; with 16 28.7 for 26.6, with 8 30.7)
  int down = 8;
  while (down < (width >= 4096 ? 32 : 128) && down * 4 < parts && width / v * down < int64_t(sm_count()) * 1024) down *= 2;
  PartSumParams q{partial, int(parts), 256 / down, width, split, {out0, out1}, {dtype0, dtype1}};
  const int64_t per_cta = int64_t(q.across) * v;
  const int grid = int((width + per_cta - 1) / per_cta);
  if (v == 4) B200_LAUNCH(part_sum_kernel<4>, grid, 256, 0, st, q);
  else B200_LAUNCH(part_sum_kernel<1>, grid, 256, 0, st, q);
  return B200_OK;
}

template <class F>
static int with_row_types(int x_dtype, int y_dtype, F f) {
  if (x_dtype != B200_DTYPE_F32) return x_dtype == B200_DTYPE_BF16 ? f(__nv_bfloat16(), __nv_bfloat16()) : f(__half(), __half());
  return with_dtype(y_dtype, [&](auto y) -> int { return f(float(), y); });
}

static int launch_layer_norm(const LayerNormParams& p, int x_dtype, int y_dtype, cudaStream_t st) {
  const bool vec = p.cols % 8 == 0 && eight_aligned(p.x, p.x_pitch, x_dtype) && eight_aligned(p.out, p.cols, y_dtype) &&
                   (!p.values || aligned(p.values, 8));
  return with_row_types(x_dtype, y_dtype, [&](auto tx, auto ty) -> int {
    return with_row_shape(p.cols, vec, [&](auto L, auto NV, auto VEC) -> int {
      constexpr int threads = kRowThreads<L()>, rpb = threads / L();
      const int64_t need = (p.rows + rpb - 1) / rpb, cap = int64_t(sm_count()) * (2048 / threads);
      B200_LAUNCH((layer_norm_kernel<decltype(tx), decltype(ty), L(), NV(), VEC()>), int(need < cap ? need : cap), threads, 0, st, p);
      return B200_OK;
    });
  });
}

static int launch_layer_norm_grad(const LayerNormParams& p, int x_dtype, int y_dtype, void* dw, void* db, int w_dtype, cudaStream_t st) {
  const bool vec = p.cols % 8 == 0 && eight_aligned(p.dy, p.dy_pitch, y_dtype) && (!p.out || eight_aligned(p.out, p.cols, x_dtype)) &&
                   (p.values ? aligned(p.values, 8) : eight_aligned(p.x, p.x_pitch, x_dtype));
  const int64_t parts = layer_norm_parts(p.rows, p.cols, vec);
  const int e = with_row_types(x_dtype, y_dtype, [&](auto tx, auto ty) -> int {
    return with_row_shape(p.cols, vec, [&](auto L, auto NV, auto VEC) -> int {
      if (p.values) B200_LAUNCH((layer_norm_grad_kernel<decltype(tx), decltype(ty), true, L(), NV(), VEC()>), int(parts), kRowThreads<L()>, 0, st, p);
      else B200_LAUNCH((layer_norm_grad_kernel<decltype(tx), decltype(ty), false, L(), NV(), VEC()>), int(parts), kRowThreads<L()>, 0, st, p);
      return B200_OK;
    });
  });
  if (e || !p.partial) return e;
  return launch_part_sum(p.partial, parts, 2 * int64_t(p.cols), p.cols, dw, w_dtype, db, w_dtype, st);
}

// ---------------------------------------------------------------------------
// The linear layer
// ---------------------------------------------------------------------------
struct LinearProduct {
  const void* a;
  int64_t a_pitch;
  bool a_mn;               // contraction across the rows of a
  const void* b;
  int64_t b_pitch;
  bool b_mn;
  void* out;
  int64_t out_pitch;
  int m, n, k;             // rows and columns of the output, length of the contraction
  int dtype, out_dtype;
  int splits = 1;          // parts of the contraction: output planes of m * n fp32 behind one another
  const float* bias = nullptr;
  int act = kActNone;
  void* save = nullptr;    // [m][n], of save_dtype
  int save_dtype = B200_DTYPE_BF16;
  const void* residual = nullptr;
  int64_t residual_pitch = 0;
  const uint8_t* values = nullptr;  // b in 8 bits, in its place: [k][n], where a and b have the contraction across their rows
  const uint8_t* exponents = nullptr;
};

static int linear_tile_n(int m, int n, int k, int splits) { return bmm_tile_n(m, n, k / splits + 1, splits, 64, 256); }

template <class T, bool A_MN, bool B_MN, int BN, bool KEPT>
static int launch_linear_tile(const LinearProduct& a, cudaStream_t st) {
  using Cfg = LinearCfg<BN>;
  LinearParams p = {};
  p.m = a.m, p.n = a.n;
  p.tiles_m = (a.m + 127) / 128, p.tiles_n = (a.n + BN - 1) / BN;
  p.k_blocks = (a.k + 63) / 64, p.splits = a.splits;
  p.act = a.act, p.out_f32 = a.out_dtype == B200_DTYPE_F32, p.save = !a.save ? 0 : a.save_dtype == B200_DTYPE_F32 ? 2 : 1;
  p.bias = a.bias, p.residual = a.residual != nullptr;
  p.values = a.values, p.exponents = a.exponents, p.k = a.k;
  // Staging: two sets of an epilogue warp's pieces where they leave the ring its stages, one otherwise.  Forward, us with a cold L2 (tile
  // width / sets): 147456 rows 128 -> 512 silu and saved value 256/1 70, 128/1 70, 128/2 84; without it 256/2 57, 256/1 59; 100000 rows
  // 128 -> 128 with a residual 128/2 22.5, 128/1 24.6; 41209 rows 512 -> 128 fp32 128/1 26.6, 128/2 32.8.
  p.set_bytes = (p.out_f32 ? 4096 : 2048) + (p.save == 2 ? 4096 : p.save ? 2048 : 0);
  p.sets = p.set_bytes <= 2048 ? 2 : 1;
  const int stages = int((227 * 1024 - Cfg::smem_bytes(0, p.sets * p.set_bytes)) / Cfg::STAGE_BYTES);
  p.stages = stages < Cfg::MAX_STAGES ? stages : Cfg::MAX_STAGES;
  // instruction descriptor: fp32 accumulator, operand type (0 fp16, 1 bf16), bits 15 / 16 for operands across their rows
  p.idesc = (make_idesc_bf16(128, BN) & ~((7u << 7) | (7u << 10))) | (uint32_t(A_MN) << 15) | (uint32_t(B_MN) << 16);
  if (a.dtype == B200_DTYPE_BF16) p.idesc |= (1u << 7) | (1u << 10);

  CUtensorMap tmA, tmB, tmY, tmSave, tmResidual;
  {
    const uint64_t dims[2] = {uint64_t(A_MN ? a.m : a.k), uint64_t(A_MN ? a.k : a.m)};
    const uint64_t str[1] = {uint64_t(a.a_pitch) * 2};
    const uint32_t box[2] = {64, A_MN ? 64u : 128u};
    if (int e = make_tmap_bf16(&tmA, a.a, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  }
  tmB = tmA;
  if (!KEPT) {
    const uint64_t dims[2] = {uint64_t(B_MN ? a.n : a.k), uint64_t(B_MN ? a.k : a.n)};
    const uint64_t str[1] = {uint64_t(a.b_pitch) * 2};
    const uint32_t box[2] = {64, B_MN ? 64u : uint32_t(BN)};
    if (int e = make_tmap_bf16(&tmB, a.b, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  }
  const size_t out_size = dtype_bytes(a.out_dtype);
  {
    const uint64_t dims[3] = {uint64_t(a.n), uint64_t(a.m), uint64_t(a.splits)};
    const uint64_t str[2] = {uint64_t(a.out_pitch) * out_size, uint64_t(a.out_pitch) * a.m * out_size};
    const uint32_t box[3] = {32, 32, 1};
    if (int e = make_tmap(&tmY, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.out, 3, dims, str, box,
                          p.out_f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return e;
  }
  tmSave = tmY;
  if (a.save) {
    const uint64_t dims[3] = {uint64_t(a.n), uint64_t(a.m), 1};
    const size_t size = dtype_bytes(a.save_dtype);
    const uint64_t str[2] = {uint64_t(a.n) * size, uint64_t(a.n) * a.m * size};
    const uint32_t box[3] = {32, 32, 1};
    if (int e = make_tmap(&tmSave, p.save == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.save, 3, dims, str,
                          box, p.save == 2 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return e;
  }
  tmResidual = tmY;
  if (a.residual) {
    const uint64_t dims[2] = {uint64_t(a.n), uint64_t(a.m)};
    const uint64_t str[1] = {uint64_t(a.residual_pitch) * out_size};
    const uint32_t box[2] = {32, 32};
    if (int e = make_tmap(&tmResidual, p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.residual, 2, dims,
                          str, box, p.out_f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return e;
  }
  const int64_t items = int64_t(p.tiles_m) * p.tiles_n * p.splits;
  const int grid = int(items < sm_count() ? items : sm_count());
  B200_LAUNCH((linear_kernel<T, A_MN, B_MN, BN, KEPT>), grid, Cfg::THREADS, Cfg::smem_bytes(p.stages, p.sets * p.set_bytes), st, tmA, tmB, tmY, tmSave, tmResidual, p);
  return B200_OK;
}

static int launch_linear(const LinearProduct& a, cudaStream_t st) {
  int bn = linear_tile_n(a.m, a.n, a.k, a.splits);
  // an fp32 piece beside another takes 96 or 128 KB of staging, which leaves a 256-wide tile one or two stages
  if (bn == 256 && a.save && (a.out_dtype == B200_DTYPE_F32 || a.save_dtype == B200_DTYPE_F32)) bn = 128;
  auto go = [&](auto t, auto amn, auto bmn, auto kept) -> int {
    using T = decltype(t);
    if (bn == 64) return launch_linear_tile<T, amn(), bmn(), 64, kept()>(a, st);
    if (bn == 128) return launch_linear_tile<T, amn(), bmn(), 128, kept()>(a, st);
    return launch_linear_tile<T, amn(), bmn(), 256, kept()>(a, st);
  };
  const std::true_type yes;
  const std::false_type no;
  auto orders = [&](auto t) -> int {
    if (a.a_mn) return a.values ? go(t, yes, yes, yes) : go(t, yes, yes, no);
    if (a.b_mn) return go(t, no, yes, no);
    return go(t, no, no, no);
  };
  return a.dtype == B200_DTYPE_BF16 ? orders(__nv_bfloat16()) : orders(__half());
}

// Parts of dw's contraction over the rows: of the numbers that fill one to four waves of CTAs, and one, the one with the least
// estimated time, in blocks of 64 rows and with about six blocks' time for an output tile and its share of the sum over the parts.
static int linear_dw_splits(int64_t rows, int n, int k) {
  const int64_t blocks = (rows + 63) / 64, sms = sm_count();
  int best = 1;
  double best_cost = 1e30;
  for (int width = 256; width >= 64; width /= 2) {
    const int64_t tiles = int64_t((n + 127) / 128) * ((k + width - 1) / width);
    for (int waves = 0; waves <= 4; ++waves) {
      const int64_t s = waves == 0 ? 1 : std::min(waves * sms / tiles, blocks);
      if (s < 1 || linear_tile_n(n, k, int(rows), int(s)) != width) continue;  // the width the product then takes
      const double cost = double((tiles * s + sms - 1) / sms) * (double((blocks + s - 1) / s) * (width == 256 ? 1.5 : width == 128 ? 1.0 : 0.76) + 6.0) +
                          (s > 1 ? double(n) * k * s * 8 / 1.2e6 : 0.0);
      if (cost < best_cost) best_cost = cost, best = int(s);
    }
  }
  return best;
}

static int64_t linear_slope_parts(int64_t rows, int n) {
  const int64_t across = (n + 255) / 256, need = (rows + 7) / 8;
  int64_t parts = (int64_t(sm_count()) * 8 + across - 1) / across;
  return need < parts ? need : parts;
}

// Pairs of CTAs that the device runs at a time (an SM holds one CTA, and a pair stays within a group of SMs).
static int linear_grad_pairs(uint32_t smem) {
  static std::atomic<int> known{0};  // every size of shared memory asked for leaves an SM one CTA
  if (int n = known.load()) return n;
  const void* kernel = reinterpret_cast<const void*>(linear_grad_kernel<__nv_bfloat16, false, true, false>);
  if (set_smem_once(kernel, smem)) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(sm_count() / 2 * 2));
  cfg.blockDim = dim3(kGradThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) return 0;
  n = std::min(n, sm_count() / 2);
  known.store(n);
  return n;
}

// The backward pass in one kernel (linear_grad.cuh): how n and k are cut, or chunks = 0 where the separate kernels serve better.
// us with a cold L2 and the host's share, in one kernel / as separate ones (rows: 1024, 4096, 9472, 18944, 41209, 100000, 200000; 8: x in 8 bits):
//   one CTA    128 -> 128 gelu, 8        20 / 23   22 / 25   24 / 29   26 / 33   36 / 43    56 / 66    87 / 107
//              128 -> 128 fp32 dy, 8     19 / 22   21 / 25   22 / 29   24 / 31   36 / 37    54 / 55    85 / 86
//              64 -> 256 silu, 8         22 / 22   24 / 25   26 / 29   28 / 33   40 / 45    60 / 72    93 / 121
//              64 -> 64, 8               15 / 21   17 / 22   17 / 25   20 / 27   26 / 32    36 / 43    52 / 64
//   two CTAs   128 -> 512 silu           28 / 25   30 / 28   34 / 33   40 / 43   56 / 68    91 / 127  150 / 219
//              128 -> 512 silu, 8        28 / 25   32 / 30   34 / 35   44 / 45   69 / 72   120 / 133  212 / 225
//              256 -> 256                24 / 25   26 / 27   30 / 29   32 / 37   46 / 49    69 / 82   110 / 133
//              256 -> 256 silu, 8        25 / 25   28 / 27   32 / 32   36 / 41   56 / 59    93 / 100  156 / 168
//              256 -> 128 fp32 dy, 8     20 / 23   21 / 27   26 / 29   30 / 33   48 / 43    81 / 68   138 / 109
// The last is what a pair does not take: x to expand and no activation to hide it behind.
struct LinearFusedPlan {
  int chunks = 0, kc = 0, splits = 0, slots = 0, x_slots = 0, tiles = 0, workers = 0;
  LinearFusedPlan(const b200_linear_grad& g) {
    if (!g.dx || !g.dw || g.n > 512 || (g.act != kActNone && g.pre_dtype != g.dtype)) return;
    if (g.dy_pitch >= (1 << 28) || g.pre_pitch >= (1 << 28)) return;  // row pitches in bytes are 32 bits there
    const int c = (g.n + 127) / 128;
    kc = c <= 2 && g.k > 64 ? 128 : 64;  // two buffers of dx and the chunks of dw, 512 columns in all
    splits = (g.k + kc - 1) / kc;
    tiles = int((g.rows + 127) / 128);
    if (splits > 2 || tiles < (splits == 1 ? 8 : 148) || (splits == 2 && g.values && g.act == kActNone)) return;
    // slots a multiple of chunks: the warps of a chunk then meet every use of their slots, as the barriers' parities want it
    for (slots = 4 / c * c; slots >= 2; slots -= c)
      for (x_slots = 2; x_slots >= 1; --x_slots)
        if (linear_grad_smem(c, kc, slots, x_slots) <= 227 * 1024) {
          workers = std::min(splits == 1 ? sm_count() : linear_grad_pairs(linear_grad_smem(c, kc, slots, x_slots)), tiles);
          if (workers >= 1) chunks = c;
          return;
        }
  }
};

// Scratch of the backward pass, in this order: d, the parts of db, the parts of dw.
struct LinearGradPlan {
  LinearFusedPlan fused;
  bool own_d;
  int64_t db_parts;
  int splits;
  size_t d, db, dw, total;
  LinearGradPlan(const b200_linear_grad& g) : fused(g) {
    if (fused.chunks) {
      own_d = false;
      splits = fused.workers;
      db_parts = int64_t(fused.workers) * fused.splits;
      d = db = 0;
      dw = (size_t(db_parts) * g.n * 4 + 1023) / 1024 * 1024;
      total = dw + size_t(fused.workers) * g.n * g.k * 4;
      return;
    }
    own_d = g.act != kActNone || g.dy_dtype != g.dtype;
    db_parts = own_d || g.db ? linear_slope_parts(g.rows, g.n) : 0;
    splits = g.dw ? linear_dw_splits(g.rows, g.n, g.k) : 1;
    auto up = [](size_t b) { return (b + 1023) / 1024 * 1024; };
    d = 0;
    db = d + (own_d ? up(size_t(g.rows) * g.n * 2) : 0);
    dw = db + (g.db ? up(size_t(db_parts) * g.n * 4) : 0);
    total = dw + (splits > 1 ? up(size_t(splits) * g.n * g.k * 4) : 0);
  }
};

static int linear_grad_fused(const b200_linear_grad& g, const LinearGradPlan& plan, uint8_t* ws, cudaStream_t st) {
  const LinearFusedPlan& f = plan.fused;
  LinearGradParams p = {};
  p.dy = g.dy, p.dy_pitch = g.dy_pitch, p.a = g.pre, p.a_pitch = g.pre_pitch, p.act = g.act;
  p.values = static_cast<const uint8_t*>(g.values), p.exponents = g.exponents;
  p.dw = reinterpret_cast<float*>(ws + plan.dw), p.db = g.db ? reinterpret_cast<float*>(ws + plan.db) : nullptr;
  p.rows = g.rows, p.n = g.n, p.k = g.k, p.chunks = f.chunks, p.kc = f.kc, p.splits = f.splits, p.tiles = f.tiles, p.workers = f.workers;
  p.groups = f.chunks <= 2 ? 1 : 2;
  p.group_warps = kGradWarps / p.groups;
  p.slots = f.slots, p.x_slots = f.x_slots;
  uint32_t type = 0;
  if (g.dtype == B200_DTYPE_BF16) type = (1u << 7) | (1u << 10);
  const uint32_t shape = make_idesc_bf16(128, f.kc) & ~((7u << 7) | (7u << 10));
  p.idesc_dx = shape | type | (1u << 16);              // w across its rows
  p.idesc_dw = shape | type | (1u << 15) | (1u << 16);
  CUtensorMap tmW, tmX, tmDx;
  auto rows_map = [&](CUtensorMap* map, const void* base, int64_t rows, int64_t pitch, uint32_t box_cols, uint32_t box_rows,
                      CUtensorMapSwizzle swizzle) {
    const uint64_t dims[2] = {uint64_t(g.k), uint64_t(rows)};
    const uint64_t str[1] = {uint64_t(pitch) * 2};
    const uint32_t box[2] = {box_cols, box_rows};
    return make_tmap_bf16(map, base, 2, dims, str, box, swizzle);
  };
  if (int e = rows_map(&tmW, g.w, g.n, g.w_pitch, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  if (int e = rows_map(&tmDx, g.dx, g.rows, g.k, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B)) return e;
  tmX = tmDx;
  if (!g.values)
    if (int e = rows_map(&tmX, g.x, g.rows, g.x_pitch, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  const uint32_t smem = linear_grad_smem(f.chunks, f.kc, f.slots, f.x_slots);
  const int grid = f.workers * f.splits;
  auto go = [&](auto t, auto wide, auto act) -> int {
    if (p.values) return launch_cluster(linear_grad_kernel<decltype(t), wide(), act(), true>, grid, f.splits, kGradThreads, smem, st, tmW, tmX, tmDx, p);
    return launch_cluster(linear_grad_kernel<decltype(t), wide(), act(), false>, grid, f.splits, kGradThreads, smem, st, tmW, tmX, tmDx, p);
  };
  auto kinds = [&](auto t) -> int {
    const bool wide = g.dy_dtype == B200_DTYPE_F32, act = g.act != kActNone;
    if (wide) return act ? go(t, std::true_type(), std::true_type()) : go(t, std::true_type(), std::false_type());
    return act ? go(t, std::false_type(), std::true_type()) : go(t, std::false_type(), std::false_type());
  };
  if (int e = g.dtype == B200_DTYPE_BF16 ? kinds(__nv_bfloat16()) : kinds(__half())) return e;
  const int64_t size = int64_t(g.n) * g.k;
  if (int e = launch_part_sum(p.dw, f.workers, size, size, g.dw, g.dtype, nullptr, 0, st)) return e;
  return g.db ? launch_part_sum(p.db, plan.db_parts, g.n, g.n, g.db, g.db_dtype, nullptr, 0, st) : B200_OK;
}

static int linear_grad(const b200_linear_grad& g, void* workspace, cudaStream_t st) {
  const LinearGradPlan plan(g);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (plan.fused.chunks) return linear_grad_fused(g, plan, ws, st);
  const void* d = g.dy;
  int64_t d_pitch = g.dy_pitch;
  if (plan.own_d || g.db) {
    LinearSlopeParams p = {};
    p.dy = g.dy, p.dy_pitch = g.dy_pitch, p.dy_f32 = g.dy_dtype == B200_DTYPE_F32;
    p.a = g.pre, p.a_pitch = g.pre_pitch, p.a_f32 = g.pre_dtype == B200_DTYPE_F32;
    p.d = plan.own_d ? ws + plan.d : nullptr;
    p.partial = g.db ? reinterpret_cast<float*>(ws + plan.db) : nullptr;
    p.rows = g.rows, p.n = g.n;
    const dim3 grid(unsigned((g.n + 255) / 256), unsigned(plan.db_parts));
    auto go = [&](auto t, auto act) -> int {
      B200_LAUNCH((linear_slope_kernel<decltype(t), act()>), grid, 256, 0, st, p);
      return B200_OK;
    };
    auto acts = [&](auto t) -> int {
      if (g.act == kActRelu) return go(t, std::integral_constant<int, kActRelu>());
      if (g.act == kActGelu) return go(t, std::integral_constant<int, kActGelu>());
      if (g.act == kActGeluTanh) return go(t, std::integral_constant<int, kActGeluTanh>());
      if (g.act == kActSilu) return go(t, std::integral_constant<int, kActSilu>());
      return go(t, std::integral_constant<int, kActNone>());
    };
    if (int e = g.dtype == B200_DTYPE_BF16 ? acts(__nv_bfloat16()) : acts(__half())) return e;
    if (plan.own_d) d = ws + plan.d, d_pitch = g.n;
    if (g.db)
      if (int e = launch_part_sum(p.partial, plan.db_parts, g.n, g.n, g.db, g.db_dtype, nullptr, 0, st)) return e;
  }
  if (g.dx) {
    LinearProduct a{d, d_pitch, false, g.w, g.w_pitch, true, g.dx, g.k, int(g.rows), g.k, g.n, g.dtype, g.dtype};
    if (int e = launch_linear(a, st)) return e;
  }
  if (g.dw) {
    LinearProduct a{d, d_pitch, true, g.x, g.x_pitch, true, g.dw, g.k, g.n, g.k, int(g.rows), g.dtype, g.dtype};
    a.values = static_cast<const uint8_t*>(g.values), a.exponents = g.exponents;
    if (plan.splits > 1) {
      a.out = ws + plan.dw, a.out_dtype = B200_DTYPE_F32, a.splits = plan.splits;
      if (int e = launch_linear(a, st)) return e;
      const int64_t size = int64_t(g.n) * g.k;
      if (int e = launch_part_sum(reinterpret_cast<const float*>(ws + plan.dw), plan.splits, size, size, g.dw, g.dtype, nullptr, 0, st)) return e;
    } else if (int e = launch_linear(a, st)) {
      return e;
    }
  }
  return B200_OK;
}

}  // namespace b200
