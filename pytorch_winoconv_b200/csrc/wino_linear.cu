// Matrix products of the fully connected layers on the tensor cores (sm_100a), 16-bit operands, fp32 accumulate:
//
//     out[row][col] = sum over i of R[row, i] C[col, i]
//
//     forward          R = x  [M][K],  C = W [N][K]       z = out + bias,  y = act(z) + residual
//     data gradient    R = dz [M][N],  C = W read down its columns        dx
//     weight gradient  R = dz and C = x, both read down their columns     dW
//
// "Down its columns" is an MN-major operand of the MMA: TMA brings [reduction][64 rows] boxes as they lie, nothing is transposed
// for it.  The kernels need no scratch and no atomics and give the same bits every time.  (What TMA does not read has been copied before:
// rows that do not start on 16 bytes and float weights by pad_rows_kernel, a W that comes transposed by torch.)  Three forms, chosen by
// linear_plan:
//
//   row kernel      one or two rows: weights read once by plain loads, FMA                        (bound by HBM)
//   cluster kernel  few rows, few tiles: 128 columns x up to 256 rows by a cluster of CTAs        (HBM, or the launch)
//   pair kernel     256 rows x 256, 128 or 64 columns by a CTA pair, persistent                   (tensor pipe, or L2)
//
// Cluster kernel.  The 128 columns (output features) are the M side of the MMA and the rows its N side, so one row costs no more
// than 16 and the weights, which are what has to be read when rows are few, stream through a ring of TMA stages.  The CTAs of a
// cluster share the reduction; the parts are added up over distributed shared memory in the same order by every CTA, vectors of four
// read from all peers at once (sending single values to the CTA that finishes a row instead took 17.5 us where this took 10.8: 509 x 1000 x
// 1531).  Two CTAs to an SM where the ring fits twice.  24 x 4096 x 16384 (f16) 23.5 us, 5.7 TB/s of weights; 64 x 4096 x 4096 10.2 us
// and 16 x 4096 x 4096 8.1 us, of which the launch, the first loads, the exchange and the end take about 5.  Of 256 x 4096 x 4096's 15.5 us
// the steps take 6.2 (L2), the hand-over 1.4, the exchange 3.5 (128 KB an SM over distributed shared memory, 19 bytes a clock: as long with
// the sums of four rows in flight) and the end 0.9.
//
// Roles: warp 0 TMA, warp 1 MMA issue; then all eight warps move the accumulator to shared memory and add up and store their share
// of the rows.  Every mbarrier wait is bounded and reports through the error word.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <set>
#include <utility>

#include "wino_e4m3.cuh"
#include "wino_launch.h"
#include "wino_linear.h"

namespace wino {

__device__ unsigned int g_linear_error = 0;

namespace linear {

using namespace sm100;

constexpr int BK = 64;                 // reduction step of a stage: 64 values of 16 bits, one row of the 128-byte swizzle
constexpr int BC = 128;                // columns of a CTA
constexpr int C_BYTES = BC * BK * 2;   // of a stage
constexpr int BAR_BYTES = 256;
constexpr int SMS = 148;               // of a B200: what plans are made for

enum ErrCode : unsigned { ERR_EMPTY = 0x601, ERR_FULL = 0x602, ERR_DONE = 0x603, ERR_ACC_EMPTY = 0x604, ERR_ACC_FULL = 0x605 };

// What the epilogues need of a problem.
struct Out {
  int rows, cols, act, layer, bias_f32, out_f32, wide;      // wide: rows of y, z and residual take vectors
  const void *bias, *residual;
  void *y, *z;
  uint8_t *z8, *z8_scale;
  long long residual_stride, y_stride, z_stride;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// The same of a CTA pair: each CTA fills its own shared memory, the bytes are counted on rank 0's barrier.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & RANK0_MASK), "r"(c0), "r"(c1) : "memory");
}
// `n` rows from `row` on, reduction from `k` on: one box, or a box per 64 rows where the rows lie contiguous.
template <bool PAIR> __device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap *map, uint32_t bar, int mn, int row, int n, int k) {
  auto load = [&](uint32_t to, int c0, int c1) {
    if (PAIR) tma_load_2d_pair(to, map, bar, c0, c1);
    else tma_load_2d(to, map, bar, c0, c1);
  };
  if (!mn) load(dst, k, row);
  else
    for (int j = 0; j < n; j += 64) load(dst + (uint32_t)j * 128u, row + j, k);
}
// The same box on its way into L2.
__device__ __forceinline__ void prefetch_operand(const CUtensorMap *map, int mn, int row, int n, int k) {
  auto fetch = [&](int c0, int c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1) : "memory");
  };
  if (!mn) fetch(k, row);
  else
    for (int j = 0; j < n; j += 64) fetch(row + j, k);
}
__device__ __forceinline__ float ld_cluster_f1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// Low descriptor word of an operand tile and the step between its 16-value slices (16-byte units).  MN-major: blocks of 64 rows
// 8 KB apart, groups of eight reduction steps 1 KB apart; K-major: groups of eight rows 1 KB apart.
__device__ __forceinline__ uint32_t operand_lo(uint32_t saddr, int mn) { return desc_lo(saddr, mn ? 8192u : 16u); }
__device__ __forceinline__ uint32_t operand_step(int mn) { return mn ? 128u : 2u; }

// Long reductions.  The tensor cores cut products and sum off about two bits below the sum's last place, at every 16 values: sums of
// one sign lose 1.7 x 2^-24 of their value for each 16 (the worst of constant columns: 3.0; sums of both signs lose nothing that is seen),
// 1e-4 over 16384.  So an accumulator takes a run of the reduction at most, and the runs are added up in fp32, rounded to nearest, in
// tensor memory: the first run's accumulator holds the sum, the others' take turns in a second one.  A run is as long as half a step of the
// result's type allows: at worst 4.6e-5 in f32 results, 1.8e-4 in f16 (half a step: 2.4e-4 to 4.9e-4), 7.3e-4 in bf16 (2.0e-3 to
// 3.9e-3).  No wait lasts longer than a run, however long the reduction.
constexpr int RUN_F32 = 4096 / BK, RUN_F16 = 16384 / BK, RUN_BF16 = 65536 / BK;      // steps
int longest_run(const LinearProblem &p) { return p.out_f32 ? RUN_F32 : p.dtype == WINOCONV_F16 ? RUN_F16 : RUN_BF16; }
// Steps of each run but the last where `steps` are shared out evenly to runs of `longest` at most.
__host__ __device__ __forceinline__ int run_of(int steps, int longest) {
  const int runs = (steps + longest - 1) / longest;
  return (steps + runs - 1) / runs;
}
// 32 lanes x 32 columns of `sum` plus those of `run`.
__device__ __forceinline__ void add_run(uint32_t sum, uint32_t run) {
  uint32_t a[32], b[32];
  tmem_ld_x32(sum, a);
  tmem_ld_x32(run, b);
  tmem_wait_ld_x32(a);
  tmem_wait_ld_x32(b);
#pragma unroll
  for (int i = 0; i < 32; ++i) a[i] = __float_as_uint(__uint_as_float(a[i]) + __uint_as_float(b[i]));
  tmem_st_x32(sum, a);
}

// A lane's four columns of a row in the cluster kernel's epilogue.  WIDE: neighbours, moved as one vector; else 32 apart, so that a
// warp's accesses of single values are contiguous.
template <bool WIDE> __device__ __forceinline__ int column_of(int lane, int j) { return WIDE ? 4 * lane + j : lane + 32 * j; }
template <typename T, bool WIDE> __device__ __forceinline__ void load4(const T *row, int lane, int cols, float (&v)[4]) {
  if constexpr (WIDE) {
    if (4 * lane < cols) VecIO<T, 4>::load(row + 4 * lane, v);
    else v[0] = v[1] = v[2] = v[3] = 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lane + 32 * j < cols ? Elem<T>::load(row + lane + 32 * j) : 0.f;
  }
}
template <typename T, bool WIDE> __device__ __forceinline__ void store4(T *row, int lane, int cols, const float (&v)[4]) {
  if constexpr (WIDE) {
    if (4 * lane < cols) VecIO<T, 4>::store(row + 4 * lane, v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (lane + 32 * j < cols) Elem<T>::store(row + lane + 32 * j, v[j]);
  }
}
// The sums v of a row's 128 columns from `col` on, finished and stored.
template <typename T, bool WIDE>
__device__ __forceinline__ void finish4(const Out &o, int row, int col, int lane, float (&v)[4], const float (&bias)[4], const float (&residual)[4]) {
  const int cols = o.cols - col;      // left of the matrix from here on
  if (o.layer) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += bias[j];
    if (o.z8) {      // (columns beyond the last are zero: no part in a block's scale)
      float top[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) top[j] = e4m3::finite_magnitude(v[j]);
      if (WIDE) {    // a block is eight lanes' columns
        float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
        top[0] = top[1] = top[2] = top[3] = t;
      } else {       // or one column of every lane
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], d));
      }
      uint8_t *dst = o.z8 + (long long)row * o.cols + col, *scale = o.z8_scale + (long long)row * ((o.cols + e4m3::BLOCK - 1) / e4m3::BLOCK) + col / e4m3::BLOCK;
      if (WIDE) {
        const uint32_t byte = e4m3::scale_byte(top[0]);
        const float inv = e4m3::inverse_scale(byte);
        if (4 * lane < cols) {
          *reinterpret_cast<uint32_t *>(dst + 4 * lane) = e4m3::pack2(v[0], v[1], inv) | (e4m3::pack2(v[2], v[3], inv) << 16);
          if ((lane & 7) == 0) scale[lane >> 3] = (uint8_t)byte;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t byte = e4m3::scale_byte(top[j]);
          if (lane + 32 * j < cols) {
            dst[lane + 32 * j] = (uint8_t)e4m3::pack2(v[j], 0.f, e4m3::inverse_scale(byte));
            if (lane == 0) scale[j] = (uint8_t)byte;
          }
        }
      }
    }
    if (o.z) store4<T, WIDE>((T *)o.z + row * o.z_stride + col, lane, cols, v);
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const act::F2 y = act::apply(act::F2(v[j], v[j + 1]), o.act);
      v[j] = y.lo() + residual[j]; v[j + 1] = y.hi() + residual[j + 1];
    }
  }
  if (o.out_f32) store4<float, WIDE>((float *)o.y + row * o.y_stride + col, lane, cols, v);
  else store4<T, WIDE>((T *)o.y + row * o.y_stride + col, lane, cols, v);
}

// A warp's rows of a tile: j0, j0 + step, ... below n.  The bias and the residuals of the first PRE rows are loaded while the
// products are still on their way.
template <typename T, bool WIDE> struct RowEnd {
  static constexpr int PRE = 4;
  float bias[4] = {}, residual[PRE][4] = {};

  __device__ __forceinline__ void load(const Out &o, int row0, int col, int lane, int j, float (&r)[4]) const {
    load4<T, WIDE>((const T *)o.residual + (row0 + j) * o.residual_stride + col, lane, o.cols - col, r);
  }
  __device__ __forceinline__ void early(const Out &o, int row0, int col, int lane, int j0, int step, int n) {
    if (!o.layer) return;
    if (o.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = col + column_of<WIDE>(lane, j);
        if (c < o.cols) bias[j] = o.bias_f32 ? reinterpret_cast<const float *>(o.bias)[c] : Elem<T>::load((const T *)o.bias + c);
      }
    }
    if (o.residual) {
#pragma unroll
      for (int i = 0; i < PRE; ++i)
        if (j0 + i * step < n) load(o, row0, col, lane, j0 + i * step, residual[i]);
    }
  }
  // sums(j, v): a lane's four columns of row j, added up over the parts of the reduction
  template <typename Sums> __device__ __forceinline__ void run(const Out &o, int row0, int col, int lane, int j0, int step, int n, Sums &&sums) {
    float v[4];
#pragma unroll
    for (int i = 0; i < PRE; ++i) {
      const int j = j0 + i * step;
      if (j >= n) return;
      sums(j, v);
      finish4<T, WIDE>(o, row0 + j, col, lane, v, bias, residual[i]);
    }
#pragma unroll 1
    for (int j = j0 + PRE * step; j < n; j += step) {
      float r[4] = {0.f, 0.f, 0.f, 0.f};
      if (o.residual) load(o, row0, col, lane, j, r);
      sums(j, v);
      finish4<T, WIDE>(o, row0 + j, col, lane, v, bias, r);
    }
  }
};

// A row's sums over the S CTAs of a cluster, from the same place in the shared memory of each: all parts' values in flight at once,
// added in the same order by every CTA.
template <int S, bool WIDE> __device__ __forceinline__ void add_parts(uint32_t sums, int j, int lane, float (&v)[4]) {
  float u[S][4];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const uint32_t row = map_to_rank(sums + (uint32_t)((j * BC + (WIDE ? 4 * lane : lane)) * 4), (uint32_t)i);
    if (WIDE) {
      const float4 t = ld_cluster_f4(row);
      u[i][0] = t.x; u[i][1] = t.y; u[i][2] = t.z; u[i][3] = t.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) u[i][c] = ld_cluster_f1(row + 128u * c);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    v[c] = u[0][c];
#pragma unroll
    for (int i = 1; i < S; ++i) v[c] += u[i][c];
  }
}

struct ClusterArgs {
  int n_steps, longest_run, n_rt, tile_rows, stages, r_mn, c_mn;
  uint32_t idesc;
};

constexpr int CLUSTER_THREADS = 256;
constexpr int CLUSTER_SMEM2 = 113 * 1024;      // of an SM's 228 KB for each of two CTAs, 1 KB of which is the system's

template <typename T, bool WIDE>
__global__ void __launch_bounds__(CLUSTER_THREADS, 2)
    cluster_kernel(const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Out o,
                   const __grid_constant__ ClusterArgs g, int split) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - raw);
  const uint32_t stage_bytes = (uint32_t)(C_BYTES + g.tile_rows * BK * 2);
  const uint32_t ring = max((uint32_t)g.stages * stage_bytes, (uint32_t)(g.tile_rows * BC * 4));      // or the sums, whichever is longer
  const uint32_t bars = base + ring;      // full[8] empty[8] done run_full run_free
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 64u + 8u * i; };
  const uint32_t done = bars + 128u, run_full = bars + 136u, run_free = bars + 144u, tmem_slot = bars + 196u;
  volatile unsigned *abort_word = reinterpret_cast<volatile unsigned *>(base_ptr + ring + 192);
  unsigned *err = &g_linear_error;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const uint32_t part = split > 1 ? cluster_ctarank() : 0u;
  const int tile = (int)blockIdx.x / split, ct = tile / g.n_rt, rt = tile - ct * g.n_rt;      // CTAs in flight share columns: the weights are read once
  const int row0 = rt * g.tile_rows, col0 = ct * BC;
  const int k0 = (int)((long long)g.n_steps * part / split), k1 = (int)((long long)g.n_steps * (part + 1) / split);
  const int run_steps = run_of(k1 - k0, g.longest_run), runs = (k1 - k0 + run_steps - 1) / run_steps;
  uint32_t acc_cols = 32;
  while (acc_cols < (uint32_t)g.tile_rows) acc_cols *= 2;
  const uint32_t tmem_cols = runs > 1 ? 2u * acc_cols : acc_cols;

  if (warp == 1 && lane == 0) prefetch_map(&map_r);
  // The first stages of C (the weights) are sent for while this kernel sets itself up and the one before it ends; into L2 only,
  // where the writes of the one before it would arrive too, should it be the one that changes them.
  if (warp == 3 && lane < g.stages && k0 + lane < k1) prefetch_operand(&map_c, g.c_mn, col0, BC, (k0 + lane) * BK);
  if (warp == 0) {
    if (lane < 8) { mbar_init(full(lane), 1); mbar_init(empty(lane), 1); }
    else if (lane == 8) { mbar_init(done, 1); mbar_init(run_full, 1); mbar_init(run_free, CLUSTER_THREADS / 32 - 2); }
    else if (lane == 9) *abort_word = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) tmem_alloc<false>(tmem_slot, tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  grid_dependency_wait();
  const int n = min(g.tile_rows, o.rows - row0);
  RowEnd<T, WIDE> end;
  end.early(o, row0, col0, lane, (int)part + warp * split, 8 * split, n);

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 1;
    for (int k = k0; k < k1; ++k) {
      if (!mbar_wait_warp(empty(s), ph, abort_word, err, ERR_EMPTY)) break;
      if (lane == 0) {
        mbar_expect_tx(full(s), stage_bytes);
        const uint32_t dst = base + (uint32_t)s * stage_bytes;
        load_operand<false>(dst, &map_c, full(s), g.c_mn, col0, BC, k * BK);
        load_operand<false>(dst + C_BYTES, &map_r, full(s), g.r_mn, row0, g.tile_rows, k * BK);
      }
      if (++s == g.stages) { s = 0; ph ^= 1u; }
    }
    if (*abort_word != 0u) {   // loads in flight must land before the shared memory goes away
      const long long start = clock64();
      while (clock64() - start < 2000000LL) { }
    }
  } else if (warp == 1) {
    int s = 0, k = k0;
    uint32_t ph = 0;
    bool alive = true;
    for (int run = 0; run < runs && alive; ++run) {
      if (run > 0) {
        if (!mbar_wait_warp(run_free, (uint32_t)(run - 1) & 1u, abort_word, err, ERR_ACC_EMPTY)) { alive = false; break; }
        tc_fence_after();
      }
      const int first = k, last = min(k + run_steps, k1);
      const uint32_t d = run > 0 ? tmem + acc_cols : tmem;
      for (; k < last; ++k) {
        if (!mbar_wait_warp(full(s), ph, abort_word, err, ERR_FULL)) { alive = false; break; }
        tc_fence_after();
        const uint32_t st = base + (uint32_t)s * stage_bytes;
        const uint32_t a = operand_lo(st, g.c_mn), b = operand_lo(st + C_BYTES, g.r_mn), hi = desc_hi(1024, 2);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            umma<false, false>(d, a + (uint32_t)j * operand_step(g.c_mn), hi, b + (uint32_t)j * operand_step(g.r_mn), hi, g.idesc, (k > first || j > 0) ? 1u : 0u);
          umma_commit<false>(empty(s), 0);
        }
        __syncwarp();
        if (++s == g.stages) { s = 0; ph ^= 1u; }
      }
      if (alive && elect_one()) umma_commit<false>(run + 1 < runs ? run_full : done, 0);
      __syncwarp();
    }
  } else {
    // every run but the last: the second accumulator into the first (all six warps answer, so that none falls two runs behind)
    for (int run = 0; run + 1 < runs; ++run) {
      if (!mbar_wait_warp(run_full, (uint32_t)run & 1u, abort_word, err, ERR_ACC_FULL)) break;
      tc_fence_after();
      if (run > 0 && warp >= 4) {
        const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < n; c += 32) add_run(at + (uint32_t)c, at + acc_cols + (uint32_t)c);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(run_free);
    }
  }
  __syncwarp();
  // sums to shared memory: [row][128 columns]
  const bool ok = mbar_wait_warp(done, 0, abort_word, err, ERR_DONE);
  grid_launch_dependents();
  float *sums = reinterpret_cast<float *>(base_ptr);
  if (ok && *abort_word == 0u) {
    tc_fence_after();
    const int q = warp & 3;
    for (int c = (warp >> 2) * 32; c < n; c += 64) {
      uint32_t v[32];
      tmem_ld_x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, v);
      tmem_wait_ld_x32(v);
      if (runs > 1) {      // the last run's
        uint32_t u[32];
        tmem_ld_x32(tmem + ((uint32_t)(q * 32) << 16) + acc_cols + (uint32_t)c, u);
        tmem_wait_ld_x32(u);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
      }
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j < n) sums[(c + j) * BC + q * 32 + lane] = __uint_as_float(v[j]);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_free<false>(tmem, tmem_cols);
  }
  __syncwarp();
  if (split > 1) cluster_sync_all();
  if (*abort_word == 0u) {
    end.run(o, row0, col0, lane, (int)part + warp * split, 8 * split, n, [&](int j, float (&v)[4]) {
      if (split == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sums[j * BC + column_of<WIDE>(lane, i)];
        return;
      }
      if (split == 2) add_parts<2, WIDE>(base, j, lane, v);
      else if (split == 4) add_parts<4, WIDE>(base, j, lane, v);
      else add_parts<8, WIDE>(base, j, lane, v);
    });
  }
  __syncwarp();
  if (split > 1) cluster_sync_all();      // no CTA leaves while another reads its shared memory
}

// ---- row kernel ------------------------------------------------------------------------------------------------------
// One or two rows against weights that are read once: a block takes four rows of W and all of x, its threads eight neighbouring
// values of the reduction each, twice before the first products; products by FMA (two values an instruction), and no set-up of
// barriers and tensor memory.  Sums: a thread's own in the order of the reduction, then over the lanes, then over the warps.
//
// What bounds it is the read of W: one row of 4096 -> 16384 or 16384 -> 4096 (bf16) 20.7 us, 6.5 TB/s; 4096 -> 4096 7.2 us for 34 MB,
// two of which are the launch (the cluster kernel: 24.0, 23.8 and 9.0 us).  Eight rows of W and one step, or no word to L2 ahead of
// the kernel before: 9.6 and 7.5 us.  From three rows on the products cost more than the set-up (10.5 us against 8.6).
constexpr int ROW_THREADS = 256, ROW_FEATURES = 4, MOST_ROWS = 2;

// Lane sums of V values by halving: afterwards v[0] of a lane is the sum over the warp of value lane / (32 / V).
template <int V> __device__ __forceinline__ void sum_lanes(float (&v)[V], int lane) {
#pragma unroll
  for (int n = V, d = 16; n > 1; n >>= 1, d >>= 1) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const bool up = (lane & d) != 0;
      const float keep = up ? v[i + n / 2] : v[i], send = up ? v[i] : v[i + n / 2];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
    }
  }
#pragma unroll
  for (int d = 16 / V; d > 0; d >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
}

template <typename T, int ROWS, bool WIDE>
__global__ void __launch_bounds__(ROW_THREADS, 3) row_kernel(const T *x, long long x_stride, const T *w, long long w_stride, int red,
                                                          const __grid_constant__ Out o) {
  using act::F2;
  constexpr int FEATURES = ROW_FEATURES, V = ROWS * FEATURES, WARPS = ROW_THREADS / 32;
  static_assert(V <= 32, "a lane for every sum");
  __shared__ float part[WARPS][V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col0 = (int)blockIdx.x * FEATURES;
  const T *wr[FEATURES];
#pragma unroll
  for (int f = 0; f < FEATURES; ++f) wr[f] = w + (long long)min(col0 + f, o.cols - 1) * w_stride;
  if (WIDE) {      // the first steps' weights on their way to L2 while the kernel before this one ends
    const int k = threadIdx.x * 64;
    if (k < min(red, ROW_THREADS * 16))
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) asm volatile("prefetch.global.L2 [%0];" ::"l"(wr[f] + k));
  }
  grid_launch_dependents();
  grid_dependency_wait();
  float v[V];
  if constexpr (WIDE) {
    F2 acc[ROWS][FEATURES];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) acc[r][f] = F2(0.f);
#pragma unroll 2
    for (int k = threadIdx.x * 8; k < red; k += ROW_THREADS * 8) {
      uint4 wv[FEATURES], xv[ROWS];
#pragma unroll
      for (int f = 0; f < FEATURES; ++f)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(wv[f].x), "=r"(wv[f].y), "=r"(wv[f].z), "=r"(wv[f].w) : "l"(wr[f] + k));
#pragma unroll
      for (int r = 0; r < ROWS; ++r) xv[r] = r < o.rows ? *reinterpret_cast<const uint4 *>(x + r * x_stride + k) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        F2 xs[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float2 t = Pair16<T>::unpack(i == 0 ? xv[r].x : i == 1 ? xv[r].y : i == 2 ? xv[r].z : xv[r].w);
          xs[r] = F2(t.x, t.y);
        }
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) {
          const float2 t = Pair16<T>::unpack(i == 0 ? wv[f].x : i == 1 ? wv[f].y : i == 2 ? wv[f].z : wv[f].w);
          const F2 ws(t.x, t.y);
#pragma unroll
          for (int r = 0; r < ROWS; ++r) acc[r][f] = act::fma2(xs[r], ws, acc[r][f]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) v[r * FEATURES + f] = acc[r][f].lo() + acc[r][f].hi();
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
#pragma unroll 2
    for (int k = threadIdx.x; k < red; k += ROW_THREADS) {
      float ws[FEATURES];
#pragma unroll
      for (int f = 0; f < FEATURES; ++f) ws[f] = Elem<T>::load(wr[f] + k);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float xs = r < o.rows ? Elem<T>::load(x + r * x_stride + k) : 0.f;
#pragma unroll
        for (int f = 0; f < FEATURES; ++f) v[r * FEATURES + f] = fmaf(xs, ws[f], v[r * FEATURES + f]);
      }
    }
  }
  sum_lanes<V>(v, lane);
  constexpr int LANES = 32 / V;
  const int index = lane / LANES;
  if (lane % LANES == 0) part[warp][index] = v[0];
  __syncthreads();
  if (threadIdx.x >= V) return;
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) z += part[i][threadIdx.x];
  const int row = threadIdx.x / FEATURES, col = col0 + threadIdx.x % FEATURES;
  if (row >= o.rows || col >= o.cols) return;
  if (o.bias) z += o.bias_f32 ? reinterpret_cast<const float *>(o.bias)[col] : Elem<T>::load((const T *)o.bias + col);
  if (o.z) Elem<T>::store((T *)o.z + row * o.z_stride + col, z);
  float y = act::apply(F2(z), o.act).lo();
  if (o.residual) y += Elem<T>::load((const T *)o.residual + row * o.residual_stride + col);
  Elem<T>::store((T *)o.y + row * o.y_stride + col, y);
}

// ---- pair kernel -----------------------------------------------------------------------------------------------------
// Many rows: a tile of 256 rows x BN columns by a CTA pair (cta_group::2, M = 256: each CTA loads half of both operands and holds
// the sums of its 128 rows), a persistent grid, two accumulators so that eight epilogue warps finish a tile beside the next one's
// products.  What bounds it: with 256 columns the tensor pipe under the power cap (8192 x 4096 x 16384 in bf16 0.65 ms in short runs,
// 1690 TFLOP/s; 0.79 ms in long ones, where the library product takes 0.78); with 128 and 64, for problems of few tiles, the L2 (a step of
// 64 takes 0.20 and 0.18 us where the pipe would take 0.14 and 0.07; four stages instead of eight 0.31, words to L2 ahead of the loads
// only add to its work; 512 x 4096 x 4096 18.1 us with 128 columns, 26.3 with 256, 22.0 by the cluster kernel).
constexpr int PAIR_THREADS = 384;
constexpr int PAIR_ROWS = 256;                                    // of a tile; a CTA holds half of each operand
constexpr int PAIR_WARPS = 8;                                     // of the epilogue
constexpr int TURN_BYTES = 2048, BIAS_BYTES = 512;                // per epilogue warp: 32 rows x 64 bytes, bias of its columns
// What a tile of BN columns takes: bytes of a stage that a CTA loads, stages, places in shared memory.
template <int BN> struct PairTile {
  static constexpr int R_BYTES = 128 * BK * 2, STAGE = R_BYTES + BN / 2 * BK * 2, STAGES = BN == 256 ? 6 : 8;
  static constexpr int OFF_TURN = STAGES * STAGE, OFF_BIAS = OFF_TURN + PAIR_WARPS * TURN_BYTES, OFF_BARS = OFF_BIAS + PAIR_WARPS * BIAS_BYTES;
  static constexpr int SMEM = 1024 + OFF_BARS + BAR_BYTES;
  static_assert(SMEM <= 227 * 1024 && STAGE % 1024 == 0, "shared memory");
};

struct PairArgs {
  int n_steps, run_steps, runs, n_rt, n_ct, n_tiles, band, r_mn, c_mn;
  uint32_t idesc;
};
// Tiles are walked in bands of tile rows, column by column: the pairs at work at one time share few rows and few columns, which then
// come from L2, and a band's rows stay there while all columns pass by.  Eight tile rows, or up to sixteen while their operand takes
// no more than 36 MB of the L2: the columns are then read half as often (8192 x 4096 x 16384 in long runs, 4 / 8 / 16: 820 / 797 / 781 us;
// 8192 x 16384 x 4096: 803 / 806 / 816).
__device__ __forceinline__ void tile_at(const PairArgs &g, int t, int &rt, int &ct) {
  const int per = g.band * g.n_ct, band = t / per, r = t - band * per, n = min(g.band, g.n_rt - band * g.band);
  ct = r / n;
  rt = band * g.band + (r - ct * n);
}
int band_of(int red) { return (int)std::min(16LL, std::max(8LL, 36000000LL / ((long long)PAIR_ROWS * red * 2))); }

// 64 bytes of each of a warp's 32 rows (lane = row), turned in shared memory so that the stores of a row are contiguous.  EL:
// bytes of an element; `rows` and `cols` are what is left of the matrix from here on.
template <int EL>
__device__ __forceinline__ void store_rows(uint8_t *turn, const uint32_t (&w)[16], uint8_t *dst, long long stride, int rows, int cols, int wide, int lane) {
  uint4 *mine = reinterpret_cast<uint4 *>(turn + lane * 64);
#pragma unroll
  for (int i = 0; i < 4; ++i) mine[i ^ ((lane >> 1) & 3)] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
  if (wide) {
    const int c = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2);
      const uint4 v = *reinterpret_cast<const uint4 *>(turn + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
      if (r < rows && c * (16 / EL) < cols) *reinterpret_cast<uint4 *>(dst + r * stride + c * 16) = v;
    }
  } else {
    constexpr int PER = 64 / EL, RS = 32 / PER;      // elements of a row, rows a time
    const int c = lane % PER;
    for (int r = lane / PER; r < min(32, rows); r += RS) {
      const uint8_t *src = turn + r * 64 + ((((c * EL) >> 4) ^ ((r >> 1) & 3)) << 4) + ((c * EL) & 15);
      if (c < cols) {
        if constexpr (EL == 2) *reinterpret_cast<uint16_t *>(dst + r * stride + c * 2) = *reinterpret_cast<const uint16_t *>(src);
        else *reinterpret_cast<float *>(dst + r * stride + c * 4) = *reinterpret_cast<const float *>(src);
      }
    }
  }
  __syncwarp();
}
// The counterpart for 16-bit rows that take no vectors: 32 columns of each row, as the lane that holds the row wants them.
__device__ __forceinline__ void load_rows(uint8_t *turn, uint32_t (&w)[16], const uint8_t *src, long long stride, int rows, int cols, int lane) {
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    const uint16_t v = r < rows && lane < cols ? *reinterpret_cast<const uint16_t *>(src + r * stride + lane * 2) : (uint16_t)0;
    *reinterpret_cast<uint16_t *>(turn + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2) = v;
  }
  __syncwarp();
  const uint4 *mine = reinterpret_cast<const uint4 *>(turn + lane * 64);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 v = mine[i ^ ((lane >> 1) & 3)];
    w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
  }
  __syncwarp();
}

// ACT: the activation of a layer; -1: the product alone.  LONG: a reduction of several runs, with any activation where it is a layer.  (A
// kernel of its own: the runs in the epilogue's loop over tiles cost the others up to 2 %, 8192 x 256 x 8192 72.0 us instead of 70.5.)
template <typename T, int ACT, int BN, bool LONG>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Out o,
                const __grid_constant__ PairArgs g) {
  using P = PairTile<BN>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - raw);
  const uint32_t bars = base + P::OFF_BARS;      // full[8] empty[8] acc_full[2] acc_empty[2]
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 64u + 8u * i; };
  auto acc_full = [&](int i) { return bars + 128u + 8u * i; };
  auto acc_empty = [&](int i) { return bars + 144u + 8u * i; };
  const uint32_t tmem_slot = bars + 196u;
  volatile unsigned *abort_word = reinterpret_cast<volatile unsigned *>(base_ptr + P::OFF_BARS + 192);
  unsigned *err = &g_linear_error;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == 1 && lane == 0) { prefetch_map(&map_r); prefetch_map(&map_c); }
  if (warp == 0) {
    if (lane < 8) { mbar_init(full(lane), 1); mbar_init(empty(lane), 1); }
    else if (lane < 10) { mbar_init(acc_full(lane - 8), 1); mbar_init(acc_empty(lane - 8), 2 * PAIR_WARPS); }
    else if (lane == 10) *abort_word = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;                   // issues the MMAs of the pair
  if (warp == 2) tmem_alloc<true>(tmem_slot, 2 * BN);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                              // the barriers of both CTAs exist before either arrives at the other's
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  tmem = __shfl_sync(0xffffffffu, tmem, 0);
  grid_launch_dependents();
  grid_dependency_wait();

  const int tile0 = (int)blockIdx.x >> 1, tile_step = (int)gridDim.x >> 1;
  if (warp == 0) {
    int s = 0;
    uint32_t ph = 1;
    bool alive = true;
    for (int t = tile0; t < g.n_tiles && alive; t += tile_step) {
      int rt, ct;
      tile_at(g, t, rt, ct);
      const int row = rt * PAIR_ROWS + (int)rank * 128, col = ct * BN + (int)rank * (BN / 2);
      for (int k = 0; k < g.n_steps; ++k) {
        if (!mbar_wait_warp(empty(s), ph, abort_word, err, ERR_EMPTY)) { alive = false; break; }
        if (lane == 0) {
          if (leader) mbar_expect_tx(full(s), 2u * P::STAGE);
          const uint32_t dst = base + (uint32_t)(s * P::STAGE);
          load_operand<true>(dst, &map_r, full(s), g.r_mn, row, 128, k * BK);
          load_operand<true>(dst + P::R_BYTES, &map_c, full(s), g.c_mn, col, BN / 2, k * BK);
        }
        if (++s == P::STAGES) { s = 0; ph ^= 1u; }
      }
    }
    if (*abort_word != 0u) {   // loads in flight must land before the shared memory goes away
      const long long start = clock64();
      while (clock64() - start < 2000000LL) { }
    }
  } else if (warp == 1 && leader) {
    int s = 0, n = 0;
    uint32_t ph = 0, used = 0;      // used: how often each accumulator has been, modulo two, a bit for each
    bool alive = true;
    const uint32_t hi = desc_hi(1024, 2), a_step = operand_step(g.r_mn), b_step = operand_step(g.c_mn);
    for (int t = tile0; t < g.n_tiles && alive; t += tile_step, ++n) {
      int k = 0;
      for (int run = 0; run < g.runs && alive; ++run) {      // the first in one accumulator, the others in turn in the other: the next tile's first
        const int buf = (n + (run > 0)) & 1;
        if (!mbar_wait_warp(acc_empty(buf), ((used >> buf) & 1u) ^ 1u, abort_word, err, ERR_ACC_EMPTY)) { alive = false; break; }
        used ^= 1u << buf;
        tc_fence_after();
        const int first = k, last = min(k + g.run_steps, g.n_steps);
        const uint32_t d = tmem + (uint32_t)(buf * BN);
        for (; k < last; ++k) {
          if (!mbar_wait_warp(full(s), ph, abort_word, err, ERR_FULL)) { alive = false; break; }
          tc_fence_after();
          const uint32_t st = base + (uint32_t)(s * P::STAGE);
          const uint32_t a = operand_lo(st, g.r_mn), b = operand_lo(st + P::R_BYTES, g.c_mn);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) umma<true, false>(d, a + (uint32_t)j * a_step, hi, b + (uint32_t)j * b_step, hi, g.idesc, (k > first || j > 0) ? 1u : 0u);
            umma_commit<true>(empty(s), 3);
          }
          __syncwarp();
          if (++s == P::STAGES) { s = 0; ph ^= 1u; }
        }
        if (alive && elect_one()) umma_commit<true>(acc_full(buf), 3);
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    const int ew = warp - 4, q = warp & 3, half = ew >> 2;
    uint8_t *turn = base_ptr + P::OFF_TURN + ew * TURN_BYTES;
    float *bias = reinterpret_cast<float *>(base_ptr + P::OFF_BIAS + ew * BIAS_BYTES);
    const int n_blk = (o.cols + e4m3::BLOCK - 1) / e4m3::BLOCK;
    int n = 0;
    [[maybe_unused]] uint32_t used = 0;
    for (int t = tile0; t < g.n_tiles; t += tile_step, ++n) {
      int rt, ct;
      tile_at(g, t, rt, ct);
      const int buf = n & 1;
      const int row0 = rt * PAIR_ROWS + (int)rank * 128 + q * 32, col0 = ct * BN + half * (BN / 2), rows = o.rows - row0;
      if (ACT >= 0) {
#pragma unroll
        for (int j = 0; j < BN / 64; ++j) {
          const int c = col0 + j * 32 + lane;
          bias[j * 32 + lane] = !o.bias || c >= o.cols ? 0.f : o.bias_f32 ? reinterpret_cast<const float *>(o.bias)[c] : Elem<T>::load((const T *)o.bias + c);
        }
        __syncwarp();
      }
      if (!mbar_wait_warp(acc_full(buf), LONG ? (used >> buf) & 1u : (uint32_t)(n >> 1) & 1u, abort_word, err, ERR_ACC_FULL)) break;
      tc_fence_after();
      if constexpr (LONG) {
        used ^= 1u << buf;
        bool alive = true;
        for (int run = 1; run < g.runs && alive; ++run) {      // the other accumulator into this one
          const int from = buf ^ 1;
          alive = mbar_wait_warp(acc_full(from), (used >> from) & 1u, abort_word, err, ERR_ACC_FULL);
          used ^= 1u << from;
          tc_fence_after();
          const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * (BN / 2));
#pragma unroll 1
          for (int ch = 0; ch < BN / 64 && alive; ++ch)
            if (rows > 0 && col0 + ch * 32 < o.cols) add_run(at + (uint32_t)(buf * BN + ch * 32), at + (uint32_t)(from * BN + ch * 32));
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_rank0(acc_empty(from));
        }
        if (!alive) break;
      }
#pragma unroll 1
      for (int ch = 0; ch < BN / 64; ++ch) {
        const int c = col0 + ch * 32, cols = o.cols - c;
        if (cols <= 0 || rows <= 0) break;
        uint32_t v[32];
        tmem_ld_x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * (BN / 2) + ch * 32), v);
        uint32_t res[16];
        if (ACT >= 0 && o.residual) {      // on its way while the accumulator is read
          const uint8_t *src = (const uint8_t *)o.residual + ((long long)row0 * o.residual_stride + c) * 2;
          if (o.wide) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 u = make_uint4(0u, 0u, 0u, 0u);
              if (lane < rows && i * 8 < cols) u = *reinterpret_cast<const uint4 *>(src + lane * o.residual_stride * 2 + i * 16);
              res[4 * i] = u.x; res[4 * i + 1] = u.y; res[4 * i + 2] = u.z; res[4 * i + 3] = u.w;
            }
          } else load_rows(turn, res, src, o.residual_stride * 2, rows, cols, lane);
        }
        tmem_wait_ld_x32(v);
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
        uint32_t w[16];
        if constexpr (ACT >= 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 b = *reinterpret_cast<const float4 *>(bias + ch * 32 + i * 4);
            f[4 * i] += b.x; f[4 * i + 1] += b.y; f[4 * i + 2] += b.z; f[4 * i + 3] += b.w;
          }
          if (o.z) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = Pair16<T>::round(f[2 * i], f[2 * i + 1]);
            store_rows<2>(turn, w, (uint8_t *)o.z + ((long long)row0 * o.z_stride + c) * 2, o.z_stride * 2, rows, cols, o.wide, lane);
          }
          if (o.z8) {      // a lane's 32 columns are a block (columns beyond the last are zero)
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, e4m3::finite_magnitude(f[i]));
            const uint32_t byte = e4m3::scale_byte(top);
            const float inv = e4m3::inverse_scale(byte);
            uint32_t p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = e4m3::pack2(f[4 * i], f[4 * i + 1], inv) | (e4m3::pack2(f[4 * i + 2], f[4 * i + 3], inv) << 16);
            uint8_t *dst = o.z8 + (long long)row0 * o.cols + c;
            if ((o.cols & 15) == 0) {
              if (lane < rows) {
                uint4 *d4 = reinterpret_cast<uint4 *>(dst + (long long)lane * o.cols);
                d4[0] = make_uint4(p[0], p[1], p[2], p[3]);
                if (cols > 16) d4[1] = make_uint4(p[4], p[5], p[6], p[7]);
              }
            } else {
              uint4 *mine = reinterpret_cast<uint4 *>(turn + lane * 32);
              mine[0] = make_uint4(p[0], p[1], p[2], p[3]);
              mine[1] = make_uint4(p[4], p[5], p[6], p[7]);
              __syncwarp();
              for (int r = 0; r < min(32, rows); ++r)
                if (lane < cols) dst[(long long)r * o.cols + lane] = turn[r * 32 + lane];
              __syncwarp();
            }
            if (lane < rows) o.z8_scale[(long long)(row0 + lane) * n_blk + c / e4m3::BLOCK] = (uint8_t)byte;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const act::F2 y = act::apply(act::F2(f[i], f[i + 1]), LONG ? o.act : ACT);
            f[i] = y.lo(); f[i + 1] = y.hi();
          }
          if (o.residual) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 r = Pair16<T>::unpack(res[i]);
              f[2 * i] += r.x;
              f[2 * i + 1] += r.y;
            }
          }
        }
        if (ACT < 0 && o.out_f32) {
          uint8_t *dst = (uint8_t *)o.y + ((long long)row0 * o.y_stride + c) * 4;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(f[16 * h + i]);
            store_rows<4>(turn, w, dst + h * 64, o.y_stride * 4, rows, cols - 16 * h, o.wide, lane);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = Pair16<T>::round(f[2 * i], f[2 * i + 1]);
          store_rows<2>(turn, w, (uint8_t *)o.y + ((long long)row0 * o.y_stride + c) * 2, o.y_stride * 2, rows, cols, o.wide, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_rank0(acc_empty(buf));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 2) {
    tc_fence_after();
    tmem_free<true>(tmem, 2 * BN);
  }
}

// Boxes of 64 x `rows` (K-major) or 64 rows x 64 reduction steps (MN-major), zeros beyond the operand's ends.
bool operand_map(CUtensorMap *m, EncodeTiledFn enc, int dtype, const MatOperand &p, int rows, int red, int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)(p.mn ? rows : red), (cuuint64_t)(p.mn ? red : rows)}, st[1] = {(cuuint64_t)p.stride * 2};
  cuuint32_t box[2] = {64u, p.mn ? 64u : (cuuint32_t)box_rows}, es[2] = {1u, 1u};
  return enc(m, map_dtype(dtype), 2, const_cast<void *>(p.ptr), dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint32_t instruction(int dtype, int a_mn, int b_mn, int m, int n) {
  const uint32_t fmt = dtype == WINOCONV_F16 ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

bool multiple(const void *p, long long stride, int el, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0 && stride * el % bytes == 0;
}

Out out_of(const LinearProblem &p, int width) {      // width: columns of a vector access
  Out o;
  o.rows = p.rows; o.cols = p.cols; o.act = p.act; o.layer = p.layer; o.bias_f32 = p.bias_f32; o.out_f32 = p.out_f32;
  o.bias = p.bias; o.residual = p.residual; o.y = p.y; o.z = p.z; o.z8 = p.z8; o.z8_scale = p.z8_scale;
  o.residual_stride = p.residual_stride; o.y_stride = p.y_stride; o.z_stride = p.z_stride;
  const int el = p.out_f32 ? 4 : 2;
  o.wide = p.cols % width == 0 && multiple(p.y, p.y_stride, el, std::min(16, el * width)) && (!p.residual || multiple(p.residual, p.residual_stride, 2, 2 * width)) &&
           (!p.z || multiple(p.z, p.z_stride, 2, 2 * width));
  return o;
}

// All of an SM's shared memory for a kernel, asked for once on each device.
cudaError_t allow_smem(const void *kern) {
  static std::mutex mu;
  static std::set<std::pair<const void *, int>> done;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kern, dev})) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
  if (e == cudaSuccess) done.insert({kern, dev});
  return e;
}

int cluster_smem(const LinearPlan &plan) {
  return 1024 + std::max(plan.stages * (C_BYTES + plan.tile_rows * BK * 2), plan.tile_rows * BC * 4) + BAR_BYTES;
}

template <typename T>
cudaError_t launch_cluster(const LinearProblem &p, const LinearPlan &plan, EncodeTiledFn enc, cudaStream_t s, const char **detail) {
  CUtensorMap mr, mc;
  if (!operand_map(&mr, enc, p.dtype, p.r, p.rows, p.red, plan.tile_rows) || !operand_map(&mc, enc, p.dtype, p.c, p.cols, p.red, BC)) {
    *detail = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  const Out o = out_of(p, 4);
  auto kern = o.wide ? cluster_kernel<T, true> : cluster_kernel<T, false>;
  cudaError_t e = allow_smem((const void *)kern);
  if (e != cudaSuccess) return e;
  ClusterArgs g;
  g.n_steps = (p.red + BK - 1) / BK;
  g.n_rt = (p.rows + plan.tile_rows - 1) / plan.tile_rows;
  g.longest_run = longest_run(p);
  g.tile_rows = plan.tile_rows; g.stages = plan.stages; g.r_mn = p.r.mn; g.c_mn = p.c.mn;
  g.idesc = instruction(p.dtype, p.c.mn, p.r.mn, 128, plan.tile_rows);
  const int n_ct = (p.cols + BC - 1) / BC;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.n_rt * n_ct * plan.split)); cfg.blockDim = dim3(CLUSTER_THREADS);
  cfg.dynamicSmemBytes = (size_t)cluster_smem(plan); cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)plan.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = plan.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, mr, mc, o, g, plan.split);
}

template <typename T> cudaError_t launch_rows(const LinearProblem &p, cudaStream_t s) {
  const bool wide = p.red % 8 == 0 && multiple(p.r.ptr, p.r.stride, 2, 16) && multiple(p.c.ptr, p.c.stride, 2, 16);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.cols + ROW_FEATURES - 1) / ROW_FEATURES)); cfg.blockDim = dim3(ROW_THREADS); cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  auto kern = p.rows == 1 ? (wide ? row_kernel<T, 1, true> : row_kernel<T, 1, false>) : (wide ? row_kernel<T, 2, true> : row_kernel<T, 2, false>);
  return cudaLaunchKernelEx(&cfg, kern, (const T *)p.r.ptr, p.r.stride, (const T *)p.c.ptr, p.c.stride, p.red, out_of(p, 1));
}

template <typename T, int ACT, int BN, bool LONG> cudaError_t launch_pair(const LinearProblem &p, EncodeTiledFn enc, cudaStream_t s, const char **detail) {
  CUtensorMap mr, mc;
  if (!operand_map(&mr, enc, p.dtype, p.r, p.rows, p.red, 128) || !operand_map(&mc, enc, p.dtype, p.c, p.cols, p.red, BN / 2)) {
    *detail = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  auto kern = pair_kernel<T, ACT, BN, LONG>;
  cudaError_t e = allow_smem((const void *)kern);
  if (e != cudaSuccess) return e;
  PairArgs g;
  g.n_steps = (p.red + BK - 1) / BK;
  g.n_rt = (p.rows + PAIR_ROWS - 1) / PAIR_ROWS; g.n_ct = (p.cols + BN - 1) / BN;
  g.n_tiles = g.n_rt * g.n_ct;
  g.run_steps = run_of(g.n_steps, longest_run(p));
  g.runs = (g.n_steps + g.run_steps - 1) / g.run_steps;
  g.band = band_of(p.red);
  g.r_mn = p.r.mn; g.c_mn = p.c.mn;
  g.idesc = instruction(p.dtype, p.r.mn, p.c.mn, PAIR_ROWS, BN);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(PAIR_THREADS);
  cfg.dynamicSmemBytes = PairTile<BN>::SMEM; cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  cfg.gridDim = dim3(2u * (unsigned)std::min(g.n_tiles, SMS / 2));
  return cudaLaunchKernelEx(&cfg, kern, mr, mc, out_of(p, 8), g);
}
bool is_long(const LinearProblem &p) { return (p.red + BK - 1) / BK > longest_run(p); }
template <typename T, int ACT> cudaError_t launch_pair(const LinearProblem &p, int bn, EncodeTiledFn enc, cudaStream_t s, const char **detail) {
  if constexpr (ACT >= 0) {      // (a product alone has columns that come in 64s, half a tile: linear_plan)
    if (bn == 64) return launch_pair<T, ACT, 64, false>(p, enc, s, detail);
  }
  return bn == 256 ? launch_pair<T, ACT, 256, false>(p, enc, s, detail) : launch_pair<T, ACT, 128, false>(p, enc, s, detail);
}
template <typename T, int ACT> cudaError_t launch_pair_long(const LinearProblem &p, int bn, EncodeTiledFn enc, cudaStream_t s, const char **detail) {
  return bn == 256 ? launch_pair<T, ACT, 256, true>(p, enc, s, detail) : launch_pair<T, ACT, 128, true>(p, enc, s, detail);
}
template <typename T> cudaError_t launch_pair(const LinearProblem &p, int bn, EncodeTiledFn enc, cudaStream_t s, const char **detail) {
  if (is_long(p)) return p.layer ? launch_pair_long<T, WINOCONV_ACT_NONE>(p, bn, enc, s, detail) : launch_pair_long<T, -1>(p, bn, enc, s, detail);
  if (!p.layer) return launch_pair<T, -1>(p, bn, enc, s, detail);
  switch (p.act) {
    case WINOCONV_ACT_RELU: return launch_pair<T, WINOCONV_ACT_RELU>(p, bn, enc, s, detail);
    case WINOCONV_ACT_GELU: return launch_pair<T, WINOCONV_ACT_GELU>(p, bn, enc, s, detail);
    case WINOCONV_ACT_GELU_TANH: return launch_pair<T, WINOCONV_ACT_GELU_TANH>(p, bn, enc, s, detail);
    case WINOCONV_ACT_SILU: return launch_pair<T, WINOCONV_ACT_SILU>(p, bn, enc, s, detail);
    default: return launch_pair<T, WINOCONV_ACT_NONE>(p, bn, enc, s, detail);
  }
}

}  // namespace linear

using namespace linear;

bool linear_by_rows(long long rows, int layer, bool z8) { return layer && rows <= MOST_ROWS && !z8; }

// The form with the smallest estimated time (us).  The constants are a fit to every form's time on 204 problems (B200, bf16: 3 to
// 8192 rows, 500 to 16384 columns, reductions of 64 to 25088, the three placements of the operands; launches in a row, operands from
// HBM): the form chosen takes 1.026 times the fastest one's time on geometric average and 1.25 times at worst.
LinearPlan linear_plan(const LinearProblem &p) {
  LinearPlan plan = {};
  plan.by_rows = linear_by_rows(p.rows, p.layer, p.z8 != nullptr);
  if (plan.by_rows) return plan;
  auto over = [](long long a, long long b) { return (a + b - 1) / b; };
  const long long n_steps = over(p.red, BK);
  const double memory = 2.0 + 2.0 * ((double)p.rows * p.red + (double)p.cols * p.red + (double)p.rows * p.cols) / 6.2e6;
  double best = 0;
  // pairs: a step's time is the tensor pipe's for 256 columns, below that the L2's (24 and 20 KB a CTA at 14.5 TB/s in all)
  const struct { int bn; double step; } pairs[3] = {{256, 0.33}, {128, 0.20}, {64, 0.18}};
  for (const auto &q : pairs) {
    if (q.bn == 64 && (p.c.mn || is_long(p))) continue;      // an MN-major operand comes in 64s: a CTA's half would be 32; long ones are built for 128 and more
    const double t = std::max(memory, 3.5 + (double)over(over(p.rows, PAIR_ROWS) * over(p.cols, q.bn), SMS / 2) * (n_steps * q.step + 0.3));
    if (plan.pair == 0 || t < best) {
      best = t;
      plan.pair = q.bn;
    }
  }
  const long long n_ct = over(p.cols, BC);
  for (int rows = p.r.mn ? 64 : 16; rows <= 256; rows *= 2) {
    const long long n_rt = over(p.rows, rows);
    if (rows < 256 && n_rt > 16) continue;                                   // many small tiles: never the fastest
    for (int split = 1; split <= 8 && split <= n_steps; split *= 2)
      for (int per_sm = 1; per_sm <= (rows == 256 ? 1 : 2); ++per_sm) {
        // CTAs that are resident at a time: clusters do not fill every group of SMs
        const int slots = per_sm * (split < 4 ? SMS : split == 4 ? (per_sm == 1 ? 132 : 142) : (per_sm == 1 ? 120 : 132));
        const double ctas = (double)(n_rt * n_ct * split), full = ctas / slots, waves = full <= 3 ? std::ceil(full) : full + 0.5;
        const double stage = C_BYTES + rows * BK * 2, shared = std::max(1.0, std::min(ctas, (double)slots) / SMS);
        const double step = std::max(0.36, stage * shared * 9.8e-6);         // what a step waits for, or an SM's share of L2
        const double end = 0.036 * rows + (split > 1 ? 1.2 : 0.0) + 0.24 * split;
        const double t = std::max(memory, waves * ((double)over(n_steps, split) * step + end));
        if (t < best) {
          best = t;
          plan.pair = 0;
          plan.tile_rows = rows;
          plan.split = split;
          plan.stages = (int)std::min(8.0, ((per_sm == 1 ? 227 * 1024 : CLUSTER_SMEM2) - 1024 - BAR_BYTES) / stage);
        }
      }
    if (rows >= p.rows) break;
  }
  return plan;
}

cudaError_t launch_linear(const LinearProblem &p, const LinearPlan &plan, cudaStream_t s, const char **detail) {
  *detail = "";
  if (plan.by_rows) return p.dtype == WINOCONV_F16 ? launch_rows<__half>(p, s) : launch_rows<__nv_bfloat16>(p, s);
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) { *detail = "cuTensorMapEncodeTiled unavailable"; return cudaErrorNotSupported; }
  if (plan.pair) return p.dtype == WINOCONV_F16 ? launch_pair<__half>(p, plan.pair, enc, s, detail) : launch_pair<__nv_bfloat16>(p, plan.pair, enc, s, detail);
  return p.dtype == WINOCONV_F16 ? launch_cluster<__half>(p, plan, enc, s, detail) : launch_cluster<__nv_bfloat16>(p, plan, enc, s, detail);
}

cudaError_t read_and_clear_linear_error(cudaStream_t s, unsigned int *code) {
  unsigned int host = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&host, g_linear_error, sizeof(host), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_linear_error, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  *code = host;
  return e;
}

}  // namespace wino
