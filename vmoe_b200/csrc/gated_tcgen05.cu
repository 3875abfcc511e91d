// Gated MLP on tcgen05: both projections, the activation and the product in one kernel, and the
// matching backward kernel.
//
//   forward   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u
//             for training also  a = act(g)  and  s = u act'(g)
//   backward  dh = dy Wo,  dg = dh s,  du = dh a   (and the column sums of both)
//
// Both are persistent warp-specialised GEMMs (TMA -> 128B-swizzled shared memory -> tcgen05.mma ->
// TMEM -> epilogue warps), with one CTA per 128-row tile or CTA pairs on 256-row tiles, like the
// plain GEMM of this library. Forward: half of a tile's accumulator columns are gate columns and half
// the up columns of the same hidden units, so a thread of the epilogue finds both factors of its
// products in its own TMEM lane; in a CTA pair the even CTA stages the gate's rows of the weights
// and the odd CTA the up projection's. Backward: the saved factors come in by TMA, two 32 x 32 tiles
// ahead of their use, and the epilogue is two products.
//
// The same kernel with a plain epilogue does the block's other two products with rows of x (output
// projection, dx) where the plain GEMM's 256-column tiles would leave SMs idle: tiles are 256, 128 or
// 64 accumulator columns wide, and the host takes the shape with the shortest estimate.
//
// Saving a and s (rounded once from fp32) instead of g and u leaves one rounding in each factor and
// no transcendental function in the backward pass; the traffic is the same. dg and du are rounded
// to bf16 because they are tensor-core operands of the next two GEMMs. With the result's own rounding
// dx and dw_in see three of them: 0.0029 of their norm, where rounding once gives 0.0017. The saved
// factors stay bf16: fp16 has more digits but s = u act'(g) passes its range, and fp32 would double
// the 434 MB that 8 experts of 6620 rows and 2048 units write and read.
//
// What bounds it: the tensor cores' power limit for many rows. Measured: 18464 rows 1024 -> 2736, forward
// 141 us of 207 GFLOP (1.47 PFLOP/s) and the output projection 82 us of 103; 8 x 6620 rows 768 -> 2048,
// forward 290 us (333 GFLOP, with 651 MB written), backward 217 us (167 GFLOP; 955 MB, 4.4 TB/s).
// HBM for few rows: 8 experts of 52 rows 1024 -> 2736, forward 23 us for 90 MB of weights, both
// kernels 37 us (3.6 TB/s, start and end of two launches included).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "ptx_sm100.cuh"
#include "tma_host.h"
#include "vmoe_api.h"

namespace vmoe {

void set_error(const char* fmt, const char* a, int code);
int make_bf16_map(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t rows, uint64_t batch,
                  uint64_t ld_elems, uint64_t batch_stride_elems, uint32_t box_rows,
                  uint32_t box_inner, CUtensorMapSwizzle swizzle);

namespace {

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int UMMA_K = 16;
constexpr int ROW_BYTES = BK * 2;           // one row of a K-major operand in a stage
constexpr int CHUNK_BYTES = 64 * BK * 2;    // one 64 x 64 MN-major box
constexpr int MAX_STAGES = 10;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int TILE_BYTES = 32 * 32 * 2;     // one staging tile: 32 rows of 64 bytes, 64B swizzle
constexpr int IN_BUFFERS = 3;               // backward: chunks of saved factors in flight or in use
// Staging tiles per epilogue warp, and stages of A rows and B rows, as many as fit the rest.
__host__ __device__ constexpr int epi_bytes(int mode) {
  return EPI_WARPS * (mode == 1 ? 2 * IN_BUFFERS : 4) * TILE_BYTES;
}
__host__ __device__ constexpr int pipe_bytes(int mode) { return (224 * 1024) - epi_bytes(mode); }
constexpr int SMEM_BYTES = 224 * 1024 + 1024 + 448;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
static_assert((2 * MAX_STAGES + 4 + EPI_WARPS * IN_BUFFERS) * 8 + 8 <= 448, "room for the barriers");

// Tiled copies with four coordinates (column, factor, row, expert).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* desc, uint32_t bar, int c0,
                                            int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      :
      : "r"(dst), "l"(reinterpret_cast<uint64_t>(desc)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const void* desc, uint32_t src, int c0, int c1, int c2,
                                             int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
      :
      : "l"(reinterpret_cast<uint64_t>(desc)), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// act(g) and act'(g) of two values through one sigmoid each: act = g s(w), act' = s (1 + g (1 - s) w').
// GELU's tanh form is w = 2 sqrt(2/pi) (g + 0.044715 g^3), SiLU is w = g. (ex2 and a reciprocal, 2^-22:
// tanh.approx would save one of the two, but its 2^-11 is several bf16 steps of act and act' where they
// fall off on the negative side.)
__device__ __forceinline__ void gate_and_slope(float g0, float g1, int act, float& a0, float& a1, float& s0,
                                               float& s1) {
  constexpr float K0 = 1.5957691216057308f, K1 = K0 * 0.044715f, L = 1.4426950408889634f;
  const float k0 = act == 0 ? K0 : 1.0f, k1 = act == 0 ? K1 : 0.0f;
  const f32x2 g = f2_pack(g0, g1), one = f2_pack(1.0f, 1.0f);
  const f32x2 g2 = f2_mul(g, g);
  float u0, u1, r0, r1;
  f2_unpack(f2_mul(g, f2_fma(g2, f2_pack(-L * k1, -L * k1), f2_pack(-L * k0, -L * k0))), u0, u1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(u0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(u1));
  f2_unpack(f2_add(f2_pack(u0, u1), one), r0, r1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r1));
  const f32x2 s = f2_pack(r0, r1);
  const f32x2 rest = f2_fma(s, f2_pack(-1.0f, -1.0f), one);
  const f32x2 dw = f2_fma(g2, f2_pack(3.0f * k1, 3.0f * k1), f2_pack(k0, k0));
  f2_unpack(f2_mul(g, s), a0, a1);
  f2_unpack(f2_mul(s, f2_fma(f2_mul(g, rest), dw, one)), s0, s1);
}

struct GatedParams {
  const void* bias;   // forward: (E, 2, M) or NULL
  const __nv_bfloat16* bias_out;  // forward: converted to fp32 for the GEMM behind, or NULL
  float* bias_out_f32;
  int bias_out_count, bias_bf16;
  float* sums;        // backward: (E, row blocks of 32, 2, M) partial column sums or NULL
  int rows, k, m, batch;
  int act;            // 0 GELU (tanh form), 1 SiLU
  int save;           // forward: write a and s
  int a_box, stages;  // rows of A per load (fewer than 128 when there are fewer), pipeline stages
  const __nv_bfloat16* residual;  // plain: (E, rows, m) with strides, or NULL
  long long ldr, r_batch_stride;
};

}  // namespace
}  // namespace vmoe

#include "gated_rows.cuh"

namespace vmoe {
namespace {

// MODE 0: forward. A = x (rows x k), B = w_in as (k, m, 2 E), both K-major.
// MODE 1: backward. A = dy (rows x k, K-major), B = w_out (m contiguous: MN-major).
// MODE 2 / 3: plain A B^T + bias + residual, B K-major / MN-major.
// BN: accumulator columns of a tile.
template <bool PAIR, int MODE, int BN>
__global__ void __launch_bounds__(THREADS, 1)
gated_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
             const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_s,
             const __grid_constant__ CUtensorMap map_d, const GatedParams p) {
  // The product behind this kernel may start as SMs become free: it fetches its weights and waits for
  // these results.
  if (MODE < 2) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  constexpr int HALF = BN / 2;
  constexpr bool B_MN = MODE == 1 || MODE == 3;
  constexpr int B_ROWS = PAIR ? HALF : BN;  // rows (columns of the result) of B this CTA stages
  constexpr int BSTAGE = B_ROWS * ROW_BYTES;
  constexpr int TMEM_COLS = 2 * BN;
  constexpr int TM = PAIR ? 2 * BM : BM;
  constexpr int TN = MODE == 0 ? HALF : BN;  // columns of the result per tile
  static_assert(!B_MN || B_ROWS % 64 == 0, "MN-major boxes are 64 columns wide");
  const int nstage = p.stages;
  // Rows of A that are not loaded keep what the stage held before: their results are not stored.
  const int a_stage = max(p.a_box, 8) * ROW_BYTES;
  uint8_t* sA = smem;
  uint8_t* sB = smem + nstage * a_stage;
  uint8_t* sEpi = smem + pipe_bytes(MODE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sEpi + epi_bytes(MODE));
  // full[stages], empty[stages], accumulator full[2], accumulator empty[2], epilogue input[8][3]
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = smem_u32(bars + nstage);
  const uint32_t bar_tfull = smem_u32(bars + 2 * nstage);
  const uint32_t bar_tempty = smem_u32(bars + 2 * nstage + 2);
  const uint32_t bar_in = smem_u32(bars + 2 * nstage + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * nstage + 4 + EPI_WARPS * IN_BUFFERS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int cta = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int ncta = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < nstage; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);
      mbar_init(bar_tempty + 8 * s, PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    for (int s = 0; s < EPI_WARPS * IN_BUFFERS; ++s) mbar_init(bar_in + 8 * s, 1);
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's barriers are initialised
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int num_m = (p.rows + TM - 1) / TM;
  const int num_n = (p.m + TN - 1) / TN;
  const int k_tiles = (p.k + BK - 1) / BK;
  const int num_tiles = p.batch * num_m * num_n;
  // Hidden units fastest, then rows, then experts: CTAs that run together share rows of A.
  auto decode = [&](int tile, int& b, int& mt, int& nt) {
    nt = tile % num_n;
    tile /= num_n;
    mt = tile % num_m;
    b = tile / num_m;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    // The whole warp walks through the steps and one elected thread issues: operands of the copies (and
    // of the products below) then are uniform across the warp. One thread alone in a branch of its own
    // took 290 ns per 64-deep step whatever the tile.
    const bool leader = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t full_base = PAIR ? mapa_shared(bar_full, 0) : bar_full;
    auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t full, int c0, int c1, int c2) {
      if (PAIR) {
        tma_load_3d_pair(dst, map, full, c0, c1, c2);
      } else {
        tma_load_3d(dst, map, full, c0, c1, c2);
      }
    };
    // Announces a stage's bytes and fetches its part of B.
    auto fill_b = [&](int st, int kt, int b, int nt) {
      const uint32_t full = full_base + 8 * st;
      if (!PAIR) {
        mbar_expect_tx(full, a_stage + BSTAGE);
      } else if (rank == 0) {
        mbar_expect_tx(bar_full + 8 * st, 2 * (a_stage + BSTAGE));
      }
      const uint32_t b_dst = smem_u32(sB + st * BSTAGE);
      const int k0 = kt * BK;
      if (MODE == 0) {
        if (PAIR) {
          load(b_dst, &map_b, full, k0, nt * TN, 2 * b + static_cast<int>(rank));
        } else {
          load(b_dst, &map_b, full, k0, nt * TN, 2 * b);
          load(b_dst + BSTAGE / 2, &map_b, full, k0, nt * TN, 2 * b + 1);
        }
      } else {
        const int n0 = nt * TN + static_cast<int>(rank) * HALF;
        if (!B_MN) {
          load(b_dst, &map_b, full, k0, n0, b);
        } else {
#pragma unroll
          for (int j = 0; j < B_ROWS / 64; ++j)
            load(b_dst + j * CHUNK_BYTES, &map_b, full, n0 + 64 * j, k0, b);
        }
      }
    };
    // A plain product's B are weights, its A is what the kernel in front writes: every stage's B is on its
    // way before that kernel is waited for.
    int early = 0;
    if (MODE >= 2) {
      int b, mt, nt;
      decode(cta, b, mt, nt);  // every CTA has a tile
      early = min(nstage, k_tiles);
      if (leader)
        for (int kt = 0; kt < early; ++kt) fill_b(kt, kt, b, nt);
      __syncwarp();
      asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    for (int tile = cta; tile < num_tiles && ok; tile += ncta) {
      int b, mt, nt;
      decode(tile, b, mt, nt);
      const int m0 = mt * TM + static_cast<int>(rank) * BM;
      for (int kt = 0; kt < k_tiles; ++kt) {
        const bool got = mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, nullptr, 0);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        if (leader) {
          if (early == 0) fill_b(stage, kt, b, nt);
          load(smem_u32(sA + stage * a_stage), &map_a, full_base + 8 * stage, kt * BK, m0, b);
        }
        __syncwarp();
        if (early > 0) --early;
        if (++stage == nstage) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {  // copies in flight get a bounded chance to land before the CTA exits
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(256);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0) {
      const bool leader = elect_one();
      const uint32_t idesc = umma_idesc_bf16(TM, BN, 0, B_MN ? 1 : 0);
      const uint32_t b_lbo = B_MN ? CHUNK_BYTES : 16, b_step = B_MN ? 2048 : 32;
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int tile = cta; tile < num_tiles && ok; tile += ncta, ++local) {
        const int slot = local & 1;
        const uint32_t use = static_cast<uint32_t>(local >> 1);
        bool got = mbar_wait(bar_tempty + 8 * slot, (use & 1) ^ 1, abort_flag, nullptr, 0);
        if (!__all_sync(0xffffffffu, got)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + slot * BN;
        for (int kt = 0; kt < k_tiles; ++kt) {
          got = mbar_wait(bar_full + 8 * stage, phase, abort_flag, nullptr, 0);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (leader) {
            const uint32_t a_addr = smem_u32(sA + stage * a_stage);
            const uint32_t b_addr = smem_u32(sB + stage * BSTAGE);
#pragma unroll
            for (int k = 0; k < BK / UMMA_K; ++k) {
              const uint64_t adesc = umma_smem_desc(a_addr + k * 32, 16, 1024);
              const uint64_t bdesc = umma_smem_desc(b_addr + k * b_step, b_lbo, 1024);
              if (PAIR) {
                umma_bf16_pair(d_tmem, adesc, bdesc, idesc, (kt > 0 || k > 0) ? 1u : 0u);
              } else {
                umma_bf16(d_tmem, adesc, bdesc, idesc, (kt > 0 || k > 0) ? 1u : 0u);
              }
            }
            if (PAIR) {
              umma_commit_pair(bar_empty + 8 * stage, 3);
            } else {
              umma_commit(bar_empty + 8 * stage);
            }
            if (kt == k_tiles - 1) {
              if (PAIR) {
                umma_commit_pair(bar_tfull + 8 * slot, 3);
              } else {
                umma_commit(bar_tfull + 8 * slot);
              }
            }
          }
          __syncwarp();
          if (++stage == nstage) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - 2;
    const int quad = warp & 3;   // TMEM lanes this warp may read
    const int half = ew >> 2;
    uint8_t* tiles = sEpi + ew * (epi_bytes(MODE) / EPI_WARPS);
    const uint32_t st_row = static_cast<uint32_t>(lane) * 64u;
    const uint32_t st_xor = (static_cast<uint32_t>(lane) >> 1) & 3u;
    constexpr int CHUNKS = TN / 32;  // 32-column chunks of a tile, shared by two warps per quadrant
    const uint32_t in_bar = bar_in + 8 * IN_BUFFERS * ew;
    const uint32_t tempty_base = PAIR ? mapa_shared(bar_tempty, 0) : bar_tempty;
    int local = 0;
    bool ok = true;
    if (MODE == 0 && p.bias_out)  // the GEMM behind this kernel takes fp32 biases
      for (int i = static_cast<int>(blockIdx.x) * 32 * EPI_WARPS + 32 * ew + lane; i < p.bias_out_count;
           i += static_cast<int>(gridDim.x) * 32 * EPI_WARPS)
        p.bias_out_f32[i] = __bfloat162float(p.bias_out[i]);
    // One row of a chunk (32 packed values) into a staging tile.
    auto stage_row = [&](uint8_t* tile, const uint32_t (&w)[16]) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(tile + st_row + ((static_cast<uint32_t>(i) ^ st_xor) << 4)) =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    };
    // Backward: this warp's chunks over all its tiles, in order. The saved factors of a chunk arrive in one
    // of IN_BUFFERS pairs of tiles, where dg and du take their place and leave. Loads run two chunks
    // ahead (a load takes longer than a chunk's arithmetic), into the next tiles too.
    int ahead_tile = cta, ahead_c = half - 2, ahead = 0, done = 0;
    auto fetch_next = [&]() {
      while (ahead_tile < num_tiles) {
        int b, mt, nt;
        decode(ahead_tile, b, mt, nt);
        ahead_c += 2;
        const int col = nt * TN + ahead_c * 32;
        if (ahead_c < CHUNKS && col < p.m) {
          if (lane == 0) {
            const int buf = ahead % IN_BUFFERS;
            const uint32_t dst = smem_u32(tiles + buf * 2 * TILE_BYTES);
            const int row = mt * TM + static_cast<int>(rank) * BM + quad * 32;
            mbar_expect_tx(in_bar + 8 * buf, 2 * TILE_BYTES);
            tma_load_4d(dst, &map_s, in_bar + 8 * buf, col, 0, row, b);
            tma_load_4d(dst + TILE_BYTES, &map_s, in_bar + 8 * buf, col, 1, row, b);
          }
          ++ahead;
          return;
        }
        ahead_tile += ncta;
        ahead_c = half - 2;
      }
    };
    if (MODE == 1)
      for (int i = 0; i < IN_BUFFERS - 1; ++i) fetch_next();
    for (int tile = cta; tile < num_tiles && ok; tile += ncta, ++local) {
      int b, mt, nt;
      decode(tile, b, mt, nt);
      const int slot = local & 1;
      const uint32_t use = static_cast<uint32_t>(local >> 1);
      const int row0 = mt * TM + static_cast<int>(rank) * BM + quad * 32;
      const int n0 = nt * TN;
      const bool got = mbar_wait(bar_tfull + 8 * slot, use & 1, abort_flag, nullptr, 0);
      if (!__all_sync(0xffffffffu, got)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = half; c < CHUNKS; c += 2) {
        const int col0 = n0 + c * 32;
        if (col0 >= p.m) break;
        const uint32_t acc =
            tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + slot * BN + c * 32;
        if (MODE == 0) {
          uint32_t rg[32], ru[32];
          tmem_ld_32x32(acc, rg);
          tmem_ld_32x32(acc + HALF, ru);
          tmem_ld_wait();
          if (p.bias && p.bias_bf16) {
            const __nv_bfloat16* bg = static_cast<const __nv_bfloat16*>(p.bias) + (2ll * b) * p.m + col0;
            const __nv_bfloat16* bu = bg + p.m;
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              if (col0 + i >= p.m) break;  // m is a multiple of 8
              const uint4 g8 = __ldg(reinterpret_cast<const uint4*>(bg + i));
              const uint4 u8 = __ldg(reinterpret_cast<const uint4*>(bu + i));
              const uint32_t gw[4] = {g8.x, g8.y, g8.z, g8.w}, uw[4] = {u8.x, u8.y, u8.z, u8.w};
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float2 gf = unpack_bf16x2(gw[q]), uf = unpack_bf16x2(uw[q]);
                rg[i + 2 * q] = __float_as_uint(__uint_as_float(rg[i + 2 * q]) + gf.x);
                rg[i + 2 * q + 1] = __float_as_uint(__uint_as_float(rg[i + 2 * q + 1]) + gf.y);
                ru[i + 2 * q] = __float_as_uint(__uint_as_float(ru[i + 2 * q]) + uf.x);
                ru[i + 2 * q + 1] = __float_as_uint(__uint_as_float(ru[i + 2 * q + 1]) + uf.y);
              }
            }
          } else if (p.bias) {
            const float* bg = static_cast<const float*>(p.bias) + (2ll * b) * p.m + col0;
            const float* bu = bg + p.m;
            if (col0 + 32 <= p.m) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 g4 = __ldg(reinterpret_cast<const float4*>(bg) + i);
                const float4 u4 = __ldg(reinterpret_cast<const float4*>(bu) + i);
                rg[4 * i] = __float_as_uint(__uint_as_float(rg[4 * i]) + g4.x);
                rg[4 * i + 1] = __float_as_uint(__uint_as_float(rg[4 * i + 1]) + g4.y);
                rg[4 * i + 2] = __float_as_uint(__uint_as_float(rg[4 * i + 2]) + g4.z);
                rg[4 * i + 3] = __float_as_uint(__uint_as_float(rg[4 * i + 3]) + g4.w);
                ru[4 * i] = __float_as_uint(__uint_as_float(ru[4 * i]) + u4.x);
                ru[4 * i + 1] = __float_as_uint(__uint_as_float(ru[4 * i + 1]) + u4.y);
                ru[4 * i + 2] = __float_as_uint(__uint_as_float(ru[4 * i + 2]) + u4.z);
                ru[4 * i + 3] = __float_as_uint(__uint_as_float(ru[4 * i + 3]) + u4.w);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col0 + i < p.m) {
                  rg[i] = __float_as_uint(__uint_as_float(rg[i]) + __ldg(bg + i));
                  ru[i] = __float_as_uint(__uint_as_float(ru[i]) + __ldg(bu + i));
                }
            }
          }
          uint32_t wh[16], wa[16], ws[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float a0, a1, s0, s1;
            const float u0 = __uint_as_float(ru[2 * i]), u1 = __uint_as_float(ru[2 * i + 1]);
            gate_and_slope(__uint_as_float(rg[2 * i]), __uint_as_float(rg[2 * i + 1]), p.act, a0, a1, s0, s1);
            wh[i] = pack_bf16x2(a0 * u0, a1 * u1);
            wa[i] = pack_bf16x2(a0, a1);
            ws[i] = pack_bf16x2(s0 * u0, s1 * u1);
          }
          // The staging tiles are free once the TMA engine has read their last contents.
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          stage_row(tiles, wh);
          if (p.save) {
            stage_row(tiles + TILE_BYTES, ws);
            stage_row(tiles + 2 * TILE_BYTES, wa);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&map_h, smem_u32(tiles), col0, row0, b);
            if (p.save) {
              tma_store_4d(&map_s, smem_u32(tiles + TILE_BYTES), col0, 0, row0, b);
              tma_store_4d(&map_s, smem_u32(tiles + 2 * TILE_BYTES), col0, 1, row0, b);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else if (MODE >= 2) {
          uint32_t r[32];
          tmem_ld_32x32(acc, r);
          const int row = row0 + lane;
          const __nv_bfloat16* res = p.residual && row < p.rows
                                         ? p.residual + b * p.r_batch_stride + row * p.ldr + col0
                                         : nullptr;
          uint4 rq[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // m is a multiple of 8
            rq[i] = make_uint4(0, 0, 0, 0);
            if (res && col0 + 8 * i < p.m) rq[i] = __ldg(reinterpret_cast<const uint4*>(res) + i);
          }
          tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {rq[i].x, rq[i].y, rq[i].z, rq[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack_bf16x2(w[j]);
              v[8 * i + 2 * j] = __uint_as_float(r[8 * i + 2 * j]) + f.x;
              v[8 * i + 2 * j + 1] = __uint_as_float(r[8 * i + 2 * j + 1]) + f.y;
            }
          }
          if (p.bias) {
            const long long at = static_cast<long long>(b) * p.m + col0;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              if (col0 + i >= p.m) break;
              float4 f;
              if (p.bias_bf16) {
                const uint2 q = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.bias) + at + i));
                const float2 f0 = unpack_bf16x2(q.x), f1 = unpack_bf16x2(q.y);
                f = make_float4(f0.x, f0.y, f1.x, f1.y);
              } else {
                f = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + at + i));
              }
              v[i] += f.x;
              v[i + 1] += f.y;
              v[i + 2] += f.z;
              v[i + 3] += f.w;
            }
          }
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          stage_row(tiles, w);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&map_h, smem_u32(tiles), col0, row0, b);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          uint32_t r[32];
          tmem_ld_32x32(acc, r);
          uint8_t* factors = tiles + (done % IN_BUFFERS) * 2 * TILE_BYTES;
          const bool in = mbar_wait(in_bar + 8 * (done % IN_BUFFERS), (done / IN_BUFFERS) & 1, abort_flag,
                                    nullptr, 0);
          ++done;
          if (!__all_sync(0xffffffffu, in)) {
            ok = false;
            break;
          }
          uint4 qs[4], qa[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t off = st_row + ((static_cast<uint32_t>(i) ^ st_xor) << 4);
            qs[i] = *reinterpret_cast<const uint4*>(factors + off);
            qa[i] = *reinterpret_cast<const uint4*>(factors + TILE_BYTES + off);
          }
          tmem_ld_wait();
          uint32_t wg[16], wu[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint4 s4 = qs[i >> 2], a4 = qa[i >> 2];
            const uint32_t sw = (i & 3) == 0 ? s4.x : (i & 3) == 1 ? s4.y : (i & 3) == 2 ? s4.z : s4.w;
            const uint32_t aw = (i & 3) == 0 ? a4.x : (i & 3) == 1 ? a4.y : (i & 3) == 2 ? a4.z : a4.w;
            const float2 fs = unpack_bf16x2(sw), fa = unpack_bf16x2(aw);
            const float d0 = __uint_as_float(r[2 * i]), d1 = __uint_as_float(r[2 * i + 1]);
            wg[i] = pack_bf16x2(d0 * fs.x, d1 * fs.y);
            wu[i] = pack_bf16x2(d0 * fa.x, d1 * fa.y);
          }
          // The chunk before this one has left its buffer (and every lane has read its column sums):
          // that buffer takes the chunk after the next.
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
          fetch_next();
          stage_row(factors, wg);  // a lane overwrites the row that it has read
          stage_row(factors + TILE_BYTES, wu);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_4d(&map_d, smem_u32(factors), col0, 0, row0, b);
            tma_store_4d(&map_d, smem_u32(factors + TILE_BYTES), col0, 1, row0, b);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          if (p.sums && row0 < p.rows) {
            // Column sums of the 32 staged rows: lanes 0-15 take the even rows, 16-31 the odd ones
            // of two columns each (rows past the end hold zeros), in fp32, of dg and du as rounded: the
            // same values that dx and dw_in are made from. Written, not added: a second kernel joins
            // the row blocks in a fixed order.
            const long long blocks = (p.rows + 31) / 32;
            const uint32_t two = lane & 15, odd = lane >> 4;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t rr = 2 * i + odd;
                const uint32_t off = rr * 64u + (((two >> 2) ^ ((rr >> 1) & 3u)) << 4) + (two & 3) * 4u;
                const float2 f = unpack_bf16x2(*reinterpret_cast<const uint32_t*>(factors + w * TILE_BYTES + off));
                s0 += f.x;
                s1 += f.y;
              }
              s0 += __shfl_xor_sync(0xffffffffu, s0, 16);
              s1 += __shfl_xor_sync(0xffffffffu, s1, 16);
              const int col = col0 + 2 * static_cast<int>(two);
              if (odd == 0 && col < p.m)
                *reinterpret_cast<float2*>(p.sums + ((b * blocks + row0 / 32) * 2 + w) * p.m + col) =
                    make_float2(s0, s1);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) {
          mbar_arrive_cluster(tempty_base + 8 * slot);
        } else {
          mbar_arrive(bar_tempty + 8 * slot);
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    if (!ok) {  // an input tile may still be in flight
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000) __nanosleep(256);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // neither CTA leaves while its peer can touch its barriers or TMEM
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) {
      tmem_dealloc_pair(tmem_base, TMEM_COLS);
    } else {
      tmem_dealloc(tmem_base, TMEM_COLS);
    }
  }
}

// One set of partial column sums: out (e, cols) (+)= sums (e, blocks, cols) over its blocks.
struct SumsPart {
  const float* sums;
  void* out;
  int blocks, cols, out_bf16, accumulate;
};

__device__ __forceinline__ void put(void* out, int is_bf16, int accumulate, long long i, float v) {
  if (is_bf16) {
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16(v);
  } else {
    float* o = static_cast<float*>(out) + i;
    *o = accumulate ? *o + v : v;
  }
}

// Blocks in order within a warp and warps in order, so the result does not depend on scheduling.
__global__ void __launch_bounds__(256)
gated_join_sums_kernel(const SumsPart a, const SumsPart b) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int a_tiles = (a.cols + 31) / 32;
  const bool in_a = static_cast<int>(blockIdx.x) < a_tiles;
  const SumsPart& p = in_a ? a : b;
  const int c = (static_cast<int>(blockIdx.x) - (in_a ? 0 : a_tiles)) * 32 + lane;
  const float* src = p.sums + static_cast<long long>(blockIdx.y) * p.blocks * p.cols;
  float s = 0.0f;
  if (c < p.cols)
    for (int i = group; i < p.blocks; i += 8) s += src[static_cast<long long>(i) * p.cols + c];
  part[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < p.cols) {
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    put(p.out, p.out_bf16, p.accumulate, static_cast<long long>(blockIdx.y) * p.cols + c, s);
  }
}

// sums (e, blocks, n) of x (e, rows, n) over blocks of ROW_BLOCK rows: 8 columns per lane, a warp
// every eighth row, its loads all in flight together.
constexpr int ROW_BLOCK = 128;
__global__ void __launch_bounds__(256)
gated_row_sums_kernel(const __nv_bfloat16* __restrict__ x, float* __restrict__ sums, int rows, int n) {
  __shared__ float part[8][256 + 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 256 + lane * 8;
  const int r0 = blockIdx.y * ROW_BLOCK + warp;
  const __nv_bfloat16* src = x + static_cast<long long>(blockIdx.z) * rows * n;
  uint4 q[ROW_BLOCK / 8];
#pragma unroll
  for (int i = 0; i < ROW_BLOCK / 8; ++i) {
    const int r = r0 + 8 * i;
    q[i] = r < rows && col < n
               ? __ldg(reinterpret_cast<const uint4*>(src + static_cast<long long>(r) * n + col))
               : make_uint4(0, 0, 0, 0);
  }
  float s[8] = {};
#pragma unroll
  for (int i = 0; i < ROW_BLOCK / 8; ++i) {
    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack_bf16x2(w[j]);
      s[2 * j] += f.x;
      s[2 * j + 1] += f.y;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) part[warp][lane * 8 + j] = s[j];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < n) {
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += part[w][threadIdx.x];
    sums[(static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * n + c] = total;
  }
}

// out (count) (+)= sum of `pieces` partial results, in order.
__global__ void __launch_bounds__(256)
gated_join_pieces_kernel(const float* __restrict__ pieces, void* __restrict__ out, long long count,
                         int n_pieces, int out_bf16, int accumulate) {
  const long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= count) return;  // count is a multiple of 64
  float4 s = __ldg(reinterpret_cast<const float4*>(pieces + i));
  for (int p = 1; p < n_pieces; ++p) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(pieces + p * count + i));
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  if (out_bf16) {
    uint2 q;
    q.x = pack_bf16x2(s.x, s.y);
    q.y = pack_bf16x2(s.z, s.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + i) = q;
  } else {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + i);
    if (accumulate) {
      const float4 v = *o;
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    *o = s;
  }
}

int fail(const char* what, int code = -1) {
  set_error("%s (code %d)", what, code);
  return code;
}

// (e, rows, 2, m) contiguous bf16 as a 4-D tensor with 32 x 32 boxes.
int make_pair_map(CUtensorMap* map, const void* ptr, uint64_t m, uint64_t rows, uint64_t e) {
  cuuint64_t dims[4] = {m, 2, rows, e};
  cuuint64_t strides[3] = {m * 2, m * 4, rows * m * 4};
  cuuint32_t box[4] = {32, 1, 32, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = tma_encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims,
                                strides, box, estr, CU_TENSOR_MAP_SWIZZLE_64B);
  return r == CUDA_SUCCESS ? 0 : fail("cuTensorMapEncodeTiled failed", -3);
}

struct DeviceInfo {
  int sms, pairs;
};

// Tile shapes: 128 rows and one CTA, or 256 rows and a CTA pair, times accumulator columns.
struct Shape {
  bool pair;
  int bn;
};
constexpr Shape SHAPES[4] = {{true, 256}, {true, 128}, {false, 128}, {false, 64}};

using Kernel = void (*)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap,
                        const CUtensorMap, const GatedParams);
template <int MODE>
Kernel kernel_in(const Shape& s) {
  if (!s.pair) return s.bn == 128 ? gated_kernel<false, MODE, 128> : gated_kernel<false, MODE, 64>;
  if (s.bn == 128) return gated_kernel<true, MODE, 128>;
  if constexpr (MODE < 2) return gated_kernel<true, MODE, 256>;
  return nullptr;  // the library's plain GEMM
}
Kernel kernel_of(int mode, const Shape& s) {
  return mode == 0 ? kernel_in<0>(s) : mode == 1 ? kernel_in<1>(s) : mode == 2 ? kernel_in<2>(s) : kernel_in<3>(s);
}

// Per-device set-up (shared-memory limits, resident CTA pairs), done once per device.
int device_info(DeviceInfo* out) {
  constexpr int MAX_DEVICES = 64;
  static DeviceInfo known[MAX_DEVICES];
  static bool ready[MAX_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= MAX_DEVICES) return fail("no current device", -4);
  if (!ready[dev]) {
    DeviceInfo d = {0, 0};
    e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
    for (int mode = 0; mode < 4; ++mode)
      for (const Shape& shape : SHAPES)
        if (e == cudaSuccess && kernel_of(mode, shape))
          e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel_of(mode, shape)),
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) {
      set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
      return -4;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute attr;
    memset(&attr, 0, sizeof(attr));
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(d.sms & ~1));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&d.pairs, gated_kernel<true, 0, 256>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      d.pairs = 0;
    }
    known[dev] = d;
    ready[dev] = true;
  }
  *out = known[dev];
  return 0;
}

// Rows of A per load: all 128, or the next of 32 and 64 that holds every row there is.
int a_box(int64_t rows, const Shape& s) { return s.pair || rows > 64 ? BM : rows > 32 ? 64 : 32; }

// Nanoseconds until the last SM is done: rounds of tiles, each the longer of its 64-deep steps and its
// epilogue, which overlaps the next tile's steps. Measured over ten sizes from 16 x 64 rows of 512 x 1024 to
// 2600 rows of 1024 x 2736: a step takes 400 ns on 256 x 256 pair tiles, 265 on 256 x 128 ones, 300 and
// 255 on single 128 x 128 and 128 x 64 tiles (each product needs shared memory for its operands twice, for
// the copy in and for the tensor core; small tiles reuse them less); an epilogue 2.5 us per 64
// hidden units forward, 1.4 us backward, 1.2 us per 64 plain columns.
double estimate(const Shape& s, int mode, int64_t e, int64_t rows, int64_t cols, int64_t k, const DeviceInfo& d) {
  if (s.pair && (d.pairs == 0 || rows <= BM)) return 1e30;
  const int64_t tm = s.pair ? 2 * BM : BM, tn = mode == 0 ? s.bn / 2 : s.bn;
  const int64_t tiles = e * ((rows + tm - 1) / tm) * ((cols + tn - 1) / tn), units = s.pair ? d.pairs : d.sms;
  const double rounds = static_cast<double>((tiles + units - 1) / units);
  const double step = s.pair ? (s.bn == 256 ? 400.0 : 265.0) : (s.bn == 128 ? 300.0 : 255.0);
  const double epilogue = (mode == 0 ? 2500.0 : mode == 1 ? 1400.0 : 1200.0) * tn / 64;
  const double work = step * ((k + BK - 1) / BK);
  return rounds * (work > epilogue ? work : epilogue) + epilogue + (s.pair ? 1000.0 : 0.0);
}

Shape choose_shape(int mode, int64_t e, int64_t rows, int64_t cols, int64_t k, const DeviceInfo& d) {
  Shape best = SHAPES[0];
  double best_ns = estimate(best, mode, e, rows, cols, k, d);
  for (const Shape& s : SHAPES) {
    const double ns = estimate(s, mode, e, rows, cols, k, d);
    if (ns < best_ns) {
      best = s;
      best_ns = ns;
    }
  }
  return best;
}

// after: the kernel in front in the stream is one of modes 0 and 1, and this one may start before its end.
int launch(int mode, const Shape& s, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mh,
           const CUtensorMap& ms, const CUtensorMap& md, GatedParams p, bool after, const DeviceInfo& info,
           cudaStream_t stream) {
  const int tm = s.pair ? 2 * BM : BM, tn = mode == 0 ? s.bn / 2 : s.bn;
  const long long tiles =
      static_cast<long long>(p.batch) * ((p.rows + tm - 1) / tm) * ((p.m + tn - 1) / tn);
  if (tiles > 0x7fffffff) return fail("gated mlp: too many tiles");
  p.a_box = a_box(p.rows, s);
  p.stages = pipe_bytes(mode) / ((p.a_box + (s.pair ? s.bn / 2 : s.bn)) * ROW_BYTES);
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  const long long most = s.pair ? info.pairs : info.sms;
  const unsigned units = static_cast<unsigned>(tiles < most ? tiles : most);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  memset(attr, 0, sizeof(attr));
  int n = 0;
  if (s.pair) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 2;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (after) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.gridDim = dim3(s.pair ? 2 * units : units);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel_of(mode, s), ma, mb, mh, ms, md, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    return -5;
  }
  return 0;
}

int check_launch() {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    return -5;
  }
  return 0;
}

int check_sizes(const VmoeGatedArgs* a) {
  if (a->e < 0 || a->rows < 0 || a->h < 1 || a->m < 1 || a->o < 1) return fail("gated mlp: bad sizes");
  if (a->rows > (1 << 28) || a->h > (1 << 24) || a->m > (1 << 24) || a->o > (1 << 24) || a->e > 32767)
    return fail("gated mlp: sizes out of range");
  if (a->h % 8 || a->m % 8 || a->o % 8 || a->ld_res % 8 || a->res_batch_stride % 8)
    return fail("gated mlp: widths and strides must be multiples of 8 elements");
  const void* ptrs[15] = {a->x,     a->w_in, a->w_out, a->b_in, a->b_out, a->residual, a->y,     a->hid,
                          a->saved, a->dy,   a->dgu,   a->dx,   a->dw_in, a->dw_out,   a->scratch};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return fail("gated mlp: operands must be 16-byte aligned");
  if (a->act != 0 && a->act != 1) return fail("gated mlp: unknown activation");
  return 0;
}

// The few-row kernel (rows of x in groups of 8) takes up to 16 rows, and up to 32 where the output projection
// has so few 64-column tiles that the tile kernel would leave most SMs idle. 1 expert of 17 rows 1280 -> 5120: 24 us
// against 36, 3 of 32 rows 1024 -> 2736: 25 against 27; but 4 of them 36 against 32 and 8 58 against 39.
// Up to 16 rows it is never behind: 8 experts of 16 rows 36 against 38, 1 of 16 rows 1280 -> 5120 17 against 36.
constexpr int FEW_ROWS = 16;
bool is_few(const VmoeGatedArgs* a, const DeviceInfo& info) {
  return a->rows <= FEW_ROWS || (a->rows <= 2 * FEW_ROWS && 3 * a->e * ((a->o + 63) / 64) <= info.sms);
}

template <int NT, bool GATED>
int launch_rows(RowsParams p, int e, int sms, cudaStream_t stream) {
  const int tiles = (p.m + 15) / 16, chunks = (p.k + 31) / 32;
  const int threads = tiles * e >= 2 * sms ? 128 : 256;
  // Share the contraction over a cluster until every SM has a CTA, while each warp keeps a chunk.
  p.split = 1;
  while (p.split < GR_MAX_SPLIT && tiles * e * p.split < sms && chunks >= 2 * p.split * (threads / 32))
    p.split *= 2;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr[2];
  memset(attr, 0, sizeof(attr));
  int n = 0;
  if (p.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(p.split);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.after) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.split), static_cast<unsigned>(e));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t err = threads == 128 ? cudaLaunchKernelEx(&cfg, gated_rows_kernel<NT, GATED, 128>, p)
                                         : cudaLaunchKernelEx(&cfg, gated_rows_kernel<NT, GATED, 256>, p);
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_error("%s (code %d)", cudaGetErrorString(err), static_cast<int>(err));
    return -5;
  }
  return 0;
}

int few_rows(const VmoeGatedArgs* a, const DeviceInfo& info, cudaStream_t stream) {
  RowsParams p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const __nv_bfloat16*>(a->x);
  p.w = static_cast<const __nv_bfloat16*>(a->w_in);
  p.bias = a->b_in;
  p.bias_bf16 = a->b_in_bf16;
  p.out = static_cast<__nv_bfloat16*>(a->hid);
  p.saved = static_cast<__nv_bfloat16*>(a->saved);
  p.ldx = a->h;
  p.x_batch_stride = a->rows * a->h;
  p.rows = static_cast<int>(a->rows);
  p.k = static_cast<int>(a->h);
  p.m = static_cast<int>(a->m);
  p.act = a->act;
  const int e = static_cast<int>(a->e);
  int rc = a->rows <= 8    ? launch_rows<1, true>(p, e, info.sms, stream)
           : a->rows <= 16 ? launch_rows<2, true>(p, e, info.sms, stream)
                           : launch_rows<4, true>(p, e, info.sms, stream);
  if (rc) return rc;
  RowsParams q;
  memset(&q, 0, sizeof(q));
  q.x = static_cast<const __nv_bfloat16*>(a->hid);
  q.w = static_cast<const __nv_bfloat16*>(a->w_out);
  q.bias = a->b_out;
  q.bias_bf16 = a->b_out_bf16;
  q.residual = static_cast<const __nv_bfloat16*>(a->residual);
  q.out = static_cast<__nv_bfloat16*>(a->y);
  q.ldx = a->m;
  q.x_batch_stride = a->rows * a->m;
  q.ldr = a->ld_res;
  q.r_batch_stride = a->res_batch_stride;
  q.rows = static_cast<int>(a->rows);
  q.k = static_cast<int>(a->m);
  q.m = static_cast<int>(a->o);
  q.after = 1;
  return a->rows <= 8    ? launch_rows<1, false>(q, e, info.sms, stream)
         : a->rows <= 16 ? launch_rows<2, false>(q, e, info.sms, stream)
                         : launch_rows<4, false>(q, e, info.sms, stream);
}

void gemm_operands(VmoeGemmArgs* g, const void* a, int64_t lda, int64_t sa, int a_mn, const void* b,
                   int64_t ldb, int64_t sb, int b_mn, int64_t m, int64_t n, int64_t k, int64_t batch) {
  memset(g, 0, sizeof(*g));
  g->A = a;
  g->B = b;
  g->M = m;
  g->N = n;
  g->K = k;
  g->batch = batch;
  g->lda = lda;
  g->ldb = ldb;
  g->ldc = n;
  g->a_batch_stride = batch > 1 ? sa : 0;
  g->b_batch_stride = batch > 1 ? sb : 0;
  g->c_batch_stride = batch > 1 ? m * n : 0;
  g->a_mn_major = a_mn;
  g->b_mn_major = b_mn;
  g->split_k = 1;
}

// Called right behind the kernel that writes a.
// out (e, rows, n) = a (e, rows, k) b^T + bias + residual, b (e, n, k) or, with b_mn, (e, k, n): on this
// file's tiles or on the plain GEMM, whichever is estimated to be done first. bias_f32: the plain GEMM's
// form of a bf16 bias.
int product(const void* a, const void* b, int b_mn, const void* bias, int bias_bf16, const float* bias_f32,
            const void* residual, int64_t ldr, int64_t r_batch_stride, void* out, int64_t e, int64_t rows,
            int64_t n, int64_t k, const DeviceInfo& info, cudaStream_t stream) {
  const int mode = b_mn ? 3 : 2;
  const Shape s = choose_shape(mode, e, rows, n, k, info);
  if (s.bn == 256) {
    VmoeGemmArgs g;
    gemm_operands(&g, a, k, rows * k, 0, b, b_mn ? n : k, n * k, b_mn, rows, n, k, e);
    g.C = out;
    g.cta_pair = 2;  // the tiles of the estimate
    g.bias = bias_bf16 ? bias_f32 : static_cast<const float*>(bias);
    g.bias_batch_stride = e > 1 ? n : 0;
    g.residual = residual;
    g.ldr = ldr;
    g.r_batch_stride = e > 1 ? r_batch_stride : 0;
    return vmoe_gemm_bf16(&g, stream);
  }
  CUtensorMap ma, mb, mh;
  int rc;
  if ((rc = make_bf16_map(&ma, a, k, rows, e, k, rows * k, a_box(rows, s), 64, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  const int b_rows = s.pair ? s.bn / 2 : s.bn;
  if ((rc = b_mn ? make_bf16_map(&mb, b, n, k, e, n, n * k, BK, 64, CU_TENSOR_MAP_SWIZZLE_128B)
                 : make_bf16_map(&mb, b, k, n, e, k, n * k, b_rows, 64, CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = make_bf16_map(&mh, out, n, rows, e, n, rows * n, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B))) return rc;
  GatedParams p;
  memset(&p, 0, sizeof(p));
  p.bias = bias;
  p.bias_bf16 = bias_bf16;
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  p.ldr = ldr;
  p.r_batch_stride = r_batch_stride;
  p.rows = static_cast<int>(rows);
  p.k = static_cast<int>(k);
  p.m = static_cast<int>(n);
  p.batch = static_cast<int>(e);
  return launch(mode, s, ma, mb, mh, mh, mh, p, true, info, stream);
}

// Pieces that a weight gradient's contraction over `rows` is cut into: few output tiles leave SMs idle in
// the last round; each piece costs writing and reading its fp32 result once (1.85 ps per element), joining
// them 4 us and rows that do not divide 20 us (a product of its own). Both gradients of 18464 rows
// 384 -> 1024 take 75 us in pieces and 233 without, of 18464 rows 1024 -> 2736 297 and 318; of 6304
// rows 768 -> 2048 77 with dw_out in two, 91 without pieces and 88 with two for both.
int gradient_pieces(int64_t e, int64_t n, int64_t k, int64_t rows) {
  const int64_t tiles = e * ((n + 255) / 256) * ((k + 255) / 256), pairs = 74;
  if (e > 1 || tiles >= 2 * pairs || rows < 4096) return 1;
  const double round_s = 2.0 * 256 * 256 * rows / (1.5e15 / pairs), piece_s = n * k * 1.85e-12;
  int best = 1;
  double best_s = round_s * ((tiles + pairs - 1) / pairs);
  for (int s = 2; s <= 8 && rows / s >= 1024; ++s) {
    const double t = round_s / s * ((tiles * s + pairs - 1) / pairs) + s * piece_s + 4e-6 +
                     (rows % s ? 20e-6 : 0.0);
    if (t < best_s) {
      best = s;
      best_s = t;
    }
  }
  return best;
}

// dw (e, n, k) = dy (e, rows, n)^T x (e, rows, k); mode: VMOE_GRAD_*.
int weight_gradient(const void* dy, const void* x, int64_t e, int64_t rows, int64_t n, int64_t k,
                    void* dw, int mode, float* pieces, cudaStream_t stream) {
  const size_t width = mode == VMOE_GRAD_BF16 ? 2 : 4;
  if (rows == 0) {
    if (mode != VMOE_GRAD_ADD) cudaMemsetAsync(dw, 0, static_cast<size_t>(e * n * k) * width, stream);
    return check_launch();
  }
  VmoeGemmArgs g;
  const int cut = gradient_pieces(e, n, k, rows);
  if (cut == 1) {
    gemm_operands(&g, dy, n, rows * n, 1, x, k, rows * k, 1, n, k, rows, e);
    g.C = dw;
    g.c_fp32 = mode != VMOE_GRAD_BF16;
    g.c_atomic = mode == VMOE_GRAD_ADD;
    return vmoe_gemm_bf16(&g, stream);
  }
  const int64_t piece = rows / cut, left = rows % cut;
  gemm_operands(&g, dy, n, piece * n, 1, x, k, piece * k, 1, n, k, piece, cut);
  g.C = pieces;
  g.c_fp32 = 1;
  int rc = vmoe_gemm_bf16(&g, stream);
  if (rc) return rc;
  if (left) {
    gemm_operands(&g, static_cast<const __nv_bfloat16*>(dy) + cut * piece * n, n, 0, 1,
                  static_cast<const __nv_bfloat16*>(x) + cut * piece * k, k, 0, 1, n, k, left, 1);
    g.C = pieces;
    g.c_fp32 = 1;
    g.c_atomic = 1;
    if ((rc = vmoe_gemm_bf16(&g, stream))) return rc;
  }
  const long long count = n * k;
  gated_join_pieces_kernel<<<static_cast<unsigned>((count / 4 + 255) / 256), 256, 0, stream>>>(
      pieces, dw, count, cut, mode == VMOE_GRAD_BF16, mode == VMOE_GRAD_ADD);
  return check_launch();
}

// Scratch of the backward pass, in floats: row-block sums of dg / du and of dy, gradient pieces.
struct BackwardScratch {
  int64_t sums, dy_sums, pieces, total;
  explicit BackwardScratch(const VmoeGatedArgs* a) {
    sums = a->db_in ? a->e * ((a->rows + 31) / 32) * 2 * a->m : 0;
    dy_sums = a->db_out ? a->e * ((a->rows + ROW_BLOCK - 1) / ROW_BLOCK) * a->o : 0;
    const int in = a->dw_in ? gradient_pieces(a->e, 2 * a->m, a->h, a->rows) : 1;
    const int out = a->dw_out ? gradient_pieces(a->e, a->o, a->m, a->rows) : 1;
    pieces = 0;
    if (in > 1) pieces = in * 2 * a->m * a->h;
    if (out > 1 && out * a->o * a->m > pieces) pieces = out * a->o * a->m;
    sums = (sums + 3) / 4 * 4;
    dy_sums = (dy_sums + 3) / 4 * 4;
    total = sums + dy_sums + pieces;
  }
};

}  // namespace
}  // namespace vmoe

using namespace vmoe;

extern "C" int64_t vmoe_gated_scratch_bytes(const VmoeGatedArgs* a, int32_t backward) {
  if (backward) return BackwardScratch(a).total * 4;
  return a->rows > FEW_ROWS && a->b_out && a->b_out_bf16 ? a->e * a->o * 4 : 0;
}

extern "C" int vmoe_gated_fwd(const VmoeGatedArgs* a, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_sizes(a);
  if (rc) return rc;
  if (a->e == 0 || a->rows == 0) return 0;
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  if (is_few(a, info)) return few_rows(a, info, stream);
  CUtensorMap ma, mb, mh, ms;
  memset(&ms, 0, sizeof(ms));
  const Shape shape = choose_shape(0, a->e, a->rows, a->m, a->h, info);
  if ((rc = make_bf16_map(&ma, a->x, a->h, a->rows, a->e, a->h, a->rows * a->h, a_box(a->rows, shape), 64,
                          CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = make_bf16_map(&mb, a->w_in, a->h, a->m, 2 * a->e, a->h, a->m * a->h, shape.bn / 2, 64,
                          CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  if ((rc = make_bf16_map(&mh, a->hid, a->m, a->rows, a->e, a->m, a->rows * a->m, 32, 32,
                          CU_TENSOR_MAP_SWIZZLE_64B)))
    return rc;
  if (a->saved && (rc = make_pair_map(&ms, a->saved, a->m, a->rows, a->e))) return rc;
  GatedParams p;
  memset(&p, 0, sizeof(p));
  p.bias = a->b_in;
  p.bias_bf16 = a->b_in_bf16;
  if (a->b_out && a->b_out_bf16) {
    if (!a->scratch) return fail("gated mlp: scratch is missing");
    p.bias_out = static_cast<const __nv_bfloat16*>(a->b_out);
    p.bias_out_f32 = a->scratch;
    p.bias_out_count = static_cast<int>(a->e * a->o);
  }
  p.rows = static_cast<int>(a->rows);
  p.k = static_cast<int>(a->h);
  p.m = static_cast<int>(a->m);
  p.batch = static_cast<int>(a->e);
  p.act = a->act;
  p.save = a->saved != nullptr;
  if ((rc = launch(0, shape, ma, mb, mh, ms, ms, p, false, info, stream))) return rc;
  return product(a->hid, a->w_out, 0, a->b_out, a->b_out_bf16, a->scratch, a->residual, a->ld_res,
                 a->res_batch_stride, a->y, a->e, a->rows, a->o, a->m, info, stream);
}

extern "C" int vmoe_gated_bwd(const VmoeGatedArgs* a, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_sizes(a);
  if (rc) return rc;
  if (a->e == 0) return 0;
  const BackwardScratch size(a);
  if (size.total && !a->scratch) return fail("gated mlp: scratch is missing");
  float* sums = a->scratch;
  float* dy_sums = a->scratch + size.sums;
  float* pieces = dy_sums + size.dy_sums;
  DeviceInfo info;
  if ((rc = device_info(&info))) return rc;
  const bool inner = a->dx || a->dw_in || a->db_in;
  if (a->rows > 0 && a->db_out) {
    if (a->rows > 65535ll * ROW_BLOCK) return fail("gated mlp: too many rows");
    gated_row_sums_kernel<<<dim3(static_cast<unsigned>((a->o + 255) / 256),
                                 static_cast<unsigned>((a->rows + ROW_BLOCK - 1) / ROW_BLOCK),
                                 static_cast<unsigned>(a->e)),
                            256, 0, stream>>>(static_cast<const __nv_bfloat16*>(a->dy), dy_sums,
                                              static_cast<int>(a->rows), static_cast<int>(a->o));
    if ((rc = check_launch())) return rc;
  }
  if (a->rows > 0 && inner) {
    CUtensorMap ma, mb, ms, md;
    const Shape shape = choose_shape(1, a->e, a->rows, a->m, a->o, info);
    if ((rc = make_bf16_map(&ma, a->dy, a->o, a->rows, a->e, a->o, a->rows * a->o, a_box(a->rows, shape), 64,
                            CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
    if ((rc = make_bf16_map(&mb, a->w_out, a->m, a->o, a->e, a->m, a->m * a->o, BK, 64,
                            CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
    if ((rc = make_pair_map(&ms, a->saved, a->m, a->rows, a->e))) return rc;
    if ((rc = make_pair_map(&md, a->dgu, a->m, a->rows, a->e))) return rc;
    GatedParams p;
    memset(&p, 0, sizeof(p));
    p.sums = a->db_in ? sums : nullptr;
    p.rows = static_cast<int>(a->rows);
    p.k = static_cast<int>(a->o);
    p.m = static_cast<int>(a->m);
    p.batch = static_cast<int>(a->e);
    if ((rc = launch(1, shape, ma, mb, ms, ms, md, p, false, info, stream))) return rc;
  }
  if (a->dx && a->rows > 0 &&
      (rc = product(a->dgu, a->w_in, 1, nullptr, 0, nullptr, nullptr, 0, 0, a->dx, a->e, a->rows, a->h,
                    2 * a->m, info, stream)))
    return rc;
  if (a->db_in || a->db_out) {
    SumsPart u = {sums, a->db_in, static_cast<int>((a->rows + 31) / 32),
                  a->db_in ? static_cast<int>(2 * a->m) : 0, a->db_in_mode == VMOE_GRAD_BF16,
                  a->db_in_mode == VMOE_GRAD_ADD};
    SumsPart v = {dy_sums, a->db_out, static_cast<int>((a->rows + ROW_BLOCK - 1) / ROW_BLOCK),
                  a->db_out ? static_cast<int>(a->o) : 0, a->db_out_mode == VMOE_GRAD_BF16,
                  a->db_out_mode == VMOE_GRAD_ADD};
    gated_join_sums_kernel<<<dim3((u.cols + 31) / 32 + (v.cols + 31) / 32, static_cast<unsigned>(a->e)),
                             256, 0, stream>>>(u, v);
    if ((rc = check_launch())) return rc;
  }
  if (a->dw_in && (rc = weight_gradient(a->dgu, a->x, a->e, a->rows, 2 * a->m, a->h, a->dw_in,
                                        a->dw_in_mode, pieces, stream)))
    return rc;
  if (a->dw_out && (rc = weight_gradient(a->dy, a->hid, a->e, a->rows, a->o, a->m, a->dw_out,
                                         a->dw_out_mode, pieces, stream)))
    return rc;
  return 0;
}
