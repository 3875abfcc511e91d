// Gated MLP of a few rows: the weights are read once, straight from global memory into the tensor
// core's register fragments.
//
// With R <= 32 rows the work is reading the weights (2 M K and O M elements), a few microseconds of
// HBM time, so what counts is how soon all of them are in flight. A CTA takes 16 hidden units (their
// gate and their up row) or 16 outputs; its warps, and the 1, 2, 4 or 8 CTAs of a cluster when
// there are few units, share the contraction in units of 64 elements (a 128-byte line of every row;
// units of 32 took 12 % longer over 32 experts of 512 x 1024), and a warp has two units' loads in
// flight. CTAs have 8 warps, or 4 when there are two CTAs for every SM anyway (32 experts x 4 rows
// 512 -> 1024: 21 us against 28; 1 row 768 -> 2048: 9.7 us against 8.6). m16n8k16 products take 16 weight
// rows as A and 8 rows of x as B; the contraction's order is free, so a thread's fragments of two products are 16 consecutive
// bytes of a weight row and of a row of x, and neither needs shared memory. Partial sums meet in
// shared memory, then over the cluster, in a fixed order. The tile kernel's 128-row tiles, TMA
// pipeline and TMEM would stay nearly empty here.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace vmoe {
namespace {

constexpr int GR_MAX_SPLIT = 8;
constexpr int GR_AHEAD = 4;  // chunks of 32 elements a warp loads before it multiplies the first one

struct RowsParams {
  const __nv_bfloat16* x;  // (E, rows, k)
  const __nv_bfloat16* w;  // forward: (E, 2, m, k); output projection: (E, m, k)
  const void* bias;        // (E, 2, m) / (E, m) or NULL
  const __nv_bfloat16* residual;
  __nv_bfloat16* out;      // (E, rows, m)
  __nv_bfloat16* saved;    // (E, rows, 2, m) or NULL
  long long ldx, x_batch_stride, ldr, r_batch_stride;
  int rows, k, m, split, bias_bf16, act, after;  // after: wait for the kernel in front
};

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float load_bias(const void* bias, int is_bf16, long long i) {
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i])
                 : static_cast<const float*>(bias)[i];
}

__device__ __forceinline__ uint4 ld_stream(const __nv_bfloat16* p) {  // read once: no L1 line
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}

// G weight groups of 16 rows: 2 (gate and up, gated = true) or 1; NT groups of 8 rows of x.
template <int NT, bool GATED, int GR_THREADS>
__global__ void __launch_bounds__(GR_THREADS, 512 / GR_THREADS) gated_rows_kernel(const RowsParams p) {
  constexpr int GR_WARPS = GR_THREADS / 32;
  constexpr int G = GATED ? 2 : 1;
  constexpr int COLS = NT * 8;
  constexpr int X_AHEAD = NT <= 2 ? GR_AHEAD : 1;  // registers for more of x's rows than 16 are not left
  __shared__ float part[GR_WARPS][G][16][COLS + 1];
  __shared__ float joined[G][16][COLS];
  // The output projection may start now: it fetches its weights and waits for these results.
  if (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int e = blockIdx.y;
  const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit0 = static_cast<int>(blockIdx.x) / p.split * 16;
  const int chunks = (p.k + 31) / 32;
  const int stride = GR_WARPS * p.split, first = rank * GR_WARPS + warp;

  // Rows past the end repeat the last one; their sums are not used.
  const __nv_bfloat16* wrow[G][2];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int unit = min(unit0 + g + 8 * j, p.m - 1);
      wrow[i][j] = p.w + ((static_cast<long long>(e) * G + i) * p.m + unit) * p.k;
    }
  const __nv_bfloat16* xrow[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    xrow[j] = p.x + e * p.x_batch_stride + static_cast<long long>(min(j * 8 + g, p.rows - 1)) * p.ldx;

  float acc[G][NT][4];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.0f;

  const uint4 zero = make_uint4(0, 0, 0, 0);
  bool waited = !p.after;
  for (int c0 = first; c0 * 2 < chunks; c0 += GR_AHEAD / 2 * stride) {
    uint4 wq[GR_AHEAD][G][2], xq[X_AHEAD][NT];
#pragma unroll
    for (int u = 0; u < GR_AHEAD; ++u) {
      const int k0 = (c0 + (u >> 1) * stride) * 64 + (u & 1) * 32 + t * 8;
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) wq[u][i][j] = k0 < p.k ? ld_stream(wrow[i][j] + k0) : zero;
    }
    if (!waited) {
      // The weights are on their way; x is what the kernel in front writes.
      asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
    }
    auto load_x = [&](int u, uint4 (&to)[NT]) {
      const int k0 = (c0 + (u >> 1) * stride) * 64 + (u & 1) * 32 + t * 8;
#pragma unroll
      for (int j = 0; j < NT; ++j)
        to[j] = k0 < p.k ? *reinterpret_cast<const uint4*>(xrow[j] + k0) : zero;
    };
#pragma unroll
    for (int u = 0; u < X_AHEAD; ++u) load_x(u, xq[u]);
#pragma unroll
    for (int u = 0; u < GR_AHEAD; ++u) {
      uint4 (&x)[NT] = xq[u % X_AHEAD];
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 a = wq[u][i][0], b = wq[u][i][1];
          mma_16x8x16(acc[i][j], a.x, b.x, a.y, b.y, x[j].x, x[j].y);
          mma_16x8x16(acc[i][j], a.z, b.z, a.w, b.w, x[j].z, x[j].w);
        }
      if (u + X_AHEAD < GR_AHEAD) load_x(u + X_AHEAD, x);
    }
  }
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");  // a warp without a chunk

  // Accumulator: unit g (+ 8), rows 2 t and 2 t + 1 of each group of 8.
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      part[warp][i][g][j * 8 + 2 * t] = acc[i][j][0];
      part[warp][i][g][j * 8 + 2 * t + 1] = acc[i][j][1];
      part[warp][i][g + 8][j * 8 + 2 * t] = acc[i][j][2];
      part[warp][i][g + 8][j * 8 + 2 * t + 1] = acc[i][j][3];
    }
  __syncthreads();
  constexpr int VALUES = 16 * COLS;
  for (int v = tid; v < G * VALUES; v += GR_THREADS) {
    const int i = v / VALUES, unit = v % VALUES / COLS, col = v % COLS;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < GR_WARPS; ++w) s += part[w][i][unit][col];
    joined[i][unit][col] = s;
  }
  if (p.split > 1) cluster_sync_all();
  else __syncthreads();

  // Each CTA of the cluster finishes its share of the values; units are contiguous in the output.
  for (int v = tid + rank * GR_THREADS; v < VALUES; v += GR_THREADS * p.split) {
    const int unit = v & 15, row = v >> 4;
    const int m = unit0 + unit;
    float s[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      s[i] = 0.0f;
      if (p.split == 1) {
        s[i] = joined[i][unit][row];
      } else {
        for (int q = 0; q < p.split; ++q) {
          float f;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(f)
                       : "r"(mapa_shared(smem_u32(&joined[i][unit][row]), static_cast<uint32_t>(q))));
          s[i] += f;
        }
      }
    }
    if (row >= p.rows || m >= p.m) continue;
    const long long at = (static_cast<long long>(e) * p.rows + row) * p.m + m;
    if (GATED) {
      float gate = s[0], up = s[G - 1];
      if (p.bias) {
        gate += load_bias(p.bias, p.bias_bf16, 2ll * e * p.m + m);
        up += load_bias(p.bias, p.bias_bf16, (2ll * e + 1) * p.m + m);
      }
      float a, slope, unused_a, unused_slope;
      gate_and_slope(gate, gate, p.act, a, unused_a, slope, unused_slope);
      p.out[at] = __float2bfloat16(a * up);
      if (p.saved) {
        const long long sat = (static_cast<long long>(e) * p.rows + row) * 2 * p.m + m;
        p.saved[sat] = __float2bfloat16(slope * up);
        p.saved[sat + p.m] = __float2bfloat16(a);
      }
    } else {
      float y = s[0];
      if (p.bias) y += load_bias(p.bias, p.bias_bf16, static_cast<long long>(e) * p.m + m);
      if (p.residual)
        y += __bfloat162float(p.residual[e * p.r_batch_stride + row * p.ldr + m]);
      p.out[at] = __float2bfloat16(y);
    }
  }
  if (p.split > 1) cluster_sync_all();  // no CTA leaves while another may read its sums
}

}  // namespace
}  // namespace vmoe
