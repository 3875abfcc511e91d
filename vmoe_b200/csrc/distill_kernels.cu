// Distillation from a teacher's top logits: selection of the k largest logits of every example
// with the log-sum-exp of all the others, and the divergence of a student from such a teacher
// with its gradient. Logits are bf16, fp16 or fp32 rows of any stride and alignment.
//
// Every kernel gives a row to one CTA, or to a cluster of 2, 4 or 8 CTAs that share it when there
// are few rows (each takes a range of columns, results meet in distributed shared memory), reads
// it in 16-byte vectors from the first aligned address on and the at most 14 edge elements one by
// one.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "ptx_sm100.cuh"
#include "vmoe_api.h"

namespace vmoe {

void set_error(const char* fmt, const char* a, int code);

namespace {

constexpr int DT = 256;  // threads per CTA of the kernels in this file
constexpr int DW = DT / 32;
constexpr int MAX_PARTS = 8;  // CTAs that can share a row (portable cluster size)

typedef unsigned long long u64;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }

// The 16 bytes of a vector as floats and back.
template <typename T>
struct Vec {
  static constexpr int W = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4], float) {
  v[0] = __uint_as_float(q.x);
  v[1] = __uint_as_float(q.y);
  v[2] = __uint_as_float(q.z);
  v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8], __half) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack(const float (&v)[4], float) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                    __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __nv_bfloat16) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8], __half) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of the values as unsigned integers: -inf < ... < -0 = +0 < ... < +inf < NaN; 0 is below
// every value and stands for "nothing here".
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((b & 0x7fffffffu) == 0) return 0x80000000u;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// Values beyond this are not multiplied by log2(e) / temperature before the row's anchor is taken
// off: masks of the type's lowest value would overflow.
constexpr float FAR = 1e30f;

// Where the vectors of a row start: `head` elements before the first 16-byte boundary, then
// `vectors` whole vectors, the rest of the n elements behind them.
template <typename T>
struct RowLayout {
  int head, vectors, tail;
  __device__ __forceinline__ RowLayout(const T* row, int n) {
    constexpr int W = Vec<T>::W;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = off == 0 ? 0 : min(W - off, n);
    vectors = (n - head) / W;
    tail = n - head - vectors * W;
  }
};

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* red, Op op) {  // result in every thread
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();  // `red` may still be read by an earlier reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int i = 1; i < DW; ++i) t = op(t, red[i]);
  return t;
}
struct Sum {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
  __device__ __forceinline__ double operator()(double a, double b) const { return a > b || a != a ? a : b; }
};
struct Min {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a < b ? a : b; }
};

// ------------------------------------------------------------------------------- top logits
constexpr int TOP_CAP = 2048;  // candidates that shared memory holds
constexpr int TOP_K_MAX = 256;

// One part of a row: NV vectors per thread stay in registers. The k largest of the threads'
// maxima (found by bisection on their order keys with one block-wide count per step) bound the
// k-th largest value from below, so everything not below that bound is a candidate: about k of
// them for values in no particular order. Candidates are ranked by counting larger ones. Ties
// that would overflow the candidate list (a row of equal values) take an exact bisection over
// values and then positions instead. The same pass sums the exponentials of everything that is
// not a candidate, relative to the bound; candidates that lose and a sum that underflows get
// anchors of their own, so that `rest` is right however far below the kept values it lies.
template <typename T, int NV>
__global__ void __launch_bounds__(DT)
top_logits_kernel(const T* __restrict__ logits, long long ld, int n, int k, float c, double inv_t,
                  int parts, T* __restrict__ values, int* __restrict__ indices,
                  float* __restrict__ rest) {
  constexpr int W = Vec<T>::W;
  __shared__ u64 cand[TOP_CAP];
  __shared__ u64 top[TOP_K_MAX];
  __shared__ uint32_t red_u[DW];
  __shared__ float red_f[DW];
  __shared__ int count;
  __shared__ float2 part_rest[MAX_PARTS];
  const int tid = threadIdx.x;
  const int part = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long r = blockIdx.x / parts;
  const T* x = logits + r * ld;
  const RowLayout<T> lay(x, n);
  const int per = (lay.vectors + parts - 1) / parts;
  const int v0 = min(part * per, lay.vectors), v1 = min(v0 + per, lay.vectors);
  const uint4* xv = reinterpret_cast<const uint4*>(x + lay.head);

  // This part's elements: up to NV vectors per thread, and one edge element in part 0.
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = v0 + tid + i * DT;
    if (j < v1) raw[i] = __ldg(xv + j);
  }
  const int edges = part == 0 ? lay.head + lay.tail : 0;
  const bool has_edge = tid < edges;
  const int edge_at = tid < lay.head ? tid : n - lay.tail + (tid - lay.head);
  const float edge = has_edge ? to_float(x[edge_at]) : -INFINITY;
  if (tid == 0) count = 0;

  uint32_t best = has_edge ? key_of(edge) : 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (v0 + tid + i * DT < v1) {
      float v[W];
      unpack(raw[i], v, T());
#pragma unroll
      for (int e = 0; e < W; ++e) best = max(best, key_of(v[e]));
    }
  }
  const int mine = min(k, (v1 - v0) * W + edges);  // entries this part can contribute

  // Bound: at least `mine` elements have a key >= bound (0: all elements).
  const int filled = __syncthreads_count(best != 0);
  uint32_t bound = 0;
  if (filled >= mine && mine > 0) {
    const uint32_t hi0 = block_reduce(best, red_u, Max());
    const uint32_t lo0 = block_reduce(best ? best : 0xffffffffu, red_u, Min());
    uint32_t lo = lo0, hi = hi0;  // count(>= lo) >= mine; the bound is <= hi
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      const int got = __syncthreads_count(best >= mid);
      if (got >= mine) {
        lo = mid;
        if (got <= mine + mine / 4 + 8) break;
      } else {
        hi = mid - 1;
      }
    }
    bound = lo;
  }

  int last_at = 0x7fffffff;  // elements equal to the bound count up to this position
  float m = 0.0f, s = 0.0f;  // the sum of what is not kept, as sum of 2^((x - m) c)
  for (int attempt = 0;; ++attempt) {
    // Everything not a candidate lies at or below the bound. A bound that cannot be an anchor
    // (infinite, NaN, a mask's value) leaves the sum to the code behind the ranking.
    m = bound ? value_of(bound) : -INFINITY;
    const bool near = fabsf(m) < FAR;
    const float anchor = near ? -m * c : 0.0f;
    s = 0.0f;
    auto element = [&](float v, int at) {
      const uint32_t key = key_of(v);
      if (key > bound || (key == bound && at <= last_at)) {
        const int pos = atomicAdd(&count, 1);
        if (pos < TOP_CAP)
          cand[pos] = (static_cast<u64>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(at));
      } else if (near) {
        s += exp2_approx(fmaf(v, c, anchor));
      }
    };
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = v0 + tid + i * DT;
      if (j < v1) {
        float v[W];
        unpack(raw[i], v, T());
#pragma unroll
        for (int e = 0; e < W; ++e) element(v[e], lay.head + j * W + e);
      }
    }
    if (has_edge) element(edge, edge_at);
    if (near) s *= exp2_approx(-fmaf(m, c, anchor));  // the anchor's own rounding
    __syncthreads();
    if (count <= TOP_CAP || attempt == 1) break;
    // Too many candidates: the exact k-th largest key, then the position of the last element
    // equal to it that still belongs to the k largest.
    auto count_if = [&](auto test) {
      int got = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = v0 + tid + i * DT;
        if (j < v1) {
          float v[W];
          unpack(raw[i], v, T());
#pragma unroll
          for (int e = 0; e < W; ++e) got += test(key_of(v[e]), lay.head + j * W + e) ? 1 : 0;
        }
      }
      if (has_edge) got += test(key_of(edge), edge_at) ? 1 : 0;
      return static_cast<int>(block_reduce(static_cast<uint32_t>(got), red_u, Sum()));
    };
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t trial = kth | (1u << bit);
      if (count_if([&](uint32_t key, int) { return key >= trial; }) >= mine) kth = trial;
    }
    const int need = mine - count_if([&](uint32_t key, int) { return key > kth; });
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (count_if([&](uint32_t key, int at) { return key == kth && at <= mid; }) >= need) hi = mid;
      else lo = mid + 1;
    }
    bound = kth;
    last_at = lo;
    __syncthreads();
    if (tid == 0) count = 0;
  }
  const int found = count;

  // Rank of every candidate; the first `mine` in order go to top[].
  uint32_t lost = 0;  // largest key of this thread's candidates that lose
  uint32_t lost_mask = 0;
#pragma unroll 1
  for (int i = tid, q = 0; i < found; i += DT, ++q) {
    const u64 me = cand[i];
    int rank = 0;
    for (int j = 0; j < found; ++j) rank += cand[j] > me ? 1 : 0;
    if (rank < mine) {
      top[rank] = me;
    } else {
      lost = max(lost, static_cast<uint32_t>(me >> 32));
      lost_mask |= 1u << q;
    }
  }
  s = block_reduce(s, red_f, Sum());
  lost = block_reduce(lost, red_u, Max());  // its barriers also publish top[]
  // Adds values (each thread's own, through `each`) whose largest key is `key` to the sum; none of
  // them lies below what is in the sum already.
  auto add_at = [&](uint32_t key, auto each) {
    const float top_value = value_of(key);
    if (!(top_value < INFINITY)) {  // +inf or NaN: so is the sum
      m = 0.0f;
      s = top_value;
      return;
    }
    float t = 0.0f;
    if (top_value > -INFINITY) {
      each([&](float v) { t += exp2_approx((v - top_value) * c); });
      t = block_reduce(t, red_f, Sum());
      s = (s > 0.0f ? s * exp2_approx((m - top_value) * c) : s) + t;
      m = top_value;
    }
  };
  if (lost) {
    // The losing candidates are at or above the bound: their largest is the new anchor.
    add_at(lost, [&](auto add) {
#pragma unroll 1
      for (int i = tid, q = 0; i < found; i += DT, ++q)
        if (lost_mask >> q & 1) add(value_of(static_cast<uint32_t>(cand[i] >> 32)));
    });
  } else if (s < 1e-30f) {
    // Nothing, or all of it far below the bound: anchor at the largest of it.
    auto below = [&](float v, int at) {
      const uint32_t key = key_of(v);
      return !(key > bound || (key == bound && at <= last_at)) ? key : 0u;
    };
    auto walk = [&](auto visit) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = v0 + tid + i * DT;
        if (j < v1) {
          float v[W];
          unpack(raw[i], v, T());
#pragma unroll
          for (int e = 0; e < W; ++e) visit(v[e], lay.head + j * W + e);
        }
      }
      if (has_edge) visit(edge, edge_at);
    };
    uint32_t low = 0;
    walk([&](float v, int at) { low = max(low, below(v, at)); });
    low = block_reduce(low, red_u, Max());
    s = 0.0f;
    if (low)
      add_at(low, [&](auto add) {
        walk([&](float v, int at) {
          if (below(v, at)) add(v);
        });
      });
  }

  auto emit = [&](int rank, u64 entry) {
    const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(entry));
    indices[r * k + rank] = at;
    values[r * k + rank] = x[at];
  };
  auto log_of = [&](float top_value, float sum) {
    return sum == 0.0f ? -INFINITY
                       : static_cast<float>(top_value * inv_t + log(static_cast<double>(sum)));
  };
  if (parts == 1) {
    for (int i = tid; i < mine; i += DT) emit(i, top[i]);
    if (tid == 0) rest[r] = log_of(m, s);
    return;
  }

  // The parts' sorted lists meet: an entry's place in the row is its place here plus the number
  // of larger entries in the other lists.
  for (int i = tid; i < TOP_K_MAX; i += DT)
    if (i >= mine) top[i] = 0;
  cluster_sync_all();
  u64* lists = cand;  // [parts][TOP_K_MAX], this CTA's candidates are no longer needed
  static_assert(TOP_CAP >= MAX_PARTS * TOP_K_MAX, "the parts' lists take the candidates' place");
  for (int i = tid; i < parts * k; i += DT) {
    const int p = i / k, q = i % k;
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];"
                 : "=l"(v)
                 : "r"(mapa_shared(smem_u32(top + q), static_cast<uint32_t>(p))));
    lists[p * TOP_K_MAX + q] = v;
  }
  __syncthreads();
  uint32_t out_key = 0;
  u64 me = 0;
  if (tid < mine) {
    me = top[tid];
    int rank = tid;
    for (int p = 0; p < parts; ++p) {
      if (p == part) continue;
      int lo = 0, hi = k;  // first position whose entry is smaller
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (lists[p * TOP_K_MAX + mid] > me) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < k) emit(rank, me);
    else out_key = static_cast<uint32_t>(me >> 32);
  }
  const uint32_t high = block_reduce(out_key, red_u, Max());
  if (high)
    add_at(high, [&](auto add) {
      if (out_key) add(value_of(out_key));
    });
  if (tid == 0) {
    const uint32_t dst = mapa_shared(smem_u32(part_rest + part), 0);
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(m), "f"(s) : "memory");
  }
  cluster_sync_all();  // also: no CTA leaves while another may read its list
  if (part == 0 && tid == 0) {
    float top_value = -INFINITY, total = 0.0f;
    for (int p = 0; p < parts; ++p)
      if (part_rest[p].y != 0.0f) top_value = fmaxf(top_value, part_rest[p].x);
    for (int p = 0; p < parts; ++p) {
      const float2 pr = part_rest[p];
      if (pr.y != 0.0f) total += pr.y * exp2_approx((pr.x - top_value) * c);
    }
    rest[r] = log_of(top_value, total);
  }
}

// ------------------------------------------------------------------------------- divergence
__device__ __forceinline__ double load_value(const void* p, int dtype, long long i) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ int load_index(const void* p, int wide, long long i, int n) {
  const long long v = wide ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
  return v >= 0 && v < n ? static_cast<int>(v) : -1;
}

struct DistillParams {
  const void* values;
  const void* indices;
  const float* rest;  // NULL: the kept classes are the teacher's whole distribution
  float* loss;
  float2* stats;      // per row: anchor and factor of the classes that are not kept
  float* slopes;      // per kept class: student's minus teacher's probability
  long long ld, ld_values, ld_indices;
  int n, k, values_dtype, indices_wide, parts;
  float c;            // log2(e) / temperature
  double temperature;
};

// Running sum of exponentials with the largest x so far as anchor: s * 2^-a = sum of 2^(x c) with
// a = -m c rounded to fp32, or s = sum of 2^((x - m) c) where m lies beyond FAR.
struct Running {
  float m, a, s;
  __device__ __forceinline__ bool far() const { return !(fabsf(m) < FAR); }
  // What a sum relative to (m0, a0) is worth relative to this anchor.
  __device__ __forceinline__ float worth(float m0, float a0, float s0, float c) const {
    if (s0 == 0.0f) return 0.0f;
    return s0 * exp2_approx(far() || !(fabsf(m0) < FAR) ? (m0 - m) * c : a - a0);
  }
  __device__ __forceinline__ void raise(float top, float c) {
    if (top > m) {
      const Running old = *this;
      m = top;
      a = -top * c;
      s = worth(old.m, old.a, old.s, c);
    }
  }
  __device__ __forceinline__ float of(float x, float c) const {
    return far() ? exp2_approx((x - m) * c) : exp2_approx(fmaf(x, c, a));
  }
  __device__ __forceinline__ void join(float m0, float a0, float s0, float c) {
    raise(m0, c);
    s += worth(m0, a0, s0, c);
  }
};

// The student's exponentials are summed over the classes that are NOT kept (a bitmap in shared
// memory marks the kept ones; one byte test per 8 bf16 elements), in one pass with a running
// maximum. The at most k + 1 terms of the divergence are evaluated in 64 bits: where student and
// teacher agree their first-order parts cancel, and so do q - p in the gradient. stats and slopes
// leave nothing but one exponential per class to the backward pass.
template <typename T>
__global__ void __launch_bounds__(DT)
distill_fwd_kernel(const T* __restrict__ logits, const DistillParams p) {
  constexpr int W = Vec<T>::W;
  extern __shared__ uint32_t bitmap[];
  __shared__ double red_d[DW];
  __shared__ float4 red_run[DW];
  __shared__ float4 part_run[MAX_PARTS];
  __shared__ int repeated;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = p.parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long r = blockIdx.x / p.parts;
  const int n = p.n, k = p.k;
  const T* x = logits + r * p.ld;
  const RowLayout<T> lay(x, n);
  const int per = (lay.vectors + p.parts - 1) / p.parts;
  const int v0 = min(part * per, lay.vectors), v1 = min(v0 + per, lay.vectors);
  // Bit of element e: the part's vectors from bit W on, the edges in front of and behind them.
  const int first = lay.head + v0 * W - W;
  const int last = part == p.parts - 1 ? n : lay.head + v1 * W;
  const int words = (last - first + 31) / 32;
  for (int i = tid; i < words; i += DT) bitmap[i] = 0;
  if (tid == 0) repeated = 0;
  __syncthreads();
  for (int i = tid; i < k; i += DT) {
    const int at = load_index(p.indices, p.indices_wide, r * p.ld_indices + i, n);
    const bool here = at >= (part == 0 ? 0 : first + W) && at < last;
    if (here) {
      const int b = at - first;
      if (atomicOr(&bitmap[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) repeated = 1;
    }
  }
  __syncthreads();

  Running run = {-INFINITY, INFINITY, 0.0f};
  const float c = p.c;
  const uint4* xv = reinterpret_cast<const uint4*>(x + lay.head);
  const uint8_t* marks = reinterpret_cast<const uint8_t*>(bitmap);
  constexpr int U = 4;
  for (int j0 = v0 + tid; j0 < v1; j0 += U * DT) {
    uint4 raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j0 + i * DT < v1) raw[i] = __ldg(xv + j0 + i * DT);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = j0 + i * DT;
      if (j >= v1) break;
      float v[W];
      unpack(raw[i], v, T());
      const int b = (j - v0 + 1) * W;
      const uint32_t mark = (marks[b >> 3] >> (b & 7)) & ((1u << W) - 1u);
      if (mark) {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (mark >> e & 1) v[e] = -INFINITY;
      }
      float top = v[0];
#pragma unroll
      for (int e = 1; e < W; ++e) top = fmaxf(top, v[e]);
      run.raise(top, c);
      if (!(top == -INFINITY)) {
#pragma unroll
        for (int e = 0; e < W; ++e) run.s += run.of(v[e], c);
      }
    }
  }
  {
    const int edges = (part == 0 ? lay.head : 0) + (part == p.parts - 1 ? lay.tail : 0);
    if (tid < edges) {
      const int at = part == 0 && tid < lay.head ? tid : n - lay.tail + (tid - (part == 0 ? lay.head : 0));
      const int b = at - first;
      const float v = bitmap[b >> 5] >> (b & 31) & 1 ? -INFINITY : to_float(x[at]);
      run.raise(v, c);
      if (!(v == -INFINITY)) run.s += run.of(v, c);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, run.m, o);
    const float a = __shfl_xor_sync(0xffffffffu, run.a, o);
    const float s = __shfl_xor_sync(0xffffffffu, run.s, o);
    run.join(m, a, s, c);
  }
  if (lane == 0) red_run[warp] = make_float4(run.m, run.a, run.s, 0.0f);
  __syncthreads();
  run = {red_run[0].x, red_run[0].y, red_run[0].z};
#pragma unroll
  for (int i = 1; i < DW; ++i) run.join(red_run[i].x, red_run[i].y, red_run[i].z, c);
  if (p.parts > 1) {
    if (tid == 0) {
      const uint32_t dst = mapa_shared(smem_u32(part_run + part), 0);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(run.m),
                   "f"(run.a), "f"(run.s), "f"(__int_as_float(repeated))
                   : "memory");
    }
    cluster_sync_all();
    if (part != 0) return;
    run = {part_run[0].x, part_run[0].y, part_run[0].z};
    int any = __float_as_int(part_run[0].w);
    for (int i = 1; i < p.parts; ++i) {
      run.join(part_run[i].x, part_run[i].y, part_run[i].z, c);
      any |= __float_as_int(part_run[i].w);
    }
    if (tid == 0) repeated = any;
    __syncthreads();
  }

  // Natural-log units from here on, in 64 bits, maxima and sums kept apart (a maximum of the size
  // of a mask's value would swallow the logarithm of its sum). zm, zs: the classes not kept;
  // fmaf(m, c, a) is what rounding the anchor to fp32 left over.
  const double inv_t = 1.0 / p.temperature;
  const bool some = run.s != 0.0f;
  const double zm = some ? run.m * inv_t : -INFINITY;
  const double zs = run.far() ? run.s : run.s * exp2(-static_cast<double>(fmaf(run.m, c, run.a)));
  const double tr = p.rest ? static_cast<double>(p.rest[r]) : -INFINITY;
  auto entry = [&](int i, double& t, double& z) {  // teacher's and student's logit; false: left out
    const int at = load_index(p.indices, p.indices_wide, r * p.ld_indices + i, n);
    if (at < 0) return false;
    if (repeated)  // the first entry of a class counts
      for (int j = 0; j < i; ++j)
        if (load_index(p.indices, p.indices_wide, r * p.ld_indices + j, n) == at) return false;
    t = load_value(p.values, p.values_dtype, r * p.ld_values + i) * inv_t;
    z = to_float(x[at]) * inv_t;
    return true;
  };
  double t_max = tr, z_max = zm;
  for (int i = tid; i < k; i += DT) {
    double t, z;
    if (!entry(i, t, z)) continue;
    t_max = Max()(t, t_max);
    z_max = Max()(z, z_max);
  }
  t_max = block_reduce(t_max, red_d, Max());
  z_max = block_reduce(z_max, red_d, Max());
  auto part_of = [](double v, double top) { return v == -INFINITY ? 0.0 : exp(v - top); };
  double t_sum = 0.0, z_sum = 0.0;
  for (int i = tid; i < k; i += DT) {
    double t, z;
    if (!entry(i, t, z)) continue;
    t_sum += part_of(t, t_max);
    z_sum += part_of(z, z_max);
  }
  t_sum = block_reduce(t_sum, red_d, Sum()) + part_of(tr, t_max);
  z_sum = block_reduce(z_sum, red_d, Sum()) + part_of(zm, z_max) * zs;
  const double t_log = log(t_sum), z_log = log(z_sum);
  // Teacher's and student's probability of an outcome, and its term of the divergence. A teacher
  // without any mass (no entry left, no rest) teaches nothing.
  const bool silent = t_max == -INFINITY;
  double loss = 0.0;
  auto outcome = [&](double t, double z, double sum, double& q) {  // student: sum * e^z
    const double pt = t == -INFINITY ? 0.0 : exp(t - t_max - t_log);
    const double log_q = z == -INFINITY ? z : z - z_max + log(sum) - z_log;
    q = silent ? 0.0 : exp(log_q);
    if (pt != 0.0) loss += pt * ((t - t_max - t_log) - log_q);
    return pt;
  };
  for (int i = tid; i < k; i += DT) {
    double t, z, q;
    float slope = 0.0f;
    if (entry(i, t, z)) {
      const double pt = outcome(t, z, 1.0, q);
      slope = static_cast<float>(q - pt);
    }
    p.slopes[r * k + i] = slope;
  }
  double q_rest = 0.0, p_rest = 0.0;
  if (tid == 0) p_rest = outcome(tr, zm, zs, q_rest);
  loss = block_reduce(loss, red_d, Sum());
  if (tid == 0) {
    p.loss[r] = static_cast<float>(loss * p.temperature * p.temperature);
    // Gradient of a class that is not kept: q_j (1 - p_rest / q_rest).
    p.stats[r] = make_float2(run.m, some ? static_cast<float>((q_rest - p_rest) / run.s) : 0.0f);
  }
}

// d loss / d logits * d_loss: 2^((x - anchor) c) * factor for the classes that are not kept, the
// saved slope for the others. One read and one write of the row; a row whose d_loss is zero (padding)
// is zeroed without being read. Columns n .. n_pad (row padding of the gradient) get zeros.
template <typename T>
__global__ void __launch_bounds__(DT)
distill_bwd_kernel(const T* __restrict__ logits, const void* __restrict__ indices, int indices_wide,
                   long long ld_indices, const float2* __restrict__ stats,
                   const float* __restrict__ slopes, const float* __restrict__ d_loss,
                   long long d_loss_stride, T* __restrict__ grad, long long ld, long long ld_grad,
                   int n, int n_pad, int k, int parts, float c, float temperature) {
  constexpr int W = Vec<T>::W;
  const int tid = threadIdx.x;
  const long long r = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  const T* x = logits + r * ld;
  T* g = grad + r * ld_grad;
  const RowLayout<T> lay(x, n);
  const int per = (lay.vectors + parts - 1) / parts;
  const int v0 = min(part * per, lay.vectors), v1 = min(v0 + per, lay.vectors);
  const float scale = d_loss[r * d_loss_stride] * temperature;
  const float2 st = stats[r];
  const float factor = st.y * scale;
  const uint4* xv = reinterpret_cast<const uint4*>(x + lay.head);
  uint4* gv = reinterpret_cast<uint4*>(g + lay.head);
  const bool skip = scale == 0.0f;
  const Running run = {st.x, -st.x * c, 0.0f};  // the forward pass's anchor
  auto value = [&](float v) { return skip || factor == 0.0f ? 0.0f : run.of(v, c) * factor; };
  constexpr int U = 4;
  for (int j0 = v0 + tid; j0 < v1; j0 += U * DT) {
    uint4 raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if (!skip && j0 + i * DT < v1) raw[i] = __ldg(xv + j0 + i * DT);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (j0 + i * DT < v1) {
        float v[W];
        unpack(raw[i], v, T());
#pragma unroll
        for (int e = 0; e < W; ++e) v[e] = value(v[e]);
        gv[j0 + i * DT] = pack(v, T());
      }
    }
  }
  if (part == 0) {
    const int edges = lay.head + lay.tail;
    if (tid < edges) {
      const int at = tid < lay.head ? tid : n - lay.tail + (tid - lay.head);
      g[at] = from_float<T>(value(skip ? 0.0f : to_float(x[at])));
    }
    for (int i = n + tid; i < n_pad; i += DT) g[i] = from_float<T>(0.0f);
  }
  // The kept classes of this part's columns: written after the block's own stores above.
  if (skip) return;
  __syncthreads();
  const int c0 = lay.head + v0 * W, c1 = lay.head + v1 * W;
  for (int i = tid; i < k; i += DT) {
    const int at = load_index(indices, indices_wide, r * ld_indices + i, n);
    const bool edge = at < lay.head || at >= lay.head + lay.vectors * W;
    if (at < 0 || !(edge ? part == 0 : at >= c0 && at < c1)) continue;
    bool first = true;  // a class that is listed again has its slope at its first entry
    const float slope = slopes[r * k + i];
    if (slope == 0.0f)
      for (int j = 0; j < i && first; ++j)
        first = load_index(indices, indices_wide, r * ld_indices + j, n) != at;
    if (first) g[at] = from_float<T>(slope * scale);
  }
}

int check_launch() {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    return -5;
  }
  return 0;
}

template <typename... Params, typename... Args>
int launch_clusters(void (*kernel)(Params...), int64_t rows, int parts, size_t smem, cudaStream_t stream,
                    Args... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(parts);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(DT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    cudaGetLastError();
    return -5;
  }
  return 0;
}

int bad(const char* what) {
  set_error("%s (code %d)", what, 0);
  return -1;
}

constexpr int kTargetCtas = 296;  // two CTAs per SM

// CTAs per row: enough to give every SM two, as long as each keeps `least` vectors.
int choose_parts(int64_t rows, int vectors, int least) {
  int parts = 1;
  while (parts < MAX_PARTS && rows * parts < kTargetCtas && vectors / (2 * parts) >= least) parts *= 2;
  return parts;
}

constexpr int TOP_NV_MAX = 12;
constexpr int64_t MAX_ROWS = 1 << 27;

template <typename T>
int top_logits(const void* logits, int64_t rows, int64_t n, int64_t ld, int64_t k, double temperature,
               void* values, int32_t* indices, float* rest, cudaStream_t stream) {
  constexpr int W = Vec<T>::W;
  const int vectors = static_cast<int>(n / W);
  int parts = choose_parts(rows, vectors, DT);
  while (parts < MAX_PARTS && (vectors + parts - 1) / parts > TOP_NV_MAX * DT) parts *= 2;
  const int nv = ((vectors + parts - 1) / parts + DT - 1) / DT;
  const float c = static_cast<float>(1.4426950408889634 / temperature);
  const double inv_t = 1.0 / temperature;
#define VMOE_TOP(NV)                                                                              \
  return launch_clusters(top_logits_kernel<T, NV>, rows, parts, 0, stream,                        \
                         static_cast<const T*>(logits), static_cast<long long>(ld),               \
                         static_cast<int>(n), static_cast<int>(k), c, inv_t, parts,               \
                         static_cast<T*>(values), indices, rest)
  if (nv <= 1) VMOE_TOP(1);
  if (nv <= 2) VMOE_TOP(2);
  if (nv <= 4) VMOE_TOP(4);
  if (nv <= 8) VMOE_TOP(8);
  if (nv <= TOP_NV_MAX) VMOE_TOP(TOP_NV_MAX);
#undef VMOE_TOP
  return bad("top_logits: too many classes");
}

}  // namespace
}  // namespace vmoe

using namespace vmoe;

extern "C" int64_t vmoe_top_logits_max_classes(int32_t dtype) {
  return static_cast<int64_t>(MAX_PARTS) * TOP_NV_MAX * DT * (dtype == 0 ? 4 : 8);
}

extern "C" int vmoe_top_logits(const void* logits, int32_t dtype, int64_t rows, int64_t n, int64_t ld,
                               int64_t k, double temperature, void* values, int32_t* indices,
                               float* rest, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (rows == 0) return 0;
  if (rows < 0 || rows > MAX_ROWS || n < 1 || n > vmoe_top_logits_max_classes(dtype))
    return bad("top_logits: rows or classes out of range");
  if (k < 1 || k > n || k > TOP_K_MAX) return bad("top_logits: k must be in 1 .. min(classes, 256)");
  if (!(temperature > 0.0)) return bad("top_logits: temperature must be positive");
  switch (dtype) {
    case 0: return top_logits<float>(logits, rows, n, ld, k, temperature, values, indices, rest, stream);
    case 1: return top_logits<__nv_bfloat16>(logits, rows, n, ld, k, temperature, values, indices, rest, stream);
    case 2: return top_logits<__half>(logits, rows, n, ld, k, temperature, values, indices, rest, stream);
  }
  return bad("top_logits: unknown dtype");
}

extern "C" int64_t vmoe_distill_max_classes(void) { return 1 << 18; }

extern "C" int vmoe_distill_fwd(const VmoeDistillArgs* a, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows == 0) return 0;
  if (a->rows < 0 || a->rows > MAX_ROWS || a->n < 1 || a->n > vmoe_distill_max_classes() || a->k < 1 ||
      a->k > (1 << 20))
    return bad("distill: rows, classes or kept classes out of range");
  if (!(a->temperature > 0.0)) return bad("distill: temperature must be positive");
  DistillParams p;
  p.values = a->values;
  p.indices = a->indices;
  p.rest = a->rest;
  p.loss = a->loss;
  p.stats = reinterpret_cast<float2*>(a->stats);
  p.slopes = a->slopes;
  p.ld = a->ld;
  p.ld_values = a->ld_values;
  p.ld_indices = a->ld_indices;
  p.n = static_cast<int>(a->n);
  p.k = static_cast<int>(a->k);
  p.values_dtype = a->values_dtype;
  p.indices_wide = a->indices_wide;
  p.c = static_cast<float>(1.4426950408889634 / a->temperature);
  p.temperature = a->temperature;
  const int width = a->dtype == 0 ? 4 : 8;
  p.parts = choose_parts(a->rows, static_cast<int>(a->n / width), 2 * DT);
  const size_t smem = ((a->n / width + p.parts - 1) / p.parts + 4) * width / 8 + 8;
  switch (a->dtype) {
    case 0: return launch_clusters(distill_fwd_kernel<float>, a->rows, p.parts, smem, stream,
                                   static_cast<const float*>(a->logits), p);
    case 1: return launch_clusters(distill_fwd_kernel<__nv_bfloat16>, a->rows, p.parts, smem, stream,
                                   static_cast<const __nv_bfloat16*>(a->logits), p);
    case 2: return launch_clusters(distill_fwd_kernel<__half>, a->rows, p.parts, smem, stream,
                                   static_cast<const __half*>(a->logits), p);
  }
  return bad("distill: unknown dtype");
}

extern "C" int vmoe_distill_bwd(const VmoeDistillArgs* a, const float* d_loss, int64_t d_loss_stride,
                                void* grad, int64_t ld_grad, int64_t n_pad, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows == 0) return 0;
  if (a->rows < 0 || a->rows > MAX_ROWS || a->n < 1 || a->n > vmoe_distill_max_classes() ||
      n_pad < a->n || n_pad > ld_grad)
    return bad("distill: rows or classes out of range");
  const int itemsize = a->dtype == 0 ? 4 : 2;
  // Gradient rows are written in the logits' vectors: both must start at the same offset
  // within 16 bytes, row by row.
  if ((reinterpret_cast<uintptr_t>(a->logits) - reinterpret_cast<uintptr_t>(grad)) % 16 ||
      ((a->ld - ld_grad) * itemsize) % 16)
    return bad("distill: gradient rows must have the alignment of the logits' rows");
  const int parts = choose_parts(a->rows, static_cast<int>(a->n / (16 / itemsize)), DT);
  const unsigned grid = static_cast<unsigned>(a->rows * parts);
  const float c = static_cast<float>(1.4426950408889634 / a->temperature);
#define VMOE_DISTILL_BWD(T)                                                                         \
  distill_bwd_kernel<T><<<grid, DT, 0, stream>>>(                                                   \
      static_cast<const T*>(a->logits), a->indices, a->indices_wide, a->ld_indices,                 \
      reinterpret_cast<const float2*>(a->stats), a->slopes, d_loss, d_loss_stride,                  \
      static_cast<T*>(grad), a->ld, ld_grad, static_cast<int>(a->n), static_cast<int>(n_pad),       \
      static_cast<int>(a->k), parts, c, static_cast<float>(a->temperature))
  switch (a->dtype) {
    case 0: VMOE_DISTILL_BWD(float); break;
    case 1: VMOE_DISTILL_BWD(__nv_bfloat16); break;
    case 2: VMOE_DISTILL_BWD(__half); break;
    default: return bad("distill: unknown dtype");
  }
#undef VMOE_DISTILL_BWD
  return check_launch();
}
