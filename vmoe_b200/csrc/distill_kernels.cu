// Distillation from a teacher's top logits: selection of the k largest logits of every example
// with the log-sum-exp of all the others, and the divergence of a student from such a teacher
// with its gradient. Logits are bf16, fp16 or fp32 rows of any stride and alignment.
//
// The selection brings a row to shared memory first: one bulk asynchronous copy of its whole 16-byte
// vectors, which needs no registers and has the whole row in flight at once; the at most two partial
// vectors at the ends are filled element by element, padded with -inf. A second pass over the row
// then costs no memory traffic. A row belongs to one CTA, or to a cluster of 2, 4 or 8 CTAs when there
// are few rows or the row does not fit one (each takes a range of vectors, results meet in
// distributed shared memory). The divergence reads its rows as a stream.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "ptx_sm100.cuh"
#include "vmoe_api.h"

namespace vmoe {

void set_error(const char* fmt, const char* a, int code);

namespace {

constexpr int MAX_PARTS = 8;  // CTAs that can share a row (portable cluster size)
constexpr int MAX_PART_BYTES = 176 * 1024;  // of a row in one CTA's shared memory

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

// Order of the values as unsigned integers (16 bits of them for 16-bit types): -inf < ... < -0 = +0
// < ... < +inf < NaN; 0 is below every value and stands for "nothing here".
template <typename T>
struct Order;
template <>
struct Order<float> {
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if ((b & 0x7fffffffu) == 0) return 0x80000000u;
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    if (key == 0xffffffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
  }
  // Largest of a vector joined with `m`; NaN wins.
  static __device__ __forceinline__ uint32_t largest(uint32_t m, const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    float f = __uint_as_float(m);
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(f) : "f"(__uint_as_float(w[i])));
    return __float_as_uint(f);
  }
  static constexpr uint32_t kLow = 0xff800000u;  // -inf, as `largest` starts
  static __device__ __forceinline__ uint32_t key_of_largest(uint32_t m) { return key(m); }
  static __device__ __forceinline__ float value_of_largest(uint32_t m) { return __uint_as_float(m); }
  static __device__ __forceinline__ bool all_below(uint32_t m, float bound) {
    return __uint_as_float(m) < bound;
  }
};
template <typename T>
struct Order16 {
  static constexpr uint32_t kInf = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  static __device__ __forceinline__ uint32_t key(uint32_t b) {
    if ((b & 0x7fffu) > kInf) return 0xffffu;
    if ((b & 0x7fffu) == 0) return 0x8000u;
    return b ^ ((b >> 15) ? 0xffffu : 0x8000u);
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    const uint32_t b = key == 0xffffu ? 0x7fffu : key ^ ((key >> 15) ? 0x8000u : 0xffffu);
    const unsigned short h = static_cast<unsigned short>(b);
    return to_float(*reinterpret_cast<const T*>(&h));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    if (std::is_same<T, __half>::value) {
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    } else {
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    }
    return r;
  }
  static __device__ __forceinline__ uint32_t largest(uint32_t m, const uint4& q) {
    return max2(m, max2(max2(q.x, q.y), max2(q.z, q.w)));
  }
  static constexpr uint32_t kLow = 0x80008000u | kInf | (kInf << 16);
  static __device__ __forceinline__ uint32_t key_of_largest(uint32_t m) {
    const uint32_t a = key(m & 0xffffu), b = key(m >> 16);
    return a > b ? a : b;
  }
  static __device__ __forceinline__ float value_of_largest(uint32_t m) {
    const uint32_t one = max2(m, m >> 16);  // the larger half in the low 16 bits
    const unsigned short h = static_cast<unsigned short>(one);
    return to_float(*reinterpret_cast<const T*>(&h));
  }
  static __device__ __forceinline__ bool all_below(uint32_t m, float bound) {
    const unsigned short h0 = static_cast<unsigned short>(m), h1 = static_cast<unsigned short>(m >> 16);
    return to_float(*reinterpret_cast<const T*>(&h0)) < bound &&
           to_float(*reinterpret_cast<const T*>(&h1)) < bound;
  }
};
template <>
struct Order<__nv_bfloat16> : Order16<__nv_bfloat16> {};
template <>
struct Order<__half> : Order16<__half> {};

// Bits of element e of a vector.
template <typename T>
__device__ __forceinline__ uint32_t bits_at(const uint4& q, int e) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if (sizeof(T) == 4) return w[e];
  return e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
}

template <typename T>
__device__ __forceinline__ uint4 low_vector() {  // -inf everywhere
  constexpr uint32_t w = Order<T>::kLow;
  return make_uint4(w, w, w, w);
}

// -inf in place of the elements whose bit is set in `mark`.
__device__ __forceinline__ void mask_vector(uint4& q, uint32_t mark, float) {
  if (mark & 1) q.x = 0xff800000u;
  if (mark & 2) q.y = 0xff800000u;
  if (mark & 4) q.z = 0xff800000u;
  if (mark & 8) q.w = 0xff800000u;
}
template <typename T>
__device__ __forceinline__ void mask_vector(uint4& q, uint32_t mark, T) {
  // Four bits to the tops of four bytes, each top to 16 bits.
  const uint32_t lo = ((mark & 15u) * 0x10204080u) & 0x80808080u;
  const uint32_t hi = (((mark >> 4) & 15u) * 0x10204080u) & 0x80808080u;
  uint32_t m[4];  // selector 8 + i: the sign of byte i, eight times
  asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m[0]) : "r"(lo));
  asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m[1]) : "r"(lo));
  asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m[2]) : "r"(hi));
  asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(m[3]) : "r"(hi));
  constexpr uint32_t low = Order<T>::kLow;
  q.x = (q.x & ~m[0]) | (low & m[0]);
  q.y = (q.y & ~m[1]) | (low & m[1]);
  q.z = (q.z & ~m[2]) | (low & m[2]);
  q.w = (q.w & ~m[3]) | (low & m[3]);
}

// Sum of 2^(x c + a) over a vector, as two partial sums.
template <typename T>
__device__ __forceinline__ f32x2 exponentials(const uint4& q, float c, float a) {
  constexpr int W = Vec<T>::W;
  float v[W];
  unpack(q, v, T());
  const f32x2 cc = f2_pack(c, c), aa = f2_pack(a, a);
  f32x2 sum = 0;  // two zeros
#pragma unroll
  for (int e = 0; e < W; e += 2) {
    float t0, t1;
    f2_unpack(f2_fma(f2_pack(v[e], v[e + 1]), cc, aa), t0, t1);
    const f32x2 two = f2_pack(exp2_approx(t0), exp2_approx(t1));
    sum = e == 0 ? two : f2_add(sum, two);
  }
  return sum;
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

template <int DT, typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* red, Op op) {  // result in every thread
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();  // `red` may still be read by an earlier reduction
  if (lane == 0) red[warp] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int i = 1; i < DT / 32; ++i) t = op(t, red[i]);
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

// Adds the warp's counts to a counter in shared memory with one atomic (they queue up on one address:
// 250 of them cost 10 000 cycles) and returns where this lane's share starts.
__device__ __forceinline__ int claim(int* counter, int mine) {
  const int lane = threadIdx.x & 31;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  int base = 0;
  if (lane == 31 && upto) base = atomicAdd(counter, upto);
  return __shfl_sync(0xffffffffu, base, 31) + upto - mine;
}

// The vectors v0 .. v1 - 1 of a row that belong to this CTA, on their way to shared memory. Vector j
// holds the elements j W - off .. j W - off + W - 1 (off: the row's place within 16 bytes).
template <typename T, int DT>
struct StagedRow {
  static constexpr int W = Vec<T>::W;
  int n, off, vectors, v0, v1;
  const uint4* row;  // [v1 - v0] in shared memory

  __device__ __forceinline__ StagedRow(const T* x, int n_, int part, int parts, uint4* smem, uint32_t bar)
      : n(n_), row(smem) {
    off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    vectors = (off + n + W - 1) / W;
    const int per = (vectors + parts - 1) / parts;
    v0 = min(part * per, vectors);
    v1 = min(v0 + per, vectors);
    const int b0 = v0 + (v0 == 0 && off > 0 ? 1 : 0);
    const int b1 = v1 - (v1 == vectors && (off + n) % W ? 1 : 0);
    const int tid = threadIdx.x;
    if (tid == 0) {
      mbar_init(bar, 1);
      fence_mbar_init();
      const uint32_t bytes = b1 > b0 ? static_cast<uint32_t>(b1 - b0) * 16u : 0u;
      mbar_expect_tx(bar, bytes);
      if (bytes)
        asm volatile(
            "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
            :
            : "r"(smem_u32(smem + (b0 - v0))), "l"(x - off + static_cast<long long>(b0) * W), "r"(bytes),
              "r"(bar)
            : "memory");
    }
    // Partial vectors at the row's ends (one vector may be both).
    const int e = tid % W;
    const int j = tid < W ? 0 : vectors - 1;
    if (tid < 2 * W && j >= v0 && j < v1 && (j < b0 || j >= b1)) {
      const int at = j * W + e - off;
      reinterpret_cast<T*>(smem + (j - v0))[e] =
          at >= 0 && at < n ? x[at] : from_float<T>(-INFINITY);
    }
  }
  __device__ __forceinline__ int elements() const {  // real elements of this part
    return v1 > v0 ? min(n, v1 * W - off) - max(0, v0 * W - off) : 0;
  }
  __device__ __forceinline__ int position(int i, int e) const { return (v0 + i) * W + e - off; }
  __device__ __forceinline__ bool holds(int position) const {
    return position >= 0 && position < n && position + off >= v0 * W && position + off < v1 * W;
  }
  __device__ __forceinline__ uint32_t bits(int position) const {
    using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, unsigned short>::type;
    return reinterpret_cast<const Bits*>(row)[position + off - v0 * W];
  }
  __device__ __forceinline__ T at(int position) const {
    return reinterpret_cast<const T*>(row)[position + off - v0 * W];
  }
};

// ------------------------------------------------------------------------------- top logits
constexpr int TOP_K_MAX = 256;
// Elements that are ranked without a bound: 512 rows of 100 with k = 50 take 8.9 us so and 14.4 with
// the bisection over elements, 512 rows of 1000 with k = 200 48 us and 22.
constexpr int RANK_ALL = 256;

// The k largest of the threads' maxima (found by bisection on their order keys) bound the
// k-th largest value from below, so everything not below that bound is a candidate: somewhat more
// than k of them for values in no particular order. Where there are too many (more kept than
// threads, rows of equal values) the bisection goes on over all values, and over positions among
// equal ones. The second pass over the row sums the exponentials relative to the bound and only
// lists the vectors that hold a candidate: with some 100 candidates in 2700 vectors nearly every
// warp would run through the code for them at every step. They are taken apart afterwards, one per
// thread, and ranked by counting the larger ones. Candidates that lose and a sum that underflows get
// anchors of their own, so that `rest` is right however far below the kept values it lies. Sums do not
// depend on the order in which threads run.
//
// Measured: 4096 rows of 21843 bf16, k = 64: 68 us (2.6 TB/s; two thirds of the issue slots are used: the
// instructions of all phases bound it, some 13 000 warp instructions per row). 24 rows of 131101, k = 200, 8 CTAs
// each: 20 us, all of it latency: copy, bounds, cluster joins, ranking of the kept. One row of 1000
// fp32: 5 us.
template <typename T, int DT>
__global__ void __launch_bounds__(DT)
top_logits_kernel(const T* __restrict__ logits, long long ld, int n, int k, float c, double inv_t,
                  int parts, int list_offset, T* __restrict__ values, int* __restrict__ indices,
                  float* __restrict__ rest) {
  constexpr int W = Vec<T>::W;
  constexpr int TOP_CAP = 2 * DT;  // candidates that shared memory holds
  using Ord = Order<T>;
  extern __shared__ __align__(16) uint4 row_smem[];
  __shared__ __align__(16) u64 cand[TOP_CAP];
  __shared__ __align__(16) u64 sorted[TOP_CAP];
  __shared__ __align__(16) uint32_t brief[TOP_CAP];
  __shared__ uint32_t red_u[DT / 32];
  __shared__ float red_f[DT / 32];
  __shared__ float2 part_rest[MAX_PARTS];
  __shared__ __align__(8) uint64_t bar_mem;
  __shared__ int count, hot_count, gave_up, too_wide;
  __shared__ uint2 red_range[DT / 32];
  __shared__ u64 part_bound[MAX_PARTS];
  __shared__ int list_length[MAX_PARTS];
  __shared__ u64 odd_sum;
  const int tid = threadIdx.x;
  const int part = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long r = blockIdx.x / parts;
  const T* x = logits + r * ld;
  const uint32_t bar = smem_u32(&bar_mem);
  const StagedRow<T, DT> st(x, n, part, parts, row_smem, bar);
  const int nv = st.v1 - st.v0;
  const int mine = min(k, st.elements());  // entries this part can contribute
  if (tid == 0) count = hot_count = gave_up = too_wide = 0, odd_sum = 0;
  __syncthreads();
  if (!mbar_wait(bar, 0, &gave_up, nullptr, 0)) gave_up = 1;

  uint32_t m0 = Ord::kLow, m1 = Ord::kLow;
  int i = tid;
  for (; i + DT < nv; i += 2 * DT) {
    m0 = Ord::largest(m0, st.row[i]);
    m1 = Ord::largest(m1, st.row[i + DT]);
  }
  if (i < nv) m0 = Ord::largest(m0, st.row[i]);
  const uint32_t best = tid < nv ? max(Ord::key_of_largest(m0), Ord::key_of_largest(m1)) : 0u;

  auto count_if = [&](auto test) {
    int got = 0;
    for (int j = tid; j < nv; j += DT) {
      const uint4 q = st.row[j];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int at = st.position(j, e);
        if (static_cast<unsigned>(at) < static_cast<unsigned>(n))
          got += test(Ord::key(bits_at<T>(q, e)), at) ? 1 : 0;
      }
    }
    return static_cast<int>(block_reduce<DT>(static_cast<uint32_t>(got), red_u, Sum()));
  };

  // Bound: at least `mine` elements have a key >= bound (0: all elements).
  uint32_t bound = 0;
  const int maxima = __syncthreads_count(best != 0);
  if (maxima < mine + mine / 2 && mine > 0) {
    // Too few maxima for a useful bound (they belong to single vectors): bisection over the elements, unless
    // ranking all of them costs less.
    if (st.elements() > RANK_ALL && st.elements() > mine + mine / 8 + 4) {
      uint32_t hi = block_reduce<DT>(best, red_u, Max());
      while (bound < hi) {
        const uint32_t mid = bound + (hi - bound) / 2 + 1;
        const int got = count_if([&](uint32_t key, int) { return key >= mid; });
        if (got >= mine) {
          bound = mid;
          if (got <= mine + mine / 8 + 4) break;
        } else {
          hi = mid - 1;
        }
      }
    }
  } else if (mine > 0) {
    uint32_t lo = __reduce_min_sync(0xffffffffu, best ? best : 0xffffffffu);
    uint32_t hi = __reduce_max_sync(0xffffffffu, best);
    if ((tid & 31) == 0) red_range[tid >> 5] = make_uint2(lo, hi);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < DT / 32; ++q) {
      lo = min(lo, red_range[q].x);
      hi = max(hi, red_range[q].y);
    }
    while (lo < hi) {  // count(>= lo) >= mine; the bound is <= hi
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      const int got = __syncthreads_count(best >= mid);
      if (got >= mine) {
        lo = mid;
        if (got <= mine + mine / 8 + 4) break;
      } else {
        hi = mid - 1;
      }
    }
    bound = lo;
  }

  int last_at = 0x7fffffff;  // elements equal to the bound count up to this position
  auto taken = [&](uint32_t key, int at) { return key > bound || (key == bound && at <= last_at); };
  float m = 0.0f, s = 0.0f;  // the sum of what is not kept, as sum of 2^((x - m) c)
  int* hot = reinterpret_cast<int*>(sorted);  // vectors that hold candidates
  for (int attempt = 0;; ++attempt) {
    // Everything not a candidate lies at or below the bound. A bound that cannot be an anchor
    // (infinite, NaN, a mask's value) leaves the sum to the code behind the ranking.
    m = bound ? Ord::value(bound) : -INFINITY;
    const bool near = fabsf(m) < FAR;
    const float anchor = near ? -m * c : 0.0f;
    f32x2 acc = 0;
    u64 odd = 0;  // what shares a vector with a candidate, in units of 2^-28
    // Candidates of the vector j (none if `has` is false); all lanes of a warp take part.
    auto take_apart = [&](bool has, int j) {
      uint32_t hits = 0;
      if (has && attempt == 0 && near) {
        // An ordinary bound: whatever is not below it is a candidate (padding is -inf).
        float v[W], below = 0.0f;
        unpack(st.row[j], v, T());
#pragma unroll
        for (int e = 0; e < W; ++e) {
          if (v[e] < m) below += exp2_approx(fmaf(v[e], c, anchor));
          else hits |= 1u << e;
        }
        odd += __float2uint_rn(below * 0x1p28f);
      } else if (has) {
        const uint4 q = st.row[j];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const uint32_t key = Ord::key(bits_at<T>(q, e));
          const int at = st.position(j, e);
          if (static_cast<unsigned>(at) >= static_cast<unsigned>(n)) continue;
          if (taken(key, at)) hits |= 1u << e;
          else if (near) odd += __float2uint_rn(exp2_approx(fmaf(Ord::value(key), c, anchor)) * 0x1p28f);
        }
      }
      int pos = claim(&count, __popc(hits));
      for (; hits && pos < TOP_CAP; hits &= hits - 1, ++pos) {
        const int at = st.position(j, __ffs(hits) - 1);
        const uint32_t key = Ord::key(st.bits(at));
        cand[pos] = (static_cast<u64>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(at));
        if (sizeof(T) == 2) {  // order in 32 bits, where key and position fit
          brief[pos] = ((key - bound) << 20) | (0xfffffu - static_cast<uint32_t>(at));
          if (key - bound >= 4096u) too_wide = 1;
        }
      }
    };
    if (attempt == 0) {
      u64 mine_hot = 0;  // bit i: vector tid + i DT (at most MAX_PART_BYTES / 16 / DT = 44 of them)
      int i = 0;
#pragma unroll 2
      for (int j = tid; j < nv; j += DT, ++i) {
        const uint4 q = st.row[j];
        const f32x2 sum = exponentials<T>(q, c, anchor);
        if (Ord::all_below(Ord::largest(Ord::kLow, q), m)) acc = f2_add(acc, sum);
        else mine_hot |= 1ull << i;
      }
      int pos = claim(&hot_count, __popcll(mine_hot));
      for (; mine_hot && pos < TOP_CAP; mine_hot &= mine_hot - 1, ++pos)
        hot[pos] = tid + (__ffsll(mine_hot) - 1) * DT;
    } else {  // exact bounds: any number of vectors may hold values equal to the bound
      for (int j0 = 0; j0 < nv; j0 += DT) {
        const int j = j0 + tid;
        const uint4 q = j < nv ? st.row[j] : make_uint4(0, 0, 0, 0);
        const bool below = j < nv && Ord::all_below(Ord::largest(Ord::kLow, q), m);
        if (below) acc = f2_add(acc, exponentials<T>(q, c, anchor));
        take_apart(j < nv && !below, j);
      }
    }
    __syncthreads();
    if (hot_count <= TOP_CAP) {
      for (int h0 = 0; h0 < hot_count; h0 += DT) {
        const int h = h0 + tid;
        const bool has = h < hot_count;
        if (!__any_sync(0xffffffffu, has)) break;  // whole warps only
        take_apart(has, has ? hot[h] : 0);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) odd += __shfl_xor_sync(0xffffffffu, odd, o);
    if (odd && (tid & 31) == 0) atomicAdd(&odd_sum, odd);  // integers: the order does not matter
    float s0, s1;
    f2_unpack(acc, s0, s1);
    s = near ? s0 + s1 : 0.0f;
    __syncthreads();
    if ((hot_count <= TOP_CAP && count <= TOP_CAP) || attempt == 1) break;
    uint32_t lo = bound, hi = sizeof(T) == 4 ? 0xffffffffu : 0xffffu;
    int got = TOP_CAP + 1;
    while (lo < hi && got > TOP_CAP) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      const int above = count_if([&](uint32_t key, int) { return key >= mid; });
      if (above >= mine) {
        lo = mid;
        got = above;
      } else {
        hi = mid - 1;
      }
    }
    bound = lo;
    if (got > TOP_CAP) {  // too many elements equal to the k-th largest: the first ones of them
      const int need = mine - count_if([&](uint32_t key, int) { return key > lo; });
      int a0 = 0, a1 = n - 1;
      while (a0 < a1) {
        const int mid = a0 + (a1 - a0) / 2;
        if (count_if([&](uint32_t key, int at) { return key == lo && at <= mid; }) >= need) a1 = mid;
        else a0 = mid + 1;
      }
      last_at = a0;
    }
    __syncthreads();
    if (tid == 0) count = hot_count = 0, odd_sum = 0;
    __syncthreads();
  }
  const int found = min(count, TOP_CAP);  // >= mine

  // Rank of every candidate = number of larger ones (all are different: the position is part). Four
  // threads count for one candidate.
  if (tid < 8 && found + tid < TOP_CAP) cand[found + tid] = brief[found + tid] = 0;  // read in blocks
  __syncthreads();
  auto rank_all = [&](auto* list, auto count_larger) {
    for (int q0 = 0; q0 < found; q0 += DT / 4) {
      const int q = q0 + (tid >> 2);
      if (q0 + ((tid & ~31) >> 2) >= found) break;  // whole warps
      int rank = count_larger(list[q < found ? q : 0]);
      rank += __shfl_xor_sync(0xffffffffu, rank, 1);
      rank += __shfl_xor_sync(0xffffffffu, rank, 2);
      if (q < found && (tid & 3) == 0) sorted[rank] = cand[q];
    }
  };
  if (sizeof(T) == 2 && !too_wide && n <= (1 << 20)) {
    rank_all(brief, [&](uint32_t me) {
      int rank = 0;
      const uint4* four = reinterpret_cast<const uint4*>(brief);
#pragma unroll 2
      for (int j = tid & 3; j < (found + 3) / 4; j += 4) {
        const uint4 v = four[j];
        rank += (v.x > me ? 1 : 0) + (v.y > me ? 1 : 0) + (v.z > me ? 1 : 0) + (v.w > me ? 1 : 0);
      }
      return rank;
    });
  } else {
    rank_all(cand, [&](u64 me) {
      int rank = 0;
      const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(cand);
#pragma unroll 2
      for (int j = tid & 3; j < (found + 1) / 2; j += 4) {
        const ulonglong2 two = pairs[j];
        rank += (two.x > me ? 1 : 0) + (two.y > me ? 1 : 0);
      }
      return rank;
    });
  }
  s = block_reduce<DT>(s, red_f, Sum());  // its barriers also publish sorted[]
  if (fabsf(m) < FAR) {  // the factor takes the rounding of m c back
    s += static_cast<float>(odd_sum) * 0x1p-28f;
    // (A bound that is no element may be so large that this rounding passes fp32's range; no element
    // below it leaves anything then, and 0 times infinity must not come of it.)
    if (s != 0.0f) s *= exp2_approx(-fmaf(m, c, -m * c));
  }
  // Adds values (each thread's own, through `each`) whose largest key is `key` to the sum; none of
  // them lies below what is in the sum already.
  auto add_at = [&](uint32_t key, auto each) {
    const float top_value = Ord::value(key);
    if (!(top_value < INFINITY)) {  // +inf or NaN: so is the sum
      m = 0.0f;
      s = top_value;
      return;
    }
    float t = 0.0f;
    if (top_value > -INFINITY) {
      each([&](float v) { t += exp2_approx((v - top_value) * c); });
      t = block_reduce<DT>(t, red_f, Sum());
      s = (s > 0.0f ? s * exp2_approx((m - top_value) * c) : s) + t;
      m = top_value;
    }
  };
  if (found > mine) {
    // The losing candidates are at or above the bound: the first of them is the new anchor. They are
    // few: the first warp adds them up (only thread 0 needs the sum).
    const float top_value = Ord::value(static_cast<uint32_t>(sorted[mine] >> 32));
    if (!(top_value < INFINITY)) {
      m = 0.0f;
      s = top_value;
    } else if (tid < 32 && top_value > -INFINITY) {
      float t = 0.0f;
      for (int q = mine + tid; q < found; q += 32)
        t += exp2_approx((Ord::value(static_cast<uint32_t>(sorted[q] >> 32)) - top_value) * c);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      s = (s > 0.0f ? s * exp2_approx((m - top_value) * c) : s) + t;
      m = top_value;
    }
  } else if (s < 0.125f) {
    // Nothing, or all of it below the bound by so much that the units of odd_sum and, further down,
    // fp32 itself would show: anchor at the largest of it.
    auto walk = [&](auto visit) {
      for (int j = tid; j < nv; j += DT) {
        const uint4 q = st.row[j];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const uint32_t key = Ord::key(bits_at<T>(q, e));
          const int at = st.position(j, e);
          if (static_cast<unsigned>(at) < static_cast<unsigned>(n) && !taken(key, at)) visit(key);
        }
      }
    };
    uint32_t low = 0;
    walk([&](uint32_t key) { low = max(low, key); });
    low = block_reduce<DT>(low, red_u, Max());
    s = 0.0f;
    if (low)
      add_at(low, [&](auto add) { walk([&](uint32_t key) { add(Ord::value(key)); }); });
  }

  auto emit = [&](int rank, u64 entry) {
    const int at = static_cast<int>(0xffffffffu - static_cast<uint32_t>(entry));
    if (!st.holds(at)) return;  // cannot be; keeps a wrong entry from reading elsewhere
    indices[r * k + rank] = at;
    values[r * k + rank] = st.at(at);
  };
  auto log_of = [&](float top_value, float sum) {
    return sum == 0.0f ? -INFINITY
                       : static_cast<float>(top_value * inv_t + log(static_cast<double>(sum)));
  };
  if (parts == 1) {
    for (int q = tid; q < mine; q += DT) emit(q, sorted[q]);
    if (tid == 0) rest[r] = gave_up ? NAN : log_of(m, s);
    return;
  }

  // The parts' sorted lists meet. Every part has ceil(k / parts) entries that are not below the least of
  // the parts' entries at that place, so nothing below it can be among the k largest of the row: little
  // more than k entries are left. An entry's place in the row is its place here plus the number of
  // larger entries in the other lists.
  const int place = (k + parts - 1) / parts - 1;
  if (tid < parts) {
    const u64 v = place < mine ? sorted[place] : 0;
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(
                     mapa_shared(smem_u32(part_bound + part), static_cast<uint32_t>(tid))),
                 "l"(v)
                 : "memory");
  }
  for (int q = mine + tid; q < k; q += DT) sorted[q] = 0;
  cluster_sync_all();
  u64 floor_entry = part_bound[0];
  for (int p = 1; p < parts; ++p) floor_entry = min(floor_entry, part_bound[p]);
  u64* lists = reinterpret_cast<u64*>(row_smem) + list_offset;  // [parts][k] behind the row
  for (int p = tid >> 5; p < parts; p += DT / 32) {
    const uint32_t src = mapa_shared(smem_u32(sorted), static_cast<uint32_t>(p));
    int length = 0;
    for (int q0 = 0; q0 < k; q0 += 32) {
      const int q = q0 + (tid & 31);
      u64 v = 0;
      if (q < k) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(src + 8u * q));
      const bool in = v != 0 && v >= floor_entry;
      if (in) lists[p * k + q] = v;
      const uint32_t mask = __ballot_sync(0xffffffffu, in);
      length += __popc(mask);
      if (mask != 0xffffffffu) break;
    }
    if ((tid & 31) == 0) list_length[p] = length;
  }
  __syncthreads();
  uint32_t out_key = 0;
  if (tid < mine) {  // k <= 256 <= DT
    const u64 me = sorted[tid];
    int rank = k;
    if (me >= floor_entry) {
      // In every list the first position whose entry is not larger, all lists in step.
      int at[MAX_PARTS] = {};
#pragma unroll 1
      for (int step = 256; step > 0; step >>= 1) {
#pragma unroll
        for (int p = 0; p < MAX_PARTS; ++p)
          if (p < parts && at[p] + step <= list_length[p] && lists[p * k + at[p] + step - 1] > me)
            at[p] += step;
      }
      rank = 0;  // this CTA's own list counts its place
#pragma unroll
      for (int p = 0; p < MAX_PARTS; ++p) rank += at[p];
    }
    if (rank < k) emit(rank, me);
    else out_key = static_cast<uint32_t>(me >> 32);
  }
  const uint32_t high = block_reduce<DT>(out_key, red_u, Max());
  if (high)
    add_at(high, [&](auto add) {
      if (out_key) add(Ord::value(out_key));
    });
  if (tid == 0) {
    const uint32_t dst = mapa_shared(smem_u32(part_rest + part), 0);
    const float sum = gave_up ? NAN : s;
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(m), "f"(sum) : "memory");
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

constexpr int ST = 128;            // threads of the forward kernels
constexpr int FT = 256;            // threads of the backward kernel
constexpr int ENTRIES = 256;       // kept classes whose logits stay in shared memory (at most)
constexpr int MAX_SUM_PARTS = 32;  // parts of a row in the sums kernel

struct DistillParams {
  const void* values;
  const void* indices;
  const float* rest;  // NULL: the kept classes are the teacher's whole distribution
  float* loss;
  float2* stats;      // per row: anchor and factor of the classes that are not kept
  float* slopes;      // per kept class: student's minus teacher's probability
  long long ld, ld_values, ld_indices;
  float4* partials;   // per row and part: maximum, anchor, sum, whether a class is listed twice
  long long rows;
  int n, k, values_dtype, indices_wide, parts;
  float c;            // log2(e) / temperature
  double temperature;
};

// Running sum of exponentials with the largest x so far as anchor: s * 2^-a = sum of 2^(x c) with
// a = -m c rounded to fp32, or s = sum of 2^((x - m) c) where m lies beyond FAR_SUM: rounding -m c there
// could be off by more than the exponents that fp32 holds (c is at most 1443: off by 64 within).
constexpr float FAR_SUM = 1e6f;
struct Running {
  float m, a, s;
  __device__ __forceinline__ bool far() const { return !(fabsf(m) < FAR_SUM); }
  // What a sum relative to (m0, a0) is worth relative to this anchor.
  __device__ __forceinline__ float worth(float m0, float a0, float s0, float c) const {
    if (s0 == 0.0f) return 0.0f;
    return s0 * exp2_approx(far() || !(fabsf(m0) < FAR_SUM) ? (m0 - m) * c : a - a0);
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

// Sum of the student's exponentials over the classes that are NOT kept, per row and part: one pass
// over the logits with a running maximum per thread. A bitmap in shared memory marks the kept classes
// (one byte test per 8 bf16 elements). Nothing else is done here, so that ten small CTAs per SM,
// each with its own loads in flight, keep HBM busy (4096 rows of 21843 bf16, with the backward pass:
// 111 us with 10 CTAs of 8 vectors per thread, 114 with 12 of 4, 116 with 8 of 8); the finish kernel is launched at once and works
// on the kept classes until these sums are there.
template <typename T>
__global__ void __launch_bounds__(ST, 10)
distill_sums_kernel(const T* __restrict__ logits, const DistillParams p) {
  constexpr int W = Vec<T>::W;
  using Ord = Order<T>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint32_t bitmap[];
  __shared__ float4 red_run[ST / 32];
  __shared__ int repeated;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long r = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const int n = p.n, k = p.k;
  const T* x = logits + r * p.ld;
  const RowLayout<T> lay(x, n);
  const int per = (lay.vectors + p.parts - 1) / p.parts;
  const int v0 = min(part * per, lay.vectors), v1 = min(v0 + per, lay.vectors);
  const uint4* xv = reinterpret_cast<const uint4*>(x + lay.head);
  // Eight vectors per thread and step; -inf past the end in the last, partial step.
  constexpr int U = 8;
  uint4 raw[U];
  const int mine = v1 - v0 - tid;  // vectors from this thread's first one on
  const int full = (v1 - v0) / (U * ST);
  const uint4* next = xv + v0 + tid;
  auto fetch = [&](int step) {
    if (step < full) {
#pragma unroll
      for (int i = 0; i < U; ++i) raw[i] = __ldg(next + i * ST);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i)
        raw[i] = (step * U + i) * ST < mine ? __ldg(next + i * ST) : low_vector<T>();
    }
    next += U * ST;
  };
  fetch(0);
  // Bit of element e: the part's vectors from bit W on, the row's ends in front of and behind them.
  const int first = lay.head + v0 * W - W;
  const int last = part == p.parts - 1 ? n : lay.head + v1 * W;
  for (int i = tid; i < (last - first + 31) / 32; i += ST) bitmap[i] = 0;
  if (tid == 0) repeated = 0;
  __syncthreads();
  for (int i = tid; i < k; i += ST) {
    const int at = load_index(p.indices, p.indices_wide, r * p.ld_indices + i, n);
    if (at >= (part == 0 ? 0 : first + W) && at < last) {
      const int b = at - first;
      if (atomicOr(&bitmap[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) repeated = 1;
    }
  }
  __syncthreads();

  const float c = p.c;
  Running run = {-INFINITY, INFINITY, 0.0f};
  float limit = NAN;  // the maximum so far while it is an ordinary number: nothing is <= NaN
  f32x2 acc = 0;
  // Marks of this thread's vectors: a byte each, or half a byte with four elements to a vector.
  const uint8_t* mark_at = reinterpret_cast<const uint8_t*>(bitmap) + (W == 8 ? tid + 1 : (tid + 1) >> 1);
  const int mark_shift = W == 8 ? 0 : ((tid + 1) & 1) * 4;
  for (int step = 0; step * U * ST < mine; ++step) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (step >= full && (step * U + i) * ST >= mine) break;
      const uint32_t mark = (mark_at[i * ST * W / 8] >> mark_shift) & ((1u << W) - 1u);
      if (mark) mask_vector(raw[i], mark, T());
    }
    mark_at += U * ST * W / 8;
    uint32_t most = Ord::largest(Ord::kLow, raw[0]);
#pragma unroll
    for (int i = 1; i < U; ++i) most = Ord::largest(most, raw[i]);
    const float top = Ord::value_of_largest(most);
    if (!(top <= limit)) {  // NaN too
      float s0, s1;
      f2_unpack(acc, s0, s1);
      run.s += s0 + s1;
      acc = 0;
      run.raise(top, c);
      limit = run.far() ? NAN : run.m;
    }
    if (!run.far()) {
#pragma unroll
      for (int i = 0; i < U; ++i) acc = f2_add(acc, exponentials<T>(raw[i], c, run.a));
    } else if (run.m > -INFINITY || top != -INFINITY) {  // infinities, NaN, masks' values
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float v[W];
        unpack(raw[i], v, T());
#pragma unroll
        for (int e = 0; e < W; ++e) run.s += exp2_approx((v[e] - run.m) * c);
      }
    }
    fetch(step + 1);
  }
  float s0, s1;
  f2_unpack(acc, s0, s1);
  run.s += s0 + s1;
  const int edges = (part == 0 ? lay.head : 0) + (part == p.parts - 1 ? lay.tail : 0);
  if (tid < edges) {
    const int at = part == 0 && tid < lay.head ? tid : n - lay.tail + (tid - (part == 0 ? lay.head : 0));
    const int b = at - first;
    const float v = bitmap[b >> 5] >> (b & 31) & 1 ? -INFINITY : to_float(x[at]);
    run.raise(v, c);
    if (!(v == -INFINITY)) run.s += run.of(v, c);
  }
  const float m = Order<float>::value(__reduce_max_sync(0xffffffffu, Order<float>::key(__float_as_uint(run.m))));
  if (m > run.m) run.raise(m, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) run.s += __shfl_xor_sync(0xffffffffu, run.s, o);
  if (lane == 0) red_run[warp] = make_float4(run.m, run.a, run.s, 0.0f);
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < ST / 32; ++i) run.join(red_run[i].x, red_run[i].y, red_run[i].z, c);
    p.partials[blockIdx.x] = make_float4(run.m, run.a, run.s, __int_as_float(repeated));
  }
}

// One warp per row evaluates the at most k + 1 terms of the divergence in 64 bits, where the parts
// that cancel between a student and a teacher that agree do no harm, nor in the gradient's q - p: all
// but the student's normaliser before the sums over the other classes are waited for. stats and slopes
// leave nothing but one exponential per class to the backward pass. The first kept classes (`room` of
// them, ENTRIES at most) stay in shared memory: beside the sums kernel's stream every dependent load
// takes 2 to 3 us (37 rows of 131101 with 100 kept classes, loss and gradient: 33 us with 64 of
// them there, 30 with all).
template <typename T>
__global__ void __launch_bounds__(ST)
distill_finish_kernel(const T* __restrict__ logits, const DistillParams p) {
  constexpr int ROWS = ST / 32;
  extern __shared__ double entry_smem[];
  const int room = min(p.k, ENTRIES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long r = static_cast<long long>(blockIdx.x) * ROWS + warp;
  if (r >= p.rows) return;
  const int n = p.n, k = p.k;
  const T* x = logits + r * p.ld;
  double *ent_t = entry_smem + warp * 4 * room, *ent_z = ent_t + room, *ent_et = ent_z + room, *ent_ez = ent_et + room;
  int* ent_at = reinterpret_cast<int*>(entry_smem + ROWS * 4 * room) + warp * room;
  const float c = p.c;
  const double inv_t = 1.0 / p.temperature;
  auto load_entry = [&](int i, double& t, double& z) {
    const int at = load_index(p.indices, p.indices_wide, r * p.ld_indices + i, n);
    t = z = -INFINITY;
    if (at >= 0) {
      t = load_value(p.values, p.values_dtype, r * p.ld_values + i) * inv_t;
      z = to_float(x[at]) * inv_t;
    }
    return at;
  };
  for (int i = lane; i < room; i += 32) {
    double t, z;
    ent_at[i] = load_entry(i, t, z);
    ent_t[i] = t;
    ent_z[i] = z;
  }
  __syncwarp();
  auto class_at = [&](int i) {
    return i < room ? ent_at[i] : load_index(p.indices, p.indices_wide, r * p.ld_indices + i, n);
  };
  auto warp_max = [](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Max()(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  auto warp_sum = [](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  // Natural-log units in 64 bits, maxima and sums kept apart (a maximum of the size of a mask's value
  // would swallow the logarithm of its sum).
  const double tr = p.rest ? static_cast<double>(p.rest[r]) : -INFINITY;
  double t_max, z_max, t_sum, z_sum, t_inv, t_log, fixed_loss, mass;
  bool silent, repeated = false;
  auto part_of = [](double v, double top_value) { return v == -INFINITY ? 0.0 : exp(v - top_value); };
  auto entry = [&](int i, double& t, double& z) {  // teacher's and student's logit; false: left out
    const int at = class_at(i);
    if (at < 0) return false;
    if (repeated)  // the first entry of a class counts
      for (int j = 0; j < i; ++j)
        if (class_at(j) == at) return false;
    if (i < room) {
      t = ent_t[i];
      z = ent_z[i];
    } else {
      load_entry(i, t, z);
    }
    return true;
  };
  auto work_on_entries = [&]() {
    t_max = tr, z_max = -INFINITY;
    for (int i = lane; i < k; i += 32) {
      double t, z;
      if (!entry(i, t, z)) continue;
      t_max = Max()(t, t_max);
      z_max = Max()(z, z_max);
    }
    t_max = warp_max(t_max);
    z_max = warp_max(z_max);
    t_sum = z_sum = 0.0;
    for (int i = lane; i < k; i += 32) {
      double t, z;
      if (!entry(i, t, z)) continue;
      const double et = part_of(t, t_max), ez = part_of(z, z_max);
      t_sum += et;
      z_sum += ez;
      if (i < room) {
        ent_et[i] = et;
        ent_ez[i] = ez;
      }
    }
    t_sum = warp_sum(t_sum) + part_of(tr, t_max);
    z_sum = warp_sum(z_sum);
    silent = t_max == -INFINITY;  // a teacher without any mass (no entry, no rest) teaches nothing
    t_inv = silent ? 0.0 : 1.0 / t_sum;
    t_log = log(t_sum);
    // sum p (log p - (z - z_max)): the loss up to the student's normaliser, which every outcome shares.
    fixed_loss = mass = 0.0;
    for (int i = lane; i < k; i += 32) {
      double t, z;
      if (!entry(i, t, z)) continue;
      const double pt = (i < room ? ent_et[i] : part_of(t, t_max)) * t_inv;
      if (pt == 0.0) continue;
      fixed_loss += pt * ((t - t_max - t_log) - (z == -INFINITY ? z : z - z_max));
      mass += pt;
    }
    fixed_loss = warp_sum(fixed_loss);
    mass = warp_sum(mass);
  };
  work_on_entries();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Running run = {-INFINITY, INFINITY, 0.0f};
  int again = 0;
  if (lane < p.parts) {
    const float4 f = p.partials[r * p.parts + lane];
    run = {f.x, f.y, f.z};
    again = __float_as_int(f.w);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, run.m, o);
    const float a = __shfl_xor_sync(0xffffffffu, run.a, o);
    const float s = __shfl_xor_sync(0xffffffffu, run.s, o);
    // Both lanes of a pair add the lower lane's value first: all lanes end with the same bits.
    if (lane & o) {
      Running low = {m, a, s};
      low.join(run.m, run.a, run.s, c);
      run = low;
    } else {
      run.join(m, a, s, c);
    }
  }
  repeated = __any_sync(0xffffffffu, again);
  if (repeated) work_on_entries();  // without the entries of classes listed before
  // The classes not kept: zs * e^zm; fmaf(m, c, a) is what rounding the anchor to fp32 left over.
  const bool some = run.s != 0.0f;
  const double zm = some ? run.m * inv_t : -INFINITY;
  const double zs = run.far() ? run.s : run.s * exp2(-static_cast<double>(fmaf(run.m, c, run.a)));
  // The student's normaliser relative to z_max, through whichever maximum is larger.
  const double top = Max()(zm, z_max);
  const double e_zm = part_of(zm, top) * zs, e_zk = part_of(z_max, top);
  const double total = z_sum * e_zk + e_zm, log_total = log(total);
  const double z_log = top - z_max + log_total;  // only used with kept classes of finite logits
  const double z_inv = e_zk / total;
  for (int i = lane; i < k; i += 32) {
    double t, z;
    float slope = 0.0f;
    if (entry(i, t, z) && !silent) {
      const double et = i < room ? ent_et[i] : part_of(t, t_max);
      const double ez = i < room ? ent_ez[i] : part_of(z, z_max);
      slope = static_cast<float>((ez == 0.0 ? 0.0 : ez * z_inv) - et * t_inv);
    }
    p.slopes[r * k + i] = slope;
  }
  if (lane == 0) {
    double loss = mass > 0.0 || mass != mass ? fixed_loss + mass * (z_max == -INFINITY ? 0.0 : z_log) : 0.0;
    const double p_rest = tr == -INFINITY ? 0.0 : part_of(tr, t_max) * t_inv;
    const double q_rest = silent || !some ? 0.0 : e_zm / total;
    if (p_rest != 0.0)
      loss += p_rest * ((tr - t_max - t_log) - (some ? zm - top + log(zs) - log_total : -INFINITY));
    p.loss[r] = static_cast<float>(loss * p.temperature * p.temperature);
    // Gradient of a class that is not kept: q_j (1 - p_rest / q_rest).
    p.stats[r] = make_float2(run.m, some ? static_cast<float>((q_rest - p_rest) / run.s) : 0.0f);
  }
}

// d loss / d logits * d_loss: 2^((x - anchor) c) * factor for the classes that are not kept, the
// saved slope for the others. One read and one write of the row (4096 rows of 21843 bf16: 59 us, 6.0 TB/s);
// a row whose d_loss is zero (padding) is zeroed without being read. Columns n .. n_pad (row padding of the gradient) get zeros.
template <typename T>
__global__ void __launch_bounds__(FT)
distill_bwd_kernel(const T* __restrict__ logits, const void* __restrict__ indices, int indices_wide,
                   long long ld_indices, const float2* __restrict__ stats,
                   const float* __restrict__ slopes, const float* __restrict__ d_loss,
                   long long d_loss_stride, T* __restrict__ grad, long long ld, long long ld_grad,
                   int n, int n_pad, int k, int parts, float c, float temperature) {
  constexpr int DT = FT;
  constexpr int W = Vec<T>::W;
  const int tid = threadIdx.x;
  // The last rows first: the forward pass read them last, and L2 may still hold some of them.
  const long long r = (gridDim.x - 1 - blockIdx.x) / parts;
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
int launch_clusters(void (*kernel)(Params...), int64_t rows, int parts, int threads, size_t smem,
                    cudaStream_t stream, Args... args) {
  if (smem > 24 * 1024) {  // may pass the default limit together with the static part
    const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               MAX_PART_BYTES + MAX_PARTS * 256 * 8);
    if (e != cudaSuccess) {
      set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
      cudaGetLastError();
      return -4;
    }
  }
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(parts);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
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

// Two CTAs per SM. (24 rows of 131101: 20 us with 8 CTAs for each row; 1 row of 1000 stays with one.)
constexpr int kTargetCtas = 296;

// CTAs per row: enough to give every SM two, as long as each keeps `least` vectors.
int choose_parts(int64_t rows, int vectors, int least, int64_t target = kTargetCtas, int most = MAX_PARTS) {
  int parts = 1;
  while (parts < most && rows * parts < target && vectors / (2 * parts) >= least) parts *= 2;
  return parts;
}

constexpr int64_t MAX_ROWS = 1 << 27;

// CTAs per row of the staged kernels and the shared memory of each (bytes of its vectors; a row may
// start anywhere within 16 bytes, which adds a vector).
int staged_parts(int64_t rows, int64_t n, int itemsize, int least, size_t* bytes) {
  const int64_t vectors = (n * itemsize + 15) / 16 + 1;
  int parts = choose_parts(rows, static_cast<int>(vectors), least);
  while (parts < MAX_PARTS && (vectors + parts - 1) / parts * 16 > MAX_PART_BYTES) parts *= 2;
  *bytes = static_cast<size_t>((vectors + parts - 1) / parts * 16);
  return parts;
}

template <typename T>
int top_logits(const void* logits, int64_t rows, int64_t n, int64_t ld, int64_t k, double temperature,
               void* values, int32_t* indices, float* rest, cudaStream_t stream) {
  size_t smem = 0;  // at first of the row's part alone
  const int parts = staged_parts(rows, n, sizeof(T), 256, &smem);
  // 512 threads, where 256 maxima are too few to bound the k-th largest value with and the row has more
  // vectors than that: 4096 rows of 21843 bf16 take 141 us against 943 with k = 200, but 98 against 77
  // with k = 100; 512 rows of 1000 with k = 200 35 against 22.
  const int threads = k + k / 2 > 256 && smem / 16 > 256 ? 512 : 256;
  const int list_offset = static_cast<int>(smem / 8);
  if (parts > 1) smem += static_cast<size_t>(parts * k * 8);
  const float c = static_cast<float>(1.4426950408889634 / temperature);
  const double inv_t = 1.0 / temperature;
  auto kernel = threads == 512 ? top_logits_kernel<T, 512> : top_logits_kernel<T, 256>;
  return launch_clusters(kernel, rows, parts, threads, smem, stream, static_cast<const T*>(logits),
                         static_cast<long long>(ld), static_cast<int>(n), static_cast<int>(k), c, inv_t,
                         parts, list_offset, static_cast<T*>(values), indices, rest);
}

}  // namespace
}  // namespace vmoe

using namespace vmoe;

extern "C" int64_t vmoe_top_logits_max_classes(int32_t dtype) {
  return static_cast<int64_t>(MAX_PARTS) * MAX_PART_BYTES / (dtype == 0 ? 4 : 2) - 64;
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

extern "C" int64_t vmoe_distill_max_classes(int32_t dtype) { return 1 << 20; }

// Eight small CTAs per SM, as long as each keeps two vectors per thread; and no more than 128 K classes
// (16 KB of bitmap) per part.
static int distill_parts(int64_t rows, int64_t n, int32_t dtype) {
  int parts = choose_parts(rows, static_cast<int>(n / (dtype == 0 ? 4 : 8)), 2 * ST, 4 * kTargetCtas,
                           MAX_SUM_PARTS);
  while (parts < MAX_SUM_PARTS && n / parts > (1 << 17)) parts *= 2;
  return parts;
}

extern "C" int64_t vmoe_distill_kept_floats(int64_t rows, int64_t n, int64_t k, int32_t dtype) {
  return (rows * (k + 2) + 3) / 4 * 4 + rows * 4 * distill_parts(rows, n, dtype);
}

// The finish kernel's CTAs can only join the sums' on an SM whose shared memory is set up with room for
// them; sums alone would get little of it, and the finish kernel would wait for SMs to drain (37 rows of
// 131101, loss and gradient: 30 us so, 20 us with a quarter set aside). More takes the L1 through which
// the sums' loads pass: 4096 rows of 21843 take 111 us with a quarter, 117 with half, 129 with all.
template <typename T>
static int share_out() {
  static std::atomic<unsigned long long> done{0};  // a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && (done.load() & bit)) return 0;
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(distill_sums_kernel<T>),
                             cudaFuncAttributePreferredSharedMemoryCarveout, 25);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(distill_finish_kernel<T>),
                             cudaFuncAttributePreferredSharedMemoryCarveout,
                             cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) {
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    cudaGetLastError();
    return -4;
  }
  done.fetch_or(bit);
  return 0;
}

template <typename T>
static int distill_fwd(const VmoeDistillArgs* a, const DistillParams& p, cudaStream_t stream) {
  const T* logits = static_cast<const T*>(a->logits);
  constexpr int W = Vec<T>::W;
  const size_t smem = ((a->n / W + p.parts - 1) / p.parts + 4) * W / 8 + 8;
  int rc = share_out<T>();
  if (rc) return rc;
  distill_sums_kernel<T><<<static_cast<unsigned>(a->rows * p.parts), ST, smem, stream>>>(logits, p);
  if ((rc = check_launch())) return rc;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cudaLaunchAttribute attr;
  memset(&attr, 0, sizeof(attr));
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>((a->rows + ST / 32 - 1) / (ST / 32)));
  cfg.blockDim = dim3(ST);
  cfg.dynamicSmemBytes = (ST / 32) * (a->k < ENTRIES ? a->k : ENTRIES) * (4 * sizeof(double) + sizeof(int));
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_finish_kernel<T>, logits, p);
  if (e != cudaSuccess) {
    set_error("%s (code %d)", cudaGetErrorString(e), static_cast<int>(e));
    cudaGetLastError();
    return -5;
  }
  return 0;
}

extern "C" int vmoe_distill_fwd(const VmoeDistillArgs* a, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows == 0) return 0;
  if (a->rows < 0 || a->rows > MAX_ROWS / MAX_SUM_PARTS || a->n < 1 ||
      a->n > vmoe_distill_max_classes(a->dtype) || a->k < 1 || a->k > (1 << 20))
    return bad("distill: rows, classes or kept classes out of range");
  if (!(a->temperature > 0.0)) return bad("distill: temperature must be positive");
  if (reinterpret_cast<uintptr_t>(a->kept) & 15) return bad("distill: kept must be 16-byte aligned");
  DistillParams p;
  p.values = a->values;
  p.indices = a->indices;
  p.rest = a->rest;
  p.loss = a->loss;
  p.stats = reinterpret_cast<float2*>(a->kept);
  p.slopes = a->kept + 2 * a->rows;
  p.partials = reinterpret_cast<float4*>(a->kept + (a->rows * (a->k + 2) + 3) / 4 * 4);
  p.rows = a->rows;
  p.ld = a->ld;
  p.ld_values = a->ld_values;
  p.ld_indices = a->ld_indices;
  p.n = static_cast<int>(a->n);
  p.k = static_cast<int>(a->k);
  p.values_dtype = a->values_dtype;
  p.indices_wide = a->indices_wide;
  p.c = static_cast<float>(1.4426950408889634 / a->temperature);
  p.temperature = a->temperature;
  p.parts = distill_parts(a->rows, a->n, a->dtype);
  switch (a->dtype) {
    case 0: return distill_fwd<float>(a, p, stream);
    case 1: return distill_fwd<__nv_bfloat16>(a, p, stream);
    case 2: return distill_fwd<__half>(a, p, stream);
  }
  return bad("distill: unknown dtype");
}

extern "C" int vmoe_distill_bwd(const VmoeDistillArgs* a, const float* d_loss, int64_t d_loss_stride,
                                void* grad, int64_t ld_grad, int64_t n_pad, vmoe_stream_t stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->rows == 0) return 0;
  if (a->rows < 0 || a->rows > MAX_ROWS || a->n < 1 || a->n > vmoe_distill_max_classes(a->dtype) ||
      n_pad < a->n || n_pad > ld_grad)
    return bad("distill: rows or classes out of range");
  const int itemsize = a->dtype == 0 ? 4 : 2;
  // Gradient rows are written in the logits' vectors: both must start at the same offset
  // within 16 bytes, row by row.
  if ((reinterpret_cast<uintptr_t>(a->logits) - reinterpret_cast<uintptr_t>(grad)) % 16 ||
      ((a->ld - ld_grad) * itemsize) % 16)
    return bad("distill: gradient rows must have the alignment of the logits' rows");
  const int parts = choose_parts(a->rows, static_cast<int>(a->n / (16 / itemsize)), FT);
  const unsigned grid = static_cast<unsigned>(a->rows * parts);
  const float c = static_cast<float>(1.4426950408889634 / a->temperature);
#define VMOE_DISTILL_BWD(T)                                                                         \
  distill_bwd_kernel<T><<<grid, FT, 0, stream>>>(                                                   \
      static_cast<const T*>(a->logits), a->indices, a->indices_wide, a->ld_indices,                 \
      reinterpret_cast<const float2*>(a->kept), a->kept + 2 * a->rows, d_loss, d_loss_stride,                  \
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
