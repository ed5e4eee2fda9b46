// Products with 4-bit weights and one scale and bias per group of columns:
//   y[m, n] = sum_k x[m, k] w[n, k],  w[n, k] = scale[n, k / G] q[n, k] + bias[n, k / G]
// with q in 0 .. 15. Per group, with a = q - 8 and X = sum of the group's x,
//   y += scale * (sum a x + 8 X) + bias * X,
// so the weights are exact small integers in the matrix product and the
// scales multiply float32 sums: no weight is rounded.
//
// For a few rows of x the product is bound by the weight stream (k / 2 bytes
// per output) and, next to it, by the instructions that unpack the weights. A
// warp takes 16 output rows as the M side of m16n8k16 (fp16), the rows of x
// are its eight columns; weights go from global memory through a private
// cp.async ring to registers. fp16 has ten mantissa bits, so two nibbles of a
// 16-bit half become numbers without a shift: w & 0x000f000f | 0x64006400 is
// the pair 1024 + q, w & 0x00f000f0 | 0x64006400 the pair 1024 + 16 q (exact).
//   float32 results: one more instruction each makes them q - 8 (exact).
//   bf16 results: they stay, the odd columns of x are divided by 16, and the
//   sums 1024 X_even + 64 X_odd are taken off in float32. That loses seven bits
//   of float32, nothing in a bf16 result: 5 instructions per 8 weights, not 9.
// x is brought to fp16 by a power of two per row and group that puts the
// group's largest |x| into [2^14, 2^15): bf16 x keeps all its bits (smaller
// ones down to 2^-31 of the largest), float32 x becomes two columns, x = hi + lo
// with 22 bits. The factor multiplies the group's float32 sum. A kernel of its
// own does that once; every CTA doing it for itself took as many instructions
// as the product. The product's weights are on their way meanwhile (programmatic
// dependent launch).
//
// The k index of a product is arbitrary as long as both operands agree: lane
// (g, c) unpacks whole words of 8 columns from its own rows, in the pairs
// (0, 4), (1, 5), (2, 6), (3, 7), and x lies in shared memory in the order in
// which the lanes ask for it.
#include <cuda_fp16.h>

#include "cache_ops.cuh"
#include "cache_tile.cuh"
#include "q4.cuh"

namespace mrtdf {
namespace {

constexpr int kMaxWarps = 16;
constexpr int kStep = 128;  // columns multiplied at a time: 64 bytes of 16 rows
constexpr int kStepBytes = 16 * kStep / 2;
// A ring stage has two steps, so that a row gives 128 bytes at a time: in 64-byte
// pieces 67 MB came in 13 us, in 128-byte pieces in 11 (from L2, no products).
constexpr int kStageBytes = 2 * kStepBytes;
constexpr int kRing = 4;  // stages per warp
constexpr int kSmemMax = 224 * 1024;

// Byte offset of 16-byte chunk `ch` (0 .. 3) of row `row` of a step. Rows are
// 64 bytes apart; the swizzle puts the eight rows of one access in different
// banks.
__device__ __forceinline__ uint32_t w_at(int row, int ch) {
  return (uint32_t)(row * (kStep / 2) + ((ch ^ (row >> 1 & 3)) << 4));
}

// Words of a step that lane c multiplies for its group `gi`, from row address
// `row` (of a step, without the chunk) whose swizzle is x: WL = G / 32 words,
// columns gi * G + (c * WL + i) * 8.
template <int WL>
__device__ __forceinline__ void load_words(uint32_t* w, uint32_t row, uint32_t x, int c, int gi) {
  if constexpr (WL == 1) {
    w[0] = lds32(row + ((gi << 4) ^ x) + 4 * c);
  } else if constexpr (WL == 2) {
    const uint32_t a = row + (((2 * gi + (c >> 1)) << 4) ^ x) + 8 * (c & 1);
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    const uint32_t a = row + ((c << 4) ^ x);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(a));
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// The column pairs (0, 4), (1, 5) of w, or with w >> 8 (2, 6), (3, 7): q - 8
// (EIGHT), or 1024 + q and 1024 + 16 q.
template <bool EIGHT>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t& even, uint32_t& odd) {
  // (w & mask) | magic in one instruction each
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(even) : "r"(w), "n"(0x000f000f), "r"(0x64006400u));
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(odd) : "r"(w), "n"(0x00f000f0), "r"(0x64006400u));
  if (EIGHT) {
    const __half2 e = __hadd2(*reinterpret_cast<const __half2*>(&even), __float2half2_rn(-1032.f));
    const __half2 o = __hfma2(*reinterpret_cast<const __half2*>(&odd), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
    even = *reinterpret_cast<const uint32_t*>(&e);
    odd = *reinterpret_cast<const uint32_t*>(&o);
  }
}

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c = a b: the first product of a sum, on zeros that take no registers.
__device__ __forceinline__ void mma_f16_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A scale and its bias, side by side in shared memory.
__device__ __forceinline__ void load_pair(uint32_t at, float& s, float& b, __nv_bfloat16) {
  const uint32_t w = lds32(at);
  s = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void load_pair(uint32_t at, float& s, float& b, float) {
  uint32_t x, y;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(at));
  s = __uint_as_float(x);
  b = __uint_as_float(y);
}

template <typename T>
struct Parts;  // fp16 columns per row of x
template <>
struct Parts<__nv_bfloat16> {
  static constexpr int N = 1;
};
template <>
struct Parts<float> {
  static constexpr int N = 2;
};

// How a product is laid out over the GPU.
struct Q4Plan {
  int split;  // CTAs of a cluster: each has a slab of the columns
  int tiles;  // row tiles of 16 per cluster (and so per CTA)
  int warps;  // warps with tiles of their own, taking every warps-th
  int wk;     // warps per tile: each takes every wk-th stage of the slab
  int slab;   // steps of 128 columns per CTA
  int chunk;  // of them, those whose x is in shared memory at a time
  int part;   // of a chunk, the steps that one barrier stands for
  int rows;   // rows of x per pass (grid y)
  int steps;  // all steps
};
constexpr int kParts = 4;  // barriers of a chunk

// Shared memory of a CTA, in order: rings, x, factors of x, scales, partial
// sums, barriers.
template <typename T, int G, int NT>
struct Q4Smem {
  static constexpr int COLS = NT * 8;
  int x_bytes, x, factors, scales, part, bars, bytes;
  __host__ __device__ explicit Q4Smem(const Q4Plan& q) {
    x_bytes = q.chunk * kStep * 2 + 64;
    x = q.warps * q.wk * kRing * kStageBytes;
    factors = x + COLS * x_bytes;
    scales = factors + (q.chunk * kStep / G) * COLS * 16;
    part = scales + (q.chunk * kStep / G) * q.tiles * 16 * 2 * (int)sizeof(T);
    const int units = q.tiles > q.warps * q.wk ? q.tiles : q.warps * q.wk;
    bars = (part + units * 16 * (COLS + 1) * 4 + 7) / 8 * 8;
    bytes = bars + kParts * 8;
  }
};

// The prepared x of one pass: [COLS][steps * 128] fp16, then
// [group][COLS] {factor of the group's sum, what is added to it, X, 0}.
template <int G, int NT>
struct Q4Prepared {
  static constexpr int COLS = NT * 8;
  static __host__ __device__ int64_t x_bytes(int steps) { return (int64_t)COLS * steps * kStep * 2; }
  static __host__ __device__ int64_t bytes(int steps) { return x_bytes(steps) + (int64_t)steps * (kStep / G) * COLS * 16; }
};

__device__ __forceinline__ float ld_cluster_f32(const float* local, uint32_t rank) {
  uint32_t ra;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra) : "memory");
  return v;
}

// x to fp16: 8 columns from kk on (one word of weights) per lane, a group by
// 4 WL neighbouring lanes, all lanes of a warp together. put(h, words) gets the
// lane's eight values of part h, sums(h, {factor, addend, X, 0}) the group's.
// Rows that do not exist (m < 0) and columns past k are zero.
template <typename T, int G, bool EIGHT, typename Put, typename Sums>
__device__ __forceinline__ void bring_x(const Q4Params& p, int m, int kk, Put&& put, Sums&& sums) {
  constexpr int WL = G / 32, P = Parts<T>::N, V = 8 * (int)sizeof(T) / 16;
  float v[8], big = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (m >= 0 && kk < p.k) {
    const T* src = reinterpret_cast<const T*>(p.x) + m * p.x_stride + kk;
#pragma unroll
    for (int e = 0; e < V; ++e) Vec16<T>::unpack(*reinterpret_cast<const uint4*>(src + e * (8 / V)), v + e * (8 / V));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(v[e]));
#pragma unroll
  for (int o = 1; o < 4 * WL; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  const uint32_t ex = max(__float_as_uint(big) >> 23, 15u);
  const float up = __uint_as_float((268u - ex) << 23), down = __uint_as_float((ex - 14u) << 23);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= up;
#pragma unroll
  for (int h = 0; h < P; ++h) {
    uint32_t w[4];
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = pack_f16(v[e], v[e + 4]);
      const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      f[e] = t2.x;
      f[e + 4] = t2.y;
    }
    float even = (f[0] + f[4]) + (f[2] + f[6]), odd = (f[1] + f[5]) + (f[3] + f[7]);
#pragma unroll
    for (int o = 1; o < 4 * WL; o <<= 1) {
      even += __shfl_xor_sync(0xffffffffu, even, o);
      odd += __shfl_xor_sync(0xffffffffu, odd, o);
    }
    if (!EIGHT) {
      w[1] = pack_f16(f[1] * 0.0625f, f[5] * 0.0625f);
      w[3] = pack_f16(f[3] * 0.0625f, f[7] * 0.0625f);
    }
    put(h, make_uint4(w[0], w[1], w[2], w[3]));
    const float sum = down * (even + odd);
    sums(h, make_float4(down, EIGHT ? 8.f * sum : -down * (1024.f * even + 64.f * odd), sum, 0.f));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] -= f[e];
  }
}
// Where word wd of a row lies: words of one group and index i next to each
// other for c = 0 .. 3.
template <int WL>
__device__ __forceinline__ int word_at(int wd) {
  const int in = wd % (4 * WL);
  return wd - in + (in % WL) * 4 + in / WL;
}

template <typename T, int G, int NT, bool EIGHT>
__global__ __launch_bounds__(128) void q4_prepare_kernel(const __grid_constant__ Q4Params p, int steps, int rows) {
  constexpr int WL = G / 32, P = Parts<T>::N, COLS = NT * 8;
  pdl_launch_dependents();
  const int words = steps * (kStep / 8), lane = threadIdx.x & 31, m0 = blockIdx.y * rows, all = words * (COLS / P);
  uint8_t* out = static_cast<uint8_t*>(p.ws) + blockIdx.y * Q4Prepared<G, NT>::bytes(steps);
  float4* factor = reinterpret_cast<float4*>(out + Q4Prepared<G, NT>::x_bytes(steps));
  const int i = blockIdx.x * 128 + threadIdx.x;
  if (i - lane >= all) return;
  const int m = i / words, wd = i - m * words;
  bring_x<T, G, EIGHT>(
      p, i < all && m < rows && m0 + m < p.m ? m0 + m : -1, wd * 8,
      [&](int h, uint4 w) {
        if (i < all) *reinterpret_cast<uint4*>(out + ((int64_t)(m * P + h) * words + word_at<WL>(wd)) * 16) = w;
      },
      [&](int h, float4 f) {
        if (i < all && wd % (4 * WL) == 0) factor[wd / (4 * WL) * COLS + m * P + h] = f;
      });
}

// T: type of x, scales and biases. NT: tiles of eight columns (rows of x x
// parts). A cluster works on q.tiles row tiles, its CTAs on a slab of the
// columns each (a CTA reads half of x that way); the slabs' sums meet over
// distributed shared memory, in rank order. FUSED: x is small and every CTA
// brings its slab to fp16 itself (2 x 1024: 7 us, 10 with a launch for it).
template <typename T, typename O, int G, int NT, bool FUSED>
__global__ __launch_bounds__(kMaxWarps * 32, 1) void q4_linear_kernel(const __grid_constant__ Q4Params p,
                                                                                     const __grid_constant__ Q4Plan q) {
  constexpr int WL = G / 32, GS = kStep / G, P = Parts<T>::N, COLS = NT * 8, LD = COLS + 1;
  constexpr bool EIGHT = sizeof(O) == 4;
  extern __shared__ __align__(128) uint8_t smem[];
  const Q4Smem<T, G, NT> at(q);
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int wt = warp % q.warps, wk = warp / q.warps, g = lane >> 2, c = lane & 3;
  const int rank = q.split > 1 ? (int)cluster_ctarank() : 0, cluster = blockIdx.x / q.split;
  const int m0 = blockIdx.y * q.rows, ms = min(q.rows, p.m - m0);
  const int tile0 = cluster * q.tiles, tiles = min(q.tiles, (p.n + 15) / 16 - tile0), stride = q.tiles * 16;
  const int groups = p.k / G, row_bytes = p.k / 2, n0 = tile0 * 16;
  const int slab0 = rank * q.slab, slab_end = min(slab0 + q.slab, q.steps);
  T* sb = reinterpret_cast<T*>(smem + at.scales);  // [group][row], scale and bias side by side
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + at.bars);
  const uint8_t* prepared = static_cast<const uint8_t*>(p.ws) + blockIdx.y * Q4Prepared<G, NT>::bytes(q.steps);
  float* part = reinterpret_cast<float*>(smem + at.part);  // [wk][row][COLS + 1]

  const uint32_t ring = smem_u32(smem) + warp * (kRing * kStageBytes);
  const int fr = lane >> 3, fc = lane & 7;  // a lane copies chunk fc of rows fr, fr + 4, ...
  const int units_max = q.tiles > q.warps * q.wk ? q.tiles : q.warps * q.wk;
  for (int i = tid; i < units_max * 16 * LD; i += threads) part[i] = 0.f;

  if (!FUSED && tid == 0) {
    for (int i = 0; i < kParts; ++i) mbar_init(bars + i, 1);
    fence_mbar_init();
  }

  for (int step0 = slab0, round = 0; step0 < slab_end; step0 += q.chunk, ++round) {
  const int steps = min(q.chunk, slab_end - step0), k0 = step0 * kStep;
  // This warp's units: its tiles, and of each its stages. Rows past n and
  // columns past k read a valid address instead: the former are not written,
  // the latter meet zeros of x.
  const int my_stages = max(0, ((steps + 1) / 2 - wk + q.wk - 1) / q.wk), my_tiles = max(0, (tiles - wt + q.warps - 1) / q.warps);
  const int units = my_stages * my_tiles;
  const int first_col = (k0 + wk * 2 * kStep) / 2 + fc * 16, last_col = row_bytes - 16, col_step = q.wk * kStep;
  int f_unit = 0, f_step = 0, f_tile = wt, f_col = first_col;  // the unit to fetch next
  uint32_t f_stage = ring + (fc >> 2) * kStepBytes;
  const uint8_t* from[4];
  auto enter = [&] {
    const int row = n0 + f_tile * 16 + fr;
#pragma unroll
    for (int i = 0; i < 4; ++i) from[i] = p.packed + (int64_t)min(row + 4 * i, p.n - 1) * row_bytes;
  };
  enter();
  auto fetch = [&] {
    const int col = min(f_col, last_col);
#pragma unroll
    for (int i = 0; i < 4; ++i) cp_async16(f_stage + w_at(fr + 4 * i, fc & 3), from[i] + col);
    f_stage += kStageBytes;
    f_col += col_step;
    if ((++f_unit & (kRing - 1)) == 0) f_stage -= kRing * kStageBytes;
    if (++f_step == my_stages) {
      f_step = 0;
      f_col = first_col;
      f_tile += q.warps;
      enter();
    }
  };
#pragma unroll
  for (int t = 0; t < kRing - 1; ++t) {
    if (f_unit < units) fetch();
    cp_async_commit();
  }

  if (round) __syncthreads();  // the chunk before is done with
  const int gn = steps * GS, g0 = k0 / G;
  if (!FUSED && round == 0) pdl_wait();  // x is prepared
  if (!FUSED && tid == 0) {
    // The chunk before was read through the generic proxy.
    if (round) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    const uint32_t factor_bytes = gn * COLS * 16;
    for (int i = 0; i < kParts; ++i) {
      const int first = i * q.part, n = min(q.part, steps - first);
      if (n <= 0) break;
      mbar_arrive_expect_tx(bars + i, COLS * n * kStep * 2 + (i == 0 ? factor_bytes : 0));
      if (i == 0)
        bulk_g2s(smem + at.factors, prepared + Q4Prepared<G, NT>::x_bytes(q.steps) + (int64_t)g0 * COLS * 16, factor_bytes, bars);
      for (int col = 0; col < COLS; ++col)
        bulk_g2s(smem + at.x + col * at.x_bytes + first * kStep * 2,
                 prepared + ((int64_t)col * q.steps + step0 + first) * (kStep * 2), n * kStep * 2, bars + i);
    }
  }
  // Scales and biases of the chunk's groups, side by side: 16 bytes at a time
  // where rows and groups allow it.
  constexpr int E = 16 / (int)sizeof(T);
  if (groups % E == 0 && g0 % E == 0) {
    const int vecs = (gn + E - 1) / E, all = tiles * 16 * vecs;
    for (int i0 = tid; i0 < all; i0 += 4 * threads) {
      uint4 s[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * threads, all - 1), r = i / vecs;
        const int64_t from = (int64_t)min(n0 + r, p.n - 1) * groups + min(g0 + (i - r * vecs) * E, groups - E);
        s[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.scales) + from);
        b[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.biases) + from);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * threads, all - 1), r = i / vecs, first = (i - r * vecs) * E;
        const T *sv = reinterpret_cast<const T*>(&s[u]), *bv = reinterpret_cast<const T*>(&b[u]);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first + e < gn) {
            sb[((first + e) * stride + r) * 2] = sv[e];
            sb[((first + e) * stride + r) * 2 + 1] = bv[e];
          }
      }
    }
  } else {
    for (int i = tid; i < gn * tiles * 16; i += threads) {
      const int r = i / gn, gr = i - r * gn;
      const int64_t from = (int64_t)min(n0 + r, p.n - 1) * groups + min(g0 + gr, groups - 1);
      sb[(gr * stride + r) * 2] = reinterpret_cast<const T*>(p.scales)[from];
      sb[(gr * stride + r) * 2 + 1] = reinterpret_cast<const T*>(p.biases)[from];
    }
  }
  if (FUSED) {
    const int words = steps * (kStep / 8), all = words * q.rows, spare = COLS - q.rows * P;
    float4* factor = reinterpret_cast<float4*>(smem + at.factors);
    for (int i0 = tid; i0 - lane < all; i0 += threads) {
      const int m = i0 / words, wd = i0 - m * words;
      bring_x<T, G, EIGHT>(
          p, i0 < all && m < ms ? m0 + m : -1, k0 + wd * 8,
          [&](int h, uint4 w) {
            if (i0 < all) *reinterpret_cast<uint4*>(smem + at.x + (m * P + h) * at.x_bytes + word_at<WL>(wd) * 16) = w;
          },
          [&](int h, float4 f) {
            if (i0 < all && wd % (4 * WL) == 0) factor[wd / (4 * WL) * COLS + m * P + h] = f;
          });
    }
    for (int i = tid; i < words * spare; i += threads)  // columns without a row of x
      *reinterpret_cast<uint4*>(smem + at.x + (COLS - spare + i / words) * at.x_bytes + (i % words) * 16) = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < gn * spare; i += threads)
      factor[i / spare * COLS + COLS - spare + i % spare] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();  // the scales are there, and the barriers (or x)

  float y[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0.f;
  // Shared addresses of this lane's operands in the unit's step.
  const uint32_t swz = (uint32_t)(g >> 1 & 3) << 4;  // of rows g and g + 8
  const uint32_t x_first = smem_u32(smem + at.x) + g * at.x_bytes + c * 16 + wk * 2 * GS * (WL * 64);
  const uint32_t f_first = smem_u32(smem + at.factors) + (wk * 2 * GS * COLS + 2 * c) * 16;
  const uint32_t s_first = smem_u32(sb) + (wk * 2 * GS * stride + wt * 16 + g) * 2 * (int)sizeof(T);
  const uint32_t x_step = GS * (WL * 64), fa_step = GS * COLS * 16, skip = 2 * q.wk - 2, s_group = stride * 2 * (int)sizeof(T);
  uint32_t xa = x_first, fa = f_first, sa = s_first, row = ring + g * (kStep / 2), st = 0;
  int tile = wt, step = 0, parts = 0;  // parts of x that have arrived
  for (int t = 0; t < units; ++t) {
    while (!FUSED && parts * q.part <= min((step * q.wk + wk) * 2 + 1, steps - 1)) mbar_wait_bounded(bars + parts++, round & 1, nullptr);
    cp_async_wait<kRing - 2>();
    __syncwarp();
    if (f_unit < units) fetch();
    cp_async_commit();
    const bool odd_end = (step * q.wk + wk) * 2 + 1 >= steps;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
    if (sub && odd_end) break;
#pragma unroll
    for (int gi = 0; gi < GS; ++gi) {
      uint32_t w0[WL], w1[WL];
      load_words<WL>(w0, row + st + sub * kStepBytes, swz, c, gi);
      load_words<WL>(w1, row + st + sub * kStepBytes + 8 * (kStep / 2), swz, c, gi);
      float s0, s1, b0, b1;
      load_pair(sa + gi * s_group, s0, b0, T());
      load_pair(sa + gi * s_group + 16 * (int)sizeof(T), s1, b1, T());
      float acc[NT][4], acd[NT][4];
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        uint32_t a0[4], a1[4];
        unpack<EIGHT>(w0[i], a0[0], a0[2]);
        unpack<EIGHT>(w1[i], a0[1], a0[3]);
        unpack<EIGHT>(w0[i] >> 8, a1[0], a1[2]);
        unpack<EIGHT>(w1[i] >> 8, a1[1], a1[3]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 b = lds128(xa + j * 8 * at.x_bytes + gi * (WL * 64) + i * 64);
          if (i == 0) {
            mma_f16_first(acc[j], a0, b.x, b.y);
            mma_f16_first(acd[j], a1, b.z, b.w);
          } else {
            mma_f16(acc[j], a0, b.x, b.y);
            mma_f16(acd[j], a1, b.z, b.w);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint4 u = lds128(fa + (gi * COLS + j * 8) * 16), v = lds128(fa + (gi * COLS + j * 8) * 16 + 16);
        const float fu = __uint_as_float(u.x), ou = __uint_as_float(u.y), xu = __uint_as_float(u.z);
        const float fv = __uint_as_float(v.x), ov = __uint_as_float(v.y), xv = __uint_as_float(v.z);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] += acd[j][e];
        y[j][0] = fmaf(s0, fmaf(fu, acc[j][0], ou), fmaf(b0, xu, y[j][0]));
        y[j][1] = fmaf(s0, fmaf(fv, acc[j][1], ov), fmaf(b0, xv, y[j][1]));
        y[j][2] = fmaf(s1, fmaf(fu, acc[j][2], ou), fmaf(b1, xu, y[j][2]));
        y[j][3] = fmaf(s1, fmaf(fv, acc[j][3], ov), fmaf(b1, xv, y[j][3]));
      }
    }
    xa += x_step;
    fa += fa_step;
    sa += GS * s_group;
    }
    st = (st + kStageBytes) & (kRing * kStageBytes - 1);
    xa += skip * x_step;
    fa += skip * fa_step;
    sa += skip * GS * s_group;
    if (++step == my_stages) {  // the tile is done
      float* to = part + ((wk * q.warps + tile) * 16 + g) * LD + 2 * c;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          to[8 * (e >> 1) * LD + j * 8 + (e & 1)] += y[j][e];
          y[j][e] = 0.f;
        }
      step = 0;
      tile += q.warps;
      xa = x_first;
      fa = f_first;
      sa = s_first + (tile - wt) * 32 * (int)sizeof(T);
    }
  }
  cp_async_wait<0>();
  // No copy is still landing when the chunk is left (or the CTA).
  while (!FUSED && parts < kParts && parts * q.part < steps) mbar_wait_bounded(bars + parts++, round & 1, nullptr);
  }

  // Sums of the warps that share tiles (then each has one), of the slabs and
  // of the parts, in a fixed order.
  if (q.wk > 1) {
    __syncthreads();
    for (int i = tid; i < tiles * 16 * COLS; i += threads) {
      const int cell = i / COLS * LD + i % COLS;
      float sum = part[cell];
      for (int w = 1; w < q.wk; ++w) sum += part[w * q.warps * 16 * LD + cell];
      part[cell] = sum;
    }
  }
  if (q.split > 1) cluster_sync();
  else __syncthreads();
  for (int i = rank * threads + tid; i < ms * tiles * 16; i += q.split * threads) {
    const int m = i / (tiles * 16), r = i - m * (tiles * 16), n = n0 + r;
    if (n >= p.n) continue;
    float sum = 0.f;
    for (int o = 0; o < q.split; ++o)
#pragma unroll
      for (int h = 0; h < P; ++h) {
        const float* from = part + r * LD + m * P + h;
        sum += q.split > 1 ? ld_cluster_f32(from, o) : *from;
      }
    reinterpret_cast<O*>(p.out)[(m0 + m) * p.out_stride + n] = from_f<O>(sum);
  }
  if (q.split > 1) cluster_sync();  // nobody leaves while its sums are read
}

// One warp per group: scale = (max - min) / 15 and bias = min, both rounded to
// T, q = round((w - bias) / scale) in 0 .. 15 with the rounded two. A group
// whose values are all equal has scale 0 and q = 0.
template <typename T>
__global__ __launch_bounds__(256) void q4_quantize_kernel(const __grid_constant__ Q4PackParams p) {
  const int lane = threadIdx.x & 31, groups = p.k / p.group, pairs = p.group / 2;
  const int64_t all = (int64_t)p.n * groups;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += (int64_t)gridDim.x * 8) {
    const int64_t n = i / groups;
    const int gr = (int)(i - n * groups);
    const T* w = reinterpret_cast<const T*>(p.w) + n * p.w_stride + (int64_t)gr * p.group;
    float v[2][2], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane + 32 * h < pairs) {
        v[h][0] = to_f(w[2 * (lane + 32 * h)]);
        v[h][1] = to_f(w[2 * (lane + 32 * h) + 1]);
        lo = fminf(lo, fminf(v[h][0], v[h][1]));
        hi = fmaxf(hi, fmaxf(v[h][0], v[h][1]));
      }
    hi = warp_max(hi);
    lo = -warp_max(-lo);
    const float scale = rnd<T>(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), bias = rnd<T>(lo);
    auto code = [&](float x) {
      const float q = scale > 0.f ? rintf(__fdiv_rn(__fsub_rn(x, bias), scale)) : 0.f;
      return (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane + 32 * h < pairs)
        p.packed[n * (p.k / 2) + (int64_t)gr * pairs + lane + 32 * h] = (uint8_t)(code(v[h][0]) | code(v[h][1]) << 4);
    if (lane == 0) {
      reinterpret_cast<T*>(p.scales)[i] = from_f<T>(scale);
      reinterpret_cast<T*>(p.biases)[i] = from_f<T>(bias);
    }
  }
}

// The layout on a GPU of `sms` multiprocessors: one CTA per SM, row tiles spread
// evenly over pairs of CTAs (1025 tiles are 74 pairs of 14), a slab of the
// columns for each of a pair where there are 16 steps or more; fewer tiles
// or columns at a time where the shared memory asks for it.
template <typename T, int G, int NT>
Q4Plan q4_plan(const Q4Params& p, int sms) {
  const int tiles = (p.n + 15) / 16;
  Q4Plan q{};
  q.steps = (p.k + kStep - 1) / kStep;
  q.rows = min(p.m, NT * 8 / Parts<T>::N);
  q.split = q.steps >= 16 ? 2 : 1;
  q.slab = (q.steps + q.split - 1) / q.split;
  q.chunk = q.slab;
  const int clusters = max(1, sms / q.split);
  q.tiles = (tiles + clusters - 1) / clusters;
  for (;;) {
    const int per_warp = (q.tiles + kMaxWarps - 1) / kMaxWarps;
    q.warps = (q.tiles + per_warp - 1) / per_warp;
    q.wk = max(1, min(kMaxWarps / q.warps, (q.chunk + 1) / 2));
    q.part = (q.chunk + kParts - 1) / kParts;
    const Q4Smem<T, G, NT> at(q);
    if (at.bytes <= kSmemMax || (q.tiles == 1 && q.chunk == 1)) return q;
    if (q.tiles == 1 || (q.chunk > 1 && at.scales - at.x > kSmemMax / 2)) q.chunk = (q.chunk + 1) / 2;
    else q.tiles = (q.tiles + 1) / 2;
  }
}

template <typename T, typename O, int G, int NT, bool FUSED>
cudaError_t q4_launch(const Q4Params& p, const Q4Plan& q, int passes, cudaStream_t s) {
  constexpr auto K = q4_linear_kernel<T, O, G, NT, FUSED>;
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (!FUSED) {
    const int words = q.steps * (kStep / 8) * (NT * 8 / Parts<T>::N);
    q4_prepare_kernel<T, G, NT, sizeof(O) == 4><<<dim3((words + 127) / 128, passes), 128, 0, s>>>(p, q.steps, q.rows);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (q.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = q.split;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(((p.n + 15) / 16 + q.tiles - 1) / q.tiles * q.split, passes);
  cfg.blockDim = dim3(q.warps * q.wk * 32);
  cfg.dynamicSmemBytes = Q4Smem<T, G, NT>(q).bytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, K, p, q);
}

template <typename T, typename O, int G, int NT>
cudaError_t q4_run(const Q4Params& p, int sms, size_t* ws_bytes, cudaStream_t s) {
  const Q4Plan q = q4_plan<T, G, NT>(p, sms);
  const int passes = (p.m + q.rows - 1) / q.rows;
  // Words of x per CTA: up to two per thread it takes them itself.
  const bool fused = q.slab * (kStep / 8) * q.rows <= 1024;
  if (ws_bytes) {
    *ws_bytes = fused ? 0 : (size_t)passes * Q4Prepared<G, NT>::bytes(q.steps);
    return cudaSuccess;
  }
  return fused ? q4_launch<T, O, G, NT, true>(p, q, passes, s) : q4_launch<T, O, G, NT, false>(p, q, passes, s);
}

template <typename T, typename O, int G>
cudaError_t q4_tiles(const Q4Params& p, int sms, size_t* ws, cudaStream_t s) {
  const int cols = p.m * Parts<T>::N;
  if (cols <= 8) return q4_run<T, O, G, 1>(p, sms, ws, s);
  if (cols <= 16) return q4_run<T, O, G, 2>(p, sms, ws, s);
  return q4_run<T, O, G, 4>(p, sms, ws, s);
}

template <typename T, typename O>
cudaError_t q4_group(const Q4Params& p, int sms, size_t* ws, cudaStream_t s) {
  if (p.group == 32) return q4_tiles<T, O, 32>(p, sms, ws, s);
  if (p.group == 64) return q4_tiles<T, O, 64>(p, sms, ws, s);
  return q4_tiles<T, O, 128>(p, sms, ws, s);
}

}  // namespace

cudaError_t launch_q4_linear(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s) {
  if (dtype == 0) return q4_group<float, float>(p, sms, ws_bytes, s);
  return out_dtype == 0 ? q4_group<__nv_bfloat16, float>(p, sms, ws_bytes, s)
                        : q4_group<__nv_bfloat16, __nv_bfloat16>(p, sms, ws_bytes, s);
}

cudaError_t launch_q4_quantize(const Q4PackParams& p, int dtype, cudaStream_t s) {
  const int64_t all = (int64_t)p.n * (p.k / p.group), want = (all + 7) / 8;
  const unsigned grid = (unsigned)(want < 148 * 32 ? want : 148 * 32);
  if (dtype == 0) q4_quantize_kernel<float><<<grid, 256, 0, s>>>(p);
  else q4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mrtdf
