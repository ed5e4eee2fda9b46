// Products with 4-bit weights and one scale and bias per group of columns:
//   y[m, n] = sum_k x[m, k] w[n, k],  w[n, k] = scale[n, k / G] q[n, k] + bias[n, k / G]
// with q in 0 .. 15. Per group, with a = q - 8 and X = sum of the group's x,
//   y += scale * (sum a x) + (bias + 8 scale) * X,
// so the weights are exact small integers in the matrix product and the
// scales multiply float32 sums: no weight is rounded. The offset 8 keeps the
// two terms from cancelling where bias is near -8 scale.
//
// For a few rows of x the product is bound by the weight stream (k / 2 bytes
// per output). A warp takes 16 output rows as the M side of m16n8k16, the rows
// of x are its eight columns; weights go from global memory through a private
// cp.async ring to registers and are unpacked there: (w >> s) & 0x000f000f |
// 0x43004300 is the bf16 pair 128 + q (exact), minus 136 is q - 8 (exact).
// float32 rows of x are split into three bf16 columns, x = x1 + x2 + x3 with
// all 24 bits, which the same product multiplies exactly.
//
// The k index of a product is arbitrary as long as both operands agree: lane
// (g, c) unpacks whole words of 8 columns from its own rows, and x lies in
// shared memory in the order in which the lanes ask for it.
#include "cache_ops.cuh"
#include "cache_tile.cuh"
#include "q4.cuh"

namespace mrtdf {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 128;  // columns of a ring stage: 64 bytes of 16 rows
constexpr int kRing = 5;    // stages per warp
constexpr int kStageBytes = 16 * kStep / 2;
constexpr int kChunkElems = 32 * 1024;  // x values (bf16) in shared memory at a time

// Byte offset of 16-byte chunk `ch` (0 .. 3) of row `row` of a stage. Rows are
// 64 bytes apart; the swizzle puts the eight rows of one access in different
// banks.
__device__ __forceinline__ uint32_t w_at(int row, int ch) {
  return (uint32_t)(row * (kStep / 2) + ((ch ^ (row >> 1 & 3)) << 4));
}

// Words of a stage that lane (row, c) multiplies for group-in-stage `gi`:
// WL = G / 32 words, columns gi * G + (c * WL + i) * 8.
template <int WL>
__device__ __forceinline__ void load_words(uint32_t* w, uint32_t stage, int row, int c, int gi) {
  if constexpr (WL == 1) {
    w[0] = lds32(stage + w_at(row, gi) + 4 * c);
  } else if constexpr (WL == 2) {
    const uint32_t a = stage + w_at(row, 2 * gi + (c >> 1)) + 8 * (c & 1);
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    const uint32_t a = stage + w_at(row, c);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(a));
  }
}

// Nibbles s / 4 and s / 4 + 4 of w, minus 8, as a bf16 pair.
template <int SHIFT>
__device__ __forceinline__ uint32_t nibbles(uint32_t w) {
  uint32_t v = (w >> SHIFT) & 0x000f000fu | 0x43004300u;
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));  // 136
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
struct Parts;  // bf16 columns per row of x
template <>
struct Parts<__nv_bfloat16> {
  static constexpr int N = 1;
};
template <>
struct Parts<float> {
  static constexpr int N = 3;
};

// T: type of x, scales and biases. NT: tiles of eight columns (rows of x x
// parts). WR: warps with rows of their own; the other kWarps / WR split k.
template <typename T, typename O, int G, int NT, int WR>
__global__ __launch_bounds__(kThreads) void q4_linear_kernel(const __grid_constant__ Q4Params p, int rows_per_pass,
                                                              int chunk) {
  constexpr int WL = G / 32, GS = kStep / G, WK = kWarps / WR, P = Parts<T>::N, COLS = NT * 8;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wr = warp % WR, wk = warp / WR;
  const int g = lane >> 2, c = lane & 3;
  const int m0 = blockIdx.y * rows_per_pass, ms = min(rows_per_pass, p.m - m0);
  const int row0 = (blockIdx.x * WR + wr) * 16, groups = p.k / G;
  const uint32_t ring = smem_u32(smem) + warp * (kRing * kStageBytes);
  // x: column i at i * x_stride bytes; 64 bytes past a multiple of 128, so two
  // columns of one access lie in different banks. Group sums behind it.
  const int x_bytes = chunk * 2 + 64;
  uint8_t* xs = smem + kWarps * kRing * kStageBytes;
  float* sums = reinterpret_cast<float*>(xs + COLS * x_bytes);  // [group of the chunk][COLS]

  const int steps = (p.k + kStep - 1) / kStep;
  // Stage t of this warp: columns (t * WK + wk) * 128.
  const int mine = (steps - wk + WK - 1) / WK;
  auto fetch = [&](int t) {
    const int k0 = (t * WK + wk) * kStep;
    const uint32_t st = ring + (t % kRing) * kStageBytes;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int idx = lane + 32 * i, row = idx >> 2, ch = idx & 3, n = row0 + row, kb = k0 / 2 + ch * 16;
      const bool on = n < p.n && kb < p.k / 2;
      cp_async16_zfill(st + w_at(row, ch), p.packed + (on ? (int64_t)n * (p.k / 2) + kb : 0), on);
    }
  };
#pragma unroll
  for (int t = 0; t < kRing - 1; ++t) {
    if (t < mine) fetch(t);
    cp_async_commit();
  }

  const T* sc0 = reinterpret_cast<const T*>(p.scales) + (int64_t)min(row0 + g, p.n - 1) * groups;
  const T* sc1 = reinterpret_cast<const T*>(p.scales) + (int64_t)min(row0 + g + 8, p.n - 1) * groups;
  const T* bi0 = reinterpret_cast<const T*>(p.biases) + (int64_t)min(row0 + g, p.n - 1) * groups;
  const T* bi1 = reinterpret_cast<const T*>(p.biases) + (int64_t)min(row0 + g + 8, p.n - 1) * groups;

  float y[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0.f;

  T s0[GS], s1[GS], b0[GS], b1[GS];  // scales of the stage to come
  auto fetch_scales = [&](int t) {
    const int gr = (t * WK + wk) * GS;
#pragma unroll
    for (int i = 0; i < GS; ++i) {
      const int at = min(gr + i, groups - 1);
      s0[i] = sc0[at];
      s1[i] = sc1[at];
      b0[i] = bi0[at];
      b1[i] = bi1[at];
    }
  };
  fetch_scales(0);

  int t = 0;
  for (int k0 = 0; k0 < p.k; k0 += chunk) {
    const int kn = min(chunk, steps * kStep - k0);  // a multiple of 128; columns past k are zero
    if (k0) __syncthreads();
    // x into shared memory: 8 columns (one word of weights) per thread, in the
    // order (0, 4, 1, 5, 2, 6, 3, 7); words of one group and index i next to
    // each other for c = 0 .. 3.
    const int words = kn / 8;
    for (int i = tid; i < words * rows_per_pass; i += kThreads) {
      const int m = i / words, wd = i - m * words, kk = k0 + wd * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (m < ms && kk < p.k) {
        const T* src = reinterpret_cast<const T*>(p.x) + (m0 + m) * p.x_stride + kk;
#pragma unroll
        for (int e = 0; e < 8; e += 16 / (int)sizeof(T))
          Vec16<T>::unpack(*reinterpret_cast<const uint4*>(src + e), v + e);
      }
      const int gr = wd / (4 * WL), in = wd - gr * 4 * WL, at = gr * 4 * WL + (in % WL) * 4 + in / WL;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const uint4 u = make_uint4(pack_bf16(v[0], v[4]), pack_bf16(v[1], v[5]), pack_bf16(v[2], v[6]), pack_bf16(v[3], v[7]));
        *reinterpret_cast<uint4*>(xs + (m * P + q) * x_bytes + at * 16) = u;
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] -= __uint_as_float(w[e] << 16);
          v[e + 4] -= __uint_as_float(w[e] & 0xffff0000u);
        }
      }
    }
    for (int i = tid + words * rows_per_pass * P; i < words * COLS; i += kThreads)  // columns without a row of x
      *reinterpret_cast<uint4*>(xs + (i / words) * x_bytes + (i % words) * 16) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i = tid; i < kn / G * COLS; i += kThreads) {
      const int col = i % COLS, gr = i / COLS;
      float sum = 0.f;
#pragma unroll 4
      for (int w = 0; w < 4 * WL; ++w) {
        float v[8];
        Vec16<__nv_bfloat16>::unpack(*reinterpret_cast<const uint4*>(xs + col * x_bytes + (gr * 4 * WL + w) * 16), v);
        sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      }
      sums[gr * COLS + col] = sum;
    }
    __syncthreads();

    for (; t < mine && (t * WK + wk) * kStep < k0 + kn; ++t) {
      cp_async_wait<kRing - 2>();
      __syncwarp();
      if (t + kRing - 1 < mine) fetch(t + kRing - 1);
      cp_async_commit();
      float fs0[GS], fs1[GS], fb0[GS], fb1[GS];
#pragma unroll
      for (int i = 0; i < GS; ++i) {
        fs0[i] = to_f(s0[i]);
        fs1[i] = to_f(s1[i]);
        fb0[i] = fmaf(8.f, fs0[i], to_f(b0[i]));
        fb1[i] = fmaf(8.f, fs1[i], to_f(b1[i]));
      }
      if (t + 1 < mine) fetch_scales(t + 1);
      const uint32_t st = ring + (t % kRing) * kStageBytes;
      const int at = (t * WK + wk) * kStep - k0;  // first column of the stage in the chunk
#pragma unroll
      for (int gi = 0; gi < GS; ++gi) {
        uint32_t w0[WL], w1[WL];
        load_words<WL>(w0, st, g, c, gi);
        load_words<WL>(w1, st, g + 8, c, gi);
        float acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
        for (int i = 0; i < WL; ++i) {
          const uint32_t a0[4] = {nibbles<0>(w0[i]), nibbles<0>(w1[i]), nibbles<4>(w0[i]), nibbles<4>(w1[i])};
          const uint32_t a1[4] = {nibbles<8>(w0[i]), nibbles<8>(w1[i]), nibbles<12>(w0[i]), nibbles<12>(w1[i])};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 b = *reinterpret_cast<const uint4*>(xs + (j * 8 + g) * x_bytes +
                                                            ((at / G + gi) * 4 * WL + i * 4 + c) * 16);
            mma_m16n8k16(acc[j], a0, b.x, b.y);
            mma_m16n8k16(acc[j], a1, b.z, b.w);
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 x2 = *reinterpret_cast<const float2*>(sums + (at / G + gi) * COLS + j * 8 + 2 * c);
          y[j][0] += fs0[gi] * acc[j][0] + fb0[gi] * x2.x;
          y[j][1] += fs0[gi] * acc[j][1] + fb0[gi] * x2.y;
          y[j][2] += fs1[gi] * acc[j][2] + fb1[gi] * x2.x;
          y[j][3] += fs1[gi] * acc[j][3] + fb1[gi] * x2.y;
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // Sums of the k splits and of the parts, in a fixed order; x's space.
  float* part = reinterpret_cast<float*>(xs);  // [wk][WR * 16][COLS + 1]
  constexpr int LD = COLS + 1;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      part[(wk * WR * 16 + wr * 16 + g + 8 * (e >> 1)) * LD + j * 8 + 2 * c + (e & 1)] = y[j][e];
  __syncthreads();
  for (int i = tid; i < ms * WR * 16; i += kThreads) {
    const int r = i % (WR * 16), m = i / (WR * 16), n = blockIdx.x * WR * 16 + r;
    if (n >= p.n) continue;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w)
#pragma unroll
      for (int q = 0; q < P; ++q) sum += part[(w * WR * 16 + r) * LD + m * P + q];
    reinterpret_cast<O*>(p.out)[(m0 + m) * p.out_stride + n] = from_f<O>(sum);
  }
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

template <typename T, typename O, int G, int NT, int WR>
cudaError_t q4_run(const Q4Params& p, cudaStream_t s) {
  constexpr int COLS = NT * 8, WK = kWarps / WR, P = Parts<T>::N;
  const int rows = COLS / P;  // rows of x per pass
  const int per = p.m < rows ? p.m : rows;
  const int unit = kStep * WK;
  const int padded = (p.k + kStep - 1) / kStep * kStep;
  int chunk = kChunkElems / COLS / unit * unit;  // columns of x held at a time
  static_assert(kChunkElems / COLS >= kStep * WK, "a chunk has a stage for every warp");
  if (chunk > padded) chunk = padded;
  int body = COLS * (chunk * 2 + 64) + chunk / G * COLS * 4;
  const int tail = WK * WR * 16 * (COLS + 1) * 4;
  const int bytes = kWarps * kRing * kStageBytes + (body > tail ? body : tail);
  constexpr auto K = q4_linear_kernel<T, O, G, NT, WR>;
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  const dim3 grid((p.n + WR * 16 - 1) / (WR * 16), (p.m + rows - 1) / rows);
  K<<<grid, kThreads, bytes, s>>>(p, per, chunk);
  return cudaGetLastError();
}

// Rows per CTA: as many as still give every SM a CTA (x is read once per CTA).
template <typename T, typename O, int G, int NT>
cudaError_t q4_rows(const Q4Params& p, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int n = op_sm_count(dev);
  if (p.n > 64 * n) return q4_run<T, O, G, NT, 4>(p, s);
  if (p.n > 32 * n) return q4_run<T, O, G, NT, 2>(p, s);
  return q4_run<T, O, G, NT, 1>(p, s);
}

template <typename T, typename O, int G>
cudaError_t q4_tiles(const Q4Params& p, cudaStream_t s) {
  const int cols = p.m * Parts<T>::N;
  if (cols <= 8) return q4_rows<T, O, G, 1>(p, s);
  if (cols <= 16) return q4_rows<T, O, G, 2>(p, s);
  if constexpr (Parts<T>::N == 3) {
    if (cols <= 24) return q4_rows<T, O, G, 3>(p, s);
  }
  return q4_rows<T, O, G, 4>(p, s);
}

template <typename T, typename O>
cudaError_t q4_group(const Q4Params& p, cudaStream_t s) {
  if (p.group == 32) return q4_tiles<T, O, 32>(p, s);
  if (p.group == 64) return q4_tiles<T, O, 64>(p, s);
  return q4_tiles<T, O, 128>(p, s);
}

}  // namespace

cudaError_t launch_q4_linear(const Q4Params& p, int dtype, int out_dtype, cudaStream_t s) {
  if (dtype == 0) return q4_group<float, float>(p, s);
  return out_dtype == 0 ? q4_group<__nv_bfloat16, float>(p, s) : q4_group<__nv_bfloat16, __nv_bfloat16>(p, s);
}

cudaError_t launch_q4_quantize(const Q4PackParams& p, int dtype, cudaStream_t s) {
  const int64_t all = (int64_t)p.n * (p.k / p.group), want = (all + 7) / 8;
  const unsigned grid = (unsigned)(want < 148 * 32 ? want : 148 * 32);
  if (dtype == 0) q4_quantize_kernel<float><<<grid, 256, 0, s>>>(p);
  else q4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mrtdf
