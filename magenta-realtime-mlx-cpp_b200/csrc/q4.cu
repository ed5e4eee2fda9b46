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
// cp.async ring to registers, where two nibbles of a 16-bit half become q - 8 in
// two instructions and without a shift (unpack, q4_tile.cuh). Without the second,
// an offset of 1024 per weight goes through the products' sums and comes off
// afterwards; the matrix instructions cut sums off towards zero, so x of one sign
// (after a gated activation) then put every result 2.3e-4 of its size too low (16384
// x 8192: 8 rows 24.0 us, 22.8 with the offset; one row 21.6, 19.6 with it).
// x is brought to fp16 by a power of two per row and group that puts the
// group's largest |x| into [2^14, 2^15): bf16 x keeps all its bits (smaller
// ones down to 2^-31 of the largest), float32 x becomes two columns, x = hi + lo
// with 22 bits. The factor multiplies the group's float32 sum at the end. Here every CTA
// does that for itself, which is right for small x only: for more, and for what
// does not fit the shared memory, see q4_wide.cu.
//
// The k index of a product is arbitrary as long as both operands agree: lane
// (g, c) unpacks whole words of 8 columns from its own rows, in the pairs
// (0, 4), (1, 5), (2, 6), (3, 7), and x lies in shared memory in the order in
// which the lanes ask for it.
#include "q4_tile.cuh"

namespace mrtdf {
namespace {

constexpr int kMaxWarps = 16;
constexpr int kStepBytes = 16 * kStep / 2;
// A ring stage has two steps, so that a row gives 128 bytes at a time: in 64-byte
// pieces 67 MB came in 13 us, in 128-byte pieces in 11 (from L2, no products).
constexpr int kStageBytes = 2 * kStepBytes;
constexpr int kRing = 4;  // stages per warp
constexpr int kSmemMax = 224 * 1024;
constexpr int kCols = 8;  // columns of the product: rows of x x parts

// How a product is laid out over the GPU.
struct Q4Plan {
  int split;  // CTAs of a cluster: each has a slab of the columns
  int tiles;  // row tiles of 16 per cluster (and so per CTA)
  int warps;  // warps with tiles of their own, taking every warps-th
  int wk;     // warps per tile: each takes every wk-th stage of the slab
  int slab;   // steps of 128 columns per CTA
  int steps;  // all steps
};

// Shared memory of a CTA, in order: rings, x, factors of x, scales, partial
// sums.
template <typename T, int G>
struct Q4Smem {
  int x_bytes, x, factors, scales, part, bytes;
  __host__ __device__ explicit Q4Smem(const Q4Plan& q) {
    x_bytes = q.slab * kStep * 2 + 64;
    x = q.warps * q.wk * kRing * kStageBytes;
    factors = x + kCols * x_bytes;
    scales = factors + (q.slab * kStep / G) * kCols * 8;
    part = scales + (q.slab * kStep / G) * q.tiles * 16 * 2 * (int)sizeof(T);
    const int units = q.tiles > q.warps * q.wk ? q.tiles : q.warps * q.wk;
    bytes = part + units * 16 * (kCols / Parts<T>::N + 1) * 4;
  }
};

__device__ __forceinline__ float ld_cluster_f32(const float* local, uint32_t rank) {
  uint32_t ra;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra) : "memory");
  return v;
}

// Where word wd of a row lies: words of one group and index i next to each
// other for c = 0 .. 3.
template <int WL>
__device__ __forceinline__ int word_at(int wd) {
  const int in = wd % (4 * WL);
  return wd - in + (in % WL) * 4 + in / WL;
}

// T: type of x, scales and biases. A cluster works on q.tiles row tiles, its
// CTAs on a slab of the columns each; the slabs' sums meet over distributed
// shared memory, in rank order. Every CTA brings its slab of x to fp16 itself.
template <typename T, typename O, int G>
__global__ __launch_bounds__(kMaxWarps * 32, 1) void q4_linear_kernel(const __grid_constant__ Q4Params p,
                                                                      const __grid_constant__ Q4Plan q) {
  constexpr int WL = G / 32, GS = kStep / G, P = Parts<T>::N, ROWS = kCols / P, LD = ROWS + 1;  // rows of x
  extern __shared__ __align__(128) uint8_t smem[];
  const Q4Smem<T, G> at(q);
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int wt = warp % q.warps, wk = warp / q.warps, g = lane >> 2, c = lane & 3;
  const int rank = q.split > 1 ? (int)cluster_ctarank() : 0, cluster = blockIdx.x / q.split;
  const int tile0 = cluster * q.tiles, tiles = min(q.tiles, (p.n + 15) / 16 - tile0), stride = q.tiles * 16;
  const int groups = p.k / G, row_bytes = p.k / 2, n0 = tile0 * 16;
  const int step0 = rank * q.slab, steps = min(q.slab, q.steps - step0), k0 = step0 * kStep;
  auto* sb = reinterpret_cast<ScalePair<T>*>(smem + at.scales);  // [group][row]
  float* part = reinterpret_cast<float*>(smem + at.part);  // [wk][row][LD]

  const uint32_t ring = smem_u32(smem) + warp * (kRing * kStageBytes);
  const int fr = lane >> 3, fc = lane & 7;  // a lane copies chunk fc of rows fr, fr + 4, ...
  const int units_max = q.tiles > q.warps * q.wk ? q.tiles : q.warps * q.wk;
  for (int i = tid; i < units_max * 16 * LD; i += threads) part[i] = 0.f;

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

  const int gn = steps * GS, g0 = k0 / G;
  // Scales and biases of the slab's groups, side by side: 16 bytes at a time
  // where rows, groups and the two addresses allow it.
  constexpr int E = 16 / (int)sizeof(T);
  if (groups % E == 0 && g0 % E == 0 && ((uintptr_t)p.scales | (uintptr_t)p.biases) % 16 == 0) {
    const int vecs = (gn + E - 1) / E, all = tiles * 16 * vecs;
    for (int i0 = tid; i0 < all; i0 += 4 * threads) {
      uint4 s[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * threads, all - 1), r = i / vecs, gr = g0 + (i - r * vecs) * E;
        const int64_t from = (int64_t)min(n0 + r, p.n - 1) * groups + gr;
        s[u] = b[u] = make_uint4(0, 0, 0, 0);  // past the last column
        if (gr < groups) {
          s[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.scales) + from);
          b[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.biases) + from);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * threads, all - 1), r = i / vecs, first = (i - r * vecs) * E;
        const T *sv = reinterpret_cast<const T*>(&s[u]), *bv = reinterpret_cast<const T*>(&b[u]);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first + e < gn) sb[(first + e) * stride + r] = ScalePair<T>{sv[e], bv[e]};
      }
    }
  } else {
    for (int i = tid; i < gn * tiles * 16; i += threads) {
      const int r = i / gn, gr = i - r * gn;
      const int64_t from = (int64_t)min(n0 + r, p.n - 1) * groups + g0 + gr;
      ScalePair<T> pair{from_f<T>(0.f), from_f<T>(0.f)};
      if (g0 + gr < groups) pair = {reinterpret_cast<const T*>(p.scales)[from], reinterpret_cast<const T*>(p.biases)[from]};
      sb[gr * stride + r] = pair;
    }
  }
  const int words = steps * (kStep / 8), all_words = words * p.m, spare = kCols - p.m * P;
  float2* factor = reinterpret_cast<float2*>(smem + at.factors);
  for (int i0 = tid; i0 - lane < all_words; i0 += threads) {
    const int m = i0 / words, wd = i0 - m * words;
    bring_x<T, G>(
        p, i0 < all_words ? m : -1, k0 + wd * 8,
        [&](int h, uint4 w) {
          if (i0 < all_words) *reinterpret_cast<uint4*>(smem + at.x + (m * P + h) * at.x_bytes + word_at<WL>(wd) * 16) = w;
        },
        [&](int h, float2 f) {
          if (i0 < all_words && wd % (4 * WL) == 0) factor[wd / (4 * WL) * kCols + m * P + h] = f;
        });
  }
  for (int i = tid; i < words * spare; i += threads)  // columns without a row of x
    *reinterpret_cast<uint4*>(smem + at.x + (kCols - spare + i / words) * at.x_bytes + (i % words) * 16) = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < gn * spare; i += threads)
    factor[i / spare * kCols + kCols - spare + i % spare] = make_float2(0.f, 0.f);
  __syncthreads();

  float y[4 / P] = {};
  // Shared addresses of this lane's operands in the unit's step.
  const uint32_t swz = (uint32_t)(g >> 1 & 3) << 4;  // of rows g and g + 8
  const uint32_t x_first = smem_u32(smem + at.x) + g * at.x_bytes + c * 16 + wk * 2 * GS * (WL * 64);
  const uint32_t f_first = smem_u32(smem + at.factors) + (wk * 2 * GS * kCols + 2 * c) * 8;
  const uint32_t s_first = smem_u32(sb) + (wk * 2 * GS * stride + wt * 16 + g) * 2 * (int)sizeof(T);
  const uint32_t x_step = GS * (WL * 64), fa_step = GS * kCols * 8, skip = 2 * q.wk - 2, s_group = stride * 2 * (int)sizeof(T);
  uint32_t xa = x_first, fa = f_first, sa = s_first, row = ring + g * (kStep / 2), st = 0;
  int tile = wt, step = 0;
  for (int t = 0; t < units; ++t) {
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
        float acc[4], acd[4];
#pragma unroll
        for (int i = 0; i < WL; ++i) {
          uint32_t a0[4], a1[4];
          unpack(w0[i], a0[0], a0[2]);
          unpack(w1[i], a0[1], a0[3]);
          unpack(w0[i] >> 8, a1[0], a1[2]);
          unpack(w1[i] >> 8, a1[1], a1[3]);
          const uint4 b = lds128(xa + gi * (WL * 64) + i * 64);
          if (i == 0) {
            mma_f16_first(acc, a0, b.x, b.y);
            mma_f16_first(acd, a1, b.z, b.w);
          } else {
            mma_f16(acc, a0, b.x, b.y);
            mma_f16(acd, a1, b.z, b.w);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += acd[e];
        add_group<P>(y, acc, lds128(fa + gi * kCols * 8), s0, b0, s1, b1);
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
      float* to = part + ((wk * q.warps + tile) * 16 + g) * LD + c * (2 / P);
#pragma unroll
      for (int e = 0; e < 4 / P; ++e) {
        to[P == 2 ? 8 * e * LD : 8 * (e >> 1) * LD + (e & 1)] += y[e];
        y[e] = 0.f;
      }
      step = 0;
      tile += q.warps;
      xa = x_first;
      fa = f_first;
      sa = s_first + (tile - wt) * 32 * (int)sizeof(T);
    }
  }
  cp_async_wait<0>();

  // Sums of the warps that share tiles (then each has one) and of the slabs, in
  // a fixed order.
  if (q.wk > 1) {
    __syncthreads();
    for (int i = tid; i < tiles * 16 * ROWS; i += threads) {
      const int cell = i / ROWS * LD + i % ROWS;
      float sum = part[cell];
      for (int w = 1; w < q.wk; ++w) sum += part[w * q.warps * 16 * LD + cell];
      part[cell] = sum;
    }
  }
  if (q.split > 1) cluster_sync();
  else __syncthreads();
  for (int i = rank * threads + tid; i < p.m * tiles * 16; i += q.split * threads) {
    const int m = i / (tiles * 16), r = i - m * (tiles * 16), n = n0 + r;
    if (n >= p.n) continue;
    float sum = 0.f;
    const float* from = part + r * LD + m;
    for (int o = 0; o < q.split; ++o) sum += q.split > 1 ? ld_cluster_f32(from, o) : *from;
    reinterpret_cast<O*>(p.out)[m * p.out_stride + n] = from_f<O>(sum);
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
// columns for each of a pair where there are 16 steps or more.
Q4Plan q4_plan(const Q4Params& p, int sms) {
  const int tiles = (p.n + 15) / 16;
  Q4Plan q{};
  q.steps = (p.k + kStep - 1) / kStep;
  q.split = q.steps >= 16 ? 2 : 1;
  q.slab = (q.steps + q.split - 1) / q.split;
  const int clusters = max(1, sms / q.split);
  q.tiles = (tiles + clusters - 1) / clusters;
  const int per_warp = (q.tiles + kMaxWarps - 1) / kMaxWarps;
  q.warps = (q.tiles + per_warp - 1) / per_warp;
  q.wk = max(1, min(kMaxWarps / q.warps, (q.slab + 1) / 2));
  return q;
}

template <typename T, typename O, int G>
cudaError_t q4_launch(const Q4Params& p, const Q4Plan& q, cudaStream_t s) {
  constexpr auto K = q4_linear_kernel<T, O, G>;
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = q.split;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(((p.n + 15) / 16 + q.tiles - 1) / q.tiles * q.split);
  cfg.blockDim = dim3(q.warps * q.wk * 32);
  cfg.dynamicSmemBytes = Q4Smem<T, G>(q).bytes;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = q.split > 1;
  return cudaLaunchKernelEx(&cfg, K, p, q);
}

// This kernel where x is small, so that every CTA can bring it to fp16 for
// itself (up to a word per thread), has one tile of columns, and all fits the
// shared memory; otherwise the one that streams everything. Microseconds, bf16,
// group 128, this kernel and the other:
//   rows of x        1           4           8
//   1024 x 1024      4.2  6.2    5.7  6.3    7.3  6.2
//   4096 x 4096      7.6  9.0    8.7  9.4    (does not fit)
//   16388 x 1024     6.4  8.4    7.2  8.9    7.7  9.2
//   16384 x 8192    21.6 23.1   23.5 23.6   26.2 23.7
// (a word per thread decides: 4 rows of 4096 and 8 rows of 16388 x 1024 would
// gain 7 and 17 %, 8 rows of the other sizes lose as much).
template <typename T, typename O, int G>
cudaError_t q4_run(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s) {
  const Q4Plan q = q4_plan(p, sms);
  if (p.m * Parts<T>::N > kCols || (int64_t)q.slab * (kStep / 8) * p.m > kMaxWarps * 32 || Q4Smem<T, G>(q).bytes > kSmemMax)
    return launch_q4_wide(p, dtype, out_dtype, sms, ws_bytes, s);
  if (ws_bytes) {
    *ws_bytes = 0;
    return cudaSuccess;
  }
  return q4_launch<T, O, G>(p, q, s);
}

template <typename T, typename O>
cudaError_t q4_group(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws, cudaStream_t s) {
  if (p.group == 32) return q4_run<T, O, 32>(p, dtype, out_dtype, sms, ws, s);
  if (p.group == 64) return q4_run<T, O, 64>(p, dtype, out_dtype, sms, ws, s);
  return q4_run<T, O, 128>(p, dtype, out_dtype, sms, ws, s);
}

}  // namespace

cudaError_t launch_q4_linear(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s) {
  if (dtype == 0) return q4_group<float, float>(p, dtype, out_dtype, sms, ws_bytes, s);
  return out_dtype == 0 ? q4_group<__nv_bfloat16, float>(p, dtype, out_dtype, sms, ws_bytes, s)
                        : q4_group<__nv_bfloat16, __nv_bfloat16>(p, dtype, out_dtype, sms, ws_bytes, s);
}

cudaError_t launch_q4_quantize(const Q4PackParams& p, int dtype, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int64_t all = (int64_t)p.n * (p.k / p.group), want = (all + 7) / 8, most = 32 * op_sm_count(dev);
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (dtype == 0) q4_quantize_kernel<float><<<grid, 256, 0, s>>>(p);
  else q4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mrtdf
