// Products with 4-bit weights for more than eight columns of x (rows x parts),
// and for those that do not fit the other kernel's shared memory. Everything
// streams: a stage is 128 rows of the weights x 256 columns (two TMA boxes of
// 64 bytes, 64-byte swizzle), x of these columns in the order of the matrix
// instructions' fragments (one bulk copy, 16 bytes per lane and instruction
// pair, without bank conflicts), and the scales and biases (through registers:
// their rows are as short as two bytes per stage).
//
// The stages of all row blocks stand in one line and every CTA takes an equal
// run of them (128 row blocks on 148 SMs are 128 runs' worth of work for 148
// CTAs); a row block that two or more CTAs share is summed from their partial
// sums by a second kernel, in the order of the columns.
//
// One warp loads a row's 16 outputs x all columns of x; up to 16 columns two
// warps share the rows and each take one of a stage's two steps. What bounds
// it: for eight columns the chain of a warp's step (load, unpack, product,
// scale), twice the weights' time over HBM; from 32 on the products themselves
// (mma.sync) and then, with small groups, the scaling. Microseconds of the
// whole call, bf16, 16384 x 8192, rows of x 8, 16, 32, 64, groups of 128: 23.7,
// 30.3, 43.1, 74.4 (weights alone 10.9); groups of 32: 30.0, 42.1, 59.3, 102.9;
// float32, groups of 128: 29.0, 38.0, 62.6, 114.6. With the rows of x resident instead, in as many chunks as the shared memory
// asked for, groups of 128 took 21.8, 35.6, 77.6, 153, groups of 32 143 to 614.
#include "q4_tile.cuh"
#include "tcgen05.cuh"

namespace mrtdf {
namespace {

constexpr int kBlock = 128;                 // rows of the weights per block
constexpr int kBoxBytes = kBlock * kStep / 2;
constexpr int kWideSmem = 200 * 1024;       // the rest stays L1, for the scales
constexpr int kScaleWarps = kBlock / 32;

template <typename T, int G, int NT>
struct Wide {
  static constexpr int COLS = NT * 8, GS = kStep / G, P = Parts<T>::N;
  static constexpr int Y = 4 / P;         // sums of a lane per tile of eight columns
  static constexpr int ROWS = COLS / P;   // rows of x
  static constexpr int CW = NT <= 2 ? 16 : 8;  // warps that multiply
  static constexpr int WK = CW / 8;            // of them, those that share 16 rows
  static constexpr bool APART = NT <= 2;  // a warp of its own issues the copies: the loaders would be too slow for both
  static constexpr int kThreads = (CW + kScaleWarps + APART) * 32;
  static constexpr bool TWO = NT <= 2;  // two chains of products, where there are few to overlap
  static constexpr int kXStep = COLS * 256 + GS * COLS * 8;  // bytes of x and its factors per step
  static constexpr int kX = 2 * kBoxBytes, kScales = kX + 2 * kXStep;
  static constexpr int kStage = (kScales + 2 * GS * kBlock * 2 * (int)sizeof(T) + 511) / 512 * 512;
  static constexpr int kMerge = WK > 1 ? 8 * 32 * NT * Y * 4 : 0;
  static constexpr int kStages = (kWideSmem - kMerge - 1024) / kStage < 8 ? (kWideSmem - kMerge - 1024) / kStage : 8;
  static constexpr int kBytes = kStages * kStage + kMerge + 512 + 2 * 8 * kStages;
  static_assert(kStages >= 3, "a ring");
  static constexpr int64_t x_bytes(int pairs) { return (int64_t)pairs * 2 * kXStep; }
};

// Runs of stages: CTA c of `grid` has [run(c), run(c + 1)).
struct Runs {
  int pairs;   // stages per row block
  int total;   // of all row blocks and passes
  int grid;
  int passes, rows;
  __host__ __device__ int start(int c) const { return (int)((int64_t)c * total / grid); }
  __host__ __device__ int owner(int u) const { return (int)((((int64_t)u + 1) * grid - 1) / total); }
};

template <typename T, int G, int NT>
__global__ __launch_bounds__(128) void q4_wide_prepare_kernel(const __grid_constant__ Q4Params p, int pairs, int rows) {
  using C = Wide<T, G, NT>;
  constexpr int WL = G / 32, P = C::P;
  pdl_launch_dependents();
  const int words = pairs * 2 * (kStep / 8), lane = threadIdx.x & 31, m0 = blockIdx.y * rows, all = words * (C::COLS / P);
  uint8_t* out = static_cast<uint8_t*>(p.ws) + blockIdx.y * C::x_bytes(pairs);
  const int i = blockIdx.x * 128 + threadIdx.x;
  if (i - lane >= all) return;
  const int m = i / words, wd = i - m * words, in = wd % (4 * WL), gi = wd % 16 / (4 * WL);
  uint8_t* step = out + (int64_t)(wd / 16) * C::kXStep;
  bring_x<T, G>(
      p, i < all && m < rows && m0 + m < p.m ? m0 + m : -1, wd * 8,
      [&](int h, uint4 w) {
        const int col = m * P + h;
        if (i < all)
          *reinterpret_cast<uint4*>(step + (((gi * WL + in % WL) * NT + col / 8) * 32 + col % 8 * 4 + in / WL) * 16) = w;
      },
      [&](int h, float2 f) {
        if (i < all && in == 0) *reinterpret_cast<float2*>(step + C::COLS * 256 + (gi * C::COLS + m * P + h) * 8) = f;
      });
}

// 2 GS scales and biases of a row, as loaded.
template <typename T, int GS>
struct alignas(16) ScaleVec {
  static constexpr int N = 2 * GS;
  alignas(16) T s[N];
  alignas(16) T b[N];
};

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <typename T, typename O, int G, int NT>
__global__ __launch_bounds__((Wide<T, G, NT>::kThreads), 1) void q4_wide_kernel(const __grid_constant__ CUtensorMap map,
                                                                              const __grid_constant__ Q4Params p,
                                                                              const __grid_constant__ Runs q) {
  using C = Wide<T, G, NT>;
  constexpr int WL = G / 32, GS = C::GS, P = C::P, Y = C::Y, COLS = C::COLS, ST = C::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((512 - (smem_u32(raw) & 511)) & 511);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * C::kStage + C::kMerge);
  uint64_t* empty = full + ST;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int abort_flag;
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(full + i, 1 + kScaleWarps);
      mbar_init(empty + i, C::CW);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  const int u0 = q.start(blockIdx.x), u1 = q.start(blockIdx.x + 1);
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(p.ws) + q.passes * C::x_bytes(q.pairs)) +
                (int64_t)blockIdx.x * 2 * C::ROWS * kBlock;

  // A wait that runs out ends all of the CTA's: copies stop, the sums become NaN.
  // `once`: it looks once and gives up (the waits for a free place in the ring,
  // when p.wait_once asks for it; in the products' own the test costs 1 to 2.5 %).
  auto wait = [&](uint64_t* bar, uint32_t parity, bool once = false) {
    if (once ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if (*(volatile int*)&abort_flag) return false;
    if (!once && mbar_wait_bounded(bar, parity, nullptr)) return true;
    *(volatile int*)&abort_flag = 1;
    return false;
  };

  if (warp >= C::CW) {
    // One thread issues the copies.
    const bool issues = tid == (C::APART ? C::CW + kScaleWarps : C::CW) * 32;
    const uint8_t* prepared = static_cast<const uint8_t*>(p.ws);
    struct At {  // a stage: its pass, row and columns, and its place in the ring
      int pass, row, pr, st;
    };
    auto begin = [&] {
      const int item = u0 / q.pairs;
      return At{item % q.passes, item / q.passes * kBlock, u0 - item * q.pairs, 0};
    };
    auto next = [&](At& a) {
      if (++a.st == ST) a.st = 0;
      if (++a.pr < q.pairs) return;
      a.pr = 0;
      if (++a.pass < q.passes) return;
      a.pass = 0;
      a.row += kBlock;
    };
    auto weights = [&](const At& a) {
      uint8_t* to = smem + a.st * C::kStage;
      mbar_arrive_expect_tx(full + a.st, 2 * kBoxBytes + 2 * C::kXStep);
      tcg::tma_load_2d(to, &map, a.pr * kStep, a.row, full + a.st);
      tcg::tma_load_2d(to + kBoxBytes, &map, a.pr * kStep + kStep / 2, a.row, full + a.st);
    };
    auto rows_of_x = [&](const At& a) {
      bulk_g2s(smem + a.st * C::kStage + C::kX, prepared + a.pass * C::x_bytes(q.pairs) + (int64_t)a.pr * 2 * C::kXStep,
               2 * C::kXStep, full + a.st);
    };
    const int head = min(u1, u0 + ST);
    int issued = head;  // stages [u0, issued)
    // No copy may still be landing when the CTA exits. After an aborted wait a
    // stage may lack its scales and never be full; its copies and the others' have
    // landed by the end of one such wait.
    auto landed = [&] {
      for (int u = max(u0, issued - ST); u < issued; ++u)
        if (!mbar_wait_bounded(full + (u - u0) % ST, (u - u0) / ST & 1, nullptr)) break;
    };
    At to_copy = begin();
    if (issues)
      for (int u = u0; u < head; ++u, next(to_copy)) weights(to_copy);
    auto prologue = [&] {
      pdl_wait();  // x is prepared
      At a = begin();
      for (int u = u0; u < head; ++u, next(a)) rows_of_x(a);
    };
    if (C::APART && warp == C::CW + kScaleWarps) {
      if (issues) {
        prologue();
        for (int u = head, turn = 0; u < u1 && wait(empty + to_copy.st, turn, p.wait_once); ++u, next(to_copy)) {
          weights(to_copy);
          rows_of_x(to_copy);
          issued = u + 1;
          if (to_copy.st == ST - 1) turn ^= 1;
        }
        landed();
      }
      return;
    }
    // A thread has a row: it loads the scales of a stage a few stages ahead.
    constexpr int kAhead = GS * (int)sizeof(T) >= 16 ? 2 : 4;
    const int r = tid - C::CW * 32, groups = p.k / G;
    using V = ScaleVec<T, GS>;
    constexpr int kVec = V::N * (int)sizeof(T);  // bytes of a stage: 4 .. 32
    constexpr int kLoad = kVec < 16 ? kVec : 16;
    const bool wide = groups % V::N == 0 && ((uintptr_t)p.scales | (uintptr_t)p.biases) % kLoad == 0;
    V ahead[kAhead];
    At to_load = begin();
    auto load = [&](V& v, int u) {
      const int g0 = to_load.pr * V::N, n = to_load.row + r;
      next(to_load);
      const int64_t from = (int64_t)n * groups + g0;
      const T *s = static_cast<const T*>(p.scales) + from, *b = static_cast<const T*>(p.biases) + from;
      if (u >= u1 || n >= p.n) {
#pragma unroll
        for (int e = 0; e < V::N; ++e) v.s[e] = v.b[e] = from_f<T>(0.f);
      } else if (wide) {
        if constexpr (kLoad == 4) {
          *reinterpret_cast<uint32_t*>(v.s) = __ldg(reinterpret_cast<const uint32_t*>(s));
          *reinterpret_cast<uint32_t*>(v.b) = __ldg(reinterpret_cast<const uint32_t*>(b));
        } else if constexpr (kLoad == 8) {
          *reinterpret_cast<uint2*>(v.s) = __ldg(reinterpret_cast<const uint2*>(s));
          *reinterpret_cast<uint2*>(v.b) = __ldg(reinterpret_cast<const uint2*>(b));
        } else {
#pragma unroll
          for (int e = 0; e < kVec / 16; ++e) {
            reinterpret_cast<uint4*>(v.s)[e] = __ldg(reinterpret_cast<const uint4*>(s) + e);
            reinterpret_cast<uint4*>(v.b)[e] = __ldg(reinterpret_cast<const uint4*>(b) + e);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < V::N; ++e) {
          v.s[e] = g0 + e < groups ? s[e] : from_f<T>(0.f);
          v.b[e] = g0 + e < groups ? b[e] : from_f<T>(0.f);
        }
      }
    };
#pragma unroll
    for (int d = 0; d < kAhead; ++d) load(ahead[d], u0 + d);
    if (!C::APART && issues) prologue();
    int st = 0, turn = 0;
    bool on = true;
    for (int u = u0; u < u1 && on; u += kAhead) {
#pragma unroll
      for (int d = 0; d < kAhead; ++d) {
        if (u + d >= u1) break;
        if (u + d >= head) {
          on = __all_sync(0xffffffffu, wait(empty + st, turn, p.wait_once));
          if (!on) break;
          if (!C::APART && issues) {
            weights(to_copy);
            rows_of_x(to_copy);
            next(to_copy);
            issued = u + d + 1;
          }
        }
        auto* to = reinterpret_cast<ScalePair<T>*>(smem + st * C::kStage + C::kScales);
#pragma unroll
        for (int e = 0; e < V::N; ++e) to[e * kBlock + r] = ScalePair<T>{ahead[d].s[e], ahead[d].b[e]};
        __syncwarp();
        if (lane == 0) mbar_arrive(full + st);
        if (++st == ST) {
          st = 0;
          if (u + d >= head) turn ^= 1;
        }
        load(ahead[d], u + d + kAhead);
      }
    }
    if (!C::APART && issues) landed();
  } else {
    const int wt = warp & 7, wk = warp >> 3, g = lane >> 2, c = lane & 3;
    const uint32_t swz = (uint32_t)(g >> 1 & 3) << 4;  // of rows g and g + 8
    const uint32_t base = smem_u32(smem);
    float y[NT][Y] = {};
    int item = u0 / q.pairs, pr = u0 - item * q.pairs, st = 0, phase = 0;
    bool whole = pr == 0;  // the row block from its first stage on
    bool on = true;        // after a wait that ran out no other is begun: each may take the hardware's time for one look
    for (int u = u0; u < u1; ++u) {
      on = on && wait(full + st, phase);
      const uint32_t stage = base + st * C::kStage;
#pragma unroll
      for (int half = 0; half < 2 / C::WK; ++half) {
        const int sub = C::WK > 1 ? wk : half;
        const uint32_t row = stage + sub * kBoxBytes + (wt * 16 + g) * (kStep / 2), xa = stage + C::kX + sub * C::kXStep + lane * 16;
        const uint32_t fa = stage + C::kX + sub * C::kXStep + COLS * 256 + 2 * c * 8;
        const uint32_t sa = stage + C::kScales + (sub * GS * kBlock + wt * 16 + g) * 2 * (int)sizeof(T);
#pragma unroll
        for (int gi = 0; gi < GS; ++gi) {
          uint32_t w0[WL], w1[WL];
          load_words<WL>(w0, row, swz, c, gi);
          load_words<WL>(w1, row + 8 * (kStep / 2), swz, c, gi);
          float s0, s1, b0, b1;
          load_pair(sa + gi * kBlock * 2 * (int)sizeof(T), s0, b0, T());
          load_pair(sa + (gi * kBlock + 8) * 2 * (int)sizeof(T), s1, b1, T());
          float acc[NT][4], acd[C::TWO ? NT : 1][4];
#pragma unroll
          for (int i = 0; i < WL; ++i) {
            uint32_t a0[4], a1[4];
            unpack(w0[i], a0[0], a0[2]);
            unpack(w1[i], a0[1], a0[3]);
            unpack(w0[i] >> 8, a1[0], a1[2]);
            unpack(w1[i] >> 8, a1[1], a1[3]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const uint4 b = lds128(xa + ((gi * WL + i) * NT + j) * 512);
              if (i == 0) mma_f16_first(acc[j], a0, b.x, b.y);
              else mma_f16(acc[j], a0, b.x, b.y);
              if (!C::TWO) mma_f16(acc[j], a1, b.z, b.w);
              else if (i == 0) mma_f16_first(acd[j], a1, b.z, b.w);
              else mma_f16(acd[j], a1, b.z, b.w);
            }
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (C::TWO) {
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[j][e] += acd[j][e];
            }
            add_group<P>(y[j], acc[j], lds128(fa + (gi * COLS + j * 8) * 8), s0, b0, s1, b1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + st);
      if (++st == ST) {
        st = 0;
        phase ^= 1;
      }
      const bool ends = ++pr == q.pairs;
      if (ends || u + 1 == u1) {
        if (*(volatile int*)&abort_flag) {
#pragma unroll
          for (int i = 0; i < NT * Y; ++i) y[i / Y][i % Y] = NAN;
        }
        if (C::WK > 1) {  // the other warp's sums of these rows
          float* merge = reinterpret_cast<float*>(smem + ST * C::kStage) + wt * 32 + lane;
          if (wk) {
#pragma unroll
            for (int i = 0; i < NT * Y; ++i) merge[i * 256] = y[i / Y][i % Y];
          }
          asm volatile("bar.sync 1, %0;" ::"n"(C::CW * 32) : "memory");
          if (!wk) {
#pragma unroll
            for (int i = 0; i < NT * Y; ++i) y[i / Y][i % Y] += merge[i * 256];
          }
          asm volatile("bar.sync 1, %0;" ::"n"(C::CW * 32) : "memory");
        }
        if (wk == 0) {
          const int m0 = item % q.passes * q.rows, n0 = item / q.passes * kBlock;
          float* to = part + (u0 / q.pairs != item ? C::ROWS * kBlock : 0);
          O* out = reinterpret_cast<O*>(p.out) + n0;
#pragma unroll
          for (int i = 0; i < NT * Y; ++i) {
            const int m = P == 2 ? i / Y * 4 + c : i / Y * 8 + 2 * c + (i & 1), r = wt * 16 + g + 8 * (P == 2 ? i & 1 : i >> 1 & 1);
            if (!(whole && ends)) to[m * kBlock + r] = y[i / Y][i % Y];
            else if (n0 + r < p.n && m < q.rows && m0 + m < p.m) out[(m0 + m) * p.out_stride + r] = from_f<O>(y[i / Y][i % Y]);
          }
        }
#pragma unroll
        for (int i = 0; i < NT * Y; ++i) y[i / Y][i % Y] = 0.f;
        ++item;
        pr = 0;
        whole = true;
      }
    }
  }
}

// Sums of a row block that begins in CTA c - 1 and goes on in c and maybe
// later ones: two rows of x per CTA.
template <typename T, typename O, int G, int NT>
__global__ __launch_bounds__(256) void q4_wide_join_kernel(const __grid_constant__ Q4Params p, const __grid_constant__ Runs q) {
  using C = Wide<T, G, NT>;
  const int c = blockIdx.x + 1, u = q.start(c), item = u / q.pairs, first = item * q.pairs;
  const bool joins = u != first && q.start(c - 1) <= first;
  const int last = q.owner(first + q.pairs - 1), m0 = item % q.passes * q.rows, n0 = item / q.passes * kBlock;
  const int m = blockIdx.y * 2 + (threadIdx.x >> 7), r = threadIdx.x & 127;
  // Every CTA waits, those without work too: the join is done when the products
  // are, and so what comes next on the stream may use them.
  pdl_wait();
  if (!joins || m >= q.rows || m0 + m >= p.m || n0 + r >= p.n) return;
  const float* part = reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.ws) + q.passes * C::x_bytes(q.pairs)) + m * kBlock + r;
  float sum = 0.f;
  for (int o = c - 1; o <= last; ++o) sum += part[((int64_t)o * 2 + (o == c - 1 && q.start(o) != first)) * C::ROWS * kBlock];
  reinterpret_cast<O*>(p.out)[(m0 + m) * p.out_stride + n0 + r] = from_f<O>(sum);
}

template <typename T, typename O, int G, int NT>
cudaError_t wide_run(const Q4Params& p, int sms, size_t* ws_bytes, cudaStream_t s) {
  using C = Wide<T, G, NT>;
  Runs q{};
  q.rows = p.m < C::ROWS ? p.m : C::ROWS;
  q.passes = (p.m + q.rows - 1) / q.rows;
  q.pairs = (p.k + 2 * kStep - 1) / (2 * kStep);
  q.total = (p.n + kBlock - 1) / kBlock * q.passes * q.pairs;
  q.grid = q.total < sms ? q.total : sms;
  if (ws_bytes) {
    *ws_bytes = (size_t)(q.passes * C::x_bytes(q.pairs)) + (size_t)q.grid * 2 * C::ROWS * kBlock * 4;
    return cudaSuccess;
  }
  CUtensorMap map;
  const auto encode = tcg::encode_tiled_fn();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)p.k / 2, (cuuint64_t)p.n}, strides[1] = {(cuuint64_t)p.k / 2};
  const cuuint32_t box[2] = {kStep / 2, kBlock}, step[2] = {1, 1};
  if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(p.packed), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorInvalidValue;
  constexpr auto K = q4_wide_kernel<T, O, G, NT>;
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  const int words = q.pairs * 2 * (kStep / 8) * C::ROWS;
  q4_wide_prepare_kernel<T, G, NT><<<dim3((words + 127) / 128, q.passes), 128, 0, s>>>(p, q.pairs, q.rows);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(q.grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kBytes;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, K, map, p, q);
  // A row block is one CTA's alone where runs end with it.
  if (e != cudaSuccess || q.grid == 1 || q.pairs == 1 || (q.total % q.grid == 0 && q.total / q.grid % q.pairs == 0)) return e;
  cfg.gridDim = dim3(q.grid - 1, (q.rows + 1) / 2);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, q4_wide_join_kernel<T, O, G, NT>, p, q);
}

template <typename T, typename O, int G>
cudaError_t wide_tiles(const Q4Params& p, int sms, size_t* ws, cudaStream_t s) {
  const int cols = p.m * Parts<T>::N;
  if (cols <= 8) return wide_run<T, O, G, 1>(p, sms, ws, s);
  if (cols <= 16) return wide_run<T, O, G, 2>(p, sms, ws, s);
  if (cols <= 32) return wide_run<T, O, G, 4>(p, sms, ws, s);
  return wide_run<T, O, G, 8>(p, sms, ws, s);
}

template <typename T, typename O>
cudaError_t wide_group(const Q4Params& p, int sms, size_t* ws, cudaStream_t s) {
  if (p.group == 32) return wide_tiles<T, O, 32>(p, sms, ws, s);
  if (p.group == 64) return wide_tiles<T, O, 64>(p, sms, ws, s);
  return wide_tiles<T, O, 128>(p, sms, ws, s);
}

}  // namespace

cudaError_t launch_q4_wide(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s) {
  if (dtype == 0) return wide_group<float, float>(p, sms, ws_bytes, s);
  return out_dtype == 0 ? wide_group<__nv_bfloat16, float>(p, sms, ws_bytes, s)
                        : wide_group<__nv_bfloat16, __nv_bfloat16>(p, sms, ws_bytes, s);
}

}  // namespace mrtdf
