// Attention of a drafted tree over a KV cache (bf16) on the 5th-generation
// tensor cores, for trees and head groups of more than a few rows. The
// mathematics is that of cache_attn.cu.
//
// The rows of one kv head (nodes x its query heads) are the M side of
// tcgen05.mma, 128 at a time. With 128 rows a tile of 64 keys takes some 800
// clocks of products (head_dim 128) and its 32 KB of K and V come in 1400 at
// the memory's rate, so padding to 128 rows costs nothing while the cache is
// read from HBM. The A operands (the queries, and the weights in the place of
// the scores they came from) are in TMEM: read from shared memory, 64 columns at
// a time, they alone kept the products at a third of their rate.
//
// CTA of 576 threads, one per SM, over an equal run of the key tiles of all
// items (cache_sched.cuh); roles and hand-over as in enc_attn_tc.cu:
//   warps 0-15 softmax: two groups of eight warps take turns at the tiles, each
//              with a running maximum and an accumulator of its own, so that
//              one's exponentials overlap the other's products; two threads per
//              query row, each with 32 of the 64 columns, who tell each other
//              their maxima (rows that do not exist skip the work: their
//              queries are zero, their scores stay zero bits);
//   warp 16    TMA producer: K and V tiles through a ring, 128-byte swizzle,
//              over the items of the run without a stop;
//   warp 17    MMA issuer: S = Q K^T into one of three TMEM buffers, two
//              tiles ahead, then O_g += P V for the tile's group g, weights as
//              two bf16 parts (16 bits of a weight).
//              V is an MN-major operand of 64-column parts kSub bytes apart.
// A maximum is raised only when a tile exceeds it by 8 units of its scale.
// The drafted rows are a tile of their own behind the cached ones.
//
// Values that no row sees must not meet the products, where 0 x NaN is NaN:
// rows behind the length are zeroed in the last cached tile, and in the drafted
// tile single values that are not finite, which the rows that do see them take
// from global memory at the end.
//
// Measured on a B200, us in a graph: 4 sequences x 8 kv heads of 128, 24 nodes of
// four heads each (96 rows), 4097 to 16360 rows, 169 MB: 64 (2.6 TB/s, 275
// TFLOP/s of real rows). A tile of 64 keys takes 0.95 us per SM, 0.75 of it its
// products (two for the weights, since they keep 16 bits); the run's start (the
// schedule and the queries to TMEM) 6, its end 4, the join of split items 3. With
// heads of 64 a tile takes 0.86 us: the chain scores - maximum - exponentials -
// weights - products of one tile, with two tiles in flight, not the products.
#include <cuda.h>

#include "cache_sched.cuh"
#include "tcgen05.cuh"

namespace mrtdf {
namespace {

using namespace tcg;
typedef __nv_bfloat16 bf16;

constexpr int kRows = 128;
constexpr int kSoft = 512;              // softmax threads
constexpr int kTcThreads = kSoft + 64;  // and the TMA and MMA warps
constexpr int kSub = 64 * 128;          // 64 rows of 128 bytes (64 columns)
constexpr float kLazy = 8.f;

template <int D>
struct TcCfg {
  static constexpr int kSubs = D / 64;  // 64-column parts of a row
  static constexpr int kStagesKv = D == 64 ? 8 : 6;
  static constexpr int kKvBytes = kSub * kSubs;
  static constexpr int kOffBar = kStagesKv * 2 * kKvBytes;
  static constexpr int kOffSched = kOffBar + 256;
  static int smem(int batch) { return kOffSched + (2 * batch + 1) * 4 + 1024; }
};
// TMEM columns: the scores of a tile, then its weights (32 columns of high
// parts, 32 of low ones), three times; O_0 and O_1; the queries.
constexpr int kBufs = 3;
constexpr uint32_t kTmem = 512, kColO = kBufs * 64;
template <int D>
constexpr uint32_t kColQ = kColO + 2 * D;
// kind::f16, D f32, A / B bf16, M 128, K-major B of 64 rows; PV: B MN-major.
constexpr uint32_t idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
constexpr uint32_t kMnMajorB = 1u << 16;

struct TcMaps {
  CUtensorMap k, v, kn, vn;
};

// A in TMEM (row = lane, two bf16 per column), B in shared memory. One lane of
// the warp issues; the operands are the same in all of them, so they can be
// kept in uniform registers (a single lane's branch has to move five operands
// there for every product, 80 clocks each).
__device__ __forceinline__ void umma(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ bool elected() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

template <int D, bool BIAS>
__global__ __launch_bounds__(kTcThreads, 1) void tree_attn_tc_kernel(const __grid_constant__ TcMaps maps,
                                                                       const __grid_constant__ TreeParams p) {
  using C = TcCfg<D>;
  constexpr int NS = C::kStagesKv, SUBS = C::kSubs;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t *q_full = bar, *o_done = bar + 1, *drain = bar + 2, *kv_full = bar + 3, *kv_empty = bar + 3 + NS;
  uint64_t *s_full = bar + 3 + 2 * NS, *p_full = s_full + kBufs, *p_empty = p_full + kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_empty + kBufs);
  int* lens = reinterpret_cast<int*>(smem + C::kOffSched);
  int* first = lens + p.c.batch;
  __shared__ int abort_flag;
  __shared__ unsigned long long seen[kOpMaxNodes], poison;
  __shared__ float xm[2][kRows], xl[4][kRows], tops[2][2][2][kRows];  // tops: [slot][group][half][row]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int batch = p.c.batch, blocks = p.row_blocks, items = p.c.kv_heads * blocks, nodes = p.nodes;
  const int heads_per = p.heads / p.c.kv_heads, rows = heads_per * nodes;

  pdl_launch_dependents();  // the grid is resident at once: the join may take its places beside it
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    mbar_init(q_full, kSoft / 32);
    mbar_init(o_done, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, kSoft / 64);  // the warps of one group
      mbar_init(p_empty + i, 1);
    }
    fence_mbar_init();
    abort_flag = 0;
  }
  tc_fence_before();
  build_schedule<true>(p.c, batch, items, nodes, lens, first);  // ends with a barrier
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int total = first[batch], parts = active(p.grid, total);
  const bool idle = (int)blockIdx.x >= parts;
  const int w0 = idle ? 0 : share(blockIdx.x, parts, total), w1 = idle ? 0 : share(blockIdx.x + 1, parts, total);
  Cursor<true> cur;
  cur.seek(w0, lens, first, batch, blocks, nodes);

  // A wait that runs out makes all of the CTA's later ones give up at once. The
  // copies and the products stop there; the softmax warps go on to the end with
  // what they find, since they meet at barriers (the two warps of a row in every
  // tile, all of them at an item's ends) and one that left would keep the others.
  auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
    if (*(volatile int*)&abort_flag) return false;
    if (p.wait_once ? mbar_test_wait(b, parity) : mbar_wait_bounded(b, parity, nullptr)) return true;
    *(volatile int*)&abort_flag = 1;
    return false;
  };

  if (idle) {
  } else if (warp == kSoft / 32) {
    // ---- TMA producer ----
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; cur.w < w1; ++i) {
        const int st = i % NS;
        if (i >= NS && !wait(kv_empty + st, (uint32_t)((i / NS - 1) & 1))) break;
        uint8_t* ks = smem + st * 2 * C::kKvBytes;
        const bool fresh = cur.tile + 1 == cur.tiles;  // the drafted rows
        mbar_arrive_expect_tx(kv_full + st, 2 * C::kKvBytes);
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
          const int row = fresh ? 0 : cur.tile * kTile;
          tma_load_4d(ks + u * kSub, fresh ? &maps.kn : &maps.k, u * 64, row, cur.outer, cur.b, kv_full + st);
          tma_load_4d(ks + C::kKvBytes + u * kSub, fresh ? &maps.vn : &maps.v, u * 64, row, cur.outer, cur.b, kv_full + st);
        }
        issued = i + 1;
        cur.next(lens, batch, p.c.kv_heads, blocks, nodes);
      }
      // No copy may still be landing when the CTA exits.
      for (int i = max(0, issued - NS); i < issued; ++i) mbar_wait_bounded(kv_full + i % NS, (uint32_t)((i / NS) & 1), nullptr);
    }
  } else if (warp == kSoft / 32 + 1) {
    // ---- MMA issuer ----
    // The whole warp goes through it with the same values.
    auto all = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    auto wait_all = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
    const uint32_t tm = (uint32_t)all((int)tmem);
    // Descriptors differ in the start address alone (units of 16 bytes, which
    // do not carry out of their field): one add per product.
    const uint64_t dk0 = smem_desc_sw128(smem_u32(smem));
    const uint64_t dv0 = (dk0 & ~((uint64_t)0x3fff << 16)) | (uint64_t)(kSub / 16) << 16;  // LBO: the next 64 columns
    const uint32_t k_lo = (uint32_t)all((int)(uint32_t)dk0), k_hi = (uint32_t)(dk0 >> 32);
    const uint32_t v_lo = (uint32_t)all((int)(uint32_t)dv0), v_hi = (uint32_t)(dv0 >> 32);
    bool ok = true;
    auto issue_s = [&](int i) -> bool {
      const int st = i % NS, sb = i % kBufs;
      if (!wait_all(kv_full + st, (uint32_t)((i / NS) & 1))) return false;
      if (i >= kBufs && !wait_all(p_empty + sb, (uint32_t)((i / kBufs - 1) & 1))) return false;
      tc_fence_after();
      const uint32_t lo = k_lo + (uint32_t)(st * 2 * C::kKvBytes / 16), d = tm + (uint32_t)(sb * 64);
      if (elected()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma(d, tm + kColQ<D> + kk * 8, lo + ((kk >> 2) * kSub + (kk & 3) * 32) / 16, k_hi, idesc(64), kk != 0);
        mma_commit(s_full + sb);
      }
      __syncwarp();
      return true;
    };
    int i = 0;
    const int end = all(w1);
    int w = all(cur.w);
    for (int seg = 0; ok && w < end; ++seg) {
      const int n = all(min(cur.tiles - cur.tile, w1 - cur.w));  // tiles of the item's run
      if (!(ok = wait_all(q_full, (uint32_t)(seg & 1)))) break;
      for (int t = 0; ok && t < min(n, 2); ++t) ok = issue_s(i + t);
      for (int t = 0; ok && t < n; ++t, ++i) {
        const int st = i % NS, pb = i % kBufs, og = i & 1;
        if (!(ok = wait_all(p_full + pb, (uint32_t)((i / kBufs) & 1)))) break;
        // The next scores of the group that made these weights come first: it
        // has nothing else to do. Their buffer was the tile's before, whose
        // products are long done.
        if (t + 2 < n && !(ok = issue_s(i + 2))) break;
        tc_fence_after();
        const uint32_t lo = v_lo + (uint32_t)((st * 2 + 1) * C::kKvBytes / 16), d = tm + kColO + (uint32_t)(og * D);
        const uint32_t a = tm + (uint32_t)(pb * 64);
        if (elected()) {
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma(d, a + part * 32 + kk * 8, lo + kk * 2048 / 16, v_hi, idesc(D) | kMnMajorB, (part || kk) ? 1u : (uint32_t)(t >= 2));
          mma_commit(p_empty + pb);
          mma_commit(kv_empty + st);
        }
        __syncwarp();
      }
      if (ok && elected()) mma_commit(o_done);
      __syncwarp();
      // To the next item.
      cur.w += n - 1;
      cur.tile += n - 1;
      cur.next(lens, batch, p.c.kv_heads, blocks, nodes);
      w += n;
    }
    // Every product issued so far has retired before TMEM is released.
    if (elected()) mma_commit(drain);
    __syncwarp();
    mbar_wait_bounded(drain, 0, nullptr);
  } else {
    // ---- softmax ----
    const int row = tid & (kRows - 1), group = (tid >> 7) & 1, half = tid >> 8, part4 = group * 2 + half;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ocol = kColO + (uint32_t)(group * D + half * (D / 2));  // this thread's columns of O when it is scaled
    constexpr bool POW2 = !BIAS;
    // Not zero: it multiplies -inf.
    const float unit = fmaxf(fabsf(POW2 ? p.scale * kLog2e : p.scale), 1e-30f);
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;  // a negative scale is the queries'
    const int c0 = half * 32;  // first column of this thread's half
    auto weight = [](float x) { return ex2(POW2 ? x : x * kLog2e); };
    // The two threads of each row of this warp's quarter.
    auto row_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + group * 4 + (warp & 3)) : "memory"); };
    // One arrival per warp: 256 of them one after the other took longer than the
    // weights.
    auto warp_arrive = [&](uint64_t* b) {
      __syncwarp();
      if (lane == 0) arrive(b);
    };
    auto soft_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory"); };
    // The same barrier; whether `v` holds in all of the threads.
    auto soft_all = [](bool v) -> bool {
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.and.pred q, 1, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(all)
          : "r"((uint32_t)v), "n"(kSoft)
          : "memory");
      return all != 0;
    };
    bool ok = true;
    int i = 0, masks_of = -1;
    for (int seg = 0; cur.w < w1; ++seg) {
      const int n = min(cur.tiles - cur.tile, w1 - cur.w), first_tile = cur.tile, kvh = cur.outer, b = cur.b;
      const int len = max(cur.len, 0), row0 = cur.inner * kRows, here = min(kRows, rows - row0);
      const bool last = first_tile + n == cur.tiles, live = (warp & 3) * 32 < here;
      // The item's rows: into shared memory, and this thread's own.
      const int hd = (row0 + row) / nodes, nd = row0 + row - hd * nodes, head = kvh * heads_per + hd;
      // 32 columns of this row's query (head_dim 64: two threads have them all).
      const bool takes = D == 128 || half == 0;
      const int q_part = D == 128 ? part4 : group;
      const bf16* q = reinterpret_cast<const bf16*>(p.q.ptr) + b * p.q.sb + head * p.q.sh + nd * p.q.sn + q_part * 32;
      uint4 qv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        qv[e] = takes && row < here ? *reinterpret_cast<const uint4*>(q + 8 * e) : make_uint4(0, 0, 0, 0);
      const int next = p.c.next_pos ? p.c.next_pos[b] : len;
      if (takes) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[4 * e] = qv[e].x ^ flip;
          w[4 * e + 1] = qv[e].y ^ flip;
          w[4 * e + 2] = qv[e].z ^ flip;
          w[4 * e + 3] = qv[e].w ^ flip;
        }
        tmem_st16(tmem + lane_base + kColQ<D> + (uint32_t)(q_part * 16), w);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(q_full);
      // The masks, while the first scores are made.
      if (masks_of != b) {
        masks_of = b;
        if (warp == 0) node_masks(seen, p.parents ? p.parents + b * nodes : nullptr, nodes, cur.len >= 0, lane);
      }
      if (tid == 0) poison = 0;
      soft_sync();
      const unsigned long long see = row < here ? seen[nd] : 0ull;
      const int at = (int)((unsigned)next + (unsigned)(see ? __popcll(see) - 1 : 0));
      const float* tab = BIAS ? p.rel_bias + (row < here ? (int64_t)head * p.rel_len : 0) : nullptr;
      const float far = BIAS ? tab[p.rel_len - 1] : 0.f;
      const int32_t* ps = BIAS && p.c.pos ? p.c.pos + (int64_t)(b * p.c.kv_heads + kvh) * p.c.capacity : nullptr;

      float m = -INFINITY, l = 0.f;
      for (int t = (group ^ i) & 1; t < n; t += 2) {
        const int it = i + t, tile = first_tile + t, st = it % NS;
        const bool fresh = tile + 1 == cur.tiles;
        const int key0 = tile * kTile, valid = fresh ? nodes : len - key0;  // columns that exist
        // Positions of this half's keys, one per lane.
        int mine = 0;
        bool near = false;
        if (BIAS) {
          const int k = c0 + lane;
          if (fresh) {
            const unsigned long long s = k < nodes ? seen[k] : 0ull;
            mine = (int)((unsigned)next + (unsigned)(s ? __popcll(s) - 1 : 0));
          } else {
            mine = ps ? ps[min(key0 + k, max(len - 1, 0))] : key0 + k;
          }
          near = __any_sync(0xffffffffu, k < valid && (int)((unsigned)next - (unsigned)mine) < p.rel_len - 1);
        }
        const int buf = it % kBufs;
        // The TMEM accesses below are .sync.aligned: the warp goes on together.
        ok = __all_sync(0xffffffffu, ok && wait(s_full + buf, (uint32_t)((it / kBufs) & 1))) != 0;
        tc_fence_after();
        const uint32_t scores = tmem + lane_base + (uint32_t)(buf * 64);
        float x[32];
        if (live) {
          tmem_ld16(scores + (uint32_t)c0, reinterpret_cast<uint32_t*>(x));
          tmem_ld16(scores + (uint32_t)(c0 + 16), reinterpret_cast<uint32_t*>(x) + 16);
          tmem_wait_ld();
        }
        // Values that must not meet the products.
        const bool cleaned = fresh || (tile + 1) * kTile > len;
        if (cleaned) ok = __all_sync(0xffffffffu, ok && wait(kv_full + st, (uint32_t)((it / NS) & 1))) != 0;
        if (cleaned && ok) {
          uint8_t* vs = smem + st * 2 * C::kKvBytes + C::kKvBytes;
          for (int x4 = half * kRows + row; x4 < kTile * (D / 8); x4 += 2 * kRows) {
            const int r = x4 / (D / 8), ch = x4 % (D / 8);
            uint4* v4 = reinterpret_cast<uint4*>(vs + (ch >> 3) * kSub + sw128(r, ch & 7));
            if (!fresh) {
              if (key0 + r >= len) *v4 = make_uint4(0, 0, 0, 0);
            } else {
              uint4 v = *v4;
              uint32_t* w = reinterpret_cast<uint32_t*>(&v);
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u, bad = true;
                if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu, bad = true;
              }
              if (bad) {
                *v4 = v;
                if (r < nodes) atomicOr(&poison, 1ull << r);
              }
            }
          }
          fence_async();
        }
        if (live) {
          if (BIAS) {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] *= unit;
            if (near) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int pos = __shfl_sync(0xffffffffu, mine, e);
                x[e] += __ldg(tab + min(max((int)((unsigned)at - (unsigned)pos), 0), p.rel_len - 1));
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] += far;
            }
          }
          if (fresh) {
            const uint32_t bits = (uint32_t)(see >> c0);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(bits >> e & 1)) x[e] = -INFINITY;
          } else if (valid < kTile || !see) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c0 + e >= valid || !see) x[e] = -INFINITY;
          }
          float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int e = 4; e < 32; ++e) top[e & 3] = fmaxf(top[e & 3], x[e]);
          float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          // The row's: the other thread has its scores in registers, too, when
          // it tells its maximum, so the weights may take their place.
          const int slot = (it >> 1) & 1;
          tops[slot][group][half][row] = mt;
          row_sync();
          mt = fmaxf(mt, tops[slot][group][half ^ 1][row]);
          if (!BIAS) mt *= unit;  // x itself is scaled where its weight is taken
          float alpha = 1.f;
          bool scale = false;
          if (mt > m + kLazy) {  // also the first tile with a key (m = -inf)
            if (m != -INFINITY) {
              alpha = weight(m - mt);
              scale = true;
            }
            m = mt;
            l *= alpha;
          }
          if (__any_sync(0xffffffffu, scale)) {
            // O holds products made with the old maximum: scale it once the
            // last of them (this group's tile before) has retired.
            ok = __all_sync(0xffffffffu, ok && wait(p_empty + (it - 2) % kBufs, (uint32_t)(((it - 2) / kBufs) & 1))) != 0;
            tc_fence_after();
#pragma unroll
            for (int cc = 0; cc < D / 2; cc += 16) {
              uint32_t o[16];
              tmem_ld16(tmem + lane_base + ocol + (uint32_t)cc, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(tmem + lane_base + ocol + (uint32_t)cc, o);
            }
          }
          const float u = m == -INFINITY ? 0.f : m;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          // Into the place of the scores.
#pragma unroll
          for (int cc = 0; cc < 32; cc += 16) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = weight(BIAS ? x[cc + 2 * e] - u : fmaf(x[cc + 2 * e], unit, -u));
              const float d = weight(BIAS ? x[cc + 2 * e + 1] - u : fmaf(x[cc + 2 * e + 1], unit, -u));
              sum[e & 3] += a + d;
              hi[e] = pack_bf16(a, d);
              lo[e] = pack_bf16(a - __uint_as_float(hi[e] << 16), d - __uint_as_float(hi[e] & 0xffff0000u));
            }
            tmem_st8(scores + (uint32_t)((c0 + cc) / 2), hi);
            tmem_st8(scores + (uint32_t)(32 + (c0 + cc) / 2), lo);
          }
          tmem_wait_st();
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        tc_fence_before();
        warp_arrive(p_full + buf);
      }
      i += n;
      ok = __all_sync(0xffffffffu, ok && wait(o_done, (uint32_t)(seg & 1))) != 0;
      // Join the groups; every softmax thread passes here once per item.
      if (half == 0) xm[group][row] = m;
      xl[part4][row] = l;
      // A row's columns, its sum and its parts' joins go by several threads: where
      // one has given up, all of them write NaN (also where nothing was summed yet).
      ok = soft_all(ok);
      const float m0 = xm[0][row], m1 = xm[1][row], mx = fmaxf(m0, m1), u = mx == -INFINITY ? 0.f : mx;
      const float a0 = weight(m0 - u), a1 = weight(m1 - u), sum = (xl[0][row] + xl[1][row]) * a0 + (xl[2][row] + xl[3][row]) * a1;
      const float mn = POW2 ? mx * kLn2 : mx;
      const bool whole = first_tile == 0 && last, empty = !see || sum == 0.f;
      const unsigned long long bad = last ? poison & see : 0ull;
      if (live) {
        tc_fence_after();
        const float inv = !ok ? NAN : empty ? 0.f : whole ? 1.f / sum : 1.f;
        float* part = p.ws + (int64_t)(blockIdx.x * 2 + (first_tile == 0)) * kRows * (D + 2) + row * 4;
        bf16* out = row < here ? reinterpret_cast<bf16*>(const_cast<void*>(p.out.ptr)) + b * p.out.sb + head * p.out.sh + nd * p.out.sn
                               : nullptr;
        // A quarter of this row's columns.
#pragma unroll
        for (int cc = 0; cc < D / 4; cc += 16) {
          const int col = part4 * (D / 4) + cc;
          float o0[16], o1[16];
          tmem_ld16(tmem + lane_base + kColO + (uint32_t)col, reinterpret_cast<uint32_t*>(o0));
          tmem_ld16(tmem + lane_base + kColO + (uint32_t)(D + col), reinterpret_cast<uint32_t*>(o1));
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // A group that had no tile has no accumulator either.
            const float both = (m0 == -INFINITY ? 0.f : o0[e] * a0) + (m1 == -INFINITY ? 0.f : o1[e] * a1);
            o0[e] = empty && ok ? 0.f : both * inv;
          }
          for (unsigned long long s = bad; s; s &= s - 1) {
            const int j = __ffsll((long long)s) - 1;
            const bf16* vr = reinterpret_cast<const bf16*>(p.v_new.ptr) + b * p.v_new.sb + kvh * p.v_new.sh + j * p.v_new.sn + col;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float v = to_f(vr[e]);
              if (!(fabsf(v) < INFINITY)) o0[e] += v;
            }
          }
          if (row < here) {
            if (whole) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack_bf16(o0[2 * e], o0[2 * e + 1]);
              *reinterpret_cast<uint4*>(out + col) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(out + col + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<float4*>(part + (col + e) * kRows) = make_float4(o0[e], o0[e + 1], o0[e + 2], o0[e + 3]);
            }
          }
        }
        if (row < here && part4 == 0) {
          if (whole) {
            if (p.lse) p.lse[((int64_t)b * p.heads + head) * nodes + nd] = !ok ? NAN : empty ? -INFINITY : mn + logf(sum);
          } else {
            float* stat = p.ws + (int64_t)(blockIdx.x * 2 + (first_tile == 0)) * kRows * (D + 2) + kRows * D;
            stat[row] = empty ? -INFINITY : mn;
            stat[kRows + row] = !ok ? NAN : empty ? 0.f : sum;
          }
        }
      }
      tc_fence_before();
      soft_sync();  // xm, xl, seen and poison are used again
      cur.w += n - 1;
      cur.tile += n - 1;
      cur.next(lens, batch, p.c.kv_heads, blocks, nodes);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
  }
}

// A tensor map of (head_dim, rows, heads, batch) rows: boxes of 64 columns x 64
// rows, 128-byte swizzle, zeros outside. Strides of dimensions of one element
// are set to a row's bytes.
bool make_map(CUtensorMap* m, const void* base, int d, int64_t rows, int heads, int batch, int64_t sn, int64_t sh, int64_t sb) {
  auto fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t row = (cuuint64_t)d * 2;
  const cuuint64_t strides[3] = {sn ? (cuuint64_t)sn * 2 : row, sh ? (cuuint64_t)sh * 2 : row, sb ? (cuuint64_t)sb * 2 : row};
  const cuuint32_t box[4] = {64, 64, 1, 1}, step[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BIAS>
cudaError_t tc_run(const TreeParams& p, cudaStream_t s) {
  TcMaps maps;
  const CacheView& c = p.c;
  if (!make_map(&maps.k, c.k, D, c.capacity, c.kv_heads, c.batch, c.st, c.sh, c.sb) ||
      !make_map(&maps.v, c.v, D, c.capacity, c.kv_heads, c.batch, c.st, c.sh, c.sb) ||
      !make_map(&maps.kn, p.k_new.ptr, D, p.nodes, c.kv_heads, c.batch, p.k_new.sn, p.k_new.sh, p.k_new.sb) ||
      !make_map(&maps.vn, p.v_new.ptr, D, p.nodes, c.kv_heads, c.batch, p.v_new.sn, p.v_new.sh, p.v_new.sb))
    return cudaErrorInvalidValue;
  constexpr auto K = tree_attn_tc_kernel<D, BIAS>;
  constexpr int kMost = 216 * 1024;  // next to 8 KB of static shared memory
  static_assert(TcCfg<D>::kOffSched + (2 * kOpMaxBatch + 1) * 4 + 1024 <= kMost, "fits");
  cudaError_t e = allow_smem<K, kMost>();
  if (e != cudaSuccess) return e;
  K<<<p.grid, kTcThreads, TcCfg<D>::smem(c.batch), s>>>(maps, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = join_grid(p, kRows, D);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (2 * c.batch + 1) * 4;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_join_kernel<bf16, D, true>, p, kRows, join_by_item(p));
}

}  // namespace

// Strides that a tensor map takes: not zero where there is more than one
// element (an expanded tensor).
bool tree_attention_tc_takes(const TreeParams& p) {
  const CacheView& c = p.c;
  auto fits = [&](int64_t stride, int64_t extent) { return extent <= 1 || stride > 0; };
  return c.dtype != 0 && fits(c.st, c.capacity) && fits(c.sh, c.kv_heads) && fits(c.sb, c.batch) &&
         fits(p.k_new.sn, p.nodes) && fits(p.k_new.sh, c.kv_heads) && fits(p.k_new.sb, c.batch) && fits(p.v_new.sn, p.nodes) &&
         fits(p.v_new.sh, c.kv_heads) && fits(p.v_new.sb, c.batch);
}

void plan_tree_attention_tc(TreeParams& p, int sms, size_t* ws_floats) {
  const int rows = p.heads / p.c.kv_heads * p.nodes;
  p.row_blocks = (rows + kRows - 1) / kRows;
  const long long items = (long long)p.c.batch * p.c.kv_heads * p.row_blocks, most = (p.c.capacity + kTile - 1) / kTile + 1;
  p.stream = 1;
  p.grid = (int)min((long long)sms, max(1ll, items * most / 2));
  *ws_floats = (size_t)p.grid * 2 * kRows * (p.c.head_dim + 2);
}

cudaError_t launch_tree_attention_tc(const TreeParams& p, cudaStream_t s) {
  if (p.c.head_dim == 64) return p.rel_bias ? tc_run<64, true>(p, s) : tc_run<64, false>(p, s);
  return p.rel_bias ? tc_run<128, true>(p, s) : tc_run<128, false>(p, s);
}

}  // namespace mrtdf
