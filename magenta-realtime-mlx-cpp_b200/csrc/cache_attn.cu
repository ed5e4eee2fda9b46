// Attention of a tree of drafted tokens over a KV cache, and the attention
// weight that each cached row has collected.
//
// Tree attention. Node i of sequence b sits at depth d_i (its proper ancestors
// in the tree); row (head, i) sees every cached row t < len and the drafted
// rows of its ancestors and itself:
//   x_t = scale q . k_t + bias[head, clamp(next_pos + d_i - pos_t, 0, R - 1)]
//   out = sum_t exp(x_t - m) v_t / sum_t exp(x_t - m),  lse = m + ln sum
// in one pass over the rows with a running maximum m. All statistics and
// sums are float32.
//
// The work is bound by the cache: 2 head_dim elements per cached row are read
// for at most 64 x group queries. The nodes of one kv head's query heads are
// stacked to one operand of up to 64 rows (more: several blocks, which read
// the cache from L2 after the first). A CTA of four warps works on tiles of 64
// keys; WM warps share a key range with 16 rows each, and the 4 / WM key
// groups stream their own 16 * WM keys of each tile through a private
// cp.async ring, so a group waits for nobody until its item ends.
//
// Measured on a B200 (us in a graph; copies run at 6.57 TB/s):
//   128 sequences x 16 heads of 64, one token, 1006 rows, bf16, 527 MB: 90
//     (5.8 TB/s; four CTAs per SM are what the registers allow);
//   2 x 16 heads of 64, 16 nodes, 50 rows: 7.3. Latency: of the kernel's 6.3 us
//     the schedule takes 0.7, finding the run and asking for its first keys 1.3,
//     the queries 1.3, a tile 1 to 2 and the groups' join 0.5;
//   2 x 16 heads of 64, 8 nodes, 700 to 1006 rows, float32, 14 MB: 15.2, of which
//     the join of the split items is 3;
//   21 x 4 heads of 128, one token, 1334 rows, float32, 115 MB: 52 (2.2 TB/s:
//     bound by issue, a float32 product is three of tf32 and the splitting).
#include "cache_sched.cuh"

namespace mrtdf {
namespace {

constexpr int kStages = 3;

template <int WM>
__device__ __forceinline__ void group_sync(int group) {
  if constexpr (WM == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(WM * 32) : "memory");
}

__device__ __forceinline__ bool nonfinite(uint32_t w, __nv_bfloat16) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ bool nonfinite(uint32_t w, float) { return (w & 0x7f800000u) == 0x7f800000u; }

// Columns 8 n + 2 c, + 1 of value row `row`.
template <int D>
__device__ __forceinline__ float2 val2(uint32_t vals, int row, int n, int c, __nv_bfloat16) {
  const uint32_t w = lds32(vals + Rows<__nv_bfloat16, D>::at(row, n) + 4 * c);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <int D>
__device__ __forceinline__ float2 val2(uint32_t vals, int row, int n, int c, float) {
  const uint32_t at = vals + Rows<float, D>::at(row, 2 * n + (c >> 1)) + 8 * (c & 1);
  return make_float2(__uint_as_float(lds32(at)), __uint_as_float(lds32(at + 4)));
}

// Rows of 512 bytes (float32, 128): a tile's keys and values take 64 KB, three
// stages leave room for one CTA, whose four warps issue 1.1 instructions a
// clock. So the ring holds three halves there, the keys of a tile or its values,
// and the groups' sums are joined one after another: two CTAs fit (21 sequences
// x 4 heads x 1334 keys: 67 us with one, 52 with two).
template <typename T, int D>
constexpr bool halves() {
  return sizeof(T) * D == 512;
}

// Shared memory of the attention kernel.
template <typename T, int D, int WM>
struct TreeSmem {
  static constexpr bool HALVES = halves<T, D>();
  static constexpr int kStageBytes = (HALVES ? 1 : 2) * kTile * Rows<T, D>::kBytes;
  static constexpr int kMergeBytes = WM == 4 ? 0 : (HALVES ? 1 : 2) * 16 * D * 4;
  static constexpr int kScoreBytes = 16 * kTile * WM * 4;  // four warps x 16 rows x 16 WM keys
  static constexpr int kScratch = kMergeBytes > kScoreBytes ? kMergeBytes : kScoreBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kPos = kStages * kTile * 4;
  static constexpr int kStat = 4 * 32 * 16;        // four floats per lane
  static constexpr int kSeen = 4 * kOpMaxNodes * 8;
  static constexpr int kFixed = kRing + kScratch + kStat + kSeen + kPos;
  static int bytes(int batch) { return kFixed + (2 * batch + 1) * 4; }
};

// HALF: at most eight rows, so lanes' rows g + 8 do not exist. CTAs per SM
// follow the shared memory (56 KB: four of them, three with a bias, whose
// positions take the registers of the fourth).
template <typename T, int D, bool BIAS>
constexpr int tree_ctas() {
  return sizeof(T) * D == 128 ? (BIAS ? 3 : 4) : 2;
}
template <typename T, int D, int WM, bool BIAS, bool HALF>
__global__ __launch_bounds__(kThreads, tree_ctas<T, D, BIAS>()) void tree_attn_kernel(const __grid_constant__ TreeParams p) {
  using R = Rows<T, D>;
  using S = TreeSmem<T, D, WM>;
  constexpr int WK = 4 / WM, KT = 16 * WM, NT = KT / 8, MB = 16 * WM, ND = D / 8;
  constexpr int ROWS = HALF ? 2 : 4;  // a lane's scores of eight keys
  // bf16 scores without a bias are kept in powers of two (one multiply and one
  // add per weight). The others stay in natural units: a bias may be the
  // lowest float32, and float32 weights keep the last bits of x - m.
  constexpr bool POW2 = !BIAS && sizeof(T) == 2;
  const float unit = POW2 ? p.scale * kLog2e : p.scale;
  auto weight = [](float x) { return ex2(POW2 ? x : x * kLog2e); };
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* scratch = smem + S::kRing;
  float4* stat = reinterpret_cast<float4*>(scratch + S::kScratch);
  unsigned long long* seen_all = reinterpret_cast<unsigned long long*>(scratch + S::kScratch + S::kStat);
  int* pos_s = reinterpret_cast<int*>(scratch + S::kScratch + S::kStat + S::kSeen);
  int* lens = pos_s + kStages * kTile;
  int* first = lens + p.c.batch;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, group = warp / WM;
  const int g = lane >> 2, c = lane & 3, gt = wm * 32 + lane;
  unsigned long long* seen = seen_all + warp * kOpMaxNodes;
  const int batch = p.c.batch, blocks = p.row_blocks, items = p.c.kv_heads * blocks, nodes = p.nodes;
  const int heads_per = p.heads / p.c.kv_heads, rows = heads_per * nodes;
  // The grid is resident at once: the join may take its places beside it.
  pdl_launch_dependents();
  build_schedule<false>(p.c, batch, items, nodes, lens, first);

  // This CTA's run of tiles.
  const int total = first[batch];
  int w0, w1, parts;
  if (p.stream) {
    parts = active(p.grid, total);
    if ((int)blockIdx.x >= parts) return;
    w0 = share(blockIdx.x, parts, total);
    w1 = share(blockIdx.x + 1, parts, total);
  } else {
    const int all = batch * items, i0 = share(blockIdx.x, p.grid, all), i1 = share(blockIdx.x + 1, p.grid, all);
    parts = 0;
    if (i0 >= i1) return;
    auto start = [&](int i) {
      if (i == all) return total;
      const int b = i / items;
      return first[b] + (i - b * items) * tiles_of<false>(lens[b], nodes);
    };
    w0 = start(i0);
    w1 = start(i1);
  }

  constexpr bool HALVES = S::HALVES;
  const uint32_t ring = smem_u32(smem) + group * ((HALVES ? 1 : 2) * KT * R::kBytes);
  const T* kc = reinterpret_cast<const T*>(p.c.k);
  const T* vc = reinterpret_cast<const T*>(p.c.v);
  const T* kn = reinterpret_cast<const T*>(p.k_new.ptr);
  const T* vn = reinterpret_cast<const T*>(p.v_new.ptr);

  // Group's keys of the tile at `ahead` into ring stage `st`. A lane copies one
  // 16-byte chunk of rows r0, r0 + RS, ...: the rows' swizzle is a constant
  // apart (r0 < RS), so a chunk costs two 64-bit adds for its sources.
  constexpr int CH = R::kChunks, RS = WM * 32 / CH, COPIES = KT / RS;
  const int r0 = gt / CH, ch = gt % CH;
  const uint32_t x0 = (uint32_t)((ch ^ (r0 & 7)) << 4);
  const int64_t row_step = (int64_t)RS * p.c.st;
  Cursor<false> ahead;
  ahead.seek(w0, lens, first, batch, blocks, nodes);
  const T *kb = nullptr, *vb = nullptr;  // this lane's chunk of row 0 of ahead's item
  auto enter = [&] {
    const int64_t at = ahead.b * p.c.sb + ahead.outer * p.c.sh + ch * (16 / (int)sizeof(T));
    kb = kc + at;
    vb = vc + at;
  };
  // The tile's keys (with their positions, in place `ps_at`) to kd, its values to vd.
  auto copy = [&](uint32_t kd, uint32_t vd, int ps_at, bool keys, bool vals) {
    const int len = max(ahead.len, 0), key0 = ahead.tile * kTile + group * KT;
    kd += r0 * R::kBytes;
    vd += r0 * R::kBytes;
    if (key0 + KT <= len) {
      const int64_t at = (int64_t)(key0 + r0) * p.c.st;
      const T *ks = kb + at, *vs = vb + at;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const uint32_t to = i * RS * R::kBytes + (x0 ^ ((i * RS & 7) << 4));
        if (keys) cp_async16(kd + to, ks);
        if (vals) cp_async16(vd + to, vs);
        ks += row_step;
        vs += row_step;
      }
    } else {
#pragma unroll 2
      for (int i = 0; i < COPIES; ++i) {
        const int j = key0 + r0 + i * RS, n = min(j - len, nodes - 1), el = ch * (16 / (int)sizeof(T));
        const T* ks = j < len ? kb + j * p.c.st : kn + ahead.b * p.k_new.sb + ahead.outer * p.k_new.sh + n * p.k_new.sn + el;
        const T* vs = j < len ? vb + j * p.c.st : vn + ahead.b * p.v_new.sb + ahead.outer * p.v_new.sh + n * p.v_new.sn + el;
        const uint32_t to = i * RS * R::kBytes + (x0 ^ ((i * RS & 7) << 4));
        if (keys) cp_async16_zfill(kd + to, ks, j < len + nodes);
        if (vals) cp_async16_zfill(vd + to, vs, j < len + nodes);
      }
    }
    if (BIAS && p.c.pos && keys && gt < KT) {
      const int j = key0 + gt;
      const int32_t* ps = p.c.pos + (int64_t)(ahead.b * p.c.kv_heads + ahead.outer) * p.c.capacity;
      cp_async4_zfill(smem_u32(pos_s + ps_at * kTile + group * KT + gt), ps + min(j, max(len - 1, 0)), j < len);
    }
    if (vals && ahead.next(lens, batch, p.c.kv_heads, blocks, nodes)) enter();
  };
  auto fetch = [&](int st) {
    const uint32_t to = ring + st * S::kStageBytes;
    copy(to, to + KT * R::kBytes, st, true, true);
  };

  Cursor<false> cur = ahead;
  enter();
  // HALVES: slots of this tile's keys and values; the next tile's keys go where
  // the values before these were, its values where these keys are.
  int k_slot = 0, v_slot = 1, free_slot = 2, turn = 0;
  auto slot = [&](int i) { return ring + i * S::kStageBytes; };
  if (HALVES) {
    copy(slot(k_slot), 0, 0, true, false);
    cp_async_commit();
    copy(0, slot(v_slot), 0, false, true);
    cp_async_commit();
  } else {
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (ahead.w < w1) fetch(i);
      cp_async_commit();
    }
  }

  QFrag<T, D> q;
  float o[ND][4], m0 = 0, m1 = 0, l0 = 0, l1 = 0, far0 = 0, far1 = 0;
  unsigned long long see0 = 0, see1 = 0;
  const float *tab0 = nullptr, *tab1 = nullptr;
  int at0 = 0, at1 = 0, next = 0, masks_of = -1, first_tile = 0;
  bool fresh = true;

  for (int st = 0, fill = kStages - 1; cur.w < w1; cur.next(lens, batch, p.c.kv_heads, blocks, nodes)) {
    if (HALVES) {
      cp_async_wait<1>();  // the keys; the values are still on their way
      group_sync<WM>(group);
      if (ahead.w < w1) copy(slot(free_slot), 0, turn ^ 1, true, false);
    } else {
      cp_async_wait<kStages - 2>();
      group_sync<WM>(group);
      if (ahead.w < w1) fetch(fill);
    }
    cp_async_commit();
    const int len = max(cur.len, 0), kvh = cur.outer, row0 = cur.inner * MB + wm * 16;

    if (fresh) {  // a new item: its rows, statistics and masks
      fresh = false;
      first_tile = cur.tile;
      if (masks_of != cur.b) {
        masks_of = cur.b;
        __syncwarp();
        node_masks(seen, p.parents ? p.parents + cur.b * nodes : nullptr, nodes, cur.len >= 0, lane);
        next = p.c.next_pos ? p.c.next_pos[cur.b] : len;
      }
      const T *q0 = nullptr, *q1 = nullptr;
      see0 = see1 = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + g + 8 * h;
        if (r < rows) {
          const int hd = r / nodes, n = r - hd * nodes, head = kvh * heads_per + hd;
          const T* qr = reinterpret_cast<const T*>(p.q.ptr) + cur.b * p.q.sb + head * p.q.sh + n * p.q.sn;
          const unsigned long long s = seen[n];
          (h ? q1 : q0) = qr;
          (h ? see1 : see0) = s;
          if (BIAS) {
            const float* t = p.rel_bias + (int64_t)head * p.rel_len;
            (h ? tab1 : tab0) = t;
            (h ? at1 : at0) = (int)((unsigned)next + (unsigned)(__popcll(s) - (s ? 1 : 0)));
            (h ? far1 : far0) = t[p.rel_len - 1];
          }
        } else if (BIAS) {
          (h ? tab1 : tab0) = p.rel_bias;
        }
      }
      q.load(q0, q1, lane);
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    }

    const uint32_t keys = HALVES ? slot(k_slot) : ring + st * S::kStageBytes, vals = HALVES ? slot(v_slot) : keys + KT * R::kBytes;
    const int pos_at = (HALVES ? turn : st) * kTile + group * KT;
    const int key0 = cur.tile * kTile + group * KT;
    const bool any = key0 < len + nodes;  // for the whole group of warps
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    if (any) qk_tile<D, NT>(s, q, keys, lane);
    if (HALVES) {
      group_sync<WM>(group);  // the keys are read: the next tile's values
      if (ahead.w < w1) copy(0, slot(k_slot), 0, false, true);
      cp_async_commit();
      const int was = k_slot;
      k_slot = free_slot;
      free_slot = v_slot;
      v_slot = was;
      cp_async_wait<2>();
      group_sync<WM>(group);
    }
    if (any) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < ROWS; ++e) s[j][e] *= unit;

      const bool tail = key0 + KT > len;
      // Position of this lane's key 8 j + 2 c + e: stored, the slot, or the
      // drafted node's.
      auto key_pos = [&](int k) {
        const int key = key0 + k;
        if (key >= len) {
          const unsigned long long s = key - len < nodes ? seen[key - len] : 0ull;
          return (int)((unsigned)next + (unsigned)(__popcll(s) - (s ? 1 : 0)));
        }
        return p.c.pos ? pos_s[pos_at + k] : key;
      };
      if (BIAS) {
        int ps[NT][2];
        bool near = tail;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            ps[j][e] = key_pos(8 * j + 2 * c + e);
            near |= (int)((unsigned)next - (unsigned)ps[j][e]) < p.rel_len - 1;
          }
        if (__any_sync(0xffffffffu, near)) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d0 = min(max((int)((unsigned)at0 - (unsigned)ps[j][e]), 0), p.rel_len - 1);
              s[j][e] += __ldg(tab0 + d0);
              if (!HALF) {
                const int d1 = min(max((int)((unsigned)at1 - (unsigned)ps[j][e]), 0), p.rel_len - 1);
                s[j][2 + e] += __ldg(tab1 + d1);
              }
            }
        } else {  // every key is further than the table: its last entry
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            s[j][0] += far0;
            s[j][1] += far0;
            if (!HALF) {
              s[j][2] += far1;
              s[j][3] += far1;
            }
          }
        }
      }
      auto visible = [&](int key, unsigned long long see) {
        if (key < len) return see != 0;
        return key - len < nodes && (see >> (key - len) & 1) != 0;
      };
      if (tail) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + 8 * j + 2 * c + e;
            if (!visible(key, see0)) s[j][e] = -INFINITY;
            if (!HALF && !visible(key, see1)) s[j][2 + e] = -INFINITY;
          }
      }

      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
        if (!HALF) x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
      }
#pragma unroll
      for (int i = 1; i < 4; i <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, i));
        if (!HALF) x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, i));
      }
      if (__any_sync(0xffffffffu, x0 > m0 || (!HALF && x1 > m1))) {
        x0 = fmaxf(x0, m0);
        x1 = fmaxf(x1, m1);
        const float f0 = x0 == -INFINITY ? 1.f : weight(m0 - x0), f1 = x1 == -INFINITY ? 1.f : weight(m1 - x1);
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          o[n][0] *= f0;
          o[n][1] *= f0;
          o[n][2] *= f1;
          o[n][3] *= f1;
        }
        m0 = x0;
        m1 = x1;
      }
      // A row that has seen nothing keeps m = -inf; 0 stands in for it.
      const float u0 = m0 == -INFINITY ? 0.f : m0, u1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        s[j][0] = weight(s[j][0] - u0);
        s[j][1] = weight(s[j][1] - u0);
        l0 += s[j][0] + s[j][1];
        if (!HALF) {
          s[j][2] = weight(s[j][2] - u1);
          s[j][3] = weight(s[j][3] - u1);
          l1 += s[j][2] + s[j][3];
        }
      }

      // 0 x inf: where a drafted value row that some row must not see is not
      // finite, the products are added one by one, only where they count.
      bool odd = false;
      if (tail) {
        for (int i = lane; i < KT * R::kBytes / 4; i += 32) odd |= nonfinite(lds32(vals + 4 * i), T());
        odd = __any_sync(0xffffffffu, odd);
      }
      if (odd) {
        float* ps = reinterpret_cast<float*>(scratch) + warp * (16 * KT);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) ps[(g + 8 * (e >> 1)) * KT + 8 * j + 2 * c + (e & 1)] = s[j][e];
        __syncwarp();
        for (int k = 0; k < KT; ++k) {
          const bool v0 = visible(key0 + k, see0), v1 = visible(key0 + k, see1);
          const float p0 = ps[g * KT + k], p1 = ps[(g + 8) * KT + k];
#pragma unroll
          for (int n = 0; n < ND; ++n) {
            const float2 v = val2<D>(vals, k, n, c, T());
            if (v0) {
              o[n][0] += p0 * v.x;
              o[n][1] += p0 * v.y;
            }
            if (v1) {
              o[n][2] += p1 * v.x;
              o[n][3] += p1 * v.y;
            }
          }
        }
        __syncwarp();
      } else {
        pv_tile<D, NT, HALF>(o, s, vals, lane, T());
      }
    }
    st = st + 1 == kStages ? 0 : st + 1;
    fill = fill + 1 == kStages ? 0 : fill + 1;
    turn ^= 1;

    if (cur.tile + 1 < cur.tiles && cur.w + 1 < w1) continue;
    // ---- the item's run ends here: join the key groups, write ----------------
    fresh = true;
#pragma unroll
    for (int i = 1; i < 4; i <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, i);
      l1 += __shfl_xor_sync(0xffffffffu, l1, i);
    }
    if constexpr (WK > 1) {
      float4* buf = reinterpret_cast<float4*>(scratch);
      __syncthreads();  // nobody still reads scores or an earlier join there
      // Half of the groups to the other half, or (HALVES) one after another,
      // the columns in two parts where two warps share a group.
      constexpr bool BY_ONE = HALVES && WM == 1;
      constexpr int PARTS = HALVES && WM == 2 ? 2 : 1, NP = ND / PARTS;
#pragma unroll
      for (int step = BY_ONE ? WK - 1 : WK / 2; step >= 1; BY_ONE ? --step : step >>= 1) {
        const bool gives = BY_ONE ? group == step : group >= step && group < 2 * step;
        const bool takes = BY_ONE ? group == 0 : group < step;
        const int at = BY_ONE ? 0 : (group % step) * WM + wm;
        float a0 = 0, a1 = 0, b0 = 0, b1 = 0;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          if (gives) {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
              const float* v = o[part * NP + n];
              buf[(at * NP + n) * 32 + lane] = make_float4(v[0], v[1], v[2], v[3]);
            }
            stat[at * 32 + lane] = make_float4(m0, m1, l0, l1);
          }
          __syncthreads();
          if (takes) {
            if (part == 0) {
              const float4 t = stat[at * 32 + lane];
              const float x0 = fmaxf(m0, t.x), x1 = fmaxf(m1, t.y);
              const float u0 = x0 == -INFINITY ? 0.f : x0, u1 = x1 == -INFINITY ? 0.f : x1;
              a0 = weight(m0 - u0);
              a1 = weight(m1 - u1);
              b0 = weight(t.x - u0);
              b1 = weight(t.y - u1);
              l0 = l0 * a0 + t.z * b0;
              l1 = l1 * a1 + t.w * b1;
              m0 = x0;
              m1 = x1;
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
              const float4 v = buf[(at * NP + n) * 32 + lane];
              float* to = o[part * NP + n];
              to[0] = to[0] * a0 + v.x * b0;
              to[1] = to[1] * a0 + v.y * b0;
              to[2] = to[2] * a1 + v.z * b1;
              to[3] = to[3] * a1 + v.w * b1;
            }
          }
          __syncthreads();
        }
      }
    }
    if (group == 0) {
      const bool whole = first_tile == 0 && cur.tile + 1 == cur.tiles;
      if (POW2) {  // partial rows and lse are in natural units
        m0 *= kLn2;
        m1 *= kLn2;
      }
      if (!see0) {
        m0 = -INFINITY;
        l0 = 0.f;
      }
      if (!see1) {
        m1 = -INFINITY;
        l1 = 0.f;
      }
      if (whole) {
#pragma unroll
        for (int h = 0; h < ROWS / 2; ++h) {
          const int r = row0 + g + 8 * h;
          if (r >= rows) continue;
          const int hd = r / nodes, n = r - hd * nodes, head = kvh * heads_per + hd;
          const float l = h ? l1 : l0, m = h ? m1 : m0, inv = l == 0.f ? 0.f : 1.f / l;
          T* dst = reinterpret_cast<T*>(const_cast<void*>(p.out.ptr)) + cur.b * p.out.sb + head * p.out.sh + n * p.out.sn;
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const float a = h ? o[i][2] : o[i][0], b = h ? o[i][3] : o[i][1];
            store2(dst + 8 * i + 2 * c, l == 0.f ? 0.f : a * inv, l == 0.f ? 0.f : b * inv);
          }
          if (p.lse && c == 0)
            p.lse[((int64_t)cur.b * p.heads + head) * nodes + n] = l == 0.f ? -INFINITY : m + logf(l);
        }
      } else {
        // Slot 1: a run that starts an item; slot 0: one that goes on with it.
        float* part = p.ws + (int64_t)(blockIdx.x * 2 + (first_tile == 0)) * MB * (D + 2);
#pragma unroll
        for (int h = 0; h < ROWS / 2; ++h) {
          const int r = wm * 16 + g + 8 * h;
#pragma unroll
          for (int i = 0; i < ND; ++i)
            store2(part + ((2 * i + (c >> 1)) * MB + r) * 4 + 2 * (c & 1), h ? o[i][2] : o[i][0], h ? o[i][3] : o[i][1]);
          if (c == 0) {
            part[MB * D + r] = h ? m1 : m0;
            part[MB * D + MB + r] = h ? l1 : l0;
          }
        }
      }
    }
  }
}

// ---- collected weight ------------------------------------------------------------
// mass_out[t] = decay mass[t] + sum over the accepted path's rows (head, i) of
// exp(x_t - lse) for cached rows t < len, and for the path's own rows, which
// commit will put at len + j, the sum over i >= j. The softmax statistics come
// from the attention (lse), so only the keys are read again: head_dim elements
// and 8 bytes of weight per cached row bound it. A warp owns 16 keys of a tile
// and sums its columns over all rows, so every sum has one owner and one order.
// 2 layers x 8 sequences x 8 kv heads x 3001 to 8190 rows of 128, bf16, five
// nodes of four heads each: 41 us for 190 MB (4.7 TB/s; the exponentials of 32
// padded rows, of which 20 count, go beside the keys; with the weights so far
// asked for in the tile that adds to them, 50 us); with a bias and stored positions
// 57; 2 x 16 heads of 64 over 250 rows, float32: 6.9 us, latency.
constexpr int kMassRows = 64;  // query rows held in shared memory at a time

// Rows of 512 bytes: two stages, so that two CTAs fit an SM.
template <typename T, int D>
struct MassSmem {
  static constexpr int kStages = sizeof(T) * D == 512 ? 2 : 3;
  static constexpr int kStageBytes = kTile * Rows<T, D>::kBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kQ = kMassRows * Rows<T, D>::kBytes;
  static constexpr int kFixed = kRing + kQ + kStages * kTile * 4 + 3 * kMassRows * 4 + kOpMaxNodes * 4;
  static int bytes(int batch) { return kFixed + (2 * batch + 1) * 4; }
};

// Row fragments from shared memory rows in the key layout.
template <int D>
__device__ __forceinline__ void q_from_smem(QFrag<__nv_bfloat16, D>& q, uint32_t base, int lane) {
  const int m = lane >> 3, r = lane & 7;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    ldsm_x4_g(q.a[ks], base + Rows<__nv_bfloat16, D>::at((m & 1) * 8 + r, 2 * ks + (m >> 1)));
}
template <int D>
__device__ __forceinline__ void q_from_smem(QFrag<float, D>& q, uint32_t base, int lane) {
  const int m = lane >> 3, r = lane & 7;
#pragma unroll
  for (int ks = 0; ks < D / 8; ++ks)
    ldsm_x4_g(q.a[ks], base + Rows<float, D>::at((m & 1) * 8 + r, 2 * ks + (m >> 1)));
}

// CTAs per SM, by shared memory (67 KB for bf16 rows of 128: three).
template <typename T, int D>
constexpr int mass_ctas() {
  return sizeof(T) * D == 128 ? 4 : sizeof(T) * D == 256 ? 3 : 2;
}
template <typename T, int D, bool BIAS>
__global__ __launch_bounds__(kThreads, mass_ctas<T, D>()) void cache_mass_kernel(const __grid_constant__ MassParams p) {
  using R = Rows<T, D>;
  using S = MassSmem<T, D>;
  constexpr int kStages = S::kStages;
  // As in the attention: powers of two where the last bits do not matter.
  constexpr bool POW2 = !BIAS && sizeof(T) == 2;
  const float unit = POW2 ? p.scale * kLog2e : p.scale;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* q_s = smem + S::kRing;
  int* pos_s = reinterpret_cast<int*>(q_s + S::kQ);
  float* lse_s = reinterpret_cast<float*>(pos_s + kStages * kTile);
  int* node_s = reinterpret_cast<int*>(lse_s + kMassRows);  // of each row: its place on the path,
  int* head_s = node_s + kMassRows;                         // its query head of the kv head
  int* path_s = head_s + kMassRows;
  int* lens = path_s + kOpMaxNodes;
  int* first = lens + p.c.batch;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int batch = p.c.batch, kv = p.c.kv_heads, items = p.c.layers * kv, extra = p.path_len;
  const int heads_per = p.heads / p.c.kv_heads;
  build_schedule<false>(p.c, batch, items, extra, lens, first);
  const int total = first[batch], parts = active(p.grid, total);
  if ((int)blockIdx.x >= parts) return;
  const int w0 = share(blockIdx.x, parts, total), w1 = share(blockIdx.x + 1, parts, total);
  const uint32_t ring = smem_u32(smem) + warp * (16 * R::kBytes);

  Cursor<false> cur;
  cur.seek(w0, lens, first, batch, kv, extra);
  while (cur.w < w1) {
    // One item's run of tiles [t0, t1): layer, sequence, kv head.
    const int layer = cur.outer, kvh = cur.inner, b = cur.b;
    const int t0 = cur.tile, t1 = min(cur.tiles, cur.tile + (w1 - cur.w)), len = max(cur.len, 0);
    const bool there = cur.len >= 0;
    __syncthreads();  // the item before is done with the path and the rows
    int count = 0;
    if (there) count = accepted(p.path + b * p.path_len, p.path_len, p.nodes, p.c.capacity - len, lane);
    for (int i = tid; i < p.path_len; i += kThreads) path_s[i] = i < count ? p.path[b * p.path_len + i] : 0;
    const int rows = heads_per * count, next = p.c.next_pos ? p.c.next_pos[b] : len;
    const int64_t row_at = ((int64_t)(layer * batch + b) * p.c.kv_heads + kvh) * p.c.capacity;
    const T* kb = reinterpret_cast<const T*>(p.c.k) + layer * p.c.sl + b * p.c.sb + kvh * p.c.sh;
    const T* kn = reinterpret_cast<const T*>(p.k_new.ptr) + layer * p.k_new.sl + b * p.k_new.sb + kvh * p.k_new.sh;
    __syncthreads();

    // As in tree_attn_kernel: a lane copies one chunk of every RS-th row.
    constexpr int CH = R::kChunks, RS = 32 / CH;
    const int r0 = lane / CH, ch = lane % CH, el = ch * (16 / (int)sizeof(T));
    const uint32_t x0 = (uint32_t)((ch ^ (r0 & 7)) << 4);
    const T* kl = kb + el;
    auto fetch = [&](int tile, int st) {
      const int key0 = tile * kTile + warp * 16;
      const uint32_t kd = ring + st * S::kStageBytes + r0 * R::kBytes;
      if (key0 + 16 <= len && rows > 0) {
        const T* ks = kl + (int64_t)(key0 + r0) * p.c.st;
#pragma unroll
        for (int i = 0; i < 16 / RS; ++i) {
          cp_async16(kd + i * RS * R::kBytes + (x0 ^ ((i * RS & 7) << 4)), ks);
          ks += RS * p.c.st;
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < 16 / RS; ++i) {
          const int j = key0 + r0 + i * RS;
          const T* ks = j < len ? kl + j * p.c.st : kn + path_s[min(j - len, p.path_len - 1)] * p.k_new.sn + el;
          cp_async16_zfill(kd + i * RS * R::kBytes + (x0 ^ ((i * RS & 7) << 4)), ks, rows > 0 && j < len + count);
        }
      }
      if (BIAS && p.c.pos && lane < 16) {
        const int j = key0 + lane;
        cp_async4_zfill(smem_u32(pos_s + st * kTile + warp * 16 + lane), p.c.pos + row_at + min(j, max(len - 1, 0)), j < len);
      }
    };

    // Rows in blocks of 64 (one block where the path is empty: the decay).
    for (int rb = 0; rb == 0 || rb < rows; rb += kMassRows) {
      const int here = min(kMassRows, rows - rb);
      if (rb) __syncthreads();
      for (int i = tid; i < kMassRows * R::kChunks; i += kThreads) {
        const int row = i / R::kChunks, ch = i % R::kChunks, r = rb + row;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (ch == 0) {  // a row that does not exist: weights of exp(-inf)
          lse_s[row] = INFINITY;
          node_s[row] = head_s[row] = 0;
        }
        if (row < here) {
          const int hd = r / count, at = r - hd * count, n = path_s[at], head = kvh * heads_per + hd;
          v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q.ptr) + layer * p.q.sl + b * p.q.sb +
                                              head * p.q.sh + n * p.q.sn + ch * (16 / sizeof(T)));
          if (ch == 0) {
            // A row whose softmax is empty (lse = -inf) gives nothing either.
            const float lse = p.lse[((int64_t)(layer * batch + b) * p.heads + head) * p.nodes + n];
            lse_s[row] = lse == -INFINITY ? INFINITY : POW2 ? lse * kLog2e : lse;
            node_s[row] = at;
            head_s[row] = hd;
          }
        }
        *reinterpret_cast<uint4*>(q_s + R::at(row, ch)) = v;
      }
      for (int i = 0; i < kStages - 1; ++i) {
        if (t0 + i < t1) fetch(t0 + i, i);
        cp_async_commit();
      }
      __syncthreads();
      QFrag<T, D> q;
      if (here <= 16) q_from_smem<D>(q, smem_u32(q_s), lane);

      // A lane's weights so far, keys 8 j + 2 c + e of a tile, in the lanes with
      // g = 0: asked for a tile ahead.
      auto before = [&](int t, float (*to)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = t * kTile + warp * 16 + 8 * j + 2 * c + e;
            to[j][e] = 0.f;
            if (g == 0 && t < t1 && there && key < (rb ? len + count : len)) to[j][e] = (rb ? p.mass_out : p.mass)[row_at + key];
          }
      };
      const float decay = rb ? 1.f : p.decay;
      float ahead[2][2];
      before(t0, ahead);
      for (int t = t0, st = 0, fill = kStages - 1; t < t1; ++t) {
        float old[2][2] = {{ahead[0][0], ahead[0][1]}, {ahead[1][0], ahead[1][1]}};
        before(t + 1, ahead);
        cp_async_wait<kStages - 2>();
        __syncwarp();
        if (t + kStages - 1 < t1) fetch(t + kStages - 1, fill);
        cp_async_commit();
        const int key0 = t * kTile + warp * 16;
        const uint32_t keys = ring + st * S::kStageBytes;
        float col[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        const bool tail = key0 + 16 > len;
        for (int mt = 0; mt * 16 < here; ++mt) {
          if (here > 16) q_from_smem<D>(q, smem_u32(q_s) + mt * 16 * R::kBytes, lane);
          float s[2][4] = {};
          qk_tile<D, 2>(s, q, keys, lane);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = mt * 16 + g + 8 * h, i = BIAS || tail ? node_s[row] : 0;
            const float lse = lse_s[row];
            // A row that gives nothing is left out by a choice: its weight would
            // be exp(x - inf), NaN where a key makes x one (0 x inf among them).
            const bool gives = lse != INFINITY;
            const float* tab = BIAS ? p.rel_bias + (int64_t)(kvh * heads_per + head_s[row]) * p.rel_len : nullptr;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int k = 8 * j + 2 * c + e;
                float x = s[j][2 * h + e] * unit;
                if (BIAS) {
                  const int at = key0 + k >= len ? next + (key0 + k - len)
                                 : p.c.pos       ? pos_s[st * kTile + warp * 16 + k]
                                                 : key0 + k;
                  x += __ldg(tab + min(max((int)((unsigned)(next + i) - (unsigned)at), 0), p.rel_len - 1));
                }
                const float w = ex2(POW2 ? x - lse : (x - lse) * kLog2e);
                col[j][e] += gives && (!tail || key0 + k - len <= i) ? w : 0.f;
              }
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) col[j][e] += __shfl_xor_sync(0xffffffffu, col[j][e], o);
            const int key = key0 + 8 * j + 2 * c + e;
            if (g == 0 && key < len + count && there)
              p.mass_out[row_at + key] = (rb || key < len ? decay * old[j][e] : 0.f) + col[j][e];
          }
        st = st + 1 == kStages ? 0 : st + 1;
        fill = fill + 1 == kStages ? 0 : fill + 1;
      }
      cp_async_wait<0>();
    }
    // To the next item.
    cur.w += t1 - t0;
    if (t1 == cur.tiles && cur.w < w1) {
      cur.w -= 1;
      cur.tile = cur.tiles - 1;
      cur.next(lens, batch, p.c.layers, kv, extra);
    }
  }
}

// ---- host --------------------------------------------------------------------------
template <typename T, int D, int WM, bool BIAS, bool HALF>
cudaError_t tree_run(const TreeParams& p, cudaStream_t s) {
  constexpr auto K = tree_attn_kernel<T, D, WM, BIAS, HALF>;
  static_assert(TreeSmem<T, D, WM>::kFixed + (2 * kOpMaxBatch + 1) * 4 <= kOpMaxSmem, "fits");
  const int bytes = TreeSmem<T, D, WM>::bytes(p.c.batch);
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  K<<<p.grid, kThreads, bytes, s>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess || !p.stream) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = join_grid(p, 16 * WM, D);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (2 * p.c.batch + 1) * 4;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_join_kernel<T, D, false>, p, 16 * WM, join_by_item(p));
}

template <typename T, int D, bool BIAS>
cudaError_t tree_variant(const TreeParams& p, int wm, cudaStream_t s) {
  if (p.heads / p.c.kv_heads * p.nodes <= 8) return tree_run<T, D, 1, BIAS, true>(p, s);
  if constexpr (sizeof(T) == 2)
    if (wm == 4) return tree_run<T, D, 4, BIAS, false>(p, s);
  return wm == 1 ? tree_run<T, D, 1, BIAS, false>(p, s) : tree_run<T, D, 2, BIAS, false>(p, s);
}
template <typename T, int D>
cudaError_t tree_variant(const TreeParams& p, int wm, cudaStream_t s) {
  return p.rel_bias ? tree_variant<T, D, true>(p, wm, s) : tree_variant<T, D, false>(p, wm, s);
}

// Warps that share a key range: one per 16 query rows, up to four. float32: up
// to two, since each takes all the keys apart for its products (96 rows of 128
// x 1334 keys, 21 sequences of 4 heads: 381 us with four, 220 with two).
int tree_wm(const TreeParams& p) {
  const int rows = p.heads / p.c.kv_heads * p.nodes;
  return rows <= 16 ? 1 : rows <= 32 || p.c.dtype == 0 ? 2 : 4;
}
int tree_smem(const TreeParams& p, int wm) {
  const int b = p.c.batch;
  const bool f = p.c.dtype == 0;
  if (p.c.head_dim == 64) {
    if (f) return wm == 1 ? TreeSmem<float, 64, 1>::bytes(b) : TreeSmem<float, 64, 2>::bytes(b);
    return wm == 1 ? TreeSmem<__nv_bfloat16, 64, 1>::bytes(b) : wm == 2 ? TreeSmem<__nv_bfloat16, 64, 2>::bytes(b) : TreeSmem<__nv_bfloat16, 64, 4>::bytes(b);
  }
  if (f) return wm == 1 ? TreeSmem<float, 128, 1>::bytes(b) : TreeSmem<float, 128, 2>::bytes(b);
  return wm == 1 ? TreeSmem<__nv_bfloat16, 128, 1>::bytes(b) : wm == 2 ? TreeSmem<__nv_bfloat16, 128, 2>::bytes(b) : TreeSmem<__nv_bfloat16, 128, 4>::bytes(b);
}

constexpr int kSmSmem = 227 * 1024;
// Which bf16 calls the tcgen05 kernel takes. us, mma.sync / tcgen05, 16
// sequences of 4 kv heads without a bias (which costs the first 1.2 to 1.8
// times as much, the second 1.1 times):
//                    32 rows      64 rows      128 rows     256 rows
//   64 x   300     13.2/ 16.4   16.7/ 17.5    19.7/ 20.8   31.1/ 24.3
//   64 x  1024     17.5/ 19.7   23.1/ 21.2    28.6/ 24.6   42.8/ 32.4
//   64 x  4096     27.2/ 33.8   39.9/ 37.9    60.5/ 41.3    106/ 65
//   64 x 16384     63.9/ 88.1    104/ 103      188/ 106     356/ 194
//  128 x   300     16.7/ 22.6   21.3/ 23.7    26.3/ 27.1   46.6/ 34.5
//  128 x  1024     22.0/ 26.8   30.2/ 28.2    44.0/ 31.7   75.0/ 43.9
//  128 x  4096     47.3/ 47.9   67.8/ 51.8     116/ 56      217/ 85
//  128 x 16384      139/ 112     207/ 125      396/ 131     773/ 239
// (256 kv heads alike; head_dim 64 and 64 rows even out there.) The rule goes by
// capacity, since lengths are not known on the host: a long buffer that is mostly
// empty is priced as a full one.
bool tree_uses_tc(const TreeParams& p, int rows) {
  const int cap = p.c.capacity;
  if (rows > 64) return cap > 512;
  if (rows > 32) return cap > (p.c.head_dim == 128 ? 768 : 2048);
  return rows > 16 && p.c.head_dim == 128 && cap > 4096;
}

}  // namespace

cudaError_t plan_tree_attention(TreeParams& p, int sms, size_t* ws_floats) {
  const int wm = tree_wm(p), mb = 16 * wm, rows = p.heads / p.c.kv_heads * p.nodes;
  p.tc = tree_uses_tc(p, rows) && tree_attention_tc_takes(p);
  if (p.tc) {
    plan_tree_attention_tc(p, sms, ws_floats);
    return cudaSuccess;
  }
  p.row_blocks = (rows + mb - 1) / mb;
  const int items = p.c.batch * p.c.kv_heads * p.row_blocks;
  const int per_sm = max(1, min(p.rel_bias && p.c.dtype != 0 ? 3 : 4, kSmSmem / (tree_smem(p, wm) + 1024)));
  const int slots = sms * per_sm, most = (p.c.capacity + p.nodes + kTile - 1) / kTile;
  // Short caches: an item is a few tiles, whole items per CTA need no join.
  p.stream = most > 4;
  p.grid = p.stream ? (int)min((long long)slots, max(1ll, (long long)items * most / 2)) : min(items, slots);
  *ws_floats = p.stream ? (size_t)p.grid * 2 * mb * (p.c.head_dim + 2) : 0;
  return cudaSuccess;
}

cudaError_t launch_tree_attention(const TreeParams& p, cudaStream_t s) {
  if (p.tc) return launch_tree_attention_tc(p, s);
  const int wm = tree_wm(p);
  if (p.c.dtype == 0) return p.c.head_dim == 64 ? tree_variant<float, 64>(p, wm, s) : tree_variant<float, 128>(p, wm, s);
  return p.c.head_dim == 64 ? tree_variant<__nv_bfloat16, 64>(p, wm, s) : tree_variant<__nv_bfloat16, 128>(p, wm, s);
}

namespace {
template <typename T, int D, bool BIAS>
cudaError_t mass_run(MassParams& p, cudaStream_t s) {
  constexpr auto K = cache_mass_kernel<T, D, BIAS>;
  const int bytes = MassSmem<T, D>::bytes(p.c.batch);
  cudaError_t e = allow_smem<K>();
  if (e != cudaSuccess) return e;
  int dev = 0;
  e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const int per_sm = max(1, min(mass_ctas<T, D>(), kSmSmem / (bytes + 1024)));
  const long long most = (long long)p.c.batch * p.c.layers * p.c.kv_heads * ((p.c.capacity + p.path_len + kTile - 1) / kTile);
  p.grid = (int)min((long long)op_sm_count(dev) * per_sm, max(1ll, most / 2));
  K<<<p.grid, kThreads, bytes, s>>>(p);
  return cudaGetLastError();
}
template <typename T, int D>
cudaError_t mass_variant(MassParams& p, cudaStream_t s) {
  return p.rel_bias ? mass_run<T, D, true>(p, s) : mass_run<T, D, false>(p, s);
}
}  // namespace

cudaError_t launch_cache_mass(MassParams& p, cudaStream_t s) {
  if (p.c.dtype == 0) return p.c.head_dim == 64 ? mass_variant<float, 64>(p, s) : mass_variant<float, 128>(p, s);
  return p.c.head_dim == 64 ? mass_variant<__nv_bfloat16, 64>(p, s) : mass_variant<__nv_bfloat16, 128>(p, s);
}

}  // namespace mrtdf
