// How the attention over a cache is spread over the GPU, shared by its kernels
// (cache_attn.cu, cache_attn_tc.cu): a list of key tiles of all (sequence, kv
// head, row block) items, equal runs of it per CTA, the drafted tree's masks,
// the accepted path (cache_move.cu reads it too), and the join of items that
// several CTAs worked on.
#pragma once

#include "cache_ops.cuh"
#include "cache_tile.cuh"

namespace mrtdf {

constexpr int kTile = 64;      // keys per CTA tile
constexpr int kThreads = 128;  // four warps

// ---- schedule ----------------------------------------------------------------
// A sequence's tiles: ceil((len + nodes) / 64), or with APART the drafted rows
// in a tile of their own behind ceil(len / 64); at least one. A length outside
// [0, capacity] makes the sequence empty (len -1 here).
__device__ __forceinline__ int checked_len(const CacheView& c, int b) {
  const int l = c.lens[b];
  return l < 0 || l > c.capacity ? -1 : l;
}
template <bool APART>
__device__ __forceinline__ int tiles_of(int len, int extra) {
  return (max(len, 0) + (APART ? kTile : extra) + kTile - 1) / kTile;
}

// lens[b] and first[b] = tiles of all items before sequence b's, for b <= B.
// All threads of the block; the first 128 do the work; ends with a barrier.
template <bool APART>
__device__ void build_schedule(const CacheView& c, int batch, int items, int extra, int* lens, int* first) {
  __shared__ int warp_sum[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, per = (batch + kThreads - 1) / kThreads;
  int sum = 0;
  for (int i = 0; i < per && tid < kThreads; ++i) {
    const int b = tid * per + i;
    if (b < batch) {
      const int l = checked_len(c, b);
      lens[b] = l;
      sum += tiles_of<APART>(l, extra) * items;
    }
  }
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31 && tid < kThreads) warp_sum[tid >> 5] = run;
  __syncthreads();
  run -= sum;
  for (int w = 0; w < (tid >> 5) && tid < kThreads; ++w) run += warp_sum[w];
  for (int i = 0; i < per && tid < kThreads; ++i) {
    const int b = tid * per + i;
    if (b < batch) {
      first[b] = run;
      run += tiles_of<APART>(lens[b], extra) * items;
      if (b == batch - 1) first[batch] = run;
    }
  }
  __syncthreads();
}

// Position in the list of tiles: sequence-major, then outer, inner (an item is
// one pair of them), then tile.
template <bool APART>
struct Cursor {
  int w, b, outer, inner, tile, tiles, len;
  __device__ __forceinline__ void seek(int at, const int* lens, const int* first, int batch, int inners, int extra) {
    w = at;
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    len = lens[b];
    tiles = tiles_of<APART>(len, extra);
    const int rem = at - first[b], item = rem / tiles;
    tile = rem - item * tiles;
    outer = item / inners;
    inner = item - outer * inners;
  }
  // True when the next tile is another item's.
  __device__ __forceinline__ bool next(const int* lens, int batch, int outers, int inners, int extra) {
    ++w;
    if (++tile < tiles) return false;
    tile = 0;
    if (++inner == inners) {
      inner = 0;
      if (++outer == outers) {
        outer = 0;
        if (++b < batch) {
          len = lens[b];
          tiles = tiles_of<APART>(len, extra);
        }
      }
    }
    return true;
  }
};

// CTA c of g takes tiles [share(c), share(c + 1)) of `total`.
__device__ __forceinline__ int share(int c, int g, int total) { return (int)((long long)c * total / g); }
// The CTA whose run holds tile w.
__device__ __forceinline__ int owner(int w, int g, int total) {
  return (int)((((long long)w + 1) * g - 1) / total);
}
// CTAs that take part: a run has two tiles or more, or there is one tile each.
__device__ __forceinline__ int active(int grid, int total) { return max(1, min(grid, total / 2)); }

// ---- the tree ------------------------------------------------------------------
// seen[i]: bit j set when node j is node i or an ancestor; 0 for a node that is
// absent (its chain holds a parent outside [-1, i)). One warp; pointer
// doubling: after k rounds a node knows 2^k links of its chain.
__device__ inline void node_masks(unsigned long long* seen, const int32_t* parents, int nodes, bool there, int lane) {
  constexpr int kRoot = -1, kAbsent = -2;
  unsigned long long m[2];
  int up[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h;
    const int p = i < nodes ? (parents ? parents[i] : i - 1) : kAbsent;
    up[h] = p < kRoot || p >= i ? kAbsent : p;
    m[h] = 1ull << i;
  }
#pragma unroll
  for (int round = 0; round < 6; ++round) {
    unsigned long long om[2];
    int ou[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int from = up[h] & 31;
      const unsigned long long a = __shfl_sync(0xffffffffu, m[0], from), b = __shfl_sync(0xffffffffu, m[1], from);
      const int c = __shfl_sync(0xffffffffu, up[0], from), d = __shfl_sync(0xffffffffu, up[1], from);
      om[h] = up[h] >= 32 ? b : a;
      ou[h] = up[h] >= 32 ? d : c;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (up[h] >= 0) {
        m[h] |= om[h];
        up[h] = ou[h];
      }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h;
    seen[i] = there && i < nodes && up[h] == kRoot ? m[h] : 0ull;
  }
  __syncwarp();
}

// Nodes of the accepted path: up to the first entry that is not a node after
// the one before it, as many as fit into the cache. One warp.
__device__ inline int accepted(const int32_t* path, int path_len, int nodes, int room, int lane) {
  int n = 0;
  for (int base = 0; base < path_len; base += 32) {
    const int i = base + lane;
    const int v = i < path_len ? path[i] : -1, before = i > 0 && i <= path_len ? path[i - 1] : -1;
    const unsigned ok = __ballot_sync(0xffffffffu, v > before && v >= 0 && v < nodes);
    const int run = ok == 0xffffffffu ? 32 : __ffs(~ok) - 1;
    n += run;
    if (run < 32) break;
  }
  return min(n, room);
}

__device__ __forceinline__ void store2(__nv_bfloat16* p, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }

// Joins the partial rows of items that several CTAs worked on. A CTA's two
// partial blocks of mb rows hold [head_dim / 4][row][4] sums, then the rows'
// maxima (natural units) and sums of weights. A thread per row and four columns.
// A part that a row saw nothing in has the maximum -inf and the sum 0. One whose
// scores are all NaN has the maximum -inf too, since a maximum passes NaN over,
// but a sum of NaN, which makes the row NaN as it does where one CTA has the item;
// so does a NaN value whose weight is 0 beside another part's.
// blockIdx.x is an item, or where there are more items than CTAs, a CTA whose run
// may begin inside one (the first such run of an item joins it).
inline bool join_by_item(const TreeParams& p) { return p.c.batch * p.c.kv_heads * p.row_blocks <= p.grid; }
inline dim3 join_grid(const TreeParams& p, int mb, int d) {
  return dim3(join_by_item(p) ? p.c.batch * p.c.kv_heads * p.row_blocks : p.grid, (mb * d / 4 + kThreads - 1) / kThreads);
}
template <typename T, int D, bool APART>
__global__ __launch_bounds__(kThreads) void tree_join_kernel(const __grid_constant__ TreeParams p, int mb, bool by_item) {
  extern __shared__ __align__(16) int sched[];
  int *lens = sched, *first = sched + p.c.batch;
  const int items = p.c.kv_heads * p.row_blocks, nodes = p.nodes;
  build_schedule<APART>(p.c, p.c.batch, items, nodes, lens, first);
  const int total = first[p.c.batch], parts = active(p.grid, total), mine = blockIdx.x;
  Cursor<APART> cur;
  if (by_item) {
    const int b = mine / items;
    cur.seek(first[b] + (mine - b * items) * tiles_of<APART>(lens[b], nodes), lens, first, p.c.batch, p.row_blocks, nodes);
  } else {
    cur.seek(share(min(mine, parts - 1), parts, total), lens, first, p.c.batch, p.row_blocks, nodes);
  }
  const int b = cur.b, w = cur.w - cur.tile;
  const int c0 = owner(w, parts, total), c1 = owner(w + cur.tiles - 1, parts, total);
  pdl_wait();
  if (by_item ? c0 == c1 : mine >= parts || cur.tile == 0 || c0 + 1 != mine) return;
  const int heads_per = p.heads / p.c.kv_heads;
  // The first CTA began with the item (its block 1), the others went on with it.
  auto part = [&](int c) { return p.ws + (int64_t)(c * 2 + (c == c0)) * mb * (D + 2); };
  const int at = blockIdx.y * kThreads + threadIdx.x, r = at % mb, quad = at / mb, row = cur.inner * mb + r;
  if (quad < D / 4 && row < heads_per * nodes) {
    float m = -INFINITY;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) m = fmaxf(m, part(c)[mb * D + r]);
    const float u = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float* src = part(c);
      const float f = ex2((src[mb * D + r] - u) * kLog2e), l = src[mb * D + mb + r];
      const float4 v = *reinterpret_cast<const float4*>(src + (quad * mb + r) * 4);
      if (l == 0.f) continue;  // an empty part's columns may be anything
      sum += l * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    const int hd = row / nodes, n = row - hd * nodes, head = cur.outer * heads_per + hd;
    T* dst = reinterpret_cast<T*>(const_cast<void*>(p.out.ptr)) + b * p.out.sb + head * p.out.sh + n * p.out.sn + quad * 4;
    const bool empty = sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    store2(dst, empty ? 0.f : acc.x * inv, empty ? 0.f : acc.y * inv);
    store2(dst + 2, empty ? 0.f : acc.z * inv, empty ? 0.f : acc.w * inv);
    if (p.lse && quad == 0) p.lse[((int64_t)b * p.heads + head) * nodes + n] = empty ? -INFINITY : m + logf(sum);
  }
}

}  // namespace mrtdf
