// Rows of a KV cache that move: commit of an accepted path, eviction by
// collected weight. Both are bound by the rows they move (head_dim elements
// of K and V, read once and written once) and by latency when there are few.
#include "cache_sched.cuh"

namespace mrtdf {
namespace {

constexpr int kMoveThreads = 256;

// K[len + j] = K_new[path[j]], V alike, pos[len + j] = next_pos + j for every
// layer and kv head of sequence blockIdx.y. The accepted rows of all layers
// are one flat list of 16-byte chunks, so a sequence's CTAs share it evenly
// whatever its path length. Each thread has four K and four V loads in flight.
// 20 layers x 2 x 16 heads of 64, bf16, five rows each: 4.1 us (one launch of
// dependent loads: length, path, rows). 32 layers x 32 x 8 heads of 128, float32,
// up to twelve rows: 21 us for 100 MB (4.7 TB/s, reads and writes).
template <int CH>  // 16-byte chunks per row
__global__ __launch_bounds__(kMoveThreads) void cache_commit_kernel(const __grid_constant__ CommitParams p, int esize) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int len = p.c.lens[b];
  const bool there = len >= 0 && len <= p.c.capacity;
  const int count = there ? accepted(p.path + (int64_t)b * p.path_len, p.path_len, p.nodes, p.c.capacity - len, lane) : 0;
  const int next = p.c.next_pos ? p.c.next_pos[b] : len;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.lens_out[b] = len + count;
    if (p.next_pos_out) p.next_pos_out[b] = (int)((unsigned)next + (unsigned)count);
  }
  if (!count) return;
  const int heads = p.c.layers * p.c.kv_heads;
  const long long total = (long long)heads * count * CH;
  const long long stride = (long long)gridDim.x * kMoveThreads;
  uint8_t *kc = (uint8_t*)p.c.k, *vc = (uint8_t*)p.c.v;
  const uint8_t *kn = (const uint8_t*)p.k_new.ptr, *vn = (const uint8_t*)p.v_new.ptr;
  for (long long i0 = (long long)blockIdx.x * kMoveThreads + threadIdx.x; i0 < total; i0 += 4 * stride) {
    uint4 kv[4], vv[4];
    int64_t to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long i = i0 + u * stride;
      if (i >= total) continue;
      const int ch = (int)(i % CH), row = (int)(i / CH), j = row % count, hd = row / count;
      const int layer = hd / p.c.kv_heads, kvh = hd - layer * p.c.kv_heads;
      const int n = p.path[(int64_t)b * p.path_len + j];
      const int64_t kf = layer * p.k_new.sl + b * p.k_new.sb + kvh * p.k_new.sh + n * p.k_new.sn;
      const int64_t vf = layer * p.v_new.sl + b * p.v_new.sb + kvh * p.v_new.sh + n * p.v_new.sn;
      kv[u] = *reinterpret_cast<const uint4*>(kn + kf * esize + ch * 16);
      vv[u] = *reinterpret_cast<const uint4*>(vn + vf * esize + ch * 16);
      to[u] = (layer * p.c.sl + b * p.c.sb + kvh * p.c.sh + (int64_t)(len + j) * p.c.st) * esize + ch * 16;
      if (ch == 0 && p.c.pos)
        p.c.pos[((int64_t)(layer * p.c.batch + b) * p.c.kv_heads + kvh) * p.c.capacity + len + j] =
            (int)((unsigned)next + (unsigned)j);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * stride >= total) continue;
      *reinterpret_cast<uint4*>(kc + to[u]) = kv[u];
      *reinterpret_cast<uint4*>(vc + to[u]) = vv[u];
    }
  }
}

// ---- eviction ----------------------------------------------------------------------
// One thread-block cluster per (layer, sequence, kv head); CTA r looks after
// slots [r * slice, (r + 1) * slice). Kept are the `budget` slots that come
// first by (protected, weight from the largest, slot from the lowest); a
// weight that is NaN comes last. The threshold is found by three histogram
// passes over an order-preserving 32-bit key (11, 11, 10 bits); a CTA adds its
// occupied bins to every CTA's totals over distributed shared memory, one
// cluster barrier per pass. Short caches (512 slots) count for each slot the
// slots before it instead. Kept slots go into a bitmap; the i-th evicted slot
// below the budget (a hole) takes the i-th kept slot at or above it. Holes are
// below the budget and sources at or above it, so every row moves once, in
// place, in any order.
// 4 layers x 4 x 8 heads, 9000 to 16384 rows of 128 to 2048, bf16, 250 MB: 72 us
// (3.5 TB/s; float32, 485 MB: 115): the passes 17, bitmap and lists 15, both bound by shared memory and
// barriers with one wave of clusters resident, the moves 30 at the memory's rate.
// 2 x 16 heads, 50 rows to 40: 5.2 us, latency. 44 heads of up to 369: 9.9 us.
constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kSliceMax = 1 << 17;  // slots per CTA: the bitmap's size
constexpr int kKeysMax = 16384;     // slots whose keys stay in shared memory
constexpr int kListMax = 2048;      // moves per CTA and round
constexpr int kCountMax = 512;      // slots ranked by counting

struct alignas(16) EvictSmem {
  int hist[kBins];
  int all[2][kBins];  // totals over the cluster; the passes take turns
  int cluster_eq[kMaxCluster], cluster_hole[kMaxCluster], cluster_fill[kMaxCluster];
  int warp_a[kEvictWarps], warp_b[kEvictWarps], warp_c[kEvictWarps];
  int found[3];
  // behind it: keys of the slice where they fit (read 16 bytes at a time),
  // bitmap of the slice, list_to[list], list_from[list]
};

__device__ __forceinline__ void add_cluster(int* local, uint32_t rank, int v) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(ra), "r"(v) : "memory");
}

// Order of weights: larger first, -0 = +0, NaN last (0).
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : float_order_key(w + 0.f); }

__global__ __launch_bounds__(kEvictThreads, 4) void cache_evict_kernel(const __grid_constant__ EvictParams p, int ranks,
                                                                        int chunks, int esize, int list, int words_max,
                                                                        int keys_max) {
  extern __shared__ __align__(16) uint8_t raw[];
  EvictSmem& s = *reinterpret_cast<EvictSmem*>(raw);
  uint32_t* keys = reinterpret_cast<uint32_t*>(raw + sizeof(EvictSmem));
  uint32_t* bitmap = keys + keys_max;
  int* list_to = reinterpret_cast<int*>(bitmap + words_max);
  int* list_from = list_to + list;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ranks > 1 ? (int)cluster_ctarank() : 0;
  const int item = blockIdx.x / ranks, kvh = item % p.c.kv_heads, lb = item / p.c.kv_heads;
  const int b = lb % p.c.batch, layer = lb / p.c.batch;
  const int raw_len = p.c.lens[b], cap = p.c.capacity;
  const long long safe_from = (long long)p.c.next_pos[b] - p.recent;
  const int len = raw_len < 0 || raw_len > cap ? 0 : raw_len;
  if (item == b * p.c.kv_heads && rank == 0 && tid == 0) p.lens_out[b] = raw_len > cap ? raw_len : min(raw_len, p.budget);
  const int64_t row_at = (int64_t)item * cap;
  const float* mass = p.mass + row_at;
  const int32_t* pos = p.c.pos + row_at;
  float* mass_out = p.mass_out + row_at;
  int32_t* pos_out = p.pos_out + row_at;
  const bool apart = mass != mass_out || pos != pos_out;

  if (len <= p.budget) {  // uniform over the cluster
    if (apart)
      for (int t = rank * kEvictThreads + tid; t < len; t += ranks * kEvictThreads) {
        mass_out[t] = mass[t];
        pos_out[t] = pos[t];
      }
    return;
  }

  // Slots of this CTA and of each of its warps, both multiples of 32 long.
  const int per_warp = ((len + ranks * kEvictWarps - 1) / (ranks * kEvictWarps) + 31) / 32 * 32;
  const int slice = per_warp * kEvictWarps, lo = min(rank * slice, len), hi = min(lo + slice, len);
  const bool held = slice <= keys_max, counted = ranks == 1 && len <= kCountMax && held;
  auto key_of = [&](int at, float w) { return at >= safe_from || at < p.sinks ? 0xffffffffu : weight_key(w); };
  auto meet = [&] {
    if (ranks > 1) cluster_sync();
    else __syncthreads();
  };

  uint32_t edge = 0;      // slots above this key are kept,
  int need = p.budget;    // `need` of its equals too (the lowest ones),
  bool some = false;      // which are not all of them
  if (counted) {
    for (int t = tid; t < slice; t += kEvictThreads) {
      uint32_t k = 0;
      if (t < len) {
        const int at = pos[t];
        const float w = mass[t];
        k = key_of(at, w);
        if (apart && t < p.budget) {
          mass_out[t] = w;
          pos_out[t] = at;
        }
      }
      keys[t] = k;
    }
    __syncthreads();
  } else {
    for (int i = tid; i < kBins; i += kEvictThreads) s.hist[i] = s.all[0][i] = s.all[1][i] = 0;
    meet();  // every CTA's totals are zero
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, bins = 1 << bits;
      constexpr int U = 8;  // keys in flight per thread
      for (int t0 = lo + tid; t0 < hi; t0 += U * kEvictThreads) {
        uint32_t k[U];
        if (held && pass) {
#pragma unroll
          for (int u = 0; u < U; ++u) k[u] = keys[min(t0 + u * kEvictThreads, hi - 1) - lo];
        } else {
          int at[U];
          float w[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int t = min(t0 + u * kEvictThreads, hi - 1);
            at[u] = pos[t];
            w[u] = mass[t];
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            k[u] = key_of(at[u], w[u]);
            const int t = t0 + u * kEvictThreads;
            if (held && t < hi) keys[t - lo] = k[u];
            // What stays in its slot; a hole's entry is written again when it is
            // filled, barriers later.
            if (pass == 0 && apart && t < hi && t < p.budget) {
              mass_out[t] = w[u];
              pos_out[t] = at[u];
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t0 + u * kEvictThreads < hi && (pass == 0 || (k[u] >> (shift + bits)) == edge))
            atomicAdd(&s.hist[(k[u] >> shift) & (bins - 1)], 1);
      }
      __syncthreads();
      int* all = s.hist;
      if (ranks > 1) {
        all = s.all[pass & 1];
        for (int i = tid; i < kBins; i += kEvictThreads) {
          const int n = s.hist[i];
          if (n)
            for (int r = 0; r < ranks; ++r) add_cluster(&all[i], r, n);
        }
        meet();
      }
      // Bins from the top: thread i has bins [top - 8 i, top - 8 (i + 1)).
      constexpr int kPer = kBins / kEvictThreads;
      const int top = kBins - 1 - tid * kPer;
      int n[kPer], mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        n[i] = all[top - i];
        mine += n[i];
      }
      int run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      if (lane == 31) s.warp_a[warp] = run;
      __syncthreads();
      // Clear for the passes to come: the histogram and the other totals (the
      // ones just read are not added to before the next barrier).
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        s.hist[top - i] = 0;
        if (pass == 1) s.all[0][top - i] = 0;
      }
      for (int w = 0; w < warp; ++w) run += s.warp_a[w];
      int before = run - mine;
      if (before < need && run >= need) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (before < need && before + n[i] >= need) {
            s.found[0] = top - i;
            s.found[1] = need - before;
            s.found[2] = n[i];
          }
          before += n[i];
        }
      }
      __syncthreads();
      edge = edge << bits | (uint32_t)s.found[0];
      need = s.found[1];
      some = need < s.found[2];
      if (pass == 1 && ranks > 1) meet();  // all[0] is clear everywhere before the last pass adds to it
    }
  }

  const int w_lo = min(lo + warp * per_warp, hi), w_hi = min(w_lo + per_warp, hi);
  auto key_at = [&](int t) { return held ? keys[t - lo] : key_of(pos[t], mass[t]); };
  auto tell = [&](int* slots, int value) {  // value of this CTA into slots[rank] of every CTA
    if (ranks > 1) {
      if (tid < ranks) st_cluster_u32(&slots[rank], tid, (uint32_t)value);
    } else if (tid == 0) {
      slots[0] = value;
    }
  };
  auto sum_of = [&](const int* v, int n) {
    int x = 0;
    for (int i = 0; i < n; ++i) x += v[i];
    return x;
  };
  int eq_before = 0;
  if (some) {  // equal slots before each warp's first one, over CTAs and warps in slot order
    int eq = 0;
    for (int t = w_lo + lane; t < w_hi; t += 32) eq += key_at(t) == edge;
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) s.warp_b[warp] = eq;
    __syncthreads();
    tell(s.cluster_eq, sum_of(s.warp_b, kEvictWarps));
    meet();
    eq_before = sum_of(s.cluster_eq, rank) + sum_of(s.warp_b, warp);
    __syncthreads();
  }

  // Bitmap of kept slots; holes and fills of each warp.
  int holes = 0, fills = 0;
  uint32_t* words = bitmap + warp * (per_warp / 32);
  for (int t = w_lo; t < w_hi; t += 32) {
    const bool in = t + lane < w_hi;
    const uint32_t k = in ? key_at(t + lane) : 0u;
    bool keep;
    if (counted) {
      // Slots that come before this one: of those before this warp's 32 the
      // equal ones too, of those behind only the larger ones.
      int ahead = 0;
      const int end = (len + 3) / 4 * 4;
#pragma unroll 8
      for (int j = 0; j < t; j += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(keys + j);
        ahead += (v.x >= k) + (v.y >= k) + (v.z >= k) + (v.w >= k);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t v = __shfl_sync(0xffffffffu, k, i);
        ahead += v > k || (v == k && i < lane);
      }
#pragma unroll 8
      for (int j = t + 32; j < end; j += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(keys + j);
        ahead += (v.x > k) + (v.y > k) + (v.z > k) + (v.w > k);
      }
      keep = in && ahead < p.budget;
    } else {
      const unsigned same = some ? __ballot_sync(0xffffffffu, in && k == edge) : 0u;
      keep = in && (k > edge || (k == edge && (!some || eq_before + __popc(same & ((1u << lane) - 1)) < need)));
      eq_before += __popc(same);
    }
    const unsigned kept = __ballot_sync(0xffffffffu, keep), used = __ballot_sync(0xffffffffu, in);
    const unsigned below = t + 32 <= p.budget ? 0xffffffffu : t >= p.budget ? 0u : (1u << (p.budget - t)) - 1;
    holes += __popc(~kept & used & below);
    fills += __popc(kept & ~below);
    if (lane == 0) words[(t - w_lo) / 32] = kept;
  }
  if (lane == 0) {
    s.warp_b[warp] = holes;
    s.warp_c[warp] = fills;
  }
  __syncthreads();
  tell(s.cluster_hole, sum_of(s.warp_b, kEvictWarps));
  tell(s.cluster_fill, sum_of(s.warp_c, kEvictWarps));
  meet();
  const int hole0 = sum_of(s.cluster_hole, rank) + sum_of(s.warp_b, warp);
  const int fill0 = sum_of(s.cluster_fill, rank) + sum_of(s.warp_c, warp);
  const int moves = sum_of(s.cluster_hole, ranks);

  // Rounds of up to `list` moves per CTA: move m is CTA m % ranks's (a power of two).
  const int log_ranks = __ffs(ranks) - 1;
  uint8_t* kc = (uint8_t*)p.c.k + (layer * p.c.sl + b * p.c.sb + kvh * p.c.sh) * esize;
  uint8_t* vc = (uint8_t*)p.c.v + (layer * p.c.sl + b * p.c.sb + kvh * p.c.sh) * esize;
  const int64_t row_bytes = p.c.st * esize;
  for (int from = 0; from < moves; from += list * ranks) {
    const int upto = min(moves, from + list * ranks);
    int h = hole0, f = fill0;
    for (int t = w_lo; t < w_hi && (h < upto || f < upto); t += 32) {
      const unsigned kept = words[(t - w_lo) / 32], used = w_hi - t >= 32 ? 0xffffffffu : (1u << (w_hi - t)) - 1;
      const unsigned below = t + 32 <= p.budget ? 0xffffffffu : t >= p.budget ? 0u : (1u << (p.budget - t)) - 1;
      const unsigned hm = ~kept & used & below, fm = kept & ~below, lt = (1u << lane) - 1;
      // A lane's slot is a hole or a fill, not both.
      const bool hole = hm >> lane & 1;
      const int m = hole ? h + __popc(hm & lt) : f + __popc(fm & lt);
      if (((hm | fm) >> lane & 1) && m >= from && m < upto) {
        const unsigned at = (unsigned)(m - from) >> log_ranks, to = (unsigned)(m - from) & (ranks - 1);
        int* slot = (hole ? list_to : list_from) + at;
        if (ranks > 1) st_cluster_u32(slot, to, (uint32_t)(t + lane));
        else *slot = t + lane;
      }
      h += __popc(hm);
      f += __popc(fm);
    }
    meet();
    // chunks is a power of two; a warp's lanes copy neighbouring chunks.
    const int mine = (upto - from - rank + ranks - 1) / ranks, work = mine * chunks, log = __ffs(chunks) - 1;
    for (int i0 = tid; i0 < work; i0 += 4 * kEvictThreads) {
      uint4 kv[4], vv[4];
      int64_t to[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = min(i0 + u * kEvictThreads, work - 1);
        const int m = i >> log, ch = (i & (chunks - 1)) * 16;
        const int64_t src = list_from[m] * row_bytes + ch;
        to[u] = list_to[m] * row_bytes + ch;
        kv[u] = *reinterpret_cast<const uint4*>(kc + src);
        vv[u] = *reinterpret_cast<const uint4*>(vc + src);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i0 + u * kEvictThreads >= work) continue;
        *reinterpret_cast<uint4*>(kc + to[u]) = kv[u];
        *reinterpret_cast<uint4*>(vc + to[u]) = vv[u];
      }
    }
    for (int i = tid; i < mine; i += kEvictThreads) {
      const int src = list_from[i], dst = list_to[i];
      mass_out[dst] = mass[src];
      pos_out[dst] = pos[src];
    }
    if (from + list * ranks < moves) meet();  // the lists are used again
  }
  if (ranks > 1) cluster_sync();  // no CTA leaves while another may still write its lists
}

}  // namespace

cudaError_t launch_cache_commit(const CommitParams& p, cudaStream_t s) {
  const int esize = p.c.dtype == 0 ? 4 : 2, chunks = p.c.head_dim * esize / 16;
  const long long most = (long long)p.c.layers * p.c.kv_heads * p.path_len * chunks;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // Four chunks per thread, at most a few waves over the batch.
  const long long want = (most + 4 * kMoveThreads - 1) / (4 * kMoveThreads);
  const int waves = max(1, 16 * op_sm_count(dev) / p.c.batch);
  const dim3 grid((unsigned)min(want, (long long)waves), p.c.batch);
  switch (chunks) {
    case 8: cache_commit_kernel<8><<<grid, kMoveThreads, 0, s>>>(p, esize); break;
    case 16: cache_commit_kernel<16><<<grid, kMoveThreads, 0, s>>>(p, esize); break;
    default: cache_commit_kernel<32><<<grid, kMoveThreads, 0, s>>>(p, esize); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_cache_evict(const EvictParams& p, cudaStream_t s) {
  const int esize = p.c.dtype == 0 ? 4 : 2, chunks = p.c.head_dim * esize / 16;
  const int items = p.c.layers * p.c.batch * p.c.kv_heads, cap = p.c.capacity;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  // Enough CTAs to fill the GPU twice, with at least 512 slots each.
  int ranks = 1;
  while (ranks < kMaxCluster && (cap > ranks * (kSliceMax / 2) || (items * ranks < 2 * op_sm_count(dev) && cap >= ranks * 1024)))
    ranks *= 2;
  const int per_warp = ((cap + ranks * kEvictWarps - 1) / (ranks * kEvictWarps) + 31) / 32 * 32;
  const int slice = per_warp * kEvictWarps, words = slice / 32, keys = slice <= kKeysMax ? slice : 0;
  const int list = min(kListMax, (min(p.budget, cap) + ranks - 1) / ranks);
  const int bytes = (int)sizeof(EvictSmem) + (2 * list + words + keys) * 4;
  e = allow_smem<cache_evict_kernel>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(items * ranks));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, cache_evict_kernel, p, ranks, chunks, esize, list, words, keys);
}

}  // namespace mrtdf
