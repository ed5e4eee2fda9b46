// Cache operators on caller-owned device buffers: parameters, limits and
// launchers. Kernels in cache_attn.cu (tree attention, collected weight) and
// cache_move.cu (commit, eviction); argument checks in cache_ops.cpp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace mrtdf {

// Lets kernel `K` use up to `BYTES` of dynamic shared memory (next to a little
// static) on the current device; the attribute is set once per device.
constexpr int kOpMaxSmem = 226 * 1024;
template <auto K, int BYTES = kOpMaxSmem>
cudaError_t allow_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Rows of head_dim contiguous elements: row (l, b, h, n) starts at
// ptr + l * sl + b * sb + h * sh + n * sn elements, 16-byte aligned.
struct RowsView {
  const void* ptr;
  int64_t sl, sb, sh, sn;
};

struct CacheView {
  void* k;
  void* v;
  int64_t sl, sb, sh, st;
  int layers, batch, kv_heads, capacity, head_dim, dtype;
  const int32_t* lens;      // (batch)
  int32_t* pos;             // (layers, batch, kv_heads, capacity) or NULL: the slot number
  const int32_t* next_pos;  // (batch) or NULL: lens
};

constexpr int kOpMaxNodes = 64;
constexpr int kOpMaxRows = 1024;  // nodes (or path nodes) x query heads of one kv head
constexpr int kOpMaxBatch = 1024;
constexpr int kOpMaxCapacity = 1 << 24;

struct TreeParams {
  CacheView c;
  RowsView q, k_new, v_new, out;
  float* lse;              // (batch, heads, nodes) or NULL
  const int32_t* parents;  // (batch, nodes) or NULL: a chain
  const float* rel_bias;   // (heads, rel_len) or NULL
  float* ws;               // partial rows, tree_workspace_floats()
  int heads, nodes, rel_len;
  float scale;
  int grid;       // CTAs of the attention kernel
  int row_blocks; // blocks of query rows per (sequence, kv head)
  int tc;         // 1: the tcgen05 kernel
  int stream;     // 1: equal runs of key tiles per CTA, joined afterwards; 0: whole items
  int wait_once;  // 1: a device wait looks once and gives up (failure detection)
};

struct MassParams {
  CacheView c;
  RowsView q, k_new;
  const float* lse;      // (layers, batch, heads, nodes)
  const int32_t* path;   // (batch, path_len)
  const float* rel_bias;
  const float* mass;     // (layers, batch, kv_heads, capacity)
  float* mass_out;
  int heads, nodes, path_len, rel_len;
  float scale, decay;
  int grid;
};

struct CommitParams {
  CacheView c;
  RowsView k_new, v_new;
  const int32_t* path;
  int32_t* lens_out;
  int32_t* next_pos_out;
  int nodes, path_len;
};

struct EvictParams {
  CacheView c;
  const float* mass;
  float* mass_out;
  int32_t* pos_out;
  int32_t* lens_out;
  int budget, recent, sinks;
};

// Multiprocessors of a device, asked once (148 when the driver does not say).
int op_sm_count(int device);

// Chooses the variant and the grid (p.grid, p.row_blocks, p.stream) for a GPU
// of `sms` multiprocessors; gives the floats of workspace the launch needs.
cudaError_t plan_tree_attention(TreeParams& p, int sms, size_t* ws_floats);
cudaError_t launch_tree_attention(const TreeParams& p, cudaStream_t s);
// The tcgen05 kernel's part of the two (cache_attn_tc.cu).
bool tree_attention_tc_takes(const TreeParams& p);
void plan_tree_attention_tc(TreeParams& p, int sms, size_t* ws_floats);
cudaError_t launch_tree_attention_tc(const TreeParams& p, cudaStream_t s);
cudaError_t launch_cache_mass(MassParams& p, cudaStream_t s);
cudaError_t launch_cache_commit(const CommitParams& p, cudaStream_t s);
cudaError_t launch_cache_evict(const EvictParams& p, cudaStream_t s);

}  // namespace mrtdf
