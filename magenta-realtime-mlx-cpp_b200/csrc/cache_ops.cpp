// C ABI of the operators on caller-owned device buffers (include/mrtdf.h,
// "operators"): argument checks, the device switch and the launches. Nothing
// here allocates, synchronises or reads device memory.
#include <atomic>
#include <initializer_list>
#include <string>

#include "cache_ops.cuh"
#include "host_util.h"
#include "q4.cuh"

namespace mrtdf {

int op_sm_count(int device) {
  static std::atomic<int> counts[64];
  if (device < 0 || device >= 64) return 148;
  int n = counts[device].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    counts[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace mrtdf

using namespace mrtdf;

namespace {

[[noreturn]] void invalid(const std::string& what) { throw Error{MRTDF_ERR_INVALID, what}; }
[[noreturn]] void out_of_range(const std::string& what) { throw Error{MRTDF_ERR_RANGE, what}; }

void cuda_check(cudaError_t e, const char* op) {
  if (e != cudaSuccess) {
    cudaGetLastError();  // do not leave it for the caller's next check
    throw Error{MRTDF_ERR_CUDA, std::string(op) + ": " + cudaGetErrorString(e)};
  }
}

// Makes `device` current for the call and puts the caller's back.
struct DeviceScope {
  int before = -1;
  DeviceScope(int device, const char* op) {
    int now = -1;
    cuda_check(cudaGetDevice(&now), op);
    if (now == device) return;
    cuda_check(cudaSetDevice(device), op);
    before = now;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int dtype_bytes(int dtype, const char* op) {
  if (dtype == MRTDF_DTYPE_FP32) return 4;
  if (dtype == MRTDF_DTYPE_BF16) return 2;
  invalid(std::string(op) + ": dtype must be MRTDF_DTYPE_FP32 or MRTDF_DTYPE_BF16");
}

// Steps over a dimension of one element do not matter.
int64_t step(int64_t stride, int64_t extent, int esize, const char* op, const char* what) {
  if (extent <= 1) return 0;
  if (stride < 0) invalid(std::string(op) + ": negative stride of " + what);
  if (stride * esize % 16 != 0) invalid(std::string(op) + ": rows of " + what + " must start on 16-byte boundaries");
  return stride;
}

RowsView rows_view(const mrtdf_rows& r, int64_t l, int64_t b, int64_t h, int64_t n, int esize, const char* op, const char* what) {
  if (!r.ptr) invalid(std::string(op) + ": " + what + " is NULL");
  if (!aligned16(r.ptr)) invalid(std::string(op) + ": " + what + " must be 16-byte aligned");
  RowsView v{};
  v.ptr = r.ptr;
  v.sl = step(r.stride_l, l, esize, op, what);
  v.sb = step(r.stride_b, b, esize, op, what);
  v.sh = step(r.stride_h, h, esize, op, what);
  v.sn = step(r.stride_n, n, esize, op, what);
  return v;
}

// `values`: whether the operator reads or writes V.
CacheView cache_view(const mrtdf_cache* c, const char* op, bool values) {
  if (!c) invalid(std::string(op) + ": cache is NULL");
  if (c->struct_bytes != sizeof(mrtdf_cache)) invalid(std::string(op) + ": cache.struct_bytes is not sizeof(mrtdf_cache)");
  const int esize = dtype_bytes(c->dtype, op);
  if (c->layers < 1 || c->batch < 1 || c->kv_heads < 1 || c->capacity < 1) invalid(std::string(op) + ": cache sizes must be positive");
  if (c->head_dim != 64 && c->head_dim != 128) invalid(std::string(op) + ": head_dim must be 64 or 128");
  if (c->batch > kOpMaxBatch || c->layers > 1024 || c->kv_heads > 1024 || c->capacity > kOpMaxCapacity)
    out_of_range(std::string(op) + ": at most 1024 sequences, layers and kv heads and 2^24 cached rows");
  if (!c->k || (values && !c->v) || !c->lens) invalid(std::string(op) + ": cache.k, cache.v and cache.lens must not be NULL");
  if (!aligned16(c->k) || (values && !aligned16(c->v))) invalid(std::string(op) + ": the cache must be 16-byte aligned");
  if (c->device < 0) invalid(std::string(op) + ": cache.device is negative");
  if (c->pos && !c->next_pos) invalid(std::string(op) + ": cache.pos needs cache.next_pos");
  CacheView v{};
  v.k = c->k;
  v.v = c->v;
  v.layers = c->layers;
  v.batch = c->batch;
  v.kv_heads = c->kv_heads;
  v.capacity = c->capacity;
  v.head_dim = c->head_dim;
  v.dtype = c->dtype;
  v.sl = step(c->stride_l, c->layers, esize, op, "the cache");
  v.sb = step(c->stride_b, c->batch, esize, op, "the cache");
  v.sh = step(c->stride_h, c->kv_heads, esize, op, "the cache");
  v.st = step(c->stride_t, c->capacity, esize, op, "the cache");
  v.lens = c->lens;
  v.pos = c->pos;
  v.next_pos = c->next_pos;
  return v;
}

// Rows that are written: a step of zero would put several into one.
void apart(std::initializer_list<std::pair<int64_t, int64_t>> steps_and_extents, const char* op, const char* what) {
  for (const auto& s : steps_and_extents)
    if (s.second > 1 && s.first == 0) invalid(std::string(op) + ": rows of " + what + " are written and must not share memory (zero stride)");
}
void apart(const CacheView& c, const char* op) {
  apart({{c.sl, c.layers}, {c.sb, c.batch}, {c.sh, c.kv_heads}, {c.st, c.capacity}}, op, "the cache");
}

// A buffer that is written is none of the others of the call (NULL ones aside).
void own_buffer(const void* written, std::initializer_list<const void*> others, const char* op, const char* what) {
  for (const void* o : others)
    if (written && written == o) invalid(std::string(op) + ": " + what + " must be another buffer than the other operands");
}

// Addresses of elements of `esize` bytes.
void check_element(const void* p, int esize, const char* op, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % esize) invalid(std::string(op) + ": " + what + " is not aligned to its elements");
}

void check_heads(const char* op, int heads, int kv_heads, int nodes) {
  if (heads < 1 || heads % kv_heads) invalid(std::string(op) + ": heads must be a multiple of kv_heads");
  if (nodes < 1) invalid(std::string(op) + ": nodes must be positive");
  if (nodes > kOpMaxNodes) out_of_range(std::string(op) + ": at most 64 nodes");
  if (heads / kv_heads > 64 || heads / kv_heads * nodes > kOpMaxRows)
    out_of_range(std::string(op) + ": at most 64 heads per kv head and 1024 rows (nodes x heads) per kv head");
}

// Key tiles of 64 of a call, counted in 32 bits by the kernels.
void check_tiles(const char* op, int64_t items, int64_t rows) {
  if (items * ((rows + 63) / 64) >= (int64_t)1 << 31) out_of_range(std::string(op) + ": the call has 2^31 key tiles or more");
}

void check_bias(const char* op, const float* table, int len, float scale) {
  if (table && (len < 1 || len > (1 << 20))) invalid(std::string(op) + ": rel_len must be 1 .. 2^20");
  if (!(scale == scale)) invalid(std::string(op) + ": scale is NaN");
}

TreeParams tree_params(const mrtdf_cache* cache, const mrtdf_tree_args* a, const char* op) {
  TreeParams p{};
  p.c = cache_view(cache, op, true);
  if (!a) invalid(std::string(op) + ": args is NULL");
  if (a->struct_bytes != sizeof(mrtdf_tree_args)) invalid(std::string(op) + ": args.struct_bytes is not sizeof(mrtdf_tree_args)");
  if (p.c.layers != 1) invalid(std::string(op) + ": attention runs layer by layer (cache.layers must be 1)");
  check_heads(op, a->heads, p.c.kv_heads, a->nodes);
  check_bias(op, a->rel_bias, a->rel_len, a->scale);
  check_tiles(op, (int64_t)p.c.batch * p.c.kv_heads * ((a->heads / p.c.kv_heads * a->nodes + 15) / 16),
              (int64_t)p.c.capacity + a->nodes);
  const int es = dtype_bytes(p.c.dtype, op), b = p.c.batch, kv = p.c.kv_heads, n = a->nodes;
  p.q = rows_view(a->q, 1, b, a->heads, n, es, op, "q");
  p.k_new = rows_view(a->k_new, 1, b, kv, n, es, op, "k_new");
  p.v_new = rows_view(a->v_new, 1, b, kv, n, es, op, "v_new");
  p.out = rows_view(a->out, 1, b, a->heads, n, es, op, "out");
  apart({{p.out.sb, b}, {p.out.sh, a->heads}, {p.out.sn, n}}, op, "out");
  const std::initializer_list<const void*> read = {p.q.ptr, p.k_new.ptr, p.v_new.ptr, p.c.k, p.c.v, p.c.lens, p.c.pos, p.c.next_pos,
                                                    a->parents, a->rel_bias};
  own_buffer(p.out.ptr, read, op, "out");
  own_buffer(a->lse, read, op, "lse");
  own_buffer(a->lse, {p.out.ptr}, op, "lse");
  p.lse = a->lse;
  p.parents = a->parents;
  p.rel_bias = a->rel_bias;
  p.rel_len = a->rel_bias ? a->rel_len : 1;
  p.scale = a->scale;
  p.heads = a->heads;
  p.nodes = a->nodes;
  return p;
}

Q4Params q4_params(const mrtdf_q4_args* a, const char* op) {
  if (!a) invalid("q4_linear: args is NULL");
  if (a->struct_bytes != sizeof(mrtdf_q4_args)) invalid("q4_linear: args.struct_bytes is not sizeof(mrtdf_q4_args)");
  const int es = dtype_bytes(a->dtype, op);
  dtype_bytes(a->out_dtype, op);
  if (a->dtype == MRTDF_DTYPE_FP32 && a->out_dtype != MRTDF_DTYPE_FP32) invalid("q4_linear: float32 x gives float32 out");
  if (a->group != 32 && a->group != 64 && a->group != 128) invalid("q4_linear: group must be 32, 64 or 128");
  if (a->m < 1 || a->n < 1 || a->k < 1 || a->k % a->group) invalid("q4_linear: sizes must be positive and k a multiple of the group");
  if (a->m > kQ4MaxRows || a->k > kQ4MaxIn || a->n > (1 << 24)) out_of_range("q4_linear: at most 64 rows of x, k 2^17, n 2^24");
  if (!a->x || !a->packed || !a->scales || !a->biases || !a->out) invalid("q4_linear: NULL argument");
  if (!aligned16(a->x) || !aligned16(a->packed)) invalid("q4_linear: x and packed must be 16-byte aligned");
  if (a->device < 0) invalid("q4_linear: device is negative");
  own_buffer(a->out, {a->x, a->packed, a->scales, a->biases}, op, "out");
  check_element(a->scales, es, op, "scales");
  check_element(a->biases, es, op, "biases");
  check_element(a->out, a->out_dtype == MRTDF_DTYPE_FP32 ? 4 : 2, op, "out");
  Q4Params p{};
  p.x = a->x;
  p.packed = static_cast<const uint8_t*>(a->packed);
  p.scales = a->scales;
  p.biases = a->biases;
  p.out = a->out;
  p.x_stride = step(a->x_stride, a->m, es, op, "x");
  p.out_stride = a->out_stride;
  if (a->m > 1 && a->out_stride < a->n) invalid("q4_linear: out_stride is less than n");
  p.m = a->m;
  p.n = a->n;
  p.k = a->k;
  p.group = a->group;
  return p;
}

void run_q4_linear(const mrtdf_q4_args* a, bool wait_once, void* stream, const char* op) {
  Q4Params p = q4_params(a, op);
  p.wait_once = wait_once;
  size_t need = 0;
  const int sms = op_sm_count(a->device);
  cuda_check(launch_q4_linear(p, a->dtype, a->out_dtype, sms, &need, nullptr), op);
  if (need) {
    if (!a->workspace || a->workspace_bytes < need)
      invalid("q4_linear: the workspace is smaller than mrtdf_q4_linear_workspace says (" + std::to_string(need) + " bytes)");
    if (!aligned16(a->workspace)) invalid("q4_linear: the workspace must be 16-byte aligned");
    p.ws = a->workspace;
  }
  DeviceScope on(a->device, op);
  cuda_check(launch_q4_linear(p, a->dtype, a->out_dtype, sms, nullptr, static_cast<cudaStream_t>(stream)), op);
}

void run_tree_attention(const mrtdf_cache* cache, const mrtdf_tree_args* args, bool wait_once, void* stream, const char* op) {
  TreeParams p = tree_params(cache, args, op);
  p.wait_once = wait_once;
  size_t floats = 0;
  cuda_check(plan_tree_attention(p, op_sm_count(cache->device), &floats), op);
  if (floats) {
    if (!args->workspace || args->workspace_bytes < floats * sizeof(float))
      invalid(std::string(op) + ": the workspace is smaller than mrtdf_tree_attention_workspace says (" +
              std::to_string(floats * sizeof(float)) + " bytes)");
    if (!aligned16(args->workspace)) invalid(std::string(op) + ": the workspace must be 16-byte aligned");
    p.ws = static_cast<float*>(args->workspace);
  }
  DeviceScope on(cache->device, op);
  cuda_check(launch_tree_attention(p, static_cast<cudaStream_t>(stream)), op);
}

}  // namespace

extern "C" {

int mrtdf_tree_attention_workspace(const mrtdf_cache* cache, const mrtdf_tree_args* args, size_t* bytes) {
  return guarded([&] {
    const char* op = "tree_attention_workspace";
    if (!bytes) invalid("tree_attention_workspace: bytes is NULL");
    TreeParams p = tree_params(cache, args, op);
    size_t floats = 0;
    cuda_check(plan_tree_attention(p, op_sm_count(cache->device), &floats), op);
    *bytes = floats * sizeof(float);
  });
}

int mrtdf_tree_attention(const mrtdf_cache* cache, const mrtdf_tree_args* args, void* stream) {
  return guarded([&] { run_tree_attention(cache, args, false, stream, "tree_attention"); });
}

int mrtdf_check_tree_attention_wait(const mrtdf_cache* cache, const mrtdf_tree_args* args, void* stream) {
  return guarded([&] { run_tree_attention(cache, args, true, stream, "check_tree_attention_wait"); });
}

int mrtdf_cache_mass(const mrtdf_cache* cache, const mrtdf_mass_args* a, void* stream) {
  return guarded([&] {
    const char* op = "cache_mass";
    MassParams p{};
    p.c = cache_view(cache, op, false);
    if (!a) invalid("cache_mass: args is NULL");
    if (a->struct_bytes != sizeof(mrtdf_mass_args)) invalid("cache_mass: args.struct_bytes is not sizeof(mrtdf_mass_args)");
    check_heads(op, a->heads, p.c.kv_heads, a->nodes);
    check_bias(op, a->rel_bias, a->rel_len, a->scale);
    if (a->path_len < 1 || a->path_len > a->nodes) invalid("cache_mass: path_len must be 1 .. nodes");
    if (!a->lse || !a->path || !a->mass || !a->mass_out) invalid("cache_mass: lse, path, mass and mass_out must not be NULL");
    if (!(a->decay == a->decay)) invalid("cache_mass: decay is NaN");
    check_tiles(op, (int64_t)p.c.layers * p.c.batch * p.c.kv_heads, (int64_t)p.c.capacity + a->path_len);
    const int es = dtype_bytes(p.c.dtype, op), l = p.c.layers, b = p.c.batch;
    p.q = rows_view(a->q, l, b, a->heads, a->nodes, es, op, "q");
    p.k_new = rows_view(a->k_new, l, b, p.c.kv_heads, a->nodes, es, op, "k_new");
    own_buffer(a->mass_out, {p.q.ptr, p.k_new.ptr, p.c.k, p.c.lens, p.c.pos, p.c.next_pos, a->lse, a->path, a->rel_bias}, op, "mass_out");
    p.lse = a->lse;
    p.path = a->path;
    p.rel_bias = a->rel_bias;
    p.rel_len = a->rel_bias ? a->rel_len : 1;
    p.mass = a->mass;
    p.mass_out = a->mass_out;
    p.heads = a->heads;
    p.nodes = a->nodes;
    p.path_len = a->path_len;
    p.scale = a->scale;
    p.decay = a->decay;
    DeviceScope on(cache->device, op);
    cuda_check(launch_cache_mass(p, static_cast<cudaStream_t>(stream)), op);
  });
}

int mrtdf_cache_commit(const mrtdf_cache* cache, const mrtdf_commit_args* a, void* stream) {
  return guarded([&] {
    const char* op = "cache_commit";
    CommitParams p{};
    p.c = cache_view(cache, op, true);
    if (!a) invalid("cache_commit: args is NULL");
    if (a->struct_bytes != sizeof(mrtdf_commit_args)) invalid("cache_commit: args.struct_bytes is not sizeof(mrtdf_commit_args)");
    if (a->nodes < 1) invalid("cache_commit: nodes must be positive");
    if (a->nodes > kOpMaxNodes) out_of_range("cache_commit: at most 64 nodes");
    if (a->path_len < 1 || a->path_len > a->nodes) invalid("cache_commit: path_len must be 1 .. nodes");
    if (!a->path || !a->lens_out) invalid("cache_commit: path and lens_out must not be NULL");
    if (a->next_pos_out && !p.c.next_pos) invalid("cache_commit: next_pos_out needs cache.next_pos");
    const int es = dtype_bytes(p.c.dtype, op), l = p.c.layers, b = p.c.batch, kv = p.c.kv_heads;
    if ((int64_t)l * kv * a->path_len >= (int64_t)1 << 26) out_of_range("cache_commit: too many rows");
    apart(p.c, op);
    p.k_new = rows_view(a->k_new, l, b, kv, a->nodes, es, op, "k_new");
    p.v_new = rows_view(a->v_new, l, b, kv, a->nodes, es, op, "v_new");
    if (p.k_new.ptr == p.c.k || p.k_new.ptr == p.c.v || p.v_new.ptr == p.c.v || p.v_new.ptr == p.c.k)
      invalid("cache_commit: the new rows must be another buffer than the cache");
    const std::initializer_list<const void*> read = {p.c.lens, p.c.next_pos, p.c.pos, a->path, p.c.k, p.c.v, p.k_new.ptr, p.v_new.ptr};
    own_buffer(a->lens_out, read, op, "lens_out");
    own_buffer(a->next_pos_out, read, op, "next_pos_out");
    own_buffer(a->next_pos_out, {a->lens_out}, op, "next_pos_out");
    own_buffer(p.c.pos, {p.c.lens, p.c.next_pos, a->path}, op, "pos");
    p.path = a->path;
    p.lens_out = a->lens_out;
    p.next_pos_out = a->next_pos_out;
    p.nodes = a->nodes;
    p.path_len = a->path_len;
    DeviceScope on(cache->device, op);
    cuda_check(launch_cache_commit(p, static_cast<cudaStream_t>(stream)), op);
  });
}

int mrtdf_cache_evict(const mrtdf_cache* cache, const mrtdf_evict_args* a, void* stream) {
  return guarded([&] {
    const char* op = "cache_evict";
    EvictParams p{};
    p.c = cache_view(cache, op, true);
    if (!a) invalid("cache_evict: args is NULL");
    if (a->struct_bytes != sizeof(mrtdf_evict_args)) invalid("cache_evict: args.struct_bytes is not sizeof(mrtdf_evict_args)");
    if (p.c.capacity > (1 << 20)) out_of_range("cache_evict: at most 2^20 cached rows");
    if ((int64_t)p.c.layers * p.c.batch * p.c.kv_heads > (1 << 24)) out_of_range("cache_evict: too many heads");
    if (!p.c.pos) invalid("cache_evict: cache.pos and cache.next_pos must not be NULL");
    if (!a->mass || !a->mass_out || !a->pos_out || !a->lens_out)
      invalid("cache_evict: mass, mass_out, pos_out and lens_out must not be NULL");
    if (a->budget < 1) invalid("cache_evict: budget must be positive");
    if (a->recent < 0 || a->sinks < 0 || (int64_t)a->recent + a->sinks > a->budget)
      invalid("cache_evict: recent and sinks must be >= 0 and fit into the budget together");
    apart(p.c, op);
    own_buffer(a->lens_out, {p.c.lens, p.c.next_pos, p.c.pos, p.c.k, p.c.v, a->mass, a->mass_out, a->pos_out}, op, "lens_out");
    own_buffer(a->mass_out, {p.c.lens, p.c.next_pos, p.c.pos, p.c.k, p.c.v}, op, "mass_out");
    own_buffer(a->pos_out, {p.c.lens, p.c.next_pos, p.c.k, p.c.v, a->mass, a->mass_out}, op, "pos_out");
    p.mass = a->mass;
    p.mass_out = a->mass_out;
    p.pos_out = a->pos_out;
    p.lens_out = a->lens_out;
    p.budget = a->budget;
    p.recent = a->recent;
    p.sinks = a->sinks;
    DeviceScope on(cache->device, op);
    cuda_check(launch_cache_evict(p, static_cast<cudaStream_t>(stream)), op);
  });
}

int mrtdf_q4_linear_workspace(const mrtdf_q4_args* a, size_t* bytes) {
  return guarded([&] {
    if (!bytes) invalid("q4_linear_workspace: bytes is NULL");
    const Q4Params p = q4_params(a, "q4_linear_workspace");
    cuda_check(launch_q4_linear(p, a->dtype, a->out_dtype, op_sm_count(a->device), bytes, nullptr), "q4_linear_workspace");
  });
}

int mrtdf_q4_linear(const mrtdf_q4_args* a, void* stream) {
  return guarded([&] { run_q4_linear(a, false, stream, "q4_linear"); });
}

int mrtdf_check_q4_linear_wait(const mrtdf_q4_args* a, void* stream) {
  return guarded([&] { run_q4_linear(a, true, stream, "check_q4_linear_wait"); });
}

int mrtdf_q4_quantize(const mrtdf_q4_pack_args* a, void* stream) {
  return guarded([&] {
    const char* op = "q4_quantize";
    if (!a) invalid("q4_quantize: args is NULL");
    if (a->struct_bytes != sizeof(mrtdf_q4_pack_args)) invalid("q4_quantize: args.struct_bytes is not sizeof(mrtdf_q4_pack_args)");
    dtype_bytes(a->dtype, op);
    if (a->group != 32 && a->group != 64 && a->group != 128) invalid("q4_quantize: group must be 32, 64 or 128");
    if (a->n < 1 || a->k < 1 || a->k % a->group) invalid("q4_quantize: sizes must be positive and k a multiple of the group");
    if (a->k > kQ4MaxIn || a->n > (1 << 24)) out_of_range("q4_quantize: k at most 2^17, n at most 2^24");
    if (!a->w || !a->packed || !a->scales || !a->biases) invalid("q4_quantize: NULL argument");
    if (a->n > 1 && a->w_stride < a->k) invalid("q4_quantize: w_stride is less than k");
    if (a->device < 0) invalid("q4_quantize: device is negative");
    const int es = dtype_bytes(a->dtype, op);
    check_element(a->w, es, op, "w");
    check_element(a->scales, es, op, "scales");
    check_element(a->biases, es, op, "biases");
    own_buffer(a->packed, {a->w, a->scales, a->biases}, op, "packed");
    own_buffer(a->scales, {a->w, a->biases}, op, "scales");
    own_buffer(a->biases, {a->w}, op, "biases");
    Q4PackParams p{};
    p.w = a->w;
    p.packed = static_cast<uint8_t*>(a->packed);
    p.scales = a->scales;
    p.biases = a->biases;
    p.w_stride = a->w_stride;
    p.n = a->n;
    p.k = a->k;
    p.group = a->group;
    DeviceScope on(a->device, op);
    cuda_check(launch_q4_quantize(p, a->dtype, static_cast<cudaStream_t>(stream)), op);
  });
}

}  // extern "C"
