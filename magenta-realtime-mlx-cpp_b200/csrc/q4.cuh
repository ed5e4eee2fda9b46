// Products with 4-bit weights: parameters and launchers (kernels in q4.cu,
// argument checks in cache_ops.cpp).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mrtdf {

constexpr int kQ4MaxRows = 64;
constexpr int kQ4MaxIn = 1 << 17;

struct Q4Params {
  const void* x;           // (m, k), row stride x_stride elements
  const uint8_t* packed;   // (n, k / 2): column 2 j in the low half of byte j
  const void* scales;      // (n, k / group)
  const void* biases;      // (n, k / group)
  void* ws;                // x as the product takes it
  void* out;               // (m, n), row stride out_stride elements
  int64_t x_stride, out_stride;
  int m, n, k, group;
  int wait_once;  // 1: a wait of the copying warps looks once and gives up (failure detection)
};

struct Q4PackParams {
  const void* w;  // (n, k), row stride w_stride elements
  uint8_t* packed;
  void* scales;
  void* biases;
  int64_t w_stride;
  int n, k, group;
};

// dtype (of x, scales, biases) and out_dtype: MRTDF_DTYPE_*.
// With ws_bytes: only the size of the workspace that the call needs, on a GPU of
// `sms` multiprocessors.
cudaError_t launch_q4_linear(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s);
// The part for wide x (q4_wide.cu).
cudaError_t launch_q4_wide(const Q4Params& p, int dtype, int out_dtype, int sms, size_t* ws_bytes, cudaStream_t s);
cudaError_t launch_q4_quantize(const Q4PackParams& p, int dtype, cudaStream_t s);

}  // namespace mrtdf
