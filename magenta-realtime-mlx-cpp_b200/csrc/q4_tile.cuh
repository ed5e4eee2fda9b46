// Products with 4-bit weights: what the two kernels share (q4.cu, q4_wide.cu).
#pragma once

#include <cuda_fp16.h>

#include "cache_ops.cuh"
#include "cache_tile.cuh"
#include "q4.cuh"

namespace mrtdf {
namespace {

constexpr int kStep = 128;  // columns multiplied at a time: 64 bytes of 16 rows

// Byte offset of 16-byte chunk `ch` (0 .. 3) of row `row` of a step. Rows are
// 64 bytes apart; the swizzle puts the eight rows of one access in different
// banks.
__device__ __forceinline__ uint32_t w_at(int row, int ch) {
  return (uint32_t)(row * (kStep / 2) + ((ch ^ (row >> 1 & 3)) << 4));
}

// Words of a step that lane c multiplies for its group `gi`, from row address
// `row` (of a step, without the chunk) whose swizzle is x: WL = G / 32 words,
// columns gi * G + (c * WL + i) * 8.
template <int WL>
__device__ __forceinline__ void load_words(uint32_t* w, uint32_t row, uint32_t x, int c, int gi) {
  if constexpr (WL == 1) {
    w[0] = lds32(row + ((gi << 4) ^ x) + 4 * c);
  } else if constexpr (WL == 2) {
    const uint32_t a = row + (((2 * gi + (c >> 1)) << 4) ^ x) + 8 * (c & 1);
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    const uint32_t a = row + ((c << 4) ^ x);
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(a));
  }
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// q - 8 of the column pairs (0, 4), (1, 5) of w, or with w >> 8 (2, 6), (3, 7). The
// nibbles go under the bits of 1024 (an fp16 whose last place is 1, a published
// way to make small integers floating): 1024 + q and 1024 + 16 q, exactly, then
// - 1032 and / 16 - 72, exactly too.
__device__ __forceinline__ void unpack(uint32_t w, uint32_t& even, uint32_t& odd) {
  // (w & mask) | magic in one instruction each
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(even) : "r"(w), "n"(0x000f000f), "r"(0x64006400u));
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(odd) : "r"(w), "n"(0x00f000f0), "r"(0x64006400u));
  const __half2 e = __hadd2(*reinterpret_cast<const __half2*>(&even), __float2half2_rn(-1032.f));
  const __half2 o = __hfma2(*reinterpret_cast<const __half2*>(&odd), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
  even = *reinterpret_cast<const uint32_t*>(&e);
  odd = *reinterpret_cast<const uint32_t*>(&o);
}

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c = a b: the first product of a sum, on zeros that take no registers.
__device__ __forceinline__ void mma_f16_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// A scale and its bias, side by side in shared memory.
template <typename T>
struct alignas(2 * sizeof(T)) ScalePair {
  T s, b;
};
__device__ __forceinline__ void load_pair(uint32_t at, float& s, float& b, __nv_bfloat16) {
  const uint32_t w = lds32(at);
  s = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void load_pair(uint32_t at, float& s, float& b, float) {
  uint32_t x, y;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(at));
  s = __uint_as_float(x);
  b = __uint_as_float(y);
}

template <typename T>
struct Parts;  // fp16 columns per row of x
template <>
struct Parts<__nv_bfloat16> {
  static constexpr int N = 1;
};
template <>
struct Parts<float> {
  static constexpr int N = 2;
};
// x to fp16: 8 columns from kk on (one word of weights) per lane, a group by
// 4 WL neighbouring lanes, all lanes of a warp together. put(h, words) gets the
// lane's eight values of part h, sums(h, {factor, X}) the group's power of two and
// sum, the latter of the values as the product takes them: x is both multiplied.
// Rows that do not exist (m < 0) and columns past k are zero.
template <typename T, int G, typename Put, typename Sums>
__device__ __forceinline__ void bring_x(const Q4Params& p, int m, int kk, Put&& put, Sums&& sums) {
  constexpr int WL = G / 32, P = Parts<T>::N, V = 8 * (int)sizeof(T) / 16;
  float v[8], big = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (m >= 0 && kk < p.k) {
    const T* src = reinterpret_cast<const T*>(p.x) + m * p.x_stride + kk;
#pragma unroll
    for (int e = 0; e < V; ++e) Vec16<T>::unpack(*reinterpret_cast<const uint4*>(src + e * (8 / V)), v + e * (8 / V));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(v[e]));
#pragma unroll
  for (int o = 1; o < 4 * WL; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  const uint32_t ex = max(__float_as_uint(big) >> 23, 15u);
  const float up = __uint_as_float((268u - ex) << 23), down = __uint_as_float((ex - 14u) << 23);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= up;
#pragma unroll
  for (int h = 0; h < P; ++h) {
    uint32_t w[4];
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = pack_f16(v[e], v[e + 4]);
      const float2 t2 = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      f[e] = t2.x;
      f[e + 4] = t2.y;
    }
    float sum = ((f[0] + f[4]) + (f[2] + f[6])) + ((f[1] + f[5]) + (f[3] + f[7]));
#pragma unroll
    for (int o = 1; o < 4 * WL; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    put(h, make_uint4(w[0], w[1], w[2], w[3]));
    sums(h, make_float2(down, sum));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] -= f[e];
  }
}

// A group's products, scaled, onto y: rows g and g + 8 of the weights and columns
// 2 c, 2 c + 1, whose factors and sums {f, X} are in `u`. The two are two rows of x
// (y[0], y[1] of row g, y[2], y[3] of row g + 8), or the parts of one (y[0] and
// y[1]; one factor), which are added before a scale meets them.
//   y += f (s (acc + 8 X) + b X)
// The power of two comes last: s and b shrink the sums first, so nothing on the
// way to a finite y is too large for float32 (|x| near its largest number
// included) as long as s and b are below 2^100.
template <int P>
__device__ __forceinline__ void add_group(float* y, const float* acc, uint4 u, float s0, float b0, float s1, float b1) {
  const float fu = __uint_as_float(u.x), xu = __uint_as_float(u.y), fv = __uint_as_float(u.z), xv = __uint_as_float(u.w);
  auto add = [](float y, float f, float acc, float x, float s, float b) { return fmaf(f, fmaf(s, fmaf(8.f, x, acc), b * x), y); };
  if constexpr (P == 2) {
    y[0] = add(y[0], fu, acc[0] + acc[1], xu + xv, s0, b0);
    y[1] = add(y[1], fu, acc[2] + acc[3], xu + xv, s1, b1);
  } else {
    y[0] = add(y[0], fu, acc[0], xu, s0, b0);
    y[1] = add(y[1], fv, acc[1], xv, s0, b0);
    y[2] = add(y[2], fu, acc[2], xu, s1, b1);
    y[3] = add(y[3], fv, acc[3], xv, s1, b1);
  }
}

}  // namespace
}  // namespace mrtdf
