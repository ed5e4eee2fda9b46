// Tile products of the cache operators: 16 query rows x 8 keys on the warp
// matrix instructions, for bf16 (m16n8k16) and float32 (m16n8k8 tf32, each
// operand split in two tf32 parts), from rows in swizzled shared memory.
//
// float32: x = hi + lo + r with hi, lo of 11 significant bits, |r| <= 2^-24 |x|
// or so; hi hi + hi lo + lo hi leaves out lo lo (2^-24 relative), so a product
// is as exact as a float32 multiply. The matrix instructions truncate their
// sums; the small products therefore go to accumulators of their own, and a
// tile's p . v is summed apart and added with a rounded add (one accumulator
// through a cache of 1006 rows: 1.1e-6 off against 5.6e-7 for float32 FMAs).
// Three m16n8k8 issue faster than the 1024 FMAs they replace, which keeps a
// few rows bound by memory.
//
// Shared-memory rows hold head_dim elements in 16-byte chunks; chunk c of row
// r sits at chunk c ^ (r & 7), so the eight rows of one ldmatrix lie in
// different banks; so do the four rows 2 c (+1) of which float32 value rows are
// read a word per lane.
#pragma once

#include "common.cuh"
#include "decode_device.cuh"

namespace mrtdf {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, both tf32 (the low part of the rest is dropped).
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(x)));
  const float rest = __uint_as_float(x) - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Shared-memory geometry of rows of D elements of T.
template <typename T, int D>
struct Rows {
  static constexpr int kChunks = D * (int)sizeof(T) / 16;  // 16-byte chunks per row
  static constexpr int kBytes = D * (int)sizeof(T);
  __device__ __forceinline__ static uint32_t at(int row, int chunk) {
    return (uint32_t)(row * kBytes + ((chunk ^ (row & 7)) << 4));
  }
};

// One 16-row block of queries in the A-operand layout of the products:
// lane (g = lane / 4, c = lane % 4) holds rows g and g + 8.
template <typename T, int D>
struct QFrag;

template <int D>
struct QFrag<__nv_bfloat16, D> {
  uint32_t a[D / 16][4];
  __device__ __forceinline__ void load(const __nv_bfloat16* r0, const __nv_bfloat16* r1, int lane) {
    const int c = lane & 3;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      a[ks][0] = r0 ? *reinterpret_cast<const uint32_t*>(r0 + 16 * ks + 2 * c) : 0u;
      a[ks][1] = r1 ? *reinterpret_cast<const uint32_t*>(r1 + 16 * ks + 2 * c) : 0u;
      a[ks][2] = r0 ? *reinterpret_cast<const uint32_t*>(r0 + 16 * ks + 8 + 2 * c) : 0u;
      a[ks][3] = r1 ? *reinterpret_cast<const uint32_t*>(r1 + 16 * ks + 8 + 2 * c) : 0u;
    }
  }
};

template <int D>
struct QFrag<float, D> {
  uint32_t a[D / 8][4];  // split into tf32 parts where they are used
  __device__ __forceinline__ void load(const float* r0, const float* r1, int lane) {
    const int c = lane & 3;
#pragma unroll
    for (int ks = 0; ks < D / 8; ++ks) {
      a[ks][0] = r0 ? __float_as_uint(r0[8 * ks + c]) : 0u;
      a[ks][1] = r1 ? __float_as_uint(r1[8 * ks + c]) : 0u;
      a[ks][2] = r0 ? __float_as_uint(r0[8 * ks + 4 + c]) : 0u;
      a[ks][3] = r1 ? __float_as_uint(r1[8 * ks + 4 + c]) : 0u;
    }
  }
};

// s[j][.] += q . key rows 8 j .. 8 j + 7 of the tile at `keys`. Lane (g, c):
// s[j][0..1] = row g, keys 8 j + 2 c, + 1; s[j][2..3] = row g + 8.
template <int D, int NT>
__device__ __forceinline__ void qk_tile(float (*s)[4], const QFrag<__nv_bfloat16, D>& q, uint32_t keys, int lane) {
  using R = Rows<__nv_bfloat16, D>;
  const int m = lane >> 3, r = lane & 7;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
    for (int jp = 0; jp < NT / 2; ++jp) {
      uint32_t b[4];
      ldsm_x4_g(b, keys + R::at(16 * jp + (m >> 1) * 8 + r, 2 * ks + (m & 1)));
      mma_m16n8k16(s[2 * jp], q.a[ks], b[0], b[1]);
      mma_m16n8k16(s[2 * jp + 1], q.a[ks], b[2], b[3]);
    }
  }
}

// float32: three products of tf32 parts, the small ones apart. The tensor cores
// cut off what does not fit an accumulator, always towards zero, so the large
// products are summed over 32 columns at most before they are added, rounded, to
// the score (chains over all 128 columns doubled the result's error).
template <int D, int NT>
__device__ __forceinline__ void qk_tile(float (*s)[4], const QFrag<float, D>& q, uint32_t keys, int lane) {
  using R = Rows<float, D>;
  constexpr int CHAIN = 4;
  const int m = lane >> 3, r = lane & 7;
  float low[NT][4] = {};
#pragma unroll
  for (int k0 = 0; k0 < D / 8; k0 += CHAIN) {
    float high[NT][4] = {};
#pragma unroll
    for (int ks = k0; ks < k0 + CHAIN; ++ks) {
      uint32_t ah[4], al[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_tf32(q.a[ks][i], ah[i], al[i]);
#pragma unroll
      for (int jp = 0; jp < NT / 2; ++jp) {
        uint32_t b[4], bh[4], bl[4];
        ldsm_x4_g(b, keys + R::at(16 * jp + (m >> 1) * 8 + r, 2 * ks + (m & 1)));
#pragma unroll
        for (int i = 0; i < 4; ++i) split_tf32(b[i], bh[i], bl[i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_tf32(low[2 * jp + h], al, bh[2 * h], bh[2 * h + 1]);
          mma_tf32(low[2 * jp + h], ah, bl[2 * h], bl[2 * h + 1]);
          mma_tf32(high[2 * jp + h], ah, bh[2 * h], bh[2 * h + 1]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] += high[j][e];
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[j][e] += low[j][e];
}

// o[n][.] += p . value rows of the tile at `vals` (p in the layout of s).
// bf16: p goes in as two bf16 parts, hi + lo, so that the weights keep 16
// bits; the second product is free while the tile waits for memory. An infinite
// value meets parts of either sign or 0 and comes out as NaN.
// HALF: rows g + 8 do not exist, their weights are taken as zero.
template <int D, int NT, bool HALF>
__device__ __forceinline__ void pv_tile(float (*o)[4], const float (*p)[4], uint32_t vals, int lane, __nv_bfloat16) {
  using R = Rows<__nv_bfloat16, D>;
  const int m = lane >> 3, r = lane & 7;
#pragma unroll
  for (int jp = 0; jp < NT / 2; ++jp) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (HALF && (i & 1)) {
        hi[i] = lo[i] = 0u;
        continue;
      }
      const float x = p[2 * jp + (i >> 1)][2 * (i & 1)], y = p[2 * jp + (i >> 1)][2 * (i & 1) + 1];
      hi[i] = pack_bf16(x, y);
      lo[i] = pack_bf16(x - __uint_as_float(hi[i] << 16), y - __uint_as_float(hi[i] & 0xffff0000u));
    }
#pragma unroll
    for (int np = 0; np < D / 16; ++np) {
      uint32_t b[4];
      ldsm_x4_t(b, vals + R::at(16 * jp + (m & 1) * 8 + r, 2 * np + (m >> 1)));
      mma_m16n8k16(o[2 * np], hi, b[0], b[1]);
      mma_m16n8k16(o[2 * np + 1], hi, b[2], b[3]);
      mma_m16n8k16(o[2 * np], lo, b[0], b[1]);
      mma_m16n8k16(o[2 * np + 1], lo, b[2], b[3]);
    }
  }
}

template <int D, int NT, bool HALF>
__device__ __forceinline__ void pv_tile(float (*o)[4], const float (*p)[4], uint32_t vals, int lane, float) {
  using R = Rows<float, D>;
  const int g = lane >> 2, c = lane & 3;
  // k index c of a product is key 2 c of its eight, c + 4 is key 2 c + 1, so
  // the scores' layout is the operand's layout.
  uint32_t ah[NT][4], al[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    split_tf32(__float_as_uint(p[j][0]), ah[j][0], al[j][0]);
    split_tf32(HALF ? 0u : __float_as_uint(p[j][2]), ah[j][1], al[j][1]);
    split_tf32(__float_as_uint(p[j][1]), ah[j][2], al[j][2]);
    split_tf32(HALF ? 0u : __float_as_uint(p[j][3]), ah[j][3], al[j][3]);
  }
#pragma unroll
  for (int n = 0; n < D / 8; ++n) {
    const int chunk = 2 * n + (g >> 2);
    float add[4] = {};
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t bh[2], bl[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        split_tf32(lds32(vals + R::at(8 * j + 2 * c + h, chunk) + 4 * (g & 3)), bh[h], bl[h]);
      mma_tf32(add, al[j], bh[0], bh[1]);
      mma_tf32(add, ah[j], bl[0], bl[1]);
      mma_tf32(add, ah[j], bh[0], bh[1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] += add[e];
  }
}

}  // namespace mrtdf
