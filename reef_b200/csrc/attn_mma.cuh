// attn_mma.cuh -- warp-level pieces shared by the int8 cache attention kernels
// (decode_attn.cu: one query per sequence; tree_attn.cu: drafted tokens).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace reef {

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// D (16x8 s32) += A (16x32 s8, row) x B (32x8 s8, col)
__device__ __forceinline__ void mma_s8_16832(int (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D (16x8 f32) += A (16x16 f16, row) x B (16x8 f16, col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
      "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A word of an ldmatrix .trans over int8 pairs: bytes (k, d), (k, d+1),
// (k+1, d), (k+1, d+1).  Out: the f16 pairs {(k, d), (k+1, d)} and
// {(k, d+1), (k+1, d+1)}, each value v + 1152 exactly (byte v ^ 0x80 = v +
// 128 as the mantissa under the exponent byte 0x64, i.e. 1024 + v + 128).
__device__ __forceinline__ void split_biased(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t u = w ^ 0x80808080u;
  even = __byte_perm(u, 0x64646464u, 0x4240);
  odd = __byte_perm(u, 0x64646464u, 0x4341);
}

// 2^x (ex2.approx.ftz: 2 ulp; -inf -> 0, results below 2^-126 flush to 0)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// int32 -> fp32, exact for |v| < 2^22 (an int8 dot over 128 dims is at most
// 128 * 127 * 127 < 2^21): v + 1.5 * 2^23 as float bits, minus 1.5 * 2^23
__device__ __forceinline__ float small_i2f(int v) {
  return __fadd_rn(__int_as_float(v + 0x4B400000), -12582912.0f);
}

// byte offset of (row, 16-byte chunk) in a tile written by TMA with the
// 128-byte swizzle (rows of 128 bytes, 1024-aligned tile)
__device__ __forceinline__ uint32_t sw128(int row, int chunk) {
  return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}

}  // namespace reef
