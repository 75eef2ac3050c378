// Entries held in 4 bits: 32 neighbouring entries share a scale d, a code c in 0..15 stands for d (c - 8).
//
// Where the codes lie follows from what reads them.  A lane of a warp-wide 16 x 8 x 16 product wants registers of two entries that are
// neighbours along the summed axis, so a 32-bit word holds eight codes that one lane uses, the two of register r in nibbles r and r + 4:
//
//   key-like rows (summed along the row: keys, weights): a row of D entries has four quarters of D / 8 bytes, one per lane of a quad; word j of
//     quarter t holds entries 32 j + 8 t + i, i = 0..7, even i in nibble i / 2, odd i in nibble 4 + i / 2.
//   value-like rows (summed over positions): two positions share D bytes, eight chunks of D / 8 bytes; word j of chunk g holds entries
//     32 j + 4 g + r, r = 0..3, of the even position in nibble r and of the odd one in nibble 4 + r.  Chunk g lies at place g ^ x(pair): with
//     x the eight lanes of a phase of a shared-memory load meet all banks; without it two or four of them would share theirs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace hb {
namespace q4 {

constexpr int kGroup = 32;
constexpr int kPage = 64;
// one (page, kv head) of a plane: 64 rows of codes, then 64 rows of D / 32 bf16 scales
__host__ __device__ constexpr int code_bytes(int D) { return kPage * D / 2; }
__host__ __device__ constexpr int block_bytes(int D) { return kPage * D / 2 + kPage * (D / kGroup) * 2; }
__host__ __device__ constexpr int place_xor(int D, int pair) { return D == 128 ? (pair & 3) << 1 : (pair & 2) << 1; }

#ifdef __CUDACC__
// (a & m) | o in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t m, uint32_t o) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(m), "r"(o));
  return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t bfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// The four registers (c - 8 of nibbles r and r + 4, exact) of a word, two instructions each.  A byte (c + 16 c') in the low mantissa bits of 1024 is
// v = 1024 + c + 16 c'; with its low nibble replaced by 8 it is u = 1032 + 16 c'.  v - u = c - 8 and u / 16 - 72.5 = c' - 8, each in one step.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t v = __byte_perm(w, 0x64646464u, h ? 0x4341 : 0x4240), u = and_or(v, 0xfff0fff0u, 0x00080008u);
    a[2 * h] = hsub2(v, u);
    a[2 * h + 1] = hfma2(u, 0x2c002c00u, 0xd488d488u);
  }
}
// As bf16: seven mantissa bits, c in the lowest of 128
__device__ __forceinline__ void codes_bf16(uint32_t w, uint32_t (&a)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) a[r] = bfma2(and_or(w >> (4 * r), 0x000f000fu, 0x43004300u), 0x3f803f80u, 0xc308c308u);  // - 136
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same from zero
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit entries, lane 4 g + t holding row g, columns 2 t and 2 t + 1: transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
#endif

}  // namespace q4
}  // namespace hb
