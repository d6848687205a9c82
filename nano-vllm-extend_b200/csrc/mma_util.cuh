// Warp-level tensor-core helpers (mma.sync / ldmatrix) for products whose
// operands or results live in registers: the tree operators' small tiles.
#pragma once

#include "common.cuh"

namespace gdn {
namespace mm {

// D[16x8] += A[16x16] B[16x8], bf16 operands, fp32 accumulators.  With g =
// lane / 4 and t = lane % 4: a0/a1/a2/a3 hold (row g, k 2t..), (row g + 8, k
// 2t..), (row g, k 2t + 8..), (row g + 8, k 2t + 8..); b0/b1 (k 2t.., column g),
// (k 2t + 8.., column g); d0..d3 (row g, column 2t), (g, 2t + 1), (g + 8, 2t),
// (g + 8, 2t + 1).
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D[16x8] += A[16x8] B[8x8], tf32 operands (fp32 registers, the low 13 bits
// ignored), fp32 accumulators: a0..a3 hold (row g, k t), (g + 8, t), (g, t + 4),
// (g + 8, t + 4); b0, b1 (k t, column g), (t + 4, g); d as above.
__device__ __forceinline__ void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x = hi + lo as operands of tf32 products: hi the 11 bits that a product keeps,
// lo the rest, of which it keeps 11 more.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

// Four 8x8 bf16 matrices; lanes 8i..8i+7 give the row addresses of matrix i.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// (lo, hi) = h + l with both parts bf16: 16 bits of the fp32 mantissas.
__device__ __forceinline__ void split2(float lo, float hi, uint32_t& h, uint32_t& l) {
  h = pack2(lo, hi);
  l = pack2(lo - __uint_as_float(h << 16), hi - __uint_as_float(h & 0xffff0000u));
}

}  // namespace mm
}  // namespace gdn
