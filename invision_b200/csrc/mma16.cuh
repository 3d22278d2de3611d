// mma16.cuh -- warp-level pieces that the 4-bit kernels share: m16n8k16 products with fp16 operands
// and fp32 sums, m16n8k32 products of bytes with 32-bit sums, an 8 x 8 transpose in registers,
// unpacking, untiled bulk copies and reads of a cluster's shared memory.
//
// mma.sync rather than tcgen05: a code has to be unpacked in registers and its group's scale has to
// meet the fp32 sum of that group alone, so both operands and accumulators live in registers.  The
// tensor pipe is 23 to 26% busy in the linear and in long decodes, 36% in a chunk of 128 queries.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace envg {

ENVG_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
// The same from a zero accumulator.
ENVG_DEV void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(0.0f));
}
// Transpose of an 8 x 8 matrix of halves; thread 4 r + c holds row r, columns 2 c and 2 c + 1.
ENVG_DEV uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
ENVG_DEV uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
ENVG_DEV __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// 2^x for softmax weights: within about 2^-22, and 0 where it would be a denormal.
ENVG_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (v & mask) | magic in one instruction: both constants stay in registers.
ENVG_DEV uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(magic));
  return r;
}
ENVG_DEV uint32_t in_register(uint32_t v) {
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
ENVG_DEV void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// Sixteen bytes from global to shared memory by this thread, in its current group of such copies.
ENVG_DEV void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(__cvta_generic_to_global(src)) : "memory");
}
ENVG_DEV void copy_group_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N of this thread's newest groups are still under way.
template <int N>
ENVG_DEV void copy_groups_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// m16n8k32 on 8-bit integers with 32-bit sums, 16-row operand unsigned, 8-column operand signed;
// from a zero accumulator where ZERO.
template <bool ZERO>
ENVG_DEV void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (ZERO)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with the 8-column operand unsigned, from the accumulator c; and with a signed 16-row
// operand from zero.
ENVG_DEV void mma_u8u8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
ENVG_DEV void mma_s8u8_zero(int (&d)[4], uint32_t a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%4,%4,%4}, {%5,%6}, {%7,%7,%7,%7};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a), "r"(b0), "r"(b1), "r"(0));
}
// A fixed-point value as four signed digits to the base 256, one to a byte.
ENVG_DEV uint32_t digits256(int x) { return ((uint32_t)x + 0x80808080u) ^ 0x80808080u; }
// The power of two e that takes a row's largest magnitude to [2^29, 2^30), where it and all smaller
// fp32 values down to 2^-6 of it are held exactly.  At most 149, which makes every fp32 number an
// integer: below 2^-120 nothing is rounded at all.
ENVG_DEV int fixed_exp(float top) {
  const int field = (int)(__float_as_uint(top) >> 23);
  return field == 255 ? 0 : min(149, 156 - field);
}
ENVG_DEV float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
ENVG_DEV float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// The power of two e that takes a row's largest magnitude to [2^14, 2^15) (at most 2^126; 0 for an
// infinity, whose row ends non-finite anyway), and 2^e.
ENVG_DEV int scale_exp(float top) {
  const int field = (int)(__float_as_uint(top) >> 23);
  return field == 255 ? 0 : min(126, 141 - field);
}
ENVG_DEV float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
// 2^-e for the e of fixed_exp: from 127 on a denormal, which holds it exactly.
ENVG_DEV float fixed_unit(int e) { return e <= 126 ? pow2(-e) : __int_as_float(1 << (149 - e)); }

// n / d for 0 <= n < 2^32 by a multiplication (Granlund and Montgomery, PLDI 1994).
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t by) : d(by), mul(0), shift(0) {
    while (shift < 32 && (1ull << shift) < by) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
  ENVG_DEV uint32_t div(uint32_t n) const {
    const uint32_t t = __umulhi(mul, n);
    return shift ? (t + ((n - t) >> 1)) >> (shift - 1) : n;
  }
};

// Four consecutive floats, as one access where `vec` (the address is 16-byte aligned).
ENVG_DEV float4 ld_f4(const float* p, bool vec) {
  if (vec) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}
ENVG_DEV void st_f4(float* p, float4 v, bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
  }
}

}  // namespace envg
