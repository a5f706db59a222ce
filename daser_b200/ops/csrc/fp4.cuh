// The 4-bit codec (fp4b16) in registers, shared by the kernels of the 4-bit pool.
//
// A group of 16 dims holds x = s * v with v in e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one 8-bit
// scale.  A scale is never negative, so its byte is the upper 8 of the 15 magnitude bits of an f16: five exponent
// and three mantissa bits, decoded by one shift (f16 bits = byte << 7).  That covers 2^-17 .. 10240 without a second
// scale per tensor, which a scale in e4m3 (smallest 2^-9) would need, and s * v has six significant bits: it is
// exact in bf16, and in f16 down to s = 2^-17.
//
//   s = round4(f16(absmax * fl(1/6))), four significant bits, ties to even, at most 10240
//   v = e2m1(fl(x / s)), ties to even, saturating at 6
//
// Rounding s to nearest (not up) lets the largest value of a group saturate by at most half a scale step (6 %),
// which is less than the half step of 1 that e2m1 has above 4.  A group with an infinity or a NaN gets scale
// byte 255 and reads back as NaN: nothing that is not finite turns into a number.
#pragma once
#include "common.cuh"
#include "kv4.h"

namespace daser {

__device__ __forceinline__ float fp4_scale(uint32_t byte) {
  return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// Four bytes of codes -> eight values as four f16x2 (the low half of a byte in the low half).
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

// Eight floats -> four bytes of codes (round to nearest even, saturating).
__device__ __forceinline__ uint32_t floats_to_e2m1x8(const float* x) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}\n"
      : "=r"(w)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return w;
}

// Two floats a register pair: one instruction for both, each rounded as the scalar one would be.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// (a, b) rotated: a' = a c - b s, b' = b c + a s, every product and sum rounded (the CPU oracle's bits).  The sums are scalar: a packed
// sum of packed products comes out of the compiler as one fused operation.
__device__ __forceinline__ void rotate2(uint64_t& a, uint64_t& b, uint64_t c, uint64_t s) {
  float ac0, ac1, bs0, bs1, bc0, bc1, as0, as1;
  unpair2(mul2(a, c), ac0, ac1);
  unpair2(mul2(b, s), bs0, bs1);
  unpair2(mul2(b, c), bc0, bc1);
  unpair2(mul2(a, s), as0, as1);
  a = pair2(__fsub_rn(ac0, bs0), __fsub_rn(ac1, bs1));
  b = pair2(__fadd_rn(bc0, as0), __fadd_rn(bc1, as1));
}

// The largest magnitude, NaN if there is one.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int N>
__device__ __forceinline__ float fp4_absmax(const uint64_t (&x)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float a, b;
    unpair2(x[i], a, b);
    m = max3_nan(m, fabsf(a), fabsf(b));
  }
  return m;
}

__device__ __forceinline__ uint32_t fp4_scale_byte(float absmax) {
  if (!(absmax < INFINITY)) return 255u;
  const float t = fminf(__fmul_rn(absmax, 1.0f / 6.0f), 10240.f);
  const uint32_t b = __half_as_ushort(__float2half_rn(t));
  return (b + 63u + ((b >> 7) & 1u)) >> 7;
}

// Pairs of values -> codes; inv = fp4_inverse(scale_byte).  The quotient x / s is correctly rounded, as two fused corrections of x * (1 / s): with inv the
// correctly rounded reciprocal and q within one unit of the quotient, q + (x - q s) * inv rounds correctly (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  x * inv alone is not enough:
// 3.5 * 1.875 / 1.875 would come out above the border between 3 and 4.
__device__ __forceinline__ float fp4_inverse(uint32_t scale_byte) {
  const float s = fp4_scale(scale_byte);
  return s > 0.f ? __frcp_rn(s) : 0.f;
}
template <int N>
__device__ __forceinline__ void fp4_encode(const uint64_t (&x)[N], uint32_t scale_byte, float inv, uint32_t (&codes)[N / 4]) {
  const float s = fp4_scale(scale_byte);
  const uint64_t inv2 = pair2(inv, inv), ns2 = pair2(-s, -s);
  float y[2 * N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint64_t q = mul2(x[i], inv2);
    unpair2(fma2(fma2(q, ns2, x[i]), inv2, q), y[2 * i], y[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) codes[i] = floats_to_e2m1x8(y + 8 * i);
}

// 8 codes and their scale byte -> floats (exact).
__device__ __forceinline__ void fp4_decode8(uint32_t w, uint32_t scale_byte, float* x) {
  uint32_t h[4];
  e2m1x8_to_f16x2(w, h);
  const float s = fp4_scale(scale_byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    x[2 * i] = __fmul_rn(f.x, s);
    x[2 * i + 1] = __fmul_rn(f.y, s);
  }
}

// Byte offset, inside a record, of the codes of (kv, token, 8-dim piece p = dim / 8) and of (kv, token, group).
__device__ __forceinline__ int kv4_code_at(int kv, int tok, int p) {
  return kv == 0 ? tok * 64 + p * 4 : DASER_KV4_V + (tok >> 3) * 512 + (p >> 1) * 64 + (tok & 7) * 8 + (p & 1) * 4;
}
__device__ __forceinline__ int kv4_scale_at(int kv, int tok, int g) {
  return kv == 0 ? DASER_KV4_KS + tok * 8 + g : DASER_KV4_VS + (tok >> 3) * 64 + g * 8 + (tok & 7);
}

// Host-side checks every entry point of the 4-bit pool makes.
static inline int kv4_check_pool(const DaserKV4Pool* p, int layer, int rank) {
  if (!p || p->n_ranks < 1 || p->n_ranks > DASER_MAX_RANKS || p->num_blocks <= 0 || p->heads_per_rank <= 0) return DASER_ERR_BAD_ARG;
  if (layer < 0 || layer >= p->num_layers || rank < 0 || rank >= p->n_ranks || !p->records[rank]) return DASER_ERR_BAD_ARG;
  if ((p->stride_layer | p->stride_block | p->stride_head | (int64_t)(uintptr_t)p->records[rank]) % 16) return DASER_ERR_UNSUPPORTED;
  return 0;
}

}  // namespace daser
