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

// The largest magnitude as bits: integer order is float order, and puts infinities and NaNs on top.
template <int N>
__device__ __forceinline__ uint32_t fp4_absmax_bits(const float (&x)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t absmax_bits) {
  if (absmax_bits >= 0x7f800000u) return 255u;
  const float t = fminf(__fmul_rn(__uint_as_float(absmax_bits), 1.0f / 6.0f), 10240.f);
  const uint32_t b = __half_as_ushort(__float2half_rn(t));
  return (b + 63u + ((b >> 7) & 1u)) >> 7;
}

// x / s, correctly rounded, as two fused corrections of x * (1 / s): with inv the correctly rounded
// reciprocal and q within one unit of the quotient, q + r * inv rounds correctly (P. Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990).  x * inv alone is not enough: 3.5 * 1.875 / 1.875 would come out
// above the border between 3 and 4.
__device__ __forceinline__ float fp4_quotient(float x, float s, float inv) {
  const float q = __fmul_rn(x, inv);
  return __fmaf_rn(__fmaf_rn(-q, s, x), inv, q);
}

template <int N>
__device__ __forceinline__ void fp4_encode(const float (&x)[N], uint32_t scale_byte, uint32_t (&codes)[N / 8]) {
  const float s = fp4_scale(scale_byte);
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fp4_quotient(x[i], s, inv);
#pragma unroll
  for (int i = 0; i < N / 8; ++i) codes[i] = floats_to_e2m1x8(y + 8 * i);
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
