// Shared by the attention kernels over the 4-bit pool: launch parameters and small PTX helpers.
#pragma once
#include "attention_params.cuh"
#include "fp4.cuh"
#include "tcgen05.cuh"

namespace daser {

struct Attn4Params {
  const __nv_bfloat16* q;       // [Tq, Hq, 128]
  __nv_bfloat16* out;           // [Tq, Hq, 128]
  float* part_o;                // partial outputs, 128 floats each, normalised ...
  float* part_lse;              // ... and their log2-sum-exp (where they lie: attention4.cu)
  int2* shared;                 // decode: of every item, the first CTA that has a part of it, and how many have
  const uint8_t* records;       // the layer's records
  int64_t stride_block, stride_head;
  const int32_t* block_tables;  // [num_seqs, max_blocks]
  const int32_t* q_start;       // [num_seqs + 1]
  const int32_t* ctx_lens;      // [num_seqs]
  const int32_t* pages;         // sparse: [Tq, Hkv, n_pages] logical pages, ascending, -1 behind the last
  int max_blocks, num_blocks, num_seqs, Hq, Hkv, G;
  int n_pages;                  // sparse: pages listed per (query row, KV head)
  int workers;                  // decode: CTAs that share all pages evenly, 0 = one CTA per item
  int tiles;                    // decode: row tiles of the longest query block
  int nsplit, split_pages;      // prefill: splits of a context, of split_pages pages each
  float scale_log2;             // softmax scale * log2(e)
  uint32_t q_lo, q_hi;          // bf16 bits: a row whose largest query is in [q_lo, q_hi) goes into f16 with that scale
  int total_q;
  int max_q_len;                // query tokens of a sequence beyond it are left alone (decode: `shared` has no place for them)
};

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Queries are scaled and rounded to f16, which has 11 bits between 2^-14 and 65504.  A row whose largest value would end up outside
// [2^-14, 2^15) gets a scale of its own, a power of two away, that brings it to 2^12, and its scores are multiplied by that power; the scores
// of a row with an infinity by NaN.  (Queries below 2^-112 keep fewer bits; beyond a factor of 2^120 scores leave fp32.)
__device__ __forceinline__ uint32_t top_bf16(uint32_t seen, const uint4& w) {  // of either half: the largest magnitude (of what is a number)
  auto up = [](uint32_t a, uint32_t b) {
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tabs.bf16x2 t, %2;\n\tmax.bf16x2 %0, %1, t;\n\t}\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
  };
  return up(up(up(up(seen, w.x), w.y), w.z), w.w);
}
__device__ __forceinline__ uint32_t top_half(uint32_t top) { return max(top & 0xffffu, top >> 16); }
__device__ __forceinline__ bool odd_row(uint32_t top, uint32_t q_lo, uint32_t q_hi) { return top - q_lo >= q_hi - q_lo && top != 0u; }
struct RowScale {
  float scale, factor;  // of the row's queries; of its scores
};
__device__ __forceinline__ RowScale row_scale(uint32_t top, float scale_log2, uint32_t q_lo, uint32_t q_hi) {
  if (!odd_row(top, q_lo, q_hi)) return {scale_log2, 1.f};
  if (top >= 0x7f80u) return {scale_log2, NAN};
  const int se = (int)(__float_as_uint(scale_log2) >> 23 & 0xffu) - 127;
  int e = (int)(top >> 7) - 127 + se - 12;
  e = max(max(-120, se - 125), min(e, 120));
  return {scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23), __uint_as_float((uint32_t)(127 + e) << 23)};
}
__device__ __forceinline__ uint32_t bperm(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

}  // namespace daser

// Chunked prefill over the 4-bit pool (attention4_tc.cu): one CTA per 128 query rows of a KV head and per split.
int daser_launch_attention4_tc(const daser::Attn4Params& p, int max_q_len, cudaStream_t stream);
