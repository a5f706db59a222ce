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
  int total_q;
  int max_q_len;                // query tokens of a sequence beyond it are left alone (decode: `shared` has no place for them)
};

__device__ __forceinline__ float ex2f(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t bperm(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

}  // namespace daser

// Chunked prefill over the 4-bit pool (attention4_tc.cu): one CTA per 128 query rows of a KV head and per split.
int daser_launch_attention4_tc(const daser::Attn4Params& p, int max_q_len, cudaStream_t stream);
