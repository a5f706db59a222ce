// Paged attention over the 4-bit pool for few query rows: decode steps, short query blocks, and decode over a list of
// selected pages.
//
//   o_r = sum_k softmax_k(scale q_r . k_k) v_k over the keys k <= pos_r (of the listed pages, in the sparse form)
//
// In the reference's serving stack this is stock vLLM's paged decode kernel over a bf16 cache.  Here a step's time is
// the 2304-byte records of the pages (0.5625 B per element against 2), as long as the tensor pipe and the dequantisation
// keep up: per page and warp 64 conversions, 64 multiplications by scales, 16 MMAs.
//
// * One warp is one worker.  The four warps of a CTA take the pages of its split in turn; lane 0 fetches a page with one bulk copy
//   into the warp's own ring (6 records), so no CTA-wide barrier exists before the final merge.
// * The cache is the A operand of mma.sync m16n8k16, the queries the B operand: S^T = K Q^T (16 tokens x 8 rows) and
//   O^T = V^T P^T (16 dims x 8 rows).  With at most 8 query heads per KV head that is half the MMAs (16 a page) of the form that puts
//   queries in the 16 rows of A.  The contraction index may be permuted as long as A and B agree, so a lane (g = lane / 4,
//   t = lane % 4) takes 16 contiguous bytes of K row g: dims [32t, 32t + 32); and of V the scale group g of tokens 2t, 2t + 1
//   (+ 8): the record stores V by groups so that these 16 bytes are contiguous too, and both reads hit all banks once.
//   P^T in the layout of B is the transpose of S^T as it comes out: one movmatrix per 8 tokens.
// * The running maximum is raised only when a page exceeds it by 2^8 (P is f16, sums are fp32): one vote a page instead of six
//   shuffles.  Scores, sums and O are fp32; K, V are exact in f16; Q and P are rounded to f16 (2^-11, finer than bf16's 2^-8).
// * Splits of a context go to CTAs of their own and meet in attn4_merge_kernel.
#include "attention4_params.cuh"

namespace daser {
using namespace sm100;

constexpr int A4_WARPS = 4;
constexpr int A4_STAGES = 6;
constexpr int A4_RING = A4_STAGES * DASER_KV4_RECORD;  // per warp
constexpr int A4_OPITCH = 132;                         // floats per row of the merge buffer
constexpr float A4_RAISE_AT = 8.f;

__device__ uint32_t g_attn4_status = 0;  // bit 0: a bounded wait ran out

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int NT, bool SPARSE>
__global__ void __launch_bounds__(A4_WARPS * 32, NT == 1 ? 4 : 3)
attn4_kernel(const Attn4Params p) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t a4_smem[];
  __shared__ __align__(8) uint64_t s_bar[A4_WARPS][A4_STAGES];
  __shared__ uint32_t s_abort;
  __shared__ float s_m[A4_WARPS][ROWS], s_l[A4_WARPS][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.x, seq = blockIdx.y;
  const int tile = blockIdx.z / p.nsplit, sp = blockIdx.z % p.nsplit;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < A4_STAGES; ++s) mbar_init(&s_bar[warp][s], 1);
    if (warp == 0) s_abort = 0u;
    mbar_init_fence();
  }
  __syncthreads();  // s_abort and the barriers, before any wait looks at them
  pdl_enter();

  // rows of the tile: dense, 8 NT consecutive rows (query token major, then head of the group); sparse, the heads of one query
  const int G = p.G;
  const int q0 = p.q_start[seq];
  const int q_len = min(p.q_start[seq + 1], p.total_q) - q0;
  const int n_rows = SPARSE ? G : q_len * G;
  const int row0 = SPARSE ? 0 : tile * ROWS;
  const int tok0 = SPARSE ? tile : row0 / G;
  if (q0 < 0 || (SPARSE ? tile >= q_len : row0 >= n_rows)) return;  // uniform over the CTA
  const int ctx = p.ctx_lens[seq];
  const int first_pos = ctx - (p.q_start[seq + 1] - q0) + tok0;  // last key the first row may see
  const int last_tok = SPARSE ? tok0 : min((row0 + ROWS - 1) / G, q_len - 1);
  const int limit = first_pos + (last_tok - tok0) + 1;  // keys the last row sees
  const int32_t* list = SPARSE ? p.pages + ((int64_t)(q0 + tok0) * p.Hkv + kvh) * p.n_pages : nullptr;
  int n_all = limit > 0 ? (min(limit, p.max_blocks * DASER_KV4_TOKENS) + DASER_KV4_TOKENS - 1) / DASER_KV4_TOKENS : 0;
  if (SPARSE) {  // up to the last entry that names a page
    int last = -1;
    for (int i = lane; i < p.n_pages; i += 32)
      if (list[i] >= 0) last = i;
    n_all = __reduce_max_sync(0xffffffffu, last) + 1;
  }
  const int page_begin = sp * p.split_pages;
  const int page_end = min(page_begin + p.split_pages, n_all);
  const int mine = page_end - page_begin > warp ? (page_end - page_begin - warp + A4_WARPS - 1) / A4_WARPS : 0;  // pages of this warp

  // ---- page fetch ----
  // Logical pages of the next 32 fetches sit one per lane (page_of), read a window ahead of their use.
  uint8_t* ring = a4_smem + warp * A4_RING;
  const uint32_t ring_u32 = smem_u32(ring);
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks;
  auto window = [&](int i, int& logical, int& block) {  // this lane's entry of fetches i .. i + 31
    logical = -1;
    block = -1;
    const int k = i + lane;
    if (k < mine) {
      const int at = page_begin + warp + k * A4_WARPS;
      logical = SPARSE ? list[at] : at;
      if (logical >= 0 && logical < p.max_blocks && logical * DASER_KV4_TOKENS < limit) block = table[logical];
      else logical = -1;
      block = block < 0 ? 0 : (block >= p.num_blocks ? p.num_blocks - 1 : block);
    }
  };
  int log_cur, blk_cur, log_nxt, blk_nxt;  // windows of the fetches
  window(0, log_cur, blk_cur);
  window(32, log_nxt, blk_nxt);
  int use_cur = log_cur, use_nxt = log_nxt;  // windows of the uses, which run behind
  auto fetch = [&](int i) {  // all lanes; fetches run 0, 1, 2, ...
    if ((i & 31) == 0 && i > 0) {
      log_cur = log_nxt;
      blk_cur = blk_nxt;
      window(i + 32, log_nxt, blk_nxt);
    }
    const int blk = __shfl_sync(0xffffffffu, blk_cur, i & 31);
    if (lane == 0) {
      uint64_t* bar = &s_bar[warp][i % A4_STAGES];
      mbar_expect_tx(bar, DASER_KV4_RECORD);
      bulk_load(ring_u32 + (i % A4_STAGES) * DASER_KV4_RECORD, p.records + (int64_t)blk * p.stride_block + (int64_t)kvh * p.stride_head,
                DASER_KV4_RECORD, bar);
    }
  };
  int fetched = 0;
  for (; fetched < A4_STAGES - 1 && fetched < mine; ++fetched) fetch(fetched);

  // ---- queries: B fragments, scaled, f16.  Column g of n-tile nt is row row0 + 8 nt + g ----
  uint32_t qf[NT][16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + 8 * nt + g;
    const bool ok = r < n_rows;
    const int tq = SPARSE ? tok0 : r / G, h = SPARSE ? r : r % G;
    const __nv_bfloat16* qp = p.q + ((int64_t)(q0 + tq) * p.Hq + kvh * G + h) * ATT_D + 32 * t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if (ok) w = *reinterpret_cast<const uint4*>(qp + 8 * i);
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[nt][4 * i + e] = pack_half2(bf16_lo(ww[e]) * p.scale_log2, bf16_hi(ww[e]) * p.scale_log2);
    }
  }
  // last visible key of this lane's columns 2t, 2t + 1 of every n-tile
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[nt][e] = SPARSE ? first_pos : first_pos + (row0 + 8 * nt + 2 * t + e) / G - tok0;

  float o[NT][8][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
  }

  int used = 0;
  bool fail = false;
  for (; used < mine; ++used) {
    int logical = page_begin + warp + used * A4_WARPS;
    if (SPARSE) {
      // fetches run less than a window ahead: when a use enters window k, the fetches' next window is k + 1
      if ((used & 31) == 0) {
        if (used > 0) use_cur = use_nxt;
        use_nxt = log_nxt;
      }
      logical = __shfl_sync(0xffffffffu, use_cur, used & 31);
    }
    if (!mbar_wait(&s_bar[warp][used % A4_STAGES], (used / A4_STAGES) & 1, &s_abort)) { fail = true; break; }
    __syncwarp();
    const uint8_t* st = ring + (used % A4_STAGES) * DASER_KV4_RECORD;
    const int key0 = logical * DASER_KV4_TOKENS;
    const bool edge = key0 + DASER_KV4_TOKENS - 1 > first_pos;  // some key of the page is hidden from some row
    if (logical >= 0) {
      // ---- S^T = K Q^T ----
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
      {
        const uint4 ka = *reinterpret_cast<const uint4*>(st + g * 64 + t * 16);
        const uint4 kb = *reinterpret_cast<const uint4*>(st + (g + 8) * 64 + t * 16);
        const uint32_t sa = *reinterpret_cast<const uint16_t*>(st + DASER_KV4_KS + g * 8 + 2 * t);
        const uint32_t sb = *reinterpret_cast<const uint16_t*>(st + DASER_KV4_KS + (g + 8) * 8 + 2 * t);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          // f16 scale of group 2t (words 0, 1) or 2t + 1 (words 2, 3) in both halves
          const uint32_t s2a = bperm(sa, 0u, w < 2 ? 0x4040u : 0x4141u) << 7, s2b = bperm(sb, 0u, w < 2 ? 0x4040u : 0x4141u) << 7;
          uint32_t ha[4], hb[4];
          e2m1x8_to_f16x2(wa[w], ha);
          e2m1x8_to_f16x2(wb[w], hb);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ha[e] = hmul2_u32(ha[e], s2a);
            hb[e] = hmul2_u32(hb[e], s2b);
          }
#pragma unroll
          for (int e = 0; e < 4; e += 2)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], ha[e], hb[e], ha[e + 1], hb[e + 1], qf[nt][4 * w + e], qf[nt][4 * w + e + 1]);
        }
      }
      // ---- mask, running maximum, P ----
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key0 + g > pos[nt][e]) s[nt][e] = -INFINITY;
            if (key0 + g + 8 > pos[nt][e]) s[nt][2 + e] = -INFINITY;
          }
      }
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mx = fmaxf(s[nt][e], s[nt][2 + e]);
          raise |= mx > m[nt][e] + A4_RAISE_AT || (m[nt][e] == -INFINITY && mx > -INFINITY);
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(s[nt][e], s[nt][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(mx, m[nt][e]);
            const float al = m[nt][e] == -INFINITY ? 0.f : ex2f(m[nt][e] - mx);
            m[nt][e] = mx;
            l[nt][e] *= al;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[nt][j][e] *= al;
              o[nt][j][2 + e] *= al;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float b0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
        const float p0 = ex2f(s[nt][0] - b0), p1 = ex2f(s[nt][1] - b1), p2 = ex2f(s[nt][2] - b0), p3 = ex2f(s[nt][3] - b1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        pb[nt][0] = movmatrix_t(pack_half2(p0, p1));
        pb[nt][1] = movmatrix_t(pack_half2(p2, p3));
      }
      // ---- O^T += V^T P^T ----
      {
        const uint4 va = *reinterpret_cast<const uint4*>(st + DASER_KV4_V + g * 64 + t * 16);
        const uint4 vb = *reinterpret_cast<const uint4*>(st + DASER_KV4_V + 512 + g * 64 + t * 16);
        // f16 scales of tokens (2t, 2t + 1) and (2t + 8, 2t + 9)
        uint32_t s2a = bperm(*reinterpret_cast<const uint16_t*>(st + DASER_KV4_VS + g * 8 + 2 * t), 0u, 0x4140u) << 7;
        uint32_t s2b = bperm(*reinterpret_cast<const uint16_t*>(st + DASER_KV4_VS + 64 + g * 8 + 2 * t), 0u, 0x4140u) << 7;
        if (key0 + DASER_KV4_TOKENS > limit) {
          // tokens behind the last key: whatever the page's last owner left there must not meet P = 0 as a NaN
          const int left = limit - key0 - 2 * t;  // tokens 2t .. that exist
          s2a &= left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
          s2b &= left >= 10 ? 0xffffffffu : left == 9 ? 0xffffu : 0u;
        }
        const uint32_t w0[2] = {va.x, va.y}, w1[2] = {va.z, va.w}, w2[2] = {vb.x, vb.y}, w3[2] = {vb.z, vb.w};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          // bytes of (token 2t in the low half, token 2t + 1 in the high half): even dims, odd dims
          uint32_t he[4], ho[4], ge[4], go[4];
          e2m1x8_to_f16x2((w0[w] & 0x0f0f0f0fu) | ((w1[w] << 4) & 0xf0f0f0f0u), he);
          e2m1x8_to_f16x2(((w0[w] >> 4) & 0x0f0f0f0fu) | (w1[w] & 0xf0f0f0f0u), ho);
          e2m1x8_to_f16x2((w2[w] & 0x0f0f0f0fu) | ((w3[w] << 4) & 0xf0f0f0f0u), ge);
          e2m1x8_to_f16x2(((w2[w] >> 4) & 0x0f0f0f0fu) | (w3[w] & 0xf0f0f0f0u), go);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a0 = hmul2_u32(he[e], s2a), a1 = hmul2_u32(ho[e], s2a), a2 = hmul2_u32(ge[e], s2b), a3 = hmul2_u32(go[e], s2b);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * w + e], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane is done with this stage before it is filled again
    if (fetched < mine) fetch(fetched++);
  }
  if (fail) {
    // give the copies in flight their own bounded wait before the shared memory goes away
    for (int i = used + 1; i < fetched; ++i) {
      uint32_t none = 0u;
      mbar_wait(&s_bar[warp][i % A4_STAGES], (i / A4_STAGES) & 1, &none);
    }
    if (lane == 0) atomicOr(&g_attn4_status, 1u);
  }

  // ---- merge the four warps: O in shared memory over the rings ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      if (g == 0) {
        s_m[warp][8 * nt + 2 * t + e] = m[nt][e];
        s_l[warp][8 * nt + 2 * t + e] = l[nt][e];
      }
    }
  __syncthreads();  // rings are dead from here on
  float* buf = reinterpret_cast<float*>(a4_smem);  // [warp][row][A4_OPITCH]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* dst = buf + (warp * ROWS + 8 * nt + 2 * t + e) * A4_OPITCH + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(o[nt][j][e], o[nt][j][2 + e], o[nt][j + 1][e], o[nt][j + 1][2 + e]);
    }
  __syncthreads();
  const int c = threadIdx.x & 31;  // four dims; a warp finishes every fourth row
#pragma unroll
  for (int r = warp; r < ROWS; r += A4_WARPS) {
    const int row = row0 + r;
    if (row >= n_rows) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float lt = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) {
      const float f = s_m[w][r] == -INFINITY ? 0.f : ex2f(s_m[w][r] - base);
      const float4 v = *reinterpret_cast<const float4*>(buf + (w * ROWS + r) * A4_OPITCH + 4 * c);
      lt += f * s_l[w][r];
      acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
    }
    const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);  // no key: zeros; NaN stays
    const int tq = SPARSE ? tok0 : row / G, h = SPARSE ? row : row % G;
    const int64_t at = (int64_t)(q0 + tq) * p.Hq + kvh * G + h;
    if (p.nsplit == 1) {
      uint2 w2;
      w2.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w2.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + at * ATT_D + 4 * c) = w2;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (at * p.nsplit + sp) * ATT_D + 4 * c) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (c == 0) p.part_lse[at * p.nsplit + sp] = lt > 0.f ? mx + log2f(lt) : (lt == 0.f ? -INFINITY : lt);
    }
  }
}

// out = sum_s w_s O_s / sum_s w_s, w_s = 2^(lse_s - max): one CTA per output row.  The weights are made once, then its warps
// take the splits in turn, eight loads in flight each: a few rows with many splits (one long sequence on one KV head) are
// a matter of latency.  The order of the sums is fixed.
constexpr int MERGE_WARPS = 8;
constexpr int MERGE_MAX_SPLITS = 256;
__global__ void __launch_bounds__(MERGE_WARPS * 32)
attn4_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse, __nv_bfloat16* __restrict__ out,
                   const int32_t* __restrict__ q_start, int num_seqs, int Hq, int nsplit) {
  __shared__ float s_w[MERGE_MAX_SPLITS];
  __shared__ float s_max[MERGE_WARPS], s_sum[MERGE_WARPS];
  __shared__ __align__(16) float s_o[MERGE_WARPS][ATT_D];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_enter();
  if (row >= (int64_t)q_start[num_seqs] * Hq) return;  // a row behind the last sequence: nobody wrote its partials
  const float lse = tid < nsplit ? part_lse[row * nsplit + tid] : -INFINITY;
  const float* src = part_o + row * nsplit * ATT_D + 4 * lane;
  // NaN marks a row that saw one: it has to survive the maximum
  const bool nan = lse != lse;
  const float wm = warp_max(nan ? INFINITY : lse);
  if (lane == 0) s_max[warp] = wm;
  __syncthreads();
  float mx = s_max[0];
#pragma unroll
  for (int w = 1; w < MERGE_WARPS; ++w) mx = fmaxf(mx, s_max[w]);
  const float wt = nan ? NAN : (lse == -INFINITY ? 0.f : ex2f(lse - mx));
  s_w[tid] = wt;
  const float ws = warp_sum(wt);
  if (lane == 0) s_sum[warp] = ws;
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = warp; s0 < nsplit; s0 += 8 * MERGE_WARPS) {
    float4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u * MERGE_WARPS;
      x[u] = s < nsplit ? *reinterpret_cast<const float4*>(src + (int64_t)s * ATT_D) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + u * MERGE_WARPS;
      const float w = s < nsplit ? s_w[s] : 0.f;
      acc.x += w * x[u].x; acc.y += w * x[u].y; acc.z += w * x[u].z; acc.w += w * x[u].w;
    }
  }
  *reinterpret_cast<float4*>(&s_o[warp][4 * lane]) = acc;
  __syncthreads();
  if (tid < ATT_D) {
    float total = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < MERGE_WARPS; ++w) {
      total += s_sum[w];
      v += s_o[w][tid];
    }
    out[row * ATT_D + tid] = __float2bfloat16(total == 0.f ? 0.f : v / total);  // no key: zeros
  }
}

template <int NT, bool SPARSE>
static int launch_attn4(const Attn4Params& p, int tiles, cudaStream_t stream) {
  static bool configured[DASER_MAX_DEVICES] = {false};  // per device: the attribute is the device's
  constexpr int smem = A4_WARPS * A4_RING;
  static_assert(A4_WARPS * 8 * NT * A4_OPITCH * 4 <= smem, "the merge buffer lies over the rings");
  if (daser_first_use_on_device(configured)) {
    cudaError_t e = cudaFuncSetAttribute(attn4_kernel<NT, SPARSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
  }
  const int64_t z = (int64_t)tiles * p.nsplit;
  if (z > 65535 || p.num_seqs > 65535) return DASER_ERR_TOO_LARGE;
  return (int)launch_pdl(attn4_kernel<NT, SPARSE>, dim3(p.Hkv, p.num_seqs, (unsigned)z), dim3(A4_WARPS * 32), smem, stream, p);
}

static int fill_attn4(Attn4Params& p, const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                      int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                      int num_seqs, int total_q, int max_q_len, int Hq, int nsplit, int split_pages, float softmax_scale) {
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  const int Hkv = pool->heads_per_rank;
  if (Hq <= 0 || Hq % Hkv || num_seqs < 0 || total_q < 0 || max_q_len < 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (nsplit < 1 || split_pages < 1 || (nsplit > 1 && (!part_o || !part_lse))) return DASER_ERR_BAD_ARG;
  if (nsplit > MERGE_MAX_SPLITS) return DASER_ERR_TOO_LARGE;
  if (max_blocks > 0x7fffffff / DASER_KV4_TOKENS || total_q > 0x7fffffff / Hq) return DASER_ERR_TOO_LARGE;
  if (Hq / Hkv > 16) return DASER_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)part_o) % 16) return DASER_ERR_UNSUPPORTED;
  p.q = (const __nv_bfloat16*)q;
  p.out = (__nv_bfloat16*)out;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.records = pool->records[rank] + (int64_t)layer * pool->stride_layer;
  p.stride_block = pool->stride_block;
  p.stride_head = pool->stride_head;
  p.block_tables = block_tables;
  p.q_start = q_start;
  p.ctx_lens = ctx_lens;
  p.pages = nullptr;
  p.max_blocks = max_blocks;
  p.num_blocks = pool->num_blocks;
  p.num_seqs = num_seqs;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.n_pages = 0;
  p.nsplit = nsplit;
  p.split_pages = split_pages;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.total_q = total_q;
  return 0;
}

static int merge_attn4(const Attn4Params& p, cudaStream_t stream) {
  if (p.nsplit == 1) return 0;
  return (int)launch_pdl(attn4_merge_kernel, dim3((unsigned)(p.total_q * p.Hq)), dim3(MERGE_WARPS * 32), 0, stream, (const float*)p.part_o,
                         (const float*)p.part_lse, p.out, p.q_start, p.num_seqs, p.Hq, p.nsplit);
}

}  // namespace daser

// Rows from which a block of queries goes to the tcgen05 kernel: half of its 128-row tile.
#define A4_TC_MIN_ROWS 64

// Causal paged attention over the 4-bit pool.  part_o / part_lse: scratch of total_q * Hq * nsplit * (128 + 1) floats when nsplit > 1.
// A split is split_pages pages; nsplit * split_pages has to cover the longest context.
DASER_API int daser_paged_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                                        int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                        const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq, int nsplit,
                                        int split_pages, float softmax_scale, cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, nsplit, split_pages, softmax_scale))
    return e;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens) return DASER_ERR_BAD_ARG;
  const int64_t rows = (int64_t)max_q_len * p.G;
  int rc;
  if (rows >= A4_TC_MIN_ROWS) rc = daser_launch_attention4_tc(p, max_q_len, stream);
  else if (rows <= 8) rc = launch_attn4<1, false>(p, 1, stream);
  else rc = launch_attn4<2, false>(p, (int)((rows + 15) / 16), stream);
  return rc ? rc : merge_attn4(p, stream);
}

// The same over the pages listed for every (query row, KV head): pages int32 [total_q][Hkv][n_pages], ascending, -1 behind the last.
// A split is split_pages entries of the list.
DASER_API int daser_sparse_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                                         int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                         const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq,
                                         const int32_t* pages, int n_pages, int nsplit, int split_pages, float softmax_scale,
                                         cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, nsplit, split_pages, softmax_scale))
    return e;
  if (n_pages < 1 || (int64_t)nsplit * split_pages < n_pages) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens || !pages) return DASER_ERR_BAD_ARG;
  p.pages = pages;
  p.n_pages = n_pages;
  const int rc = p.G <= 8 ? launch_attn4<1, true>(p, max_q_len, stream) : launch_attn4<2, true>(p, max_q_len, stream);
  return rc ? rc : merge_attn4(p, stream);
}

// Non-zero once any CTA of the 4-bit decode kernels gave up on a bounded wait (synchronises the device).
DASER_API int daser_attention4_status(uint32_t* out) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, daser::g_attn4_status, sizeof(v));
  if (out) *out = v;
  return (int)e;
}
