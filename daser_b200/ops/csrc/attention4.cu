// Paged attention over the 4-bit pool for few query rows: decode steps, short query blocks, and decode over a list of
// selected pages.
//
//   o_r = sum_k softmax_k(scale q_r . k_k) v_k over the keys k <= pos_r (of the listed pages, in the sparse form)
//
// In the reference's serving stack this is stock vLLM's paged decode kernel over a bf16 cache.  Here a step's time is
// the 2304-byte records of the pages (0.5625 B per element against 2), as long as the tensor pipe and the dequantisation
// keep up: per page and warp 64 conversions, 64 multiplications by scales, 16 MMAs.
//
// * One warp is one worker.  The eight warps of a CTA take pairs of pages of its range in turn; two lanes fetch a pair with one bulk copy
//   each into the warp's own ring (3 pairs), so no CTA-wide barrier exists before the merge of the warps.
// * An item is (sequence, tile of query rows, KV head).  With many pages a fixed number of CTAs (two a SM) shares the pages of ALL
//   items evenly: CTA c takes [c T / W, (c + 1) T / W) of the T pages in item order, whatever the lengths are, so that
//   all finish together (splits of a fixed length left the last wave a third empty: 73 us against 5x us at 8 sequences of
//   16k - 32k tokens).  An item that lies in several CTAs is put together by attn4_merge_kernel from their partial results.
// * The cache is the A operand of mma.sync m16n8k16, the queries the B operand: S^T = K Q^T (16 tokens x 8 rows) and
//   O^T = V^T P^T (16 dims x 8 rows).  With at most 8 query heads per KV head that is half the MMAs (16 a page) of the form that puts
//   queries in the 16 rows of A.  The contraction index may be permuted as long as A and B agree, so a lane (g = lane / 4,
//   t = lane % 4) takes 16 contiguous bytes of K row g: dims [32t, 32t + 32); and of V the scale group g of tokens 2t, 2t + 1
//   (+ 8): the record stores V by groups so that these 16 bytes are contiguous too, and both reads hit all banks once.
//   P^T in the layout of B is the transpose of S^T as it comes out: one movmatrix per 8 tokens.
// * The running maximum is raised only when a page exceeds it by 2^8 (P is f16, sums are fp32): one vote a page instead of six
//   shuffles.  Scores, sums and O are fp32; K, V are exact in f16; Q and P are rounded to f16 (2^-11, finer than bf16's 2^-8).
#include "attention4_params.cuh"

namespace daser {
using namespace sm100;

constexpr int A4_WARPS = 8;
constexpr int A4_PAIR = 2 * DASER_KV4_RECORD;
constexpr int A4_STAGES = 3;                           // pairs of pages
constexpr int A4_RING = A4_STAGES * A4_PAIR;           // per warp
constexpr int A4_OPITCH = 132;                         // floats per row of the merge buffer
constexpr float A4_RAISE_AT = 8.f;

__device__ uint32_t g_attn4_status = 0;  // bit 0: a bounded wait ran out

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a chain: d = a b + (i0, i1, i0, i1).
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                              float i0, float i1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(i0), "f"(i1));
}
// h * (lo, lo) or h * (hi, hi) of s: the broadcast is part of the multiplication.
__device__ __forceinline__ uint32_t hmul2_lo(uint32_t h, uint32_t s) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&h), __low2half2(*reinterpret_cast<__half2*>(&s)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2_hi(uint32_t h, uint32_t s) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&h), __high2half2(*reinterpret_cast<__half2*>(&s)));
  return *reinterpret_cast<const uint32_t*>(&r);
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

// Pages of an item of the dense form: (query rows [row0, row0 + ROWS) of a sequence of q_len new tokens and ctx keys) sees the keys
// below limit.  Every item counts one page at least: somebody has to write its zeros.
__device__ __forceinline__ int item_limit(int q_len, int q_all, int ctx, int G, int row0, int rows) {
  return ctx - q_all + min((row0 + rows - 1) / G, q_len - 1) + 1;
}
__device__ __forceinline__ int item_pages(const Attn4Params& p, int limit) {
  return limit > 0 ? (min(limit, p.max_blocks * DASER_KV4_TOKENS) + DASER_KV4_TOKENS - 1) / DASER_KV4_TOKENS : 0;
}
struct SeqInfo {
  int q0, q_all, q_len, ctx;  // first row, new tokens, those that have a row, keys
};
__device__ __forceinline__ SeqInfo seq_info(const Attn4Params& p, int seq) {
  SeqInfo s;
  s.q0 = p.q_start[seq];
  const int q1 = p.q_start[seq + 1];
  s.q_all = q1 - s.q0;
  s.q_len = s.q0 < 0 ? 0 : max(0, min(q1, p.total_q) - s.q0);
  s.ctx = p.ctx_lens[seq];
  return s;
}
// Pages of all items of a sequence.
template <int ROWS, bool SPARSE>
__device__ __forceinline__ int64_t seq_pages(const Attn4Params& p, int seq) {
  const SeqInfo s = seq_info(p, seq);
  if (SPARSE) return (int64_t)s.q_len * p.Hkv * p.n_pages;
  int64_t n = 0;
  for (int row0 = 0; row0 < s.q_len * p.G; row0 += ROWS) n += max(1, item_pages(p, item_limit(s.q_len, s.q_all, s.ctx, p.G, row0, ROWS)));
  return n * p.Hkv;
}
__device__ __forceinline__ int64_t warp_sum_i64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Pages of all sequences below `upto` (every lane of a warp calls it, and gets the sum).
template <int ROWS, bool SPARSE>
__device__ __forceinline__ int64_t pages_below(const Attn4Params& p, int upto) {
  int64_t n = 0;
  for (int s = threadIdx.x & 31; s < upto; s += 32) n += seq_pages<ROWS, SPARSE>(p, s);
  return warp_sum_i64(n);
}
// The CTA that owns page x of T when W share them: CTA c owns [floor(c T / W), floor((c + 1) T / W)).
__device__ __forceinline__ int owner_of(int64_t x, int64_t T, int W) { return (int)(((x + 1) * W - 1) / T); }

template <int NT, bool SPARSE>
__global__ void __launch_bounds__(A4_WARPS * 32, NT == 1 ? 2 : 1)
attn4_kernel(const Attn4Params p) {
  constexpr int ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t a4_smem[];
  __shared__ __align__(8) uint64_t s_bar[A4_WARPS][A4_STAGES];
  __shared__ uint32_t s_abort;
  __shared__ float s_m[A4_WARPS][ROWS], s_l[A4_WARPS][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < A4_STAGES; ++s) mbar_init(&s_bar[warp][s], 1);
    if (warp == 0) s_abort = 0u;
    mbar_init_fence();
  }
  __syncthreads();  // s_abort and the barriers, before any wait looks at them
  pdl_enter();

  const int G = p.G;
  // ---- where this CTA starts: item (seq, tile, kvh), page p0 of it, and how many pages it takes ----
  int seq, tile, kvh, p0 = 0;
  int64_t todo = 1;  // pages left to this CTA (one CTA per item: the whole item, see below)
  SeqInfo si;
  if (p.workers == 0) {
    kvh = blockIdx.x;
    seq = blockIdx.y;
    tile = blockIdx.z;
    si = seq_info(p, seq);
    if (SPARSE ? tile >= si.q_len : tile * ROWS >= si.q_len * G) return;  // uniform over the CTA
  } else {
    const int64_t T = pages_below<ROWS, SPARSE>(p, p.num_seqs);
    int64_t at = (int64_t)blockIdx.x * T / p.workers;
    todo = (int64_t)(blockIdx.x + 1) * T / p.workers - at;
    if (todo == 0) return;
    // the sequence that page `at` is in
    seq = 0;
    for (int base = 0;; base += 32) {
      int64_t mine = base + lane < p.num_seqs ? seq_pages<ROWS, SPARSE>(p, base + lane) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, upto > at);
      if (behind != 0u) {
        const int who = __ffs(behind) - 1;
        seq = base + who;
        at -= __shfl_sync(0xffffffffu, upto - mine, who);
        break;
      }
      at -= __shfl_sync(0xffffffffu, upto, 31);
    }
    si = seq_info(p, seq);
    for (tile = 0;; ++tile) {
      const int n = SPARSE ? p.n_pages : max(1, item_pages(p, item_limit(si.q_len, si.q_all, si.ctx, G, tile * ROWS, ROWS)));
      if (at < (int64_t)n * p.Hkv) {
        kvh = (int)(at / n);
        p0 = (int)(at - (int64_t)kvh * n);
        break;
      }
      at -= (int64_t)n * p.Hkv;
    }
  }
  uint8_t* ring = a4_smem + warp * A4_RING;
  const uint32_t ring_u32 = smem_u32(ring);
  // the ring of this warp, over all items: where the next record goes, where the next one to use is, and its phase
  int put = 0, get = 0;
  uint32_t phase = 0;

  while (todo > 0) {
  // ---- the item ----
  // rows: dense, ROWS consecutive rows (query token major, then head of the group); sparse, the heads of one query token
  const int q0 = si.q0;
  const int n_rows = SPARSE ? G : si.q_len * G;
  const int row0 = SPARSE ? 0 : tile * ROWS;
  const int tok0 = SPARSE ? tile : row0 / G;
  const int first_pos = si.ctx - si.q_all + tok0;  // last key the first row may see
  const int limit = SPARSE ? first_pos + 1 : item_limit(si.q_len, si.q_all, si.ctx, G, row0, ROWS);  // keys the last row sees
  const int32_t* list = SPARSE ? p.pages + ((int64_t)(q0 + tok0) * p.Hkv + kvh) * p.n_pages : nullptr;
  const int real = SPARSE ? p.n_pages : item_pages(p, limit);
  const int n_item = max(1, real);
  if (p.workers == 0) todo = n_item;
  const int p1 = (int)min((int64_t)n_item, p0 + todo);
  const int page_begin = p0, page_end = min(p1, real);
  const int n_pairs = (page_end - page_begin + 1) >> 1;  // negative or zero: nothing to read
  const int mine = n_pairs > warp ? (n_pairs - warp + A4_WARPS - 1) / A4_WARPS : 0;  // pairs of this warp: warp, warp + 8, ...

  // ---- page fetch ----
  // Page k of this warp (k = 2 * pair + which) is entry k & 31 of window k / 32, one per lane: its logical page (negative: skipped)
  // and its record's offset, read a window ahead of their use.
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks;
  auto window = [&](int w, int& logical, int64_t& offset) {
    const int k = 32 * w + lane;
    const int at = page_begin + 2 * (warp + (k >> 1) * A4_WARPS) + (k & 1);
    logical = -1;
    offset = 0;
    if ((k >> 1) < mine && at < page_end) {
      logical = SPARSE ? list[at] : at;
      if (logical >= 0 && logical < p.max_blocks && (int64_t)logical * DASER_KV4_TOKENS < limit) {
        int block = table[logical];
        block = block < 0 ? 0 : (block >= p.num_blocks ? p.num_blocks - 1 : block);
        offset = (int64_t)block * p.stride_block + (int64_t)kvh * p.stride_head;
      } else {
        logical = -1;
      }
    }
  };
  int log_cur, log_nxt;  // windows of the fetches
  int64_t off_cur, off_nxt;
  window(0, log_cur, off_cur);
  window(1, log_nxt, off_nxt);
  int use_cur = log_cur, use_nxt = log_nxt;  // windows of the uses, which run behind
  auto fetch = [&](int i) {  // all lanes; pairs 0, 1, 2, ...
    const int e = (2 * i) & 31;
    if (e == 0 && i > 0) {
      log_cur = log_nxt;
      off_cur = off_nxt;
      window((i >> 4) + 1, log_nxt, off_nxt);
    }
    const int from = e + (lane & 1);
    const int64_t off = __shfl_sync(0xffffffffu, off_cur, from);
    const bool there = __shfl_sync(0xffffffffu, log_cur, from) >= 0;
    const uint32_t pair = __ballot_sync(0xffffffffu, there) & 3u;
    uint64_t* bar = &s_bar[warp][put];
    if (lane == 0) mbar_expect_tx(bar, __popc(pair) * DASER_KV4_RECORD);
    __syncwarp();
    if (lane < 2 && there) bulk_load(ring_u32 + put * A4_PAIR + lane * DASER_KV4_RECORD, p.records + off, DASER_KV4_RECORD, bar);
    put = put == A4_STAGES - 1 ? 0 : put + 1;
  };
  int fetched = 0;
  for (; fetched < A4_STAGES && fetched < mine; ++fetched) fetch(fetched);

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

  // base: what the exponents are relative to: the running maximum, up to 2^8 behind it; 0 until the row has seen a key
  float o[NT][8][4], base[NT][2], l[NT][2];
  bool seen[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    base[nt][0] = base[nt][1] = 0.f;
    seen[nt][0] = seen[nt][1] = false;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
  }
  bool fresh = true;  // some row has seen no key yet

  // ---- a pair of pages at a time: their chains of dependent MMAs run side by side ----
  bool fail = false;
  int used = 0;
  for (; used < mine; ++used) {
    int key0[2];
    if (SPARSE) {
      // fetches run less than a window ahead: when a use enters window k, the fetches' next window is k + 1
      const int e = (2 * used) & 31;
      if (e == 0) {
        if (used > 0) use_cur = use_nxt;
        use_nxt = log_nxt;
      }
      key0[0] = __shfl_sync(0xffffffffu, use_cur, e);
      key0[1] = __shfl_sync(0xffffffffu, use_cur, e + 1);
    } else {
      key0[0] = page_begin + 2 * (warp + used * A4_WARPS);
      key0[1] = key0[0] + 1 < page_end ? key0[0] + 1 : -1;
    }
    // a page that is not there lies beyond every limit: its scores become -inf, its scales 0
    key0[0] = key0[0] < 0 ? 1 << 29 : key0[0] * DASER_KV4_TOKENS;
    key0[1] = key0[1] < 0 ? 1 << 29 : key0[1] * DASER_KV4_TOKENS;
    const uint8_t* st[2] = {ring + get * A4_PAIR, ring + get * A4_PAIR + DASER_KV4_RECORD};
    if (!mbar_wait(&s_bar[warp][get], phase, &s_abort)) { fail = true; break; }
    if (++get == A4_STAGES) { get = 0; phase ^= 1u; }
    __syncwarp();
    // some key of the pair is hidden from some row (pages are in ascending order)
    const bool special = max(key0[0], key0[1]) + DASER_KV4_TOKENS - 1 > first_pos;
    // ---- S^T - base = K Q^T - base: the tensor core takes the difference ----
    float s[2][NT][4];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4 ka = *reinterpret_cast<const uint4*>(st[x] + g * 64 + t * 16);
      const uint4 kb = *reinterpret_cast<const uint4*>(st[x] + (g + 8) * 64 + t * 16);
      // f16 scales of groups 2t (low half) and 2t + 1 of tokens g, g + 8
      const uint32_t sa = bperm(*reinterpret_cast<const uint16_t*>(st[x] + DASER_KV4_KS + g * 8 + 2 * t), 0u, 0x4140u) << 7;
      const uint32_t sb = bperm(*reinterpret_cast<const uint16_t*>(st[x] + DASER_KV4_KS + (g + 8) * 8 + 2 * t), 0u, 0x4140u) << 7;
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t ha[4], hb[4];
        e2m1x8_to_f16x2(wa[w], ha);
        e2m1x8_to_f16x2(wb[w], hb);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ha[e] = w < 2 ? hmul2_lo(ha[e], sa) : hmul2_hi(ha[e], sa);
          hb[e] = w < 2 ? hmul2_lo(hb[e], sb) : hmul2_hi(hb[e], sb);
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (w == 0 && e == 0) mma_f16_first(s[x][nt], ha[0], hb[0], ha[1], hb[1], qf[nt][0], qf[nt][1], -base[nt][0], -base[nt][1]);
            else mma_f16(s[x][nt], ha[e], hb[e], ha[e + 1], hb[e + 1], qf[nt][4 * w + e], qf[nt][4 * w + e + 1]);
          }
      }
    }
    if (special) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key0[x] + g > pos[nt][e]) s[x][nt][e] = -INFINITY;
            if (key0[x] + g + 8 > pos[nt][e]) s[x][nt][2 + e] = -INFINITY;
          }
    }
    // ---- raise the base where a score is more than 2^8 above it; P ----
    float top = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[x][nt][i]);
    if (__any_sync(0xffffffffu, fresh || top > A4_RAISE_AT)) {
      bool none = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[0][nt][e], s[0][nt][2 + e]), fmaxf(s[1][nt][e], s[1][nt][2 + e]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          // relative to the old base: to the first maximum wherever it lies, then upwards only
          const float up = mx == -INFINITY ? 0.f : (seen[nt][e] ? fmaxf(mx, 0.f) : mx);
          seen[nt][e] |= mx > -INFINITY;
          none |= !seen[nt][e];
          const float al = ex2f(-up);
          base[nt][e] += up;
          l[nt][e] *= al;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            s[x][nt][e] -= up;
            s[x][nt][2 + e] -= up;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[nt][j][e] *= al;
            o[nt][j][2 + e] *= al;
          }
        }
      fresh = __any_sync(0xffffffffu, none);
    }
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float e0 = ex2f(s[x][nt][0]), e1 = ex2f(s[x][nt][1]), e2 = ex2f(s[x][nt][2]), e3 = ex2f(s[x][nt][3]);
        l[nt][0] += e0 + e2;
        l[nt][1] += e1 + e3;
        pb[x][nt][0] = movmatrix_t(pack_half2(e0, e1));
        pb[x][nt][1] = movmatrix_t(pack_half2(e2, e3));
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4 va = *reinterpret_cast<const uint4*>(st[x] + DASER_KV4_V + g * 64 + t * 16);
      const uint4 vb = *reinterpret_cast<const uint4*>(st[x] + DASER_KV4_V + 512 + g * 64 + t * 16);
      // f16 scales of tokens (2t, 2t + 1) and (2t + 8, 2t + 9)
      uint32_t s2a = bperm(*reinterpret_cast<const uint16_t*>(st[x] + DASER_KV4_VS + g * 8 + 2 * t), 0u, 0x4140u) << 7;
      uint32_t s2b = bperm(*reinterpret_cast<const uint16_t*>(st[x] + DASER_KV4_VS + 64 + g * 8 + 2 * t), 0u, 0x4140u) << 7;
      if (special) {
        // tokens behind the last key: whatever the page's last owner left there must not meet P = 0 as a NaN
        const int left = limit - key0[x] - 2 * t;  // tokens 2t .. that exist
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
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * w + e], a0, a1, a2, a3, pb[x][nt][0], pb[x][nt][1]);
        }
      }
    }
    __syncwarp();  // every lane is done with this stage before it is filled again
    if (fetched < mine) fetch(fetched++);
  }
  if (fail) {
    // give the copies in flight their own bounded wait before the shared memory goes away (`get` is the one that gave up)
    for (int i = used + 1; i < fetched; ++i) {
      if (++get == A4_STAGES) { get = 0; phase ^= 1u; }
      uint32_t none = 0u;
      mbar_wait(&s_bar[warp][get], phase, &none);
    }
    if (lane == 0) atomicOr(&g_attn4_status, 1u);
  }

  // ---- merge the warps: O in shared memory over the rings ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      if (g == 0) {
        s_m[warp][8 * nt + 2 * t + e] = l[nt][e] == 0.f ? -INFINITY : base[nt][e];
        s_l[warp][8 * nt + 2 * t + e] = l[nt][e];
      }
    }
  if (__syncthreads_or(fail)) return;  // (the output of this launch is void; the status word says so)
  float* buf = reinterpret_cast<float*>(a4_smem);  // [warp][row][A4_OPITCH]: every record has been used
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
  const bool whole = p0 == 0 && p1 == n_item;
  const int64_t slot = ((int64_t)blockIdx.x * 2 + (p0 == 0 ? 1 : 0)) * ROWS;  // of a partial: 0 continues an item, 1 begins one
#pragma unroll
  for (int r = warp; r < ROWS; r += A4_WARPS) {  // a warp finishes a row, a lane four dims
    const int row = row0 + r;
    if (row >= n_rows) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float lt = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < A4_WARPS; ++w) {
      const float f = s_m[w][r] == -INFINITY ? 0.f : ex2f(s_m[w][r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(buf + (w * ROWS + r) * A4_OPITCH + 4 * lane);
      lt += f * s_l[w][r];
      acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
    }
    const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);  // no key: zeros; NaN stays
    if (whole) {
      const int tq = SPARSE ? tok0 : row / G, h = SPARSE ? row : row % G;
      uint2 w2;
      w2.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w2.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + ((int64_t)(q0 + tq) * p.Hq + kvh * G + h) * ATT_D + 4 * lane) = w2;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (slot + r) * ATT_D + 4 * lane) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (lane == 0) p.part_lse[slot + r] = lt > 0.f ? mx + log2f(lt) : (lt == 0.f ? -INFINITY : lt);
    }
  }
  // ---- the next item ----
  todo -= p1 - p0;
  if (todo > 0) {
    p0 = 0;
    if (++kvh == p.Hkv) {
      kvh = 0;
      ++tile;
      if (SPARSE ? tile >= si.q_len : tile * ROWS >= si.q_len * G) {
        tile = 0;
        // (pages are left, so a sequence with queries is)
        do si = seq_info(p, ++seq);
        while (si.q_len == 0 && seq + 1 < p.num_seqs);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the rings are written by copies again
    __syncthreads();
  }
  }
}

// out = sum_i w_i O_i / sum_i w_i, w_i = 2^(lse_i - max): one CTA per output row.  The weights are made once, then its warps
// take the partials in turn, eight loads in flight each: a few rows with many partials (one long sequence on one KV head) are
// a matter of latency.  The order of the sums is fixed.
// ROWS > 0: the partials of the CTAs that share the pages (attn4_kernel with tiles of ROWS rows): the first is the
// begun item of its CTA, the others continue it.  ROWS = 0: nsplit partials per row (the prefill kernel).
constexpr int MERGE_WARPS = 8;
constexpr int MERGE_MAX = 512;
template <int ROWS, bool SPARSE>
__global__ void __launch_bounds__(MERGE_WARPS * 32)
attn4_merge_kernel(const Attn4Params p) {
  __shared__ float s_w[MERGE_MAX];
  __shared__ float s_max[MERGE_WARPS], s_sum[MERGE_WARPS];
  __shared__ __align__(16) float s_o[MERGE_WARPS][ATT_D];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_enter();
  const int tok = (int)(row / p.Hq), hq = (int)(row % p.Hq);
  if (tok >= p.q_start[p.num_seqs]) return;  // a row behind the last sequence: nobody wrote its partials
  int n;             // partials
  int64_t at0, at1;  // where the first and the second of them are
  int64_t step;      // from one to the next, from the second on
  if constexpr (ROWS > 0) {
    // the row's sequence: as many end at or before it
    int seq = 0;
    for (int s = lane; s < p.num_seqs; s += 32) seq += p.q_start[s + 1] <= tok;
    seq = __reduce_add_sync(0xffffffffu, seq);
    const SeqInfo si = seq_info(p, seq);
    const int64_t before = pages_below<ROWS, SPARSE>(p, seq), T = pages_below<ROWS, SPARSE>(p, p.num_seqs);
    const int kvh = hq / p.G, off = tok - si.q0;
    const int in_seq = SPARSE ? hq % p.G : off * p.G + hq % p.G;  // row among the sequence's rows of this KV head
    const int tile = SPARSE ? off : in_seq / ROWS, r = SPARSE ? in_seq : in_seq % ROWS;
    int64_t begin = before;
    int pages = p.n_pages;
    if (SPARSE) {
      begin += ((int64_t)tile * p.Hkv + kvh) * p.n_pages;
    } else {
      for (int x = 0; x <= tile; ++x) {
        pages = max(1, item_pages(p, item_limit(si.q_len, si.q_all, si.ctx, p.G, x * ROWS, ROWS)));
        if (x < tile) begin += (int64_t)pages * p.Hkv;
      }
      begin += (int64_t)kvh * pages;
    }
    const int c0 = owner_of(begin, T, p.workers), c1 = owner_of(begin + pages - 1, T, p.workers);
    n = c1 - c0 + 1;
    if (n == 1) return;  // one CTA had it all and wrote the result
    at0 = ((int64_t)c0 * 2 + 1) * ROWS + r;
    at1 = (int64_t)(c0 + 1) * 2 * ROWS + r;
    step = 2 * ROWS;
  } else {
    n = p.nsplit;
    at0 = row * n;
    at1 = at0 + 1;
    step = 1;
  }
  auto where = [&](int i) { return i == 0 ? at0 : at1 + (i - 1) * step; };
  // NaN marks a row that saw one: it has to survive the maximum
  float lse[MERGE_MAX / (MERGE_WARPS * 32)], wm = -INFINITY;
#pragma unroll
  for (int u = 0; u < MERGE_MAX / (MERGE_WARPS * 32); ++u) {
    const int i = tid + u * MERGE_WARPS * 32;
    lse[u] = i < n ? p.part_lse[where(i)] : -INFINITY;
    wm = fmaxf(wm, lse[u] != lse[u] ? INFINITY : lse[u]);
  }
  wm = warp_max(wm);
  if (lane == 0) s_max[warp] = wm;
  __syncthreads();
  float mx = s_max[0];
#pragma unroll
  for (int w = 1; w < MERGE_WARPS; ++w) mx = fmaxf(mx, s_max[w]);
  float ws = 0.f;
#pragma unroll
  for (int u = 0; u < MERGE_MAX / (MERGE_WARPS * 32); ++u) {
    const float wt = lse[u] != lse[u] ? NAN : (lse[u] == -INFINITY ? 0.f : ex2f(lse[u] - mx));
    s_w[tid + u * MERGE_WARPS * 32] = wt;
    ws += wt;
  }
  ws = warp_sum(ws);
  if (lane == 0) s_sum[warp] = ws;
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = warp; i0 < n; i0 += 8 * MERGE_WARPS) {
    float4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * MERGE_WARPS;
      x[u] = i < n ? *reinterpret_cast<const float4*>(p.part_o + where(i) * ATT_D + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * MERGE_WARPS;
      const float w = i < n ? s_w[i] : 0.f;
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
    p.out[row * ATT_D + tid] = __float2bfloat16(total == 0.f ? 0.f : v / total);  // no key: zeros
  }
}

template <int ROWS, bool SPARSE>
static int launch_merge(const Attn4Params& p, cudaStream_t stream) {
  return (int)launch_pdl(attn4_merge_kernel<ROWS, SPARSE>, dim3((unsigned)(p.total_q * p.Hq)), dim3(MERGE_WARPS * 32), 0, stream, p);
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
  if (tiles > 65535 || p.num_seqs > 65535) return DASER_ERR_TOO_LARGE;
  const dim3 grid = p.workers ? dim3((unsigned)p.workers) : dim3(p.Hkv, p.num_seqs, (unsigned)tiles);
  const int rc = (int)launch_pdl(attn4_kernel<NT, SPARSE>, grid, dim3(A4_WARPS * 32), smem, stream, p);
  return rc || p.workers == 0 ? rc : launch_merge<8 * NT, SPARSE>(p, stream);
}

static int fill_attn4(Attn4Params& p, const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                      int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                      int num_seqs, int total_q, int max_q_len, int Hq, int parts, float softmax_scale) {
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  const int Hkv = pool->heads_per_rank;
  if (Hq <= 0 || Hq % Hkv || num_seqs < 0 || total_q < 0 || max_q_len < 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (parts < 0 || (parts > 1 && (!part_o || !part_lse))) return DASER_ERR_BAD_ARG;
  if (parts > MERGE_MAX || max_blocks > 0x7fffffff / DASER_KV4_TOKENS || total_q > 0x7fffffff / Hq) return DASER_ERR_TOO_LARGE;
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
  p.workers = 0;
  p.nsplit = 1;
  p.split_pages = 0;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.total_q = total_q;
  return 0;
}

}  // namespace daser

// Rows from which a block of queries goes to the tcgen05 kernel: half of its 128-row tile.
#define A4_TC_MIN_ROWS 64

// Causal paged attention over the 4-bit pool.
// Fewer than A4_TC_MIN_ROWS query rows per KV head (max_q_len * heads per KV head): parts is the number of CTAs that share the pages
// (0: one CTA per item, no scratch); part_o / part_lse: parts * 2 * 16 partials of 128 floats / one float.
// Else parts is the number of splits per context, of split_pages pages (parts * split_pages has to cover the longest
// context); scratch for total_q * Hq * parts partials when parts > 1.
DASER_API int daser_paged_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                                        int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                        const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq, int parts,
                                        int split_pages, float softmax_scale, cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, parts, softmax_scale))
    return e;
  const int64_t rows = (int64_t)max_q_len * p.G;
  if (rows >= A4_TC_MIN_ROWS ? parts < 1 || split_pages < 1 : parts == 1) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens) return DASER_ERR_BAD_ARG;
  if (rows >= A4_TC_MIN_ROWS) {
    p.nsplit = parts;
    p.split_pages = split_pages;
    const int rc = daser_launch_attention4_tc(p, max_q_len, stream);
    return rc || parts == 1 ? rc : launch_merge<0, false>(p, stream);
  }
  p.workers = parts;
  return rows <= 8 ? launch_attn4<1, false>(p, 1, stream) : launch_attn4<2, false>(p, (int)((rows + 15) / 16), stream);
}

// The same over the pages listed for every (query row, KV head): pages int32 [total_q][Hkv][n_pages], ascending, -1 behind the last.
// workers as parts above.
DASER_API int daser_sparse_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, const DaserKV4Pool* pool, int layer,
                                         int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                         const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq,
                                         const int32_t* pages, int n_pages, int workers, float softmax_scale, cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, workers, softmax_scale))
    return e;
  if (n_pages < 1 || workers == 1) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens || !pages) return DASER_ERR_BAD_ARG;
  p.pages = pages;
  p.n_pages = n_pages;
  p.workers = workers;
  return p.G <= 8 ? launch_attn4<1, true>(p, max_q_len, stream) : launch_attn4<2, true>(p, max_q_len, stream);
}

// Non-zero once any CTA of the 4-bit decode kernels gave up on a bounded wait (synchronises the device).
DASER_API int daser_attention4_status(uint32_t* out) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, daser::g_attn4_status, sizeof(v));
  if (out) *out = v;
  return (int)e;
}
