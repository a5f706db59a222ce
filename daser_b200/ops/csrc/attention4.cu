// Paged attention over the 4-bit pool for few query rows: decode steps, short query blocks, and decode over a list of
// selected pages.
//
//   o_r = sum_k softmax_k(scale q_r . k_k) v_k over the keys k <= pos_r (of the listed pages, in the sparse form)
//
// In the reference's serving stack this is stock vLLM's paged decode kernel over a bf16 cache.  Here a step's time is
// the 2304-byte records of the pages (0.5625 B per element against 2), as long as the dequantisation keeps up: per page 64 conversions, 64
// multiplications by scales and 16 MMAs of a warp, about 60 cycles of an SM where the memory needs 100.
//
// * A CTA (one per SM) has 16 warps that take pairs of pages in turn and fetch their own, three pairs ahead, with 16-byte asynchronous
//   copies: nine a lane and pair, no barrier in the CTA before an item is put together.  (One bulk copy a page, by each warp or by
//   a producer warp, was measured first: the copy engine of an SM took about 90 cycles for a record of 2304 bytes whoever asked, which
//   is 26 bytes a cycle, and a lane that asks waits for it: 150 us against 130 for 32 sequences of 4k - 32k tokens.)  The next
//   item's first pages are on their way while the parts of the last one are put together.
// * An item is (sequence, tile of query rows, KV head).  With many pages a fixed number of CTAs shares the pages of ALL
//   items evenly: CTA c takes [c T / W, (c + 1) T / W) of the T pages in item order, whatever the lengths are, so that
//   all finish together (splits of a fixed length left the last wave a third empty).  An item that lies in several CTAs is put
//   together by attn4_merge_kernel from their partial results.  W is the number of CTAs, or T if that is less (CTAs are planned for the
//   longest context there can be, T comes from the lengths there are): each of the W has a page then, so that
//   every CTA between the first and the last of an item leaves a part of it.
// * The cache is the A operand of mma.sync m16n8k16, the queries the B operand: S^T = K Q^T (16 tokens x 8 rows) and
//   O^T = V^T P^T (16 dims x 8 rows).  With at most 8 query heads per KV head that is half the MMAs (16 a page) of the form that puts
//   queries in the 16 rows of A.  The contraction index may be permuted as long as A and B agree, so a lane (g = lane / 4,
//   t = lane % 4) takes 16 contiguous bytes of K row g: dims [32t, 32t + 32); and of V the scale group g of tokens 2t, 2t + 1
//   (+ 8): the record stores V by groups so that these 16 bytes are contiguous too, and both reads hit all banks once.
//   P^T in the layout of B is the transpose of S^T as it comes out: one movmatrix per 8 tokens.
// * The running maximum is raised only when a page exceeds it by 2^8 (P is f16, sums are fp32): one vote a page instead of six
//   shuffles.  Scores, sums and O are fp32; K, V are exact in f16; Q and P are rounded to f16, because the MMA takes no fp32 operand that
//   keeps up with the memory: 2^-11 of their size, finer than bf16's 2^-8 (a query at least 2^-25, which is 2^-11 of its row's largest;
//   rows that f16 does not hold: plain_row).  P of the maximum is 2^7 to 2^15, so that weights have those 11
//   bits down to 2^-21 of the largest and an absolute error of at most 2^-32 of it below (with P of 1 to 2^8 a long tail 2^-20 below one
//   loud key was off by 2 %).
//
// Measured (L2 flushed in front of each call): 32 sequences of 4k - 32k tokens, 64 / 8 heads, 681 MB: 132 us, 5.2 TB/s (a copy: 6.5);
// the ALU is 56 % busy (conversions, byte selection), the tensor pipe 28 %.  4 sequences of 50k - 120k tokens on one KV head, 49 MB: 22 us +
// merge, of which 3 go by before the first page is asked for (lengths, table: dependent misses), 6 until the first pair of all
// warps is there, and 3 for putting warps and CTAs together.  One sequence of 327 keys: 6 us, latency alone.  16 lists of 128
// pages, 64 / 8 heads, 38 MB: 17 us.  More query rows take more passes over the pages, 16 rows each, with 8 warps a CTA (240 registers): 16
// sequences of 8k - 16k tokens and 64 / 8 heads, 229 MB, take 144 us for 4 new tokens each and 232 for 7, 180 TFLOP/s either
// way; 16 heads per KV head, 32 sequences of 4k - 32k tokens, 170 MB: 61 us.
// Registers bind the form for 8 rows: at 128 a thread the dense kernel spills 24 bytes, and code added to the loop over pages costs some
// 2 % whether it runs or not.
#include "attention4_params.cuh"

namespace daser {
using namespace sm100;

constexpr int A4_PAIR = 2 * DASER_KV4_RECORD;
constexpr int A4_OPITCH = 132;  // floats per row of a warp's part
// Warps and ring depth (pairs per warp) for NT column tiles: two tiles need twice the accumulators.
template <int NT> struct A4 {
  static constexpr int ROWS = 8 * NT;
  static constexpr int WARPS = NT == 1 ? 16 : 8;
  static constexpr int STAGES = NT == 1 ? 3 : 4;
  static constexpr int RING = WARPS * STAGES * A4_PAIR;
  // Where a warp leaves its part of an item: in the stage of its last pair if it fits in there.
  static constexpr int PART = ROWS * A4_OPITCH * 4;
  static constexpr bool IN_RING = PART <= A4_PAIR;
  static constexpr int SMEM = RING + (IN_RING ? 0 : WARPS * PART);
};
constexpr float A4_TOP = 7.f, A4_RAISE_AT = 15.f;  // P of a new maximum is 2^7, raised when a score would make it more than 2^15

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
// What beginning and finishing an item costs a CTA, in pages: items count that much more when the pages are shared out (about 8000
// cycles against 100 a page; 32 sequences of 4k - 32k tokens: 148 us with 1, 133 with 48, 130 with 72 to 128).
constexpr int A4_ITEM_COST = 80;
// Pages of an item of the dense form: (query rows [row0, row0 + ROWS) of a sequence of q_len new tokens and ctx keys) sees the keys
// below limit.
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
  s.q_len = s.q0 < 0 ? 0 : min(max(0, min(q1, p.total_q) - s.q0), p.max_q_len);
  s.ctx = p.ctx_lens[seq];
  return s;
}
// Pages of all items of a sequence, with what an item costs.
template <int ROWS, bool SPARSE>
__device__ __forceinline__ int64_t seq_pages(const Attn4Params& p, int seq) {
  const SeqInfo s = seq_info(p, seq);
  if (SPARSE) return (int64_t)s.q_len * p.Hkv * (p.n_pages + A4_ITEM_COST);
  int64_t n = 0;
  for (int row0 = 0; row0 < s.q_len * p.G; row0 += ROWS) n += item_pages(p, item_limit(s.q_len, s.q_all, s.ctx, p.G, row0, ROWS)) + A4_ITEM_COST;
  return n * p.Hkv;
}
__device__ __forceinline__ int64_t warp_sum_i64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The CTAs that have pages, of `workers` launched ones: no more than there are pages.
__device__ __forceinline__ int sharers(int64_t T, int workers) { return (int)min(T, (int64_t)workers); }
// The CTA that owns page x of T when W <= T share them: CTA c owns [floor(c T / W), floor((c + 1) T / W)).
__device__ __forceinline__ int owner_of(int64_t x, int64_t T, int W) { return (int)(((x + 1) * W - 1) / T); }

// The items of a CTA, one after the other; its warps walk them on their own.
template <int NT, bool SPARSE>
struct Walk {
  int seq, tile, kvh;  // the item
  int p0;              // its first page that is this CTA's
  int64_t todo;        // pages left to this CTA from there on
  SeqInfo si;
  // of the item:
  int row0, tok0, n_rows;  // rows: dense, ROWS consecutive ones (query token major, then head of the group); sparse, the heads of one token
  int first_pos, limit;    // last key the first row may see, keys the last row sees
  int n_item, p1;          // pages and the item's cost, end of this CTA's part
  int page_end;            // the same of the pages alone
  const int32_t* list;

  __device__ __forceinline__ void item(const Attn4Params& p) {
    constexpr int ROWS = A4<NT>::ROWS;
    n_rows = SPARSE ? p.G : si.q_len * p.G;
    row0 = SPARSE ? 0 : tile * ROWS;
    tok0 = SPARSE ? tile : row0 / p.G;
    first_pos = si.ctx - si.q_all + tok0;
    limit = SPARSE ? first_pos + 1 : item_limit(si.q_len, si.q_all, si.ctx, p.G, row0, ROWS);
    list = SPARSE ? p.pages + ((int64_t)(si.q0 + tok0) * p.Hkv + kvh) * p.n_pages : nullptr;
    const int real = SPARSE ? p.n_pages : item_pages(p, limit);
    n_item = real + A4_ITEM_COST;
    if (p.workers == 0) todo = n_item;
    p1 = (int)min((int64_t)n_item, p0 + todo);
    page_end = min(p1, real);
  }
  // The first item; false if there is none.  at: p0 in the order of all pages, T: pages of all items.
  __device__ __forceinline__ bool start(const Attn4Params& p, int64_t& at, int64_t& T) {
    constexpr int ROWS = A4<NT>::ROWS;
    const int lane = threadIdx.x & 31;
    p0 = 0;
    at = T = 0;
    if (p.workers == 0) {
      kvh = blockIdx.x;
      seq = blockIdx.y;
      tile = blockIdx.z;
      si = seq_info(p, seq);
      if (SPARSE ? tile >= si.q_len : tile * ROWS >= si.q_len * p.G) return false;
      item(p);
      return true;
    }
    int64_t mine = lane < p.num_seqs ? seq_pages<ROWS, SPARSE>(p, lane) : 0;  // of sequence base + lane
    T = warp_sum_i64(mine);
    for (int s = 32 + lane; s - lane < p.num_seqs; s += 32) T += warp_sum_i64(s < p.num_seqs ? seq_pages<ROWS, SPARSE>(p, s) : 0);
    const int W = sharers(T, p.workers);
    if ((int)blockIdx.x >= W) return false;
    at = (int64_t)blockIdx.x * T / W;
    todo = (int64_t)(blockIdx.x + 1) * T / W - at;
    int64_t x = at;  // relative to the sequence, the tile, the item
    for (int base = 0;; base += 32) {
      if (base > 0) mine = base + lane < p.num_seqs ? seq_pages<ROWS, SPARSE>(p, base + lane) : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t behind = __ballot_sync(0xffffffffu, upto > x);
      if (behind != 0u) {
        const int who = __ffs(behind) - 1;
        seq = base + who;
        x -= __shfl_sync(0xffffffffu, upto - mine, who);
        break;
      }
      x -= __shfl_sync(0xffffffffu, upto, 31);
    }
    si = seq_info(p, seq);
    for (tile = 0;; ++tile) {
      const int n = (SPARSE ? p.n_pages : item_pages(p, item_limit(si.q_len, si.q_all, si.ctx, p.G, tile * ROWS, ROWS))) + A4_ITEM_COST;
      if (x < (int64_t)n * p.Hkv) {
        kvh = (int)(x / n);
        p0 = (int)(x - (int64_t)kvh * n);
        break;
      }
      x -= (int64_t)n * p.Hkv;
    }
    item(p);
    return true;
  }
  __device__ __forceinline__ bool next(const Attn4Params& p) {
    todo -= p1 - p0;
    if (todo <= 0) return false;
    p0 = 0;
    if (++kvh == p.Hkv) {
      kvh = 0;
      ++tile;
      if (SPARSE ? tile >= si.q_len : tile * A4<NT>::ROWS >= si.q_len * p.G) {
        tile = 0;
        // (pages are left, so a sequence with queries is)
        do si = seq_info(p, ++seq);
        while (si.q_len == 0 && seq + 1 < p.num_seqs);
      }
    }
    item(p);
    return true;
  }
};

// ONE: the rows of an item are heads of one token and see the same keys (sparse, and dense with at most one query token per sequence).
// One query row over pages [p0, page_end) of an item in plain fp32 products: for queries that f16 does not hold (scaled and rounded to f16 the
// largest of a row is outside [2^-14, 2^15), where it would be infinite or few bits would be left).  The row is looked at when it is put
// together, so that the warps that work on its pages have nothing to do with it.  With an infinite query the sum is NaN.
// A warp; a lane has 4 dims.  One sequence of 4096 keys, 64 / 8 heads: 246 us for such queries, 13 for others.
struct PlainItem {
  const uint8_t* records;  // of the layer and KV head
  int64_t stride_block;
  const int32_t* table;
  const int32_t* list;     // sparse
  int p0, page_end, max_blocks, num_blocks;
  float scale_log2;
};
struct PlainRow {
  float4 acc;
  float m, l;
};
__device__ __noinline__ void plain_row(const PlainItem* item, uint2 w, int pos, PlainRow* out) {
  const PlainItem it = *item;
  const int lane = threadIdx.x & 31;
  const float qs[4] = {bf16_lo(w.x) * it.scale_log2, bf16_hi(w.x) * it.scale_log2, bf16_lo(w.y) * it.scale_log2, bf16_hi(w.y) * it.scale_log2};
  const float top = warp_max(fmaxf(fmaxf(fabsf(qs[0]), fabsf(qs[1])), fmaxf(fabsf(qs[2]), fabsf(qs[3]))));
  PlainRow r = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
  for (int at = it.p0; at < it.page_end; ++at) {
    const int page = it.list ? it.list[at] : at;
    if (page < 0 || page >= it.max_blocks) continue;
    const int blk = it.table[page];
    const uint8_t* rec = it.records + (int64_t)(blk < 0 ? 0 : (blk >= it.num_blocks ? it.num_blocks - 1 : blk)) * it.stride_block;
    for (int tok = 0; tok < DASER_KV4_TOKENS && page * DASER_KV4_TOKENS + tok <= pos; ++tok) {
      float k[8], v[8];
      fp4_decode8(*reinterpret_cast<const uint32_t*>(rec + kv4_code_at(0, tok, lane >> 1)), rec[kv4_scale_at(0, tok, lane >> 2)], k);
      fp4_decode8(*reinterpret_cast<const uint32_t*>(rec + kv4_code_at(1, tok, lane >> 1)), rec[kv4_scale_at(1, tok, lane >> 2)], v);
      const bool h = lane & 1;  // which half of the 8 dims
      const float s = warp_sum(qs[0] * (h ? k[4] : k[0]) + qs[1] * (h ? k[5] : k[1]) + qs[2] * (h ? k[6] : k[2]) + qs[3] * (h ? k[7] : k[3]));
      const float m = fmaxf(r.m, s), al = r.m == m ? 1.f : ex2f(r.m - m), e = top < INFINITY ? ex2f(s - m) : NAN;
      r.m = m;
      r.l = r.l * al + e;
      r.acc.x = r.acc.x * al + e * (h ? v[4] : v[0]);
      r.acc.y = r.acc.y * al + e * (h ? v[5] : v[1]);
      r.acc.z = r.acc.z * al + e * (h ? v[6] : v[2]);
      r.acc.w = r.acc.w * al + e * (h ? v[7] : v[3]);
    }
  }
  *out = r;
}

template <int NT, bool SPARSE, bool ONE>
__global__ void __launch_bounds__(A4<NT>::WARPS * 32, 1)
attn4_kernel(const Attn4Params p) {
  using C = A4<NT>;
  constexpr int ROWS = C::ROWS, WARPS = C::WARPS, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t a4_smem[];  // ring [warp][stage][2 records], parts [warp][row][A4_OPITCH]
  __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
  __shared__ int s_part[WARPS];
  __shared__ PlainItem s_item;
  __shared__ int64_t s_at, s_T;  // where this CTA is in the order of all pages, and how many there are: thread 0's, out of its registers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = p.G;
  pdl_enter();
  Walk<NT, SPARSE> it;
  {
    int64_t at, T;
    if (!it.start(p, at, T)) return;  // uniform over the CTA
    if (threadIdx.x == 0) { s_at = at; s_T = T; }
  }

  const uint8_t* ring = a4_smem + warp * STAGES * A4_PAIR;
  const uint32_t ring_u32 = smem_u32(ring);
  // Page k of this warp (k = 2 * pair + which) of an item is entry k & 31 of window k / 32, one per lane: its logical page (sparse;
  // negative: none) and its block (negative: not fetched), read a window ahead of their use.
  int log_cur, log_nxt, blk_cur, blk_nxt;  // windows of the fetches
  auto window = [&](int w, int& logical, int& block) {
    const int k = 32 * w + lane;
    const int at = it.p0 + 2 * (warp + (k >> 1) * WARPS) + (k & 1);
    logical = -1;
    block = -1;
    if (at < it.page_end) {
      logical = SPARSE ? it.list[at] : at;
      if (logical >= 0 && logical < p.max_blocks && (int64_t)logical * DASER_KV4_TOKENS < it.limit) {
        block = p.block_tables[(int64_t)it.seq * p.max_blocks + logical];
        block = block < 0 ? 0 : (block >= p.num_blocks ? p.num_blocks - 1 : block);
      } else {
        logical = -1;
      }
    }
  };
  int put = 0, get = 0;  // stages
  // Pair i (0, 1, 2, ... of the item) into the next stage: 288 pieces of 16 bytes, page 0 then page 1.  One group a call.
  auto fetch = [&](int i) {
    const int e = (2 * i) & 31;
    if (e == 0 && i > 0) {
      log_cur = log_nxt;
      blk_cur = blk_nxt;
      window((i >> 4) + 1, log_nxt, blk_nxt);
    }
    const int b0 = __shfl_sync(0xffffffffu, blk_cur, e), b1 = __shfl_sync(0xffffffffu, blk_cur, e + 1);
    const uint8_t* head = p.records + (int64_t)it.kvh * p.stride_head + lane * 16;
    const uint8_t* r0 = head + (int64_t)b0 * p.stride_block;
    const uint8_t* r1 = head + (int64_t)b1 * p.stride_block - DASER_KV4_RECORD;  // piece 144 is its first
    const uint32_t dst = ring_u32 + put * A4_PAIR + lane * 16;
    if (b0 >= 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) cp_async16(dst + u * 512, r0 + u * 512);
    }
    if (lane < 16 ? b0 >= 0 : b1 >= 0) cp_async16(dst + 4 * 512, (lane < 16 ? r0 : r1) + 4 * 512);
    if (b1 >= 0) {
#pragma unroll
      for (int u = 5; u < 9; ++u) cp_async16(dst + u * 512, r1 + u * 512);
    }
    cp_async_commit();
    put = put == STAGES - 1 ? 0 : put + 1;
  };
  auto first_windows = [&] {
    window(0, log_cur, blk_cur);
    window(1, log_nxt, blk_nxt);
  };
  uint4 qr[NT][4];  // the rows of the queries that this lane holds, as they are
  auto load_q = [&] {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = it.row0 + 8 * nt + g;
      const int tq = SPARSE ? it.tok0 : r / G, h = SPARSE ? r : r % G;
      const __nv_bfloat16* qp = p.q + ((int64_t)(it.si.q0 + tq) * p.Hq + it.kvh * G + h) * ATT_D + 32 * t;
#pragma unroll
      for (int i = 0; i < 4; ++i) qr[nt][i] = r < it.n_rows ? *reinterpret_cast<const uint4*>(qp + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  first_windows();
#pragma unroll
  for (int i = 0; i < STAGES; ++i) fetch(i);  // (a pair that is not there is an empty group)
  load_q();
  bool parts_read = true;  // false: the parts of the last item are still being read

  bool more;
  do {
  const int row0 = it.row0, tok0 = it.tok0, n_rows = it.n_rows, first_pos = it.first_pos, kvh = it.kvh, q0 = it.si.q0;
  const int limit = ONE ? first_pos + 1 : it.limit;
  int use_cur = log_cur, use_nxt = log_nxt;  // windows of the uses, which run behind those of the fetches
  // ---- queries: B fragments, scaled, f16.  Column g of n-tile nt is row row0 + 8 nt + g ----
  uint32_t qf[NT][16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t ww[4] = {qr[nt][i].x, qr[nt][i].y, qr[nt][i].z, qr[nt][i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[nt][4 * i + e] = pack_half2(bf16_lo(ww[e]) * p.scale_log2, bf16_hi(ww[e]) * p.scale_log2);
    }
  // last visible key of this lane's columns 2t, 2t + 1 of every n-tile
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[nt][e] = ONE ? first_pos : first_pos + (row0 + 8 * nt + 2 * t + e) / G - tok0;

  // base: what the exponents are relative to: 7 less than the running maximum, which may be up to 8 behind; 0 until the row has seen a key
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

  int part = -1;  // where this warp's part goes; none without a page
  int used = 0;
  for (int page = it.p0 + 2 * warp; page < it.page_end; page += 2 * WARPS, ++used) {
    if (parts_read) cp_async_wait<STAGES - 1>();
    else cp_async_wait<STAGES - 2>();  // one group fewer is out
    __syncwarp();
    const uint8_t* st[2] = {ring + get * A4_PAIR, ring + get * A4_PAIR + DASER_KV4_RECORD};
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
      key0[0] = page;
      key0[1] = page + 1 < it.page_end ? page + 1 : -1;
    }
    // a page that is not there lies beyond every limit: its scores become -inf, its scales 0
    key0[0] = key0[0] < 0 ? 1 << 29 : key0[0] * DASER_KV4_TOKENS;
    key0[1] = key0[1] < 0 ? 1 << 29 : key0[1] * DASER_KV4_TOKENS;
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
      if (!ONE && limit - 1 > first_pos) {
        // A key that only the later rows see must not reach the others as 0 * NaN: a group of its value that is not finite leaves the
        // product (its scale becomes 0), and NaN goes into the rows that see it.
        int bad = 1 << 30;  // the first such key of group g
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = i >> 2, tok = 2 * t + (i & 1) + 4 * (i & 2);
          uint8_t* const at = const_cast<uint8_t*>(st[x]) + kv4_scale_at(1, tok, g);
          if (key0[x] + tok < limit && *at >= 0xf8u) {
            *at = 0;
            bad = min(bad, key0[x] + tok);
          }
        }
        if (__any_sync(0xffffffffu, bad < 1 << 30)) {
          bad = min(bad, __shfl_xor_sync(0xffffffffu, bad, 1));
          bad = min(bad, __shfl_xor_sync(0xffffffffu, bad, 2));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (bad <= pos[nt][e]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[nt][j][e] = o[nt][j][2 + e] = NAN;
              }
        }
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
          // relative to the old base: to 7 below the first maximum wherever that lies, then upwards only
          const float up = mx == -INFINITY ? 0.f : fmaxf(mx - A4_TOP, seen[nt][e] ? 0.f : -INFINITY);
          seen[nt][e] |= mx > -INFINITY;
          none |= !seen[nt][e];
          const float al = ex2f(fminf(-up, 0.f));  // (a row's first maximum may lie far below 0: there is nothing to scale yet)
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
    __syncwarp();  // every lane is done with this stage
    part = C::IN_RING ? (warp * STAGES + get) * A4_PAIR : C::RING + warp * C::PART;
    get = get == STAGES - 1 ? 0 : get + 1;
    if (!parts_read) {
      __syncthreads();  // the stage that held this warp's part, and what was said about it, are free
      parts_read = true;
      fetch(STAGES - 1);
    }
    if (page + 2 * WARPS < it.page_end) fetch(used + STAGES);
  }
  if (!parts_read) {
    __syncthreads();
    parts_read = true;
    fetch(STAGES - 1);
  }

  // ---- put the warps' parts together ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
      l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
      const int r = 8 * nt + 2 * t + e;
      if (g == 0) {
        s_m[warp][r] = l[nt][e] == 0.f ? -INFINITY : base[nt][e];
        s_l[warp][r] = l[nt][e];
      }
      float* dst = reinterpret_cast<float*>(a4_smem + max(part, 0)) + r * A4_OPITCH + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        if (part >= 0) *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(o[nt][j][e], o[nt][j][2 + e], o[nt][j + 1][e], o[nt][j + 1][2 + e]);
    }
  if (lane == 0) s_part[warp] = part;
  if (threadIdx.x == 32)
    s_item = {p.records + (int64_t)kvh * p.stride_head, p.stride_block, p.block_tables + (int64_t)it.seq * p.max_blocks, it.list, it.p0, it.page_end,
              p.max_blocks, p.num_blocks, p.scale_log2};
  const bool begins = it.p0 == 0, whole = begins && it.p1 == it.n_item;
  const int64_t slot = ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * ROWS;  // of a partial: 0 continues an item, 1 begins one
  if (p.workers && threadIdx.x == 0) {
    if (begins) {
      // who has the rest of the item: the owner of its last page is the last
      const int64_t id = SPARSE ? (int64_t)(q0 + tok0) * p.Hkv + kvh : ((int64_t)it.seq * p.tiles + it.tile) * p.Hkv + kvh;
      const int n = whole ? 1 : owner_of(s_at + it.n_item - 1, s_T, sharers(s_T, p.workers)) - (int)blockIdx.x + 1;
      p.shared[id] = make_int2((int)blockIdx.x, n);
    }
    s_at += it.p1 - it.p0;
  }
  // ---- the next item: its first pages, but for the stage that holds this warp's part ----
  cp_async_wait<0>();  // (groups that were empty)
  more = it.next(p);
  put = get;
  if (more) {
    first_windows();
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  }
  __syncthreads();
#pragma unroll
  for (int r = warp; r < ROWS; r += WARPS) {  // a warp finishes a row, a lane four dims
    const int row = row0 + r;
    if (row >= n_rows) break;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, s_m[w][r]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float lt = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      // a warp that saw no key: its part may not even be there.  No branch, so that the loads of all warps' parts go out together.
      const bool there = s_m[w][r] != -INFINITY;
      const float f = there ? ex2f(s_m[w][r] - ref) : 0.f;
      const float4 v = *reinterpret_cast<const float4*>(a4_smem + max(s_part[w], 0) + (r * A4_OPITCH + 4 * lane) * 4);
      lt += f * s_l[w][r];
      acc.x += there ? f * v.x : 0.f; acc.y += there ? f * v.y : 0.f; acc.z += there ? f * v.z : 0.f; acc.w += there ? f * v.w : 0.f;
    }
    const int tq = SPARSE ? tok0 : row / G, h = SPARSE ? row : row % G;
    const int64_t at = ((int64_t)(q0 + tq) * p.Hq + kvh * G + h) * ATT_D;  // in q and out
    const uint2 qw = *reinterpret_cast<const uint2*>(p.q + at + 4 * lane);
    if (odd_row(__reduce_max_sync(0xffffffffu, top_half(top_bf16(0u, make_uint4(qw.x, qw.y, 0u, 0u)))), p.q_lo, p.q_hi)) {
      PlainRow pr;
      plain_row(&s_item, qw, first_pos + tq - tok0, &pr);
      acc = pr.acc;
      mx = pr.m;
      lt = pr.l;
    }
    const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);  // no key: zeros; NaN stays
    if (whole) {
      uint2 w2;
      w2.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w2.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + at + 4 * lane) = w2;
    } else {
      *reinterpret_cast<float4*>(p.part_o + (slot + r) * ATT_D + 4 * lane) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (lane == 0) p.part_lse[slot + r] = lt > 0.f ? mx + log2f(lt) : (lt == 0.f ? -INFINITY : lt);
    }
  }
  if (more) load_q();
  parts_read = false;  // warps that finish no row go on with the next item
  } while (more);
}

// out = sum_i w_i O_i / sum_i w_i, w_i = 2^(lse_i - max): one CTA per output row.  The weights are made once, then its warps
// take the partials in turn, eight loads in flight each: a few rows with many partials (one long sequence on one KV head) are
// a matter of latency.  The order of the sums is fixed.
// The partials of the CTAs that share the pages (attn4_kernel with tiles of ROWS rows): the first is the begun item of its CTA, the
// others continue it; grid (KV head, sequence, row) or (KV head, query row, head).
constexpr int MERGE_WARPS = 4;
constexpr int MERGE_MAX = 256;
template <int ROWS, bool SPARSE>
__global__ void __launch_bounds__(MERGE_WARPS * 32)
attn4_merge_kernel(const Attn4Params p) {
  __shared__ float s_w[MERGE_MAX];
  __shared__ float s_max[MERGE_WARPS], s_sum[MERGE_WARPS];
  __shared__ __align__(16) float s_o[MERGE_WARPS][ATT_D];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_enter();
  int n;             // partials
  int64_t at0, at1;  // where the first and the second of them are
  int64_t step;      // from one to the next, from the second on
  int64_t row;       // of the output
  const int kvh = blockIdx.x;
  int r;
  int64_t id;
  if (SPARSE) {
    const int tok = blockIdx.y;
    r = blockIdx.z;
    // a row that no CTA worked on has no entry in `shared`: in front of, between or behind the sequences, beyond max_q_len
    bool found = false;
    for (int base = 0; base < p.num_seqs && !found; base += 32) {
      const int seq = base + lane;
      bool mine = false;
      if (seq < p.num_seqs) {
        const int q0 = p.q_start[seq], q1 = p.q_start[seq + 1];
        mine = q0 >= 0 && tok >= q0 && tok < q1 && tok - q0 < p.max_q_len;
      }
      found = __any_sync(0xffffffffu, mine);
    }
    if (!found) return;  // (every warp of the CTA alike)
    id = (int64_t)tok * p.Hkv + kvh;
    row = (int64_t)tok * p.Hq + kvh * p.G + r;
  } else {
    const int seq = blockIdx.y, in_seq = blockIdx.z;
    const int q0 = p.q_start[seq], q1 = min(p.q_start[seq + 1], p.total_q);
    const int tok = in_seq / p.G;
    if (q0 < 0 || q0 + tok >= q1) return;
    r = in_seq % ROWS;
    id = ((int64_t)seq * p.tiles + in_seq / ROWS) * p.Hkv + kvh;
    row = (int64_t)(q0 + tok) * p.Hq + kvh * p.G + in_seq % p.G;
  }
  const int2 s = p.shared[id];
  n = s.y;
  // 1: one CTA had it all and wrote the result.  (The rest: a row that no sequence has, in a list that is not one of prefix sums.)
  if (n < 2 || s.x < 0 || n > p.workers - s.x) return;
  at0 = ((int64_t)s.x * 2 + 1) * ROWS + r;
  at1 = (int64_t)(s.x + 1) * 2 * ROWS + r;
  step = 2 * ROWS;
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
  float total = 0.f, v = 0.f;
#pragma unroll
  for (int w = 0; w < MERGE_WARPS; ++w) {
    total += s_sum[w];
    v += s_o[w][tid];
  }
  p.out[row * ATT_D + tid] = __float2bfloat16(total == 0.f ? 0.f : v / total);  // no key: zeros
}

// The same for nsplit partials per row, one behind the other (the prefill kernel's): many rows with few partials, a warp per row.
__global__ void __launch_bounds__(MERGE_WARPS * 32)
attn4_merge_rows_kernel(const Attn4Params p) {
  const int lane = threadIdx.x & 31;
  pdl_enter();
  const int q0 = p.q_start[blockIdx.y], q_len = min(min(p.q_start[blockIdx.y + 1], p.total_q) - q0, p.max_q_len);
  const int64_t in_seq = (int64_t)blockIdx.x * MERGE_WARPS + (threadIdx.x >> 5), row = (int64_t)q0 * p.Hq + in_seq;
  if (q0 < 0 || q_len <= 0 || in_seq >= (int64_t)q_len * p.Hq) return;  // a row of no sequence: nobody wrote its partials
  const int n = p.nsplit;
  const float* lse = p.part_lse + row * n;
  const float* part = p.part_o + row * n * ATT_D + 4 * lane;
  float wm = -INFINITY;
  for (int i = lane; i < n; i += 32) wm = fmaxf(wm, lse[i] != lse[i] ? INFINITY : lse[i]);  // a NaN has to survive the maximum
  const float mx = warp_max(wm);
  float total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float mine = i0 + lane < n ? lse[i0 + lane] : -INFINITY;
    const float wt = mine != mine ? NAN : (mine == -INFINITY ? 0.f : ex2f(mine - mx));
    total += wt;
    for (int i = 0; i < 32 && i0 + i < n; i += 8) {
      float4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        x[u] = i0 + i + u < n ? *reinterpret_cast<const float4*>(part + (int64_t)(i0 + i + u) * ATT_D) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __shfl_sync(0xffffffffu, wt, i + u);  // (0 behind the last)
        acc.x += w * x[u].x; acc.y += w * x[u].y; acc.z += w * x[u].z; acc.w += w * x[u].w;
      }
    }
  }
  total = warp_sum(total);
  auto div = [&](float v) { return total == 0.f ? 0.f : v / total; };  // no key: zeros
  uint2 w2;
  w2.x = pack_bf16x2(div(acc.x), div(acc.y));
  w2.y = pack_bf16x2(div(acc.z), div(acc.w));
  *reinterpret_cast<uint2*>(p.out + row * ATT_D + 4 * lane) = w2;
}

template <int ROWS, bool SPARSE>
static int launch_merge(const Attn4Params& p, int max_q_len, cudaStream_t stream) {
  const dim3 grid = SPARSE ? dim3((unsigned)p.Hkv, (unsigned)p.total_q, (unsigned)p.G)
                           : dim3((unsigned)p.Hkv, (unsigned)p.num_seqs, (unsigned)(max_q_len * p.G));
  return (int)launch_pdl(attn4_merge_kernel<ROWS, SPARSE>, grid, dim3(MERGE_WARPS * 32), 0, stream, p);
}

template <int NT, bool SPARSE, bool ONE>
static int launch_attn4(Attn4Params& p, int max_q_len, cudaStream_t stream) {
  using C = A4<NT>;
  static bool configured[DASER_MAX_DEVICES] = {false};  // per device: the attribute is the device's
  constexpr int smem = C::SMEM;
  if (daser_first_use_on_device(configured)) {
    cudaError_t e = cudaFuncSetAttribute(attn4_kernel<NT, SPARSE, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    daser_used_on_device(configured);
  }
  p.max_q_len = max_q_len;
  p.tiles = SPARSE ? max_q_len : (max_q_len * p.G + C::ROWS - 1) / C::ROWS;
  if (p.tiles > 65535 || p.num_seqs > 65535 || (SPARSE && p.total_q > 65535)) return DASER_ERR_TOO_LARGE;
  const dim3 grid = p.workers ? dim3((unsigned)p.workers) : dim3((unsigned)p.Hkv, (unsigned)p.num_seqs, (unsigned)p.tiles);
  const int rc = (int)launch_pdl(attn4_kernel<NT, SPARSE, ONE>, grid, dim3(C::WARPS * 32), smem, stream, p);
  return rc || p.workers == 0 ? rc : launch_merge<C::ROWS, SPARSE>(p, max_q_len, stream);
}

static int fill_attn4(Attn4Params& p, const void* q, void* out, float* part_o, float* part_lse, void* shared, const DaserKV4Pool* pool, int layer,
                      int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                      int num_seqs, int total_q, int max_q_len, int Hq, int parts, float softmax_scale) {
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  const int Hkv = pool->heads_per_rank;
  if (Hq <= 0 || Hq % Hkv || num_seqs < 0 || total_q < 0 || max_q_len < 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (parts < 0 || (parts > 1 && (!part_o || !part_lse))) return DASER_ERR_BAD_ARG;
  if (parts > MERGE_MAX || max_blocks > (1 << 29) / DASER_KV4_TOKENS || total_q > 0x7fffffff / Hq) return DASER_ERR_TOO_LARGE;
  if (Hq / Hkv > 16) return DASER_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)part_o) % 16) return DASER_ERR_UNSUPPORTED;
  p.q = (const __nv_bfloat16*)q;
  p.out = (__nv_bfloat16*)out;
  p.part_o = part_o;
  p.part_lse = part_lse;
  p.shared = (int2*)shared;
  p.tiles = 0;
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
  // with the scale's exponent e, |q| in [2^(-14 - e), 2^(14 - e)) keeps |q scale| in [2^-14, 2^15)
  int e = 0;
  if (p.scale_log2 != 0.f && isfinite(p.scale_log2)) frexpf(p.scale_log2, &e), --e;
  const int lo = 127 - 14 - e, hi = 127 + 14 - e;
  p.q_lo = (uint32_t)(lo < 0 ? 0 : lo > 255 ? 255 : lo) << 7;
  p.q_hi = (uint32_t)(hi < 0 ? 0 : hi > 255 ? 255 : hi) << 7;
  p.total_q = total_q;
  return 0;
}

}  // namespace daser

// Rows from which a block of queries goes to the tcgen05 kernel: half of its 128-row tile.
#define A4_TC_MIN_ROWS 64

// Causal paged attention over the 4-bit pool.
// Fewer than A4_TC_MIN_ROWS query rows per KV head (max_q_len * heads per KV head): parts is the number of CTAs that share the pages
// (0: one CTA per item, no scratch); part_o / part_lse: parts * 2 * 16 partials of 128 floats / one float; shared: two
// ints per (sequence, tile of 8 rows, KV head), sparse per (query row, KV head).
// Else parts is the number of splits per context, of split_pages pages (parts * split_pages has to cover the longest
// context); scratch for total_q * Hq * parts partials when parts > 1.
DASER_API int daser_paged_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, void* shared, const DaserKV4Pool* pool, int layer,
                                        int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                        const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq, int parts,
                                        int split_pages, float softmax_scale, cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, shared, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, parts, softmax_scale))
    return e;
  const int64_t rows = (int64_t)max_q_len * p.G;
  if (rows >= A4_TC_MIN_ROWS ? parts < 1 || split_pages < 1 : parts == 1) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens) return DASER_ERR_BAD_ARG;
  if (rows >= A4_TC_MIN_ROWS) {
    p.nsplit = parts;
    p.max_q_len = max_q_len;
    p.split_pages = split_pages;
    const int rc = daser_launch_attention4_tc(p, max_q_len, stream);
    if (rc || parts == 1) return rc;
    const int64_t ctas = ((int64_t)max_q_len * Hq + MERGE_WARPS - 1) / MERGE_WARPS;  // (max_q_len: bounded by the launch in front)
    return (int)launch_pdl(attn4_merge_rows_kernel, dim3((unsigned)ctas, (unsigned)num_seqs), dim3(MERGE_WARPS * 32), 0, stream, p);
  }
  p.workers = parts;
  if (parts && !shared) return DASER_ERR_BAD_ARG;
  // a single token's rows need no look at values that some of them do not see: 146 us against 150 for 32 sequences of 4k - 32k tokens
  if (max_q_len == 1) return rows <= 8 ? launch_attn4<1, false, true>(p, max_q_len, stream) : launch_attn4<2, false, true>(p, max_q_len, stream);
  return rows <= 8 ? launch_attn4<1, false, false>(p, max_q_len, stream) : launch_attn4<2, false, false>(p, max_q_len, stream);
}

// The same over the pages listed for every (query row, KV head): pages int32 [total_q][Hkv][n_pages], ascending, -1 behind the last.
// workers as parts above.
DASER_API int daser_sparse_attention_kv4(const void* q, void* out, float* part_o, float* part_lse, void* shared, const DaserKV4Pool* pool, int layer,
                                         int rank, const int32_t* block_tables, int max_blocks, const int32_t* q_start,
                                         const int32_t* ctx_lens, int num_seqs, int total_q, int max_q_len, int Hq,
                                         const int32_t* pages, int n_pages, int workers, float softmax_scale, cudaStream_t stream) {
  using namespace daser;
  Attn4Params p;
  if (int e = fill_attn4(p, q, out, part_o, part_lse, shared, pool, layer, rank, block_tables, max_blocks, q_start, ctx_lens, num_seqs, total_q,
                         max_q_len, Hq, workers, softmax_scale))
    return e;
  if (n_pages < 1 || workers == 1) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !out || !block_tables || !q_start || !ctx_lens || !pages) return DASER_ERR_BAD_ARG;
  p.pages = pages;
  p.n_pages = n_pages;
  p.workers = workers;
  if (workers && !shared) return DASER_ERR_BAD_ARG;
  return p.G <= 8 ? launch_attn4<1, true, true>(p, max_q_len, stream) : launch_attn4<2, true, true>(p, max_q_len, stream);
}
