// Chunked-prefill attention over the 4-bit pool on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// One CTA per SM works on two tiles of 128 query rows (128 / G query tokens x the G heads of one KV head, each) against tiles of 64 keys, so
// that a tile of keys is dequantised once for 256 rows and one row tile's softmax runs under the other's MMAs.  14 warps:
//   * 0-3, 4-7   softmax of row tile 0, 1: a thread owns a row of S (tcgen05.ld 32x32b), takes it into registers and frees it at once,
//                so that the next S is under way while P = 2^(S - m) is made: f16, back into TMEM, as the MMA operand.  m is 7 less than
//                the running maximum and raised only when a tile exceeds that by 2^8, and only then is O rescaled (tcgen05.ld / st);
//   * 8-11       dequantise: K as [key][dim], V transposed to [dim][key], f16 (exact), in the 128-byte-swizzled K-major layout of the
//                MMA descriptors, two buffers each.  V's codes of two neighbouring tokens are interleaved nibble by nibble, so that
//                one conversion yields the two neighbours of a V^T row.  A row of ones in V^T sums the rows of the P that was multiplied;
//   * 12         issues the MMAs, S0(i), O0 += P0(i-1) V(i-1), S1(i), O1 += P1(i-1) V(i-1): M 128, N 64, K 128 and M 128, N 144, K 64;
//   * 13         fetches: a tile is four bulk copies of 2304 bytes, three tiles ahead.
// Measured: 2048 tokens over 8192 keys, 32 / 8 heads, 241 GFLOP: 283 us, 850 TFLOP/s.  256 CTAs on 148 SMs are 1.73 waves: of the
// cycles that an SM is at work the tensor pipe is active in 46 %, the ALU in 39 and the exponential's unit in 43.  What binds is shared
// memory: a tile moves 174 KB (Q and K into the scores 96, V^T 37, dequantised tiles 32, records 9), 1360 cycles at 128 bytes, of the
// some 2000 that it takes; the warp that issues the MMAs waits for operands in a quarter of them only.  (Exponents before the wait
// for the last P V were 3 % slower, their maximum in packed f16 6 %.)  64 tokens over 3328 keys, 64 / 8 heads (9 splits of 6 tiles): 25 us with
// the merge, half of it before the first MMA and behind the last.
// Rounded to f16: Q and P, 2^-11 of their size, P below 2^-21 of a row's maximum to 2^-32 of that.  Exponents are fp32: an f16 exponential
// of rounded exponents was 1.4 % faster, but off by up to 2^-8 where the maximum lags, and P of 1 to 2^8 lost what
// lies 2^-20 below the maximum, 2 % of a long flat tail.  Rows whose queries f16 does not hold have a scale of their own (row_scale).
// Every mbarrier wait is bounded; on expiry the CTA records it in a status word, frees its TMEM and returns.
#include "attention4_params.cuh"

namespace daser {
using namespace sm100;

constexpr int T4_NK = 64;                               // keys per tile
constexpr int T4_PAGES = T4_NK / DASER_KV4_TOKENS;
constexpr int T4_PITCH = DASER_KV4_RECORD + 16;         // of a page in shared memory: pages start on other banks
constexpr int T4_RAW = T4_PAGES * T4_PITCH;
constexpr int T4_STAGES = 3;
constexpr int T4_Q_BYTES = 128 * ATT_D * 2;             // of a row tile: two sub-tiles [128 rows][64 dims]
constexpr int T4_K_BYTES = T4_NK * ATT_D * 2;           // two sub-tiles [64 keys][64 dims]
constexpr int T4_ON = ATT_D + 16;                       // output columns: 128 dims, the row sum, 15 unused
constexpr int T4_VT_BYTES = T4_ON * 128;
constexpr int T4_THREADS = 14 * 32;
constexpr int T4_SMEM = 1024 + 2 * T4_Q_BYTES + 2 * T4_K_BYTES + 2 * T4_VT_BYTES + T4_STAGES * T4_RAW;
constexpr uint32_t T4_TMEM_COLS = 512;
// Of row tile t: S in columns [64 t, + 64), O in [128 + 192 t, + 144), P (two f16 a column) in [288 + 192 t, + 32).
__device__ __forceinline__ uint32_t t4_s_col(int t) { return 64u * t; }
__device__ __forceinline__ uint32_t t4_o_col(int t) { return 128u + 192u * t; }
__device__ __forceinline__ uint32_t t4_p_col(int t) { return 288u + 192u * t; }
constexpr float T4_TOP = 7.f, T4_RAISE_AT = 15.f;  // P of a new maximum is 2^7, raised when a score would make it more than 2^15

__device__ uint32_t g_attn4_tc_status = 0;  // bit 0: a bounded wait ran out

__device__ __forceinline__ void t4_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void t4_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {  // 32 lanes x 16 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void t4_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void t4_tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]^T, f16.
__device__ __forceinline__ void t4_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void t4_tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void t4_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The whole warp waits; one answer for all lanes, so that they leave a loop together.
__device__ __forceinline__ bool t4_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

struct T4Bars {
  uint64_t raw_full[T4_STAGES], raw_free[T4_STAGES];
  uint64_t k_ready[2], k_free[2], v_ready[2], v_free[2];  // by buffer
  uint64_t s_ready[2], s_free[2], p_ready[2], o_done[2];  // by row tile
  uint64_t q_ready, drain;
  uint32_t tmem, abort;
  int bad_v[8];  // of every group of 16 dims: the first key whose value is not finite and that some row of the CTA does not see
};

// A key that only the later rows of a CTA see must not reach the others as 0 * NaN: a group of its value that is not finite leaves the product
// (its scale becomes 0), and the rows that see it get their NaN when they are written.  Called where the causal edge runs through
// a tile; a warp looks at the two groups of which it makes V^T.  (In line it cost every tile: 292 us against 291, 25.3 against 24.9.)
__device__ __noinline__ void t4_leave_out_bad_values(uint8_t* raw, int* bad_v, int key0, int key_end) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int rep = 0; rep < 4; ++rep) {
    const int kt = lane + 32 * (rep & 1), g = 2 * (warp - 8) + (rep >> 1);
    uint8_t* const at = raw + (kt >> 4) * T4_PITCH + kv4_scale_at(1, kt & 15, g);
    if (key0 + kt < key_end && *at >= 0xf8u) {
      *at = 0;
      atomicMin(bad_v + g, key0 + kt);
    }
  }
  __syncwarp();
}

// The scale of a query row (null: none).
__device__ __noinline__ RowScale t4_row_scale(const __nv_bfloat16* q, float scale_log2, uint32_t q_lo, uint32_t q_hi) {
  uint32_t top = 0u;
  if (q != nullptr)
    for (int i = 0; i < ATT_D / 8; ++i) top = top_bf16(top, *reinterpret_cast<const uint4*>(q + 8 * i));
  return row_scale(top_half(top), scale_log2, q_lo, q_hi);
}

__global__ void __launch_bounds__(T4_THREADS, 1)
attn4_tc_kernel(const Attn4Params p, int groups) {
  extern __shared__ uint8_t t4_smem_raw[];
  __shared__ T4Bars bars;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(t4_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;
  uint8_t* k_s = q_s + 2 * T4_Q_BYTES;
  uint8_t* vt_s = k_s + 2 * T4_K_BYTES;
  uint8_t* raw_s = vt_s + 2 * T4_VT_BYTES;
  volatile uint32_t* abort_flag = &bars.abort;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x, seq = blockIdx.y;
  const int grp = groups - 1 - (int)(blockIdx.z / p.nsplit), sp = blockIdx.z % p.nsplit;  // the longest first
  pdl_wait();  // launched ahead of its predecessor's end: nothing is read before this returns
  const int q0 = p.q_start[seq];
  const int q_all = p.q_start[seq + 1] - q0;
  const int q_len = min(min(p.q_start[seq + 1], p.total_q) - q0, p.max_q_len);
  const int G = p.G;
  const int toks = 128 / G;  // of a row tile
  const int tok0 = grp * 2 * toks;
  if (q0 < 0 || tok0 >= q_len) return;  // uniform over the CTA
  const int tiles = tok0 + toks < q_len ? 2 : 1;  // live row tiles
  const int last_tok = min(tok0 + tiles * toks, q_len) - 1;
  const int limit = p.ctx_lens[seq] - q_all + last_tok + 1;  // keys visible to the last row
  const int n_all = limit > 0 ? (min(limit, p.max_blocks * DASER_KV4_TOKENS) + DASER_KV4_TOKENS - 1) / DASER_KV4_TOKENS : 0;
  const int page_begin = sp * p.split_pages;
  const int page_end = min(page_begin + p.split_pages, n_all);
  const int n_tiles = page_begin < page_end ? (page_end - page_begin + T4_PAGES - 1) / T4_PAGES : 0;
  const int key_end = min(page_end * DASER_KV4_TOKENS, limit);
  const int seen_by_all = p.ctx_lens[seq] - q_all + tok0;  // the last key that the CTA's first row sees

  // softmax threads: this thread's row
  const int tile = warp >> 2, rt = tid & 127;
  const int tq = tok0 + tile * toks + rt / G, hq = kvh * G + rt % G;
  const bool valid = tile < tiles && rt < toks * G && tq < q_len;
  const int pos = p.ctx_lens[seq] - q_all + tq;  // last key this row may see
  const int64_t row = (int64_t)(q0 + tq) * p.Hq + hq;

  if (n_tiles == 0) {  // no keys in this split: an empty partial
    if (valid) {
      if (p.nsplit == 1) {
        __nv_bfloat16* dst = p.out + row * ATT_D;
#pragma unroll
        for (int ck = 0; ck < 16; ++ck) *reinterpret_cast<uint4*>(dst + 8 * ck) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        float* dst = p.part_o + (row * p.nsplit + sp) * ATT_D;
#pragma unroll
        for (int ck = 0; ck < 32; ++ck) *reinterpret_cast<float4*>(dst + 4 * ck) = make_float4(0.f, 0.f, 0.f, 0.f);
        p.part_lse[row * p.nsplit + sp] = -INFINITY;
      }
    }
    return;
  }

  // Q: half a warp reads a row of 256 bytes, two rows an instruction (a row per thread took 8000 cycles, tags bound).  The loads are out
  // before the barriers are set up, and so are those of the first block ids.
  uint4 qw[16];
  if (tile < tiles) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int src = 2 * i + (lane >> 4);
      const int64_t r = __shfl_sync(0xffffffffu, row, src);
      const bool live = __shfl_sync(0xffffffffu, (int)valid, src) != 0;
      qw[i] = live ? *reinterpret_cast<const uint4*>(p.q + r * ATT_D + (lane & 15) * 8) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks;
  int blk[T4_PAGES];
  auto ids = [&](int ti) {  // a tile ahead of the copies that need them
#pragma unroll
    for (int pg = 0; pg < T4_PAGES; ++pg) blk[pg] = __ldg(table + min(page_begin + ti * T4_PAGES + pg, p.max_blocks - 1));
  };
  if (warp == 13) ids(0);

  const uint32_t q_u32 = smem_u32(q_s), k_u32 = smem_u32(k_s), vt_u32 = smem_u32(vt_s), raw_u32 = smem_u32(raw_s);
  if (tid == 0) {
#pragma unroll
    for (int s = 0; s < T4_STAGES; ++s) {
      mbar_init(&bars.raw_full[s], 1);
      mbar_init(&bars.raw_free[s], 4);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars.k_ready[b], 4);
      mbar_init(&bars.k_free[b], 1);
      mbar_init(&bars.v_ready[b], 4);
      mbar_init(&bars.v_free[b], 1);
      mbar_init(&bars.s_ready[b], 1);
      mbar_init(&bars.s_free[b], 4);
      mbar_init(&bars.p_ready[b], 4);
      mbar_init(&bars.o_done[b], 1);
    }
    mbar_init(&bars.q_ready, 4 * tiles);
    mbar_init(&bars.drain, 1);
    bars.abort = 0u;
    mbar_init_fence();
  }
  if (warp == 11 && lane < 8) bars.bad_v[lane] = 0x7fffffff;
  if (warp == 12) {
    tmem_alloc(&bars.tmem, T4_TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();  // barriers initialised, TMEM address published
  tc_fence_after();
  pdl_launch_dependents();  // only now: this CTA holds its tensor memory, a successor cannot take it
  const uint32_t tmem = bars.tmem;
  bool ok = true;

  if (warp < 8) {
    // ======== softmax ========
    if (tile < tiles) {
      const uint32_t tmem_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t4_s_col(tile);
      const uint32_t tmem_o = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t4_o_col(tile);
      const uint32_t tmem_p = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t4_p_col(tile);
      uint8_t* my_q = q_s + tile * T4_Q_BYTES;
      // Q -> f16, times scale * log2(e), into the swizzled A tile.  Rows with a scale of their own (row_scale) are looked for by 8 dims: if all
      // of the warp's are in the range, or zero, so are the rows.
      RowScale rs = {p.scale_log2, 1.f};
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) odd |= odd_row(top_half(top_bf16(0u, qw[i])), p.q_lo, p.q_hi);
      odd = __any_sync(0xffffffffu, odd);
      if (odd) rs = t4_row_scale(valid ? p.q + row * ATT_D : nullptr, p.scale_log2, p.q_lo, p.q_hi);
      const bool plain = valid && rs.factor == 1.f;  // keys in front of the causal edge count as they are
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = (warp & 3) * 32 + 2 * i + (lane >> 4), ck = lane & 15;
        const uint4 w = qw[i];
        const float sc = odd ? __shfl_sync(0xffffffffu, rs.scale, 2 * i + (lane >> 4)) : p.scale_log2;
        auto two = [&](uint32_t x) { return pack_half2(bf16_lo(x) * sc, bf16_hi(x) * sc); };
        const uint4 h = make_uint4(two(w.x), two(w.y), two(w.z), two(w.w));
        *reinterpret_cast<uint4*>(my_q + (ck >> 3) * 16384 + r * 128 + (((ck & 7) ^ (r & 7)) << 4)) = h;
      }
      t4_fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.q_ready);

      float m = -INFINITY;  // what the accumulated P are relative to
      for (int ti = 0; ti < n_tiles; ++ti) {
        const int key0 = (page_begin + ti * T4_PAGES) * DASER_KV4_TOKENS;
        if (!(ok = t4_wait(&bars.s_ready[tile], ti & 1, abort_flag))) break;
        tc_fence_after();
        uint32_t sr[2][32];
        tmem_ld_32x32(tmem_s, sr[0]);
        tmem_ld_32x32(tmem_s + 32, sr[1]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.s_free[tile]);
        if (!(plain && key0 + T4_NK - 1 <= pos && key0 + T4_NK <= key_end)) {
          // the causal edge or the end of the range runs through this tile, or the row has a scale of its own
#pragma unroll
          for (int j = 0; j < T4_NK; ++j) {
            const int key = key0 + j;
            sr[j >> 5][j & 31] = valid && key < key_end && key <= pos ? __float_as_uint(__uint_as_float(sr[j >> 5][j & 31]) * rs.factor) : 0xff800000u;  // -inf
          }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          mx0 = fmaxf(mx0, __uint_as_float(sr[0][j]));
          mx1 = fmaxf(mx1, __uint_as_float(sr[1][j]));
        }
        const float mx = fmaxf(mx0, mx1);
        // raise m only when this tile is far above it: P then stays below 2^15, inside f16
        const bool raise = mx > m + T4_RAISE_AT || (m == -INFINITY && mx > -INFINITY);
        const float to = mx - T4_TOP;
        // the previous P V has completed: its P may be overwritten, and O may be touched
        if (ti > 0 && !(ok = t4_wait(&bars.o_done[tile], (ti - 1) & 1, abort_flag))) break;
        tc_fence_after();  // the stores below come behind that product's reads of P, whether or not O is touched
        if (ti > 0 && __any_sync(0xffffffffu, raise)) {
          const float alpha = raise ? ex2f(m - to) : 1.f;
#pragma unroll
          for (int cc = 0; cc < 9; ++cc) {
            uint32_t r[16];
            t4_tmem_ld16(tmem_o + 16 * cc, r);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * alpha);
            t4_tmem_st16(tmem_o + 16 * cc, r);
          }
          t4_tmem_st_wait();
        }
        if (raise) m = to;
        const float base = m == -INFINITY ? 0.f : m;
        // P, two keys a register, over the first half of the scores' registers
#pragma unroll
        for (int j = 0; j < T4_NK; j += 2)
          sr[0][j >> 1] = pack_half2(ex2f(__uint_as_float(sr[j >> 5][j & 31]) - base), ex2f(__uint_as_float(sr[(j + 1) >> 5][(j + 1) & 31]) - base));
        t4_tmem_st32(tmem_p, sr[0]);
        t4_tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_ready[tile]);
      }
      if (ok) ok = t4_wait(&bars.o_done[tile], (n_tiles - 1) & 1, abort_flag);
      if (ok) ok = t4_wait(&bars.v_ready[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, abort_flag);  // (long past: orders bad_v)
      tc_fence_after();
      if (ok) {
        // ---- O / l from TMEM (column 128 holds l).  The TMEM loads are warp-wide (.sync.aligned): every thread
        // executes them, only the global stores depend on `valid`.
        uint32_t r[32];
        tmem_ld_32x32(tmem_o + ATT_D, r);
        tmem_ld_wait();
        const bool hurt = __any_sync(0xffffffffu, bars.bad_v[lane & 7] != 0x7fffffff);
        const float l = __uint_as_float(r[0]);
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: zeros; NaN stays
        // Through shared memory, so that half a warp writes 256 bytes of a row (a row per thread: 11000 cycles for the partials).  The Q
        // tile's scores are all done, it is free: 8 KB per warp, [32 rows][16 pieces of 16 bytes], piece ^ (row & 7).
        uint8_t* stage = my_q + (warp & 3) * 8192;
        const bool partial = p.nsplit > 1;
        const int64_t at = partial ? (row * p.nsplit + sp) * (ATT_D * 4) : row * (ATT_D * 2);  // bytes
        uint8_t* const dst = (partial ? reinterpret_cast<uint8_t*>(p.part_o) : reinterpret_cast<uint8_t*>(p.out)) + (lane & 15) * 16;
        auto put = [&](int c, uint4 w) { *reinterpret_cast<uint4*>(stage + lane * 256 + ((c ^ (lane & 7)) << 4)) = w; };
        auto flush = [&](int off) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int src = 2 * i + (lane >> 4);
            const int64_t to = __shfl_sync(0xffffffffu, at, src);
            const bool live = __shfl_sync(0xffffffffu, (int)valid, src) != 0;
            const uint4 w = *reinterpret_cast<const uint4*>(stage + src * 256 + (((lane & 15) ^ (src & 7)) << 4));
            if (live) *reinterpret_cast<uint4*>(dst + to + off) = w;
          }
          __syncwarp();
        };
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          tmem_ld_32x32(tmem_o + 32 * cc, r);
          tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < 32; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * inv);
          if (hurt) {
            const bool bad0 = bars.bad_v[2 * cc] <= pos, bad1 = bars.bad_v[2 * cc + 1] <= pos;
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (x < 16 ? bad0 : bad1) r[x] = 0x7fc00000u;
          }
          if (partial) {
#pragma unroll
            for (int x = 0; x < 8; ++x) put((cc & 1) * 8 + x, make_uint4(r[4 * x], r[4 * x + 1], r[4 * x + 2], r[4 * x + 3]));
            if (cc & 1) flush((cc >> 1) * 256);
          } else {
            auto two = [&](int k) { return pack_bf16x2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])); };
#pragma unroll
            for (int x = 0; x < 4; ++x) put(cc * 4 + x, make_uint4(two(8 * x), two(8 * x + 2), two(8 * x + 4), two(8 * x + 6)));
          }
        }
        if (!partial) flush(0);
        if (valid && p.nsplit > 1) p.part_lse[row * p.nsplit + sp] = l > 0.f ? m + log2f(l) : (l == 0.f ? -INFINITY : l);
        __syncwarp();
      }
    }
  } else if (warp < 12) {
    // ======== dequantise ========
    const int dt = tid - 256;  // 0 .. 127
    {  // rows 128..143 of both V^T buffers: row 128 all ones (it sums the rows of P), the rest zero
      const uint32_t v = dt < 8 ? 0x3c003c00u : 0u;
      *reinterpret_cast<uint4*>(vt_s + ATT_D * 128 + dt * 16) = make_uint4(v, v, v, v);
      *reinterpret_cast<uint4*>(vt_s + T4_VT_BYTES + ATT_D * 128 + dt * 16) = make_uint4(v, v, v, v);
    }
    for (int ti = 0; ti < n_tiles; ++ti) {
      const int b = ti & 1;
      const uint8_t* st = raw_s + (ti % T4_STAGES) * T4_RAW;
      const int key0 = (page_begin + ti * T4_PAGES) * DASER_KV4_TOKENS;
      uint8_t* kb = k_s + b * T4_K_BYTES;
      uint8_t* vb = vt_s + b * T4_VT_BYTES;
      if (!(ok = t4_wait(&bars.raw_full[ti % T4_STAGES], (ti / T4_STAGES) & 1, abort_flag))) break;
      if (ti >= 2 && !(ok = t4_wait(&bars.k_free[b], (ti / 2 - 1) & 1, abort_flag))) break;
      // ---- K: (key, 16-dim group) items, four per thread ----
#pragma unroll
      for (int rep = 0; rep < 4; ++rep) {
        // four groups of a row on neighbouring lanes: their 16-byte pieces, and those of the row behind, are in different banks
        const int item = dt + 128 * rep;
        const int kt = (item >> 2) & 63, c = (item & 3) + 4 * (item >> 8);
        uint32_t h[8];
        if (key0 + kt < key_end) {
          const uint8_t* rec = st + (kt >> 4) * T4_PITCH;
          const int tok = kt & 15;
          const uint2 w = *reinterpret_cast<const uint2*>(rec + tok * 64 + c * 8);
          const uint32_t sc = (uint32_t)rec[DASER_KV4_KS + tok * 8 + c] * 0x00800080u;  // f16 bits = byte << 7, in both halves
          uint32_t x[4], y[4];
          e2m1x8_to_f16x2(w.x, x);
          e2m1x8_to_f16x2(w.y, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h[i] = hmul2_u32(x[i], sc);
            h[4 + i] = hmul2_u32(y[i], sc);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = 0u;
        }
        uint8_t* dst = kb + (c >> 2) * 8192 + kt * 128;
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3)) ^ (kt & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + (((2 * (c & 3) + 1) ^ (kt & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      t4_fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.k_ready[b]);
      if (key0 + T4_NK - 1 > seen_by_all) t4_leave_out_bad_values(raw_s + (ti % T4_STAGES) * T4_RAW, bars.bad_v, key0, key_end);
      if (ti >= 2 && !(ok = t4_wait(&bars.v_free[b], (ti / 2 - 1) & 1, abort_flag))) break;
      // ---- V^T: 8 keys x 8 dims per thread ----
      {
        const int ko = dt & 7, g = dt >> 4, hf = (dt >> 3) & 1;
        const uint8_t* rec = st + (ko >> 1) * T4_PITCH;
        const int left = key_end - (key0 + 8 * ko);  // keys of this octet that exist
        uint32_t v[8][4];  // [dim][key pair]
        if (left > 0) {
          const uint2 sw = *reinterpret_cast<const uint2*>(rec + DASER_KV4_VS + (ko & 1) * 64 + g * 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(rec + DASER_KV4_V + (ko & 1) * 512 + g * 64 + i * 16);
            const uint32_t w0 = hf ? w.y : w.x, w1 = hf ? w.w : w.z;  // 8 dims of tokens 2i, 2i + 1
            uint32_t sc = bperm(i < 2 ? sw.x : sw.y, 0u, (i & 1) ? 0x4342u : 0x4140u) << 7;
            sc &= left >= 2 * i + 2 ? 0xffffffffu : left == 2 * i + 1 ? 0xffffu : 0u;
            uint32_t e[4], o[4];
            e2m1x8_to_f16x2((w0 & 0x0f0f0f0fu) | ((w1 << 4) & 0xf0f0f0f0u), e);
            e2m1x8_to_f16x2(((w0 >> 4) & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u), o);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              v[2 * d][i] = hmul2_u32(e[d], sc);
              v[2 * d + 1][i] = hmul2_u32(o[d], sc);
            }
          }
        } else {
#pragma unroll
          for (int d = 0; d < 8; ++d) v[d][0] = v[d][1] = v[d][2] = v[d][3] = 0u;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = 16 * g + 8 * hf + j;
          *reinterpret_cast<uint4*>(vb + d * 128 + ((ko ^ j) << 4)) = make_uint4(v[j][0], v[j][1], v[j][2], v[j][3]);
        }
      }
      t4_fence_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars.v_ready[b]);
        mbar_arrive(&bars.raw_free[ti % T4_STAGES]);
      }
    }
  } else if (warp == 12) {
    // ======== MMAs: the warp walks the tiles together (its values stay in uniform registers), one lane issues ========
    constexpr uint32_t idesc_s = make_idesc_f16(128, T4_NK, 0);
    constexpr uint32_t idesc_o = make_idesc_f16(128, T4_ON, 0);
    const bool leader = elect_one();
    // descriptors: the low word moves by (bytes >> 4), the high word is common
    const uint32_t hi = (uint32_t)(make_desc_k_sw128(0) >> 32);
    const uint32_t lo_q = (uint32_t)make_desc_k_sw128(q_u32), lo_k = (uint32_t)make_desc_k_sw128(k_u32);
    const uint32_t lo_v = (uint32_t)make_desc_k_sw128(vt_u32);
    auto desc = [&](uint32_t lo) { return (uint64_t)hi << 32 | lo; };
    auto scores = [&](int t, int ti) {  // S of row tile t against key tile ti
      tc_fence_after();
      if (leader) {
        const uint32_t da = lo_q + t * (T4_Q_BYTES >> 4), db = lo_k + (ti & 1) * (T4_K_BYTES >> 4);
        const uint32_t d = tmem + t4_s_col(t);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          umma_f16(d, desc(da + (k >> 2) * (16384 >> 4) + 2 * (k & 3)), desc(db + (k >> 2) * (8192 >> 4) + 2 * (k & 3)), idesc_s, k ? 1u : 0u);
        umma_commit(&bars.s_ready[t]);
        if (t == tiles - 1) umma_commit(&bars.k_free[ti & 1]);
      }
      __syncwarp();
    };
    auto outputs = [&](int t, int pi) {  // O of row tile t += P V of key tile pi
      tc_fence_after();
      if (leader) {
        const uint32_t db = lo_v + (pi & 1) * (T4_VT_BYTES >> 4);
        const uint32_t d = tmem + t4_o_col(t), a = tmem + t4_p_col(t);
#pragma unroll
        for (int k = 0; k < 4; ++k) t4_umma_ts(d, a + 8 * k, desc(db + 2 * k), idesc_o, (pi | k) ? 1u : 0u);
        umma_commit(&bars.o_done[t]);
        if (t == tiles - 1) umma_commit(&bars.v_free[pi & 1]);
      }
      __syncwarp();
    };
    ok = t4_wait(&bars.q_ready, 0, abort_flag);
    for (int ti = 0; ok && ti <= n_tiles; ++ti) {
      const int pi = ti - 1;
      if (ti < n_tiles && !(ok = t4_wait(&bars.k_ready[ti & 1], (ti >> 1) & 1, abort_flag))) break;
      for (int t = 0; t < tiles; ++t) {
        if (ti < n_tiles) {
          if (ti > 0 && !(ok = t4_wait(&bars.s_free[t], pi & 1, abort_flag))) break;
          scores(t, ti);
        }
        if (ti > 0) {
          if (t == 0 && !(ok = t4_wait(&bars.v_ready[pi & 1], (pi >> 1) & 1, abort_flag))) break;
          if (!(ok = t4_wait(&bars.p_ready[t], pi & 1, abort_flag))) break;
          outputs(t, pi);
        }
      }
    }
    // nothing may be in flight when the tensor memory goes back
    if (leader) umma_commit(&bars.drain);
    __syncwarp();
    uint32_t none = 0u;
    if (!t4_wait(&bars.drain, 0, &none)) ok = false;
  } else if (lane == 0) {
    // ======== fetch ========
    const uint8_t* base = p.records + (int64_t)kvh * p.stride_head;
    int issued = 0;
    for (; issued < n_tiles; ++issued) {
      const int s = issued % T4_STAGES;
      if (issued >= T4_STAGES && !(ok = mbar_wait(&bars.raw_free[s], (issued / T4_STAGES - 1) & 1, abort_flag))) break;
      const int n = min(T4_PAGES, page_end - page_begin - issued * T4_PAGES);
      mbar_expect_tx(&bars.raw_full[s], n * DASER_KV4_RECORD);
#pragma unroll
      for (int pg = 0; pg < T4_PAGES; ++pg) {
        if (pg >= n) break;
        const int bk = blk[pg] < 0 ? 0 : (blk[pg] >= p.num_blocks ? p.num_blocks - 1 : blk[pg]);
        t4_bulk_load(raw_u32 + s * T4_RAW + pg * T4_PITCH, base + (int64_t)bk * p.stride_block, DASER_KV4_RECORD, &bars.raw_full[s]);
      }
      ids(issued + 1);
    }
    // the copies in flight have landed before the shared memory goes away (the others wait for them too, unless they gave up)
    for (int i = max(0, issued - T4_STAGES); i < issued; ++i) {
      uint32_t none = 0u;
      if (!mbar_wait(&bars.raw_full[i % T4_STAGES], (i / T4_STAGES) & 1, &none)) ok = false;
    }
  }
  tc_fence_before();
  const bool aborted = __syncthreads_or(!ok) != 0;
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, T4_TMEM_COLS);
  }
  if (aborted && tid == 0) atomicOr(&g_attn4_tc_status, 1u);
}

}  // namespace daser

int daser_launch_attention4_tc(const daser::Attn4Params& p, int max_q_len, cudaStream_t stream) {
  using namespace daser;
  static bool configured[DASER_MAX_DEVICES] = {false};  // per device: the attribute is the device's
  if (daser_first_use_on_device(configured)) {
    cudaError_t e = cudaFuncSetAttribute(attn4_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T4_SMEM);
    if (e != cudaSuccess) return (int)e;
    daser_used_on_device(configured);
  }
  const int toks = 2 * (128 / p.G);
  const int groups = (max_q_len + toks - 1) / toks;
  const int64_t z = (int64_t)groups * p.nsplit;
  if (z > 65535 || p.num_seqs > 65535) return DASER_ERR_TOO_LARGE;
  return (int)launch_pdl(attn4_tc_kernel, dim3(p.Hkv, p.num_seqs, (unsigned)z), dim3(T4_THREADS), T4_SMEM, stream, p, groups);
}

// Non-zero once any CTA of the 4-bit prefill kernel gave up on a bounded wait (synchronises the device).
DASER_API int daser_attention4_tc_status(uint32_t* out) {
  uint32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, daser::g_attn4_tc_status, sizeof(v));
  if (out) *out = v;
  return (int)e;
}
