// Which pages a query reads: a cheap upper bound on the scores of every page, and the best pages by it.
//
// For a query row and a KV head, sum over the head's query heads h of the bound of a page:
//   sum_h sum_d max(q_hd hi_d, q_hd lo_d) = sum_d Q+_d hi_d + Q-_d lo_d,   Q+ = sum_h max(q_h, 0), Q- = sum_h min(q_h, 0)
// so the heads of a group collapse into two vectors.  Q+ and Q- are rounded to int8 with one power-of-two scale (it is common to
// all pages and drops out), the bounds are int8 already: a page costs 256 integer products, |sum| <= 256 * 127^2 < 2^24, and
// its score, the sum times the page's power of two, is exact in fp32.  The choice therefore depends on no order of summation.
// The chosen pages: the first `sink`, the last `recent`, and of the others the highest scores, the lower page first among equals.
//
// attn4_score_kernel is bound by the 256 bytes of bounds per page and head and the table in front of them: 16 sequences of 16k - 64k
// tokens, 8 KV heads, 82 MB: 20 us, 4.1 TB/s (a batch of pages is read ahead of the one in work: 22 without).  attn4_select_kernel
// (one CTA per list) is bound by latency: 10 us for lists of 1k - 4k pages, 12 us for 8192: a pass over the scores, two rounds of
// bins, a pass that writes.  (Rounds of 13 bits instead of 11 clear and add up four times the bins: 12 us against 10.)
#include "attention4_params.cuh"

namespace daser {

constexpr int SCORE_PAGES = 128;    // pages per CTA of the score kernel: 8 per half-warp
constexpr int SELECT_THREADS = 1024;
constexpr int SELECT_DIGIT = 11;
constexpr int SELECT_BINS = 1 << SELECT_DIGIT;
static_assert(SELECT_THREADS == 32 * 32, "one warp can hold a value of every warp");
constexpr int SELECT_SMEM_KEYS = 40960;  // longer lists are read from global memory in every pass

struct Select4Params {
  const __nv_bfloat16* q;    // [Tq, Hq, 128]
  const int8_t* codes;       // the layer's bounds [blocks][heads][2][128]
  const int8_t* exps;        // [blocks][heads]
  const int32_t* block_tables;
  const int32_t* q_start;
  const int32_t* ctx_lens;
  float* scores;             // [Tq, Hkv, stride]
  int32_t* pages;            // [Tq, Hkv, n_pages]
  int max_blocks, num_blocks, Hq, Hkv, G, max_q_len, total_q;
  int stride, n_pages, sink, recent;
  int batches;               // of SCORE_PAGES pages per CTA of the score kernel
};

// The query row of (sequence, offset) and the pages it sees; false if there is no such row.
__device__ __forceinline__ bool select_row(const Select4Params& p, int seq, int off, int& row, int& count) {
  const int q0 = p.q_start[seq], q1 = p.q_start[seq + 1];
  row = q0 + off;
  if (q0 < 0 || row >= min(q1, p.total_q)) return false;
  const int pos = p.ctx_lens[seq] - (q1 - q0) + off;  // last visible key
  count = pos < 0 ? 0 : min(pos / DASER_KV4_TOKENS + 1, min(p.max_blocks, p.stride));
  return true;
}

__device__ __forceinline__ double warp_max_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__global__ void __launch_bounds__(256, 3)
attn4_score_kernel(const Select4Params p) {
  __shared__ double s_max[4];
  __shared__ __align__(16) int8_t s_q[2 * ATT_D];
  pdl_enter();
  const int seq = blockIdx.z / p.max_q_len, off = blockIdx.z % p.max_q_len, kvh = blockIdx.y;
  int row, count;
  if (!select_row(p, seq, off, row, count)) return;
  const int span = SCORE_PAGES * p.batches;
  const int lo_page = max(p.sink, (int)blockIdx.x * span);
  const int hi_page = min(count - p.recent, ((int)blockIdx.x + 1) * span);
  if (count <= p.n_pages || lo_page >= hi_page) return;  // everything is chosen, or nothing here needs a score

  // Sixteen lanes a page, 16 bytes a lane, eight pages a half-warp and batch.  A batch's loads are issued before the batch in front of it
  // is worked on (the first one's before the query is prepared): the block id is a dependent load in front of them, and nothing
  // else hides either.
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks;
  int my_page = blockIdx.x * span + (threadIdx.x >> 4) * 8 + (sub >> 1);  // whose score this lane ends up with
  auto block_of = [&](int page) {
    const int blk = table[min(page, count - 1)];
    return blk < 0 ? 0 : (blk >= p.num_blocks ? p.num_blocks - 1 : blk);
  };
  int4 c[8];
  int e = 0;
  auto load = [&](int blk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int b = __shfl_sync(0xffffffffu, blk, (lane & 16) + 2 * i);
      c[i] = *reinterpret_cast<const int4*>(p.codes + ((int64_t)b * p.Hkv + kvh) * (2 * ATT_D) + 16 * sub);
    }
    e = p.exps[(int64_t)blk * p.Hkv + kvh];
  };
  load(block_of(my_page));
  int blk_next = block_of(my_page + SCORE_PAGES);

  double up = 0.0, down = 0.0;  // sums of at most 16 bf16 values: exact
  if (threadIdx.x < ATT_D) {
    const __nv_bfloat16* qp = p.q + ((int64_t)row * p.Hq + kvh * p.G) * ATT_D + threadIdx.x;
    float x[16];
#pragma unroll
    for (int h = 0; h < 16; ++h) x[h] = h < p.G ? __bfloat162float(qp[h * ATT_D]) : 0.f;
#pragma unroll
    for (int h = 0; h < 16; ++h) {
      if (h >= p.G) break;
      up += (double)fmaxf(x[h], 0.f);
      down += (double)fminf(x[h], 0.f);
    }
    const double mx = warp_max_f64(fmax(up, -down));
    if (lane == 0) s_max[threadIdx.x >> 5] = mx;
  }
  __syncthreads();
  if (threadIdx.x < ATT_D) {
    const double a = fmax(fmax(s_max[0], s_max[1]), fmax(s_max[2], s_max[3]));
    double f = 1.0;  // 2^-x, x the smallest with a <= 127 * 2^x
    if (a > 0.0) {
      const uint64_t b = (uint64_t)__double_as_longlong(a);
      const int x = (int)(b >> 52) - 1022 - 7 + ((b & 0xfffffffffffffull) > (63ull << 46) ? 1 : 0);
      f = __longlong_as_double((long long)(uint64_t)(1023 - x) << 52);
    }
    s_q[threadIdx.x] = (int8_t)__double2int_rn(up * f);
    s_q[ATT_D + threadIdx.x] = (int8_t)__double2int_rn(down * f);
  }
  __syncthreads();
  const int4 qv = *reinterpret_cast<const int4*>(s_q + 16 * sub);
  float* dst = p.scores + ((int64_t)row * p.Hkv + kvh) * p.stride;
  const int batches = min(p.batches, (hi_page - (int)blockIdx.x * span + SCORE_PAGES - 1) / SCORE_PAGES);
  for (int k = 0; k < batches; ++k) {
    int dot[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dot[i] = __dp4a(c[i].x, qv.x, __dp4a(c[i].y, qv.y, __dp4a(c[i].z, qv.z, __dp4a(c[i].w, qv.w, 0))));
    // exponent 127: a key of the page is not finite; such a page is always read
    const float scale = e == 127 ? INFINITY : __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
    const int page = my_page;
    my_page += SCORE_PAGES;
    if (k + 1 < batches) {
      load(blk_next);
      blk_next = block_of(my_page + SCORE_PAGES);
    }
    // sum over the sixteen lanes and transpose: a lane keeps half of its pages at each step, in the end page sub / 2
#pragma unroll
    for (int n = 4, o = 8; n > 0; n >>= 1, o >>= 1) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const bool high = (sub & o) != 0;
        const int keep = high ? dot[n + i] : dot[i], give = high ? dot[i] : dot[n + i];
        dot[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
    dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], 1);
    if ((sub & 1) == 0 && page >= lo_page && page < hi_page) dst[page] = scale == INFINITY ? INFINITY : (float)dot[0] * scale;
  }
}

// Floats in the order of unsigned integers.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);  // -0 ranks with 0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Exclusive sum of v over the block (every thread calls it).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane] : 0u);
  return before + x - v;
}

__global__ void __launch_bounds__(SELECT_THREADS)
attn4_select_kernel(const Select4Params p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ uint32_t s_bins[SELECT_BINS];
  __shared__ uint32_t s_warp[SELECT_THREADS / 32], s_lo[SELECT_THREADS / 32], s_hi[SELECT_THREADS / 32];
  __shared__ uint32_t s_bin, s_above, s_in;
  pdl_enter();
  const int tid = threadIdx.x;
  const int seq = blockIdx.y / p.max_q_len, off = blockIdx.y % p.max_q_len, kvh = blockIdx.x;
  int row, count;
  if (!select_row(p, seq, off, row, count)) return;
  int32_t* list = p.pages + ((int64_t)row * p.Hkv + kvh) * p.n_pages;
  if (count <= p.n_pages) {
    for (int i = tid; i < p.n_pages; i += SELECT_THREADS) list[i] = i < count ? i : -1;
    return;
  }
  const int n = count - p.sink - p.recent;               // pages that compete ...
  int need = p.n_pages - p.sink - p.recent;              // ... for so many places: 0 <= need < n
  for (int i = tid; i < p.sink; i += SELECT_THREADS) list[i] = i;
  for (int i = tid; i < p.recent; i += SELECT_THREADS) list[p.n_pages - p.recent + i] = count - p.recent + i;
  if (need == 0) return;
  const float* src = p.scores + ((int64_t)row * p.Hkv + kvh) * p.stride + p.sink;
  const bool cached = n <= SELECT_SMEM_KEYS;
  uint32_t lo = 0xffffffffu, hi = 0u;
  for (int i = tid; i < n; i += SELECT_THREADS) {
    const uint32_t k = ordered(src[i]);
    if (cached) s_keys[i] = k;
    lo = min(lo, k);
    hi = max(hi, k);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((tid & 31) == 0) { s_lo[tid >> 5] = lo; s_hi[tid >> 5] = hi; }
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, s_lo[tid & 31]);
  hi = __reduce_max_sync(0xffffffffu, s_hi[tid & 31]);
  __syncthreads();  // s_lo and s_hi are used again below
  auto key = [&](int i) { return cached ? s_keys[i] : ordered(src[i]); };

  // The need-th largest key, by digits of up to SELECT_DIGIT bits from the first bit in which the keys differ.
  // Invariant: keys whose bits from `shift` up exceed `prefix` are chosen, `need` more are among those equal to it.
  int shift = lo == hi ? 0 : 32 - __clz(lo ^ hi);
  uint32_t prefix = shift >= 32 ? 0u : hi >> shift;
  bool whole = false;  // all keys that match the prefix are chosen
  while (shift > 0 && !whole) {
    const int width = min(shift, SELECT_DIGIT);
    const int at = shift - width;
    const uint32_t mask = (1u << width) - 1u;
    for (int i = tid; i < SELECT_BINS; i += SELECT_THREADS) s_bins[i] = 0u;
    __syncthreads();
    for (int i = tid; i < n; i += SELECT_THREADS) {
      const uint32_t k = key(i);
      if (shift >= 32 || (k >> shift) == prefix) atomicAdd(&s_bins[(k >> at) & mask], 1u);
    }
    __syncthreads();
    // bins from the top: two a thread
    constexpr int PER = SELECT_BINS / SELECT_THREADS;
    uint32_t c[PER], sum = 0;
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      c[x] = s_bins[SELECT_BINS - 1 - (tid * PER + x)];
      sum += c[x];
    }
    uint32_t above = block_scan(sum, s_warp);
    if (above < (uint32_t)need && above + sum >= (uint32_t)need) {
#pragma unroll
      for (int x = 0; x < PER; ++x) {
        if (above < (uint32_t)need && above + c[x] >= (uint32_t)need) {
          s_bin = SELECT_BINS - 1 - (tid * PER + x);
          s_above = above;
          s_in = c[x];
        }
        above += c[x];
      }
    }
    __syncthreads();
    prefix = (shift >= 32 ? 0u : prefix << width) | s_bin;
    need -= (int)s_above;
    whole = s_in == (uint32_t)need;
    shift = at;
    __syncthreads();
  }
  // keys above `thr` are chosen, and the first `need` of those equal to it; when all that match the prefix are, thr lies below them
  // (prefix is not zero then: some key is not chosen)
  const uint32_t thr = whole ? (prefix << shift) - 1u : prefix;
  const int eq_need = whole ? 0 : need;
  // In ascending order: a warp owns a run of keys and takes 32 at a time (contiguous in shared memory), ballots count them.
  const int lane = tid & 31, warp = tid >> 5;
  const uint32_t below = (1u << lane) - 1u;
  const int run = ((n + SELECT_THREADS - 1) / SELECT_THREADS) * 32;
  const int i0 = min(warp * run, n), i1 = min(i0 + run, n);
  uint32_t gt = 0, eq = 0;
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, in && k > thr));
    eq += __popc(__ballot_sync(0xffffffffu, in && k == thr));
  }
  if (lane == 0) { s_lo[warp] = gt; s_hi[warp] = eq; }
  __syncthreads();
  int g = 0, e = 0;
  for (int w = 0; w < warp; ++w) { g += (int)s_lo[w]; e += (int)s_hi[w]; }
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, in && k > thr), me = __ballot_sync(0xffffffffu, in && k == thr);
    const int my_e = e + __popc(me & below);
    if (in && (k > thr || (k == thr && my_e < eq_need))) list[p.sink + g + __popc(mg & below) + min(my_e, eq_need)] = p.sink + i + lane;
    g += __popc(mg);
    e += __popc(me);
  }
}

}  // namespace daser

// pages int32 [total_q][Hkv][n_pages]: for every query row and KV head the pages to read, ascending, -1 behind the last.
// scores: scratch of total_q * Hkv * stride floats, stride >= the pages of the longest context.
DASER_API int daser_select_pages_kv4(const void* q, const int8_t* codes, const int8_t* exps, int layer, int num_blocks,
                                     const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                                     int num_seqs, int total_q, int max_q_len, int Hq, int Hkv, float* scores, int stride,
                                     int32_t* pages, int n_pages, int sink, int recent, cudaStream_t stream) {
  using namespace daser;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || layer < 0 || num_blocks <= 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (num_seqs < 0 || total_q < 0 || max_q_len < 0 || stride < 1) return DASER_ERR_BAD_ARG;
  if (n_pages < 1 || sink < 0 || recent < 1 || (int64_t)sink + recent > n_pages) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !codes || !exps || !block_tables || !q_start || !ctx_lens || !scores || !pages) return DASER_ERR_BAD_ARG;
  if (Hq / Hkv > 16 || (uintptr_t)codes % 16) return DASER_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)num_seqs * max_q_len;
  if (rows > 65535 || Hkv > 65535 || max_blocks > (1 << 29) / DASER_KV4_TOKENS) return DASER_ERR_TOO_LARGE;
  Select4Params p;
  p.q = (const __nv_bfloat16*)q;
  p.codes = codes + (int64_t)layer * num_blocks * Hkv * 2 * ATT_D;
  p.exps = exps + (int64_t)layer * num_blocks * Hkv;
  p.block_tables = block_tables;
  p.q_start = q_start;
  p.ctx_lens = ctx_lens;
  p.scores = scores;
  p.pages = pages;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_q_len = max_q_len;
  p.total_q = total_q;
  p.stride = stride;
  p.n_pages = n_pages;
  p.sink = sink;
  p.recent = recent;
  static bool configured[DASER_MAX_DEVICES] = {false};  // per device: the attribute is the device's
  if (daser_first_use_on_device(configured)) {
    cudaError_t e = cudaFuncSetAttribute(attn4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SELECT_SMEM_KEYS * 4);
    if (e != cudaSuccess) return (int)e;
  }
  if (stride > n_pages) {
    // One batch a CTA while that fills the GPU no more than twice (3 resident an SM), four beyond: 16 sequences of 16k - 64k tokens 65 us
    // for the whole step with one, 59 to 63 with two to eight; 64 chunks (131072 tokens, 8 heads) fill it once.
    const int64_t chunks = (stride + SCORE_PAGES - 1) / SCORE_PAGES;
    p.batches = chunks * Hkv * rows > 2 * 148 * 3 ? 4 : 1;
    cudaError_t e = launch_pdl(attn4_score_kernel, dim3((unsigned)((chunks + p.batches - 1) / p.batches), (unsigned)Hkv, (unsigned)rows),
                               dim3(256), 0, stream, p);
    if (e != cudaSuccess) return (int)e;
  }
  const size_t smem = (size_t)(stride < SELECT_SMEM_KEYS ? stride : SELECT_SMEM_KEYS) * 4;
  return (int)launch_pdl(attn4_select_kernel, dim3((unsigned)Hkv, (unsigned)rows), dim3(SELECT_THREADS), smem, stream, p);
}
