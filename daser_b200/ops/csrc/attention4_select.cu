// Which pages a query reads: a cheap estimate of the largest score of every page, and the best pages by it.
//
// For a query row and a KV head, sum over the head's query heads h of the bound of a page:
//   sum_h sum_d max(q_hd hi_d, q_hd lo_d) = sum_d Q+_d hi_d + Q-_d lo_d,   Q+ = sum_h max(q_h, 0), Q- = sum_h min(q_h, 0)
// so the heads of a group collapse into two vectors.  Q+ and Q- are rounded to int8 with one power-of-two scale (it is common to
// all pages and drops out), to nearest, so that the score lies up to half a step per dim on either side of that bound: of 4096 pages and
// 128 places one to three go to other pages than by the bound itself with normal queries, up to 9 % of them with one loud channel.  That is the
// price of whole numbers: the bounds are int8 already, a page costs 256 integer products, |sum| <= 256 * 127^2 < 2^24, and
// its score, the sum times the page's power of two, is exact in fp32.  The choice therefore depends on no order of summation.
// (Q+ and Q- are sums of up to 16 bf16 values in fp64, exact while their exponents lie within 41 of one another, and
// always made in the order of the heads.)
// The chosen pages: the first `sink`, the last `recent`, and of the others the highest scores, the lower page first among equals.
//
// One kernel: a cluster of up to 8 CTAs makes a list.  Each scores its share of the pages, keeps the scores on chip and counts them into
// bins; the counts are read across the cluster's shared memory, so that every CTA finds the same threshold and writes its own
// part of the list.  The bounds, 256 bytes per page and head, are read once; the rest is latency: lengths, table, bounds, up to four
// rounds of bins.  Measured: 16 sequences of 16k - 64k tokens, 8 KV heads, 82 MB: 27 us (a kernel for scores and one CTA per list for the
// choice: 20 + 10); one of 131072 tokens: 16 us (8 + 12); 2 lists of 300 pages: 10 us (6 + 6).  Bins of 11 bits, eight a thread, read
// from every CTA: 30 us for the second, 124 for the first with clusters of 8: the reading across the cluster then outweighs all else.
#include "attention4_params.cuh"

namespace daser {
using namespace sm100;

constexpr int SELECT_THREADS = 512;
constexpr int SELECT_WARPS = SELECT_THREADS / 32;
constexpr int SELECT_BATCH = SELECT_THREADS / 2;  // pages per CTA and batch: 8 per half-warp
constexpr int SELECT_DIGIT = 8;     // bits a round: a bin per thread, so that reading all CTAs' bins is one load for each of them
constexpr int SELECT_BINS = 1 << SELECT_DIGIT;
static_assert(SELECT_BINS <= SELECT_THREADS, "a bin per thread");
constexpr int SELECT_KEYS = 16384;  // scores a CTA keeps on chip; longer shares are kept in global memory
constexpr int SELECT_CLUSTER = 8;   // CTAs a list at most

struct Select4Params {
  const __nv_bfloat16* q;    // [Tq, Hq, 128]
  const int8_t* codes;       // the layer's bounds [blocks][heads][2][128]
  const int8_t* exps;        // [blocks][heads]
  const int32_t* block_tables;
  const int32_t* q_start;
  const int32_t* ctx_lens;
  float* scores;             // [Tq, Hkv, stride], used when a share exceeds SELECT_KEYS
  int32_t* pages;            // [Tq, Hkv, n_pages]
  int max_blocks, num_blocks, num_seqs, Hq, Hkv, G, max_q_len, total_q;
  int by_row;                // a CTA's row comes from its index in all rows, not in num_seqs * max_q_len of them
  int stride, n_pages, sink, recent;
  int cluster;               // CTAs per list
  int keys;                  // places for scores in a CTA's shared memory; 0: they are in `scores`
};

// The i-th query row, its sequence and the pages it sees; false if there is no such row.  Whole warps call it.
__device__ __forceinline__ bool select_row(const Select4Params& p, int i, int& seq, int& row, int& count) {
  int off = 0;
  if (p.by_row) {
    const int lane = threadIdx.x & 31;
    uint32_t mine = 0;
    for (int base = 0; base < p.num_seqs && mine == 0; base += 32) {
      seq = min(base + lane, p.num_seqs - 1);
      off = i - p.q_start[seq];
      mine = __ballot_sync(0xffffffffu, base + lane < p.num_seqs && off >= 0 && i < p.q_start[seq + 1] && off < p.max_q_len);
    }
    if (mine == 0) return false;
    seq = __shfl_sync(0xffffffffu, seq, __ffs(mine) - 1);
    off = __shfl_sync(0xffffffffu, off, __ffs(mine) - 1);
  } else {
    seq = i / p.max_q_len;
    off = i - seq * p.max_q_len;
  }
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

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Of the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote(uint32_t smem_addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint2 remote_u32x2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(SELECT_THREADS, 2)
attn4_select_kernel(const Select4Params p) {
  extern __shared__ uint32_t s_keys[];
  __shared__ __align__(16) uint32_t s_bins[2][SELECT_BINS];
  __shared__ double s_max[4];
  __shared__ __align__(16) int8_t s_q[2 * ATT_D];
  __shared__ uint32_t s_warp[SELECT_WARPS], s_a[SELECT_WARPS], s_b[SELECT_WARPS];
  __shared__ __align__(8) uint2 s_share[2];  // read by the other CTAs: lowest and highest key, counts above and at the threshold
  __shared__ uint32_t s_bin, s_above, s_in;
  pdl_launch_dependents();  // (launched the plain way: its predecessor has ended)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = p.cluster, rank = blockIdx.x % C, kvh = blockIdx.x / C % p.Hkv;
  int seq, row, count;
  if (!select_row(p, blockIdx.x / C / p.Hkv, seq, row, count)) return;  // (this and the next two returns: all CTAs of the cluster alike)
  int32_t* list = p.pages + ((int64_t)row * p.Hkv + kvh) * p.n_pages;
  if (count <= p.n_pages) {
    if (rank == 0)
      for (int i = tid; i < p.n_pages; i += SELECT_THREADS) list[i] = i < count ? i : -1;
    return;
  }
  const int n = count - p.sink - p.recent;               // pages that compete ...
  int need = p.n_pages - p.sink - p.recent;              // ... for so many places: 0 <= need < n
  if (rank == 0) {
    for (int i = tid; i < p.sink; i += SELECT_THREADS) list[i] = i;
    for (int i = tid; i < p.recent; i += SELECT_THREADS) list[p.n_pages - p.recent + i] = count - p.recent + i;
  }
  if (need == 0) return;
  const int share = (n + C - 1) / C;  // of the pages that compete, [begin, end) is this CTA's
  const int begin = min(rank * share, n), end = min(begin + share, n), mine = end - begin;
  const bool cached = p.keys > 0;
  float* kept = p.scores + ((int64_t)row * p.Hkv + kvh) * p.stride + begin;

  // ---- scores ----
  // Sixteen lanes a page, 16 bytes a lane, eight pages a half-warp and batch.  A batch's loads are issued before the batch in front of
  // it is worked on (the first one's before the query is prepared): the block id is a dependent load in front of them, and
  // nothing else hides either.
  const int sub = lane & 15;
  const int32_t* table = p.block_tables + (int64_t)seq * p.max_blocks + p.sink;
  int at = (tid >> 4) * 8 + (sub >> 1);  // whose score this lane ends up with: page begin + at of those that compete
  auto block_of = [&](int i) {
    const int blk = table[min(begin + i, n - 1)];
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
  load(block_of(at));
  int blk_next = block_of(at + SELECT_BATCH);
  for (int i = tid; i < 2 * SELECT_BINS; i += SELECT_THREADS) s_bins[0][i] = 0u;

  double up = 0.0, down = 0.0;
  if (tid < ATT_D) {
    const __nv_bfloat16* qp = p.q + ((int64_t)row * p.Hq + kvh * p.G) * ATT_D + tid;
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
    if (lane == 0) s_max[warp] = mx;
  }
  __syncthreads();
  if (tid < ATT_D) {
    const double a = fmax(fmax(s_max[0], s_max[1]), fmax(s_max[2], s_max[3]));
    double f = 1.0;  // 2^-x, x the smallest with a <= 127 * 2^x
    if (a > 0.0) {
      const uint64_t b = (uint64_t)__double_as_longlong(a);
      const int x = (int)(b >> 52) - 1022 - 7 + ((b & 0xfffffffffffffull) > (63ull << 46) ? 1 : 0);
      f = __longlong_as_double((long long)(uint64_t)(1023 - x) << 52);
    }
    s_q[tid] = (int8_t)__double2int_rn(up * f);
    s_q[ATT_D + tid] = (int8_t)__double2int_rn(down * f);
  }
  __syncthreads();
  const int4 qv = *reinterpret_cast<const int4*>(s_q + 16 * sub);
  uint32_t lo = 0xffffffffu, hi = 0u;
  for (int done = 0; done < mine; done += SELECT_BATCH, at += SELECT_BATCH) {
    int dot[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dot[i] = __dp4a(c[i].x, qv.x, __dp4a(c[i].y, qv.y, __dp4a(c[i].z, qv.z, __dp4a(c[i].w, qv.w, 0))));
    // exponent 127: a key of the page is not finite; such a page is always read
    const float scale = e == 127 ? INFINITY : __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
    if (done + SELECT_BATCH < mine) {
      load(blk_next);
      blk_next = block_of(at + 2 * SELECT_BATCH);
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
    if ((sub & 1) == 0 && at < mine) {
      const uint32_t k = ordered(scale == INFINITY ? INFINITY : (float)dot[0] * scale);
      if (cached) s_keys[at] = k;
      else kept[at] = __uint_as_float(k);
      lo = min(lo, k);
      hi = max(hi, k);
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) { s_a[warp] = lo; s_b[warp] = hi; }
  __syncthreads();
  if (warp == 0) {
    lo = __reduce_min_sync(0xffffffffu, s_a[lane % SELECT_WARPS]);
    hi = __reduce_max_sync(0xffffffffu, s_b[lane % SELECT_WARPS]);
    if (lane == 0) s_share[0] = make_uint2(lo, hi);
  }
  cluster_sync();
  for (int r = 0; r < C; ++r) {
    const uint2 v = remote_u32x2(remote(smem_u32(&s_share[0]), r));
    lo = r == 0 ? v.x : min(lo, v.x);
    hi = r == 0 ? v.y : max(hi, v.y);
  }
  auto key = [&](int i) { return cached ? s_keys[i] : __float_as_uint(kept[i]); };

  // ---- the need-th largest key, by digits of up to SELECT_DIGIT bits from the first bit in which the keys differ ----
  // Invariant: keys whose bits from `shift` up exceed `prefix` are chosen, `need` more are among those equal to it.  The bins take turns: one
  // set is cleared when every CTA has passed the barrier behind its last reading.
  int shift = lo == hi ? 0 : 32 - __clz(lo ^ hi);
  uint32_t prefix = shift >= 32 ? 0u : hi >> shift;
  bool whole = false;  // all keys that match the prefix are chosen
  for (int set = 0; shift > 0 && !whole; set ^= 1) {
    const int width = min(shift, SELECT_DIGIT);
    const int low = shift - width;
    const uint32_t mask = (1u << width) - 1u;
    for (int i = tid; i < mine; i += SELECT_THREADS) {
      const uint32_t k = key(i);
      if (shift >= 32 || (k >> shift) == prefix) atomicAdd(&s_bins[set][(k >> low) & mask], 1u);
    }
    cluster_sync();
    uint32_t in = 0;  // bins from the top, one a thread
    if (tid < SELECT_BINS) {
      s_bins[set ^ 1][tid] = 0u;
      const uint32_t bin = smem_u32(&s_bins[set][SELECT_BINS - 1 - tid]);
#pragma unroll
      for (int r = 0; r < SELECT_CLUSTER; ++r)
        if (r < C) in += remote_u32(remote(bin, r));
    }
    const uint32_t above = block_scan(in, s_warp);
    if (above < (uint32_t)need && above + in >= (uint32_t)need) {
      s_bin = SELECT_BINS - 1 - tid;
      s_above = above;
      s_in = in;
    }
    __syncthreads();
    prefix = (shift >= 32 ? 0u : prefix << width) | s_bin;
    need -= (int)s_above;
    whole = s_in == (uint32_t)need;
    shift = low;
    __syncthreads();
  }
  // keys above `thr` are chosen, and the first `need` of those equal to it; when all that match the prefix are, thr lies below them
  // (prefix is not zero then: some key is not chosen)
  const uint32_t thr = whole ? (prefix << shift) - 1u : prefix;
  const int eq_need = whole ? 0 : need;
  // ---- the list, in ascending order: a warp owns a run of keys and takes 32 at a time, ballots count them ----
  const uint32_t below = (1u << lane) - 1u;
  const int run = ((mine + SELECT_THREADS - 1) / SELECT_THREADS) * 32;
  const int i0 = min(warp * run, mine), i1 = min(i0 + run, mine);
  uint32_t gt = 0, eq = 0;
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, in && k > thr));
    eq += __popc(__ballot_sync(0xffffffffu, in && k == thr));
  }
  if (lane == 0) { s_a[warp] = gt; s_b[warp] = eq; }
  __syncthreads();
  int g = 0, q = 0;  // in front of this warp
  uint32_t all_g = 0, all_q = 0;
#pragma unroll
  for (int w = 0; w < SELECT_WARPS; ++w) {
    if (w == warp) { g = (int)all_g; q = (int)all_q; }
    all_g += s_a[w];
    all_q += s_b[w];
  }
  if (tid == 0) s_share[1] = make_uint2(all_g, all_q);
  cluster_sync();
  for (int r = 0; r < rank; ++r) {
    const uint2 v = remote_u32x2(remote(smem_u32(&s_share[1]), r));
    g += (int)v.x;
    q += (int)v.y;
  }
  for (int i = i0; i < i1; i += 32) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    const uint32_t mg = __ballot_sync(0xffffffffu, in && k > thr), me = __ballot_sync(0xffffffffu, in && k == thr);
    const int my_q = q + __popc(me & below);
    if (in && (k > thr || (k == thr && my_q < eq_need))) list[p.sink + g + __popc(mg & below) + min(my_q, eq_need)] = p.sink + begin + i + lane;
    g += __popc(mg);
    q += __popc(me);
  }
  cluster_sync();  // nobody's shared memory goes away while another CTA reads it
}

}  // namespace daser

// pages int32 [total_q][Hkv][n_pages]: for every query row and KV head the pages to read, ascending, -1 behind the last.
// scores: scratch of total_q * Hkv * stride floats, stride >= the pages of the longest context; only strides above 16384 need it.
DASER_API int daser_select_pages_kv4(const void* q, const int8_t* codes, const int8_t* exps, int layer, int num_blocks,
                                     const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                                     int num_seqs, int total_q, int max_q_len, int Hq, int Hkv, float* scores, int stride,
                                     int32_t* pages, int n_pages, int sink, int recent, cudaStream_t stream) {
  using namespace daser;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || layer < 0 || num_blocks <= 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (num_seqs < 0 || total_q < 0 || max_q_len < 0 || stride < 1) return DASER_ERR_BAD_ARG;
  if (n_pages < 1 || sink < 0 || recent < 1 || (int64_t)sink + recent > n_pages) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return 0;
  if (!q || !codes || !exps || !block_tables || !q_start || !ctx_lens || !pages) return DASER_ERR_BAD_ARG;
  if (Hq / Hkv > 16 || (uintptr_t)codes % 16) return DASER_ERR_UNSUPPORTED;
  // Rows by (sequence, offset) while that many exist, as in a decode step, else by a search in q_start (one more dependent load): 32
  // sequences of one token beside a chunk of 2048 are 2080 rows, not 33 * 2048.
  const int64_t all = (int64_t)num_seqs * max_q_len, rows = all < total_q ? all : total_q;
  if (max_q_len > 65535 || max_blocks > (1 << 29) / DASER_KV4_TOKENS) return DASER_ERR_TOO_LARGE;
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
  p.num_seqs = num_seqs;
  p.by_row = all > total_q;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.max_q_len = max_q_len;
  p.total_q = total_q;
  p.stride = stride;
  p.n_pages = n_pages;
  p.sink = sink;
  p.recent = recent;
  // A batch a CTA at least, and no more CTAs than run at once (two an SM).
  int cluster = 1;
  while (cluster < SELECT_CLUSTER && cluster * SELECT_BATCH < stride && rows * Hkv * cluster * 2 <= 2 * 148) cluster *= 2;
  p.cluster = cluster;
  const int share = (stride + cluster - 1) / cluster;
  p.keys = share <= SELECT_KEYS ? share : 0;
  if (p.keys == 0 && !scores) return DASER_ERR_BAD_ARG;
  if (rows * Hkv > 0x7fffffff / cluster) return DASER_ERR_TOO_LARGE;
  static bool configured[DASER_MAX_DEVICES] = {false};  // per device: the attribute is the device's
  if (daser_first_use_on_device(configured)) {
    cudaError_t e = cudaFuncSetAttribute(attn4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SELECT_KEYS * 4);
    if (e != cudaSuccess) return (int)e;
    daser_used_on_device(configured);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * Hkv * cluster));
  cfg.blockDim = dim3(SELECT_THREADS);
  cfg.dynamicSmemBytes = (size_t)p.keys * 4;
  cfg.stream = stream;
  // (Not brought in ahead of its predecessor's end: clusters that wait on the SMs cost more than the launch they hide, 66 us
  // against 50 for a step of 16 sequences of 16k - 64k tokens.)
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, attn4_select_kernel, p);
}
