// What fills the 4-bit paged pool and reads it back: RoPE + cache write of a step, read by slot, restore of
// stored chunk images, save into chunk images, and the key bounds of pages.
//
// The reference has no cache codec (it copies whatever bytes its engine's pool holds,
// daser/connector/daser_connector.py:537-551,625-632); the fp8 counterparts are kv_paged.cu and rope.cuh.
#include "fp4.cuh"

namespace daser {

#define KV4_ERR_BLOCK_RANGE 2u
#define KV4_ERR_DELTA_RANGE 3u
#define KV4_ERR_NULL_SLOT 4u  // or an image off the 16-byte grid

__device__ __forceinline__ void kv4_report(uint32_t* status, uint32_t code, uint32_t slot) {
  if (status != nullptr && atomicCAS(status, 0u, code) == 0u) status[1] = slot;
}

// Eight values as they lie in memory, and as pairs of floats.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  ulonglong2 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const ulonglong2*>(p)[0];
    b = reinterpret_cast<const ulonglong2*>(p)[1];
  }
  __device__ __forceinline__ void pairs(uint64_t (&x)[4]) const { x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; }
  static __device__ __forceinline__ void zero(float* p) {
    reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(0ull, 0ull);
    reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(0ull, 0ull);
  }
};
template <> struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void pairs(uint64_t (&x)[4]) const {
    x[0] = pair2(bf16_lo(a.x), bf16_hi(a.x));
    x[1] = pair2(bf16_lo(a.y), bf16_hi(a.y));
    x[2] = pair2(bf16_lo(a.z), bf16_hi(a.z));
    x[3] = pair2(bf16_lo(a.w), bf16_hi(a.w));
  }
  static __device__ __forceinline__ void zero(__nv_bfloat16* p) { *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u); }
};
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ uint32_t bf16_pair(uint64_t v) {
  float a, b;
  unpair2(v, a, b);
  return pack_bf16x2(a, b);
}
__device__ __forceinline__ uint4 pack8(const uint64_t (&x)[4]) {
  return make_uint4(bf16_pair(x[0]), bf16_pair(x[1]), bf16_pair(x[2]), bf16_pair(x[3]));
}
__device__ __forceinline__ void load_pairs4(const float* p, uint64_t (&x)[4]) {
  const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(p), b = *reinterpret_cast<const ulonglong2*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

// ---- RoPE + cache write of a step -----------------------------------------------------------------------------
//
// y = rot(x): y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin over dims (i, i + 64); queries leave as bf16, keys (rotated) and
// values (as they are) are rounded to bf16, what a bf16 cache would hold, and then to the 4-bit format.
// Bound by bytes: the projections in, the queries out, 72 B a row into the pool.  A thread takes 8 dims and their rotary
// partners, so that a warp's access is four runs of 128 contiguous bytes and the two halves of a scale group sit
// on neighbouring lanes (one shuffle joins their maxima); it keeps the token's cosines in registers for all its heads.
// 4096 tokens of 32 / 8 heads, bf16, 88 MB: 17.2 us, 5.1 TB/s (18.4 with every trip's values read in the trip itself), 19 with the
// per-head norm (72 registers, 4 bytes spilled); 64 tokens of 64 / 8 heads, fp32: 4 us, a launch and three dependent misses.
template <typename TIn, bool QKNORM>
__global__ void __launch_bounds__(128)
kv4_write_kernel(TIn* __restrict__ qkv, int64_t qkv_stride, const int32_t* __restrict__ positions,
                 const int64_t* __restrict__ slot_mapping, const float* __restrict__ cos_sin, int max_pos,
                 __nv_bfloat16* __restrict__ q_out, int Hq, int Hkv, uint8_t* __restrict__ pool, int64_t stride_block,
                 int64_t stride_head, int num_blocks, int zero_after, const __nv_bfloat16* __restrict__ q_norm_w,
                 const __nv_bfloat16* __restrict__ k_norm_w, float norm_eps) {
  constexpr int D = DASER_KV4_DIM;
  pdl_enter();
  const int t = blockIdx.x;
  const int c = threadIdx.x & 7;  // dims [8c, 8c + 8) and [64 + 8c, 64 + 8c + 8)
  const int heads = Hq + 2 * Hkv;
  int pos = positions[t];
  pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);
  const int64_t slot = slot_mapping[t];
  const int64_t block = slot / DASER_KV4_TOKENS;
  const int tok = (int)(slot % DASER_KV4_TOKENS);
  const bool live = slot >= 0 && block < num_blocks;
  uint64_t cs[4], sn[4];
  load_pairs4(cos_sin + (int64_t)pos * D + 8 * c, cs);
  load_pairs4(cos_sin + (int64_t)pos * D + 64 + 8 * c, sn);
  TIn* row = qkv + (int64_t)t * qkv_stride;
  // every lane of a warp runs the same trips (the shuffles below are warp-wide): heads beyond the last are clamped.  A trip's values
  // are read during the trip before it.
  Raw8<TIn> ra, rb;
  auto read = [&](int h0) {
    const TIn* src = row + (int64_t)min(h0 + (int)(threadIdx.x >> 3), heads - 1) * D + 8 * c;
    ra.load(src);
    rb.load(src + 64);
  };
  read(blockIdx.y * 16);
  for (int h0 = blockIdx.y * 16; h0 < heads; h0 += gridDim.y * 16) {
    const int hd_raw = h0 + (threadIdx.x >> 3);
    const bool in = hd_raw < heads;
    const int hd = in ? hd_raw : heads - 1;
    const bool is_q = hd < Hq, is_v = hd >= Hq + Hkv;
    uint64_t a[4], b[4];
    ra.pairs(a);
    rb.pairs(b);
    const int h1 = h0 + gridDim.y * 16;
    if (h1 < heads) read(h1);
    if (in && zero_after != 0) {  // (what a clamped lane reads is not used)
      Raw8<TIn>::zero(row + (int64_t)hd * D + 8 * c);
      Raw8<TIn>::zero(row + (int64_t)hd * D + 64 + 8 * c);
    }
    if (QKNORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0, x1, y0, y1;
        unpair2(a[i], x0, x1);
        unpair2(b[i], y0, y1);
        ss += x0 * x0 + y0 * y0 + (x1 * x1 + y1 * y1);
      }
#pragma unroll
      for (int m = 4; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
      if (!is_v) {
        const float inv = rsqrtf(ss / (float)D + norm_eps);
        const __nv_bfloat16* w = (is_q ? q_norm_w : k_norm_w) + 8 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // the normalised head is a bf16 tensor in the models this follows: round before rotating
          const uint64_t wa = pair2(__bfloat162float(w[2 * i]), __bfloat162float(w[2 * i + 1]));
          const uint64_t wb = pair2(__bfloat162float(w[64 + 2 * i]), __bfloat162float(w[64 + 2 * i + 1]));
          const uint32_t ra = bf16_pair(mul2(mul2(a[i], pair2(inv, inv)), wa)), rb = bf16_pair(mul2(mul2(b[i], pair2(inv, inv)), wb));
          a[i] = pair2(bf16_lo(ra), bf16_hi(ra));
          b[i] = pair2(bf16_lo(rb), bf16_hi(rb));
        }
      }
    }
    if (!is_v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) rotate2(a[i], b[i], cs[i], sn[i]);
    }
    if (in && is_q) {
      __nv_bfloat16* dst = q_out + ((int64_t)t * Hq + hd) * D + 8 * c;
      *reinterpret_cast<uint4*>(dst) = pack8(a);
      *reinterpret_cast<uint4*>(dst + 64) = pack8(b);
    }
    if (h0 + 16 > Hq) {  // some lane of the block holds a key or value head: uniform over the block
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t ra = bf16_pair(a[i]), rb = bf16_pair(b[i]);
        a[i] = pair2(bf16_lo(ra), bf16_hi(ra));
        b[i] = pair2(bf16_lo(rb), bf16_hi(rb));
      }
      float ma = fp4_absmax<4>(a), mb = fp4_absmax<4>(b);
      ma = max3_nan(ma, __shfl_xor_sync(0xffffffffu, ma, 1), 0.f);
      mb = max3_nan(mb, __shfl_xor_sync(0xffffffffu, mb, 1), 0.f);
      const uint32_t sa = fp4_scale_byte(ma), sb = fp4_scale_byte(mb);
      uint32_t ca[1], cb[1];
      fp4_encode<4>(a, sa, fp4_inverse(sa), ca);
      fp4_encode<4>(b, sb, fp4_inverse(sb), cb);
      if (in && !is_q && live) {
        const int kv = is_v ? 1 : 0;
        uint8_t* rec = pool + block * stride_block + (int64_t)(hd - Hq - kv * Hkv) * stride_head;
        *reinterpret_cast<uint32_t*>(rec + kv4_code_at(kv, tok, c)) = ca[0];
        *reinterpret_cast<uint32_t*>(rec + kv4_code_at(kv, tok, 8 + c)) = cb[0];
        if ((c & 1) == 0) {
          rec[kv4_scale_at(kv, tok, c >> 1)] = (uint8_t)sa;
          rec[kv4_scale_at(kv, tok, 4 + (c >> 1))] = (uint8_t)sb;
        }
      }
    }
  }
}

// ---- read by slot ------------------------------------------------------------------------------------------------
//
// k, v [T][H][128] bf16 of the tokens that slot_mapping names, exact (e2m1 * scale has six significant bits); a slot below zero,
// or beyond the pool, reads as zeros.  A thread takes 8 dims: 4 bytes in, 16 out, 16 lanes a row.  Its floor is the 256 bytes written a
// row; 4096 tokens of 8 heads, 21 MB, take 7 us against 3.2: one item in flight a thread, behind the load of its slot.
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ pool, int64_t stride_block, int64_t stride_head, int num_blocks,
                const int64_t* __restrict__ slot_mapping, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v,
                int64_t items, int H) {
  pdl_enter();
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int p = (int)(it & 15);
    const int kv = (int)((it >> 4) & 1);
    const int64_t th = it >> 5;
    const int64_t t = th / H;
    const int h = (int)(th - t * H);
    const int64_t slot = slot_mapping[t];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int64_t block = slot / DASER_KV4_TOKENS;
    if (slot >= 0 && block < num_blocks) {
      const int tok = (int)(slot % DASER_KV4_TOKENS);
      const uint8_t* rec = pool + block * stride_block + h * stride_head;
      fp4_decode8(*reinterpret_cast<const uint32_t*>(rec + kv4_code_at(kv, tok, p)), rec[kv4_scale_at(kv, tok, p >> 1)], x);
    }
    *reinterpret_cast<uint4*>((kv ? v : k) + th * DASER_KV4_DIM + 8 * p) = pack8(x);
  }
}

// ---- chunk images -> pages ---------------------------------------------------------------------------------------
//
// One CTA per (slot, layer, up to KV4_HEADS heads).  An item is one scale group of a row and its rotary partner: dequantised,
// rotated by the slot's delta (keys), quantised, and put into the record's place in shared memory; whole records
// then leave as 16-byte stores.  Stored directly, the 8-byte pieces of V would each be a quarter of a 32-byte sector.
// 208 slots of 10 layers and 8 heads (85 MB in, 38 out) take 41 us from fp8 images, 47 from bf16 ones (136 MB in), where a copy of the
// bytes takes 19 and 27.  No unit is full (ALU 40 %, FMA 42, memory 45): a CTA makes its table, loads, computes and stores one after the
// other, three of them an SM (80 registers), and waits longest for its loads.  (57 us with a division per group in place of the table of
// reciprocals and without reading an item ahead.)  The pool's bases are indexed by rank, so each thread has the parameter in local
// memory (104 bytes), here and in the save.
constexpr int KV4_HEADS = 8;
constexpr int KV4_PITCH = DASER_KV4_RECORD + 32;  // of a record in shared memory: the rows of eight heads start in different banks

__device__ __forceinline__ void decode_fp8_group(const uint4& q, float scale, uint64_t (&x)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  const uint64_t s = pair2(scale, scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = e4m3x2_to_float2((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    x[i] = mul2(pair2(f.x, f.y), s);
  }
}
__device__ __forceinline__ void decode_bf16_group(const uint4& a, const uint4& b, uint64_t (&x)[8]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = pair2(bf16_lo(w[i]), bf16_hi(w[i]));
}

template <bool IMG_FP8>
__global__ void __launch_bounds__(256)
kv4_restore_kernel(const DaserKVJob job, const DaserKV4Pool pool) {
  constexpr int D = DASER_KV4_DIM, B = DASER_KV4_TOKENS;
  __shared__ __align__(16) float s_cs[D];
  __shared__ float s_inv[256];  // of every scale byte: a reciprocal, correctly rounded, takes more instructions than a group otherwise
  __shared__ __align__(16) uint8_t s_rec[KV4_HEADS * KV4_PITCH];
  const int H = job.num_kv_heads;
  const int slot = blockIdx.x / job.layer_count;
  const int layer = job.layer_begin + blockIdx.x % job.layer_count;
  const int head0 = blockIdx.y * KV4_HEADS, nh = min(KV4_HEADS, H - head0);
  const int block = job.block_id[slot];
  const uint64_t img = job.slot_ptr[slot];
  const int delta = job.delta ? job.delta[slot] : 0;
  const int64_t adelta = delta < 0 ? -(int64_t)delta : delta;
  uint32_t bad = 0;
  if (block < 0 || block >= pool.num_blocks) bad = KV4_ERR_BLOCK_RANGE;
  else if (img == 0 || img % 16 != 0) bad = KV4_ERR_NULL_SLOT;
  else if (delta != 0 && adelta >= job.max_pos) bad = KV4_ERR_DELTA_RANGE;
  if (bad) {
    if (threadIdx.x == 0) kv4_report(job.status, bad, slot);
    return;
  }
  s_inv[threadIdx.x] = fp4_inverse(threadIdx.x);
  if (delta != 0 && threadIdx.x < D) {
    const float v = job.cos_sin[adelta * D + threadIdx.x];
    s_cs[threadIdx.x] = (threadIdx.x >= D / 2 && delta < 0) ? -v : v;  // sin(-x) = -sin(x)
  }
  __syncthreads();
  const int64_t elems = (int64_t)2 * B * H * D;
  const int64_t layer_bytes = IMG_FP8 ? elems + elems / FP8_GROUP * 4 : 2 * elems;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(img) + (int64_t)layer * layer_bytes;
  const float* img_scales = reinterpret_cast<const float*>(base + elems);
  const int items = 2 * B * nh * 4;
  const int lg = (nh & (nh - 1)) == 0 ? __ffs(nh) - 1 : -1;
  // what an item reads, and its (kv * B + token, head), one item ahead of its use
  uint4 n1, n2, n3, n4;
  float ns1 = 0.f, ns2 = 0.f;
  int n_rr = 0, n_hl = 0;
  auto load = [&](int item) {
    const int r = item >> 2;
    n_rr = lg >= 0 ? r >> lg : r / nh;
    n_hl = r - n_rr * nh;
    const int e1 = (n_rr * H + head0 + n_hl) * D + (item & 3) * FP8_GROUP, e2 = e1 + D / 2;  // (a layer of a slot: far below 2^31)
    if (IMG_FP8) {
      n1 = *reinterpret_cast<const uint4*>(base + e1);
      n2 = *reinterpret_cast<const uint4*>(base + e2);
      ns1 = img_scales[e1 / FP8_GROUP];
      ns2 = img_scales[e2 / FP8_GROUP];
    } else {
      const uint4* h1 = reinterpret_cast<const uint4*>(base + 2 * e1);
      const uint4* h2 = reinterpret_cast<const uint4*>(base + 2 * e2);
      n1 = h1[0];
      n2 = h2[0];
      n3 = h1[1];
      n4 = h2[1];
    }
  };
  const int j = threadIdx.x & 3;
  if (threadIdx.x < items) load(threadIdx.x);
  for (int item = threadIdx.x; item < items; item += 256) {
    const int hl = n_hl, tok = n_rr & (B - 1), kv = n_rr / B;
    uint64_t x1[8], x2[8];
    if (IMG_FP8) {
      decode_fp8_group(n1, ns1, x1);
      decode_fp8_group(n2, ns2, x2);
    } else {
      decode_bf16_group(n1, n3, x1);
      decode_bf16_group(n2, n4, x2);
    }
    if (item + 256 < items) load(item + 256);
    if (kv == 0 && delta != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&s_cs[j * FP8_GROUP + 4 * i]);
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&s_cs[D / 2 + j * FP8_GROUP + 4 * i]);
        rotate2(x1[2 * i], x2[2 * i], c.x, s.x);
        rotate2(x1[2 * i + 1], x2[2 * i + 1], c.y, s.y);
      }
    }
    uint8_t* rec = s_rec + hl * KV4_PITCH;
    uint32_t codes[2];
    const uint32_t s1 = fp4_scale_byte(fp4_absmax<8>(x1)), s2 = fp4_scale_byte(fp4_absmax<8>(x2));
    fp4_encode<8>(x1, s1, s_inv[s1], codes);
    *reinterpret_cast<uint2*>(rec + kv4_code_at(kv, tok, 2 * j)) = make_uint2(codes[0], codes[1]);
    fp4_encode<8>(x2, s2, s_inv[s2], codes);
    *reinterpret_cast<uint2*>(rec + kv4_code_at(kv, tok, 8 + 2 * j)) = make_uint2(codes[0], codes[1]);
    rec[kv4_scale_at(kv, tok, j)] = (uint8_t)s1;
    rec[kv4_scale_at(kv, tok, 4 + j)] = (uint8_t)s2;
  }
  __syncthreads();
  // a warp a head; with more ranks than KV heads a head is kept by `replicas` ranks
  const bool wide = pool.n_ranks > H;
  const int replicas = wide ? pool.n_ranks / H : 1;
  constexpr int VECS = DASER_KV4_RECORD / 16;
  const int hl = threadIdx.x >> 5, head = head0 + hl;
  if (hl >= nh) return;
  const int rank0 = wide ? head * replicas : head / pool.heads_per_rank;
  const int64_t off = (int64_t)layer * pool.stride_layer + (int64_t)block * pool.stride_block +
                      (int64_t)(wide ? 0 : head - rank0 * pool.heads_per_rank) * pool.stride_head;
  const uint4* src = reinterpret_cast<const uint4*>(s_rec + hl * KV4_PITCH);
  for (int rep = 0; rep < replicas; ++rep) {
    uint4* dst = reinterpret_cast<uint4*>(pool.records[rank0 + rep] + off);
#pragma unroll
    for (int i = threadIdx.x & 31; i < VECS; i += 32) dst[i] = src[i];
  }
}

// ---- pages -> chunk images ---------------------------------------------------------------------------------------
//
// The mirror image: records in as 16-byte loads, rows out.  A raw image gets the values as they stand (exact in bf16), an fp8b16
// image is quantised again (group maximum 448: relative error at most 2^-4).  208 slots of 10 layers and 8 heads: into raw images (38 MB
// in, 136 out) 36 us, 4.9 TB/s; into fp8b16 ones (85 out), which is what an engine stores, 37 us, 3.3 TB/s.  The phases of a CTA, records in,
// barrier, rows out, do not overlap; the largest stall is on its loads.
template <bool IMG_FP8>
__global__ void __launch_bounds__(256)
kv4_save_kernel(const DaserKVJob job, const DaserKV4Pool pool) {
  constexpr int D = DASER_KV4_DIM, B = DASER_KV4_TOKENS;
  __shared__ __align__(16) uint8_t s_rec[KV4_HEADS * KV4_PITCH];
  const int H = job.num_kv_heads;
  const int slot = blockIdx.x / job.num_layers, layer = blockIdx.x % job.num_layers;
  const int block = job.block_id[slot];
  const uint64_t img = job.slot_ptr[slot];
  if (block < 0 || block >= pool.num_blocks || img == 0 || img % 16 != 0) {
    if (threadIdx.x == 0) kv4_report(job.status, block >= 0 && block < pool.num_blocks ? KV4_ERR_NULL_SLOT : KV4_ERR_BLOCK_RANGE, slot);
    return;
  }
  int first, owned;  // heads of this rank inside the all-head image
  if (pool.n_ranks > H) {
    const int replicas = pool.n_ranks / H;
    if (job.rank % replicas) return;  // only the first replica of a head writes it
    first = job.rank / replicas;
    owned = 1;
  } else {
    first = job.rank * pool.heads_per_rank;
    owned = pool.heads_per_rank;
  }
  const int l0 = blockIdx.y * KV4_HEADS, nh = min(KV4_HEADS, owned - l0);
  if (nh <= 0) return;
  constexpr int VECS = DASER_KV4_RECORD / 16;
  if (const int hl = threadIdx.x >> 5; hl < nh) {  // a warp a head
    const uint4* src = reinterpret_cast<const uint4*>(pool.records[job.rank] + (int64_t)layer * pool.stride_layer +
                                                      (int64_t)block * pool.stride_block + (int64_t)(l0 + hl) * pool.stride_head);
    uint4* dst = reinterpret_cast<uint4*>(s_rec + hl * KV4_PITCH);
#pragma unroll
    for (int i = threadIdx.x & 31; i < VECS; i += 32) dst[i] = src[i];
  }
  __syncthreads();
  const int64_t elems = (int64_t)2 * B * H * D;
  const int64_t layer_bytes = IMG_FP8 ? elems + elems / FP8_GROUP * 4 : 2 * elems;
  uint8_t* base = reinterpret_cast<uint8_t*>(img) + (int64_t)layer * layer_bytes;
  float* img_scales = reinterpret_cast<float*>(base + elems);
  constexpr int PIECES = IMG_FP8 ? 8 : 16;  // of a row: a scale group, or 16 bytes of bf16
  const int lg = (nh & (nh - 1)) == 0 ? __ffs(nh) - 1 : -1;
  for (int item = threadIdx.x; item < 2 * B * nh * PIECES; item += 256) {
    const int p = item % PIECES;
    const int r = item / PIECES;
    const int rr = lg >= 0 ? r >> lg : r / nh;  // kv * B + token
    const int hl = r - rr * nh;
    const int tok = rr & (B - 1), kv = rr / B;
    const uint8_t* rec = s_rec + hl * KV4_PITCH;
    const int row = rr * H + first + l0 + hl;  // (a layer of a slot: far below 2^31)
    if (IMG_FP8) {
      float x[16];
      const uint2 w = *reinterpret_cast<const uint2*>(rec + kv4_code_at(kv, tok, 2 * p));
      const uint32_t s = rec[kv4_scale_at(kv, tok, p)];
      fp4_decode8(w.x, s, x);
      fp4_decode8(w.y, s, x + 8);
      uint4 q;
      float sc;
      quant_group16(x, q, sc);
      *reinterpret_cast<uint4*>(base + row * D + p * FP8_GROUP) = q;
      img_scales[row * (D / FP8_GROUP) + p] = sc;
    } else {
      float x[8];
      fp4_decode8(*reinterpret_cast<const uint32_t*>(rec + kv4_code_at(kv, tok, p)), rec[kv4_scale_at(kv, tok, p >> 1)], x);
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(base) + row * D + 8 * p) = pack8(x);
    }
  }
}

// ---- key bounds of pages -----------------------------------------------------------------------------------------
//
// hi_d = max, lo_d = min over the page's keys, held as int8 codes times one power of two, rounded outwards (hi up, lo down), so that
// sum_d max(q_d hi_d, q_d lo_d) bounds every score of the page from above.  One warp per (page, head).
// Recomputed from the whole page, so that the result depends on the page alone; only tokens below ctx count (what lies behind
// them in a page is left over from its last owner).  A page with a key that is not finite gets exponent 127.  A decode step touches one
// page per sequence: 6 to 8 us, of which a launch is 2 and the chain of lengths, table, record about 3; the rest has not been looked into.
__device__ __forceinline__ int pow2_exponent(float a) {
  // the smallest e with a <= 127 * 2^e, for a > 0: a = m * 2^x, m in [1/2, 1), gives e = x - 7, one more if m * 128 > 127
  const int x = (int)(__float_as_uint(a) >> 23) - 126;
  return x - 7 + ((__float_as_uint(a) & 0x7fffffu) > 63u * (1u << 17) ? 1 : 0);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

__global__ void __launch_bounds__(128)
kv4_page_bounds_kernel(const uint8_t* __restrict__ pool, int64_t stride_block, int64_t stride_head, int num_blocks,
                       int8_t* __restrict__ codes, int8_t* __restrict__ exps, const int32_t* __restrict__ block_tables,
                       int max_blocks, const int32_t* __restrict__ q_start, const int32_t* __restrict__ ctx_lens, int H) {
  pdl_enter();
  const int seq = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_len = q_start[seq + 1] - q_start[seq], ctx = ctx_lens[seq];
  if (q_len <= 0 || ctx <= 0) return;
  const int first = max(ctx - q_len, 0) / DASER_KV4_TOKENS, last = (ctx - 1) / DASER_KV4_TOKENS;
  const int idx = blockIdx.x * 4 + warp;
  const int page = first + idx / H, head = idx % H;
  if (page > last || page >= max_blocks) return;
  const int blk = block_tables[(int64_t)seq * max_blocks + page];
  if (blk < 0 || blk >= num_blocks) return;
  const uint8_t* rec = pool + (int64_t)blk * stride_block + (int64_t)head * stride_head;
  const int live = min(DASER_KV4_TOKENS, ctx - page * DASER_KV4_TOKENS);
  // a lane owns 8 dims; the half-warps take alternate tokens
  const int p = lane & 15;
  float hi[8], lo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { hi[i] = -INFINITY; lo[i] = INFINITY; }
  bool bad = false;
#pragma unroll
  for (int it = 0; it < DASER_KV4_TOKENS / 2; ++it) {
    const int tok = 2 * it + (lane >> 4);
    if (tok < live) {
      const uint32_t sb = rec[kv4_scale_at(0, tok, p >> 1)];
      float x[8];
      fp4_decode8(*reinterpret_cast<const uint32_t*>(rec + kv4_code_at(0, tok, p)), sb, x);
      bad |= sb >= 0xf8u;
#pragma unroll
      for (int i = 0; i < 8; ++i) { hi[i] = fmaxf(hi[i], x[i]); lo[i] = fminf(lo[i], x[i]); }
    }
  }
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], 16));
    lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], 16));
    a = fmaxf(a, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
  }
  a = warp_max(a);
  bad = __any_sync(0xffffffffu, bad);
  const int e = bad ? 127 : (a > 0.f ? pow2_exponent(a) : -100);
  const float up = bad ? 0.f : pow2f(-e);
  // half-warp 0 writes the high codes, half-warp 1 the low ones
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // a product with a power of two: exact
    const int c = lane < 16 ? (bad ? 127 : __float2int_ru(hi[i] * up)) : (bad ? -127 : __float2int_rd(lo[i] * up));
    w[i >> 2] |= ((uint32_t)c & 0xffu) << (8 * (i & 3));
  }
  const int64_t at = (int64_t)blk * H + head;
  *reinterpret_cast<uint2*>(codes + at * 256 + (lane >> 4) * 128 + 8 * p) = make_uint2(w[0], w[1]);
  if (lane == 0) exps[at] = (int8_t)e;
}

// The bounds of listed blocks as floats [n][H][2][128]; a block outside the pool reads as zeros.
__global__ void __launch_bounds__(256)
kv4_bounds_read_kernel(const int8_t* __restrict__ codes, const int8_t* __restrict__ exps, const int32_t* __restrict__ blocks,
                       float* __restrict__ out, int64_t items, int num_blocks, int H) {
  pdl_enter();
  for (int64_t it = blockIdx.x * (int64_t)256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
    const int64_t nh = it >> 6;  // 64 pieces of four values a head
    const int64_t n = nh / H;
    const int blk = blocks[n];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (blk >= 0 && blk < num_blocks) {
      const int64_t at = (int64_t)blk * H + (nh - n * H);
      const char4 c = *reinterpret_cast<const char4*>(codes + at * 256 + (it & 63) * 4);
      const int e = exps[at];
      const float f = e == 127 ? INFINITY : pow2f(max(e, -126));
      v = make_float4(c.x * f, c.y * f, c.z * f, c.w * f);
    }
    *reinterpret_cast<float4*>(out + it * 4) = v;
  }
}

// ---- the codec on its own ----------------------------------------------------------------------------------------
//
// A thread takes a group.  67 million values: 30 us to codes (172 MB, 5.8 TB/s), 41 us back (4.2 TB/s; a thread's 32 bytes
// leave as two 16-byte stores).
__global__ void __launch_bounds__(256)
quant_fp4b16_kernel(const __nv_bfloat16* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int64_t groups) {
  for (int64_t g = blockIdx.x * (int64_t)256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
    uint64_t v[8];
    const uint4* src = reinterpret_cast<const uint4*>(x + g * 16);
    decode_bf16_group(src[0], src[1], v);
    const uint32_t s = fp4_scale_byte(fp4_absmax<8>(v));
    uint32_t c[2];
    fp4_encode<8>(v, s, fp4_inverse(s), c);
    *reinterpret_cast<uint2*>(codes + g * 8) = make_uint2(c[0], c[1]);
    scales[g] = (uint8_t)s;
  }
}
__global__ void __launch_bounds__(256)
dequant_fp4b16_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, __nv_bfloat16* __restrict__ y, int64_t groups) {
  for (int64_t g = blockIdx.x * (int64_t)256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + g * 8);
    float v[16];
    fp4_decode8(c.x, scales[g], v);
    fp4_decode8(c.y, scales[g], v + 8);
    store_bf16x16(y + g * 16, v);
  }
}

static int kv4_check_job(const DaserKVJob& j, const DaserKV4Pool& p) {
  if (j.n_slots < 0 || j.num_layers <= 0 || j.num_layers > p.num_layers || j.num_kv_heads <= 0) return DASER_ERR_BAD_ARG;
  if (j.head_dim != DASER_KV4_DIM || j.block_tokens != DASER_KV4_TOKENS) return DASER_ERR_UNSUPPORTED;
  if (p.n_ranks <= j.num_kv_heads) {
    if (j.num_kv_heads % p.n_ranks || p.heads_per_rank != j.num_kv_heads / p.n_ranks) return DASER_ERR_BAD_ARG;
  } else if (p.n_ranks % j.num_kv_heads || p.heads_per_rank != 1) {
    return DASER_ERR_BAD_ARG;
  }
  for (int r = 0; r < p.n_ranks; ++r)
    if (int e = kv4_check_pool(&p, 0, r)) return e;
  return 0;
}

}  // namespace daser

// q, k of qkv [T][(Hq + 2 Hkv) * 128] rotated; q -> q_out (bf16), k and v -> the pool at slot_mapping (negative: not written).
// q_norm_w / k_norm_w (bf16 [128], both or neither): RMSNorm over the head before the rotation.
DASER_API int daser_rope_kv4_write(void* qkv, int qkv_is_fp32, int64_t qkv_stride, const int32_t* positions,
                                   const int64_t* slot_mapping, const float* cos_sin, int max_pos, void* q_out, int T, int Hq,
                                   int Hkv, const DaserKV4Pool* pool, int layer, int rank, int zero_after,
                                   const void* q_norm_w, const void* k_norm_w, float eps, cudaStream_t stream) {
  using namespace daser;
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  if (T < 0 || Hq < 0 || Hkv <= 0 || Hkv > pool->heads_per_rank || max_pos <= 0 || (!q_norm_w) != (!k_norm_w)) return DASER_ERR_BAD_ARG;
  if (T == 0) return 0;
  if (!qkv || !positions || !slot_mapping || !cos_sin || (Hq > 0 && !q_out)) return DASER_ERR_BAD_ARG;
  if (qkv_stride % (qkv_is_fp32 ? 4 : 8) || (uintptr_t)qkv % 16 || (uintptr_t)q_out % 16 || (uintptr_t)cos_sin % 16) return DASER_ERR_UNSUPPORTED;
  // one pass over the heads per block while there are few tokens, all heads in one block (cosines read once) beyond: 4096 tokens of
  // 48 heads 17 us against 22
  const int parts = (Hq + 2 * Hkv + 15) / 16;
  const dim3 grid((unsigned)T, (unsigned)(T >= 592 ? 1 : parts));
  uint8_t* base = pool->records[rank] + (int64_t)layer * pool->stride_layer;
  cudaError_t e;
#define LAUNCH4(TIN, N)                                                                                              \
  e = launch_pdl(kv4_write_kernel<TIN, N>, grid, dim3(128), 0, stream, (TIN*)qkv, qkv_stride, positions, slot_mapping, cos_sin, \
             max_pos, (__nv_bfloat16*)q_out, Hq, Hkv, base, pool->stride_block, pool->stride_head, pool->num_blocks, \
             zero_after, (const __nv_bfloat16*)q_norm_w, (const __nv_bfloat16*)k_norm_w, eps)
  if (qkv_is_fp32) { if (q_norm_w) LAUNCH4(float, true); else LAUNCH4(float, false); }
  else { if (q_norm_w) LAUNCH4(__nv_bfloat16, true); else LAUNCH4(__nv_bfloat16, false); }
#undef LAUNCH4
  return (int)e;
}

DASER_API int daser_kv4_read(const DaserKV4Pool* pool, int layer, int rank, const int64_t* slot_mapping, void* k, void* v, int T,
                             cudaStream_t stream) {
  using namespace daser;
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  if (T < 0) return DASER_ERR_BAD_ARG;
  if (T == 0) return 0;
  if (!slot_mapping || !k || !v) return DASER_ERR_BAD_ARG;
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16) return DASER_ERR_UNSUPPORTED;
  const int64_t items = (int64_t)T * pool->heads_per_rank * 32;
  const int64_t blocks = (items + 255) / 256;
  return (int)launch_pdl(kv4_read_kernel, dim3((unsigned)(blocks < 148 * 16 ? blocks : 148 * 16)), dim3(256), 0, stream,
                         (const uint8_t*)pool->records[rank] + (int64_t)layer * pool->stride_layer, pool->stride_block,
                         pool->stride_head, pool->num_blocks, slot_mapping, (__nv_bfloat16*)k, (__nv_bfloat16*)v, items,
                         pool->heads_per_rank);
}

DASER_API int daser_kv4_restore(const DaserKVJob* job, const DaserKV4Pool* pool, cudaStream_t stream) {
  using namespace daser;
  if (!job || !pool) return DASER_ERR_BAD_ARG;
  if (int e = kv4_check_job(*job, *pool)) return e;
  if (job->n_slots == 0) return 0;
  if (!job->slot_ptr || !job->block_id || (job->delta && (!job->cos_sin || job->max_pos <= 0))) return DASER_ERR_BAD_ARG;
  if (job->layer_begin < 0 || job->layer_count < 0 || (int64_t)job->layer_begin + job->layer_count > job->num_layers) return DASER_ERR_BAD_ARG;
  DaserKVJob j = *job;
  j.layer_count = job->layer_count > 0 ? job->layer_count : job->num_layers - job->layer_begin;
  if (j.layer_count <= 0) return 0;
  if ((int64_t)j.n_slots * j.layer_count > 0x7fffffff) return DASER_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(j.n_slots * j.layer_count), (unsigned)((j.num_kv_heads + KV4_HEADS - 1) / KV4_HEADS));
  if (j.image_is_fp8) kv4_restore_kernel<true><<<grid, 256, 0, stream>>>(j, *pool);
  else kv4_restore_kernel<false><<<grid, 256, 0, stream>>>(j, *pool);
  return (int)cudaGetLastError();
}

DASER_API int daser_kv4_save(const DaserKVJob* job, const DaserKV4Pool* pool, cudaStream_t stream) {
  using namespace daser;
  if (!job || !pool) return DASER_ERR_BAD_ARG;
  if (int e = kv4_check_job(*job, *pool)) return e;
  if (job->rank < 0 || job->rank >= pool->n_ranks) return DASER_ERR_BAD_ARG;
  if (job->n_slots == 0) return 0;
  if (!job->slot_ptr || !job->block_id) return DASER_ERR_BAD_ARG;
  if ((int64_t)job->n_slots * job->num_layers > 0x7fffffff) return DASER_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(job->n_slots * job->num_layers), (unsigned)((pool->heads_per_rank + KV4_HEADS - 1) / KV4_HEADS));
  if (job->image_is_fp8) kv4_save_kernel<true><<<grid, 256, 0, stream>>>(*job, *pool);
  else kv4_save_kernel<false><<<grid, 256, 0, stream>>>(*job, *pool);
  return (int)cudaGetLastError();
}

// Bounds of the pages that hold the last q_start[s + 1] - q_start[s] keys of every sequence.  codes int8 [layers][blocks][heads][2][128]
// (high, low), exps int8 [layers][blocks][heads].  max_q_len: no sequence has more new tokens.
DASER_API int daser_kv4_page_bounds(const DaserKV4Pool* pool, int layer, int rank, int8_t* codes, int8_t* exps,
                                    const int32_t* block_tables, int max_blocks, const int32_t* q_start, const int32_t* ctx_lens,
                                    int num_seqs, int max_q_len, cudaStream_t stream) {
  using namespace daser;
  if (int e = kv4_check_pool(pool, layer, rank)) return e;
  if (num_seqs < 0 || max_q_len < 0 || max_blocks <= 0) return DASER_ERR_BAD_ARG;
  if (num_seqs == 0 || max_q_len == 0) return 0;
  if (!codes || !exps || !block_tables || !q_start || !ctx_lens) return DASER_ERR_BAD_ARG;
  if ((uintptr_t)codes % 8 || num_seqs > 65535) return DASER_ERR_UNSUPPORTED;
  const int64_t H = pool->heads_per_rank;
  // max_q_len tokens lie in at most (max_q_len + 14) / 16 + 1 pages
  const int64_t warps = ((max_q_len + 14) / DASER_KV4_TOKENS + 1) * H;
  const int64_t rows = (int64_t)layer * pool->num_blocks * H;
  return (int)launch_pdl(kv4_page_bounds_kernel, dim3((unsigned)((warps + 3) / 4), (unsigned)num_seqs), dim3(128), 0, stream,
                         (const uint8_t*)pool->records[rank] + (int64_t)layer * pool->stride_layer, pool->stride_block,
                         pool->stride_head, pool->num_blocks, codes + rows * 256, exps + rows, block_tables, max_blocks, q_start,
                         ctx_lens, (int)H);
}

// Bounds of `n` listed blocks as floats [n][heads][2][128].
DASER_API int daser_kv4_bounds_read(const int8_t* codes, const int8_t* exps, int layer, int num_blocks, int heads, const int32_t* blocks,
                                    float* out, int n, cudaStream_t stream) {
  using namespace daser;
  if (layer < 0 || num_blocks <= 0 || heads <= 0 || n < 0) return DASER_ERR_BAD_ARG;
  if (n == 0) return 0;
  if (!codes || !exps || !blocks || !out) return DASER_ERR_BAD_ARG;
  if ((uintptr_t)codes % 4 || (uintptr_t)out % 16) return DASER_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)layer * num_blocks * heads, items = (int64_t)n * heads * 64, grid = (items + 255) / 256;
  return (int)launch_pdl(kv4_bounds_read_kernel, dim3((unsigned)(grid < 148 * 8 ? grid : 148 * 8)), dim3(256), 0, stream, codes + rows * 256,
                         exps + rows, blocks, out, items, num_blocks, heads);
}

DASER_API int daser_quant_fp4b16(const void* x, void* codes, void* scales, int64_t n_elems, cudaStream_t stream) {
  if (n_elems < 0 || n_elems % 16) return DASER_ERR_BAD_ARG;
  if (n_elems == 0) return 0;
  if (!x || !codes || !scales) return DASER_ERR_BAD_ARG;
  if ((uintptr_t)x % 16 || (uintptr_t)codes % 8) return DASER_ERR_UNSUPPORTED;
  const int64_t g = n_elems / 16, blocks = (g + 255) / 256;
  daser::quant_fp4b16_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>((const __nv_bfloat16*)x, (uint8_t*)codes,
                                                                                            (uint8_t*)scales, g);
  return (int)cudaGetLastError();
}

DASER_API int daser_dequant_fp4b16(const void* codes, const void* scales, void* y, int64_t n_elems, cudaStream_t stream) {
  if (n_elems < 0 || n_elems % 16) return DASER_ERR_BAD_ARG;
  if (n_elems == 0) return 0;
  if (!codes || !scales || !y) return DASER_ERR_BAD_ARG;
  if ((uintptr_t)codes % 8 || (uintptr_t)y % 16) return DASER_ERR_UNSUPPORTED;
  const int64_t g = n_elems / 16, blocks = (g + 255) / 256;
  daser::dequant_fp4b16_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales,
                                                                                              (__nv_bfloat16*)y, g);
  return (int)cudaGetLastError();
}
