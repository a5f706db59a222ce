"""The operators of the 4-bit pool on the GPU against plain forms in 64 bits."""

import pytest
import torch

from daser_b200.kv import codec
from daser_b200.kv.layout import KVGeometry, tp_head_range
from daser_b200.position import inv_freq_table

pytestmark = pytest.mark.gpu

D, B = 128, 16
BF16_HALF, F16_HALF = 2.0**-8, 2.0**-11  # eps / 2


def _ops():
    from daser_b200.ops import attention, elementwise, kv_ops

    return attention, elementwise, kv_ops


# -- codec -------------------------------------------------------------------------------


def test_codec_matches_the_oracle_bit_for_bit():
    _, _, kv_ops = _ops()
    torch.manual_seed(0)
    x = torch.randn(777, 4, 128) * torch.exp(3 * torch.randn(777, 4, 1))
    x[0] = 0
    x[1, 0, 5] = float("inf")
    x[1, 1, 20] = float("nan")
    x[2, 0] = 1e-8
    x[2, 1] = 1e30
    # ties of every scale
    x[3:11, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 2) * torch.arange(8, 16)[:, None] / 8
    x = x.to(torch.bfloat16)
    codes, scales = kv_ops.quantize_fp4b16(x.cuda())
    want_c, want_s = codec.quantize_fp4b16(x)
    assert torch.equal(scales.cpu(), want_s)
    finite = (want_s < 248).repeat_interleave(8, -1)  # the codes of a group that is not finite are free
    assert torch.equal(codes.cpu()[finite], want_c[finite])
    y = kv_ops.dequantize_fp4b16(codes, scales).float().cpu()
    ref = codec.dequantize_fp4b16(want_c, want_s)
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    assert torch.equal(y[~torch.isnan(ref)], ref[~torch.isnan(ref)])


# -- write and read ----------------------------------------------------------------------


def _rope_ref(x, cs):
    """fp32, operation for operation what the kernel does."""
    c, s = cs[:, None, :64], cs[:, None, 64:]
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("T,hq,hkv,f32,pad", [(1, 8, 1, True, 0), (5, 64, 8, True, 2), (64, 32, 8, False, 0), (37, 10, 2, False, 36),
                                              (130, 3, 3, True, 1), (700, 16, 1, False, 9), (601, 40, 8, True, 0), (3, 0, 2, False, 0)])
def test_write_and_read_are_exact(T, hq, hkv, f32, pad):
    attention, ew, kv_ops = _ops()
    torch.manual_seed(T)
    blocks = -(-T // B) + 3
    cols = (hq + 2 * hkv) * D
    wide = torch.randn(T, cols + 64).to(torch.float32 if f32 else torch.bfloat16)  # rows with a stride
    qkv = wide.cuda()[:, :cols]
    pos = torch.randint(-3, 520, (T,), dtype=torch.int32)  # also outside the table: clamped
    slots = torch.randperm(blocks * B)[:T].to(torch.int64)
    slots[T - pad :] = -1
    if T > 4:
        slots[2] = blocks * B + 5  # beyond the pool: not written
    cos_sin = kv_ops.rope_table(512, inv_freq_table(D, 10000.0), "cuda")
    big = torch.full((2, blocks, hkv + 1, 2304), 0x5A, dtype=torch.uint8, device="cuda")
    pool = kv_ops.PagedKV4Pool.from_tensors([big[:, :, :hkv]])  # strides of a larger tensor
    q_out = torch.zeros(T, hq, D, dtype=torch.bfloat16, device="cuda")
    ew.rope_kv_write(qkv, pos.cuda(), slots.cuda(), cos_sin, q_out, hq, hkv, D, B, pool, 1, zero_after=f32)
    k, v = kv_ops.kv_read(pool, 1, slots.cuda())
    torch.cuda.synchronize()
    x = wide[:, :cols].float().reshape(T, -1, D)
    cs = cos_sin.cpu()[pos.long().clamp(0, 511)]
    assert torch.equal(q_out.cpu(), _rope_ref(x[:, :hq], cs).to(torch.bfloat16))
    ref = torch.cat([_rope_ref(x[:, hq : hq + hkv], cs), x[:, hq + hkv :]], 1).to(torch.bfloat16)
    ref = codec.dequantize_fp4b16(*codec.quantize_fp4b16(ref))
    live = (slots >= 0) & (slots < blocks * B)
    ref[~live] = 0
    assert torch.equal(k.float().cpu(), ref[:, :hkv]) and torch.equal(v.float().cpu(), ref[:, hkv:])
    rec = big.cpu()
    assert (rec[0] == 0x5A).all() and (rec[:, :, hkv] == 0x5A).all()  # another layer, a neighbouring head
    untouched = torch.ones(blocks * B, dtype=torch.bool)
    untouched[slots[live]] = False
    for s in untouched.nonzero().flatten().tolist()[:40]:
        assert (rec[1, s // B, 0, (s % B) * 64 : (s % B) * 64 + 64] == 0x5A).all()
    if f32:
        assert (qkv == 0).all()  # accumulators are handed back zeroed


def test_write_with_the_per_head_norm():
    """The sum of squares has no fixed order, so a value may land on the other side of a border: within one step of the format."""
    _, ew, kv_ops = _ops()
    torch.manual_seed(3)
    T, hq, hkv, eps = 33, 8, 2, 1e-6
    qkv = torch.randn(T, (hq + 2 * hkv) * D, device="cuda").to(torch.bfloat16)
    qw, kw = (1 + 0.1 * torch.randn(2, D, device="cuda")).to(torch.bfloat16)
    cos_sin = kv_ops.rope_table(64, inv_freq_table(D, 10000.0), "cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    slots = torch.arange(T, dtype=torch.int64, device="cuda")
    pool = kv_ops.PagedKV4Pool.zeros(1, 3, hkv, "cuda")
    q_out = torch.zeros(T, hq, D, dtype=torch.bfloat16, device="cuda")
    ew.rope_kv_write(qkv, pos, slots, cos_sin, q_out, hq, hkv, D, B, pool, 0, qk_norm=(qw, kw, eps))
    k, v = kv_ops.kv_read(pool, 0, slots)
    x = qkv.double().cpu().reshape(T, -1, D)
    cs = cos_sin.double().cpu()[:T]

    def normed(h, w):
        y = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
        return _rope_ref(y.to(torch.bfloat16).double(), cs)

    q_ref, k_ref = normed(x[:, :hq], qw), normed(x[:, hq : hq + hkv], kw)
    # y may round to the neighbouring bf16 (one step, 2 * half, of each of the two values that a rotation mixes), then one rounding
    size = torch.cat([normed_abs := q_ref.abs()[..., :64] + q_ref.abs()[..., 64:], normed_abs], -1)
    assert ((q_out.double().cpu() - q_ref).abs() <= BF16_HALF * q_ref.abs() + 4 * BF16_HALF * size + 1e-6).all()
    got = k.double().cpu()
    s = codec.fp4_scale_values(codec.quantize_fp4b16(k_ref.float())[1]).double().repeat_interleave(16, -1)
    # half a step of e2m1 (at most s), a neighbouring scale (2^-3 of a value up to 6 s), a moved value (2^-6 of 6 s)
    assert ((got - k_ref).abs() <= s * (1.0 + 0.75 + 0.1)).all()
    assert ((got - k_ref).norm() / k_ref.norm()).item() < 0.15  # rms of a uniform error of half a step, with margin
    assert torch.equal(v.float().cpu(), codec.dequantize_fp4b16(*codec.quantize_fp4b16(x[:, hq + hkv :].float())))


# -- restore and save --------------------------------------------------------------------


def _images(geo, n, seed):
    torch.manual_seed(seed)
    slots = []
    for _ in range(n):
        ks = [(torch.randn(B, geo.num_kv_heads, D) * 0.5).to(torch.bfloat16) for _ in range(geo.num_layers)]
        vs = [(torch.randn(B, geo.num_kv_heads, D) * 0.5).to(torch.bfloat16) for _ in range(geo.num_layers)]
        slots.append(codec.pack_slot(geo, ks, vs))
    return torch.stack(slots)


def _pools(kv_ops, geo, blocks, tp, heads=None):
    hn = tp_head_range(geo.num_kv_heads, tp, 0)[1]
    recs = [torch.zeros(geo.num_layers, blocks, hn, 2304, dtype=torch.uint8, device="cuda") for _ in range(tp)]
    return recs, kv_ops.PagedKV4Pool.from_tensors(recs)


@pytest.mark.parametrize("img", ["fp8b16", "raw"])
@pytest.mark.parametrize("H,tp", [(4, 1), (4, 2), (2, 4), (10, 1), (1, 1)])
def test_restore_is_exact_and_save_gives_it_back(img, H, tp):
    """Ranks are pools on one GPU, written by one kernel."""
    _, _, kv_ops = _ops()
    geo = KVGeometry(3, H, D, B, 2, img)
    inv = inv_freq_table(D, 10000.0)
    n, blocks = 5, 11
    images = _images(geo, n, H)
    staging = images.cuda()
    ids, deltas = [7, 0, 10, 3, 5], [0, 17, -5, 300, 1]
    work = kv_ops.KVWorkList(staging.data_ptr() + torch.arange(n, dtype=torch.int64, device="cuda") * geo.slot_size,
                             torch.tensor(ids, dtype=torch.int32, device="cuda"), torch.tensor(deltas, dtype=torch.int32, device="cuda"))
    recs, pool = _pools(kv_ops, geo, blocks, tp)
    table = kv_ops.rope_table(512, inv, "cuda")
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    # in two pieces of layers, as a pipelined restore makes them
    kv_ops.kv_restore(work, geo, pool, table, status, layer_begin=0, layer_count=2)
    kv_ops.kv_restore(work, geo, pool, table, status, layer_begin=2)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    t = table.cpu()
    want = torch.empty(n, geo.num_layers, 2, B, H, D)
    for i in range(n):
        for layer in range(geo.num_layers):
            k, v = codec.unpack_layer(geo, images[i][layer * geo.layer_size : (layer + 1) * geo.layer_size])
            if deltas[i]:
                cs = t[abs(deltas[i])].clone()
                if deltas[i] < 0:
                    cs[64:] = -cs[64:]
                k = _rope_ref(k, cs.expand(B, D))
            want[i, layer, 0] = codec.dequantize_fp4b16(*codec.quantize_fp4b16(k))
            want[i, layer, 1] = codec.dequantize_fp4b16(*codec.quantize_fp4b16(v))
    for r in range(tp):
        h0, hn = tp_head_range(H, tp, r)
        k, v = codec.unpack_kv4_records(recs[r].cpu()[:, ids])  # [layers, n, heads, 16, 128]
        assert torch.equal(k, want[:, :, 0, :, h0 : h0 + hn].permute(1, 0, 3, 2, 4))
        assert torch.equal(v, want[:, :, 1, :, h0 : h0 + hn].permute(1, 0, 3, 2, 4))
        assert (recs[r][:, 1] == 0).all()  # a block nobody named
    # and back: every rank saves its heads into the same images
    raw = geo.with_codec("raw")
    out = torch.zeros(n, raw.slot_size, dtype=torch.uint8, device="cuda")
    back = kv_ops.KVWorkList(out.data_ptr() + torch.arange(n, dtype=torch.int64, device="cuda") * raw.slot_size, work.block_ids)
    for r in range(tp):
        kv_ops.kv_save(back, raw, pool, r, status)
    got = out.cpu().view(torch.bfloat16).reshape(want.shape)
    assert status.tolist() == [0, 0] and torch.equal(got.float(), want)
    # an fp8 image of the same pages: the oracle's payload and scales
    fp8 = geo.with_codec("fp8b16")
    out8 = torch.zeros(n, fp8.slot_size, dtype=torch.uint8, device="cuda")
    for r in range(tp):
        kv_ops.kv_save(kv_ops.KVWorkList(out8.data_ptr() + torch.arange(n, dtype=torch.int64, device="cuda") * fp8.slot_size, work.block_ids), fp8, pool, r, status)
    for i in range(n):
        assert torch.equal(out8.cpu()[i], codec.pack_slot(fp8, list(want[i, :, 0]), list(want[i, :, 1])))


def test_restore_and_save_report_bad_slots_instead_of_faulting():
    _, _, kv_ops = _ops()
    geo = KVGeometry(1, 2, D, B, 2, "fp8b16")
    image = _images(geo, 1, 0).cuda()
    _, pool = _pools(kv_ops, geo, 4, 1)
    table = kv_ops.rope_table(32, inv_freq_table(D, 10000.0), "cuda")
    for ptr, block, delta, code in ((image.data_ptr(), 4, 0, 2), (image.data_ptr(), -1, 0, 2), (0, 1, 0, 4), (image.data_ptr(), 1, 32, 3),
                                    (image.data_ptr(), 1, -2**31, 3)):
        status = torch.zeros(2, dtype=torch.int32, device="cuda")
        work = kv_ops.KVWorkList(torch.tensor([image.data_ptr(), ptr], dtype=torch.int64, device="cuda"),
                                 torch.tensor([0, block], dtype=torch.int32, device="cuda"), torch.tensor([0, delta], dtype=torch.int32, device="cuda"))
        kv_ops.kv_restore(work, geo, pool, table, status)
        assert status.tolist() == [code, 1]
        if code != 3:
            status.zero_()
            kv_ops.kv_save(work, geo, pool, 0, status)
            assert status.tolist() == [code, 1]
    with pytest.raises(Exception):
        kv_ops.kv_restore(work, KVGeometry(1, 2, 64, B, 2, "fp8b16"), pool, table, status)  # another head_dim
    with pytest.raises(Exception):
        kv_ops.kv_restore(work, KVGeometry(2, 2, D, B, 2, "fp8b16"), pool, table, status)   # more layers than the pool


@pytest.mark.parametrize("img", ["fp8b16", "raw"])
def test_an_image_off_the_16_byte_grid_is_reported(img):
    _, _, kv_ops = _ops()
    geo = KVGeometry(1, 2, D, B, 2, img)
    image = torch.zeros(geo.slot_size + 16, dtype=torch.uint8, device="cuda")
    records, pool = _pools(kv_ops, geo, 4, 1)
    before = [r.clone() for r in records]
    for off in (1, 4, 8):
        work = kv_ops.KVWorkList(torch.tensor([image.data_ptr() + off], dtype=torch.int64, device="cuda"),
                                 torch.tensor([2], dtype=torch.int32, device="cuda"))
        for call in (lambda s: kv_ops.kv_restore(work, geo, pool, None, s), lambda s: kv_ops.kv_save(work, geo, pool, 0, s)):
            status = torch.zeros(2, dtype=torch.int32, device="cuda")
            call(status)
            assert status.tolist() == [4, 0]
    assert all(torch.equal(a, b) for a, b in zip(records, before)) and not image.any()


# -- attention ---------------------------------------------------------------------------


def _records(n, h, seed, layers=1, loud=0.5):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(layers, n, h, B, D, generator=g) * torch.exp(loud * torch.randn(D, generator=g))
    v = torch.randn(layers, n, h, B, D, generator=g)
    return codec.pack_kv4_records(k, v)


def _oracle(rec, tables, q, q_lens, ctx_lens, scale, pages=None, prefill=False):
    """(output in 64 bits, bound on what the kernel's roundings may change), row by row.

    q is scaled and rounded to f16 (each product off by 2^-11), p = exp(s - m) is rounded to f16 (2^-11; the maximum may lag by
    2^8, so the smallest f16 step is at most 2^-24 of the true maximum), in the prefill kernel also the exponent (2^-11 of its
    size times ln 2) and the f16 exponential itself (2^-10); fp32 sums and scores add at most 2^-14 here.  The output is a weighted mean:
    weights off by e_k change it by at most sum p_k e_k (|v_k| + |o|).  Then one rounding to bf16."""
    k_all, v_all = codec.unpack_kv4_records(rec)
    hkv = rec.shape[1]
    G = q.shape[1] // hkv
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    row = 0
    for s, (n, ctx) in enumerate(zip(q_lens, ctx_lens)):
        for t in range(n):
            last = ctx - n + t
            for h in range(hkv):
                if last < 0:
                    continue
                if pages is None:
                    lp = torch.arange(last // B + 1)
                else:
                    lp = pages[row + t, h].long()
                    lp = lp[(lp >= 0) & (lp * B <= last)]
                if lp.numel() == 0:
                    continue
                at = tables[s, lp].long()
                key = (lp[:, None] * B + torch.arange(B)).flatten()
                ok = key <= last
                k = k_all[at, h].reshape(-1, D)[ok].double()
                v = v_all[at, h].reshape(-1, D)[ok].double()
                qq = q[row + t, h * G : (h + 1) * G].double()
                sc = qq @ k.t() * scale
                a = sc - sc.max(-1, keepdim=True).values
                p = torch.softmax(sc, -1)
                o = p @ v
                e = F16_HALF * (qq.abs() @ k.abs().t()) * scale + F16_HALF + 2.0**-14
                if prefill:
                    e = e + F16_HALF * a.abs() + F16_HALF * 8 + 2.0**-10
                w = p * e + 2.0**-24 * p.max(-1, keepdim=True).values
                out[row + t, h * G : (h + 1) * G] = o
                tol[row + t, h * G : (h + 1) * G] = w @ v.abs() + w.sum(-1, keepdim=True) * o.abs() + BF16_HALF * o.abs() + 1e-6
        row += n
    return out, tol


def _setup(q_lens, ctx_lens, hq, hkv, seed=0, extra_rows=0, layers=1):
    _, _, kv_ops = _ops()
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // B) for c in ctx_lens]
    blocks = sum(need) + 3
    rec = _records(blocks, hkv, seed + 1, layers)
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    tables = torch.full((len(ctx_lens), max(need + [1]) + 1), -7, dtype=torch.int32)  # entries behind the context are not read
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = perm[at : at + n]
        at += n
    rows = sum(q_lens)
    q = (torch.randn(rows + extra_rows, hq, D, generator=g) * 1.3).to(torch.bfloat16)
    pool = kv_ops.PagedKV4Pool.from_tensors([rec.cuda()])
    start = torch.tensor([0] + torch.tensor(q_lens).cumsum(0).tolist(), dtype=torch.int32)
    return pool, rec, tables, q, start


def _attend(pool, layer, tables, q, start, ctx_lens, max_q, hkv, split=None, ws=None, max_ctx=None, out=None):
    attention, _, _ = _ops()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    kw = {} if split is None else dict(nsplit=split)
    attention.paged_attention(q.cuda(), out, pool, layer, tables.cuda(), start.cuda(), torch.tensor(ctx_lens, dtype=torch.int32, device="cuda"),
                              max_q, max_ctx or max(ctx_lens), hkv, D**-0.5, ws, **kw)
    torch.cuda.synchronize()
    assert attention.kv4_status() == 0
    return out.double().cpu()


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,split", [
    ([1], [1], 8, 1, None),
    ([1], [16], 8, 1, None),
    ([1], [17], 4, 4, None),                                 # one head per KV head
    ([1, 1, 1, 1], [15, 100, 33, 512], 16, 2, None),
    ([1, 1], [700, 1500], 64, 8, None),
    ([1, 1], [700, 1500], 64, 8, 9),                         # nine CTAs share the pages of sixteen items
    ([1, 1], [2500, 90], 10, 2, 7),                          # five heads per KV head
    ([1], [3000], 7, 1, 0),                                  # seven
    ([1, 1], [900, 40], 32, 2, None),                        # sixteen: two column tiles
    ([2, 1, 3], [40, 300, 3], 8, 1, None),                   # several query rows; pure prefill of the last sequence
    ([5, 0, 2], [37, 64, 1000], 16, 4, 5),                   # a sequence without queries
    ([9], [333], 14, 2, None),                               # 63 rows: four row tiles
    ([9, 1, 4], [333, 20, 700], 14, 2, 6),                   # tiles of several sequences over the CTAs
    ([1, 1, 1], [0, 20, 0], 8, 2, None),                     # no keys at all: zeros
    ([4], [2], 8, 2, None),                                  # the first rows see no key
    ([1], [9000], 8, 1, 0),                                  # 71 pages a warp: the page windows turn over twice
    ([1], [9000], 8, 1, 200),                                # CTAs with less than a page a warp
    ([1, 0, 1, 2], [0, 0, 1700, 5], 4, 2, 50),               # items without keys between shared ones
    ([1] * 40, list(range(3, 1203, 30)), 8, 1, 31),          # more sequences than a warp has lanes
])
def test_decode_matches_the_formula(q_lens, ctx_lens, hq, hkv, split):
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=len(q_lens) + hq, extra_rows=2)
    got = _attend(pool, 0, tables, q, start, ctx_lens, max(q_lens), hkv, split)
    rows = sum(q_lens)
    want, tol = _oracle(rec[0], tables, q[:rows], q_lens, ctx_lens, D**-0.5)
    assert ((got[:rows] - want).abs() <= tol).all(), (got[:rows] - want).abs().max()
    assert (got[rows:] == 7.0).all()  # rows behind the last sequence are left as they were


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,split", [
    ([64], [320], 8, 1, None),
    ([16], [16], 8, 1, None),                                # a single tile, causal inside it
    ([100], [100], 16, 2, None),
    ([20, 33], [500, 81], 32, 8, None),
    ([13], [650], 32, 2, 3),                                # sixteen heads per KV head
    ([70], [257], 2, 2, 1),                                  # one head per KV head: 70 rows of a tile
    ([14, 0, 15], [214, 50, 15], 10, 2, 2),                  # five heads: 125 rows a tile; an empty sequence
    ([30], [12], 8, 2, None),                                # more queries than keys: the first rows see none
    ([130], [130], 7, 1, None),                              # 18 tokens of seven heads a tile
])
def test_prefill_matches_the_formula(q_lens, ctx_lens, hq, hkv, split):
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=len(q_lens) + hq, extra_rows=3)
    got = _attend(pool, 0, tables, q, start, ctx_lens, max(q_lens), hkv, split)
    rows = sum(q_lens)
    want, tol = _oracle(rec[0], tables, q[:rows], q_lens, ctx_lens, D**-0.5, prefill=True)
    assert ((got[:rows] - want).abs() <= tol).all(), ((got[:rows] - want).abs() - tol).max()
    assert (got[rows:] == 7.0).all()


@pytest.mark.parametrize("q_len", [1, 3, 32])
def test_what_lies_behind_the_context_does_not_reach_the_output(q_len):
    """Tokens behind the last one, in the same page and in pages behind it, hold NaN and infinity scales."""
    _, _, kv_ops = _ops()
    ctx = [200, 33]
    pool, rec, tables, q, start = _setup([q_len] * 2, ctx, 8, 1, seed=4)
    dirty = rec.clone()
    for s, c in enumerate(ctx):
        page = dirty[0, tables[s, (c - 1) // B].long(), 0]
        for t in range((c - 1) % B + 1, B):
            page[2048 + 8 * t : 2056 + 8 * t] = 0xFF
            for g in range(8):
                page[2176 + (t // 8) * 64 + 8 * g + t % 8] = 0xF8 if g & 1 else 0xFF
    used = set(tables[tables >= 0].tolist())
    for blk in set(range(rec.shape[1])) - used:
        dirty[0, blk] = 0xFF
    pool = kv_ops.PagedKV4Pool.from_tensors([dirty.cuda()])
    got = _attend(pool, 0, tables.clamp(min=0), q, start, ctx, q_len, 1)
    want, tol = _oracle(rec[0], tables, q, [q_len] * 2, ctx, D**-0.5, prefill=q_len * 8 >= 64)
    assert ((got - want).abs() <= tol).all()


def test_a_key_that_is_not_finite_shows():
    """A NaN in a visible key or value is not turned into a number, in either kernel and through a merge of splits."""
    for q_len, split in ((1, None), (1, 3), (16, None), (16, 2)):
        pool, rec, tables, q, start = _setup([q_len], [300], 8, 1, seed=5)
        rec[0, tables[0, 4].long(), 0, 2048 : 2056] = 0xFF  # the scales of key 64
        from daser_b200.ops import kv_ops

        got = _attend(kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables, q, start, [300], q_len, 1, split)
        assert torch.isnan(got).all()


def test_scores_far_apart_and_large_values():
    """Maxima that rise page after page (the accumulator is rescaled each time) and a single dominating key."""
    _, _, kv_ops = _ops()
    for q_len in (1, 16):
        ctx = 400
        _, rec, tables, q, start = _setup([q_len], [ctx], 8, 1, seed=6)
        k = torch.randn(26, 1, B, D) * 0.05
        q = torch.ones(q_len, 8, D).to(torch.bfloat16)
        for i in range(25):
            k[i] += 0.12 * (i + 1)
        v = torch.randn(26, 1, B, D) * 1000
        rec = codec.pack_kv4_records(k, v)[None]
        tables = torch.arange(26, dtype=torch.int32)[None]
        got = _attend(kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables, q, start, [ctx], q_len, 1)
        want, tol = _oracle(rec[0], tables, q, [q_len], [ctx], D**-0.5, prefill=q_len > 1)
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def test_layers_and_strided_pools():
    _, _, kv_ops = _ops()
    pool, rec, tables, q, start = _setup([1, 1], [130, 77], 8, 2, seed=7, layers=3)
    big = torch.zeros(3, rec.shape[1], 5, 2304, dtype=torch.uint8, device="cuda")
    big[:, :, 1:5:2] = rec.cuda()
    strided = kv_ops.PagedKV4Pool.from_tensors([big[:, :, 1:5:2]])
    for layer in (0, 2):
        want, tol = _oracle(rec[layer], tables, q, [1, 1], [130, 77], D**-0.5)
        for p in (pool, strided):
            assert ((_attend(p, layer, tables, q, start, [130, 77], 1, 2) - want).abs() <= tol).all()


def test_record_offsets_beyond_two_gigabytes():
    """A pool of 2.3 GB: the last blocks lie beyond 2^31 bytes."""
    _, ew, kv_ops = _ops()
    blocks = 1_000_000
    pool = kv_ops.PagedKV4Pool.zeros(1, blocks, 1, "cuda")
    rec = _records(3, 1, 9)
    last = torch.tensor([[blocks - 1, blocks - 3, blocks - 2]], dtype=torch.int32)
    pool.keepalive[0][0][0, last[0].long().cuda()] = rec[0].cuda()
    q = torch.randn(1, 8, D).to(torch.bfloat16)
    got = _attend(pool, 0, last, q, torch.tensor([0, 1], dtype=torch.int32), [41], 1, 1)
    want, tol = _oracle(rec[0], torch.tensor([[0, 1, 2]]), q, [1], [41], D**-0.5)
    assert ((got - want).abs() <= tol).all()
    slots = torch.tensor([blocks * B - 1, blocks * B - 17, 5], dtype=torch.int64, device="cuda")
    k, v = kv_ops.kv_read(pool, 0, slots)
    rk, rv = codec.unpack_kv4_records(rec[0])
    assert torch.equal(k[0].float().cpu(), rk[0, :, 15]) and torch.equal(v[1].float().cpu(), rv[2, :, 15]) and (k[2] == 0).all()


# -- bounds, selection, sparse attention ---------------------------------------------------


def _bounds_oracle(k):
    """fp64 keys ``[tokens, 128]`` -> (codes, exponent)."""
    hi, lo = k.max(0).values, k.min(0).values
    a = torch.maximum(hi.abs(), lo.abs()).max().item()
    if a == 0:
        return torch.zeros(2, D), -100
    e = -150
    while a > 127 * 2.0**e:
        e += 1
    return torch.stack([torch.ceil(hi / 2.0**e), torch.floor(lo / 2.0**e)]), e


@pytest.mark.parametrize("ctx,q_lens", [([1, 16, 17], [1, 1, 1]), ([100, 45, 70], [100, 3, 0]), ([33, 0, 500], [2, 0, 37])])
def test_page_bounds_are_exact_and_only_of_the_pages_touched(ctx, q_lens):
    _, _, kv_ops = _ops()
    pool, rec, tables, _, start = _setup(q_lens, ctx, 8, 2, seed=11, layers=2)
    rec[1, tables[0, 0].long(), 1, 0:1024] = 0  # a page of zeros
    pool = kv_ops.PagedKV4Pool.from_tensors([rec.cuda()])
    bounds = kv_ops.PageBounds.for_pool(pool)
    bounds.codes.fill_(55)
    bounds.exps.fill_(33)
    kv_ops.update_page_bounds(pool, bounds, 1, tables.cuda(), start.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), max(q_lens))
    torch.cuda.synchronize()
    k, _ = codec.unpack_kv4_records(rec[1])
    touched = {}
    for s, (c, n) in enumerate(zip(ctx, q_lens)):
        if n:
            for p in range(max(c - n, 0) // B, (c - 1) // B + 1):
                touched[int(tables[s, p])] = min(B, c - B * p)
    codes, exps = bounds.codes.cpu(), bounds.exps.cpu()
    for blk in range(rec.shape[1]):
        for h in range(2):
            if blk in touched:
                want, e = _bounds_oracle(k[blk, h, : touched[blk]].double())
                assert torch.equal(codes[1, blk, h].double(), want.double()) and exps[1, blk, h] == e
            else:
                assert (codes[1, blk, h] == 55).all() and exps[1, blk, h] == 33
    assert (codes[0] == 55).all()
    read = bounds.read(1, torch.tensor(sorted(touched), dtype=torch.int32, device="cuda")).cpu().double()
    for i, blk in enumerate(sorted(touched)):
        kk = k[blk, :, : touched[blk]].double()
        assert (read[i, :, 0] >= kk.max(1).values).all() and (read[i, :, 1] <= kk.min(1).values).all()
        assert torch.equal(read[i], codes[1, blk].double() * torch.exp2(exps[1, blk].double())[:, None, None])


def test_page_bounds_of_a_key_that_is_not_finite():
    """Such a page has infinite bounds, so that it is always among the selected ones; one behind the context does not count."""
    _, _, kv_ops = _ops()
    rec = _records(3, 1, 13)
    rec[0, 1, 0, 2048 + 8 * 5 + 3] = 0xFF  # token 5
    rec[0, 2, 0, 2048 + 8 * 5 + 3] = 0xFF
    pool = kv_ops.PagedKV4Pool.from_tensors([rec.cuda()])
    bounds = kv_ops.PageBounds.for_pool(pool)
    i32 = dict(dtype=torch.int32, device="cuda")
    kv_ops.update_page_bounds(pool, bounds, 0, torch.tensor([[0, 1, 2]], **i32), torch.tensor([0, 36], **i32), torch.tensor([36], **i32), 36)
    read = bounds.read(0, torch.tensor([[0, 1], [2, 3]], **i32))
    assert read.shape == (2, 2, 1, 2, 128) and torch.isfinite(read[0, 0]).all() and torch.isfinite(read[1, 0]).all()
    assert (read[0, 1, 0, 0] == float("inf")).all() and (read[0, 1, 0, 1] == -float("inf")).all()
    assert (read[1, 1] == 0).all()  # a block outside the pool


def _select_oracle(q, codes, exps, tables, q_lens, ctx_lens, n_pages, sink, recent):
    """In whole numbers."""
    hkv = exps.shape[1]
    G = q.shape[1] // hkv
    out = torch.full((q.shape[0], hkv, n_pages), -1, dtype=torch.int32)
    row = 0
    for s, (n, ctx) in enumerate(zip(q_lens, ctx_lens)):
        for t in range(n):
            count = (ctx - n + t) // B + 1
            for h in range(hkv):
                if count <= n_pages:
                    pages = list(range(max(count, 0)))
                else:
                    x = q[row + t, h * G : (h + 1) * G].double()
                    up, down = x.clamp(min=0).sum(0), x.clamp(max=0).sum(0)
                    a, e = max(up.max().item(), -down.min().item()), -150
                    if a > 0:
                        while a > 127 * 2.0**e:
                            e += 1
                    iq = torch.stack([torch.round(up / 2.0**e), torch.round(down / 2.0**e)]).long()
                    blk = tables[s, :count].long()
                    dots = (codes[blk, h].long() * iq).sum((-2, -1)).tolist()
                    score = [d * 2.0 ** int(x) if x < 127 else float("inf") for d, x in zip(dots, exps[blk, h].tolist())]
                    rest = sorted(range(sink, count - recent), key=lambda p: (-score[p], p))[: n_pages - sink - recent]
                    pages = list(range(sink)) + sorted(rest) + list(range(count - recent, count))
                out[row + t, h, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
        row += n
    return out


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,n_pages,sink,recent", [
    ([1], [1000], 8, 1, 9, 1, 4),
    ([1, 1, 1], [5000, 3200, 100], 16, 2, 17, 2, 1),
    ([2, 0, 3], [2000, 70, 1999], 10, 2, 32, 0, 3),
    ([1], [900], 8, 2, 5, 1, 4),           # no place left to compete for
    ([1], [9000], 16, 1, 550, 1, 4),       # nearly all
    ([1, 1], [0, 16], 4, 4, 3, 1, 1),      # no key; one page
    ([1], [16 * 33], 8, 1, 32, 1, 4),      # one page too many
])
def test_selection_matches_whole_number_arithmetic(q_lens, ctx_lens, hq, hkv, n_pages, sink, recent):
    attention, _, kv_ops = _ops()
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=n_pages)
    bounds = kv_ops.PageBounds.for_pool(pool)
    ctx = torch.tensor(ctx_lens, dtype=torch.int32, device="cuda")
    full = torch.tensor([0] + torch.tensor(ctx_lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    kv_ops.update_page_bounds(pool, bounds, 0, tables.cuda(), full, ctx, max(ctx_lens))
    for ws in (None, attention.AttentionWorkspace("cuda")):
        got = attention.select_pages(q.cuda(), bounds, 0, tables.cuda(), start.cuda(), ctx, max(q_lens), max(ctx_lens), n_pages, sink, recent, ws)
        want = _select_oracle(q, bounds.codes[0].cpu(), bounds.exps[0].cpu(), tables, q_lens, ctx_lens, n_pages, sink, recent)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kind", ["ties", "all equal", "zero query", "poisoned", "long"])
def test_selection_of_hard_scores(kind):
    attention, _, kv_ops = _ops()
    torch.manual_seed(12)
    pages = 45000 if kind == "long" else 1500
    codes = torch.randint(-127, 128, (1, pages, 1, 2, D), dtype=torch.int8)
    exps = torch.randint(-9, 3, (1, pages, 1), dtype=torch.int8)
    if kind == "ties":  # 1500 pages with three different contents
        codes = codes[:, torch.arange(pages) % 3]
        exps.fill_(-3)
    if kind == "all equal":
        codes = codes[:, :1].expand(1, pages, 1, 2, D).contiguous()
        exps.fill_(0)
    if kind == "poisoned":
        exps[0, [7, 700, 1400], 0] = 127
    q = torch.randn(1, 8, D).to(torch.bfloat16)
    if kind == "zero query":
        q.zero_()
    bounds = kv_ops.PageBounds(codes.cuda(), exps.cuda())
    tables = torch.randperm(pages).to(torch.int32)[None]
    if kind == "ties":
        tables = torch.arange(pages, dtype=torch.int32)[None]
    i32 = dict(dtype=torch.int32, device="cuda")
    for n in (6, 64, 333):
        got = attention.select_pages(q.cuda(), bounds, 0, tables.cuda(), torch.tensor([0, 1], **i32), torch.tensor([pages * B], **i32), 1, pages * B, n)
        want = _select_oracle(q, codes[0], exps[0], tables, [1], [pages * B], n, 1, 4)
        assert torch.equal(got.cpu(), want), n


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,n_pages", [([1], [1000], 8, 1, 9), ([1, 1], [900, 30], 32, 8, 17), ([3, 0, 1], [700, 9, 400], 10, 2, 12),
                                                            ([1], [2600], 32, 2, 140), ([2], [1], 8, 2, 5)])
def test_sparse_attention_matches_the_formula_over_the_listed_pages(q_lens, ctx_lens, hq, hkv, n_pages):
    attention, _, kv_ops = _ops()
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=n_pages, extra_rows=1)
    rows = sum(q_lens)
    pages = torch.full((rows + 1, hkv, n_pages), -1, dtype=torch.int32)
    row = 0
    for n, ctx in zip(q_lens, ctx_lens):
        for t in range(n):
            have = -(-ctx // B)
            for h in range(hkv):
                take = torch.randperm(have)[: min(have, n_pages - 1)].sort().values
                pages[row, h, : take.numel()] = take.to(torch.int32)
                pages[row, h, take.numel()] = 10**6  # outside the context: skipped
            row += 1
    ctx = torch.tensor(ctx_lens, dtype=torch.int32, device="cuda")
    want, tol = _oracle(rec[0], tables, q[:rows], q_lens, ctx_lens, D**-0.5, pages=pages)
    for ws in (None, attention.AttentionWorkspace("cuda")):
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
        attention.sparse_paged_attention(q.cuda(), out, pool, 0, tables.cuda(), start.cuda(), ctx, pages.cuda(), max(q_lens), D**-0.5, ws)
        got = out.double().cpu()
        assert attention.kv4_status() == 0
        assert ((got[:rows] - want).abs() <= tol).all()
        assert (got[rows:] == 7.0).all()


def test_all_pages_listed_is_dense_attention():
    attention, _, kv_ops = _ops()
    pool, rec, tables, q, start = _setup([1, 1], [777, 300], 16, 2, seed=21)
    bounds = kv_ops.PageBounds.for_pool(pool)
    ctx = torch.tensor([777, 300], dtype=torch.int32, device="cuda")
    pages = attention.select_pages(q.cuda(), bounds, 0, tables.cuda(), start.cuda(), ctx, 1, 777, 49)
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    attention.sparse_paged_attention(q.cuda(), out, pool, 0, tables.cuda(), start.cuda(), ctx, pages, 1, D**-0.5)
    want, tol = _oracle(rec[0], tables, q, [1, 1], [777, 300], D**-0.5)
    assert ((out.double().cpu() - want).abs() <= tol).all()


# -- a run of them together ---------------------------------------------------------------


def _decode_steps(steps, hq, hkv, ctx0, n_pages, stream=None, graph=False):
    """Prefill ctx0 tokens, then `steps` decode steps: write, bounds, selection, sparse and dense attention.  Returns what each step gave and
    the plain K and V (as the format holds them)."""
    attention, ew, kv_ops = _ops()
    g = torch.Generator().manual_seed(31)
    total = ctx0 + steps
    blocks = -(-total // B) + 2
    pool = kv_ops.PagedKV4Pool.zeros(1, blocks, hkv, "cuda")
    bounds = kv_ops.PageBounds.for_pool(pool)
    table = torch.randperm(blocks, generator=g).to(torch.int32)[None]
    tables = table.cuda()
    cos_sin = kv_ops.rope_table(total, inv_freq_table(D, 10000.0), "cuda")
    x = torch.randn(total, (hq + 2 * hkv) * D, generator=g).to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    ws = attention.AttentionWorkspace("cuda")
    slot_of = lambda i: int(table[0, i // B]) * B + i % B  # noqa: E731

    def buffers(n):
        return dict(x=torch.zeros(n, x.shape[1], dtype=torch.bfloat16, device="cuda"), pos=torch.zeros(n, **i32), slot=torch.zeros(n, dtype=torch.int64, device="cuda"),
                    start=torch.tensor([0, n], **i32), ctx=torch.zeros(1, **i32), q=torch.zeros(n, hq, D, dtype=torch.bfloat16, device="cuda"),
                    dense=torch.zeros(n, hq, D, dtype=torch.bfloat16, device="cuda"), sparse=torch.zeros(n, hq, D, dtype=torch.bfloat16, device="cuda"))

    def fill(b, i, n):
        b["x"].copy_(x[i : i + n])
        b["pos"].copy_(torch.arange(i, i + n, dtype=torch.int32))
        b["slot"].copy_(torch.tensor([slot_of(j) for j in range(i, i + n)]))
        b["ctx"].fill_(i + n)

    def step(b, n, sparse):
        ew.rope_kv_write(b["x"], b["pos"], b["slot"], cos_sin, b["q"], hq, hkv, D, B, pool, 0)
        kv_ops.update_page_bounds(pool, bounds, 0, tables, b["start"], b["ctx"], n)
        attention.paged_attention(b["q"], b["dense"], pool, 0, tables, b["start"], b["ctx"], n, total, hkv, D**-0.5, ws)
        if sparse:
            b["pages"] = attention.select_pages(b["q"], bounds, 0, tables, b["start"], b["ctx"], n, total, n_pages, workspace=ws)
            attention.sparse_paged_attention(b["q"], b["sparse"], pool, 0, tables, b["start"], b["ctx"], b["pages"], n, D**-0.5, ws)

    got = []
    with torch.cuda.stream(stream or torch.cuda.current_stream()):
        b = buffers(ctx0)
        fill(b, 0, ctx0)
        step(b, ctx0, False)
        got.append((b["q"].cpu(), b["dense"].cpu(), None, None))
        b = buffers(1)
        replay = None
        for i in range(steps):
            fill(b, ctx0 + i, 1)
            if graph and i == 1:
                torch.cuda.synchronize()
                replay = torch.cuda.CUDAGraph()
                with torch.cuda.graph(replay):
                    step(b, 1, True)
            if replay is not None:
                replay.replay()
            else:
                step(b, 1, True)
            got.append((b["q"].cpu(), b["dense"].cpu(), b["sparse"].cpu(), b["pages"].cpu()))
        torch.cuda.synchronize()
    assert attention.kv4_status() == 0
    return got, pool.keepalive[0][0][0].cpu(), table


@pytest.mark.parametrize("how", ["eager", "stream", "graph"])
def test_prefill_then_decode_steps_with_sparse_attention(how):
    hq, hkv, ctx0, steps, n_pages = 16, 2, 170, 20, 8
    side = torch.cuda.Stream() if how == "stream" else None
    got, rec, table = _decode_steps(steps, hq, hkv, ctx0, n_pages, side, how == "graph")
    q, dense, _, _ = got[0]
    want, tol = _oracle(rec, table, q, [ctx0], [ctx0], D**-0.5, prefill=True)
    assert ((dense.double() - want).abs() <= tol).all()
    for i in range(steps):
        ctx = ctx0 + i + 1
        q, dense, sparse, pages = got[1 + i]
        want, tol = _oracle(rec, table, q, [1], [ctx], D**-0.5)
        assert ((dense.double() - want).abs() <= tol).all(), i
        assert pages[0, 0, 0] == 0 and pages[0, :, -4:].tolist() == [list(range((ctx - 1) // B - 3, (ctx - 1) // B + 1))] * hkv
        want, tol = _oracle(rec, table, q, [1], [ctx], D**-0.5, pages=pages)
        assert ((sparse.double() - want).abs() <= tol).all(), i


def test_two_captured_graphs_with_workspaces_of_their_own_replay_side_by_side():
    attention, _, _ = _ops()
    made = []
    for seed in (41, 42):
        pool, rec, tables, q, start = _setup([1], [2000], 16, 2, seed=seed)
        args = (q.cuda(), torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), pool, 0, tables.cuda(), start.cuda(),
                torch.tensor([2000], dtype=torch.int32, device="cuda"), 1, 2000, 2, D**-0.5, None)  # no workspace: the call's own
        attention.paged_attention(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attention.paged_attention(*args)
        made.append((graph, args, _oracle(rec[0], tables, q, [1], [2000], D**-0.5)))  # a graph's inputs live as long as it does
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (graph, _, _), s in zip(made, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, args, (want, tol) in made:
        assert ((args[1].double().cpu() - want).abs() <= tol).all()


def test_results_repeat_bit_for_bit():
    attention, _, _ = _ops()
    pool, rec, tables, q, start = _setup([1] * 6, [3000, 20, 800, 1601, 2999, 1], 64, 8, seed=51)
    ws = attention.AttentionWorkspace("cuda")
    first = _attend(pool, 0, tables, q, start, [3000, 20, 800, 1601, 2999, 1], 1, 8, 70, ws)
    for _ in range(3):
        assert torch.equal(_attend(pool, 0, tables, q, start, [3000, 20, 800, 1601, 2999, 1], 1, 8, 70, ws), first)


def test_refusals_on_the_gpu():
    attention, ew, kv_ops = _ops()
    pool, rec, tables, q, start = _setup([1], [40], 8, 2, seed=61)
    t, s, c, qd = tables.cuda(), start.cuda(), torch.tensor([40], dtype=torch.int32, device="cuda"), q.cuda()
    out = torch.empty_like(qd)
    good = dict(q=qd, out=out, pool=pool, layer=0, block_tables=t, q_start=s, ctx_lens=c, max_q_len=1, max_ctx=40, num_kv_heads=2,
                softmax_scale=1.0, workspace=None)
    attention.paged_attention(**good)
    for change in (dict(layer=1), dict(layer=-1), dict(rank=1), dict(num_kv_heads=1), dict(q=qd.half()), dict(q=qd[..., :64]), dict(q=qd[:, :3]),
                   dict(out=out.float()), dict(out=out[:0]), dict(block_tables=t.long()), dict(block_tables=t[:0]), dict(q_start=s[:1]),
                   dict(ctx_lens=c.cpu()), dict(block_tokens=32), dict(nsplit=1), dict(nsplit=-1), dict(nsplit=2, split_tokens=16),
                   dict(q=torch.zeros(1, 64, 128, dtype=torch.bfloat16, device="cuda"), out=torch.zeros(1, 64, 128, dtype=torch.bfloat16, device="cuda")),
                   dict(q=qd.expand(2, 8, 128), out=torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            attention.paged_attention(**{**good, **change})
    bounds = kv_ops.PageBounds.for_pool(pool)
    for bad in (dict(num_pages=4), dict(sink_pages=-1), dict(recent_pages=0), dict(layer=1)):
        with pytest.raises(ValueError):
            attention.select_pages(**{**dict(q=qd, bounds=bounds, layer=0, block_tables=t, q_start=s, ctx_lens=c, max_q_len=1, max_ctx=40, num_pages=8), **bad})
    with pytest.raises(ValueError):
        attention.sparse_paged_attention(qd, out, pool, 0, t, s, c, torch.zeros(1, 1, 4, dtype=torch.int32, device="cuda"), 1, 1.0)
    with pytest.raises(ValueError):
        kv_ops.update_page_bounds(kv_ops.PagedKV4Pool.zeros(1, 2, 2, "cuda"), bounds, 0, t, s, c, 1)
    x = torch.zeros(1, 12 * 128, device="cuda")
    one = dict(qkv=x, positions=c, slot_mapping=c.long(), cos_sin=torch.zeros(4, 128, device="cuda"), q_out=out, num_q_heads=8, num_kv_heads=2,
               head_dim=128, block_tokens=16, pool=pool, layer=0)
    for change in (dict(num_kv_heads=1), dict(head_dim=64), dict(block_tokens=32), dict(qkv=x.half()), dict(qkv=x[:, :512]), dict(positions=c.long()),
                   dict(slot_mapping=c), dict(cos_sin=torch.zeros(4, 64, device="cuda")), dict(q_out=out.float()), dict(layer=3),
                   dict(qk_norm=(x[0, :128], x[0, :128], 1e-6))):
        with pytest.raises(ValueError):
            ew.rope_kv_write(**{**one, **change})


def test_work_lists_that_do_not_fit_are_refused():
    _, _, kv_ops = _ops()
    geo = KVGeometry(1, 2, D, B, 2, "fp8b16")
    _, pool = _pools(kv_ops, geo, 4, 1)
    image = torch.zeros(geo.slot_size, dtype=torch.uint8, device="cuda")
    ptr, blk, dlt = (torch.tensor([v], dtype=t, device="cuda") for v, t in ((image.data_ptr(), torch.int64), (0, torch.int32), (1, torch.int32)))
    table = kv_ops.rope_table(32, inv_freq_table(D, 10000.0), "cuda")
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    W = kv_ops.KVWorkList
    kv_ops.kv_restore(W(ptr, blk, dlt), geo, pool, table, status)
    for work in (W(ptr.int(), blk), W(ptr, blk.long()), W(ptr, blk, dlt.long()), W(ptr, blk.repeat(2)), W(ptr, blk, dlt[:0]), W(ptr.cpu(), blk),
                 W(ptr.repeat(2), blk.repeat(4)[::2], None)):
        with pytest.raises(ValueError):
            kv_ops.kv_restore(work, geo, pool, table, status)
        with pytest.raises(ValueError):
            kv_ops.kv_save(work, geo, pool, 0, status)
    for bad in (table[:, :64], table.double(), table.cpu()):
        with pytest.raises(ValueError):
            kv_ops.kv_restore(W(ptr, blk, dlt), geo, pool, bad, status)
    for bad in (status[:1], status.long()):
        with pytest.raises(ValueError):
            kv_ops.kv_restore(W(ptr, blk, dlt), geo, pool, table, bad)
    with pytest.raises(ValueError):
        kv_ops.kv_restore(W(ptr, blk), KVGeometry(1, 2, D, B, 4, "raw"), pool, None, status)  # four bytes a value
    with pytest.raises(ValueError):
        pool.c_struct()  # operators of the fp8 pool


@pytest.mark.parametrize("split", [0, 5])
def test_query_tokens_beyond_max_q_len_are_left_alone(split):
    """A caller's max_q_len that is too small: rows below it are right, and nothing is written outside the call's own memory."""
    attention, _, kv_ops = _ops()
    q_lens, ctx_lens = [3, 9, 2], [300, 900, 500]
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, 8, 2, seed=71)
    ws = attention.AttentionWorkspace(torch.device("cuda"))
    ws.ensure(16, 148, D)
    places = ws.ensure_shared(200)
    places.fill_(77)
    out = _attend(pool, 0, tables, q, start, ctx_lens, 2, 2, split, ws)
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5)
    at = 0
    for n in q_lens:
        assert ((out - want).abs() <= tol)[at : at + 2].all()
        assert (out[at + 2 : at + n] == 7.0).all()
        at += n
    assert (places[2 * 3 * 2 :] == 77).all()  # 3 sequences x one tile x 2 KV heads, two words each


def test_rows_in_front_of_the_first_sequence_are_left_alone():
    attention, _, kv_ops = _ops()
    pool, rec, tables, q, start = _setup([1, 1], [700, 900], 8, 2, seed=72, extra_rows=3)
    start = start + 2  # rows 0, 1 belong to nobody; the places of their items are whatever the workspace holds
    q = torch.cat([q[2:4], q])[: 2 + 2 + 1]
    pages = torch.arange(12, dtype=torch.int32).expand(5, 2, 12).contiguous().cuda()
    c = torch.tensor([700, 900], dtype=torch.int32, device="cuda")
    for junk in (0, 1, 3, 2**30, -5):
        ws = attention.AttentionWorkspace(torch.device("cuda"))
        ws.ensure(16, 148, D)
        ws.ensure_shared(64).fill_(junk)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
        attention._attention_kv4(q.cuda(), out, pool, 0, tables.cuda(), start.cuda(), c, 1, 0, D**-0.5, ws, 0, pages, 3)
        torch.cuda.synchronize()
        want, tol = _oracle(rec[0], tables, q[2:4], [1, 1], [700, 900], D**-0.5, pages=pages[2:4].cpu())
        assert ((out[2:4].double().cpu() - want).abs() <= tol).all()
        assert (out[4:] == 7.0).all()


def test_prefill_tokens_beyond_max_q_len_are_left_alone():
    q_lens, ctx_lens = [100, 3], [300, 900]
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, 8, 2, seed=73)
    out = _attend(pool, 0, tables, q, start, ctx_lens, 64, 2, 3)  # a CTA has 64 tokens
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5, prefill=True)
    assert ((out - want).abs() <= tol)[list(range(64)) + [100, 101, 102]].all()
    assert (out[64:100] == 7.0).all()


@pytest.mark.parametrize("seqs,hkv", [(40, 4), (20, 4), (9, 4), (3, 4), (1, 1)])
def test_selection_with_any_number_of_lists(seqs, hkv):
    """The more lists, the fewer CTAs work on one: 160 lists to 1, of 200 to 560 pages."""
    attention, _, kv_ops = _ops()
    g = torch.Generator().manual_seed(13)
    ctx = torch.randint(200 * B, 560 * B, (seqs,), generator=g).tolist()
    ctx[0] = 560 * B - 1
    pages, width = 700, 560
    codes = torch.randint(-127, 128, (1, pages, hkv, 2, D), dtype=torch.int8, generator=g)
    exps = torch.randint(-6, -2, (1, pages, hkv), dtype=torch.int8, generator=g)
    tables = torch.stack([torch.randperm(pages, generator=g)[:width] for _ in range(seqs)]).to(torch.int32)
    q = torch.randn(seqs, 2 * hkv, D, generator=g).to(torch.bfloat16)
    bounds = kv_ops.PageBounds(codes.cuda(), exps.cuda())
    start, lens = torch.arange(seqs + 1, dtype=torch.int32, device="cuda"), torch.tensor(ctx, dtype=torch.int32, device="cuda")
    want = _select_oracle(q, codes[0], exps[0], tables, [1] * seqs, ctx, 40, 1, 4)
    for max_ctx in (max(ctx), 300_000, 2_300_000):  # scores on chip, scratch at hand, scratch in use by a list of 8 CTAs
        if max_ctx > 10**6 and seqs > 3:
            continue
        got = attention.select_pages(q.cuda(), bounds, 0, tables.cuda(), start, lens, 1, max_ctx, 40)
        assert torch.equal(got.cpu(), want), max_ctx


def _junk_workspace(attention):
    """A workspace whose partials hold large finite numbers with weights to match: what an earlier call may have left."""
    ws = attention.AttentionWorkspace(torch.device("cuda"))
    ws.ensure(32, 256, D)
    ws.part_o.fill_(1e4)
    ws.part_lse.fill_(60.0)
    return ws


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,max_ctx,split", [
    ([1], [500], 8, 1, 131072, None),                                  # planned for a capacity: 112 units, 148 CTAs
    ([1], [100], 8, 1, 131072, None),
    ([1], [500], 8, 1, 65536, None),
    ([1], [0], 8, 1, 131072, None),                                    # no key at all
    ([0, 0, 1, 0, 0, 0, 0, 0], [40, 40, 320, 40, 40, 40, 40, 40], 8, 1, 16384, None),  # one of eight has a query
    ([1] + [0] * 63, [77] * 64, 8, 1, 32768, None),
    ([0, 0], [40, 300], 8, 1, 131072, None),                           # nobody has one
    ([1], [40], 8, 1, None, 200),                                      # more CTAs asked for than there are units
    ([1], [300], 16, 1, 131072, None),                                 # two column tiles
    ([3, 1], [90, 20], 8, 1, 131072, 250),
])
def test_more_ctas_than_there_is_work_to_share(q_lens, ctx_lens, hq, hkv, max_ctx, split):
    """CTAs are planned from max_ctx, the work comes from the lengths: what no CTA wrote must not be merged."""
    attention, _, _ = _ops()
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=81, extra_rows=1)
    got = _attend(pool, 0, tables, q, start, ctx_lens, max(max(q_lens), 1), hkv, split, _junk_workspace(attention), max_ctx)
    rows = sum(q_lens)
    want, tol = _oracle(rec[0], tables, q[:rows], q_lens, ctx_lens, D**-0.5)
    assert ((got[:rows] - want).abs() <= tol).all(), (got[:rows] - want).abs().max()
    assert (got[rows:] == 7.0).all()


def test_a_captured_decode_step_planned_for_its_capacity():
    """One graph for contexts of 17 to 2000 keys: with few keys there are fewer units than CTAs."""
    attention, _, _ = _ops()
    pool, rec, tables, q, start = _setup([1], [2000], 8, 1, seed=82)
    ctx = torch.tensor([2000], dtype=torch.int32, device="cuda")
    ws = _junk_workspace(attention)
    args = (q.cuda(), torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda"), pool, 0, tables.cuda(), start.cuda(), ctx, 1, 131072, 1, D**-0.5, ws)
    attention.paged_attention(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention.paged_attention(*args)
    for n in (2000, 1100, 300, 17, 1, 1500):
        ctx.fill_(n)
        ws.part_o.fill_(1e4)
        graph.replay()
        want, tol = _oracle(rec[0], tables, q, [1], [n], D**-0.5)
        assert ((args[1].double().cpu() - want).abs() <= tol).all(), n


def test_sparse_rows_of_no_sequence_leave_fewer_units_than_ctas():
    attention, _, _ = _ops()
    pool, rec, tables, q, start = _setup([1], [400], 8, 1, seed=83, extra_rows=30)
    pages = torch.arange(20, dtype=torch.int32).expand(31, 1, 20).contiguous()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    attention._attention_kv4(q.cuda(), out, pool, 0, tables.cuda(), start.cuda(), torch.tensor([400], dtype=torch.int32, device="cuda"), 1, 0,
                             D**-0.5, _junk_workspace(attention), 0, pages.cuda(), 148)
    want, tol = _oracle(rec[0], tables, q[:1], [1], [400], D**-0.5, pages=pages)
    assert ((out[:1].double().cpu() - want).abs() <= tol).all()
    assert (out[1:] == 7.0).all()


@pytest.mark.parametrize("max_q,split", [(70, 1), (70, 2), (65, None), (64, 1)])
def test_prefill_rows_beyond_max_q_len_inside_a_tile_are_left_alone(max_q, split):
    """A CTA has 64 tokens here: max_q_len ends inside its second tile."""
    q_lens, ctx_lens = [100, 3], [300, 900]
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, 8, 2, seed=74)
    out = _attend(pool, 0, tables, q, start, ctx_lens, max_q, 2, split)
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5, prefill=True)
    assert ((out - want).abs() <= tol)[list(range(max_q)) + [100, 101, 102]].all()
    assert (out[max_q:100] == 7.0).all()


@pytest.mark.parametrize("parts", [0, 3])
@pytest.mark.parametrize("front", [0, 2])
def test_sparse_rows_outside_the_call_are_left_alone(parts, front):
    """Rows in front of the first sequence, tokens beyond max_q_len (select_pages leaves their lists unset) and rows behind the last
    sequence, with places in the workspace that an earlier call may have left."""
    attention, _, _ = _ops()
    q_lens, ctx_lens = [3, 1, 2] + [0] * 40 + [2], [300, 90, 150] + [5] * 40 + [200]  # more sequences than a warp has lanes
    pool, rec, tables, q, start = _setup(q_lens, ctx_lens, 8, 2, seed=75, extra_rows=front + 2)
    start, rows = start + front, q.shape[0]
    pages = torch.arange(12, dtype=torch.int32).expand(rows, 2, 12).contiguous()
    c = torch.tensor(ctx_lens, dtype=torch.int32, device="cuda")
    live, at = [], front
    for n in q_lens:
        live += list(range(at, at + min(n, 1)))
        at += n
    want, tol = _oracle(rec[0], tables, q[front : front + sum(q_lens)], q_lens, ctx_lens, D**-0.5, pages=pages[front:])
    for junk in ((0, 2), (1, 2), (0, 3), (0, 1)):
        ws = attention.AttentionWorkspace(torch.device("cuda"))
        ws.ensure(16, 148, D)
        ws.part_o.fill_(1e4)
        ws.part_lse.fill_(3.0)
        ws.ensure_shared(256).copy_(torch.tensor(junk, dtype=torch.int32).repeat(256))
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
        attention._attention_kv4(q.cuda(), out, pool, 0, tables.cuda(), start.cuda(), c, 1, 0, D**-0.5, ws, 0, pages.cuda(), parts)
        got = out.double().cpu()
        rest = [r for r in range(rows) if r not in live]
        assert (got[rest] == 7.0).all(), junk
        of = [r - front for r in live]
        assert ((got[live] - want[of]).abs() <= tol[of]).all()


@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,split,bad", [
    ([3], [40], 8, 1, None, 38),            # few rows: the second of three new tokens
    ([3], [40], 8, 1, 0, 39),
    ([5, 2], [700, 90], 16, 2, 7, 698),     # pages of the items shared by seven CTAs
    ([9], [333], 14, 2, None, 330),         # 63 rows: four row tiles
    ([9], [333], 14, 2, 5, 325),
    ([4], [50], 32, 2, None, 48),           # sixteen heads per KV head
    ([20], [40], 8, 1, None, 30),           # tensor cores: one row tile
    ([64], [320], 8, 1, 1, 300),            # two row tiles
    ([64], [320], 8, 1, 3, 257),            # splits
    ([100], [100], 16, 2, None, 0),         # every row sees it
    ([100], [100], 16, 2, None, 50),
    ([70], [257], 2, 2, 1, 255),
    ([130], [130], 7, 1, None, 64),
])
def test_a_value_that_is_not_finite_stays_in_the_rows_that_see_it(q_lens, ctx_lens, hq, hkv, split, bad):
    """A NaN in the value of key `bad` of the first sequence, in one group of 16 dims: rows in front of it do not change, rows from it on
    have NaN in those dims and the formula in the others."""
    from daser_b200.ops import kv_ops

    _, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=91)
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5, prefill=max(q_lens) * hq // hkv >= 64)
    dirty, t, head, group = rec.clone(), bad % B, hkv - 1, 5
    dirty[0, tables[0, bad // B].long(), head, 2176 + (t // 8) * 64 + 8 * group + t % 8] = 0xFF
    got = _attend(kv_ops.PagedKV4Pool.from_tensors([dirty.cuda()]), 0, tables, q, start, ctx_lens, max(q_lens), hkv, split)
    sees = torch.zeros(q.shape, dtype=torch.bool)
    first, G = max(0, bad - (ctx_lens[0] - q_lens[0])), hq // hkv
    sees[first : q_lens[0], head * G : (head + 1) * G, 16 * group : 16 * group + 16] = True
    assert torch.isnan(got[sees]).all()
    assert ((got - want).abs() <= tol)[~sees].all(), (got - want)[~sees].abs().max()


def test_prefill_whose_maximum_is_never_raised():
    """The largest score comes first, so that P is replaced tile after tile while O is never touched in between: right, and the same each time."""
    _, _, kv_ops = _ops()
    ctx, q_len = 2500, 32
    _, rec, tables, q, start = _setup([q_len], [ctx], 8, 1, seed=76)
    g = torch.Generator().manual_seed(77)
    k = torch.randn(rec.shape[1], 1, B, D, generator=g) * 0.3
    q = (q.abs() + 0.1).to(torch.bfloat16)
    k[tables[0, 0].long(), 0, 0] = 1.0  # key 0: above all others
    rec = codec.pack_kv4_records(k, torch.randn(k.shape, generator=g))[None]
    pool = kv_ops.PagedKV4Pool.from_tensors([rec.cuda()])
    want, tol = _oracle(rec[0], tables, q, [q_len], [ctx], D**-0.5, prefill=True)
    first = None
    for _ in range(20):
        got = _attend(pool, 0, tables, q, start, [ctx], q_len, 1, 1)
        assert ((got - want).abs() <= tol).all()
        first = got if first is None else first
        assert torch.equal(got, first)


@pytest.mark.parametrize("q_lens,front,behind", [([1] * 32 + [2048], 0, 0), ([3] + [0] * 40 + [1, 7], 2, 3), ([2, 2, 2], 0, 2)])
def test_selection_in_a_step_of_unequal_sequences(q_lens, front, behind):
    """Decode steps beside a chunk of a prompt: the lists are those of the rows there are, not of sequences times the longest."""
    attention, _, _ = _ops()
    from daser_b200.ops import kv_ops

    g = torch.Generator().manual_seed(14)
    pages, width, n_pages, T = 300, 160, 8, sum(q_lens)
    ctx = [n + int(torch.randint(B, width * B - n, (1,), generator=g)) for n in q_lens]
    codes = torch.randint(-127, 128, (1, pages, 1, 2, D), dtype=torch.int8, generator=g)
    exps = torch.randint(-6, -2, (1, pages, 1), dtype=torch.int8, generator=g)
    tables = torch.stack([torch.randperm(pages, generator=g)[:width] for _ in q_lens]).to(torch.int32)
    q = torch.randn(front + T + behind, 4, D, generator=g).to(torch.bfloat16)
    start = torch.tensor([0] + torch.tensor(q_lens).cumsum(0).tolist(), dtype=torch.int32) + front
    got = attention.select_pages(q.cuda(), kv_ops.PageBounds(codes.cuda(), exps.cuda()), 0, tables.cuda(), start.cuda(),
                                 torch.tensor(ctx, dtype=torch.int32, device="cuda"), max(q_lens), max(ctx), n_pages).cpu()
    want = _select_oracle(q[front : front + T], codes[0], exps[0], tables, q_lens, ctx, n_pages, 1, 4)
    assert torch.equal(got[front : front + T], want)


@pytest.mark.parametrize("scale_byte_of_16ths", [11, 13, 15])
@pytest.mark.parametrize("q_len,ctx", [(1, 32768), (16, 32768), (2, 9000)])
def test_a_long_flat_tail_far_below_the_maximum_keeps_its_mass(scale_byte_of_16ths, q_len, ctx):
    """One loud key in every second page of the first 32 (each warp of a CTA meets one at once), the other keys 16.5, 19.5 or 22.5 below them in
    log2, all equal.  The loud keys' values are 0, the others' 1, so an output is the tail's share.

    P of the tail is 2^(7 - gap) in f16: off by 2^-11 of itself or, below 2^-14, by 2^-25; scores, whole multiples of 2^-7 here, are exact up to
    their fp32 sum (2^-18 of them); ex2 and the sums in fp32 2^-14 in all; then one rounding to bf16."""
    import math

    from daser_b200.ops import attention, kv_ops

    n = -(-ctx // B)
    k, v = torch.zeros(n, 1, B, D), torch.ones(n, 1, B, D)
    loud = 6 * scale_byte_of_16ths / 64  # absmax 6 s with s = m / 64, four bits: exact in the format
    k[0:32:2, 0, 0], v[0:32:2, 0, 0] = loud, 0.0
    rec = codec.pack_kv4_records(k, v)[None]
    kk, vv = codec.unpack_kv4_records(rec[0])
    assert kk.max() == loud and (kk.unique().numel(), vv.unique().numel()) == (2, 2)
    q = torch.ones(q_len, 8, D).to(torch.bfloat16)
    tables = torch.arange(n, dtype=torch.int32)[None].cuda()
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    attention.paged_attention(q.cuda(), out, kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables, torch.tensor([0, q_len], **i32),
                              torch.tensor([ctx], **i32), q_len, ctx, 1, 0.125 / math.log2(math.e), None, nsplit=0 if q_len < 8 else 1)
    gap = 0.125 * D * loud
    one = float(vv.max())
    for t in range(q_len):
        tail = ctx - q_len + t + 1 - 16
        share = tail * 2.0**-gap / (16 + tail * 2.0**-gap)
        rel = max(2.0**-11, 2.0**-25 * 2.0 ** (gap - 7)) + gap * 2.0**-18 + 2.0**-14 + BF16_HALF
        assert ((out[t].double().cpu() - one * share).abs() <= rel * one * share).all(), (gap, t, out[t, 0, 0].item() / (one * share))


@pytest.mark.parametrize("size,key,scale", [(2e5, 2e-5, 1.0), (1e30, 4e-6, 1e-25), (1.0, 3e4, 1e-6), (1e-30, 5.0, 1e29), (5e37, 4e-6, 1e-33)])
@pytest.mark.parametrize("q_len,split", [(1, None), (1, 5), (5, 0), (16, None), (40, 2)])
def test_queries_beyond_the_range_of_f16(q_len, split, size, key, scale):
    """Scaled queries far above 65504 and far below 2^-14 (where f16 has fewer bits): each row as the formula has it.  One row of ordinary
    size, one of zeros among them."""
    from daser_b200.ops import attention, kv_ops

    ctx = 300
    _, rec, tables, q, start = _setup([q_len], [ctx], 8, 1, seed=95)
    g = torch.Generator().manual_seed(96)
    k, v = torch.randn(rec.shape[1], 1, B, D, generator=g) * key, torch.randn(rec.shape[1], 1, B, D, generator=g)
    rec = codec.pack_kv4_records(k, v)[None]
    q = (q.float() * size / 2).to(torch.bfloat16)
    q[0, 3] = 0
    q[-1, 5] = torch.randn(D, generator=g).to(torch.bfloat16)
    assert torch.isfinite(q.float()).all()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    attention.paged_attention(q.cuda(), out, kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables.cuda(), start.cuda(), torch.tensor([ctx], **i32),
                              q_len, ctx, 1, scale, None, nsplit=split)
    want, tol = _oracle(rec[0], tables, q, [q_len], [ctx], scale, prefill=q_len > 7)
    got = out.double().cpu()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("q_len,split", [(1, None), (3, 4), (16, None)])
def test_small_queries_against_large_keys(q_len, split):
    """A scaled query of 2.5 * 2^-24 is 2 * 2^-24 in f16, a fifth less: values that have the sign of their key's score show it."""
    import math

    from daser_b200.ops import attention, kv_ops

    ctx, scale = 300, 2.5 * 2.0**-24 / math.log2(math.e)
    _, rec, tables, q, start = _setup([q_len], [ctx], 8, 1, seed=97)
    g = torch.Generator().manual_seed(98)
    sign = torch.where(torch.randn(D, generator=g) > 0, 1.0, -1.0)
    q = sign.expand(q.shape).to(torch.bfloat16).contiguous()
    k = torch.randn(rec.shape[1], 1, B, D, generator=g) * 1e4 + sign * 4e3 * torch.randn(rec.shape[1], 1, B, 1, generator=g)
    v = torch.sign((k * sign).sum(-1, keepdim=True)).expand(k.shape)
    rec = codec.pack_kv4_records(k, v)[None]
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    attention.paged_attention(q.cuda(), out, kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables.cuda(), start.cuda(), torch.tensor([ctx], **i32),
                              q_len, ctx, 1, scale, None, nsplit=split)
    want, tol = _oracle(rec[0], tables, q, [q_len], [ctx], scale, prefill=q_len > 7)
    got = out.double().cpu()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("q_len,split", [(1, None), (1, 5), (2, 0), (16, None), (40, 2)])
def test_a_query_that_is_not_finite_is_nan_in_its_row_alone(q_len, split):
    """Also where every score is minus infinity, which is not the same as no key."""
    from daser_b200.ops import kv_ops

    ctx = 300
    _, rec, tables, q, start = _setup([q_len], [ctx], 8, 1, seed=99)
    k, v = codec.unpack_kv4_records(rec[0])
    rec = codec.pack_kv4_records(-k.abs() - 0.5, v)[None]  # no key of 0
    want, tol = _oracle(rec[0], tables, q, [q_len], [ctx], D**-0.5, prefill=q_len > 7)
    q[0, 3, 77], q[-1, 6, 5] = float("inf"), float("nan")
    q[0, 1, 0] = float("-inf")
    got = _attend(kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables, q, start, [ctx], q_len, 1, split)
    bad = torch.zeros(q_len, 8, dtype=torch.bool)
    bad[0, 1] = bad[0, 3] = bad[-1, 6] = True
    assert torch.isnan(got[bad]).all() and ((got - want).abs() <= tol)[~bad].all()


@pytest.mark.parametrize("parts", [0, 7])
def test_sparse_queries_beyond_the_range_of_f16(parts):
    attention, _, _ = _ops()
    from daser_b200.ops import kv_ops

    q_lens, ctx_lens = [1, 2], [500, 230]
    _, rec, tables, q, start = _setup(q_lens, ctx_lens, 32, 2, seed=100)
    g = torch.Generator().manual_seed(101)
    k, v = torch.randn(rec.shape[1], 2, B, D, generator=g) * 2e-5, torch.randn(rec.shape[1], 2, B, D, generator=g)
    rec = codec.pack_kv4_records(k, v)[None]
    q = (q.float() * 1e6).to(torch.bfloat16)
    q[1, 17:30] *= 1e-6
    pages = torch.full((3, 2, 12), -1, dtype=torch.int32)
    pages[:, 0, :9] = torch.tensor([0, 2, 3, 5, 7, 8, 11, 13, 14])
    pages[:, 1, :5] = torch.tensor([1, 4, 6, 10, 12])
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    attention._attention_kv4(q.cuda(), out, kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables.cuda(), start.cuda(),
                             torch.tensor(ctx_lens, dtype=torch.int32, device="cuda"), 2, 0, D**-0.5, None, 0, pages.cuda(), parts)
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5, pages=pages)
    assert ((out.double().cpu() - want).abs() <= tol).all()


def test_first_calls_of_a_process_from_several_threads():
    """A kernel's shared memory has to be asked for once per device before its first launch: by whichever thread is first."""
    import os
    import subprocess
    import sys

    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kv4_threads_worker.py")
    done = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_row_strides_of_the_projections():
    """One row of a tensor whose rows are off the vector grid is taken; rows that are one row repeated are read, but not zeroed under one another."""
    _, ew, kv_ops = _ops()
    hq, hkv = 8, 2
    cols = (hq + 2 * hkv) * D
    pool = kv_ops.PagedKV4Pool.zeros(1, 2, hkv, "cuda")
    cos_sin = kv_ops.rope_table(32, inv_freq_table(D, 10000.0), "cuda")
    q_out = torch.zeros(3, hq, D, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(102)
    wide = torch.randn(3, cols + 3, generator=g).cuda()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    ew.rope_kv_write(wide[:1, :cols], i(3), i(5).long(), cos_sin, q_out, hq, hkv, D, B, pool, 0)
    want = _rope_ref(wide[:1, : hq * D].float().reshape(1, hq, D).cpu(), cos_sin.cpu()[3:4]).to(torch.bfloat16)
    assert torch.equal(q_out[:1].cpu(), want)
    k, v = kv_ops.kv_read(pool, 0, i(5).long())
    assert torch.equal(v.float().cpu()[0], codec.dequantize_fp4b16(*codec.quantize_fp4b16(wide[0, (hq + hkv) * D : cols].reshape(hkv, D).to(torch.bfloat16).float().cpu())))
    with pytest.raises(Exception):
        ew.rope_kv_write(wide[:3, :cols], i(3, 3, 3), i(5, 6, 7).long(), cos_sin, q_out, hq, hkv, D, B, pool, 0)  # three such rows
    same = torch.randn(1, cols, generator=g).cuda()
    rep = same.expand(3, cols)
    ew.rope_kv_write(rep, i(3, 3, 3), i(5, 6, 7).long(), cos_sin, q_out, hq, hkv, D, B, pool, 0)
    assert torch.equal(q_out[0], q_out[2])
    before = same.clone()
    with pytest.raises(ValueError):
        ew.rope_kv_write(rep, i(3, 3, 3), i(5, 6, 7).long(), cos_sin, q_out, hq, hkv, D, B, pool, 0, zero_after=True)
    assert torch.equal(same, before)


@pytest.mark.parametrize("level", [-1e4, -200.0, -100.0, 100.0, 1e4])
@pytest.mark.parametrize("q_lens,ctx_lens,hq,hkv,split", [([1], [300], 8, 1, None), ([1, 1], [300, 40], 16, 2, 5), ([1], [900], 16, 1, 0), ([3], [70], 8, 1, None),
                                                          ([20], [200], 8, 1, 1), ([40], [300], 8, 1, 3)])
def test_scores_that_all_lie_far_from_zero(q_lens, ctx_lens, hq, hkv, split, level):
    """Every score of a row is near `level` (in log2): the first maximum a warp meets is far above or below what it starts from."""
    from daser_b200.ops import kv_ops

    _, rec, tables, q, start = _setup(q_lens, ctx_lens, hq, hkv, seed=110)
    g = torch.Generator().manual_seed(111)
    k = torch.randn(rec.shape[1], hkv, B, D, generator=g)
    k[..., :16] = level / (16 * 0.1275)  # a group of 16 dims carries the level, the others the differences
    q = (q.float() / 1.3).to(torch.bfloat16)
    q[..., :16] = 1.0
    rec = codec.pack_kv4_records(k, torch.randn(k.shape, generator=g))[None]
    got = _attend(kv_ops.PagedKV4Pool.from_tensors([rec.cuda()]), 0, tables, q, start, ctx_lens, max(q_lens), hkv, split)
    want, tol = _oracle(rec[0], tables, q, q_lens, ctx_lens, D**-0.5, prefill=max(q_lens) * hq // hkv >= 64)
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
