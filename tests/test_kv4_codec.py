"""The 4-bit format on the CPU: codec, record layout, and what the operators of the 4-bit pool refuse."""

import ctypes as C
import math

import pytest
import torch

from daser_b200.kv import codec

MAGS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest_even(y):
    """The e2m1 value nearest to ``y`` (a Python float), the even code at a tie."""
    a = min(abs(y), 6.0)
    best = min(range(8), key=lambda i: (abs(MAGS[i] - a), i % 2))
    return math.copysign(MAGS[best], y)


def test_every_scale_byte_and_code_decodes_to_its_definition():
    scales = torch.arange(256, dtype=torch.uint8)
    got = codec.fp4_scale_values(scales).tolist()
    for b in range(248):
        e, m = b >> 3, b & 7
        assert got[b] == (m * 2.0**-17 if e == 0 else (1 + m / 8) * 2.0 ** (e - 15))
    assert math.isinf(got[248]) and all(math.isnan(x) for x in got[249:])
    codes = torch.tensor([i | (15 - i) << 4 for i in range(16)], dtype=torch.uint8)[None, :8]
    vals = codec.dequantize_fp4b16(codes, torch.tensor([[120]], dtype=torch.uint8))[0].tolist()  # byte 120: scale 1
    table = MAGS + [-x for x in MAGS]
    assert vals[0::2] == table[:8] and vals[1::2] == table[:7:-1]


@pytest.mark.parametrize("mant", range(8, 16))
def test_rounding_is_to_nearest_with_ties_to_the_even_code_for_every_scale(mant):
    s = mant / 8.0
    ys = [0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, -5.0, 6.0]
    x = torch.tensor([y * s for y in ys])
    codes, byte = codec.quantize_fp4b16(x)
    assert codec.fp4_scale_values(byte).item() == s
    assert (codec.dequantize_fp4b16(codes, byte) / s).tolist() == [_nearest_even(y) for y in ys]


def test_error_is_within_half_a_step_of_the_scale():
    torch.manual_seed(0)
    x = torch.randn(4096, 64) * torch.exp(3 * torch.randn(4096, 1))
    codes, byte = codec.quantize_fp4b16(x)
    y = codec.dequantize_fp4b16(codes, byte)
    g, r = x.view(4096, 4, 16).double(), y.view(4096, 4, 16).double()
    s = codec.fp4_scale_values(byte).double().unsqueeze(-1)
    amax = g.abs().amax(-1, keepdim=True)
    # the scale: four significant bits (half a step: 2^-4) of an f16 (2^-11) of absmax * fl(1/6) (2^-23); below 2^-14, where f16 is
    # subnormal, scales are multiples of 2^-17 (half a step: 2^-18) of f16 multiples of 2^-24 (2^-25); at most 10240
    ideal = (amax / 6).clamp(max=10240)
    assert ((s - ideal).abs() <= torch.clamp((2.0**-4 + 2.0**-10) * ideal, min=2.0**-18 + 2.0**-24)).all()
    s = s.clamp(min=2.0**-300)  # a scale of zero holds zeros: the error is the value itself
    q = g.abs() / s
    half = torch.where(q <= 2, 0.25, torch.where(q <= 4, 0.5, 1.0)) * s
    assert ((g - r).abs() <= torch.maximum(half, (q - 6).clamp(min=0) * s) * (1 + 2.0**-20)).all()


def test_zero_tiny_huge_and_not_finite_groups():
    rows = torch.zeros(6, 16)
    rows[1] = 1e-7            # rounds to nothing
    rows[2, 3] = 3.0e38       # saturates
    rows[3, 5] = float("inf")
    rows[4, 7] = float("nan")
    rows[5] = 2.0**-17 * 6    # the smallest scale
    rows[5, 0] = -rows[5, 1]
    codes, byte = codec.quantize_fp4b16(rows)
    y = codec.dequantize_fp4b16(codes, byte)
    assert (y[0] == 0).all() and (y[1] == 0).all()
    assert y[2, 3] == 6 * codec.FP4_MAX_SCALE and torch.isfinite(y[2]).all()
    assert byte[3].item() == 255 and byte[4].item() == 255 and torch.isnan(y[3:5]).all()
    assert torch.equal(y[5], rows[5])


def test_values_of_the_format_survive_another_quantisation_and_bf16():
    torch.manual_seed(1)
    y = codec.dequantize_fp4b16(*codec.quantize_fp4b16(torch.randn(512, 128)))
    assert torch.equal(y.to(torch.bfloat16).float(), y)
    assert torch.equal(codec.dequantize_fp4b16(*codec.quantize_fp4b16(y)), y)


def test_record_layout_by_hand():
    k, v = torch.zeros(16, 128), torch.zeros(16, 128)
    k[3, 37] = 6.0    # token 3, group 2, an odd dim: high half of byte 37 // 2
    v[11, 66] = -3.0  # token 11, group 4, dim 2 of the group: low half
    rec = codec.pack_kv4_records(k, v)
    assert rec.shape == (2304,)
    want = torch.zeros(2304, dtype=torch.uint8)
    want[3 * 64 + 18] = 7 << 4
    want[1024 + 512 + 4 * 64 + 3 * 8 + 1] = 15
    want[2048 + 3 * 8 + 2] = 120       # scale 1
    want[2176 + 64 + 4 * 8 + 3] = 112  # scale 0.5
    # negative zeros keep their sign bit nowhere here: all other values are +0
    assert torch.equal(rec, want)
    torch.manual_seed(2)
    k, v = torch.randn(3, 2, 16, 128), torch.randn(3, 2, 16, 128)
    rk, rv = codec.unpack_kv4_records(codec.pack_kv4_records(k, v))
    assert torch.equal(rk, codec.dequantize_fp4b16(*codec.quantize_fp4b16(k)))
    assert torch.equal(rv, codec.dequantize_fp4b16(*codec.quantize_fp4b16(v)))


# -- refusals ----------------------------------------------------------------------------


def test_pool_and_bounds_refuse_other_shapes():
    from daser_b200.ops import kv_ops

    ok = torch.zeros(2, 5, 3, 2304, dtype=torch.uint8)
    pool = kv_ops.PagedKV4Pool.from_tensors([ok])
    assert (pool.num_layers, pool.num_blocks, pool.heads_per_rank, pool.n_ranks) == (2, 5, 3, 1)
    for bad in (ok[..., :2288], ok.to(torch.int8), ok[0], ok.transpose(2, 3)):
        with pytest.raises(ValueError):
            kv_ops.PagedKV4Pool.from_tensors([bad])
    with pytest.raises(ValueError):
        kv_ops.PagedKV4Pool.from_tensors([ok, ok[:, :4]])
    with pytest.raises(ValueError):  # records off the 16-byte grid
        kv_ops.PagedKV4Pool.from_tensors([torch.zeros(2 * 2305 + 8, dtype=torch.uint8)[8:].as_strided((1, 2, 1, 2304), (2304, 2305, 2304, 1))])
    with pytest.raises(ValueError):
        kv_ops.PagedKV4Pool.from_tensors([ok] * 9)
    codes, exps = torch.zeros(2, 5, 3, 2, 128, dtype=torch.int8), torch.zeros(2, 5, 3, dtype=torch.int8)
    kv_ops.PageBounds(codes, exps)
    for c, e in ((codes[..., :64], exps), (codes, exps[:1]), (codes.float(), exps), (codes.transpose(1, 2), exps.transpose(1, 2))):
        with pytest.raises(ValueError):
            kv_ops.PageBounds(c, e)


def test_operators_refuse_cpu_tensors_instead_of_launching():
    from daser_b200.ops import attention, elementwise, kv_ops

    pool = kv_ops.PagedKV4Pool.from_tensors([torch.zeros(1, 4, 2, 2304, dtype=torch.uint8)])
    bounds = kv_ops.PageBounds.for_pool(pool)
    i32, q = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    tables = torch.zeros(1, 4, dtype=torch.int32)
    calls = [
        lambda: kv_ops.kv_read(pool, 0, torch.zeros(1, dtype=torch.int64)),
        lambda: kv_ops.update_page_bounds(pool, bounds, 0, tables, i32, i32[:1], 1),
        lambda: kv_ops.quantize_fp4b16(q),
        lambda: kv_ops.dequantize_fp4b16(torch.zeros(8, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8)),
        lambda: attention.paged_attention(q, q, pool, 0, tables, i32, i32[:1], 1, 16, 2, 1.0, None),
        lambda: attention.select_pages(q, bounds, 0, tables, i32, i32[:1], 1, 64, 8),
        lambda: attention.sparse_paged_attention(q, q, pool, 0, tables, i32, i32[:1], torch.zeros(1, 2, 4, dtype=torch.int32), 1, 1.0),
        lambda: elementwise.rope_kv_write(torch.zeros(1, 12 * 128), i32[:1], torch.zeros(1, dtype=torch.int64), torch.zeros(4, 128), q, 8, 2,
                                          128, 16, pool, 0),
    ]
    for call in calls:
        with pytest.raises(ValueError):
            call()


def _c_pool(**kw):
    from daser_b200.ops import _lib

    p = _lib.KV4Pool()
    p.records[0] = 1 << 20  # never dereferenced on the host
    p.stride_layer, p.stride_block, p.stride_head = 4 * 2 * 2304, 2 * 2304, 2304
    p.num_layers, p.num_blocks, p.n_ranks, p.heads_per_rank = 1, 4, 1, 2
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(n_ranks=0), -1), (dict(n_ranks=9), -1), (dict(num_blocks=0), -1), (dict(heads_per_rank=0), -1), (dict(num_layers=0), -1),
    (dict(stride_block=2 * 2304 + 8), -2), (dict(stride_head=2305), -2), (dict(stride_layer=24), -2),
])
def test_c_entry_points_refuse_bad_pools(change, code):
    """Every entry point checks the pool before it launches: the code comes back without a GPU."""
    from daser_b200.ops import _lib

    pool = _c_pool(**change)
    p = C.addressof(pool)
    a = 1 << 21  # an aligned address that nothing reads
    assert _lib.kv4_fn("daser_kv4_read")(p, 0, 0, a, a, a, 1, None) == code
    assert _lib.kv4_fn("daser_rope_kv4_write")(a, 1, 1536, a, a, a, 8, a, 1, 8, 2, p, 0, 0, 0, None, None, 0.0, None) == code
    assert _lib.kv4_fn("daser_kv4_page_bounds")(p, 0, 0, a, a, a, 4, a, a, 1, 1, None) == code
    assert _lib.kv4_fn("daser_paged_attention_kv4")(a, a, a, a, a, p, 0, 0, a, 4, a, a, 1, 1, 1, 8, 1, 4, 1.0, None) == code
    assert _lib.kv4_fn("daser_sparse_attention_kv4")(a, a, a, a, a, p, 0, 0, a, 4, a, a, 1, 1, 1, 8, a, 4, 2, 1.0, None) == code


def test_c_entry_points_refuse_bad_arguments():
    from daser_b200.ops import _lib

    pool = _c_pool()
    p, a = C.addressof(pool), 1 << 21
    read, att = _lib.kv4_fn("daser_kv4_read"), _lib.kv4_fn("daser_paged_attention_kv4")
    assert read(p, 1, 0, a, a, a, 1, None) == -1 and read(p, -1, 0, a, a, a, 1, None) == -1  # layer
    assert read(p, 0, 1, a, a, a, 1, None) == -1                                              # rank
    assert read(p, 0, 0, a, a + 8, a, 1, None) == -2 and read(p, 0, 0, None, a, a, 1, None) == -1
    write = _lib.kv4_fn("daser_rope_kv4_write")
    ok = [a, 1, 1536, a, a, a, 8, a, 1, 8, 2, p, 0, 0, 0, None, None, 0.0, None]
    for at, bad, code in ((10, 3, -1), (8, -1, -1), (6, 0, -1), (0, None, -1), (7, None, -1), (2, 1537, -2), (0, a + 4, -2), (15, a, -1)):
        args = list(ok)
        args[at] = bad
        assert write(*args) == code, at
    ok = [a, a, a, a, a, p, 0, 0, a, 4, a, a, 1, 1, 1, 8, 2, 4, 1.0, None]
    for at, bad, code in ((15, 7, -1), (15, 34, -2), (16, 1, -1), (16, -1, -1), (16, 257, -3), (2, None, -1), (4, None, -1), (9, 0, -1),
                          (0, a + 2, -2), (12, -1, -1)):
        args = list(ok)
        args[at] = bad
        assert att(*args) == code, at
    sparse = _lib.kv4_fn("daser_sparse_attention_kv4")
    assert sparse(a, a, a, a, a, p, 0, 0, a, 4, a, a, 1, 1, 1, 8, a, 9, 1, 1.0, None) == -1  # one CTA has nothing to share
    assert sparse(a, a, a, a, a, p, 0, 0, a, 4, a, a, 1, 1, 1, 8, a, 0, 2, 1.0, None) == -1
    prefill = [a, a, a, a, None, p, 0, 0, a, 4, a, a, 1, 64, 64, 8, 2, 4, 1.0, None]  # 4 heads x 64 queries: splits
    for at, bad in ((16, 0), (17, 0)):
        args = list(prefill)
        args[at] = bad
        assert att(*args) == -1, at
    sel = _lib.kv4_fn("daser_select_pages_kv4")
    ok = [a, a, a, 0, 4, a, 4, a, a, 1, 1, 1, 8, 2, a, 4, a, 8, 1, 4, None]
    for at, bad, code in ((17, 4, -1), (18, -1, -1), (19, 0, -1), (12, 9, -1), (12, 34, -2), (1, a + 4, -2), (15, 0, -1), (11, 70000, -3)):
        args = list(ok)
        args[at] = bad
        assert sel(*args) == code, at
    # nothing to do is not an error, and launches nothing
    assert read(p, 0, 0, None, None, None, 0, None) == 0
    assert att(a, a, None, None, None, p, 0, 0, a, 4, a, a, 0, 0, 0, 8, 0, 0, 1.0, None) == 0


@pytest.mark.parametrize("off,code", [((2, 0, 0), -2), ((8, 0, 0), -2), ((0, 4, 0), -2), ((0, 1, 0), -2)])
def test_the_codec_refuses_addresses_off_its_vectors(off, code):
    """bf16 values are read 16 bytes at a time, codes 8: a view that starts elsewhere is refused before a launch."""
    from daser_b200.ops import _lib

    a = 1 << 21
    x, codes, scales = a + off[0], a + off[1], a + off[2]
    assert _lib.kv4_fn("daser_quant_fp4b16")(x, codes, scales, 64, None) == code
    assert _lib.kv4_fn("daser_dequant_fp4b16")(codes, scales, x, 64, None) == code
    for args in ((None, a, a), (a, None, a), (a, a, None)):
        assert _lib.kv4_fn("daser_quant_fp4b16")(*args, 64, None) == -1
        assert _lib.kv4_fn("daser_dequant_fp4b16")(*args, 64, None) == -1


def test_plans_cover_the_context():
    from daser_b200.ops import attention

    for seqs in (1, 3, 64):
        for heads, group in ((1, 8), (8, 8), (8, 5), (2, 16), (4, 1)):
            for q in (1, 2, 9, 64, 500):
                for pages in (0, 1, 2, 15, 17, 129, 8192, 65536):
                    n, per = attention.plan_kv4(seqs, heads, q, group, pages, rows=seqs * q * heads * group)
                    if q * group >= 64:
                        assert n >= 1 and per >= 1 and n * per >= pages
                        assert n == 1 or (n - 1) * per < pages  # no split is empty for the longest context
                        assert n == 1 or n * seqs * q * heads * group <= attention.MAX_ROW_SPLITS
                    else:
                        assert n == 0 or 2 <= n <= 148


def test_outgrown_workspace_buffers_stay_alive():
    from daser_b200.ops import attention

    ws = attention.AttentionWorkspace("cpu")
    ws.ensure(4, 2, 128)
    first = ws.part_o
    ws.ensure(40, 2, 128)
    assert ws.part_o is not first and any(t is first for t in ws._outgrown)
    assert ws.ensure_scores(10).numel() == 10 and ws.ensure_scores(5).numel() == 10


def test_a_workspace_keeps_what_it_outgrew_and_not_more_than_that():
    """Captured graphs may hold the smaller buffers' addresses; growing in small steps must not pile them up."""
    from daser_b200.ops import attention

    ws = attention.AttentionWorkspace(torch.device("cpu"))
    for rows in range(1, 2000, 3):
        ws.ensure(rows, 2, 4)
        ws.ensure_shared(rows)
        assert ws.ensure_scores(rows).numel() >= rows
        assert ws.part_lse.numel() >= 2 * rows and ws.part_o.numel() == 4 * ws.part_lse.numel() and ws.shared.numel() >= 2 * rows
    held = sum(t.numel() for t in ws._outgrown)
    assert held <= ws.part_o.numel() + ws.part_lse.numel() + ws.shared.numel() + ws.scores.numel()
    assert all(t is not None for t in ws._outgrown)


def test_chunks_of_a_4_bit_engine_are_found_by_engines_of_its_kind_alone(live_plane):
    """Two schedulers on one store, as GpuRagEngine makes them for the two formats."""
    from daser_b200.connector.core import SchedulerHalf
    from daser_b200.hashing import hash_tokens

    fp8 = SchedulerHalf(live_plane.socket_path, 16, "m")
    kv4 = SchedulerHalf(live_plane.socket_path, 16, "m+fp4b16", also_reads=("m",))
    try:
        mine, theirs = list(range(32)), list(range(100, 148))
        for half, tokens in ((kv4, mine), (fp8, theirs)):
            spec = half.reserve_chunk_store("s", tokens, list(range(3)))
            half._ipc.commit_chunk(spec.chunk_key)
            half.request_finished("s")
        places = [(hash_tokens(mine), 0), (hash_tokens(theirs), 32), (hash_tokens([7] * 16), 80)]
        got8, got4 = fp8.plan_chunk_loads("a", places), kv4.plan_chunk_loads("b", places)
        assert [s is not None for s in got8] == [False, True, False]
        assert [s is not None for s in got4] == [True, True, False]
        assert got4[0].num_slots == 2 and got4[1].num_slots == 3 and got4[1].start_slot == got8[1].start_slot
        combo = [mine, list(range(200, 216))]
        spec = fp8.reserve_chunk_store("c", [t for c in combo for t in c], [0, 1, 2])
        fp8._ipc.commit_chunk(spec.chunk_key)
        assert len(kv4.merge_composed(combo)) == len(fp8.merge_composed(combo)) == 1
    finally:
        fp8.close()
        kv4.close()
