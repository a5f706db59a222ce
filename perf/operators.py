"""The 4-bit KV cache and the operators that write, read and attend over it.

Four families of cases, each one pass through what a serving program calls:

* ``write``    rotate a step's queries and keys, write its keys and values into the 4-bit paged pool and read
               the same tokens back (``rope_kv_write`` + ``kv_read``);
* ``restore``  stored chunk images (block-scaled fp8) into 4-bit pages at new positions, and pages back out to
               raw bf16 images (``kv_restore`` + ``kv_save``);
* ``attend``   causal paged attention over 4-bit pages: decode steps and chunked prefill (``paged_attention``);
* ``sparse``   the step's key bounds, the pages that a bound on the scores selects for every query and KV head,
               and attention over those pages (``update_page_bounds`` + ``select_pages`` +
               ``sparse_paged_attention``).

The format (``fp4b16``): groups of 16 consecutive dims share one scale.  A value is held as e2m1 (sign, two
exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), a scale as the upper 8 of the 15 magnitude bits of an
f16 (5 exponent bits, 3 mantissa bits, no sign); scale = absmax / 6.  A page of 16 tokens of one KV head is
one record of 2304 bytes: K codes [token][64 bytes], V codes [token / 8][group][token % 8][8 bytes], K scales
[token][group], V scales [token / 8][group][token % 8].

``run`` computes in plain torch operations where ``own`` is false, with the framework's kernels where it is true.
"""

import math

import torch

own = False

D, B, G16 = 128, 16, 16
RECORD = 2304
DEV = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- the cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # a decode step of 64 running sequences of a 64 / 8 head model: split-K accumulators in, five padded rows
        {"name": "write decode 64", "kind": "write", "tokens": 64, "pad": 5, "hq": 64, "hkv": 8, "f32": True},
        # a prefill step of a 32 / 8 head model, bf16 projections
        {"name": "write prefill 4096", "kind": "write", "tokens": 4096, "pad": 0, "hq": 32, "hkv": 8, "f32": False},
        # one retrieved chunk of 301 tokens, one group of four layers
        {"name": "restore chunk", "kind": "restore", "slots": 19, "layers": 4, "hkv": 8},
        # a request's whole context of about 3.3k tokens, one group of ten layers
        {"name": "restore request", "kind": "restore", "slots": 208, "layers": 10, "hkv": 8},
        # one short sequence: the latency of a call
        {"name": "decode one short", "kind": "attend", "seqs": 1, "q_len": 1, "lo": 327, "hi": 327, "hq": 64, "hkv": 8},
        # one of eight tensor-parallel ranks (8 query heads, 1 KV head), a few very long sequences
        {"name": "decode long shard", "kind": "attend", "seqs": 4, "q_len": 1, "lo": 50001, "hi": 120007, "hq": 8, "hkv": 1},
        # a decode batch with ragged contexts of 4k to 32k
        {"name": "decode batch 32", "kind": "attend", "seqs": 32, "q_len": 1, "lo": 4096, "hi": 32768, "hq": 64, "hkv": 8},
        # the question of a retrieval request over its restored chunks
        {"name": "prefill question", "kind": "attend", "seqs": 1, "q_len": 64, "lo": 3328, "hi": 3328, "hq": 64, "hkv": 8},
        # a chunk of a long prompt
        {"name": "prefill chunk", "kind": "attend", "seqs": 1, "q_len": 2048, "lo": 8192, "hi": 8192, "hq": 32, "hkv": 8},
        # a short context on one tensor-parallel rank: the latency of the three calls
        {"name": "sparse short shard", "kind": "sparse", "seqs": 2, "q_len": 1, "lo": 4001, "hi": 5003, "hq": 8, "hkv": 1, "pages": 64},
        # one user with a book in the context
        {"name": "sparse one long", "kind": "sparse", "seqs": 1, "q_len": 1, "lo": 131072, "hi": 131072, "hq": 32, "hkv": 8, "pages": 256},
        # a batch of long-context decodes
        {"name": "sparse batch 16", "kind": "sparse", "seqs": 16, "q_len": 1, "lo": 16384, "hi": 65536, "hq": 64, "hkv": 8, "pages": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "restore", "attend", "attend", "sparse"))
    hq, hkv = rng.choice(((64, 8), (32, 8), (8, 1), (16, 2), (4, 4), (16, 1), (40, 8)))
    if kind == "write":
        tokens = _log(rng, 1, 4000)
        return {"kind": kind, "tokens": tokens, "pad": rng.randrange(0, 1 + tokens // 8), "hq": min(hq, 32) if hkv != 8 else hq, "hkv": hkv,
                "f32": rng.random() < 0.5}
    if kind == "restore":
        return {"kind": kind, "slots": _log(rng, 1, 200), "layers": rng.randint(1, 10), "hkv": rng.choice((1, 2, 4, 8))}
    if kind == "attend":
        if rng.random() < 0.5:
            seqs, q_len, hi = _log(rng, 1, 32), rng.choice((1, 1, 1, 2, 3, 5)), _log(rng, 64, 32000)
        else:
            seqs, q_len, hi = rng.randint(1, 3), _log(rng, 9, 400), _log(rng, 800, 5000)
        return {"kind": kind, "seqs": seqs, "q_len": q_len, "lo": max(q_len, hi // rng.randint(1, 6)), "hi": hi, "hq": hq, "hkv": hkv}
    hi = _log(rng, 1500, 100000)
    seqs = max(1, min(_log(rng, 1, 16), 500000 // hi))
    return {"kind": kind, "seqs": seqs, "q_len": rng.choice((1, 1, 1, 2, 4)), "lo": hi // rng.randint(1, 4), "hi": hi, "hq": hq, "hkv": hkv,
            "pages": rng.choice((17, 32, 64, 128, 256))}


SINK, RECENT = 1, 4  # pages that every sparse query reads: the first, and the last ones


def _lens(case):
    """Context and query lengths of every sequence, ragged, from the case alone."""
    n, lo, hi, q = case["seqs"], case["lo"], case["hi"], case["q_len"]
    ctx = [hi if n == 1 else lo + (hi - lo) * ((i * 7) % n if math.gcd(7, n) == 1 else i) // (n - 1) for i in range(n)]
    ql = [max(1, q - (i * 5) % max(1, q // 3)) if i else q for i in range(n)]
    return ctx, [min(a, b) for a, b in zip(ql, ctx)]


def work(case):
    hkv, rec = case["hkv"], RECORD
    if case["kind"] == "write":
        t, live = case["tokens"], case["tokens"] - case["pad"]
        n = case["hq"] + 2 * hkv
        moved = t * n * D * (4 if case["f32"] else 2) + t * case["hq"] * D * 2  # projections in, queries out
        moved += 2 * live * hkv * 2 * 72 + t * hkv * 2 * D * 2  # 4-bit rows written and read back, values out
        return {"bytes": moved, "flops": 10 * t * n * D}
    if case["kind"] == "restore":
        n = case["slots"] * case["layers"] * hkv
        return {"bytes": n * (2 * B * D * 1.25 + 2 * rec + 2 * B * D * 2), "flops": 10 * n * 2 * B * D}
    ctx, ql = _lens(case)
    qo = sum(ql) * case["hq"] * D * 4
    if case["kind"] == "attend":
        pages = sum(-(-c // B) for c in ctx)
        pairs = sum(q * (c - q) + q * (q + 1) // 2 for c, q in zip(ctx, ql))
        return {"bytes": qo + pages * hkv * rec, "flops": 4 * D * case["hq"] * pairs}
    pages = sum(-(-c // B) for c in ctx)  # a sequence's bounds are read once however many queries it has
    chosen = sum(min(case["pages"], -(-c // B)) * q for c, q in zip(ctx, ql))
    scored = sum(-(-c // B) * q for c, q in zip(ctx, ql))
    return {"bytes": qo + pages * hkv * 257 + chosen * hkv * rec, "flops": hkv * scored * 4 * D + 4 * D * case["hq"] * chosen * B}


# ---- the format --------------------------------------------------------------------------------------------------


def _quantize(x):
    """fp32 ``[..., 128]`` -> (codes uint8 ``[..., 128]``, scale bytes uint8 ``[..., 8]``)."""
    g = x.reshape(*x.shape[:-1], D // G16, G16)
    amax = g.abs().amax(-1)
    t = (amax * torch.full((), 1.0 / 6.0, dtype=torch.float32, device=x.device)).clamp(max=10240.0)
    bits = t.to(torch.float16).view(torch.int16).to(torch.int32)
    byte = (bits + 63 + ((bits >> 7) & 1)) >> 7  # to three mantissa bits, ties to even
    byte = torch.where(torch.isfinite(amax), byte, torch.full_like(byte, 255))
    s = _scale(byte.to(torch.uint8)).unsqueeze(-1)
    y = torch.where(s > 0, g / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    a = y.abs()
    code = (a > 0.25).to(torch.uint8)
    for at, closed in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= at) if closed else (a > at)
    code |= torch.signbit(y).to(torch.uint8) << 3
    return code.reshape(x.shape), byte.to(torch.uint8)


def _scale(byte):
    return (byte.to(torch.int32) << 7).to(torch.int16).view(torch.float16).float()


def _pairs():
    """The two values of every byte of codes: ``[256, 2]``, the even dim (low half) first."""
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=DEV)
    b = torch.arange(256, device=DEV)
    return torch.stack([v[b & 15], v[b >> 4]], -1)


def _pack(k, v):
    """fp32 ``[N, H, 16, 128]`` keys and values -> records ``[N, H, 2304]``."""
    n, h = k.shape[:2]
    (kc, ks), (vc, vs) = _quantize(k), _quantize(v)
    kb = kc[..., 0::2] | (kc[..., 1::2] << 4)
    vb = (vc[..., 0::2] | (vc[..., 1::2] << 4)).reshape(n, h, 2, 8, 8, 8).transpose(3, 4)
    vs = vs.reshape(n, h, 2, 8, 8).transpose(3, 4)
    return torch.cat([kb.reshape(n, h, -1), vb.reshape(n, h, -1), ks.reshape(n, h, -1), vs.reshape(n, h, -1)], -1)


def _unpack(rec):
    """records ``[..., 2304]`` -> fp32 keys and values ``[..., 16, 128]``."""
    lead = rec.shape[:-1]
    table = _pairs()

    def values(b):
        return table.index_select(0, b.reshape(-1).to(torch.int32)).reshape(*b.shape[:-1], b.shape[-1] * 2)

    k = values(rec[..., :1024].reshape(*lead, 16, 8, 8)) * _scale(rec[..., 2048:2176].reshape(*lead, 16, 8)).unsqueeze(-1)
    vb = rec[..., 1024:2048].reshape(*lead, 2, 8, 8, 8).transpose(-3, -2)  # [.., token / 8, token % 8, group, 8]
    vs = rec[..., 2176:].reshape(*lead, 2, 8, 8).transpose(-2, -1)
    v = values(vb) * _scale(vs).unsqueeze(-1)
    return k.reshape(*lead, 16, D), v.reshape(*lead, 16, D)


def _dequantized(x):
    """fp32 ``[..., 128]`` through the 4-bit format and back."""
    code, byte = _quantize(x)
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=DEV)
    y = v.index_select(0, code.reshape(-1).to(torch.int32)).reshape(*x.shape[:-1], D // G16, G16) * _scale(byte).unsqueeze(-1)
    return y.reshape(x.shape)


def _bounds(k, live):
    """Bounds of fp32 keys ``[..., 16, 128]`` over the first ``live`` tokens: (codes int8 ``[..., 2, 128]`` (high, low),
    exponents int8 ``[...]``), values = code * 2^exponent, rounded outwards."""
    seen = (torch.arange(B, device=DEV) < live.unsqueeze(-1)).unsqueeze(-1)
    hi = torch.where(seen, k, torch.full_like(k, -math.inf)).amax(-2)
    lo = torch.where(seen, k, torch.full_like(k, math.inf)).amin(-2)
    both = torch.stack([hi, lo], -2)
    m, e = torch.frexp(both.abs().amax((-2, -1)))
    e = torch.where(m == 0, torch.full_like(e, -100), e - 7 + (m * 128 > 127).to(e.dtype))
    s = both * torch.exp2(-e.float()).unsqueeze(-1).unsqueeze(-1)
    codes = torch.stack([s[..., 0, :].ceil(), s[..., 1, :].floor()], -2)
    return codes.to(torch.int8), e.to(torch.int8)


# ---- inputs ------------------------------------------------------------------------------------------------------


def _rope_table(n, theta=500000.0):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    ang = torch.arange(n, dtype=torch.float64, device=DEV).unsqueeze(1) * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _keys(g, shape):
    """Normal values with a few loud channels, as keys have them, in bf16."""
    loud = torch.exp(0.6 * torch.randn(D, generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * loud).to(torch.bfloat16)


def _pool(g, layers, blocks, hkv):
    rec = torch.empty(layers, blocks, hkv, RECORD, dtype=torch.uint8, device=DEV)
    codes = torch.empty(layers, blocks, hkv, 2, D, dtype=torch.int8, device=DEV)
    exps = torch.empty(layers, blocks, hkv, dtype=torch.int8, device=DEV)
    for layer in range(layers):
        for at in range(0, blocks, 8192):
            n = min(8192, blocks - at)
            rec[layer, at : at + n] = _pack(_keys(g, (n, hkv, B, D)).float(), torch.randn(n, hkv, B, D, generator=g, device=DEV).to(torch.bfloat16).float())
    return rec, codes, exps


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    kind, hkv = case["kind"], case["hkv"]
    st = {"kind": kind, "hkv": hkv}
    if kind == "write":
        t, hq = case["tokens"], case["hq"]
        live = t - case["pad"]
        blocks = -(-live // B) + 7
        st["hq"] = hq
        st["qkv"] = torch.randn(t, (hq + 2 * hkv) * D, generator=g, device=DEV).to(torch.float32 if case["f32"] else torch.bfloat16)
        st["positions"] = torch.randint(0, 8192, (t,), generator=g, device=DEV, dtype=torch.int32)
        slots = torch.full((t,), -1, dtype=torch.int64, device=DEV)
        slots[:live] = torch.randperm(blocks * B, generator=g, device=DEV)[:live]
        st["slots"], st["cos_sin"] = slots, _rope_table(8192)
        st["q_out"] = torch.zeros(t, hq, D, dtype=torch.bfloat16, device=DEV)
        st["records"] = torch.zeros(2, blocks, hkv, RECORD, dtype=torch.uint8, device=DEV)
    elif kind == "restore":
        n, layers = case["slots"], case["layers"]
        kv = torch.randn(n, layers, 2, B, hkv, D, generator=g, device=DEV) * 0.5
        grp = kv.reshape(n, layers, -1, G16)
        amax = grp.abs().amax(-1, keepdim=True)
        payload = (grp * (448.0 / amax)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, layers, -1)
        scales = (amax / 448.0).reshape(n, layers, -1).view(torch.uint8)
        st["images"] = torch.cat([payload, scales], -1).contiguous()
        st["deltas"] = torch.randint(-300, 4000, (n,), generator=g, device=DEV, dtype=torch.int32)
        st["deltas"][:: max(2, n // 8)] = 0  # a chunk that stays where it was
        st["blocks"] = torch.randperm(n + 5, generator=g, device=DEV)[:n].to(torch.int32)
        st["cos_sin"] = _rope_table(8192)
        st["records"] = torch.zeros(layers, n + 5, hkv, RECORD, dtype=torch.uint8, device=DEV)
        st["out"] = torch.zeros(n, layers, 2, B, hkv, D, dtype=torch.bfloat16, device=DEV)
        st["layers"] = layers
        step = st["images"][0].numel()
        st["src"] = st["images"].data_ptr() + step * torch.arange(n, dtype=torch.int64, device=DEV)
        st["dst"] = st["out"].data_ptr() + st["out"][0].numel() * 2 * torch.arange(n, dtype=torch.int64, device=DEV)
        st["status"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    else:
        ctx, ql = _lens(case)
        need = [-(-c // B) for c in ctx]
        blocks, hq = sum(need) + 3, case["hq"]
        st["hq"], st["max_q"], st["max_ctx"] = hq, max(ql), max(ctx)
        st["records"], codes, exps = _pool(g, 1, blocks, hkv)
        order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
        tables = torch.zeros(len(ctx), max(need), dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at : at + n]
            at += n
        st["tables"] = tables
        st["q_start"] = torch.tensor([0] + torch.tensor(ql).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        st["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        st["q"] = (1.5 * torch.randn(sum(ql), hq, D, generator=g, device=DEV)).to(torch.bfloat16)
        st["out"] = torch.zeros(sum(ql), hq, D, dtype=torch.bfloat16, device=DEV)
        if kind == "sparse":
            st["pages"] = case["pages"]
            full = torch.full((blocks, hkv), B, device=DEV)
            for i in range(0, blocks, 8192):
                codes[0, i : i + 8192], exps[0, i : i + 8192] = _bounds(_unpack(st["records"][0, i : i + 8192])[0], full[i : i + 8192])
            # the pages that the step's new tokens are in: their bounds are not up to date
            touched = [(i, p) for i, (c, q) in enumerate(zip(ctx, ql)) for p in range((c - q) // B, (c - 1) // B + 1)]
            st["t_seq"] = torch.tensor([a for a, _ in touched], device=DEV)
            st["t_page"] = torch.tensor([p for _, p in touched], device=DEV)
            st["touched"] = tables[st["t_seq"], st["t_page"]]
            codes[0, st["touched"].long()], exps[0, st["touched"].long()] = 0, 0
            st["codes"], st["exps"] = codes, exps
    if own:
        _handles(st)
    return st


def _handles(st):
    from daser_b200.kv.layout import KVGeometry
    from daser_b200.ops import attention, kv_ops

    st["pool"] = kv_ops.PagedKV4Pool.from_tensors([st["records"]])
    if st["kind"] == "restore":
        st["geo"] = KVGeometry(st["layers"], st["hkv"], D, B, 2, "fp8b16")
        st["geo_raw"] = st["geo"].with_codec("raw")
        st["work"] = kv_ops.KVWorkList(st["src"], st["blocks"], st["deltas"])
        st["work_out"] = kv_ops.KVWorkList(st["dst"], st["blocks"])
    elif st["kind"] in ("attend", "sparse"):
        st["ws"] = attention.AttentionWorkspace(st["q"].device)
        if st["kind"] == "sparse":
            st["bounds"] = kv_ops.PageBounds(st["codes"], st["exps"])


# ---- one pass ----------------------------------------------------------------------------------------------------


def run(st):
    if own:
        return _run_own(st)
    return {"write": _plain_write, "restore": _plain_restore, "attend": _plain_attend, "sparse": _plain_sparse}[st["kind"]](st)


def _run_own(st):
    from daser_b200.ops import attention, elementwise, kv_ops

    kind, pool = st["kind"], st["pool"]
    if kind == "write":
        elementwise.rope_kv_write(st["qkv"], st["positions"], st["slots"], st["cos_sin"], st["q_out"], st["hq"], st["hkv"], D, B, pool, 1)
        k, v = kv_ops.kv_read(pool, 1, st["slots"])
        return {"q": st["q_out"], "k": k, "v": v}
    if kind == "restore":
        kv_ops.kv_restore(st["work"], st["geo"], pool, st["cos_sin"], st["status"])
        kv_ops.kv_save(st["work_out"], st["geo_raw"], pool, 0, st["status"])
        return st["out"]
    scale = D**-0.5
    if kind == "attend":
        return attention.paged_attention(st["q"], st["out"], pool, 0, st["tables"], st["q_start"], st["ctx"], st["max_q"], st["max_ctx"], st["hkv"],
                                         scale, st["ws"])
    kv_ops.update_page_bounds(pool, st["bounds"], 0, st["tables"], st["q_start"], st["ctx"], st["max_q"])
    pages = attention.select_pages(st["q"], st["bounds"], 0, st["tables"], st["q_start"], st["ctx"], st["max_q"], st["max_ctx"], st["pages"],
                                   sink_pages=SINK, recent_pages=RECENT, workspace=st["ws"])
    out = attention.sparse_paged_attention(st["q"], st["out"], pool, 0, st["tables"], st["q_start"], st["ctx"], pages, st["max_q"], scale, st["ws"])
    return {"out": out, "pages": pages, "bounds": st["bounds"].read(0, st["touched"])}


def _rotate(x, cs):
    """Rotate halves of fp32 ``x [T, H, 128]`` by ``cs [T, 128]`` (cosines, then sines)."""
    c, s = cs[:, None, : D // 2], cs[:, None, D // 2 :]
    a, b = x[..., : D // 2], x[..., D // 2 :]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_write(st):
    t, hq, hkv = st["qkv"].shape[0], st["hq"], st["hkv"]
    x = st["qkv"].float().reshape(t, hq + 2 * hkv, D)
    cs = st["cos_sin"][st["positions"].long()]
    q = _rotate(x[:, :hq], cs).to(torch.bfloat16)
    kv = torch.cat([_rotate(x[:, hq : hq + hkv], cs), x[:, hq + hkv :]], 1).to(torch.bfloat16).float()
    kv = torch.where((st["slots"] >= 0)[:, None, None], _dequantized(kv), torch.zeros_like(kv)).to(torch.bfloat16)
    return {"q": q, "k": kv[:, :hkv], "v": kv[:, hkv:]}


def _plain_restore(st):
    n, layers = st["images"].shape[:2]
    hkv = st["hkv"]
    elems = 2 * B * hkv * D
    pay = st["images"][..., :elems].contiguous().view(torch.float8_e4m3fn).float().reshape(n, layers, -1, G16)
    sc = st["images"][..., elems:].contiguous().view(torch.float32).unsqueeze(-1)
    kv = (pay * sc).reshape(n, layers, 2, B, hkv, D)
    d = st["deltas"].long()
    cs = st["cos_sin"][d.abs()]
    cs = torch.where((d < 0)[:, None] & (torch.arange(D, device=DEV) >= D // 2), -cs, cs)
    k = _rotate(kv[:, :, 0].reshape(n, -1, D), cs).reshape(n, layers, B, hkv, D)
    k = torch.where((d == 0)[:, None, None, None, None], kv[:, :, 0], k)
    return _dequantized(torch.stack([k, kv[:, :, 1]], 2)).to(torch.bfloat16)


def _rows(st):
    """(sequence, last visible key) of every query row, and the padded index of the rows."""
    qs, ctx = st["q_start"].long(), st["ctx"].long()
    t = torch.arange(st["q"].shape[0], device=DEV)
    seq = torch.searchsorted(qs[1:].contiguous(), t, right=True)
    off = t - qs[seq]
    return seq, off, ctx[seq] - (qs[seq + 1] - qs[seq]) + off


def _plain_attend(st):
    hq, hkv, q = st["hq"], st["hkv"], st["q"].float()
    seq, off, pos = _rows(st)
    n, p = st["tables"].shape
    k, v = _unpack(st["records"][0][st["tables"].long()].transpose(1, 2))  # [seqs, hkv, pages, 16, 128]
    k, v = k.reshape(n, hkv, p * B, D), v.reshape(n, hkv, p * B, D)
    rep = hq // hkv
    wide = torch.zeros(n, st["max_q"], hq, D, device=DEV)
    wide[seq, off] = q
    last = torch.full((n, st["max_q"]), -1, dtype=torch.long, device=DEV)
    last[seq, off] = pos
    wide = wide.reshape(n, -1, hkv, rep, D).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, D)
    s = torch.matmul(wide, k.transpose(2, 3)).reshape(n, hkv, rep, -1, p * B)
    s *= D**-0.5
    seen = torch.arange(p * B, device=DEV) <= last[:, :, None]  # [seqs, queries, keys]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(n, hkv, -1, p * B), v).reshape(n, hkv, rep, -1, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, hq, D)[seq, off].to(torch.bfloat16)


def _update_bounds(st):
    live = st["ctx"].long()[st["t_seq"]] - B * st["t_page"]
    touched = st["touched"].long()
    k = _unpack(st["records"][0, touched])[0]
    codes, exps = _bounds(k, live.clamp(max=B)[:, None].expand(-1, st["hkv"]))
    st["codes"][0, touched], st["exps"][0, touched] = codes, exps
    return codes.float() * torch.exp2(exps.float())[..., None, None]


def _plain_select(st):
    """The pages of every query row and KV head: ``[rows, hkv, pages]`` ascending, -1 behind the last."""
    hkv, budget = st["hkv"], st["pages"]
    seq, _, pos = _rows(st)
    rows, p = seq.numel(), st["tables"].shape[1]
    q = st["q"].double().reshape(rows, hkv, -1, D)
    q = torch.stack([q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)], -2)  # [rows, hkv, 2, 128]
    m, e = torch.frexp(q.abs().amax((-2, -1)))
    e = torch.where(m == 0, torch.zeros_like(e), e - 7 + (m * 128 > 127).to(e.dtype))
    q = torch.round(q * torch.exp2(-e.double())[..., None, None]).reshape(rows, hkv, 2 * D, 1)
    phys = st["tables"].long()
    codes = st["codes"][0][phys].transpose(1, 2).reshape(-1, hkv, p, 2 * D).float()  # whole numbers: exact in fp32 sums
    score = torch.matmul(codes[seq], q.float()).squeeze(-1)
    score *= torch.exp2(st["exps"][0][phys].transpose(1, 2)[seq].float())
    page = torch.arange(p, device=DEV)
    count = torch.div(pos, B, rounding_mode="floor") + 1
    forced = (page < SINK) | (page >= count[:, None] - RECENT)
    score = torch.where(forced[:, None], torch.full_like(score, math.inf), score)
    score = torch.where((page >= count[:, None])[:, None], torch.full_like(score, -math.inf), score)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget]
    if order.shape[-1] < budget:
        order = torch.cat([order, order.new_full((*order.shape[:-1], budget - order.shape[-1]), p)], -1)
    order = torch.where(order < count[:, None, None], order, torch.full_like(order, 1 << 30))
    order = order.sort(-1).values
    return torch.where(order < (1 << 30), order, torch.full_like(order, -1)).to(torch.int32)


def _plain_sparse(st):
    bounds = _update_bounds(st)
    pages = _plain_select(st)
    hkv = st["hkv"]
    seq, _, pos = _rows(st)
    rows = seq.numel()
    at = pages.long().clamp(min=0)
    phys = st["tables"].long()[seq[:, None, None], at]
    k, v = _unpack(st["records"][0][phys, torch.arange(hkv, device=DEV)[None, :, None]])
    k, v = k.reshape(rows, hkv, -1, D), v.reshape(rows, hkv, -1, D)
    key = (at[..., None] * B + torch.arange(B, device=DEV)).reshape(rows, hkv, -1)
    seen = (key <= pos[:, None, None]) & (pages >= 0).repeat_interleave(B, -1)
    s = torch.matmul(st["q"].float().reshape(rows, hkv, -1, D), k.transpose(2, 3)) * D**-0.5
    s = s.masked_fill(~seen[:, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).reshape(rows, -1, D)
    return {"out": o.to(torch.bfloat16), "pages": pages, "bounds": bounds}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------


def _exact_codec(x):
    """fp64 ``[..., 128]`` through the format: nearest scale of four significant bits, nearest e2m1 value."""
    g = x.reshape(*x.shape[:-1], -1, G16)
    s = (g.abs().amax(-1, keepdim=True) / 6).clamp(max=10240.0).to(torch.float16).double()
    quantum = torch.exp2(torch.floor(torch.log2(s.clamp(min=2.0**-14))) - 3)
    s = torch.round(s / quantum) * quantum
    y = torch.where(s > 0, g / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g))
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(y) * (torch.round(a / step) * step).clamp(max=6.0) * s).reshape(x.shape)


def _exact_record(rec):
    """One pass over bytes with shifts instead of a table: records -> fp64 K, V ``[..., 16, 128]``."""
    def val(n):
        e, m = (n >> 1) & 3, (n & 1).double()
        a = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
        return torch.where((n >> 3) == 1, -a, a)

    def scl(b):
        e, m = (b >> 3).double(), (b & 7).double()
        return torch.where(e == 0, m * 2.0**-17, (1 + m / 8) * torch.exp2(e - 15))

    lead = rec.shape[:-1]
    r = rec.to(torch.int16)
    kb, vb = r[..., :1024].reshape(*lead, 16, 64), r[..., 1024:2048].reshape(*lead, 2, 8, 8, 8)
    k = torch.stack([val(kb & 15), val(kb >> 4)], -1).reshape(*lead, 16, 8, 16)
    k = k * scl(r[..., 2048:2176].reshape(*lead, 16, 8, 1))
    v = torch.stack([val(vb & 15), val(vb >> 4)], -1).reshape(*lead, 2, 8, 8, 16)
    v = (v * scl(r[..., 2176:].reshape(*lead, 2, 8, 8, 1))).transpose(-3, -2)
    return k.reshape(*lead, 16, D), v.reshape(*lead, 16, D)


def _exact_rotate(x, ang):
    """Complex multiplication of dims ``(i, i + 64)`` by ``ang [..., 64]``."""
    z = torch.complex(x[..., : D // 2].contiguous(), x[..., D // 2 :].contiguous()) * ang
    return torch.cat([z.real, z.imag], -1)


def _exact_power(a):
    """The smallest power of two that brings ``a`` to at most 127; 1 for nothing."""
    e = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))) - 6
    return torch.where(a > 0, torch.exp2(torch.where(a > 127 * torch.exp2(e), e + 1, e)), torch.ones_like(a))


def _exact_bounds(st):
    """Of the touched pages, one page after the other: fp64 ``[touched, hkv, 2, 128]``."""
    out = []
    for i, p, n in zip(st["t_seq"].tolist(), st["t_page"].tolist(), st["touched"].tolist()):
        k = _exact_record(st["records"][0, n])[0][:, : int(st["ctx"][i]) - B * p]
        hi, lo = k.max(1).values, k.min(1).values
        s = _exact_power(torch.maximum(hi.abs(), lo.abs()).max(-1).values)[:, None]
        out.append(torch.stack([torch.ceil(hi / s) * s, torch.floor(lo / s) * s], 1))
    return torch.stack(out)


def _exact_choice(st, bounds, q, h, phys, count, budget):
    """The pages, as truth values over ``phys``, that one query row's heads ``q [rep, 128]`` of KV head ``h`` read."""
    page = torch.arange(phys.numel(), device=DEV)
    if count <= budget:
        return page < count
    hi_lo = st["codes"][0, phys, h].double() * torch.exp2(st["exps"][0, phys, h].double())[:, None, None]
    hi_lo = torch.where((phys[:, None] == st["touched"][None]).any(1)[:, None, None], bounds[(phys[:, None] == st["touched"][None]).int().argmax(1), h], hi_lo)
    up, down = q.clamp(min=0).sum(0), q.clamp(max=0).sum(0)
    s = _exact_power(torch.maximum(up.max(), -down.min()))
    score = hi_lo[:, 0] @ torch.round(up / s) + hi_lo[:, 1] @ torch.round(down / s)
    must = (page < SINK) | (page >= count - RECENT)
    score = torch.where(must, math.inf, torch.where(page < count, score, -math.inf))
    # a page is read if fewer than `budget` are ahead of it: of higher score, or of the same and lower number
    rank = torch.empty_like(page)
    rank[sorted(range(phys.numel()), key=lambda j, v=score.tolist(): (-v[j], j))] = page
    return rank < budget


def exact(case, seed):
    st = prepare(case, seed)
    kind, hkv = case["kind"], case["hkv"]
    if kind in ("write", "restore"):
        table = st["cos_sin"].double()
        turn = torch.complex(table[:, : D // 2].contiguous(), table[:, D // 2 :].contiguous())
    if kind == "write":
        t, hq = case["tokens"], case["hq"]
        x = st["qkv"].double().reshape(t, -1, D)
        ang = turn[st["positions"].long()][:, None]
        q, k, v = _exact_rotate(x[:, :hq], ang), _exact_rotate(x[:, hq : hq + hkv], ang), x[:, hq + hkv :]
        live = (st["slots"] >= 0).double()[:, None, None]
        # the cache holds what a bf16 cache would have held
        return {"q": q, "k": _exact_codec(k.to(torch.bfloat16).double()) * live, "v": _exact_codec(v.to(torch.bfloat16).double()) * live}
    if kind == "restore":
        n, layers = case["slots"], case["layers"]
        elems = 2 * B * hkv * D
        raw = st["images"].reshape(n, layers, -1)
        x = raw[..., :elems].contiguous().view(torch.float8_e4m3fn).double().reshape(n, layers, -1, G16)
        x = (x * raw[..., elems:].contiguous().view(torch.float32).double()[..., None]).reshape(n, layers, 2, B, hkv, D)
        d = st["deltas"].long()
        ang = torch.where((d < 0)[:, None], turn[d.abs()].conj(), turn[d.abs()])[:, None, None, None]
        return torch.stack([_exact_codec(_exact_rotate(x[:, :, 0], ang)), _exact_codec(x[:, :, 1])], 2)
    ctx, ql = _lens(case)
    outs, row = [], 0
    bounds = None
    if kind == "sparse":
        bounds = _exact_bounds(st)
    for i, (c, n) in enumerate(zip(ctx, ql)):
        phys = st["tables"][i, : -(-c // B)].long()
        for h in range(hkv):
            k, v = _exact_record(st["records"][0, phys, h])
            k, v = k.reshape(-1, D), v.reshape(-1, D)
            rep = case["hq"] // hkv
            q = st["q"][row : row + n, h * rep : (h + 1) * rep].double()
            s = torch.einsum("qrd,kd->rqk", q, k) / math.sqrt(D)
            ok = torch.arange(k.shape[0], device=DEV)[None] <= (c - n + torch.arange(n, device=DEV))[:, None]
            if kind == "sparse":
                last = [c - n + j for j in range(n)]
                chosen = torch.stack([_exact_choice(st, bounds, q[j], h, phys, last[j] // B + 1, case["pages"]) for j in range(n)])
                ok = ok & chosen.repeat_interleave(B, 1)
            outs.append((row, h, torch.einsum("rqk,kd->qrd", torch.softmax(s.masked_fill(~ok, -math.inf), -1), v)))
        row += n
    o = torch.empty(row, case["hq"], D, dtype=torch.float64, device=DEV)
    for r, h, x in outs:
        o[r : r + x.shape[0], h * x.shape[1] : (h + 1) * x.shape[1]] = x
    return {"out": o, "pages": None, "bounds": bounds} if kind == "sparse" else o
