"""The runner and the RAG engine on a 4-bit pool (``kv_format="fp4b16"``)."""

import random

import pytest
import torch

from conftest import LiveControlPlane
from daser_b200.models.llama import PRESETS, LlamaWeights
from test_gpu_kv4 import D, _oracle, _ops

pytestmark = pytest.mark.gpu


def _step(runner, seqs):
    out = runner.forward(runner.stage_inputs(seqs)).clone()
    torch.cuda.synchronize()
    return out.tolist()


@pytest.mark.parametrize("preset", ["tiny-gqa", "tiny-8kv", "tiny-gqa-qk"])
def test_the_runners_attention_is_the_formula_over_its_pool(preset):
    """After each step the last layer's queries, its pool and its attention output are still in the runner's buffers.  Prompts of
    several lengths in one step (prefill kernel), then decode steps: eager, captured and replayed."""
    from daser_b200.engine.runner import GpuModelRunner

    cfg = PRESETS[preset]
    w = LlamaWeights.random(cfg, "cuda", torch.bfloat16, seed=3, std=0.05)
    runner = GpuModelRunner(cfg, w, num_blocks=64, max_tokens=256, max_seqs=8, max_blocks=32, kv_format="fp4b16")
    rng = random.Random(0)
    lens = [33, 7, 90]
    perm = torch.randperm(64, generator=torch.Generator().manual_seed(1)).tolist()
    seqs, at = [], 0
    for n in lens:
        need = -(-(n + 5) // 16)
        seqs.append({"tokens": [rng.randrange(cfg.vocab_size) for _ in range(n)], "start_pos": 0, "block_table": perm[at : at + need]})
        at += need
    tables = torch.zeros(3, 32, dtype=torch.int64)
    for i, s in enumerate(seqs):
        tables[i, : len(s["block_table"])] = torch.tensor(s["block_table"])
    for step in range(4):
        nxt = _step(runner, seqs)
        q_lens, ctx = [len(s["tokens"]) for s in seqs], [s["start_pos"] + len(s["tokens"]) for s in seqs]
        T = sum(q_lens)
        rec = runner.local_pool.keepalive[0][0][len(w.layers) - 1].cpu()
        q = runner.q_rot[:T].float().cpu()
        group = runner.hq // runner.hkv
        want, tol = _oracle(rec, tables, q, q_lens, ctx, D**-0.5, prefill=max(q_lens) * group >= 64)
        got = runner.attn_out[:T].view(T, runner.hq, D).double().cpu()
        assert (got.isfinite().all()) and ((got - want).abs() <= tol).all(), (step, ((got - want).abs() / tol).max())
        seqs = [{"tokens": [t], "start_pos": c, "block_table": s["block_table"]} for s, t, c in zip(seqs, nxt, ctx)]
    runner.check_status()


def test_replayed_steps_across_the_contexts_at_which_they_are_planned_anew():
    """Steps of one shape share a graph over a range of context lengths.  A long prompt in pieces, then decode steps from 2040 keys on:
    the plan changes behind 2048, every step's attention is the formula's.  (Tokens are not compared with an eager run's: projections
    that are split along K add their parts in no fixed order.)"""
    from daser_b200.engine.runner import GpuModelRunner

    cfg = PRESETS["tiny-gqa"]
    w = LlamaWeights.random(cfg, "cuda", torch.bfloat16, seed=5, std=0.05)
    rng = random.Random(4)
    prompt = [rng.randrange(cfg.vocab_size) for _ in range(2040)]
    table = list(range(160, 160 - 131, -1))
    runner = GpuModelRunner(cfg, w, num_blocks=161, max_tokens=256, max_seqs=4, max_blocks=256, kv_format="fp4b16")

    def check(n, ctx):
        rec = runner.local_pool.keepalive[0][0][len(w.layers) - 1].cpu()
        want, tol = _oracle(rec, torch.tensor([table]), runner.q_rot[:n].float().cpu(), [n], [ctx], D**-0.5, prefill=n > 1)
        got = runner.attn_out[:n].view(n, runner.hq, D).double().cpu()
        assert ((got - want).abs() <= tol).all(), (n, ctx, ((got - want).abs() / tol).max())

    for i in range(0, len(prompt), 256):
        piece = prompt[i : i + 256]
        token = _step(runner, [{"tokens": piece, "start_pos": i, "block_table": table}])
    check(len(piece), len(prompt))
    for i in range(14):
        token = _step(runner, [{"tokens": token, "start_pos": len(prompt) + i, "block_table": table}])
        check(1, len(prompt) + i + 1)
    runner.check_status()
    assert len(runner._graphs) >= 2 * len(runner.layer_groups)  # pieces of 256 tokens, decode steps


def test_rag_engine_restores_into_a_4_bit_pool(tmp_path):
    from daser_b200.engine.rag_gpu import GpuRagEngine, RagRequest

    _, _, kv_ops = _ops()
    cfg = PRESETS["tiny-gqa"]
    lp = LiveControlPlane(tmp_path, total_slots=256,
                          slot_size=cfg.num_layers * 2 * 16 * cfg.num_kv_heads * cfg.head_dim * 5 // 4).start()
    eng = GpuRagEngine(cfg, lp.socket_path, lp.cfg.store_path, num_blocks=256, max_tokens=128, hbm_slots=64, kv_format="fp4b16")
    try:
        rng = random.Random(1)
        chunks = [[rng.randrange(cfg.vocab_size) for _ in range(n)] for n in (64, 128, 48)]
        for c in chunks:
            eng.store_chunk(c)
        query = [rng.randrange(cfg.vocab_size) for _ in range(20)]
        runs = []
        for attempt in range(2):  # from the store file, then from the HBM tier
            req = eng.generate([chunks[2], chunks[0], chunks[1]], query, max_new_tokens=4)
            assert req.restored_chunks == 3 and len(req.generated) == 4
            runs.append(req.generated)
        assert runs[0] == runs[1]  # the same slots, the same kernels
        r = eng.submit(RagRequest([chunks[2], chunks[0]], query, 2))
        eng._ttft_step(eng.waiting.pop(0))
        off = len(chunks[2])
        restored = r.block_table[off // 16 : (off + 64) // 16]
        fresh = eng.blocks.alloc(4)
        eng._prefill_tokens(chunks[0], off, [0] * (off // 16) + fresh)
        slots = lambda blocks: (torch.tensor(blocks)[:, None] * 16 + torch.arange(16)).flatten().cuda()
        pool = eng.runner.local_pool
        # Layer 0 depends on token and position alone.  With largest magnitude A, a rounding to 4 bits is off by at most one scale, 0.178 A
        # (A / 6 * (1 + 2^-4)); the stored value was rounded so, then to fp8 for the slot (2^-4 of itself), and again after its rotation,
        # which mixes two values of a key (factor sqrt 2, before and behind it); the fresh one once.  2^-4: the largest value's
        # own rounding; 2^-6: the products' order and bf16.  In the mean each rounding changes some 10 % of the root mean square.
        for got, want, p in zip(kv_ops.kv_read(pool, 0, slots(restored)), kv_ops.kv_read(pool, 0, slots(fresh)), (2**0.5, 1.0)):
            got, want = got.float().flatten(), want.float().flatten()
            e1 = (0.178 + 2.0**-4 * 1.178) * p * p
            bound = (e1 + 0.178 * (1 + e1) + 0.178 + 2.0**-6) / (1 - 2.0**-4)
            assert (got - want).abs().max() <= bound * want.abs().max()
            assert torch.nn.functional.cosine_similarity(got, want, dim=0) > 0.9
        eng.runner.check_status()
    finally:
        eng.close()
        lp.stop()


def test_the_runner_refuses_what_the_pool_cannot_hold():
    from daser_b200.engine.runner import GpuModelRunner

    w = LlamaWeights.random(PRESETS["toy-qk"], "cuda", torch.bfloat16)  # head_dim 64
    with pytest.raises(ValueError, match="head_dim 128"):
        GpuModelRunner(PRESETS["toy-qk"], w, num_blocks=8, max_tokens=16, kv_format="fp4b16")
    with pytest.raises(ValueError, match="kv_format"):
        GpuModelRunner(PRESETS["toy-qk"], w, num_blocks=8, max_tokens=16, kv_format="int4")


@pytest.mark.parametrize("kv_format", ["fp4b16", "fp8b16"])
def test_a_padding_row_leaves_the_cache_alone(kv_format):
    """A batch padded with a copy of its first sequence: the copy has no slot, the cache is what the batch without it writes, and the copy
    attends as the first row does."""
    from daser_b200.engine.runner import GpuModelRunner

    cfg = PRESETS["tiny-gqa"]
    w = LlamaWeights.random(cfg, "cuda", torch.bfloat16, seed=7, std=0.05)
    runner = GpuModelRunner(cfg, w, num_blocks=16, max_tokens=64, max_seqs=4, max_blocks=8, kv_format=kv_format)
    _step(runner, [{"tokens": list(range(3, 23)), "start_pos": 0, "block_table": [4, 2]}])
    seq = {"tokens": [9], "start_pos": 20, "block_table": [4, 2]}
    inp = runner.stage_inputs([seq, dict(seq, write=False)])
    assert inp.slot_mapping.tolist() == [2 * 16 + 4, -1]
    pool = (lambda: runner.local_pool.keepalive[0][0]) if kv_format == "fp4b16" else (lambda: runner.kv_payload)
    before = pool().clone()
    runner.forward(runner.stage_inputs([dict(seq, write=False)]))
    assert torch.equal(pool(), before)
    runner.forward(runner.stage_inputs([seq, dict(seq, write=False)]))  # (a step's inputs live in the runner's buffers)
    assert not torch.equal(pool(), before)
    if kv_format == "fp4b16":  # the last layer's queries and outputs are still there
        rec = runner.local_pool.keepalive[0][0][len(w.layers) - 1].cpu()
        want, tol = _oracle(rec, torch.tensor([[4, 2]] * 2), runner.q_rot[:2].float().cpu(), [1, 1], [21, 21], D**-0.5)
        assert ((runner.attn_out[:2].view(2, runner.hq, D).double().cpu() - want).abs() <= tol).all()
    runner.check_status()


def test_engines_of_both_formats_on_one_store(tmp_path):
    """The 4-bit engine restores what the fp8 engine stored; the fp8 engine computes what only the 4-bit engine has."""
    from daser_b200.engine.rag_gpu import GpuRagEngine

    cfg = PRESETS["tiny-gqa"]
    lp = LiveControlPlane(tmp_path, total_slots=256, slot_size=cfg.num_layers * 2 * 16 * cfg.num_kv_heads * cfg.head_dim * 5 // 4).start()
    make = lambda fmt: GpuRagEngine(cfg, lp.socket_path, lp.cfg.store_path, num_blocks=64, max_tokens=64, model_id="m", kv_format=fmt)  # noqa: E731
    fp8, kv4 = make("fp8b16"), make("fp4b16")
    try:
        rng = random.Random(2)
        a, b = ([rng.randrange(cfg.vocab_size) for _ in range(32)] for _ in range(2))
        kv4.store_chunk(a)
        fp8.store_chunk(b)
        query = [rng.randrange(cfg.vocab_size) for _ in range(9)]
        assert fp8.generate([a, b], query, max_new_tokens=2).restored_chunks == 1
        assert kv4.generate([a, b], query, max_new_tokens=2).restored_chunks == 2
        for eng in (fp8, kv4):
            eng.runner.check_status()
    finally:
        fp8.close()
        kv4.close()
        lp.stop()


def test_pipeline_stages_on_4_bit_pools():
    """Two stages of one layer each hand the residual stream over in this process: every stage's attention is the formula over its own pool,
    and what comes out points the way it does in one runner with both layers.  (It is not equal: projections that are split along K add in no
    fixed order, and a last bit may move a key or value to the next of the format's values.  An unrelated stream has a cosine near 0.)"""
    from daser_b200.engine.runner import GpuModelRunner

    class Link:
        def __init__(self, stage, box):
            self.stage, self.first, self.last, self.box = stage, stage == 0, stage == 1, box

        def drain(self):
            pass

        def send_next(self, t):
            self.box.append(t.clone())

        def recv_prev_into(self, buf):
            buf.copy_(self.box.pop())

    cfg = PRESETS["tiny-gqa"]
    assert cfg.num_layers == 2
    box, stages = [], []
    for i in range(2):
        w = LlamaWeights.random(cfg, "cuda", torch.bfloat16, seed=11, std=0.05, layers=range(i, i + 1))
        stages.append(GpuModelRunner(cfg, w, num_blocks=16, max_tokens=64, max_seqs=2, max_blocks=8, layer_range=range(i, i + 1), pool_layers=1,
                                     pp_link=Link(i, box), kv_format="fp4b16"))
    whole = GpuModelRunner(cfg, LlamaWeights.random(cfg, "cuda", torch.bfloat16, seed=11, std=0.05), num_blocks=16, max_tokens=64, max_seqs=2,
                           max_blocks=8, kv_format="fp4b16")
    table, rng = [5, 9, 1, 14], random.Random(5)
    tokens, pos = [rng.randrange(cfg.vocab_size) for _ in range(37)], 0
    for step in range(4):
        seq = {"tokens": tokens, "start_pos": pos, "block_table": table}
        assert stages[0].forward(stages[0].stage_inputs([seq])) is None
        got = stages[1].forward(stages[1].stage_inputs([seq])).tolist()
        n, ctx = len(tokens), pos + len(tokens)
        for r in stages:
            want, tol = _oracle(r.local_pool.keepalive[0][0][0].cpu(), torch.tensor([table]), r.q_rot[:n].float().cpu(), [n], [ctx], D**-0.5,
                                prefill=n > 1)
            assert ((r.attn_out[:n].view(n, r.hq, D).double().cpu() - want).abs() <= tol).all(), step
        whole.forward(whole.stage_inputs([seq]))
        a, b = stages[1].normed[n - 1].float(), whole.normed[n - 1].float()
        assert torch.nn.functional.cosine_similarity(a, b, dim=0) > 0.99
        tokens, pos = got, ctx
    for r in (*stages, whole):
        r.check_status()
