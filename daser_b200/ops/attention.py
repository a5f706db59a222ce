"""Paged attention over the block-scaled fp8 pool (``ops/csrc/attention.cu``) and over the 4-bit pool
(``ops/csrc/attention4.cu``, ``attention4_tc.cu``), there also over pages selected per query
(``ops/csrc/attention4_select.cu``)."""

from __future__ import annotations

import ctypes as C
import functools
import os
from typing import Optional

import torch

from daser_b200.ops import _lib
from daser_b200.ops.kv_ops import KV4_DIM, KV4_TOKENS, PageBounds, PagedKV4Pool, PagedKVPool, check_sequences

NUM_SMS = 148
MAX_ROW_SPLITS = 262144  # (query rows x KV splits) the split-KV scratch is sized for (135 MB)


SELECT_ON_CHIP = 16384  # pages of a context up to which select_pages needs no scratch
TC_MIN_ROWS = 64  # query rows per KV head from which chunked prefill runs on the tcgen05 kernel
TC_KEY_TILE = 64
_tc_enabled = os.environ.get("DASER_ATTN_TC", "1") != "0"


def set_tensor_core_prefill(enabled: bool) -> None:
    """Route chunked prefill to the tcgen05 kernel (default) or to the mma.sync one."""
    global _tc_enabled
    _tc_enabled = bool(enabled)
    _lib.lib().daser_attention_set_tc(1 if enabled else 0)


def tc_status() -> int:
    """Non-zero if a tcgen05 attention CTA ever gave up on a bounded wait (synchronises)."""
    out = C.c_uint32(0)
    _lib.check(_lib.lib().daser_attention_tc_status(C.byref(out)), "attention_tc_status")
    return int(out.value)


def plan_splits(num_seqs: int, kv_heads: int, max_q_len: int, group: int, max_ctx: int,
                block_tokens: int = 16, rows: int = 0) -> tuple[int, int]:
    """(nsplit, split_tokens): enough work items to fill the GPU."""
    if _tc_enabled and max_q_len * group >= TC_MIN_ROWS and 128 % group == 0:
        # tcgen05 kernel: the unit is a CTA of 128 query rows, two per SM, 64 keys per tile
        base_items = num_seqs * kv_heads * -(-max_q_len * group // 128)
        want = max(1, (NUM_SMS * 2) // max(base_items, 1))
        max_splits = max(1, -(-max_ctx // (2 * TC_KEY_TILE)))  # splits of two key tiles at the shortest
        nsplit = max(1, min(want, max_splits, 64))
        if rows > 0:
            nsplit = max(1, min(nsplit, MAX_ROW_SPLITS // rows))
        per = -(-max_ctx // nsplit)
        split_tokens = -(-per // TC_KEY_TILE) * TC_KEY_TILE
        return -(-max_ctx // split_tokens), split_tokens
    row_tiles = -(-max_q_len * group // 16)
    base_items = num_seqs * kv_heads * row_tiles
    # Measured on the batch-64, 4k-32k decode case: 1024-token splits reach 0.80 of the copy
    # bandwidth, 2048 -> 0.78, 8192 -> 0.53, 256 -> 0.69.  So: splits of about 1024 tokens
    # whenever that still yields several waves of warps, never shorter than 256.
    target_items = NUM_SMS * 8 * 4
    if row_tiles > 1:
        # prefill kernel: the work unit is a CTA of four row tiles, three CTAs fit an SM
        base_items = num_seqs * kv_heads * -(-row_tiles // 4)
        target_items = NUM_SMS * 3 * 2
    want = max(1, -(-target_items // max(base_items, 1)))
    by_len = max(1, max_ctx // 1024)
    max_splits = max(1, max_ctx // 256)
    nsplit = max(1, min(max(want, by_len), max_splits, 128))
    if rows > 0:
        nsplit = max(1, min(nsplit, MAX_ROW_SPLITS // rows))
    per = -(-max_ctx // nsplit)
    split_tokens = -(-per // block_tokens) * block_tokens
    nsplit = -(-max_ctx // split_tokens)
    return nsplit, split_tokens


def kv4_status() -> int:
    """Non-zero if a CTA of the 4-bit prefill kernel ever gave up on a bounded wait (synchronises)."""
    out = C.c_uint32(0)
    _lib.check(_lib.lib().daser_attention4_tc_status(C.byref(out)), "attention4_tc_status")
    return int(out.value)


@functools.lru_cache(maxsize=4096)
def plan_kv4(num_seqs: int, kv_heads: int, max_q_len: int, group: int, max_pages: int, rows: int = 0) -> tuple[int, int]:
    """(parts, pages per split) of attention over the 4-bit pool; ``max_pages``: of the longest context, or of a page list.

    From 64 query rows per KV head on (the tcgen05 kernel) parts are splits per context.  Below, they are the CTAs that share all
    pages evenly, 0 for one CTA per (sequence, row tile, KV head) and no merge."""
    max_pages = max(1, max_pages)
    if max_q_len * group >= TC_MIN_ROWS:
        # a CTA of two tiles of 128 query rows, one per SM, tiles of four pages; splits of two tiles at the shortest
        items = num_seqs * kv_heads * -(-max_q_len // (2 * (128 // group)))
        nsplit = max(1, min(NUM_SMS // max(items, 1), -(-max_pages // 8), 64))
        if rows > 0:
            nsplit = max(1, min(nsplit, MAX_ROW_SPLITS // rows))
        per = -(--(-max_pages // nsplit) // 4) * 4
        return -(-max_pages // per), per
    # One CTA per item: about 2 us and 0.051 us a page, in as many waves as the items need.  Shared: the same over all pages and 80 pages'
    # time per item, and 6 us for the merge kernel and the partial results.  Measured: 128 items of 128 pages 9 us against
    # 24, 8 items of 256 pages 17 against 15, 256 items of 256 - 2048 pages 210 against 130.
    items = max(1, num_seqs) * kv_heads * -(-max_q_len * group // (8 if max_q_len * group <= 8 else 16))
    workers = min(NUM_SMS, items * max_pages // 32)  # a pair of pages a warp at least
    if workers < 2:
        return 0, 0
    alone = -(-items // NUM_SMS) * (2.0 + 0.051 * max_pages)
    shared = 8.0 + 0.051 * items * (max_pages + 80) / workers
    return (0 if alone <= shared else workers), 0


class AttentionWorkspace:
    """Scratch for split-KV partials, grown on demand and reused.

    Calls that use one workspace have to be ordered (one stream, or events between streams), graph replays included.  When it
    grows, to twice the size at least, it keeps the smaller buffers, whose addresses captured graphs may hold."""

    def __init__(self, device) -> None:
        self.device = device
        self.part_o: Optional[torch.Tensor] = None
        self.part_lse: Optional[torch.Tensor] = None
        self.scores: Optional[torch.Tensor] = None  # of select_pages
        self.shared: Optional[torch.Tensor] = None  # which CTAs share an item of the 4-bit decode kernel
        self._outgrown: list = []

    def ensure(self, rows: int, nsplit: int, head_dim: int) -> None:
        need = rows * nsplit
        if self.part_lse is None or self.part_lse.numel() < need:
            if self.part_lse is not None:
                self._outgrown += [self.part_o, self.part_lse]
                need = max(need, 2 * self.part_lse.numel())
            self.part_o = torch.empty(need * head_dim, dtype=torch.float32, device=self.device)
            self.part_lse = torch.empty(need, dtype=torch.float32, device=self.device)

    def ensure_shared(self, items: int) -> torch.Tensor:
        if self.shared is None or self.shared.numel() < 2 * items:
            need = 2 * items
            if self.shared is not None:
                self._outgrown.append(self.shared)
                need = max(need, 2 * self.shared.numel())
            self.shared = torch.empty(need, dtype=torch.int32, device=self.device)
        return self.shared

    def ensure_scores(self, need: int) -> torch.Tensor:
        if self.scores is None or self.scores.numel() < need:
            if self.scores is not None:
                self._outgrown.append(self.scores)
                need = max(need, 2 * self.scores.numel())
            self.scores = torch.empty(need, dtype=torch.float32, device=self.device)
        return self.scores


def paged_attention(
    q: torch.Tensor,
    out: torch.Tensor,
    pool: PagedKVPool | PagedKV4Pool,
    layer: int,
    block_tables: torch.Tensor,
    q_start: torch.Tensor,
    ctx_lens: torch.Tensor,
    max_q_len: int,
    max_ctx: int,
    num_kv_heads: int,
    softmax_scale: float,
    workspace: Optional[AttentionWorkspace],
    rank: int = 0,
    block_tokens: int = 16,
    nsplit: Optional[int] = None,
    split_tokens: Optional[int] = None,
) -> torch.Tensor:
    """``q, out``: bf16 ``[Tq, Hq, D]``; sequences given by ``q_start`` (prefix sums) and ``ctx_lens``.

    The K/V of the new tokens must already be in the pool; row ``t`` of a sequence attends
    keys ``0 .. ctx_len - q_len + t`` (a row with none gets zeros); rows of no sequence are left as they were.

    Over a :class:`~daser_b200.ops.kv_ops.PagedKV4Pool` any group of up to 16 query heads per KV head is taken,
    ``max_ctx`` has to be at least the longest context (it may be a capacity), ``max_q_len`` at least the most query tokens of a sequence (those
    beyond it are left alone), and ``workspace`` may be ``None`` (scratch of the call's own).  A value that is not finite shows in the rows that see
    it.  Queries are rounded to f16 once they are scaled; a row that f16 does not hold takes a slower way (scores have to fit fp32).
    ``nsplit`` then is the first value of :func:`plan_kv4`.
    """
    if isinstance(pool, PagedKV4Pool):
        _lib.require(block_tokens == KV4_TOKENS and num_kv_heads == pool.heads_per_rank, "block_tokens or num_kv_heads are not the pool's")
        _lib.require(split_tokens is None, "a 4-bit pool takes nsplit alone")
        return _attention_kv4(q, out, pool, layer, block_tables, q_start, ctx_lens, max_q_len, max_ctx, softmax_scale, workspace, rank,
                              None, nsplit)
    Tq, Hq, D = q.shape
    num_seqs = ctx_lens.numel()
    assert block_tables.dtype == torch.int32 and q_start.dtype == torch.int32 and ctx_lens.dtype == torch.int32
    if nsplit is None or split_tokens is None:
        nsplit, split_tokens = plan_splits(num_seqs, num_kv_heads, max_q_len, Hq // num_kv_heads, max_ctx, block_tokens)
    if nsplit > 1:
        workspace.ensure(Tq * Hq, nsplit, D)
    pool_c = pool.c_struct()
    po = workspace.part_o.data_ptr() if nsplit > 1 else None
    pl = workspace.part_lse.data_ptr() if nsplit > 1 else None
    _lib.check(
        _lib.lib().daser_paged_attention_fp8(
            C.c_void_p(q.data_ptr()), C.c_void_p(out.data_ptr()), C.c_void_p(po), C.c_void_p(pl),
            C.byref(pool_c), layer, rank, C.c_void_p(block_tables.data_ptr()), int(block_tables.shape[1]),
            C.c_void_p(q_start.data_ptr()), C.c_void_p(ctx_lens.data_ptr()), num_seqs, Tq, max_q_len,
            Hq, num_kv_heads, D, block_tokens, nsplit, split_tokens, C.c_float(softmax_scale),
            _lib.stream_ptr(),
        ),
        "paged_attention_fp8",
    )
    if nsplit > 1:
        _lib.launch_count += 1  # the merge kernel
    return out


def _check_step(q, out, index, kv_heads, block_tables, q_start, ctx_lens, max_q_len) -> tuple[int, int, int]:
    """The arguments every 4-bit attention call shares; (query rows, query heads, sequences)."""
    bf16 = torch.bfloat16
    if not (q.dtype is bf16 and q.get_device() == index and q.is_contiguous()):
        _lib.check_tensor(q, "q", bf16, index)
    if q.dim() != 3 or q.shape[2] != KV4_DIM:
        raise ValueError("q: [rows, heads, 128]")
    Tq, Hq, _ = q.shape
    if not (Hq > 0 and Hq % kv_heads == 0 and Hq // kv_heads <= 16 and max_q_len >= 0):
        raise ValueError("1 to 16 query heads per KV head; max_q_len is not negative")
    if out is not None:
        if not (out.dtype is bf16 and out.get_device() == index and out.is_contiguous()):
            _lib.check_tensor(out, "out", bf16, index)
        if out.numel() < q.numel():
            raise ValueError("out is smaller than q")
    return Tq, Hq, check_sequences(index, block_tables, q_start, ctx_lens)


def _attention_kv4(q, out, pool, layer, block_tables, q_start, ctx_lens, max_q_len, max_ctx, softmax_scale, workspace, rank, pages,
                   parts) -> torch.Tensor:
    pool.check(layer, rank)
    Hkv = pool.heads_per_rank
    Tq, Hq, n = _check_step(q, out, pool.index, Hkv, block_tables, q_start, ctx_lens, max_q_len)
    group = Hq // Hkv
    if pages is not None:  # every query row is an item of its own
        max_pages, rows, prefill = pages.shape[2], group, False
        planned, split_pages = plan_kv4(Tq, Hkv, 1, group, max_pages)
    else:
        max_pages, rows, prefill = -(-max_ctx // KV4_TOKENS), max_q_len * group, max_q_len * group >= TC_MIN_ROWS
        planned, split_pages = plan_kv4(n, Hkv, max_q_len, group, max_pages, Tq * Hq if prefill else 0)
    if parts is None:
        parts = planned
    elif prefill:
        _lib.require(parts >= 1, "nsplit")
        split_pages = -(--(-max_pages // parts) // 4) * 4
    else:
        _lib.require(parts >= 0 and parts != 1, "nsplit: 0, or two CTAs at least")
    po = pl = sh = None
    if parts > 1:
        if workspace is None:
            workspace = AttentionWorkspace(q.device)
        if prefill:
            workspace.ensure(Tq * Hq, parts, KV4_DIM)
        else:
            workspace.ensure(16 if rows <= 8 else 32, parts, KV4_DIM)
            sh = workspace.ensure_shared((Tq if pages is not None else n * -(-rows // 8)) * Hkv).data_ptr()
        _lib.require(workspace.part_o.get_device() == pool.index, "the workspace is on another device")
        po, pl = workspace.part_o.data_ptr(), workspace.part_lse.data_ptr()
        _lib.launch_count += 1  # the merge kernel
    if pages is None:
        _lib.call_on(pool.index, _lib.kv4_fn("daser_paged_attention_kv4"), "paged_attention_kv4", q.data_ptr(), out.data_ptr(), po, pl, sh,
                     pool.c_ptr, layer, rank, block_tables.data_ptr(), block_tables.shape[1], q_start.data_ptr(), ctx_lens.data_ptr(), n,
                     Tq, max_q_len, Hq, parts, split_pages, softmax_scale)
    else:
        _lib.call_on(pool.index, _lib.kv4_fn("daser_sparse_attention_kv4"), "sparse_attention_kv4", q.data_ptr(), out.data_ptr(), po, pl, sh,
                     pool.c_ptr, layer, rank, block_tables.data_ptr(), block_tables.shape[1], q_start.data_ptr(), ctx_lens.data_ptr(), n,
                     Tq, max_q_len, Hq, pages.data_ptr(), max_pages, parts, softmax_scale)
    return out


def select_pages(
    q: torch.Tensor,
    bounds: PageBounds,
    layer: int,
    block_tables: torch.Tensor,
    q_start: torch.Tensor,
    ctx_lens: torch.Tensor,
    max_q_len: int,
    max_ctx: int,
    num_pages: int,
    sink_pages: int = 1,
    recent_pages: int = 4,
    workspace: Optional[AttentionWorkspace] = None,
) -> torch.Tensor:
    """The pages every query row reads per KV head: int32 ``[Tq, Hkv, num_pages]``, logical pages in ascending order, -1
    behind the last.

    Always the first ``sink_pages`` and the last ``recent_pages`` (at least one: the page of the newest key, whose bounds need not be
    up to date) of the pages a row sees; the other places go to the highest estimates of the largest sum of the group's scores, the lower
    page first among equals.  The estimate is what the bounds give for the query rounded to int8 under one power of two: in whole numbers, and
    up to half a step per dim on either side of the bound itself.  A row that sees at most ``num_pages`` pages gets them all.  Rows of no
    sequence, and query tokens beyond ``max_q_len`` (at most 65535), are not set.  ``bounds`` have to cover the context
    (:func:`~daser_b200.ops.kv_ops.update_page_bounds`); other arguments as in :func:`paged_attention`.
    """
    (layers, nb, Hkv), dev = bounds.shape, bounds.index
    _lib.require(dev >= 0 and 0 <= layer < layers, "bounds on a CUDA device, layer inside them")
    Tq, Hq, n = _check_step(q, None, dev, Hkv, block_tables, q_start, ctx_lens, max_q_len)
    _lib.require(sink_pages >= 0 and recent_pages >= 1 and sink_pages + recent_pages <= num_pages, "sink_pages + recent_pages (at least 1) <= num_pages")
    pages = torch.empty((Tq, Hkv, num_pages), dtype=torch.int32, device=q.device)
    stride = max(1, -(-max_ctx // KV4_TOKENS))
    scores = None
    if stride > SELECT_ON_CHIP:
        need = Tq * Hkv * stride
        scores = workspace.ensure_scores(need) if workspace is not None else torch.empty(need, dtype=torch.float32, device=q.device)
        _lib.require(scores.get_device() == dev, "the workspace is on another device")
        scores = scores.data_ptr()
    _lib.call_on(dev, _lib.kv4_fn("daser_select_pages_kv4"), "select_pages_kv4", q.data_ptr(), bounds.codes.data_ptr(),
                 bounds.exps.data_ptr(), layer, nb, block_tables.data_ptr(), block_tables.shape[1], q_start.data_ptr(),
                 ctx_lens.data_ptr(), n, Tq, max_q_len, Hq, Hkv, scores, stride,
                 pages.data_ptr(), num_pages, sink_pages, recent_pages)
    return pages


def sparse_paged_attention(
    q: torch.Tensor,
    out: torch.Tensor,
    pool: PagedKV4Pool,
    layer: int,
    block_tables: torch.Tensor,
    q_start: torch.Tensor,
    ctx_lens: torch.Tensor,
    pages: torch.Tensor,
    max_q_len: int,
    softmax_scale: float,
    workspace: Optional[AttentionWorkspace] = None,
    rank: int = 0,
) -> torch.Tensor:
    """:func:`paged_attention` over the pages of ``pages`` (int32 ``[Tq, Hkv, n]``, as :func:`select_pages` gives them): row ``t``
    of a sequence attends the keys of its listed pages up to ``ctx_len - q_len + t``.  Every query row reads its own list: a
    decode operator, for one or a few query tokens per sequence, at most 65535 rows.  Pages have to be distinct within a list (one listed
    twice counts twice); entries outside the context are skipped.  Rows of no sequence, and query tokens beyond ``max_q_len``, are left alone."""
    _lib.require(isinstance(pool, PagedKV4Pool), "sparse attention works on a PagedKV4Pool")
    _lib.require(pages.dim() == 3 and pages.shape[2] >= 1 and tuple(pages.shape[:2]) == (q.shape[0], pool.heads_per_rank),
                 "pages: int32 [rows, KV heads, pages]")
    _lib.check_tensor(pages, "pages", torch.int32, pool.index)
    return _attention_kv4(q, out, pool, layer, block_tables, q_start, ctx_lens, max_q_len, 0, softmax_scale, workspace, rank, pages,
                          None)
