"""Python entry points of the KV kernels: codecs, fused restore, fused save, read-back, key bounds of pages.

``PagedKVPool`` describes a paged pool (one per tensor-parallel rank) with explicit
strides, so the kernels never assume an attention backend's layout; the reference
hard-codes FlashAttention's ``(2, num_blocks, block, heads, dim)`` and breaks on the
FlashInfer layout that Blackwell defaults to
(``daser/connector/daser_connector.py:404-408,544-547,627-630``).
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch

from daser_b200.ops import _lib
from daser_b200.ops._lib import KVJob, KVPool


def quantize_fp8b16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 CUDA tensor ``[..., D]`` -> (uint8 payload same shape, fp32 scales ``[..., D/16]``)."""
    assert x.is_cuda and x.dtype == torch.bfloat16 and x.is_contiguous()
    payload = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], x.shape[-1] // 16), dtype=torch.float32, device=x.device)
    _lib.check(
        _lib.lib().daser_quant_fp8b16(
            C.c_void_p(x.data_ptr()), C.c_void_p(payload.data_ptr()), C.c_void_p(scales.data_ptr()),
            C.c_int64(x.numel()), _lib.stream_ptr(),
        ),
        "quant_fp8b16",
    )
    return payload, scales


def dequantize_fp8b16(payload: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    assert payload.is_cuda and payload.dtype == torch.uint8 and payload.is_contiguous()
    assert scales.dtype == torch.float32 and scales.is_contiguous()
    out = torch.empty(payload.shape, dtype=torch.bfloat16, device=payload.device)
    _lib.check(
        _lib.lib().daser_dequant_fp8b16(
            C.c_void_p(payload.data_ptr()), C.c_void_p(scales.data_ptr()), C.c_void_p(out.data_ptr()),
            C.c_int64(payload.numel()), _lib.stream_ptr(),
        ),
        "dequant_fp8b16",
    )
    return out


@dataclass
class PagedKVPool:
    """A paged KV pool as the kernels see it.

    ``payload_ptrs[r]`` / ``scale_ptrs[r]`` are rank ``r``'s base addresses as mapped into
    *this* process (peers' pools are peer-mapped).  Strides are in elements of the payload
    dtype; the scale tensor has the same shape with ``dim / 16`` as its last dimension.
    """

    payload_ptrs: Sequence[int]
    scale_ptrs: Sequence[int]
    stride_layer: int
    stride_block: int
    stride_kv: int
    stride_tok: int
    stride_head: int
    num_blocks: int
    heads_per_rank: int
    is_fp8: bool
    keepalive: list = field(default_factory=list)

    @property
    def n_ranks(self) -> int:
        return len(self.payload_ptrs)

    def c_struct(self) -> KVPool:
        p = KVPool()
        for r, ptr in enumerate(self.payload_ptrs):
            p.payload[r] = ptr
        for r, ptr in enumerate(self.scale_ptrs):
            p.scales[r] = ptr
        p.stride_layer, p.stride_block = self.stride_layer, self.stride_block
        p.stride_kv, p.stride_tok, p.stride_head = self.stride_kv, self.stride_tok, self.stride_head
        p.num_blocks, p.n_ranks = self.num_blocks, self.n_ranks
        p.heads_per_rank, p.pool_is_fp8 = self.heads_per_rank, int(self.is_fp8)
        return p

    @classmethod
    def from_tensors(
        cls,
        payloads: Sequence[torch.Tensor],
        scales: Optional[Sequence[torch.Tensor]] = None,
        layout: str = "LNKHTD",
    ) -> "PagedKVPool":
        """Build from per-rank tensors.

        ``layout`` names the dimension order of each payload tensor with the letters
        L (layer), N (block), K (k/v), T (token), H (head), D (dim), e.g. ``LNKHTD`` for
        the native engine's head-major pool or ``LKNTHD`` for a stack of vLLM
        FlashAttention layers ``(2, num_blocks, block, heads, dim)``.
        """
        t = payloads[0]
        assert len(layout) == t.dim() and layout[-1] == "D" and t.stride(-1) == 1
        st = {ch: t.stride(i) for i, ch in enumerate(layout)}
        sh = {ch: t.shape[i] for i, ch in enumerate(layout)}
        is_fp8 = t.dtype in (torch.uint8, torch.float8_e4m3fn)
        if is_fp8 and scales is None:
            raise ValueError("an fp8 pool needs its scale tensors")
        return cls(
            payload_ptrs=[p.data_ptr() for p in payloads],
            scale_ptrs=[s.data_ptr() for s in scales] if scales is not None else [0] * len(payloads),
            stride_layer=st.get("L", 0),
            stride_block=st["N"],
            stride_kv=st["K"],
            stride_tok=st["T"],
            stride_head=st["H"],
            num_blocks=sh["N"],
            heads_per_rank=sh["H"],
            is_fp8=is_fp8,
            keepalive=[list(payloads), list(scales) if scales is not None else None],
        )


def quantize_fp4b16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 CUDA tensor ``[..., D]`` -> (uint8 codes ``[..., D/2]``, uint8 scales ``[..., D/16]``); the format is
    described in :mod:`daser_b200.kv.codec`."""
    _lib.require(x.is_cuda and x.shape[-1] % 16 == 0, "quantize_fp4b16: needs a CUDA tensor whose last dimension is a multiple of 16")
    _lib.check_tensor(x, "x", torch.bfloat16, x.get_device())
    codes = torch.empty((*x.shape[:-1], x.shape[-1] // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], x.shape[-1] // 16), dtype=torch.uint8, device=x.device)
    _lib.call_on(x.get_device(), _lib.kv4_fn("daser_quant_fp4b16"), "quant_fp4b16", x.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                 x.numel())
    return codes, scales


def dequantize_fp4b16(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values that :func:`quantize_fp4b16`'s result stands for, in bf16 (exact)."""
    _lib.require(codes.is_cuda and tuple(scales.shape) == (*codes.shape[:-1], codes.shape[-1] // 8) and codes.shape[-1] % 8 == 0,
                 "dequantize_fp4b16: codes [..., D/2] and scales [..., D/16] on a CUDA device")
    _lib.check_tensor(codes, "codes", torch.uint8, codes.get_device())
    _lib.check_tensor(scales, "scales", torch.uint8, codes.get_device())
    out = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=torch.bfloat16, device=codes.device)
    _lib.call_on(codes.get_device(), _lib.kv4_fn("daser_dequant_fp4b16"), "dequant_fp4b16", codes.data_ptr(), scales.data_ptr(),
                 out.data_ptr(), out.numel())
    return out


KV4_RECORD = 2304  # bytes of one page (16 tokens) of one KV head: ``ops/csrc/kv4.h``
KV4_TOKENS, KV4_DIM = 16, 128


class PagedKV4Pool:
    """A paged pool in the 4-bit format: one 2304-byte record per (layer, block, KV head), 0.5625 bytes per element
    (:class:`PagedKVPool` holds 1.25 in fp8 and 2 in bf16).

    It takes the place of a :class:`PagedKVPool` in ``rope_kv_write``, :func:`kv_restore`, :func:`kv_save` and
    ``paged_attention``, and is what :func:`kv_read`, :func:`update_page_bounds` and
    ``sparse_paged_attention`` work on.  16 tokens per block, head_dim 128.  ``record_ptrs[r]`` is rank ``r``'s base
    address as mapped into this process; the pool's kernels run on ``device``.

    Slots written by one call have to be distinct, and so do the blocks of one restore: of two tokens with the same slot each store
    of a few bytes is one's or the other's, so that a group may end up with the codes of one under the scale of the other.
    """

    def __init__(self, record_ptrs: Sequence[int], stride_layer: int, stride_block: int, stride_head: int, num_layers: int,
                 num_blocks: int, heads_per_rank: int, device: torch.device, keepalive: Optional[list] = None) -> None:
        _lib.require(1 <= len(record_ptrs) <= _lib.MAX_RANKS, f"1 to {_lib.MAX_RANKS} ranks")
        _lib.require(all(int(p) % 16 == 0 for p in record_ptrs) and all(x % 16 == 0 for x in (stride_layer, stride_block, stride_head)),
                     "records have to start on 16-byte boundaries")
        _lib.require(min(num_layers, num_blocks, heads_per_rank) > 0, "a 4-bit pool needs layers, blocks and heads")
        self.record_ptrs = [int(p) for p in record_ptrs]
        self.stride_layer, self.stride_block, self.stride_head = stride_layer, stride_block, stride_head
        self.num_layers, self.num_blocks, self.heads_per_rank = num_layers, num_blocks, heads_per_rank
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.index = self.device.index if self.device.type == "cuda" else -1
        self.keepalive = keepalive
        c = _lib.KV4Pool()
        for r, ptr in enumerate(self.record_ptrs):
            c.records[r] = ptr
        c.stride_layer, c.stride_block, c.stride_head = stride_layer, stride_block, stride_head
        c.num_layers, c.num_blocks, c.n_ranks, c.heads_per_rank = num_layers, num_blocks, len(self.record_ptrs), heads_per_rank
        self._c = c
        self.c_ptr = C.addressof(c)  # entry points copy the block before they return

    @property
    def n_ranks(self) -> int:
        return len(self.record_ptrs)

    @classmethod
    def from_tensors(cls, records: Sequence[torch.Tensor]) -> "PagedKV4Pool":
        """From one uint8 tensor ``[layers, blocks, heads, 2304]`` per rank; records are contiguous, the other
        strides are free (multiples of 16)."""
        t = records[0]
        for r in records:
            _lib.require(r.dtype == torch.uint8 and r.dim() == 4 and r.shape[3] == KV4_RECORD and r.stride(3) == 1,
                         "records: uint8 [layers, blocks, heads, 2304] with contiguous records")
            _lib.require(r.shape == t.shape and r.stride() == t.stride(), "every rank's records need the same shape and strides")
        return cls([r.data_ptr() for r in records], t.stride(0), t.stride(1), t.stride(2), t.shape[0], t.shape[1], t.shape[2],
                   t.device, [list(records)])

    @classmethod
    def zeros(cls, num_layers: int, num_blocks: int, num_heads: int, device) -> "PagedKV4Pool":
        return cls.from_tensors([torch.zeros(num_layers, num_blocks, num_heads, KV4_RECORD, dtype=torch.uint8, device=device)])

    def c_struct(self):
        """What the operators of a :class:`PagedKVPool` alone ask for."""
        raise ValueError("this operator takes a PagedKVPool, not a 4-bit pool")

    def check(self, layer: int, rank: int) -> None:
        if self.index < 0:
            raise ValueError("the pool's kernels need a CUDA device")
        if not (0 <= layer < self.num_layers and 0 <= rank < len(self.record_ptrs)):
            raise ValueError(f"layer {layer} or rank {rank} outside the pool")


def kv_read(pool: PagedKV4Pool, layer: int, slot_mapping: torch.Tensor, rank: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values bf16 ``[T, heads, 128]`` of the tokens at ``slot_mapping`` (int64 ``[T]``, block * 16 + offset,
    as ``rope_kv_write`` takes it), as the pool holds them; a negative slot reads as zeros."""
    pool.check(layer, rank)
    _lib.check_tensor(slot_mapping, "slot_mapping", torch.int64, pool.index)
    T = slot_mapping.numel()
    k = torch.empty((T, pool.heads_per_rank, KV4_DIM), dtype=torch.bfloat16, device=pool.device)
    v = torch.empty_like(k)
    _lib.call_on(pool.index, _lib.kv4_fn("daser_kv4_read"), "kv4_read", pool.c_ptr, layer, rank, slot_mapping.data_ptr(),
                 k.data_ptr(), v.data_ptr(), T)
    return k, v


class PageBounds:
    """Bounds of the keys of every page of a 4-bit pool: what ``select_pages`` scores.

    ``codes`` int8 ``[layers, blocks, heads, 2, 128]`` (high, low) and ``exps`` int8 ``[layers, blocks, heads]``: the keys of a
    page lie between ``codes[..., 1, :] * 2^exp`` and ``codes[..., 0, :] * 2^exp``, 257 bytes per page and head.
    """

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor) -> None:
        _lib.require(codes.dim() == 5 and tuple(codes.shape[3:]) == (2, KV4_DIM) and tuple(exps.shape) == tuple(codes.shape[:3]),
                     "codes [layers, blocks, heads, 2, 128], exps [layers, blocks, heads]")
        _lib.check_tensor(codes, "codes", torch.int8, codes.get_device())
        _lib.check_tensor(exps, "exps", torch.int8, codes.get_device())
        _lib.require(codes.data_ptr() % 16 == 0, "codes have to start on a 16-byte boundary")
        self.codes, self.exps = codes, exps
        self.index = codes.get_device()
        self.shape = tuple(exps.shape)  # (layers, blocks, heads)

    @classmethod
    def for_pool(cls, pool: PagedKV4Pool) -> "PageBounds":
        shape = (pool.num_layers, pool.num_blocks, pool.heads_per_rank)
        return cls(torch.zeros(*shape, 2, KV4_DIM, dtype=torch.int8, device=pool.device),
                   torch.zeros(shape, dtype=torch.int8, device=pool.device))

    def read(self, layer: int, blocks: torch.Tensor) -> torch.Tensor:
        """The bounds of ``blocks`` (int32, any shape) as float32 ``[..., heads, 2, 128]`` (high, low); of a page with a key that is not
        finite, infinities."""
        layers, nb, heads = self.shape
        _lib.require(self.index >= 0 and 0 <= layer < layers, "bounds on a CUDA device, layer inside them")
        _lib.check_tensor(blocks, "blocks", torch.int32, self.index)
        out = torch.empty((*blocks.shape, heads, 2, KV4_DIM), dtype=torch.float32, device=self.exps.device)
        _lib.call_on(self.index, _lib.kv4_fn("daser_kv4_bounds_read"), "kv4_bounds_read", self.codes.data_ptr(), self.exps.data_ptr(), layer,
                     nb, heads, blocks.data_ptr(), out.data_ptr(), blocks.numel())
        return out


def check_sequences(index: int, block_tables: torch.Tensor, q_start: torch.Tensor, ctx_lens: torch.Tensor) -> int:
    """How many sequences a step's tables describe (contiguous int32 tensors on CUDA device ``index``)."""
    i32 = torch.int32
    if not (block_tables.dtype is i32 and q_start.dtype is i32 and ctx_lens.dtype is i32
            and block_tables.get_device() == index and q_start.get_device() == index and ctx_lens.get_device() == index
            and block_tables.is_contiguous() and q_start.is_contiguous() and ctx_lens.is_contiguous()):
        for t, name in ((block_tables, "block_tables"), (q_start, "q_start"), (ctx_lens, "ctx_lens")):
            _lib.check_tensor(t, name, i32, index)
    n = ctx_lens.numel()
    if block_tables.dim() != 2 or block_tables.shape[0] < n or q_start.numel() != n + 1:
        raise ValueError("one row of block_tables per sequence, one entry of q_start more")
    return n


def update_page_bounds(pool: PagedKV4Pool, bounds: PageBounds, layer: int, block_tables: torch.Tensor, q_start: torch.Tensor,
                       ctx_lens: torch.Tensor, max_q_len: int, rank: int = 0) -> None:
    """Recompute the bounds of every page that holds one of a sequence's last ``q_start[s+1] - q_start[s]`` tokens (the step's
    new ones; after a restore, the restored ones).  Arguments as ``paged_attention`` takes them; call it behind the step's
    ``rope_kv_write``.  ``max_q_len`` has to be at least the most tokens of a sequence: pages beyond it are not looked at.  Of a page the
    tokens below ``ctx_len`` count; where sequences share a page that the call recomputes, they have to see the same tokens of it."""
    pool.check(layer, rank)
    _lib.require(bounds.shape == (pool.num_layers, pool.num_blocks, pool.heads_per_rank) and bounds.index == pool.index,
                 "the bounds belong to a pool of another shape or device")
    n = check_sequences(pool.index, block_tables, q_start, ctx_lens)
    _lib.call_on(pool.index, _lib.kv4_fn("daser_kv4_page_bounds"), "kv4_page_bounds", pool.c_ptr, layer, rank, bounds.codes.data_ptr(),
                 bounds.exps.data_ptr(), block_tables.data_ptr(), block_tables.shape[1], q_start.data_ptr(), ctx_lens.data_ptr(), n,
                 max_q_len)


@dataclass
class KVWorkList:
    """Device-side work list of one restore/save launch."""

    slot_ptrs: torch.Tensor  # int64 [n] addresses of slot images
    block_ids: torch.Tensor  # int32 [n]
    deltas: Optional[torch.Tensor] = None  # int32 [n]

    @property
    def n_slots(self) -> int:
        return int(self.block_ids.numel())


def _job(work, geo, image_is_fp8, cos_sin, status, rank=0) -> KVJob:
    j = KVJob()
    j.slot_ptr = work.slot_ptrs.data_ptr()
    j.block_id = work.block_ids.data_ptr()
    j.delta = work.deltas.data_ptr() if work.deltas is not None else None
    j.cos_sin = cos_sin.data_ptr() if cos_sin is not None else None
    j.status = status.data_ptr() if status is not None else None
    j.max_pos = int(cos_sin.shape[0]) if cos_sin is not None else 0
    j.n_slots = work.n_slots
    j.num_layers, j.num_kv_heads = geo.num_layers, geo.num_kv_heads
    j.head_dim, j.block_tokens = geo.head_dim, geo.block_tokens
    j.image_is_fp8 = int(image_is_fp8)
    j.rank = rank
    return j


def _check_work4(work: KVWorkList, geo, pool: PagedKV4Pool, cos_sin, status) -> None:
    """The tensors of a restore or save of a 4-bit pool: the kernels read them as they are described here."""
    for t, name, dtype in ((work.slot_ptrs, "slot_ptrs", torch.int64), (work.block_ids, "block_ids", torch.int32),
                           (work.deltas, "deltas", torch.int32), (cos_sin, "cos_sin", torch.float32), (status, "status", torch.int32)):
        if t is not None:
            _lib.check_tensor(t, name, dtype, pool.index)
    n = work.n_slots
    _lib.require(work.slot_ptrs.numel() == n and (work.deltas is None or work.deltas.numel() == n), "one entry per slot in slot_ptrs and deltas")
    _lib.require(cos_sin is None or (cos_sin.dim() == 2 and cos_sin.shape[1] == KV4_DIM), "cos_sin: [positions, 128]")
    _lib.require(status is None or status.numel() >= 2, "status: two words")
    _lib.require(geo.codec == "fp8b16" or geo.dtype_bytes == 2, "images of a 4-bit pool are fp8b16 or bf16")


def kv_restore(work: KVWorkList, geo, pool: PagedKVPool | PagedKV4Pool, cos_sin: Optional[torch.Tensor],
               status: Optional[torch.Tensor] = None, stream=None, layer_begin: int = 0,
               layer_count: int = 0) -> None:
    """Slot images -> paged pools of every rank: dequantise, rotate keys by ``deltas``, scatter.

    ``layer_begin`` / ``layer_count`` restrict the launch to a range of layers (0 = through the
    last one): a restore can then run group by group while the storage reads of later layers
    are still in flight and the model already computes on the earlier ones.

    Into a :class:`PagedKV4Pool` the (rotated) values are quantised to 4 bits on the way."""
    job = _job(work, geo, geo.codec == "fp8b16", cos_sin, status)
    job.layer_begin, job.layer_count = int(layer_begin), int(layer_count)
    if isinstance(pool, PagedKV4Pool):
        pool.check(0, 0)
        _check_work4(work, geo, pool, cos_sin, status)
        _lib.call_on(pool.index, _lib.kv4_fn("daser_kv4_restore"), "kv4_restore", C.addressof(job), pool.c_ptr, stream=stream)
        return
    pool_c = pool.c_struct()
    _lib.check(_lib.lib().daser_kv_restore(C.byref(job), C.byref(pool_c), _lib.stream_ptr(stream)), "kv_restore")


def kv_save(work: KVWorkList, geo, pool: PagedKVPool | PagedKV4Pool, rank: int = 0,
            status: Optional[torch.Tensor] = None, stream=None) -> None:
    """Rank ``rank``'s blocks -> its head slice of each slot image (compressing for fp8b16).

    Out of a :class:`PagedKV4Pool` a raw image gets the 4-bit values as they stand (exact in bf16), an fp8b16 image the
    same values quantised once more."""
    job = _job(work, geo, geo.codec == "fp8b16", None, status, rank)
    if isinstance(pool, PagedKV4Pool):
        pool.check(0, rank)
        _check_work4(work, geo, pool, None, status)
        _lib.call_on(pool.index, _lib.kv4_fn("daser_kv4_save"), "kv4_save", C.addressof(job), pool.c_ptr, stream=stream)
        return
    pool_c = pool.c_struct()
    _lib.check(_lib.lib().daser_kv_save(C.byref(job), C.byref(pool_c), _lib.stream_ptr(stream)), "kv_save")


def copy_rows(dst_ptr: int, src_ptr: int, pitch: int, width: int, rows: int, stream=None) -> None:
    """``rows`` runs of ``width`` bytes, ``pitch`` bytes apart on both sides, copied by the copy
    engine on ``stream`` (either side may be pinned host or device memory)."""
    code = _lib.lib().daser_copy_rows(C.c_void_p(dst_ptr), C.c_void_p(src_ptr), C.c_int64(pitch), C.c_int64(width),
                                      C.c_int64(rows), _lib.stream_ptr(stream))
    if code != 0:
        raise _lib.KernelError(f"copy_rows: CUDA error {code}" if code > 0 else "copy_rows: bad argument")


def rope_table(max_pos: int, inv_freq, device) -> torch.Tensor:
    """``[max_pos, D]`` fp32: cos in ``[:, :D/2]``, sin in ``[:, D/2:]`` (angles in fp64)."""
    inv = torch.as_tensor(inv_freq, dtype=torch.float64)
    ang = torch.arange(max_pos, dtype=torch.float64).unsqueeze(1) * inv.unsqueeze(0)
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32).to(device)
