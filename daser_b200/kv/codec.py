"""CPU reference for the block-scaled fp8 codec, RoPE and slot packing.

This is the oracle for the CUDA kernels (``ops/csrc/kv_codec.cu``,
``kv_restore.cu``, ``kv_save.cu``) and the implementation used by the CPU-only
engine.  The reference stores KV raw and has no codec, RoPE or repacking code
(``daser/connector/daser_connector.py:625-632`` is a byte copy), so everything
here is new.

fp8b16: groups of 16 consecutive ``dim`` elements share one fp32 scale
``s = absmax / 448`` (``s = 1`` for an all-zero group); the payload is
``rne_e4m3(x * (448 / absmax))``.  Dequantisation is ``q * s``.  All arithmetic
is IEEE fp32 so the CUDA kernels reproduce it bit for bit.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from daser_b200.config import CODEC_RAW, FP8_GROUP
from daser_b200.kv.layout import KVGeometry

E4M3_MAX = 448.0


def quantize_fp8b16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x[..., D]`` (any float dtype) -> (uint8 e4m3 payload ``[..., D]``, fp32 scales ``[..., D/16]``)."""
    if x.shape[-1] % FP8_GROUP:
        raise ValueError("last dimension must be a multiple of 16")
    xf = x.detach().to(torch.float32)
    g = xf.reshape(*xf.shape[:-1], xf.shape[-1] // FP8_GROUP, FP8_GROUP)
    absmax = g.abs().amax(dim=-1, keepdim=True)
    nz = absmax > 0
    safe = torch.where(nz, absmax, torch.ones_like(absmax))
    # tensor / tensor so both are true IEEE divisions (scalar operands make torch multiply
    # by a reciprocal, which rounds differently from the kernels' div.rn)
    top = torch.full_like(safe, E4M3_MAX)
    inv = torch.where(nz, torch.div(top, safe), torch.ones_like(absmax))
    scale = torch.where(nz, torch.div(safe, top), torch.ones_like(absmax))
    q = (g * inv).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(x.shape), scale.squeeze(-1).contiguous()


def dequantize_fp8b16(
    payload: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32
) -> torch.Tensor:
    q = payload.view(torch.float8_e4m3fn).to(torch.float32)
    g = q.reshape(*q.shape[:-1], q.shape[-1] // FP8_GROUP, FP8_GROUP)
    return (g * scales.to(torch.float32).unsqueeze(-1)).reshape(payload.shape).to(dtype)


# -- the 4-bit format ---------------------------------------------------------------
#
# fp4b16 (oracle of ``ops/csrc/fp4.cuh``): groups of 16 consecutive ``dim`` elements share one scale.  A value is e2m1 (0, 0.5, 1,
# 1.5, 2, 3, 4, 6 with a sign, two to a byte, the even element in the low half); a scale is 8 bits, the upper 8 of the 15
# magnitude bits of an f16 (five exponent and three mantissa bits).  ``s = round4(f16(absmax * fl(1/6)))``, four significant bits,
# at most 10240; the payload is ``rne_e2m1(fl(x / s))``, saturating at 6.  A group with an infinity or a NaN has
# scale byte 255 and reads back as NaN.

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP4_MAX_SCALE = 10240.0


def fp4_scale_values(scales: torch.Tensor) -> torch.Tensor:
    """uint8 scale bytes -> the fp32 values they stand for."""
    return (scales.to(torch.int32) << 7).to(torch.int16).view(torch.float16).to(torch.float32)


def quantize_fp4b16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x[..., D]`` (any float dtype) -> (uint8 codes ``[..., D/2]``, uint8 scales ``[..., D/16]``)."""
    if x.shape[-1] % FP8_GROUP:
        raise ValueError("last dimension must be a multiple of 16")
    xf = x.detach().to(torch.float32)
    g = xf.reshape(*xf.shape[:-1], xf.shape[-1] // FP8_GROUP, FP8_GROUP)
    absmax = g.abs().amax(dim=-1)  # propagates NaN
    t = (absmax * torch.tensor(1.0 / 6.0, dtype=torch.float32)).clamp(max=FP4_MAX_SCALE)
    bits = t.to(torch.float16).view(torch.int16).to(torch.int32)
    byte = (bits + 63 + ((bits >> 7) & 1)) >> 7
    byte = torch.where(torch.isfinite(absmax), byte, torch.full_like(byte, 255)).to(torch.uint8)
    s = fp4_scale_values(byte).unsqueeze(-1)
    ok = s > 0  # false for a group that rounds to nothing and for one that is not finite
    y = torch.where(ok, torch.div(g, torch.where(ok, s, torch.ones_like(s))), torch.copysign(torch.zeros_like(g), g))
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    a = y.abs()
    code = torch.bucketize(a, borders)  # borders below a: a tie goes down ...
    for i in (1, 3, 5):  # ... except where the code above is the even one
        code = torch.where(a == borders[i], torch.full_like(code, i + 1), code)
    code = (code.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def dequantize_fp4b16(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that (codes ``[..., D/2]``, scales ``[..., D/16]``) stand for (exact in bf16 and fp32)."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1))
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).reshape(*codes.shape[:-1], -1)
    g = v.reshape(*scales.shape, FP8_GROUP)
    return (g * fp4_scale_values(scales).unsqueeze(-1)).reshape(v.shape).to(dtype)


def pack_kv4_records(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """``k, v [..., 16, 128]`` of one page -> its record ``[..., 2304]`` (uint8), the layout of ``ops/csrc/kv4.h``."""
    lead = k.shape[:-2]
    (kc, ks), (vc, vs) = quantize_fp4b16(k), quantize_fp4b16(v)
    vc = vc.reshape(*lead, 2, 8, 8, 8).transpose(-3, -2)  # [token / 8][group][token % 8][8]
    vs = vs.reshape(*lead, 2, 8, 8).transpose(-2, -1)
    return torch.cat([t.reshape(*lead, -1) for t in (kc, vc, ks, vs)], dim=-1)


def unpack_kv4_records(records: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Inverse of :func:`pack_kv4_records`: fp32 ``k, v [..., 16, 128]``."""
    lead = records.shape[:-1]
    kc, vc, ks, vs = records.split([1024, 1024, 128, 128], dim=-1)
    k = dequantize_fp4b16(kc.reshape(*lead, 16, 64), ks.reshape(*lead, 16, 8))
    vc = vc.reshape(*lead, 2, 8, 8, 8).transpose(-3, -2).reshape(*lead, 16, 64)
    vs = vs.reshape(*lead, 2, 8, 8).transpose(-2, -1).reshape(*lead, 16, 8)
    return k, dequantize_fp4b16(vc, vs)


# -- RoPE ---------------------------------------------------------------------------


def rope_cos_sin(
    positions: torch.Tensor, inv_freq: Sequence[float] | torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor]:
    """cos/sin of ``positions[:, None] * inv_freq[None, :]`` computed in fp64, returned fp32."""
    inv = torch.as_tensor(inv_freq, dtype=torch.float64)
    ang = positions.to(torch.float64).reshape(-1, 1) * inv.reshape(1, -1)
    return ang.cos().to(torch.float32), ang.sin().to(torch.float32)


def rope_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half (NeoX) RoPE.  ``x[T, H, D]``, ``cos/sin[T, D/2]`` (or ``[1, D/2]``)."""
    half = x.shape[-1] // 2
    xf = x.to(torch.float32)
    x1, x2 = xf[..., :half], xf[..., half:]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def rope_delta_rotate(
    k: torch.Tensor, delta: int, inv_freq: Sequence[float] | torch.Tensor
) -> torch.Tensor:
    """Move already-rotated keys ``k[..., H, D]`` by ``delta`` positions."""
    if delta == 0:
        return k.to(torch.float32)
    cos, sin = rope_cos_sin(torch.tensor([delta]), inv_freq)
    flat = k.reshape(-1, k.shape[-2], k.shape[-1])
    return rope_rotate(flat, cos, sin).reshape(k.shape)


# -- slot images ------------------------------------------------------------------------


def pack_layer(geo: KVGeometry, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """``k, v`` of shape ``[block_tokens, H, D]`` -> the layer's bytes (uint8, 1-D)."""
    kv = torch.stack([k, v])  # [2, B, H, D]
    if geo.codec == CODEC_RAW:
        want = {2: (torch.bfloat16, torch.float16), 4: (torch.float32,), 1: (torch.uint8,)}
        if kv.dtype not in want[geo.dtype_bytes]:
            raise ValueError(f"dtype {kv.dtype} does not match dtype_bytes={geo.dtype_bytes}")
        return kv.contiguous().view(torch.uint8).reshape(-1)
    payload, scales = quantize_fp8b16(kv)
    return torch.cat([payload.reshape(-1), scales.reshape(-1).view(torch.uint8)])


def unpack_layer(
    geo: KVGeometry, raw: torch.Tensor, dtype: torch.dtype = torch.float32
) -> tuple[torch.Tensor, torch.Tensor]:
    """Inverse of :func:`pack_layer`; returns ``k, v`` ``[block_tokens, H, D]`` in ``dtype``."""
    shape = (2, geo.block_tokens, geo.num_kv_heads, geo.head_dim)
    raw = raw.reshape(-1)
    if raw.numel() != geo.layer_size:
        raise ValueError(f"layer region has {raw.numel()} bytes, expected {geo.layer_size}")
    if geo.codec == CODEC_RAW:
        src = {2: torch.bfloat16, 4: torch.float32}[geo.dtype_bytes]
        if dtype in (torch.float16,) and geo.dtype_bytes == 2:
            src = torch.float16
        kv = raw.contiguous().view(src).reshape(shape).to(dtype)
    else:
        n = geo.payload_bytes_per_layer
        payload = raw[:n].reshape(shape)
        scales = raw[n:].contiguous().view(torch.float32).reshape(*shape[:-1], -1)
        kv = dequantize_fp8b16(payload, scales, dtype)
    return kv[0], kv[1]


def pack_slot(geo: KVGeometry, ks: Sequence[torch.Tensor], vs: Sequence[torch.Tensor]) -> torch.Tensor:
    """One slot image from per-layer ``k, v`` blocks."""
    return torch.cat([pack_layer(geo, k, v) for k, v in zip(ks, vs)])


def restore_slot_reference(
    geo: KVGeometry,
    slot: torch.Tensor,
    delta: int,
    inv_freq: Sequence[float] | torch.Tensor,
    head_range: Optional[tuple[int, int]] = None,
    dtype: torch.dtype = torch.float32,
) -> list[tuple[torch.Tensor, torch.Tensor]]:
    """Oracle for the restore kernel on one slot: per layer ``(k_rotated, v)``.

    ``head_range=(first, count)`` selects one TP rank's heads.
    """
    out = []
    for layer in range(geo.num_layers):
        raw = slot[layer * geo.layer_size : (layer + 1) * geo.layer_size]
        k, v = unpack_layer(geo, raw, torch.float32)
        k = rope_delta_rotate(k, delta, inv_freq)
        if head_range is not None:
            h0, hn = head_range
            k, v = k[:, h0 : h0 + hn], v[:, h0 : h0 + hn]
        out.append((k.to(dtype), v.to(dtype)))
    return out
