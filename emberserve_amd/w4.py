"""Projections over 4-bit weights with group scales, for decode batches: `ember_w4_linear` and
`ember_w4_gate_up_silu` (libember_ops.so). The reference's weight-only path holds 8 bits
(emberserve/model/quant.py:113); this one halves a decode step's weight bytes again.

    qweight [N, K / 2] uint8, two codes to a byte (the even k in the low nibble)
    scales [N, K / G] fp16/bf16, zeros [N, K / G] uint8 in 0..15 or None (8 everywhere)
    w[n, k] = scales[n, k // G] * (code[n, k] - zeros[n, k // G])
    pack_w4(qweight, scales, zeros) -> PackedW4, once, when a model is loaded
    linear_w4(x [..., K], packed, bias) -> round(x @ w.T + bias) [..., N]
    gate_up_silu_w4(x [..., H], pack_w4_gate_up(...)) -> round(silu(gate) * up) [..., I]

The group G is K // scales.shape[-1]: 32, 64 or a multiple of 128. A leading expert dimension packs the
weights of `moe.fused_moe`. x is fp16 or bf16, whatever the scales' dtype.

Numerics: the codes enter MFMA as exact fp16/bf16 integers, the products are summed in fp32, a group's
sum is scaled in fp32, and the result is rounded once; gate_up_silu_w4 does not round between the
projection and the activation, as the 16-bit pair does. A row of x with an infinity gives NaN, and so may
one whose 31-fold sum over a group overflows fp32 (bf16 values of 2^116 and more).

A pass over the weight serves 64 tokens; more tokens take more passes, so at prefill sizes
`PackedW4.dequantize` and a library GEMM are the faster way. CPU tensors, or `EMBERSERVE_FUSED_OPS=0`, take
the eager forms.
"""

from __future__ import annotations

from ctypes import byref, c_int64

import torch
import torch.nn.functional as F
from torch import Tensor

from . import _lib
from ._scratch import SharedScratch
from .ops import _check_indices, _launch, fused_enabled

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16)
MAX_ROW_STRIDE = 1 << 23  # elements: 64 tokens are addressed with 32-bit offsets; rows farther apart are copied


def quantize_w4(weight: Tensor, group_size: int = 128, *, symmetric: bool = True) -> tuple[Tensor, Tensor, Tensor | None]:
    """(qweight, scales, zeros) of weight [..., N, K] (fp16/bf16) by rounding to nearest within each
    group: scale max|w| / 7 around 8 when symmetric (zeros None), else (max - min) / 15 with a zero
    point. The scales have the weight's dtype."""
    if weight.dtype not in SUPPORTED_DTYPES or weight.dim() < 2:
        raise ValueError(f"quantize_w4: an fp16/bf16 weight [..., N, K] expected, got {tuple(weight.shape)} "
                         f"{weight.dtype}")
    k = weight.shape[-1]
    _check_group(k, group_size)
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("quantize_w4: the weight has infinities or NaN")
    w = weight.float().reshape(*weight.shape[:-1], k // group_size, group_size)
    # a group of zeros: any scale, codes at the zero point. fp16 weights under 2^-11 have scales below
    # its normal range, whose smallest step is 2^-24
    tiny = 2.0 ** -24 if weight.dtype == torch.float16 else torch.finfo(weight.dtype).tiny
    if symmetric:
        scales = (w.abs().amax(-1) / 7.0).clamp_min(tiny).to(weight.dtype)
        zero = torch.full_like(scales, 8.0, dtype=torch.float32)
    else:
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        scales = ((hi - lo) / 15.0).clamp_min(tiny).to(weight.dtype)
        zero = torch.round(-lo / scales.float()).clamp(0, 15)
    q = torch.round(w / scales.float()[..., None] + zero[..., None]).clamp(0, 15).to(torch.uint8)
    q = q.reshape(*weight.shape[:-1], k // 2, 2)
    return q[..., 0] | (q[..., 1] << 4), scales, None if symmetric else zero.to(torch.uint8)


def dequantize_w4(qweight: Tensor, scales: Tensor, zeros: Tensor | None = None,
                  dtype: torch.dtype | None = None) -> Tensor:
    """The weight [..., N, K] in `dtype` (default: the scales')."""
    q = torch.stack((qweight & 15, qweight >> 4), dim=-1).float()
    q = q.reshape(*scales.shape, -1)
    q = q - (8.0 if zeros is None else zeros.float()[..., None])
    w = (q * scales.float()[..., None]).reshape(*qweight.shape[:-1], 2 * qweight.shape[-1])
    return w.to(scales.dtype if dtype is None else dtype)


class PackedW4:
    """A 4-bit weight [rows, k] (or [num_experts, rows, k]; gate_up: [2 rows, k], gate rows first) as the
    kernels read it: slabs of 16 rows, each one contiguous stream of MFMA operand fragments with the
    scales and zero points of every 128 k beside them. Made by `pack_w4` or `pack_w4_gate_up`; on
    the CPU it holds the unpacked parts for the eager forms."""

    def __init__(self, packed: Tensor | None, parts: tuple | None, num_experts: int | None, rows: int, k: int,
                 group: int, gate_up: bool, device: torch.device) -> None:
        self.packed, self.parts, self.num_experts = packed, parts, num_experts
        self.rows, self.k, self.group, self.gate_up, self.device = rows, k, group, gate_up, device
        # what the native host path takes of a projection's weight (None: left to the wrappers)
        self.projection = (rows, k, group, int(gate_up)) if packed is not None and num_experts is None else None

    def dequantize(self, dtype: torch.dtype) -> Tensor:
        """The weight [..., N, K] in `dtype`, from the packed form: for the eager forms and for a
        library GEMM at prefill sizes."""
        if self.parts is not None:
            return dequantize_w4(*self.parts, dtype=dtype)
        gpb, nb, e = max(1, 128 // self.group), -(-self.k // 128), self.num_experts or 1
        flat = self.packed.view(e, -1, 1024 * nb + -(-64 * gpb * nb // 128) * 128)
        slabs = flat.shape[1]
        words = flat[..., :1024 * nb].contiguous().view(torch.int32).view(e, slabs, nb, 4, 16, 4)
        q = torch.stack([(words >> (4 * (j // 2) + 16 * (j % 2))) & 15 for j in range(8)], dim=-1)
        q = q.permute(0, 1, 4, 2, 5, 3, 6).reshape(e, slabs, 16, nb * gpb, 128 // gpb)
        meta = flat[..., 1024 * nb:1024 * nb + 64 * gpb * nb].contiguous().view(torch.int32)
        meta = meta.view(e, slabs, nb, 16, gpb).transpose(2, 3).reshape(e, slabs, 16, nb * gpb, 1)
        w = (q - (meta & 15)).float() * (meta & -16).view(torch.float32)
        halves = 2 if self.gate_up else 1
        w = w.reshape(e, slabs // halves, halves, 16, -1).transpose(1, 2).reshape(e, halves, -1, nb * 128)
        w = w[:, :, :self.rows, :self.k].reshape(e, halves * self.rows, self.k).to(dtype)
        return w if self.num_experts is not None else w[0]

    def __repr__(self) -> str:
        lead = "" if self.num_experts is None else f"{self.num_experts}, "
        return f"PackedW4([{lead}{'2 x ' if self.gate_up else ''}{self.rows}, {self.k}], group {self.group})"


def _check_group(k: int, group: int) -> None:
    if group < 1 or k % group or not (group in (32, 64) or group % 128 == 0):
        raise ValueError(f"w4: groups of 32, 64 or a multiple of 128 that divide k = {k} expected, got {group}")


def _pack(what: str, qweight: Tensor, scales: Tensor, zeros: Tensor | None, gate_up: bool) -> PackedW4:
    if qweight.dtype != torch.uint8 or qweight.dim() not in (2, 3):
        raise ValueError(f"{what}: uint8 codes [N, K / 2] or [E, N, K / 2] expected, got {tuple(qweight.shape)} "
                         f"{qweight.dtype}")
    if scales.dtype not in SUPPORTED_DTYPES:
        raise TypeError(f"{what}: fp16 or bf16 scales expected, got {scales.dtype}")
    if scales.dim() != qweight.dim() or scales.shape[:-1] != qweight.shape[:-1] or 0 in qweight.shape + scales.shape:
        raise ValueError(f"{what}: codes {tuple(qweight.shape)} and scales {tuple(scales.shape)} do not match")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"{what}: uint8 zeros of the scales' shape expected, got {tuple(zeros.shape)} {zeros.dtype}")
    rows, k = qweight.shape[-2], 2 * qweight.shape[-1]
    if k % scales.shape[-1]:
        raise ValueError(f"{what}: {scales.shape[-1]} groups do not divide k = {k}")
    group = k // scales.shape[-1]
    _check_group(k, group)
    if gate_up:
        if rows % 2:
            raise ValueError(f"{what}: gate and up rows expected, got {rows} rows")
        rows //= 2
    experts = qweight.shape[0] if qweight.dim() == 3 else None
    for t in (scales, zeros):
        if t is not None and t.device != qweight.device:
            raise ValueError(f"{what}: all tensors must be on {qweight.device}, got one on {t.device}")
    if zeros is not None and bool((zeros > 15).any()):
        raise ValueError(f"{what}: zero points must be in 0..15")
    if not qweight.is_cuda:
        return PackedW4(None, (qweight, scales, zeros), experts, rows, k, group, gate_up, qweight.device)
    q, s = (t if t.stride(-1) == 1 else t.contiguous() for t in (qweight, scales))
    z = zeros if zeros is None or zeros.stride(-1) == 1 else zeros.contiguous()
    lib = _lib.load()
    n = lib.ember_w4_packed_bytes(rows, k, group, int(gate_up))
    if n < 0:
        raise ValueError(f"{what}: a weight of {rows} x {k} is too large")
    packed = torch.empty((experts or 1, n), dtype=torch.uint8, device=q.device)
    es = [t.stride(0) if t is not None and experts else 0 for t in (q, s, z)]
    _launch("ember_w4_pack_weight", lib.ember_w4_pack_weight, q.device, q.data_ptr(), es[0], q.stride(-2),
            s.data_ptr(), es[1], s.stride(-2), _lib.dtype_tag(s.dtype), None if z is None else z.data_ptr(), es[2],
            0 if z is None else z.stride(-2), experts or 1, rows, k, group, int(gate_up), packed.data_ptr())
    return PackedW4(packed, None, experts, rows, k, group, gate_up, q.device)


def pack_w4(qweight: Tensor, scales: Tensor, zeros: Tensor | None = None) -> PackedW4:
    """The packed form of a 4-bit weight [N, K], or [E, N, K] for `fused_moe`'s down projection."""
    return _pack("pack_w4", qweight, scales, zeros, False)


def pack_w4_gate_up(qweight: Tensor, scales: Tensor, zeros: Tensor | None = None) -> PackedW4:
    """The packed form of a 4-bit gate_up weight [2I, K] (rows [0, I) gate, [I, 2I) up), or [E, 2I, K]."""
    return _pack("pack_w4_gate_up", qweight, scales, zeros, True)


def linear_w4_torch(x: Tensor, weight: PackedW4, bias: Tensor | None = None) -> Tensor:
    """Eager form, in fp32."""
    y = F.linear(x.float(), weight.dequantize(torch.float32))
    return (y if bias is None else y + bias.float()).to(x.dtype)


def gate_up_silu_w4_torch(x: Tensor, weight: PackedW4) -> Tensor:
    """Eager form, in fp32."""
    g, u = F.linear(x.float(), weight.dequantize(torch.float32)).chunk(2, dim=-1)
    return (F.silu(g) * u).to(x.dtype)


def _check(what: str, x: Tensor, weight: PackedW4, gate_up: bool) -> None:
    if not isinstance(weight, PackedW4) or weight.gate_up != gate_up or weight.num_experts is not None:
        raise ValueError(f"{what}: a weight from {'pack_w4_gate_up' if gate_up else 'pack_w4'} expected, got {weight}")
    if x.dim() < 1 or x.shape[-1] != weight.k:
        raise ValueError(f"{what}: x {tuple(x.shape)} does not match {weight}")
    if x.dtype not in SUPPORTED_DTYPES:
        raise TypeError(f"{what}: fp16 or bf16 activations expected, got {x.dtype}")
    if x.device != weight.device:
        raise ValueError(f"{what}: x is on {x.device}, the weight on {weight.device}")


def _rows(x: Tensor) -> Tensor:
    """x as [T, K] rows that the kernels can read: unit inner stride, 16-byte aligned."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or x2.stride(0) % 8 or x2.stride(0) > MAX_ROW_STRIDE or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


# Sums and arrival counters of calls whose k is split over workgroups: one buffer per (thread, device,
# stream), and one per graph capture.
_SCRATCH = SharedScratch("linear_w4", per_capture=True)


def _workspace(need: int, counters: int, x: Tensor) -> tuple[int, Tensor]:
    """(0, a workspace of `need` bytes, `counters` of them at its end)."""
    return 0, _SCRATCH.get(need - counters, counters, x.device)


def linear_w4(x: Tensor, weight: PackedW4, bias: Tensor | None = None) -> Tensor:
    """round(x @ w.T + bias) [..., N] over a weight from `pack_w4`; bias [N] of x's dtype or None."""
    if type(weight) is PackedW4 and weight.projection is not None and not weight.gate_up and not _lib.tracing():
        got = _lib.fast.w4_linear(x, weight.packed, bias, weight.projection, _workspace)
        if got is not None:  # an ordinary call, answered by the native host path
            return got
    _check("linear_w4", x, weight, False)
    if bias is not None and (bias.shape != (weight.rows,) or bias.dtype != x.dtype or bias.device != x.device):
        raise ValueError(f"linear_w4: a bias of {weight.rows} elements of {x.dtype} on {x.device} expected, got "
                         f"{tuple(bias.shape)} {bias.dtype} on {bias.device}")
    if not fused_enabled(x):
        return linear_w4_torch(x, weight, bias)
    x2 = _rows(x)
    out = torch.empty((x2.shape[0], weight.rows), dtype=x.dtype, device=x.device)
    if x2.shape[0]:
        if bias is not None and bias.stride(0) != 1:
            bias = bias.contiguous()
        lib, counters, ws = _lib.load(), c_int64(0), None
        with torch.cuda.device(x.device):
            need = lib.ember_w4_linear_workspace_bytes(x2.shape[0], weight.k, weight.rows, weight.group, byref(counters))
        if need > 0:
            ws = _workspace(need, counters.value, x)[1]
        size = 0 if ws is None else ws.numel() * 4
        _launch("ember_w4_linear_split", lib.ember_w4_linear_split, x.device, x2.data_ptr(), x2.stride(0),
                weight.packed.data_ptr(), weight.group, _lib.dtype_tag(x.dtype), x2.shape[0], weight.k, weight.rows,
                None if bias is None else bias.data_ptr(), None if ws is None else ws.data_ptr(), size,
                out.data_ptr(), out.stride(0))
        if ws is not None and _check_indices():
            _SCRATCH.verify_counters(ws, size - counters.value, size)
    return out.view(*x.shape[:-1], weight.rows)


def gate_up_silu_w4(x: Tensor, weight: PackedW4) -> Tensor:
    """round(silu(gate) * up) [..., I] over a weight from `pack_w4_gate_up`: `gate_up_silu` with 4-bit
    weights."""
    if type(weight) is PackedW4 and weight.projection is not None and weight.gate_up and not _lib.tracing():
        got = _lib.fast.w4_linear(x, weight.packed, None, weight.projection, _workspace)
        if got is not None:
            return got
    _check("gate_up_silu_w4", x, weight, True)
    if not fused_enabled(x):
        return gate_up_silu_w4_torch(x, weight)
    x2 = _rows(x)
    out = torch.empty((x2.shape[0], weight.rows), dtype=x.dtype, device=x.device)
    if x2.shape[0]:
        _launch("ember_w4_gate_up_silu", _lib.load().ember_w4_gate_up_silu, x.device, x2.data_ptr(), x2.stride(0),
                weight.packed.data_ptr(), weight.group, _lib.dtype_tag(x.dtype), x2.shape[0], weight.k, weight.rows,
                out.data_ptr(), out.stride(0))
    return out.view(*x.shape[:-1], weight.rows)
