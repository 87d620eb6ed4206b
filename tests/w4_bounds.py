"""64-bit values and error bounds for the 4-bit projections and the routed experts' layer.

How far a kernel may be off, from its arithmetic (u = 2^-24, an fp32 rounding; h = eps / 2 of the
storage type, the rounding of a stored value):

* a 16-bit product sum over K terms: products of two fp16/bf16 values are exact in fp32; a term passes
  through at most 32 roundings inside an MFMA step, K / 32 of the accumulator and 32 of the joins of
  waves and splits: (K / 32 + 64) u sum |x w|;
* a 4-bit one: the group sums of x (16 + q) and of x, at most 31 sum |x| each, take G / 32 + 34 roundings
  of sizes up to 62 |s| sum |x|; the scaled groups are then joined by K / min(G, 128) + 32 roundings of
  sums no larger than sum |s x (q - z)| + the same: bounded by
  u ((G' / 32 + 34) 62 sum |s x| + (K / G' + 34) sum |x w|), G' = min(G, 128);
* silu(g) u: |d silu / d g| <= 1.1; exp, the quotient and the product are within 8 u of the value.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24


def half_ulp(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def tiny_step(t: torch.dtype) -> float:
    """Half the smallest subnormal: the rounding of values below the normal range."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def codes64(qweight, scales, zeros):
    """(weight, |scale| of every k) in 64 bits."""
    k = 2 * qweight.shape[-1]
    g = k // scales.shape[-1]
    q = torch.empty(*qweight.shape[:-1], k, dtype=torch.float64)
    q[..., 0::2] = (qweight & 15).double()
    q[..., 1::2] = (qweight >> 4).double()
    q -= 8.0 if zeros is None else zeros.double().repeat_interleave(g, -1)
    s = scales.double().repeat_interleave(g, -1)
    return q * s, s.abs()


def dot_bound(x, w, s=None, group=None):
    """(value, bound) of x @ w.T in 64 bits; s, group: the scales of a 4-bit weight."""
    y = x.double() @ w.T
    mag = x.double().abs() @ w.abs().T
    k = w.shape[-1]
    if s is None:
        return y, U * (k / 32 + 64) * mag
    g = min(group, 128)
    return y, U * ((g / 32 + 34) * 62 * (x.double().abs() @ s.T) + (k / g + 34) * mag)


def act_bound(y, dy):
    """silu(g) u of [g | u] = y and its bound."""
    inter = y.shape[-1] // 2
    g, u, dg, du = y[..., :inter], y[..., inter:], dy[..., :inter], dy[..., inter:]
    sig = torch.sigmoid(g)
    a = g * sig * u
    return a, 1.1 * dg * (u.abs() + du) + (g * sig).abs() * du + 8 * U * a.abs()


def check(got, want, bound, what=""):
    """|got - want| <= bound + the rounding of the stored value."""
    dt = got.dtype
    g = got.cpu().double()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    err = (g - want).abs()
    tol = bound + half_ulp(dt) * (want.abs() + bound) + tiny_step(dt)
    bad = ~(err <= tol)
    if bool(bad.any()):
        i = int(torch.where(bad, err / tol, torch.zeros_like(err)).nan_to_num(torch.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance, worst at "
                             f"{divmod(i, g.shape[-1])}: got {float(g.flatten()[i])!r} want "
                             f"{float(want.flatten()[i])!r} tol {float(tol.flatten()[i]):.3g}")
