"""The 4-bit projections and the experts' layer without a GPU: quantising, the eager forms against 64
bits, refusals, and the C ABI's argument checks (which answer before any device call)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from emberserve_amd import _lib, moe, w4
from tests.w4_bounds import U, act_bound, check, codes64, dot_bound, half_ulp, tiny_step

BF, HF = torch.bfloat16, torch.float16


def _w(n, k, dtype=BF, experts=None, seed=0):
    lead = () if experts is None else (experts,)
    return (torch.randn(*lead, n, k, generator=torch.Generator().manual_seed(seed)) / k ** 0.5).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_quantize_rounds_to_nearest(dtype, symmetric, group):
    """Each weight is within half a step of its group's scale, and the rounding of scale and of the zero
    point (asymmetric: half a step more at the ends of the range)."""
    w = _w(24, 512, dtype)
    w[3, :group] = 0
    q, s, z = w4.quantize_w4(w, group, symmetric=symmetric)
    assert q.shape == (24, 256) and s.shape == (24, 512 // group) and s.dtype == dtype
    assert (z is None) == symmetric
    d = w4.dequantize_w4(q, s, z, dtype=torch.float32)
    step = s.double().repeat_interleave(group, -1)
    h = half_ulp(dtype)
    slack = (7 if symmetric else 15) * step * h * 1.01 + (0 if symmetric else 0.5) * step
    assert bool(((d.double() - w.double()).abs() <= 0.5 * step * (1 + 1e-6) + slack).all())
    assert bool((d[3, :group] == 0).all())


def test_quantize_refuses_what_is_not_finite():
    for bad in (float("inf"), float("-inf"), float("nan")):
        w = _w(4, 64)
        w[2, 5] = bad
        with pytest.raises(ValueError):
            w4.quantize_w4(w, 32)


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_small_fp16_weights(symmetric):
    """Scales below fp16's normal range are multiples of 2^-24: half of one more a code for the scale's
    rounding, which may also put the ends of the range out of the codes' reach, by as much."""
    w = (_w(16, 256, torch.float32, seed=70) * 2.0 ** -10).to(HF)
    q, s, z = w4.quantize_w4(w, 64, symmetric=symmetric)
    assert float(s.max()) < torch.finfo(HF).tiny
    d = w4.dequantize_w4(q, s, z, dtype=torch.float32)
    step = s.double().repeat_interleave(64, -1)
    slack = (7 if symmetric else 15) * 2.0 ** -25 + (0 if symmetric else 0.5) * step
    assert bool(((d.double() - w.double()).abs() <= 0.5 * step * (1 + 1e-6) + slack).all())


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_eager_forms_match_64_bits(group, zeros):
    parts = w4.quantize_w4(_w(60, 384, BF), group, symmetric=not zeros)
    x = torch.randn(3, 5, 384, generator=torch.Generator().manual_seed(1)).to(BF)
    bias = torch.randn(60, generator=torch.Generator().manual_seed(2)).to(BF)
    w, _ = codes64(*parts)
    y = x.reshape(15, 384).double() @ w.T
    # fp32 sums of 384 terms in any order
    dy = 400 * U * (x.reshape(15, 384).double().abs() @ w.abs().T)
    got = w4.linear_w4(x, w4.pack_w4(*parts), bias)
    assert got.shape == (3, 5, 60)
    check(got.view(15, 60), y + bias.double(), dy + 2 * U * (y.abs() + bias.double().abs()))
    got = w4.gate_up_silu_w4(x, w4.pack_w4_gate_up(*parts))
    check(got.view(15, 30), *act_bound(y, dy))


def test_fused_moe_eager():
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(3)).to(HF)
    w1, w2 = _w(128, 64, HF, 3, seed=4), _w(64, 64, HF, 3, seed=5)
    ids = torch.tensor([[0, 2], [1, 1], [-1, 2], [-1, -1]])
    weights = torch.rand(4, 2, generator=torch.Generator().manual_seed(6))
    got = moe.fused_moe(x, ids, weights, w1, w2)
    want, bound = torch.zeros(4, 64, dtype=torch.float64), torch.zeros(4, 64, dtype=torch.float64)
    for t in range(4):
        for c in range(2):
            if ids[t, c] >= 0:
                e, wt = int(ids[t, c]), float(weights[t, c])
                a, da = act_bound(*dot_bound(x[t:t + 1], w1[e].double()))
                v, dv = dot_bound(a, w2[e].double())
                want[t] += wt * v[0]
                bound[t] += wt * (dv + da @ w2[e].double().abs().T)[0] + 4 * U * wt * v[0].abs()
    check(got, want, bound)
    assert bool((got[3] == 0).all())
    q1, q2 = w4.quantize_w4(w1, 32), w4.quantize_w4(w2, 64, symmetric=False)
    p1, p2 = w4.pack_w4_gate_up(*q1), w4.pack_w4(*q2)
    got = moe.fused_moe(x, ids, weights, None, None, packed=p1, packed_down=p2)
    d1, d2 = (w4.dequantize_w4(*q, dtype=torch.float32) for q in (q1, q2))
    assert torch.equal(got, moe.fused_moe_torch(x, ids, weights, d1, d2))


def test_quantize_and_pack_refusals():
    q, s, z = w4.quantize_w4(_w(8, 256), 64, symmetric=False)
    for group in (0, 16, 96, 512, -64):
        with pytest.raises(ValueError):
            w4.quantize_w4(_w(8, 256), group)
    with pytest.raises(ValueError):
        w4.quantize_w4(_w(8, 256).float(), 64)
    with pytest.raises(ValueError):
        w4.pack_w4(q.int(), s, z)
    with pytest.raises(TypeError):
        w4.pack_w4(q, s.float(), z)
    with pytest.raises(ValueError):
        w4.pack_w4(q, s[:7], z)
    with pytest.raises(ValueError):
        w4.pack_w4(q, s, z[:, :3])
    with pytest.raises(ValueError):
        w4.pack_w4(q, s, z + 8)
    with pytest.raises(ValueError):
        w4.pack_w4(q, s.repeat(1, 4))  # groups of 16
    with pytest.raises(ValueError):
        w4.pack_w4(q[0], s[0], z[0])
    with pytest.raises(ValueError):
        w4.pack_w4(q[:0], s[:0], z[:0])
    with pytest.raises(ValueError):
        w4.pack_w4_gate_up(q[:7], s[:7], z[:7])


def test_linear_refusals():
    parts = w4.quantize_w4(_w(16, 128), 64)
    p, gu = w4.pack_w4(*parts), w4.pack_w4_gate_up(*parts)
    experts = w4.pack_w4(*w4.quantize_w4(_w(16, 128, BF, 2), 64))
    x = torch.zeros(2, 128, dtype=BF)
    for bad in (gu, experts, parts[0]):
        with pytest.raises(ValueError):
            w4.linear_w4(x, bad)
    for bad in (p, experts):
        with pytest.raises(ValueError):
            w4.gate_up_silu_w4(x, bad)
    with pytest.raises(ValueError):
        w4.linear_w4(x[:, :64], p)
    with pytest.raises(TypeError):
        w4.linear_w4(x.float(), p)
    with pytest.raises(ValueError):
        w4.linear_w4(x, p, torch.zeros(15, dtype=BF))
    with pytest.raises(ValueError):
        w4.linear_w4(x, p, torch.zeros(16))
    with pytest.raises(ValueError):
        w4.linear_w4(x.to("meta"), p)
    assert w4.linear_w4(x[:0], p).shape == (0, 16)


def test_fused_moe_refusals():
    x, w1, w2 = torch.zeros(4, 64, dtype=BF), _w(128, 64, BF, 3), _w(64, 64, BF, 3)
    ids, wt = torch.zeros(4, 2, dtype=torch.int64), torch.ones(4, 2)
    p1, p2 = w4.pack_w4_gate_up(*w4.quantize_w4(w1, 32)), w4.pack_w4(*w4.quantize_w4(w2, 32))
    ok = dict(x=x, topk_ids=ids, topk_weights=wt, w_gate_up=w1, w_down=w2)
    assert moe.fused_moe(**ok).shape == (4, 64)

    def refused(error, **change):
        with pytest.raises(error):
            moe.fused_moe(**{**ok, **change})

    refused(ValueError, x=x[0])
    refused(ValueError, x=x[:3])
    refused(ValueError, x=x[:, :32])
    refused(ValueError, topk_ids=ids[:, 0])
    refused(ValueError, topk_ids=ids[:, :1])
    refused(ValueError, topk_ids=ids[:, :0], topk_weights=wt[:, :0])
    refused(TypeError, topk_ids=ids.short())
    refused(TypeError, topk_weights=wt.double())
    refused(TypeError, x=x.half())
    refused(TypeError, x=x.float())
    refused(ValueError, w_down=None)
    refused(ValueError, w_gate_up=None)
    refused(ValueError, w_gate_up=w1[:, :127])
    refused(ValueError, w_down=w2[:2])
    refused(ValueError, w_down=w2[:, :, :32])
    refused(ValueError, packed=p1)               # 4-bit gate_up with a 16-bit down
    refused(ValueError, packed=p2, packed_down=p2)
    refused(ValueError, packed=p1, packed_down=p1)
    refused(TypeError, packed=w1)
    refused(ValueError, topk_ids=ids.to("meta"))
    n = moe.LAYER_MAX_TOKENS + 1
    refused(ValueError, x=x[:1].expand(n, 64), topk_ids=ids[:1].expand(n, 2), topk_weights=wt[:1].expand(n, 2))
    refused(ValueError, topk_ids=ids[:, :1].expand(4, 129), topk_weights=wt[:, :1].expand(4, 129))
    with pytest.raises(ValueError):
        moe.pack_moe_down_weight(w2)  # on the CPU


def test_abi_argument_checks():
    lib = _lib.load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)  # never dereferenced: the calls are refused first
    size = lib.ember_w4_packed_bytes
    assert size(16, 128, 128, 0) == 1024 + 128 and size(17, 129 + 31, 32, 0) == 2 * (2 * 1024 + 512)
    assert size(16, 640, 64, 1) == 2 * (5 * 1024 + 640)
    for bad in ((0, 128, 128, 0), (16, 0, 128, 0), (16, 128, 96, 0), (16, 100, 32, 0), (16, 128, 256, 0),
                (16, 128, 0, 0), (16, 128, -64, 0), (1 << 28, 128, 128, 0), (16, 1 << 25, 128, 0)):
        assert size(*bad) == -1
    lin = lib.ember_w4_linear
    assert lin(p, 128, p, 128, 2, 0, 128, 16, None, p, 16, None) == 0  # no tokens: nothing to do
    assert lin(None, 128, p, 128, 2, 1, 128, 16, None, p, 16, None) == 1
    assert lin(p, 128, p, 128, 0, 1, 128, 16, None, p, 16, None) == 1   # fp32
    assert lin(p, 128, p, 48, 2, 1, 128, 16, None, p, 16, None) == 1
    assert lin(p, 128, p, 128, 2, -1, 128, 16, None, p, 16, None) == 1
    assert lin(p, 128, p, 128, 2, 1 << 22, 128, 16, None, p, 16, None) == 1
    assert lin(odd, 128, p, 128, 2, 1, 128, 16, None, p, 16, None) == 2
    assert lin(p, 132, p, 128, 2, 1, 128, 16, None, p, 16, None) == 2
    assert lib.ember_w4_gate_up_silu(p, 128, p, 96, 2, 1, 128, 16, p, 16, None) == 1
    pack = lib.ember_w4_pack_weight
    assert pack(p, 0, 64, p, 0, 1, 2, None, 0, 0, 0, 16, 128, 128, 0, p, None) == 1   # no experts
    assert pack(p, 0, 64, p, 0, 1, 0, None, 0, 0, 1, 16, 128, 128, 0, p, None) == 1   # fp32 scales
    assert pack(p, 0, 64, None, 0, 1, 2, None, 0, 0, 1, 16, 128, 128, 0, p, None) == 1
    assert pack(p, 0, 64, p, 0, 1, 2, None, 0, 0, 1, 16, 128, 128, 0, odd, None) == 2
    cnt = ctypes.c_int64(0)
    need = lib.ember_moe_layer_workspace_bytes(4, 2, 8, 128, 64, ctypes.byref(cnt))
    assert need > cnt.value > 0 and cnt.value >= 128 // 16 * 4
    for bad in ((65, 2, 8, 128, 64), (4, 0, 8, 128, 64), (64, 9, 8, 128, 64), (4, 2, 0, 128, 64), (4, 2, 1025, 128, 64),
                (4, 2, 8, 100, 64), (4, 2, 8, 128, 20), (-1, 2, 8, 128, 64)):
        assert lib.ember_moe_layer_workspace_bytes(*bad, None) == -1

    def layer(x=p, xs=128, ids=p, id_bytes=8, wt=p, wt_dtype=0, n=4, k=2, w1=p, s1=(0, 0), w2=p, s2=(0, 0), dtype=2,
              e=8, h=128, i=64, ws=p, ws_bytes=1 << 24, out=p):
        return lib.ember_moe_layer(x, xs, ids, id_bytes, wt, wt_dtype, n, k, w1, *s1, w2, *s2, dtype, e, h, i, ws,
                                   ws_bytes, out, 128, None)

    assert layer(n=0) == 0
    for bad in (dict(id_bytes=2), dict(wt_dtype=9), dict(dtype=0), dict(h=96), dict(i=32), dict(n=65), dict(k=0),
                dict(e=2000), dict(ws_bytes=256), dict(ws=None), dict(x=None), dict(w1=None), dict(w2=None),
                dict(ids=None), dict(wt=None), dict(out=None)):
        assert layer(**bad) == 1, bad
    for bad in (dict(x=odd), dict(xs=132), dict(w1=odd), dict(w2=odd), dict(s1=(128 * 128, 132)), dict(s2=(8, 60)),
                dict(ws=odd)):
        assert layer(**bad) == 2, bad
    w4_layer = lib.ember_moe_layer_w4
    assert w4_layer(p, 128, p, 8, p, 0, 0, 2, p, 128, p, 64, 2, 8, 128, 64, p, 1 << 24, p, 128, None) == 0
    assert w4_layer(p, 128, p, 8, p, 0, 4, 2, p, 128, p, 128, 2, 8, 128, 64, p, 1 << 24, p, 128, None) == 1
    down = lib.ember_moe_down_pack_weight
    assert down(p, 0, 64, 0, 1, 16, 64, p, None) == 1 and down(p, 0, 60, 2, 1, 16, 64, p, None) == 2
    assert down(p, 0, 64, 2, 0, 16, 64, p, None) == 1 and down(p, 0, 64, 2, 1, 20, 64, p, None) == 1


def test_abi_checks_of_the_split_form():
    lib = _lib.load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    cnt = ctypes.c_int64(7)
    size = lib.ember_w4_linear_workspace_bytes
    assert size(1, 4096, 4096, 128, ctypes.byref(cnt)) == 0 and cnt.value == 0  # one token: no splits
    assert size(1 << 20, 4096, 4096, 128, None) == 0
    for bad in ((-1, 128, 16, 128), (1, 128, 0, 128), (1, 100, 16, 32), (1, 128, 16, 96), (1 << 22, 128, 16, 128)):
        assert size(*bad, None) == -1
    lin = lib.ember_w4_linear_split
    assert lin(p, 128, p, 128, 2, 0, 128, 16, None, None, 0, p, 16, None) == 0
    assert lin(p, 128, p, 128, 2, 1, 128, 16, None, odd, 256, p, 16, None) == 2
    assert lin(p, 128, p, 128, 2, 1, 128, 16, None, p, 250, p, 16, None) == 2
    assert lin(None, 128, p, 128, 2, 1, 128, 16, None, p, 256, p, 16, None) == 1
    assert lin(p, (1 << 23) + 8, p, 128, 2, 1, 128, 16, None, p, 256, p, 16, None) == 1


def test_bounds_have_teeth():
    """The oracle's bound refuses a wrong zero point, scale or expert."""
    q, s, z = w4.quantize_w4(_w(16, 256), 64, symmetric=False)
    x = torch.randn(2, 256, generator=torch.Generator().manual_seed(7)).to(BF)
    w, sa = codes64(q, s, z)
    want, bound = dot_bound(x, w, sa, 64)
    check(want.to(BF), want, bound)
    for parts in ((q, s, (z + 1) % 16), (q, s * 1.02, z), (q ^ 1, s, z)):
        with pytest.raises(AssertionError):
            check((x.double() @ codes64(*parts)[0].T).to(BF), want, bound)
    assert tiny_step(BF) > 0


def test_native_host_path_declines_other_calls():
    """CPU tensors, wrong argument counts and anything but the weight's own tuple are the wrappers'."""
    _lib.load()
    x, b = torch.zeros(2, 128, dtype=BF), torch.zeros(16, 80, dtype=torch.uint8)
    ids, wt = torch.zeros(2, 1, dtype=torch.int64), torch.ones(2, 1)
    fast = _lib.fast
    assert fast.w4_linear(x, b, None, (16, 128, 128, 0)) is None and fast.w4_linear(x) is None
    assert fast.w4_linear(x, b, None, (16, 128)) is None and fast.w4_linear(x, b, "b", None) is None
    assert fast.fused_moe(x, ids, wt, b, b, (1, 128, 64, 128, 64), None) is None and fast.fused_moe() is None


def test_fused_moe_is_registered():
    from emberserve_amd import torch_ops
    x, w1, w2 = torch.randn(4, 64).to(BF), _w(128, 64, BF, 3), _w(64, 64, BF, 3)
    ids, wt = torch.tensor([[0, 2], [1, 1], [2, 0], [-1, 1]]), torch.rand(4, 2)
    torch.library.opcheck(torch.ops.emberserve.fused_moe, (x, ids, wt, w1, w2))
    assert torch.equal(torch_ops.fused_moe(x, ids, wt, w1, w2), moe.fused_moe(x, ids, wt, w1, w2))
