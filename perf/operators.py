"""The weight-streaming operators of a decode step, as timed cases with a plain form beside each:
projections over 4-bit weights with group scales (`w4.linear_w4`), the dense MLP's gate_up
projection over such weights with silu_and_mul as its epilogue (`w4.gate_up_silu_w4`), and the
routed experts' whole layer (`moe.fused_moe`) over 16-bit and over 4-bit experts.

Shapes are those of the repository's benchmark and timed cases (Qwen2.5-0.5B / 7B, Qwen3-8B,
Moonlight) and the 128-expert layer that its dispatch was measured on. Every case is a decode
step: one token to a batch of 64.
"""

from __future__ import annotations

import math

import torch

own = False  # True: the framework's operators instead of the plain forms

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DENSE = {  # hidden, intermediate, q heads, kv heads, head dim, projection bias
    "qwen2.5-0.5b": (896, 4864, 14, 2, 64, True),
    "qwen2.5-7b": (3584, 18944, 28, 4, 128, True),
    "qwen3-8b": (4096, 12288, 32, 8, 128, False),
}
VOCAB = 151936
EXPERTS = {  # hidden, expert intermediate, experts, experts a token
    "moonlight": (2048, 1408, 64, 6),
    "experts-128": (2048, 768, 128, 8),
}
GROUPS = (32, 64, 128)
MAX_TOKENS = 64
MAX_MACS = 16 * VOCAB * 4096  # the largest listed product


def listed():
    return [
        # a lone request on a small model: the qkv projection with its bias, launch latency only
        dict(name="linear_qkv_1", kind="linear", model="qwen2.5-0.5b", proj="qkv", tokens=1, group=128, zeros=True,
             dtype="fp16"),
        # the longest rows of a 7B layer, two requests
        dict(name="linear_down_2", kind="linear", model="qwen2.5-7b", proj="down", tokens=2, group=128, zeros=False,
             dtype="bf16"),
        # an output projection with the finest groups at a usual batch
        dict(name="linear_o_16", kind="linear", model="qwen3-8b", proj="o", tokens=16, group=32, zeros=False,
             dtype="bf16"),
        # an odd, nearly full batch through the qkv projection, zero points given
        dict(name="linear_qkv_61", kind="linear", model="qwen3-8b", proj="qkv", tokens=61, group=64, zeros=True,
             dtype="fp16"),
        # the largest matrix of a decode step: the vocabulary head
        dict(name="linear_head_16", kind="linear", model="qwen3-8b", proj="head", tokens=16, group=128, zeros=False,
             dtype="bf16"),
        # the MLP's gate_up of a lone request, and of an odd batch with zero points
        dict(name="gate_up_1", kind="gate_up", model="qwen3-8b", tokens=1, group=128, zeros=False, dtype="bf16"),
        dict(name="gate_up_27", kind="gate_up", model="qwen2.5-7b", tokens=27, group=64, zeros=True, dtype="fp16"),
        # the routed experts of a lone request, of a small batch, and of one that reaches every expert
        dict(name="moe_1", kind="moe", experts="moonlight", tokens=1, group=0, zeros=False, dtype="bf16"),
        dict(name="moe_9", kind="moe", experts="moonlight", tokens=9, group=0, zeros=False, dtype="fp16"),
        dict(name="moe_48", kind="moe", experts="moonlight", tokens=48, group=0, zeros=False, dtype="bf16"),
        # the same over 4-bit experts: one token, and a batch on many small experts
        dict(name="moe_w4_1", kind="moe", experts="moonlight", tokens=1, group=128, zeros=False, dtype="bf16"),
        dict(name="moe_w4_33", kind="moe", experts="experts-128", tokens=33, group=64, zeros=True, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "gate_up", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    group, zeros = rng.choice(GROUPS), rng.random() < 0.5
    if kind == "moe":
        experts = rng.choice(sorted(EXPERTS))
        if rng.random() < 0.5:
            group, zeros = 0, False
        most = 48 if group == 0 else MAX_TOKENS
        return dict(kind=kind, experts=experts, tokens=_log(rng, 1, most), group=group, zeros=zeros, dtype=dtype)
    case = dict(kind=kind, model=rng.choice(sorted(DENSE)), group=group, zeros=zeros, dtype=dtype)
    if kind == "linear":
        case["proj"] = rng.choice(["qkv", "o", "down", "head"])
    n, k = _shape(case)
    return dict(case, tokens=_log(rng, 1, min(MAX_TOKENS, MAX_MACS // (n * k))))


def _shape(case):
    """(rows, k) of the case's weight."""
    hidden, inter, hq, hk, d, _ = DENSE[case["model"]]
    if case["kind"] == "gate_up":
        return 2 * inter, hidden
    return {"qkv": ((hq + 2 * hk) * d, hidden), "o": (hidden, hq * d), "down": (hidden, inter),
            "head": (VOCAB, hidden)}[case["proj"]]


# ---- inputs --------------------------------------------------------------------------------

class _Rand:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(self, shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=self.g)


def _quantized(r, lead, n, k, group, zeros, dtype):
    """A normal weight [*lead, n, k] rounded to 4 bits by groups: codes two to a byte (the even k in
    the low nibble), scales, and zero points or None."""
    w = r.normal((*lead, n, k // group, group), torch.bfloat16, 1.0 / math.sqrt(k)).float()
    if zeros:
        lo, hi = w.amin(-1).clamp(max=0.0), w.amax(-1).clamp(min=0.0)
        scales = ((hi - lo) / 15.0).to(dtype)
        zero = torch.round(-lo / scales.float()).clamp(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7.0).to(dtype)
        zero = torch.full_like(scales, 8.0, dtype=torch.float32)
    w = w.div_(scales.float()[..., None]).round_().add_(zero[..., None]).clamp_(0, 15).to(torch.uint8)
    w = w.view(*lead, n, k // 2, 2)
    codes = w[..., 0] | (w[..., 1] << 4)
    return codes, scales, zero.to(torch.uint8) if zeros else None


def _inputs(case, seed):
    r, dt = _Rand(seed), DTYPES[case["dtype"]]
    t = case["tokens"]
    if case["kind"] != "moe":
        n, k = _shape(case)
        s = dict(x=r.normal((t, k), dt), w=_quantized(r, (), n, k, case["group"], case["zeros"], dt), bias=None)
        if case["kind"] == "linear" and case["proj"] == "qkv" and DENSE[case["model"]][5]:
            s["bias"] = r.normal((n,), dt)
        return s
    hidden, inter, experts, topk = EXPERTS[case["experts"]]
    # a trained router favours some experts: a bias beside each token's own logits
    logits = r.normal((t, experts)) + r.normal((experts,), std=0.3)
    top = torch.topk(logits, topk, dim=-1)
    s = dict(x=r.normal((t, hidden), dt), ids=top.indices.contiguous(), weights=torch.softmax(top.values, -1))
    if case["group"]:
        s["w1"] = _quantized(r, (experts,), 2 * inter, hidden, case["group"], case["zeros"], dt)
        s["w2"] = _quantized(r, (experts,), hidden, inter, case["group"], case["zeros"], dt)
    else:
        s["w1"] = r.normal((experts, 2 * inter, hidden), dt, 1.0 / math.sqrt(hidden))
        s["w2"] = r.normal((experts, hidden, inter), dt, 1.0 / math.sqrt(inter))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # weights are packed once, when a model is loaded; the packed copy is the one it keeps
        from emberserve_amd import moe, w4
        if case["kind"] == "linear":
            s["w"] = w4.pack_w4(*s["w"])
        elif case["kind"] == "gate_up":
            s["w"] = w4.pack_w4_gate_up(*s["w"])
        elif case["group"]:
            s["w1"], s["w2"] = w4.pack_w4_gate_up(*s["w1"]), w4.pack_w4(*s["w2"])
        else:
            s["w1"], s["w2"] = moe.pack_moe_gate_up_weight(s["w1"]), moe.pack_moe_down_weight(s["w2"])
    return s


# ---- one pass ------------------------------------------------------------------------------

def _dequantized(codes, scales, zeros):
    """fp32 values of a 4-bit weight: (code - zero) * scale by groups."""
    q = torch.stack((codes & 15, codes >> 4), dim=-1).float()
    q = q.view(*scales.shape, -1)
    z = 8.0 if zeros is None else zeros.float()[..., None]
    return ((q - z) * scales.float()[..., None]).view(*codes.shape[:-1], -1)


def _silu_mul(gate_up):
    g, u = gate_up.chunk(2, dim=-1)
    return g / (1.0 + torch.exp(-g)) * u


def _expert(w, e):
    """fp32 weight of expert e."""
    if isinstance(w, tuple):
        codes, scales, zeros = w
        return _dequantized(codes[e], scales[e], None if zeros is None else zeros[e])
    return w[e].float()


def _plain_moe(s):
    x, ids, weights = s["x"].float(), s["ids"], s["weights"]
    t, topk = ids.shape
    experts = s["w1"][0].shape[0] if isinstance(s["w1"], tuple) else s["w1"].shape[0]
    y = torch.zeros_like(x)
    if t * topk <= experts:  # few assignments: gather each one's expert
        for i in range(t):
            for c in range(topk):
                e = ids[i, c:c + 1]
                act = _silu_mul(_expert(s["w1"], e)[0] @ x[i])
                y[i] += weights[i, c] * (_expert(s["w2"], e)[0] @ act)
        return y.to(s["x"].dtype)
    for e in range(experts):  # every expert over all tokens, weighted by the routing
        share = torch.where(ids == e, weights, torch.zeros_like(weights)).sum(-1, keepdim=True)
        act = _silu_mul(x @ _expert(s["w1"], e).t())
        y += share * (act @ _expert(s["w2"], e).t())
    return y.to(s["x"].dtype)


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        from emberserve_amd import moe, w4
        if kind == "linear":
            return w4.linear_w4(s["x"], s["w"], s["bias"])
        if kind == "gate_up":
            return w4.gate_up_silu_w4(s["x"], s["w"])
        return moe.fused_moe(s["x"], s["ids"], s["weights"], None, None, packed=s["w1"], packed_down=s["w2"])
    if kind == "moe":
        return _plain_moe(s)
    y = s["x"].float() @ _dequantized(*s["w"]).t()
    if kind == "gate_up":
        y = _silu_mul(y)
    elif s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------

def _weight_bytes(n, k, group, zeros):
    if not group:
        return 2 * n * k
    return n * k / 2 + n * (k // group) * (3 if zeros else 2)


def work(case):
    e, t, group, zeros = 2, case["tokens"], case["group"], case["zeros"]
    if case["kind"] == "moe":
        hidden, inter, experts, topk = EXPERTS[case["experts"]]
        used = experts * (1 - (1 - topk / experts) ** t)  # expected
        one = _weight_bytes(2 * inter, hidden, group, zeros) + _weight_bytes(hidden, inter, group, zeros)
        return {"bytes": used * one + 2 * t * hidden * e + t * topk * 12, "flops": 6 * t * topk * hidden * inter}
    n, k = _shape(case)
    out = n // 2 if case["kind"] == "gate_up" else n
    return {"bytes": _weight_bytes(n, k, group, zeros) + t * (k + out) * e, "flops": 2 * t * n * k}


# ---- the same in 64 bits -------------------------------------------------------------------

def _rows64(w, lo, hi, e=None):
    """Rows [lo, hi) of a weight (of its expert e) in 64 bits."""
    if not isinstance(w, tuple):
        return w[e, lo:hi].double()
    codes, scales, zeros = (v if v is None or e is None else v[e] for v in w)
    codes, scales = codes[lo:hi].to(torch.int64), scales[lo:hi].double()
    group = 2 * codes.shape[1] // scales.shape[1]
    vals = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    vals[:, 0::2] = (codes % 16).double()
    vals[:, 1::2] = (codes // 16).double()
    vals -= 8.0 if zeros is None else zeros[lo:hi].double().repeat_interleave(group, dim=1)
    return vals * scales.repeat_interleave(group, dim=1)


def _product64(x, w, n, e=None, step=16384):
    parts = [x @ _rows64(w, lo, min(n, lo + step), e).t().contiguous() for lo in range(0, n, step)]
    return torch.cat(parts, dim=-1)


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"].double()
    if case["kind"] == "moe":
        hidden, inter, experts, _ = EXPERTS[case["experts"]]
        y = torch.zeros_like(x)
        for e in range(experts):
            rows, choice = (s["ids"] == e).nonzero(as_tuple=True)
            if rows.numel():
                gu = _product64(x[rows], s["w1"], 2 * inter, e)
                act = gu[:, :inter] * torch.sigmoid(gu[:, :inter]) * gu[:, inter:]
                y.index_add_(0, rows, s["weights"].double()[rows, choice][:, None] * _product64(act, s["w2"], hidden, e))
        return y
    n, _ = _shape(case)
    y = _product64(x, s["w"], n)
    if case["kind"] == "gate_up":
        return y[:, :n // 2] * torch.sigmoid(y[:, :n // 2]) * y[:, n // 2:]
    return y if s["bias"] is None else y + s["bias"].double()
