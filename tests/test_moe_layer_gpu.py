"""The routed experts' whole layer (`moe.fused_moe`) on the GPU against 64-bit values, with the bounds of
tests.w4_bounds carried through both products."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from emberserve_amd import _lib, moe, w4  # noqa: E402
from tests.test_w4_gpu import _dev, _weight  # noqa: E402
from tests.w4_bounds import U, act_bound, check, codes64, dot_bound, half_ulp, tiny_step  # noqa: E402

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clear_errors():
    _lib.read_errors(clear=True)
    yield
    assert _lib.read_errors() == 0


def _routing(n, k, experts, seed, ids_dtype=torch.int64, w_dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(n)]) if n else torch.empty(0, k)
    weights = torch.softmax(torch.randn(n, k, generator=g), -1)
    return ids.to(ids_dtype), weights.to(w_dtype)


def _half(experts, h, i, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    w1 = (torch.randn(experts, 2 * i, h, generator=g) / h ** 0.5).to(dtype)
    w2 = (torch.randn(experts, h, i, generator=g) / i ** 0.5).to(dtype)
    return w1, w2


def _want(x, ids, weights, w1, w2, s1=None, s2=None, g1=None, g2=None):
    """(value, bound) of the layer; w1, w2 per expert in 64 bits, s1, s2 their |scales| for 4 bits."""
    y = torch.zeros(x.shape, dtype=torch.float64)
    bound = torch.zeros_like(y)
    mag = torch.zeros_like(y)
    for t in range(ids.shape[0]):
        for c in range(ids.shape[1]):
            e, wt = int(ids[t, c]), weights[t, c].double()
            if not 0 <= e < w1.shape[0]:
                continue
            a, da = act_bound(*dot_bound(x[t:t + 1], w1[e], None if s1 is None else s1[e], g1))
            da = da + half_ulp(x.dtype) * (a.abs() + da) + tiny_step(x.dtype)
            v, dv = dot_bound(a, w2[e], None if s2 is None else s2[e], g2)
            y[t] += wt * v[0]
            bound[t] += wt.abs() * (dv + da @ w2[e].abs().T)[0]
            mag[t] += wt.abs() * v[0].abs()
    # the weighted sums of waves, splits and choices: up to 128 waves and splits join a token's sums
    return y, bound + U * (ids.shape[1] + 140) * (mag + bound)


def _w4_experts(experts, h, i, group, zeros, dtype, seed):
    return (_weight(2 * i, h, group, zeros, dtype, seed, experts), _weight(h, i, group, zeros, dtype, seed + 1, experts))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k,experts,h,i", [
    (1, 6, 64, 256, 128), (1, 1, 1, 64, 64), (2, 2, 8, 128, 192), (9, 6, 64, 192, 64), (17, 8, 128, 128, 64),
    (64, 2, 8, 128, 128), (64, 8, 9, 64, 64), (33, 1, 3, 320, 64), (5, 100, 1024, 64, 64), (20, 4, 4, 64, 448)])
def test_half_matches_64_bits(dtype, n, k, experts, h, i):
    """Unpacked, packed and mixed weights; groups of more than 16 assignments; every expert used; A = 512."""
    print(f"fused_moe n={n} k={k} E={experts} H={h} I={i} {dtype}", flush=True)
    x = torch.randn(n, h, generator=torch.Generator().manual_seed(n)).to(dtype)
    w1, w2 = _half(experts, h, i, dtype, seed=experts)
    ids, weights = _routing(n, k, experts, seed=h)
    want, bound = _want(x, ids, weights, w1.double(), w2.double())
    dx, dids, dwt, d1, d2 = (v.to(DEV) for v in (x, ids, weights, w1, w2))
    got = moe.fused_moe(dx, dids, dwt, d1, d2)
    check(got, want, bound, "unpacked")
    p1, p2 = moe.pack_moe_gate_up_weight(d1), moe.pack_moe_down_weight(d2)
    packed = moe.fused_moe(dx, dids.int(), dwt, None, None, packed=p1, packed_down=p2)
    check(packed, want, bound, "packed")
    assert torch.equal(packed, got)  # the same products in the same order
    assert torch.equal(moe.fused_moe(dx, dids, dwt, d1, None, packed_down=p2), got)
    assert torch.equal(moe.fused_moe(dx, dids, dwt, None, d2, packed=p1), got)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,k,experts,h,i,group,zeros", [
    (1, 6, 64, 256, 128, 128, False), (1, 2, 4, 96, 32, 32, True), (9, 4, 16, 416, 160, 32, True),
    (33, 8, 128, 128, 192, 64, True), (64, 2, 8, 256, 256, 256, False), (3, 1, 2, 64, 320, 64, False)])
def test_w4_matches_64_bits(dtype, n, k, experts, h, i, group, zeros):
    print(f"fused_moe w4 n={n} k={k} E={experts} H={h} I={i} g{group} {dtype}", flush=True)
    x = torch.randn(n, h, generator=torch.Generator().manual_seed(n)).to(dtype)
    q1, q2 = _w4_experts(experts, h, i, group, zeros, dtype, seed=experts)
    ids, weights = _routing(n, k, experts, seed=h)
    (w1, s1), (w2, s2) = codes64(*q1), codes64(*q2)
    want, bound = _want(x, ids, weights, w1, w2, s1, s2, group, group)
    got = moe.fused_moe(x.to(DEV), ids.to(DEV), weights.to(DEV), None, None, packed=w4.pack_w4_gate_up(*_dev(q1)),
                        packed_down=w4.pack_w4(*_dev(q2)))
    check(got, want, bound)


def test_moonlight_geometry():
    """H 2048, I 1408, 64 experts, top-6: splits of the second product, ragged groups."""
    x = torch.randn(24, 2048, generator=torch.Generator().manual_seed(1)).to(BF)
    w1, w2 = _half(64, 2048, 1408, BF, seed=2)
    for n in (1, 24):
        ids, weights = _routing(n, 6, 64, seed=n)
        want, bound = _want(x[:n], ids, weights, w1.double(), w2.double())
        got = moe.fused_moe(x[:n].to(DEV), ids.to(DEV), weights.to(DEV), w1.to(DEV), w2.to(DEV))
        check(got, want, bound, f"n={n}")


def test_absent_and_bad_ids():
    """-1 adds nothing, silently; other ids outside the experts neither, and set the error bit; a token with
    none gets zeros, and so does a step with none at all."""
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(3)).to(BF)
    w1, w2 = _half(8, 128, 64, BF, seed=4)
    ids, weights = _routing(5, 3, 8, seed=5)
    ids[0, 1] = -1
    ids[2] = -1
    want, bound = _want(x, ids, weights, w1.double(), w2.double())
    args = [v.to(DEV) for v in (x, ids, weights, w1, w2)]
    got = moe.fused_moe(*args)
    check(got, want, bound)
    assert bool((got[2] == 0).all())
    assert _lib.read_errors() == 0
    args[1][0, 1], args[1][2, 0], args[1][2, 1] = 8, -2, 2 ** 40
    assert torch.equal(moe.fused_moe(*args), got)
    assert _lib.read_errors(clear=True) == _lib.ERR_EXPERT_ID
    args[1].fill_(-1)
    assert bool((moe.fused_moe(*args) == 0).all())


def test_one_expert_twice():
    """A token that names an expert twice gets both weights; the same bits on every call."""
    x = torch.randn(40, 128, generator=torch.Generator().manual_seed(6)).to(HF)
    w1, w2 = _half(4, 128, 64, HF, seed=7)
    ids = torch.randint(0, 4, (40, 5), generator=torch.Generator().manual_seed(8))
    weights = torch.randn(40, 5, generator=torch.Generator().manual_seed(9))
    want, bound = _want(x, ids, weights, w1.double(), w2.double())
    args = [v.to(DEV) for v in (x, ids, weights, w1, w2)]
    got = moe.fused_moe(*args)
    check(got, want, bound)
    for _ in range(5):
        assert torch.equal(moe.fused_moe(*args), got)


@pytest.mark.parametrize("w_dtype", [torch.float32, BF, HF])
def test_weight_dtypes_and_strides(w_dtype):
    """Routing weights of each type; x, ids and weights as views; weights of experts far apart."""
    x = torch.randn(7, 128, generator=torch.Generator().manual_seed(10)).to(BF)
    w1, w2 = _half(6, 128, 64, BF, seed=11)
    ids, weights = _routing(7, 2, 6, seed=12, w_dtype=w_dtype)
    want, bound = _want(x, ids, weights, w1.double(), w2.double())
    wide = torch.full((7, 300), float("nan"), dtype=BF, device=DEV)
    wide[:, 1:129] = x.to(DEV)
    b1 = torch.full((6, 2, 128, 136), float("nan"), dtype=BF, device=DEV)
    b1[:, 1, :, :128] = w1.to(DEV)
    tall = torch.zeros((2, 7), dtype=torch.int64, device=DEV)
    tall.copy_(ids.T)
    got = moe.fused_moe(wide[:, 1:129], tall.T, weights.to(DEV), b1[:, 1, :, :128], w2.to(DEV))
    check(got, want, bound)


def test_nonfinite_rows_stay_their_own():
    x = torch.randn(6, 128, generator=torch.Generator().manual_seed(13)).to(BF).to(DEV)
    w1, w2 = (v.to(DEV) for v in _half(3, 128, 64, BF, seed=14))
    ids, weights = (v.to(DEV) for v in _routing(6, 2, 3, seed=15))
    want = moe.fused_moe(x, ids, weights, w1, w2)
    bad = x.clone()
    bad[4, 127] = float("nan")
    got = moe.fused_moe(bad, ids, weights, w1, w2)
    assert bool(got[4].isnan().all())
    assert torch.equal(got[[0, 1, 2, 3, 5]], want[[0, 1, 2, 3, 5]])


def test_shapes_take_turns_on_one_workspace():
    """Calls of different sizes on one stream, each on what the others left: the same bits as the first."""
    calls = []
    for n, k, experts, h, i in ((1, 6, 64, 512, 128), (64, 8, 16, 256, 64), (3, 2, 4, 2048, 64)):
        x = torch.randn(n, h, generator=torch.Generator().manual_seed(n)).to(BF).to(DEV)
        w1, w2 = (v.to(DEV) for v in _half(experts, h, i, BF, seed=n))
        ids, weights = (v.to(DEV) for v in _routing(n, k, experts, seed=n))
        calls.append((x, ids, weights, w1, w2))
    first = [moe.fused_moe(*c) for c in calls]
    for i in (2, 0, 1, 1, 0, 2):
        assert torch.equal(moe.fused_moe(*calls[i]), first[i])
    assert moe.fused_moe(calls[0][0][:0], calls[0][1][:0], calls[0][2][:0], *calls[0][3:]).shape == (0, 512)


def test_graph_replays_match_eager():
    """A captured step replayed with other routings, with eager calls and another graph in between."""
    w1, w2 = (v.to(DEV) for v in _half(16, 512, 128, BF, seed=16))
    x = torch.randn(4, 512, generator=torch.Generator().manual_seed(17)).to(BF).to(DEV)
    ids, weights = (v.to(DEV) for v in _routing(4, 3, 16, seed=18))
    moe.fused_moe(x, ids, weights, w1, w2)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(moe.fused_moe(x, ids, weights, w1, w2))
    for i in range(4):
        new_ids, new_weights = _routing(4, 3, 16, seed=30 + i)
        ids.copy_(new_ids)
        weights.copy_(new_weights)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], moe.fused_moe(x, ids, weights, w1, w2)), i


def test_two_graphs_of_one_stream_replay_at_once():
    """Two graphs captured on a stream that eager calls used have workspaces of their own."""
    w1, w2 = (v.to(DEV) for v in _half(16, 1024, 256, BF, seed=31))
    ids, weights = (v.to(DEV) for v in _routing(8, 4, 16, seed=32))
    xs = [torch.randn(8, 1024, generator=torch.Generator().manual_seed(33 + i)).to(BF).to(DEV) for i in range(3)]
    want = [moe.fused_moe(x, ids, weights, w1, w2) for x in xs]
    torch.cuda.synchronize()
    one, graphs, outs = torch.cuda.Stream(), [], []
    with torch.cuda.stream(one):
        moe.fused_moe(xs[2], ids, weights, w1, w2)
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=one):
            outs.append([moe.fused_moe(x, ids, weights, w1, w2) for _ in range(4)])
        graphs.append(g)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(one):
            eager = moe.fused_moe(xs[2], ids, weights, w1, w2)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i]) and torch.equal(eager, want[2])


@pytest.mark.parametrize("n,k,experts,h,i", [(33, 4, 8, 4096, 64), (20, 2, 4, 7168, 64), (2, 2, 2, 16384, 32)])
def test_w4_long_rows(n, k, experts, h, i):
    """Groups whose tokens take up to 128 KiB of LDS, eager and captured."""
    x = torch.randn(n, h, generator=torch.Generator().manual_seed(n)).to(BF)
    q1, q2 = _w4_experts(experts, h, i, 32, False, BF, seed=40)
    ids, weights = _routing(n, k, experts, seed=41)
    (w1, s1), (w2, s2) = codes64(*q1), codes64(*q2)
    want, bound = _want(x, ids, weights, w1, w2, s1, s2, 32, 32)
    packs = dict(packed=w4.pack_w4_gate_up(*_dev(q1)), packed_down=w4.pack_w4(*_dev(q2)))
    args = [v.to(DEV) for v in (x, ids, weights)]
    got = moe.fused_moe(*args, None, None, **packs)
    check(got, want, bound)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe.fused_moe(*args, None, None, **packs)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_w4_hidden_past_the_limit_is_refused():
    q1, q2 = _w4_experts(1, 16416, 32, 32, False, BF, seed=42)
    x, weights = torch.zeros(1, 16416, dtype=BF, device=DEV), torch.ones(1, 1, device=DEV)
    ids = torch.zeros(1, 1, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError):
        moe.fused_moe(x, ids, weights, None, None, packed=w4.pack_w4_gate_up(*_dev(q1)), packed_down=w4.pack_w4(*_dev(q2)))


@pytest.mark.parametrize("w4_bits", [False, True])
def test_more_than_64_assignments_and_fewer_agree(w4_bits):
    """The groups are found two ways, one assignment a lane (12 tokens) or by a count (24)."""
    w1, w2 = (v.to(DEV) for v in _half(32, 256, 128, BF, seed=43))
    if w4_bits:
        packs = dict(packed=w4.pack_w4_gate_up(*w4.quantize_w4(w1, 64)), packed_down=w4.pack_w4(*w4.quantize_w4(w2, 64)))
        w1 = w2 = None
    else:
        packs = {}
    x = torch.randn(24, 256, generator=torch.Generator().manual_seed(44)).to(BF).to(DEV)
    ids, weights = (v.to(DEV) for v in _routing(24, 4, 32, seed=45))
    want = torch.cat([moe.fused_moe(x[i:i + 12], ids[i:i + 12], weights[i:i + 12], w1, w2, **packs) for i in (0, 12)])
    got = moe.fused_moe(x, ids, weights, w1, w2, **packs)
    # the order of a token's choices may differ with the groups': fp32 sums of 4 terms, then one rounding
    assert float((got.float() - want.float()).abs().max()) <= 2 * half_ulp(BF) * float(want.float().abs().max())


def test_two_threads_on_one_stream():
    """A call is two launches: each host thread has a workspace of its own."""
    import threading
    w1, w2 = (v.to(DEV) for v in _half(16, 512, 256, BF, seed=61))
    ids, weights = (v.to(DEV) for v in _routing(8, 4, 16, seed=62))
    xs = [torch.randn(8, 512, generator=torch.Generator().manual_seed(63 + i)).to(BF).to(DEV) for i in range(2)]
    want = [moe.fused_moe(x, ids, weights, w1, w2) for x in xs]
    got = [[], []]
    threads = [threading.Thread(target=lambda i=i: got[i].extend(moe.fused_moe(xs[i], ids, weights, w1, w2) for _ in range(50)))
               for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(len(g) == 50 and all(torch.equal(o, want[i]) for o in g) for i, g in enumerate(got))


def test_captured_before_any_eager_call_on_its_stream():
    w1, w2 = (v.to(DEV) for v in _half(8, 256, 128, BF, seed=64))
    q = dict(packed=w4.pack_w4_gate_up(*w4.quantize_w4(w1, 32)), packed_down=w4.pack_w4(*w4.quantize_w4(w2, 64)))
    ids, weights = (v.to(DEV) for v in _routing(5, 3, 8, seed=65))
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(66)).to(BF).to(DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        half = moe.fused_moe(x, ids, weights, w1, w2)
        four = moe.fused_moe(x, ids, weights, None, None, **q)
    for i in range(3):
        x.copy_(x + 0.25)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(half, moe.fused_moe(x, ids, weights, w1, w2))
        assert torch.equal(four, moe.fused_moe(x, ids, weights, None, None, **q))


def test_two_streams():
    """Calls on two streams at once have workspaces of their own."""
    w1, w2 = (v.to(DEV) for v in _half(16, 1024, 256, BF, seed=19))
    x = torch.randn(8, 1024, generator=torch.Generator().manual_seed(20)).to(BF).to(DEV)
    ids, weights = (v.to(DEV) for v in _routing(8, 4, 16, seed=21))
    want = moe.fused_moe(x, ids, weights, w1, w2)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(moe.fused_moe(x, ids, weights, w1, w2))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_native_host_path_equals_the_wrapper(monkeypatch):
    """The same bits with and without the extension over both kinds of packed weights; what neither takes is
    refused either way."""
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(23)).to(BF).to(DEV)
    w1, w2 = (v.to(DEV) for v in _half(8, 128, 64, BF, seed=24))
    ids, weights = (v.to(DEV) for v in _routing(5, 2, 8, seed=25))
    q1, q2 = _w4_experts(8, 128, 64, 32, True, BF, seed=26)
    packs = [(moe.pack_moe_gate_up_weight(w1), moe.pack_moe_down_weight(w2)),
             (w4.pack_w4_gate_up(*_dev(q1)), w4.pack_w4(*_dev(q2)))]

    def run(p, x=x, ids=ids, weights=weights):
        return moe.fused_moe(x, ids, weights, None, None, packed=p[0], packed_down=p[1])

    def all_runs():
        return [run(p, **c) for p in packs for c in (
            {}, dict(ids=ids.int()), dict(weights=weights.to(BF)), dict(ids=ids.T.contiguous().T), dict(x=x[:1], ids=ids[:1], weights=weights[:1]),
            dict(x=torch.cat([x, x], 1)[:, 4:132].clone()[:, :128]))]

    got = all_runs()
    with monkeypatch.context() as m:
        m.setattr(_lib, "fast", _lib._Fast())
        assert all(torch.equal(g, w) for g, w in zip(got, all_runs()))
    for p in packs:
        with pytest.raises(ValueError):
            run(p, x=x.repeat(13, 1), ids=ids.repeat(13, 1), weights=weights.repeat(13, 1))  # 65 tokens
        with pytest.raises(ValueError):
            run(p, ids=ids[:4])
        with pytest.raises(TypeError):
            run(p, x=x.float())
    with pytest.raises((TypeError, ValueError)):
        run((packs[0][0], packs[1][1]))
    with pytest.raises(TypeError):
        run(packs[0], x=x.half())


def test_check_indices_reads_the_error_word(monkeypatch):
    monkeypatch.setenv("EMBERSERVE_CHECK_INDICES", "1")
    x = torch.randn(3, 128, generator=torch.Generator().manual_seed(27)).to(BF).to(DEV)
    w1, w2 = (v.to(DEV) for v in _half(4, 128, 64, BF, seed=28))
    ids, weights = (v.to(DEV) for v in _routing(3, 2, 4, seed=29))
    moe.fused_moe(x, ids, weights, w1, w2)
    ids[1, 1] = 4
    with pytest.raises(IndexError):
        moe.fused_moe(x, ids, weights, w1, w2)


def test_decode_step_of_w4_model(monkeypatch):
    """A step as a model runs it: qkv (bias), o, router, 4-bit experts and head, eager against fused."""
    h, i, experts = 256, 128, 8
    g = torch.Generator().manual_seed(22)
    x = torch.randn(5, h, generator=g).to(BF).to(DEV)
    qkv = w4.pack_w4(*w4.quantize_w4((torch.randn(3 * h, h, generator=g) / 16).to(BF).to(DEV), 64))
    o = w4.pack_w4(*w4.quantize_w4((torch.randn(h, h, generator=g) / 16).to(BF).to(DEV), 32, symmetric=False))
    up = w4.pack_w4_gate_up(*w4.quantize_w4((torch.randn(experts, 2 * i, h, generator=g) / 16).to(BF).to(DEV), 128))
    down = w4.pack_w4(*w4.quantize_w4((torch.randn(experts, h, i, generator=g) / 11).to(BF).to(DEV), 128))
    router = (torch.randn(h, experts, generator=g) / 16).to(BF).to(DEV)
    bias = torch.randn(3 * h, generator=g).to(BF).to(DEV)

    def step():
        q = w4.linear_w4(x, qkv, bias)
        y = w4.linear_w4(q[:, :h], o)
        top = torch.topk((x.float() @ router.float()), 2, dim=-1)
        return y, moe.fused_moe(y, top.indices, torch.softmax(top.values, -1), None, None, packed=up, packed_down=down)

    y, z = step()
    monkeypatch.setenv("EMBERSERVE_FUSED_OPS", "0")
    y0, z0 = step()
    # the same fp32 formulas but for the order of sums, the roundings of q, y and act and their flips (2 h each
    # of values summed at random): y within 4 h of its rms, z within 8 h
    for a, b, n in ((y, y0, 4), (z, z0, 8)):
        rms = b.double().pow(2).mean().sqrt()
        assert float((a.double() - b.double()).pow(2).mean().sqrt() / rms) < n * half_ulp(BF)
