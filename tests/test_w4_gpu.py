"""4-bit projections (`w4.linear_w4`, `w4.gate_up_silu_w4`) on the GPU against 64-bit values, with the
bounds of tests.w4_bounds."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from emberserve_amd import _lib, w4  # noqa: E402
from tests.w4_bounds import act_bound, check, codes64, dot_bound  # noqa: E402

DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _weight(n, k, group, zeros, dtype, seed, experts=None):
    g = torch.Generator().manual_seed(seed)
    lead = () if experts is None else (experts,)
    q = torch.randint(0, 256, (*lead, n, k // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand((*lead, n, k // group), generator=g) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def _x(t, k, dtype, seed):
    return torch.randn(t, k, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _dev(parts):
    return [None if p is None else p.to(DEV) for p in parts]


@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("n,k,group", [(16, 32, 32), (20, 128, 64), (6, 192, 64), (34, 416, 32), (48, 1024, 256)])
def test_pack_round_trip(n, k, group, gate_up):
    parts = _weight(n, k, group, True, HF, seed=n)
    packed = (w4.pack_w4_gate_up if gate_up else w4.pack_w4)(*_dev(parts))
    want = w4.dequantize_w4(*parts, dtype=torch.float32)
    assert torch.equal(packed.dequantize(torch.float32).cpu(), want)
    stacked = [torch.stack([p, p.flip(0)]) for p in parts]
    packed = (w4.pack_w4_gate_up if gate_up else w4.pack_w4)(*_dev(stacked))
    assert torch.equal(packed.dequantize(torch.float32).cpu(), w4.dequantize_w4(*stacked, dtype=torch.float32))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,n,k,group,zeros", [
    (1, 16, 32, 32, False), (1, 1, 64, 64, True), (3, 17, 96, 32, True), (16, 48, 896, 128, False),
    (17, 1152, 896, 64, True), (33, 100, 4864, 128, True), (64, 272, 1024, 32, False), (65, 33, 160, 32, True),
    (200, 64, 384, 128, False), (2, 3584, 2048, 512, True), (5, 40000, 256, 128, False), (31, 70001, 128, 64, True),
    (50, 70000, 64, 32, False),
    (9, 14500, 160, 32, True), (32, 14340, 384, 128, False), (40, 33000, 96, 32, False), (64, 57000, 128, 64, True),
    (90, 31000, 160, 32, True), (16, 65500, 128, 128, False)])
def test_linear_matches_64_bits(dtype, t, n, k, group, zeros):
    print(f"linear_w4 {t}x{n}x{k} g{group} zeros={zeros} {dtype}", flush=True)
    parts, x = _weight(n, k, group, zeros, dtype, seed=t + n), _x(t, k, dtype, seed=k)
    w, s = codes64(*parts)
    want, bound = dot_bound(x, w, s, group)
    packed = w4.pack_w4(*_dev(parts))
    got = w4.linear_w4(x.to(DEV), packed)
    assert got.dtype == dtype and got.shape == (t, n)
    check(got, want, bound, "no bias")
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(dtype)
    got = w4.linear_w4(x.to(DEV), packed, bias.to(DEV))
    check(got, want + bias.double(), bound + 2.0 ** -23 * (want.abs() + bias.double().abs()), "bias")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,inter,k,group,zeros", [
    (1, 16, 32, 32, True), (2, 5, 128, 128, False), (16, 4864, 896, 128, True), (27, 77, 416, 32, True),
    (64, 160, 512, 64, False), (70, 30, 256, 256, True), (9, 40000, 128, 64, False), (40, 33000, 64, 32, True),
    (9, 7200, 160, 32, True), (17, 7205, 640, 128, False), (31, 12290, 384, 64, True), (33, 16400, 96, 32, False),
    (64, 18944, 256, 128, True), (100, 16385, 128, 64, False), (12, 32760, 160, 32, False)])
def test_gate_up_matches_64_bits(dtype, t, inter, k, group, zeros):
    print(f"gate_up_silu_w4 {t}x{inter}x{k} g{group} zeros={zeros} {dtype}", flush=True)
    parts, x = _weight(2 * inter, k, group, zeros, dtype, seed=t + inter), _x(t, k, dtype, seed=k)
    w, s = codes64(*parts)
    want, bound = act_bound(*dot_bound(x, w, s, group))
    got = w4.gate_up_silu_w4(x.to(DEV), w4.pack_w4_gate_up(*_dev(parts)))
    check(got, want, bound)


def test_x_strides_and_alignment():
    """Rows far apart, rows of a transposed tensor, an odd first element: the same bits as contiguous."""
    parts = _weight(50, 256, 64, True, BF, seed=3)
    packed = w4.pack_w4(*_dev(parts))
    x = _x(9, 256, BF, seed=4).to(DEV)
    want = w4.linear_w4(x, packed)
    wide = torch.full((9, 1024), float("nan"), dtype=BF, device=DEV)
    wide[:, 256:512] = x
    assert torch.equal(w4.linear_w4(wide[:, 256:512], packed), want)
    assert torch.equal(w4.linear_w4(x.T.contiguous().T, packed), want)
    odd = torch.zeros(9 * 256 + 1, dtype=BF, device=DEV)[1:].view(9, 256)
    odd.copy_(x)
    assert torch.equal(w4.linear_w4(odd, packed), want)
    assert torch.equal(w4.linear_w4(x.view(3, 3, 256), packed), want.view(3, 3, 50))
    assert w4.linear_w4(x[:0], packed).shape == (0, 50)


def test_pack_of_strided_parts():
    """Codes, scales and zeros as views of wider tensors pack to the same array."""
    parts = _dev(_weight(48, 256, 64, True, HF, seed=5))
    want = w4.pack_w4(*parts).packed
    wide = [torch.cat([p, p.flip(0)], dim=1)[:, :p.shape[1]] for p in parts]
    assert torch.equal(w4.pack_w4(*wide).packed, want)
    cols = [p.T.contiguous().T for p in parts]
    assert torch.equal(w4.pack_w4(*cols).packed, want)


def test_nonfinite_rows_stay_their_own():
    """A token with a NaN or an infinity gives NaN in its row and leaves the others' bits alone."""
    parts = _weight(64, 416, 32, True, BF, seed=6)
    packed = w4.pack_w4(*_dev(parts))
    x = _x(20, 416, BF, seed=7).to(DEV)
    want = w4.linear_w4(x, packed)
    y = x.clone()
    y[3, 415] = float("nan")
    y[17, 0] = float("inf")
    got = w4.linear_w4(y, packed)
    assert bool(got[[3, 17]].isnan().all())
    keep = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(got[keep], want[keep])


def test_extreme_scales_and_values():
    """Zero, negative and subnormal scales, and x at the largest finite value that the sum allows."""
    q, s, z = _weight(32, 128, 32, True, HF, seed=8)
    s[0] = 0.0
    s[1] = -s[1]
    s[2] = 2.0 ** -24
    x = _x(4, 128, HF, seed=9)
    x[1] = 60000.0
    w, sa = codes64(q, s, z)
    want, bound = dot_bound(x, w, sa, 32)
    got = w4.linear_w4(x.to(DEV), w4.pack_w4(*_dev((q, s, z))))
    small = want.abs() < 65000
    check(torch.where(small.to(DEV), got, 0), torch.where(small, want, 0.0), bound)
    over = want.abs() > 66000  # past fp16's range: the rounded value is infinite
    assert bool(got.cpu()[over].isinf().all())


def test_tiny_and_large_values():
    """Subnormal x beside ordinary ones (each token its own size), and bf16 x as large as the sums hold."""
    for dtype, sizes in ((HF, (2.0 ** -24, 2.0 ** -20, 2.0 ** -14, 1.0)), (BF, (2.0 ** -130, 2.0 ** -100, 1.0, 2.0 ** 110))):
        parts = _weight(64, 256, 64, True, HF, seed=24)  # fp16 scales under either type of x
        x = torch.stack([_x(1, 256, torch.float32, seed=30 + i)[0] * v for i, v in enumerate(sizes)]).to(dtype)
        w, s = codes64(*parts)
        want, bound = dot_bound(x, w, s, 64)
        got = w4.linear_w4(x.to(DEV), w4.pack_w4(*_dev(parts)))
        # fp32 sums of such products may themselves be subnormal: 2^-149 a rounding
        check(got, want, bound + 400 * 2.0 ** -149, f"{dtype}")


def test_overlapping_rows():
    """One token for all rows, by a row stride of zero, and rows that overlap."""
    packed = w4.pack_w4(*_dev(_weight(48, 256, 64, False, BF, seed=25)))
    flat = _x(1, 512, BF, seed=26).to(DEV)[0]
    one = flat[:256].expand(9, 256)
    assert torch.equal(w4.linear_w4(one, packed), w4.linear_w4(one.contiguous(), packed))
    slide = flat.as_strided((20, 256), (8, 1))
    assert torch.equal(w4.linear_w4(slide, packed), w4.linear_w4(slide.contiguous(), packed))


@pytest.mark.parametrize("t,n,k", [(2000, 160, 256), (777, 40, 1056), (300, 24576, 128)])
def test_many_tokens(t, n, k):
    """Prefill-sized batches: many tiles of tokens, the last one ragged."""
    parts = _weight(n, k, 32, True, BF, seed=50)
    x = _x(t, k, BF, seed=51)
    w, s = codes64(*parts)
    rows = torch.cat((torch.arange(0, t, 37), torch.arange(t - 40, t)))
    want, bound = dot_bound(x[rows], w, s, 32)
    got = w4.linear_w4(x.to(DEV), w4.pack_w4(*_dev(parts)))
    check(got[rows.to(DEV)], want, bound)


def _need(t, k, n, group):
    counters = ctypes.c_int64(0)
    return _lib.load().ember_w4_linear_workspace_bytes(t, k, n, group, ctypes.byref(counters)), counters.value


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("t,n,k,group", [(24, 3584, 18944, 128), (61, 2056, 12288, 64), (17, 900, 4864, 32),
                                         (33, 40, 8224, 32), (64, 16, 16384, 256), (16, 200, 20480, 128)])
def test_long_rows_are_split(dtype, t, n, k, group):
    """A few long rows: the workgroups that share k join their sums, the same bits each time."""
    assert _need(t, k, n, group)[0] > 0
    parts = _weight(n, k, group, True, dtype, seed=70)
    x, bias = _x(t, k, dtype, seed=71), _x(1, n, dtype, seed=72)[0]
    w, s = codes64(*parts)
    want, bound = dot_bound(x, w, s, group)
    packed = w4.pack_w4(*_dev(parts))
    got = [w4.linear_w4(x.to(DEV), packed) for _ in range(4)]
    check(got[0], want, bound)
    assert all(torch.equal(g, got[0]) for g in got)
    biased = w4.linear_w4(x.to(DEV), packed, bias.to(DEV))
    y = want + bias.double()
    check(biased, y, bound + 2.0 ** -23 * y.abs())


def test_split_shapes_take_turns_graphs_and_threads():
    """Calls of several shapes on one workspace; two graphs at once beside eager calls; two host threads."""
    shapes = [(24, 1024, 8192), (61, 200, 12288), (17, 48, 16384), (3, 64, 4096), (24, 1024, 8192)]
    packs = [w4.pack_w4(*_dev(_weight(n, k, 128, False, BF, seed=80 + i))) for i, (_, n, k) in enumerate(shapes)]
    xs = [_x(t, k, BF, seed=90 + i).to(DEV) for i, (t, _, k) in enumerate(shapes)]
    assert sum(_need(t, k, n, 128)[0] > 0 for t, n, k in shapes) >= 4
    want = [w4.linear_w4(x, p) for x, p in zip(xs, packs)]
    for _ in range(3):
        for x, p, y in zip(xs, packs, want):
            assert torch.equal(w4.linear_w4(x, p), y)
    one, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=one):
            outs.append([w4.linear_w4(x, p) for x, p in zip(xs, packs)])
        graphs.append(g)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(one):
            eager = [w4.linear_w4(x, p) for x, p in zip(xs, packs)]
        torch.cuda.synchronize()
        for got in (*outs, eager):
            assert all(torch.equal(o, y) for o, y in zip(got, want))
    got = [[], []]
    threads = [threading.Thread(target=lambda i=i: got[i].extend(w4.linear_w4(xs[i], packs[i]) for _ in range(50)))
               for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(len(g) == 50 and all(torch.equal(o, want[i]) for o in g) for i, g in enumerate(got))


def test_split_with_and_without_a_workspace(monkeypatch):
    lib = _lib.load()
    t, n, k, group = 24, 1024, 8192, 128
    parts = _weight(n, k, group, False, BF, seed=100)
    packed, x = w4.pack_w4(*_dev(parts)), _x(t, k, BF, seed=101).to(DEV)
    need, counters = _need(t, k, n, group)
    ws, out = torch.zeros(need, dtype=torch.uint8, device=DEV), torch.empty(t, n, dtype=BF, device=DEV)

    def call(space, size):
        return lib.ember_w4_linear_split(x.data_ptr(), k, packed.packed.data_ptr(), group, 2, t, k, n, None, space, size,
                                         out.data_ptr(), n, torch.cuda.current_stream().cuda_stream)

    assert call(ws.data_ptr(), need - 16) == 1 and call(ws.data_ptr(), need - 8) == 2  # before any launch
    assert call(ws.data_ptr() + 8, need) == 2
    want, bound = dot_bound(x.cpu(), *codes64(*parts), group)
    for space, size in ((ws.data_ptr(), need), (None, 0)):
        out.zero_()
        assert call(space, size) == 0
        check(out, want, bound)
    assert not bool(ws[need - counters:].any())
    eager = w4.linear_w4(x, packed)
    monkeypatch.setenv("EMBERSERVE_CHECK_INDICES", "1")  # the wrapper's path, which looks at the counters
    assert torch.equal(w4.linear_w4(x, packed), eager)


def test_rows_far_apart_are_copied():
    """Row strides past what 32-bit offsets reach over 64 rows."""
    parts = _weight(48, 128, 64, False, BF, seed=52)
    packed = w4.pack_w4(*_dev(parts))
    stride = w4.MAX_ROW_STRIDE + 8
    big = torch.zeros(2 * stride + 128, dtype=BF, device=DEV)
    x = big.as_strided((3, 128), (stride, 1))
    x.copy_(_x(3, 128, BF, seed=53))
    assert torch.equal(w4.linear_w4(x, packed), w4.linear_w4(x.contiguous(), packed))


def test_rows_at_the_largest_stride():
    """64 rows at the largest stride that is read in place: offsets up to 2^30."""
    parts = _weight(32768, 128, 64, False, BF, seed=54)
    stride = w4.MAX_ROW_STRIDE
    big = torch.zeros(63 * stride + 128, dtype=BF, device=DEV)
    x = big.as_strided((64, 128), (stride, 1))
    x.copy_(_x(64, 128, BF, seed=55))
    for sub in (parts, tuple(None if p is None else p[:48] for p in parts)):
        packed = w4.pack_w4(*_dev(sub))
        assert torch.equal(w4.linear_w4(x, packed), w4.linear_w4(x.contiguous(), packed))


def test_more_threads_than_one_launch_takes():
    """2^23 slabs of 16 rows: 64 tokens a launch, the 66 take two."""
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of device memory")
    slabs = (1 << 23) - 8
    q = torch.randint(0, 256, (slabs * 16, 16), dtype=torch.uint8, device=DEV)
    s = torch.ones(slabs * 16, 1, dtype=BF, device=DEV)
    packed = w4.pack_w4(q, s)
    g = torch.Generator().manual_seed(60)
    x = torch.randint(-4, 5, (66, 32), generator=g).to(BF).to(DEV)  # sums of whole numbers, exact in fp32
    got = w4.linear_w4(x, packed)
    n = slabs * 16
    some = torch.cat((torch.arange(64), torch.randint(0, n, (256,), generator=g), torch.arange(n - 64, n))).to(DEV)
    codes = torch.stack((q[some] & 15, q[some] >> 4), -1).reshape(-1, 32).float() - 8
    assert torch.equal(got[:, some], (x.float() @ codes.T).to(BF))


def test_two_threads_on_one_stream():
    """Calls of two host threads, each into its own output."""
    parts = _weight(256, 1024, 128, False, BF, seed=56)
    packed = w4.pack_w4(*_dev(parts))
    xs = [_x(5 + 8 * i, 1024, BF, seed=57 + i).to(DEV) for i in range(2)]
    want = [w4.linear_w4(x, packed) for x in xs]
    got = [[], []]
    threads = [threading.Thread(target=lambda i=i: got[i].extend(w4.linear_w4(xs[i], packed) for _ in range(50)))
               for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(len(g) == 50 and all(torch.equal(o, want[i]) for o in g) for i, g in enumerate(got))


def test_graph_replays_match_eager():
    parts, gu = _weight(1152, 896, 128, False, BF, seed=10), _weight(2 * 304, 896, 128, False, BF, seed=11)
    packed, packed_gu = w4.pack_w4(*_dev(parts)), w4.pack_w4_gate_up(*_dev(gu))
    x = _x(3, 896, BF, seed=12).to(DEV)
    w4.linear_w4(x, packed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = w4.linear_w4(x, packed), w4.gate_up_silu_w4(x, packed_gu)
    for i in range(3):
        x.copy_(_x(3, 896, BF, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, w4.linear_w4(x, packed)) and torch.equal(b, w4.gate_up_silu_w4(x, packed_gu)), i


def test_another_stream():
    parts = _weight(256, 1024, 128, False, BF, seed=13)
    packed = w4.pack_w4(*_dev(parts))
    x = _x(4, 1024, BF, seed=14).to(DEV)
    want = w4.linear_w4(x, packed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = w4.linear_w4(x, packed)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_eager_form_of_a_gpu_weight(monkeypatch):
    """EMBERSERVE_FUSED_OPS=0 computes from the packed copy in torch."""
    parts = _weight(40, 256, 64, True, BF, seed=15)
    x = _x(5, 256, BF, seed=16)
    w, s = codes64(*parts)
    want, bound = dot_bound(x, w, s, 64)
    packed = w4.pack_w4(*_dev(parts))
    monkeypatch.setenv("EMBERSERVE_FUSED_OPS", "0")
    check(w4.linear_w4(x.to(DEV), packed), want, bound + 300 * 2.0 ** -24 * (x.double().abs() @ w.abs().T))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_native_host_path_equals_the_wrappers(dtype, monkeypatch):
    """The same bits, shapes and refusals with and without the extension, for calls it answers and calls
    it leaves alone."""
    parts, gu = _weight(40, 256, 64, True, dtype, seed=17), _weight(96, 256, 32, False, dtype, seed=18)
    packed, packed_gu = w4.pack_w4(*_dev(parts)), w4.pack_w4_gate_up(*_dev(gu))
    x = _x(6, 256, dtype, seed=19).to(DEV)
    bias = torch.randn(80, generator=torch.Generator().manual_seed(20)).to(dtype).to(DEV)
    wide = torch.zeros(6, 600, dtype=dtype, device=DEV)
    wide[:, 8:264] = x
    calls = [lambda: w4.linear_w4(x, packed), lambda: w4.linear_w4(x, packed, bias[:40]),
             lambda: w4.linear_w4(x, packed, bias[::2]), lambda: w4.linear_w4(wide[:, 8:264], packed),
             lambda: w4.linear_w4(wide[:, 9:265], packed), lambda: w4.linear_w4(x.view(2, 3, 256), packed),
             lambda: w4.linear_w4(x[0], packed), lambda: w4.linear_w4(x[:0], packed),
             lambda: w4.gate_up_silu_w4(x, packed_gu), lambda: w4.gate_up_silu_w4(x.view(3, 2, 256), packed_gu)]
    got = [c() for c in calls]
    monkeypatch.setattr(_lib, "fast", _lib._Fast())
    for g, c in zip(got, calls):
        want = c()
        assert g.shape == want.shape and g.dtype == want.dtype and torch.equal(g, want)
    monkeypatch.undo()
    for bad in (lambda: w4.linear_w4(x, packed_gu), lambda: w4.gate_up_silu_w4(x, packed),
                lambda: w4.linear_w4(x[:, :128], packed), lambda: w4.linear_w4(x, packed, bias),
                lambda: w4.linear_w4(x, packed, bias[:40].cpu())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        w4.linear_w4(x.float(), packed)


def test_registered_ops():
    """Schemas, fake kernels and results of torch.ops.emberserve's forms, and one traced by torch.compile."""
    from emberserve_amd import torch_ops
    parts, gu = _weight(48, 128, 64, True, BF, seed=21), _weight(64, 128, 32, False, BF, seed=22)
    packed, packed_gu = w4.pack_w4(*_dev(parts)), w4.pack_w4_gate_up(*_dev(gu))
    x = _x(3, 128, BF, seed=23).to(DEV)
    torch.library.opcheck(torch.ops.emberserve.linear_w4, (x, packed.packed, None, 48, 128, 64))
    torch.library.opcheck(torch.ops.emberserve.gate_up_silu_w4, (x, packed_gu.packed, 32, 128, 32))
    assert torch.equal(torch_ops.linear_w4(x, packed), w4.linear_w4(x, packed))
    assert torch.equal(torch_ops.gate_up_silu_w4(x, packed_gu), w4.gate_up_silu_w4(x, packed_gu))
    with pytest.raises(ValueError):
        torch.ops.emberserve.linear_w4(x, packed.packed[:, :1024].contiguous(), None, 48, 128, 64)
    compiled = torch.compile(lambda v: torch_ops.linear_w4(v, packed) * 2, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(x), w4.linear_w4(x, packed) * 2)


def test_no_error_bits():
    assert _lib.read_errors(clear=True) == 0
