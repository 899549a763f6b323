"""The 8-bit matrix product on gfx950 against the float64 oracle, and the 8-bit path as a model runs it.

The integer sum is exact, so a result is off by its fp32 operations (the sum's conversion, two products,
two additions: five roundings of at most E = 2^-24 of the terms' magnitudes) and one rounding to 16
bits (half a step: 2^-11 or 2^-8 of the value, 2^-25 absolute below fp16's normal range)."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import layouts, torch_ops
from oracle import rows8 as orr
from test_rows8_gpu import DT, E, TINY16, U, guarded, host, inputs, shifted

pytestmark = pytest.mark.gpu


def operands(m, k, n, kind, b, residual, seed=0):
    rng = np.random.default_rng(seed + m + 1000 * n + k)
    kp = (k + 63) // 64 * 64
    q, w = np.zeros((m, kp), np.int8), np.zeros((n, kp), np.int8)
    q[:, :k] = rng.integers(-127, 128, (m, k))
    w[:, :k] = rng.integers(-127, 128, (n, k))
    qs = rng.uniform(0.5, 2, m).astype(np.float32) / 127
    ws = (rng.uniform(0.5, 2, n) * k ** -0.5 / 60).astype(np.float32)
    t = dict(q=torch.from_numpy(q).cuda(), qs=torch.from_numpy(qs).cuda(), w=torch.from_numpy(w).cuda(),
             ws=torch.from_numpy(ws).cuda(), b=None, residual=None)
    t["wq"] = layouts.q8_blocked(t["w"])
    if b:
        t["b"] = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda()
    if residual:
        t["residual"] = torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32)).to(DT[kind]).cuda()
    return t


def call(hip, t, kind, **kw):
    return hip.q8_projection(t["q"], t["qs"], t["wq"], t["ws"], t["b"], t["residual"], DT[kind], **kw)


def check(out, t, kind, rows=slice(None)):
    # float64 on the GPU: the same products, by another route
    s = t["q"][rows].double() @ t["w"].double().t()
    out, s = out[rows], s * t["qs"][rows].double()[:, None] * t["ws"].double()
    want, mag = s, s.abs()
    for other in (t["b"], None if t["residual"] is None else t["residual"][rows]):
        if other is not None:
            want, mag = want + other.double(), mag + other.double().abs()
    err = (out.double() - want).abs()
    assert out.dtype == DT[kind] and bool((err <= U[kind] * want.abs() + 6 * E * mag + TINY16[kind]).all()), float(err.max())


def test_check_agrees_with_the_oracle(hip):
    t = operands(5, 70, 9, "f16", True, True)
    want, _ = orr.project(host(t["q"]), host(t["qs"]), host(t["w"]), host(t["ws"]), host(t["b"]), host(t["residual"]))
    got = call(hip, t, "f16")
    assert np.abs(host(got) - want).max() <= 2.0 ** -11 * np.abs(want).max() + 1e-5
    check(got, t, "f16")


@pytest.mark.parametrize("m", [1, 2, 5, 15, 16, 17, 31, 33, 48, 63, 64, 65, 100, 128, 129, 200, 256, 257, 500])
@pytest.mark.parametrize("k,n", [(64, 64), (200, 72), (512, 65), (1100, 300), (2048, 1000)])
def test_sizes(hip, m, k, n):
    for kind, b, residual in (("f16", True, False), ("bf16", False, True)):
        t = operands(m, k, n, kind, b, residual)
        check(call(hip, t, kind), t, kind)


@pytest.mark.parametrize("n", [1, 3, 4, 7, 15, 16, 17, 63, 66, 127, 128, 130, 191, 255, 256, 257])
@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_odd_channels(hip, m, n):
    for kind, b, residual in (("bf16", True, True), ("f16", False, False)):
        t = operands(m, 192, n, kind, b, residual)
        check(call(hip, t, kind), t, kind)


@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (3, 8192, 1024), (48, 4096, 2048), (147, 128, 512), (4000, 128, 512),
                                   (20011, 64, 64), (5000, 256, 128), (1531, 1100, 2050), (1024, 1024, 1024), (2048, 4096, 512),
                                   (700, 8192, 4096), (1, 64, 20000), (513, 640, 2304), (2304, 320, 2304), (4096, 2048, 4096)])
def test_large(hip, m, k, n):
    for kind, b, residual in (("f16", True, True), ("bf16", False, False)):
        t = operands(m, k, n, kind, b, residual)
        check(call(hip, t, kind), t, kind)


@pytest.mark.parametrize("k", [1, 64, 100, 128, 192, 256, 300, 512, 513])
@pytest.mark.parametrize("m,n", [(2047, 64), (2048, 8), (2049, 72), (2100, 256), (2500, 264), (3001, 520), (5003, 128),
                                 (20011, 40), (2300, 1032)])
def test_many_rows_short_k(hip, m, n, k):
    """Where rows stream past weights in registers: every depth, ends inside tiles, channels past a block."""
    for kind, b, residual in (("f16", True, True), ("bf16", True, False), ("f16", False, False)):
        t = operands(m, k, n, kind, b, residual)
        out, ok = guarded((m, n), DT[kind], 7.0)
        check(call(hip, t, kind, out=out), t, kind)
        assert ok()
    t = operands(m, k, n, "bf16", True, True)
    want = call(hip, t, "bf16")
    res = t["residual"].clone()
    assert torch.equal(call(hip, dict(t, residual=res), "bf16", out=res), want)
    assert torch.equal(call(hip, dict(t, residual=shifted(t["residual"])), "bf16"), want)
    assert torch.equal(call(hip, t, "bf16", out=shifted(want)), want)
    rows = dict(t, q=t["q"][7:60].contiguous(), qs=t["qs"][7:60].contiguous(), residual=t["residual"][7:60].contiguous())
    assert torch.equal(call(hip, rows, "bf16"), want[7:60])  # a row's result is the same in a batch of any size


@pytest.mark.parametrize("k", [64, 128, 256, 500])
@pytest.mark.parametrize("m,n", [(2048, 2), (2049, 6), (2100, 62), (2500, 130), (3001, 254), (5003, 258), (20011, 42),
                                 (2300, 1030), (2048, 510)])
def test_many_rows_even_channels(hip, m, n, k):
    """As above with rows that end inside a 16-byte piece: the cut piece and what lies behind the last row."""
    for kind, b, residual in (("f16", True, True), ("bf16", True, False), ("bf16", False, True)):
        t = operands(m, k, n, kind, b, residual)
        out, ok = guarded((m, n), DT[kind], 7.0)
        check(call(hip, t, kind, out=out), t, kind)
        assert ok()
    res = t["residual"].clone()
    assert torch.equal(call(hip, dict(t, residual=res), "bf16", out=res), out)
    rows = dict(t, q=t["q"][7:60].contiguous(), qs=t["qs"][7:60].contiguous(), residual=t["residual"][7:60].contiguous())
    assert torch.equal(call(hip, rows, "bf16"), out[7:60])


@pytest.mark.parametrize("m,k,n", [(3000, 128, 256), (300, 1024, 512), (700, 192, 130), (2304, 640, 2304)])
@pytest.mark.parametrize("residual", [False, True])
def test_results_off_lines(hip, m, k, n, residual):
    """Results that start 16 bytes (or 2) into a line are the same bits."""
    t = operands(m, k, n, "f16", True, residual)
    want = call(hip, t, "f16")
    check(want, t, "f16")
    for by in (1, 8, 40):
        flat = torch.full((m * n + 128,), 7.0, dtype=torch.float16, device="cuda")
        out = flat[by:by + m * n].view(m, n)
        assert torch.equal(call(hip, t, "f16", out=out), want)
        assert (flat[:by] == 7).all() and (flat[by + m * n:] == 7).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("k,n", [(128, 512), (500, 254), (1024, 1024), (1000, 511)])
@pytest.mark.parametrize("b,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_a_row_is_the_same_in_calls_of_any_size(hip, kind, k, n, b, residual):
    t = operands(9000, k, n, kind, b, residual)
    want = call(hip, t, kind)
    for lo, hi in ((0, 1), (5, 8), (100, 148), (300, 500), (1000, 1700), (2000, 5000), (8, 9000)):
        part = dict(t, q=t["q"][lo:hi], qs=t["qs"][lo:hi].clone(), residual=t["residual"][lo:hi].clone() if residual else None)
        assert torch.equal(call(hip, part, kind), want[lo:hi])


@pytest.mark.parametrize("m", [1, 20, 70, 300, 600])
def test_sums_are_exact(hip, m):
    """The longest rows of the largest integers: the sums reach 131008 * 128 * 128, just under 2^31, and one
    step of them is far under fp32's resolution, so neighbours that cancel are compared too."""
    kp, n = 131008, 70
    q = torch.full((m, kp), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, kp), -128, dtype=torch.int8, device="cuda")
    w[1, ::2] = 127      # nearly cancels
    w[2, 7:] = 0
    q[m // 2, 1000:] = 127
    ones = lambda r: torch.ones(r, device="cuda")  # noqa: E731
    scale = 2.0 ** -20
    t = dict(q=q, qs=ones(m), w=w, ws=ones(n) * scale, wq=layouts.q8_blocked(w), b=None, residual=None)
    check(call(hip, t, "f16"), t, "f16")
    check(call(hip, t, "bf16"), t, "bf16")


def test_special_scales(hip):
    """A row or channel whose scale is NaN is NaN, a zero scale gives the bias; the others are untouched."""
    t = operands(70, 128, 100, "f16", True, False)
    t["qs"][3], t["qs"][5] = float("nan"), 0.0
    t["ws"][7], t["ws"][9] = float("nan"), 0.0
    out = call(hip, t, "f16")
    assert torch.isnan(out[3]).all() and torch.isnan(out[:, 7]).all()
    keep_r = [i for i in range(70) if i != 3]
    keep_c = [i for i in range(100) if i != 7]
    assert not torch.isnan(out[keep_r][:, keep_c]).any()
    assert torch.equal(out[5, keep_c], t["b"][keep_c].half()) and torch.equal(out[keep_r, 9], t["b"][9].half().expand(69))


@pytest.mark.parametrize("m,n", [(1, 65), (20, 66), (70, 131), (300, 257), (600, 1000)])
def test_nothing_outside_is_written(hip, m, n):
    t = operands(m, 320, n, "bf16", True, True)
    out, ok = guarded((m, n), torch.bfloat16, 7.0)
    check(call(hip, t, "bf16", out=out), t, "bf16")
    assert ok()


@pytest.mark.parametrize("m,n", [(1, 65), (20, 64), (70, 131), (300, 256), (600, 1000)])
def test_in_place_and_odd_addresses(hip, m, n):
    t = operands(m, 320, n, "f16", True, True)
    want = call(hip, t, "f16")
    t2 = dict(t, residual=shifted(t["residual"]), b=shifted(t["b"]), qs=shifted(t["qs"]), ws=shifted(t["ws"]))
    assert torch.equal(call(hip, t2, "f16", out=t2["residual"]), want)
    assert torch.equal(call(hip, t, "f16", out=shifted(want)), want)


def test_many_row_tiles(hip):
    """More rows than 65535 tiles of 16, and offsets past 2^32 bytes in the result."""
    m, k, n = 1100003, 64, 2000
    t = operands(3, k, n, "f16", True, False)
    q = t["q"][:1].expand(m, -1).contiguous()
    q[-3:] = t["q"]
    qs = t["qs"][:1].expand(m).contiguous()
    qs[-3:] = t["qs"]
    out = hip.q8_projection(q, qs, t["wq"], t["ws"], t["b"])
    want = call(hip, t, "f16")
    check(want, t, "f16")
    assert torch.equal(out[-3:], want) and torch.equal(out[m // 2], want[0]) and torch.equal(out[m - 4], want[0])


# ---- as a model runs them --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lead,c,hidden,activation", [((1,), 256, 1024, "relu"), ((3, 17), 128, 512, "relu"),
                                                      ((130,), 200, 300, "swish_gate"), ((2, 600), 1024, 1024, "swish_gate")])
def test_transition(hip, lead, c, hidden, activation, kind):
    """norm -> product -> activation -> product + stream: each step against the oracle on that step's own
    inputs, and the whole against torch_ops.q8_transition bit for bit."""
    m = int(np.prod(lead))
    x, res, scale = inputs(m, c, kind, True)
    rng = np.random.default_rng(5)
    wide = 2 * hidden if activation == "swish_gate" else hidden
    w1, w2 = (torch.from_numpy((rng.standard_normal(s) * s[0] ** -0.5).astype(np.float32)).cuda() for s in ((c, wide), (hidden, c)))
    b1, b2 = (torch.from_numpy((0.1 * rng.standard_normal(n)).astype(np.float32)).cuda() for n in (wide, c))
    w1q, w2q = torch_ops.q8_weights(w1), torch_ops.q8_weights(w2)
    for w, (wq, ws) in ((w1, w1q), (w2, w2q)):
        ints = layouts.q8_unblocked(wq, w.shape[1]).double()[:, :w.shape[0]]
        assert bool(((ints * ws.double()[:, None] - w.double().t()).abs() <= (0.5 + 1e-4) * ws.double()[:, None]).all())
    out, total = torch_ops.q8_transition(x.view(lead + (c,)), scale, w1q, b1, w2q, b2, res.view(lead + (c,)), activation, True)
    assert out.shape == lead + (c,) and total.shape == lead + (c,)

    q, qs, s = hip.rms_norm_q8(x, scale, res)
    h = hip.q8_projection(q, qs, *w1q, b1, None, DT[kind])
    t = dict(q=q, qs=qs, w=layouts.q8_unblocked(w1q[0], wide), ws=w1q[1], b=b1, residual=None)
    check(h, t, kind)
    hq, hs = hip.quantize_rows(h, {"relu": 1, "swish_gate": 2}[activation])
    y = hip.q8_projection(hq, hs, *w2q, b2, s, DT[kind])
    t = dict(q=hq, qs=hs, w=layouts.q8_unblocked(w2q[0], c), ws=w2q[1], b=b2, residual=s)
    check(y, t, kind)
    assert torch.equal(out.view(m, c), y) and torch.equal(total.view(m, c), s)

    # against the same block in float64 without 8 bits: rows and weights are off by up to half a step, a / 254,
    # spread evenly (a / 440 in the mean square); with a at 4 to 6 spreads that is 1.4% for each of the four
    # operands, 3% for all, which the activation passes on; three times that is allowed
    sd = host(s)
    hid = orr.hidden(orr.rms_norm(sd, host(scale), 1e-5)[0] @ host(w1) + host(b1), {"relu": 1, "swish_gate": 2}[activation])
    want = hid @ host(w2) + host(b2)
    assert np.linalg.norm(host(y) - sd - want) <= 0.1 * np.linalg.norm(want) + 2 * U[kind] * np.linalg.norm(sd)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_rms_norm_autograd(hip, kind):
    x, res, w = inputs(40, 200, kind, True)
    dy, ds = torch.randn_like(x), torch.randn_like(x)
    x, res, w = (t.view(s).requires_grad_() for t, s in ((x, (8, 5, 200)), (res, (8, 5, 200)), (w, (200,))))
    y, total = torch_ops.rms_norm(x, w, res)
    gx, gr, gw = torch.autograd.grad((y, total), (x, res, w), (dy.view(8, 5, 200), ds.view(8, 5, 200)))
    s2 = total.detach().view(40, 200)
    _, _, rstd = hip.rms_norm(s2, w.detach(), want_rstd=True)
    want, wantw = hip.rms_norm_bwd(s2, w.detach(), rstd, dy, ds)
    assert torch.equal(gx.view(40, 200), want) and torch.equal(gr, gx) and torch.equal(gw, wantw)
    # without a residual, through a leaf used twice, with a 16-bit scale, and only one of the results used
    w16 = w.detach().to(DT[kind]).requires_grad_()
    y = torch_ops.rms_norm(x, w16)
    (y.float() * dy.view(8, 5, 200).float()).sum().backward()
    assert w16.grad.dtype == DT[kind] and x.grad.shape == x.shape
    x.grad = None
    y, total = torch_ops.rms_norm(x, w, x)
    total.backward(ds.view(8, 5, 200))
    assert torch.equal(x.grad, (2 * ds).view(8, 5, 200)) and w.grad is not None and (w.grad == 0).all()
    x.grad = w.grad = None
    y, total = torch_ops.rms_norm(x, w, x)
    y.backward(dy.view(8, 5, 200))
    s2 = total.detach().view(40, 200)
    _, _, rstd = hip.rms_norm(s2, w.detach(), want_rstd=True)
    assert torch.equal(x.grad.view(40, 200), 2 * hip.rms_norm_bwd(s2, w.detach(), rstd, dy)[0])


def test_rms_norm_autograd_corners(hip):
    """No rows, one value, an expanded gradient, a gradient of another type, a scale of its own shape, a
    second derivative."""
    w = torch.ones(96, device="cuda", requires_grad=True)
    x = torch.empty((0, 96), dtype=torch.float16, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(torch_ops.rms_norm(x, w), (x, w), torch.empty_like(x))
    assert gx.shape == x.shape and (gw == 0).all()
    x, _, w = inputs(5, 64, "bf16", False)
    x, w = x.view(1, 5, 64).requires_grad_(), w.view(1, 64).requires_grad_()
    y = torch_ops.rms_norm(x, w)
    g1 = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)  # a gradient without strides
    g2 = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.equal(g1[0], g2[0]) and torch.equal(g1[1], g2[1]) and g1[1].shape == w.shape
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(torch_ops.rms_norm(x, w).float().square().sum(), x, create_graph=True)[0]
        g.sum().backward()
    one = torch.full((1, 1), -3.0, dtype=torch.float16, device="cuda", requires_grad=True)
    y = torch_ops.rms_norm(one, torch.ones(1, device="cuda"), eps=0.0)
    assert y.item() == -1 and torch.autograd.grad(y, one)[0].abs().item() < 1e-3


def test_rms_norm_gradient_against_differences(hip):
    """The GPU's gradients against central differences of the float64 forward on the same values. The
    gradient carries a rounding to bf16 (2^-8 of itself), the differences an error far below that."""
    x, _, w = inputs(3, 24, "bf16", False)
    dy = torch.randn_like(x)
    x.requires_grad_()
    w.requires_grad_()
    gx, gw = torch.autograd.grad(torch_ops.rms_norm(x, w), (x, w), dy)
    f = lambda s, v: (orr.rms_norm(s, v, 1e-5)[0] * host(dy)).sum()  # noqa: E731
    s, v, h = host(x), host(w), 1e-5
    for i in range(3):
        for j in range(24):
            d = np.zeros_like(s)
            d[i, j] = h
            diff = (f(s + d, v) - f(s - d, v)) / (2 * h)
            assert abs(host(gx)[i, j] - diff) <= 2.0 ** -8 * abs(diff) + 1e-5
    for j in range(24):
        d = np.zeros_like(v)
        d[j] = h
        assert abs(host(gw)[j] - (f(s, v + d) - f(s, v - d)) / (2 * h)) <= 1e-5


def test_strided_views(hip):
    """torch_ops takes any strides; hip refuses what is not contiguous."""
    x, res, w = inputs(24, 96, "f16", True)
    big = torch.zeros((24, 200), dtype=torch.float16, device="cuda")
    big[:, 50:146] = x
    y, total = torch_ops.rms_norm(big[:, 50:146], w, res)
    want = hip.rms_norm(x, w, res)
    assert torch.equal(y, want[0]) and torch.equal(total, want[1])
    with pytest.raises(ValueError, match="contiguous"):
        hip.rms_norm(big[:, 50:146], w)
    q, qs = torch_ops.quantize_rows(big[:, 50:146])
    assert torch.equal(q, hip.quantize_rows(x)[0])


def test_graph_replays_match_eager(hip):
    """Two graphs of the whole path, each with its own buffers, replayed in turn with eager work between."""
    def calls(seed):
        x, res, w = inputs(50, 300, "f16", True, seed=seed)
        t = operands(50, 300, 300, "f16", True, True, seed=seed)
        ws = torch.empty(hip.rms_norm_bwd_workspace(x), dtype=torch.uint8, device="cuda")

        def run():
            y, total, rstd = hip.rms_norm(x, w, res, want_rstd=True)
            ds, dw = hip.rms_norm_bwd(total, w, rstd, y, x, workspace=ws)
            q, qs, _ = hip.rms_norm_q8(x, w, res)
            h = hip.q8_projection(q, qs, t["wq"], t["ws"], t["b"], t["residual"])
            hq, hs = hip.quantize_rows(h, 2)
            return [y, total, rstd, ds, dw, q, qs, h, hq, hs, hip.dequantize_rows(hq, hs)]
        return run

    runs = [calls(1), calls(2)]
    eager = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    graphs, results = [], []
    for r in runs:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            r()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(r())
        graphs.append(g)
    for replay in range(4):
        for out in results:
            for t in out:
                t.fill_(3)
        runs[replay % 2]()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, want in zip(results, eager):
            for i, (a, b) in enumerate(zip(out, want)):
                assert torch.equal(a, b), (replay, i)


def test_differentiated_call_is_refused_under_capture(hip):
    x, _, w = inputs(4, 64, "f16", False)
    x.requires_grad_()
    static = x.detach().clone()
    torch_ops.rms_norm(static, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(hip.InvalidArgument, match="cannot be captured"):
            torch_ops.rms_norm(x, w)
        y = torch_ops.rms_norm(static, w)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, torch_ops.rms_norm(static, w))


def test_backward_of_an_eager_forward_is_refused_under_capture(hip):
    """The backward node runs on its forward's stream; captured there, it raises before any gradient reaches a leaf."""
    x, _, w = inputs(4, 64, "f16", False)
    dy = torch.ones_like(x)
    x.requires_grad_()
    static = x.detach().clone()
    torch_ops.rms_norm(static, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = torch_ops.rms_norm(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        with pytest.raises(hip.InvalidArgument, match="cannot be captured"):
            y.backward(dy)
        captured = torch_ops.rms_norm(static, w)
    assert x.grad is None
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, torch_ops.rms_norm(static, w))


def cancelling(m, k, n, turns):
    """Rows and weights of [m, k] and [n, k] whose products add up to millions above 2^24, all of them again below zero, and
    the product of two small odd numbers, which 16 bits hold. The two lie in k's two halves, or (turns) 64 inputs by
    64 in turn, so that one of them is all that some parts of a divided sum have."""
    rng = np.random.default_rng(m + k + n)
    h = k // 2
    row, chan = 2 * rng.integers(0, 8, m) + 1, (2 * rng.integers(0, 8, n) + 1) * rng.choice((-1, 1), n)
    q = torch.from_numpy(rng.integers(64, 128, (m, h)).astype(np.int8)).cuda()
    q[:, -1] = torch.from_numpy(row.astype(np.int8))
    w = torch.from_numpy(rng.integers(64, 128, (n, h)).astype(np.int8)).cuda()
    w[:, -1] = 0
    less = -w
    less[:, -1] = torch.from_numpy(chan.astype(np.int8))

    def join(a, b):
        if turns:
            return torch.stack([a.view(len(a), -1, 64), b.view(len(a), -1, 64)], 2).reshape(len(a), k)
        return torch.cat([a, b], 1)
    return join(q, q).contiguous(), join(w, less).contiguous(), torch.from_numpy(np.outer(row, chan)).cuda()


@pytest.mark.parametrize("turns", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 16384, 70), (4, 130944, 70), (9, 16384, 70), (16, 130944, 70), (20, 16384, 70), (33, 16384, 130),
                                   (64, 130944, 70), (20, 16384, 4200), (40, 16384, 4200), (60, 16384, 4200),
                                   (70, 16384, 70), (300, 130944, 70), (700, 16384, 1100), (1531, 16384, 2050),
                                   (2304, 16384, 4608)])
def test_sums_that_cancel_are_exact(hip, m, k, n, turns):
    """A sum in floating point, or one that is rounded to it before its parts are joined, is off by a few here."""
    q, w, want = cancelling(m, k, n, turns)
    ones = lambda r: torch.ones(r, device="cuda")  # noqa: E731
    wq = layouts.q8_blocked(w)
    for kind in ("f16", "bf16"):
        out = hip.q8_projection(q, ones(m), wq, ones(n), dtype=DT[kind])
        assert torch.equal(out, want.to(DT[kind]))
