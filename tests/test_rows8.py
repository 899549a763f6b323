"""The RMS norm and the 8-bit path on the CPU: the float64 oracle against independent statements, the
weights' layout element by element, and every refusal of the entry points, none of which touches a
device. No kernel is launched here."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import hip as H
from colabfold_legacy_kernels import layouts, torch_ops
from oracle import rows8 as orr
from test_capi import F16, F32, S32, buf, lib  # noqa: F401

S8, BF16 = 2, 16


# ---- the oracle ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind,dtype", [("f16", torch.float16), ("bf16", torch.bfloat16)])
def test_round16_is_torchs(kind, dtype):
    rng = np.random.default_rng(0)
    v = (rng.standard_normal(4000) * 2.0 ** rng.integers(-30, 20, 4000)).astype(np.float32)
    v[:4] = [0.0, 1e-7, 65519.0, 65520.0]
    want = torch.from_numpy(v).to(dtype).double().numpy()
    assert np.array_equal(orr.round16(v, kind), want)


@pytest.mark.parametrize("with_dsum", [False, True])
def test_gradients_against_differences(with_dsum):
    """d/ds and d/dw of sum(y dy) + sum(s dsum) by central differences of the forward: with steps of 1e-5
    their error is about 1e-10 from the third derivative and 1e-16 / 1e-5 from the subtraction."""
    rng = np.random.default_rng(1)
    s, w, dy, dsum = (rng.standard_normal(n) for n in ((3, 7), 7, (3, 7), (3, 7)))
    eps, h = 1e-3, 1e-5

    def loss(s, w):
        return (orr.rms_norm(s, w, eps)[0] * dy).sum() + ((s * dsum).sum() if with_dsum else 0.0)

    ds, dw = orr.rms_norm_bwd(s, w, dy, dsum if with_dsum else None, eps)
    for i in range(3):
        for j in range(7):
            d = np.zeros((3, 7))
            d[i, j] = h
            assert abs((loss(s + d, w) - loss(s - d, w)) / (2 * h) - ds[i, j]) < 1e-8
    for j in range(7):
        d = np.zeros(7)
        d[j] = h
        assert abs((loss(s, w + d) - loss(s, w - d)) / (2 * h) - dw[j]) < 1e-8


def test_quotients_and_project():
    t = np.array([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0], [1.0, np.inf, 0.0], [np.nan, 1.0, 2.0], [1e-37, 0.0, -1e-38]])
    q, scale = orr.quotients(t)
    assert np.allclose(q[0], [63.5, -127.0, 31.75]) and scale[0] == 2.0 / 127
    assert (q[1:] == 0).all() and scale[1] == 0 and np.isnan(scale[2]) and np.isnan(scale[3]) and scale[4] == 0
    rng = np.random.default_rng(2)
    a, b = rng.integers(-127, 128, (3, 5)), rng.integers(-127, 128, (4, 5))
    out, _ = orr.project(a, [1, 2, 3], b, [1, 1, 2, 1], [0.5] * 4, np.ones((3, 4)))
    for i in range(3):
        for j in range(4):
            s = sum(int(a[i, k]) * int(b[j, k]) for k in range(5))
            assert out[i, j] == s * [1, 2, 3][i] * [1, 1, 2, 1][j] + 1.5


# ---- layouts ------------------------------------------------------------------------------

@pytest.mark.parametrize("lib_", ("numpy", "torch"))
@pytest.mark.parametrize("n,kp", [(1, 64), (64, 128), (130, 192)])
def test_q8_blocked(lib_, n, kp):
    q = np.random.default_rng(n).integers(-127, 128, (n, kp)).astype(np.int8)
    arg = torch.from_numpy(q) if lib_ == "torch" else q
    wq = layouts.q8_blocked(arg)
    assert tuple(wq.shape) == (-(-n // 64), kp // 64, 4, 4, 16, 16)
    for ch in range(0, wq.shape[0] * 64):
        for k in (0, 15, 16, kp - 1, (7 * ch) % kp):
            r, i = ch % 64, k % 64
            got = int(wq[ch // 64, k // 64, (r // 4) % 4, i // 16, 4 * (r // 16) + r % 4, i % 16])
            assert got == (int(q[ch, k]) if ch < n else 0)
    assert np.array_equal(np.asarray(layouts.q8_unblocked(wq, n)), q)


def test_q8_blocked_refuses_other_widths():
    with pytest.raises(ValueError, match="multiple of 64"):
        layouts.q8_blocked(torch.zeros((4, 65), dtype=torch.int8))


# ---- refusals of the C entry points ----------------------------------------------------------

def refs(args):
    return [a[0] for a in args]


def norm_args(m=6, c=40, act=F16, **other):
    d = dict(x=buf(act, m, c), residual=buf(act, m, c, data=0x200000), scale=buf(F32, c), sum=buf(act, m, c, data=0x300000),
             out=buf(act, m, c, data=0x400000), rstd=buf(F32, m))
    d.update(other)
    return refs(d.values())


@pytest.mark.parametrize("other,eps,message", [
    (dict(x=buf(F16, 6)), 1e-5, r"x must be \[M,C\]"),
    (dict(x=buf(F32, 6, 40)), 1e-5, "must be F16, got F32"),
    (dict(residual=buf(BF16, 6, 40)), 1e-5, "must be F16, got BF16"),
    (dict(residual=buf(F16, 6, 41)), 1e-5, "residual and sum must be like x"),
    (dict(sum=buf(F16, 5, 40)), 1e-5, "residual and sum must be like x"),
    (dict(scale=buf(F32, 41)), 1e-5, r"scale must be \[C\]"),
    (dict(out=buf(F16, 6, 39)), 1e-5, "out must be like x"),
    (dict(out=buf(F16, 6, 40, data=0x300000)), 1e-5, "must not be the same buffer"),
    (dict(rstd=buf(F32, 7)), 1e-5, r"rstd must be \[M\]"),
    (dict(), -1.0, "eps must not be negative"),
    (dict(), float("nan"), "eps must not be negative"),
])
def test_rms_norm_refusals(lib, other, eps, message):
    import re
    st = lib.clk_rms_norm(None, *norm_args(**other), eps, 1, 1)
    assert st == 3 and re.search(message, lib.clk_last_error().decode()), lib.clk_last_error()


def test_rms_norm_empty(lib):
    assert lib.clk_rms_norm(None, *norm_args(m=0), 1e-5, 1, 1) == 0
    assert lib.clk_rms_norm(None, *norm_args(c=0), 1e-5, 1, 1) == 3
    assert "C must be at least 1" in lib.clk_last_error().decode()


def test_rms_norm_q8_refusals(lib):
    a = dict(x=buf(F16, 6, 40), residual=buf(F16, 1), scale=buf(F32, 40), sum=buf(F16, 1), q=buf(S8, 6, 64), qs=buf(F32, 6))
    for other, message in ((dict(q=buf(S8, 6, 40)), "q must be [M,Kp]"), (dict(q=buf(F16, 6, 64)), "must be S8"),
                           (dict(qs=buf(F32, 5)), "q_scale must be [M]"),
                           (dict(q=buf(S8, 6, 64, data=0x100008)), "16-byte aligned")):
        assert lib.clk_rms_norm_q8(None, *refs({**a, **other}.values()), 1e-5, 0) == 3
        assert message in lib.clk_last_error().decode()


def test_rms_norm_bwd_refusals(lib):
    m, c = 6, 40
    a = dict(s=buf(F16, m, c), scale=buf(F32, c), rstd=buf(F32, m), dout=buf(F16, m, c), dsum=buf(F16, m, c),
             ds=buf(F16, m, c), dscale=buf(F32, c))
    need = lib.clk_rms_norm_bwd_workspace_size(a["s"][0])
    assert need >= 4 * c and need % 256 == 0
    for other, message in ((dict(scale=buf(F32, c + 1)), "scale and dscale must be [C]"),
                           (dict(dscale=buf(F32, c - 1)), "scale and dscale must be [C]"),
                           (dict(rstd=buf(F32, m + 1)), "rstd must be [M]"),
                           (dict(dout=buf(F16, m, c + 1)), "must be like s"), (dict(dsum=buf(F16, 1)), "must be like s"),
                           (dict(ds=buf(BF16, m, c)), "must be F16")):
        assert lib.clk_rms_norm_bwd(None, *refs({**a, **other}.values()), 1, 0x100000, need) == 3
        assert message in lib.clk_last_error().decode()
    for ws, size, message in ((0x100000, need - 1, "workspace of"), (None, need, "workspace of"),
                              (0x100010, need, "256-byte aligned")):
        assert lib.clk_rms_norm_bwd(None, *refs(a.values()), 1, ws, size) == 3
        assert message in lib.clk_last_error().decode()
    assert lib.clk_rms_norm_bwd_workspace_size(buf(F16, 0, c)[0]) == 0
    assert lib.clk_rms_norm_bwd_workspace_size(None) == 0


def test_rms_norm_bwd_of_the_longest_rows(lib):
    """Rows past 2^27 values would need more threads than a launch takes."""
    for m, c in ((1, 2 ** 27), (1, 2 ** 27 + 1), (5, 2 ** 29)):
        s = buf(F16, m, c)
        need = lib.clk_rms_norm_bwd_workspace_size(s[0])
        assert (need == 0) == (c > 2 ** 27)
        if c > 2 ** 27:
            st = lib.clk_rms_norm_bwd(None, *refs([s, buf(F32, c), buf(F32, m), s, s, s, buf(F32, c)]), 0, 0x100000, 2 ** 40)
            assert st == 3 and "rms_norm_bwd: too large" in lib.clk_last_error().decode()


def test_quantize_rows_refusals(lib):
    for x, q, s, act, message in (
            (buf(F16, 6, 40), buf(S8, 6, 64), buf(F32, 6), 3, "activation is 0 (none)"),
            (buf(F16, 6, 40), buf(S8, 6, 64), buf(F32, 6), -1, "activation is 0 (none)"),
            (buf(S32, 6, 40), buf(S8, 6, 64), buf(F32, 6), 0, "must be F16, got S32"),
            (buf(F16, 6, 41), buf(S8, 6, 64), buf(F32, 6), 2, "must be [M,2K]"),
            (buf(F16, 6, 40), buf(S8, 6, 40), buf(F32, 6), 0, "q must be [M,Kp]"),
            (buf(F16, 6, 160), buf(S8, 6, 192), buf(F32, 6), 2, "q must be [M,Kp]"),
            (buf(F16, 6, 40), buf(S8, 6, 64), buf(F32, 7), 0, "q_scale must be [M]"),
            (buf(F16, 6, 0), buf(S8, 6, 0), buf(F32, 6), 0, "C must be at least 1"),
            (buf(F16, 6), buf(S8, 6, 64), buf(F32, 6), 0, "must be [M,C]"),
            (buf(F16, 6, 40), buf(S8, 6, 64, data=0x100004), buf(F32, 6), 0, "16-byte aligned")):
        assert lib.clk_quantize_rows(None, x[0], q[0], s[0], act) == 3
        assert message in lib.clk_last_error().decode(), message
    assert lib.clk_quantize_rows(None, buf(F16, 0, 40)[0], buf(S8, 0, 64)[0], buf(F32, 0)[0], 0) == 0


def test_dequantize_rows_refusals(lib):
    for q, s, out, message in ((buf(S8, 6, 64), buf(F32, 6), buf(F16, 6, 65), "q must be [M,Kp]"),
                               (buf(S8, 6, 64), buf(F32, 5), buf(F16, 6, 64), "q_scale must be [M]"),
                               (buf(S8, 6, 64), buf(F32, 6), buf(S32, 6, 64), "must be F16, got S32"),
                               (buf(F16, 6, 64), buf(F32, 6), buf(F16, 6, 64), "must be S8")):
        assert lib.clk_dequantize_rows(None, q[0], s[0], out[0]) == 3
        assert message in lib.clk_last_error().decode()


def test_q8_projection_refusals(lib):
    m, kp, n = 6, 128, 100
    a = dict(q=buf(S8, m, kp), qs=buf(F32, m), wq=buf(S8, 2, 2, 4, 4, 16, 16), ws=buf(F32, n), b=buf(F32, n),
             residual=buf(F16, m, n), out=buf(F16, m, n))
    for other, message in ((dict(q=buf(S8, m, 96)), "Kp must be a multiple of 64"),
                           (dict(q=buf(S8, m, 131072)), "from 64 to 131008"),
                           (dict(q=buf(S8, m, 0)), "Kp must be a multiple of 64"),
                           (dict(q=buf(S8, m + 1, kp)), "q must be [M,Kp] and out [M,N]"),
                           (dict(q=buf(F16, m, kp)), "must be S8"),
                           (dict(qs=buf(F32, m - 1)), "q_scale must be [M]"),
                           (dict(wq=buf(S8, 1, 2, 4, 4, 16, 16)), "wq must be"),
                           (dict(wq=buf(S8, 2, 1, 4, 4, 16, 16)), "wq must be"),
                           (dict(wq=buf(S8, n, kp)), "wq must be"),
                           (dict(ws=buf(F32, n + 1)), "w_scale and b must be [N]"),
                           (dict(b=buf(F32, 1)), "w_scale and b must be [N]"),
                           (dict(b=buf(F16, n)), "must be F32"),
                           (dict(residual=buf(F16, 1)), "residual must be like out"),
                           (dict(residual=buf(BF16, m, n)), "must be F16, got BF16"),
                           (dict(out=buf(F32, m, n)), "must be F16"),
                           (dict(wq=buf(S8, 2, 2, 4, 4, 16, 16, data=0x100008)), "16-byte aligned")):
        st = lib.clk_q8_projection(None, *refs({**a, **other}.values()), 1, 1)
        assert st == 3 and message in lib.clk_last_error().decode(), (message, lib.clk_last_error())
    for rows, n2 in ((1, 1 << 28), (1 << 21, 1 << 16), (1 << 31, n)):  # more than a launch holds
        big = dict(a, q=buf(S8, rows, kp), qs=buf(F32, rows), wq=buf(S8, -(-n2 // 64), 2, 4, 4, 16, 16), ws=buf(F32, n2),
                   b=buf(F32, n2), residual=buf(F16, rows, n2), out=buf(F16, rows, n2))
        assert lib.clk_q8_projection(None, *refs(big.values()), 1, 1) == 3
        assert "too large" in lib.clk_last_error().decode()
    empty = dict(a, q=buf(S8, 0, kp), qs=buf(F32, 0), residual=buf(F16, 0, n), out=buf(F16, 0, n))
    assert lib.clk_q8_projection(None, *refs(empty.values()), 1, 1) == 0
    none = dict(a, wq=buf(S8, 0, 2, 4, 4, 16, 16), ws=buf(F32, 0), b=buf(F32, 0), residual=buf(F16, m, 0), out=buf(F16, m, 0))
    assert lib.clk_q8_projection(None, *refs(none.values()), 1, 1) == 0


# ---- refusals of the Python entry points -------------------------------------------------------

def test_cpu_tensors_are_refused():
    x, w = torch.zeros((4, 64), dtype=torch.float16), torch.ones(64)
    q, s = torch.zeros((4, 64), dtype=torch.int8), torch.ones(4)
    wq, ws = layouts.q8_blocked(torch.zeros((8, 64), dtype=torch.int8)), torch.ones(8)
    for call in (lambda: H.rms_norm(x, w), lambda: H.rms_norm_q8(x, w), lambda: H.quantize_rows(x),
                 lambda: H.dequantize_rows(q, s), lambda: H.q8_projection(q, s, wq, ws),
                 lambda: H.rms_norm_bwd(x, w, s, x), lambda: torch_ops.rms_norm(x, w),
                 lambda: torch_ops.q8_projection(q, s, (wq, ws))):
        with pytest.raises(H.InvalidArgument, match="must be on one GPU"):
            call()


def test_shapes_are_refused():
    x = torch.zeros((2, 4, 64), dtype=torch.float16)
    for call in (lambda: H.rms_norm(x, x), lambda: H.rms_norm_q8(x, x), lambda: H.quantize_rows(x),
                 lambda: H.dequantize_rows(x, x), lambda: H.q8_projection(x, x, x, x)):
        with pytest.raises(H.InvalidArgument, match="expected a matrix"):
            call()
    with pytest.raises(H.InvalidArgument, match="residual must be like x"):
        torch_ops.rms_norm(x, torch.ones(64), x[:1])
    with pytest.raises(H.InvalidArgument, match="activation is None"):
        torch_ops.quantize_rows(x, "gelu")


def test_padded_k():
    assert [H.padded_k(k) for k in (1, 63, 64, 65, 128, 8191)] == [64, 64, 64, 128, 128, 8192]


# ---- torch_ops.rms_norm under autograd, with torch operations in the kernels' place --------------

@pytest.fixture
def kernels_on_cpu(monkeypatch):
    """hip.rms_norm and hip.rms_norm_bwd by torch operations, with the entry points' own shapes."""
    def forward(x, scale, residual=None, eps=1e-5, want_rstd=False, out=None, sum_out=None, rstd=None):
        assert x.dim() == 2 and (out is None or out.shape == x.shape)
        s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
        r = 1 / torch.sqrt(s.float().square().mean(1) + eps)
        y = (s.float() * r[:, None] * scale.reshape(-1)).to(x.dtype)
        y = y if out is None else out.copy_(y)
        if residual is not None and sum_out is not None:
            s = sum_out.copy_(s)
        return y, None if residual is None else s, r if want_rstd else None

    def backward(s, scale, rstd, dout, dsum=None, workspace=None, grads=None):
        assert s.dim() == 2 and dout.shape == s.shape and (dsum is None or dsum.shape == s.shape)
        g, xh = dout.float() * scale.reshape(-1), s.float() * rstd[:, None]
        ds = rstd[:, None] * (g - xh * (g * xh).mean(1, keepdim=True)) + (0 if dsum is None else dsum.float())
        ds, dscale = ds.to(s.dtype), (dout.float() * xh).sum(0).reshape(scale.shape)
        return (ds, dscale) if grads is None else (grads[0].copy_(ds), grads[1].copy_(dscale))

    monkeypatch.setattr(H, "rms_norm", forward)
    monkeypatch.setattr(H, "rms_norm_bwd", backward)


def norm_leaves(shape, dtype=torch.float16):
    gen = torch.Generator().manual_seed(3)
    x, res = (torch.randn(shape, generator=gen).to(dtype).requires_grad_() for _ in range(2))
    w = (1 + 0.2 * torch.randn(shape[-1], generator=gen)).requires_grad_()
    return x, res, w, torch.randn(shape, generator=gen).to(dtype), torch.randn(shape, generator=gen).to(dtype)


@pytest.mark.parametrize("shape", [(64,), (6, 64), (2, 3, 64), (2, 3, 2, 8), (1, 1, 64), (0, 3, 64)])
@pytest.mark.parametrize("used", ["both", "norm", "sum"])
def test_gradients_accumulate_leaf_by_leaf(kernels_on_cpu, shape, used):
    """Two passes into both leaves: twice one pass's gradient in each, in memory of its own."""
    x, res, w, dy, ds = norm_leaves(shape)

    def one_pass():
        y, total = torch_ops.rms_norm(x, w, res)
        assert y.shape == x.shape and total.shape == x.shape
        outs, grads = {"both": ((y, total), (dy, ds)), "norm": ((y,), (dy,)), "sum": ((total,), (ds,))}[used]
        torch.autograd.backward(outs, grads)

    given = dy.clone(), ds.clone()
    one_pass()
    once = x.grad.clone(), res.grad.clone()
    assert torch.equal(*once) and x.grad.shape == x.shape
    one_pass()
    for leaf, g in zip((x, res), once):
        assert torch.equal(leaf.grad, 2 * g)
    if x.numel():
        owners = [t.data_ptr() for t in (x.grad, res.grad, dy, ds)]
        assert len(set(owners)) == 4
    x.grad.zero_()
    assert torch.equal(res.grad, 2 * once[1]) and torch.equal(dy, given[0]) and torch.equal(ds, given[1])


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64)])
def test_results_of_a_differentiated_norm_are_plain_tensors(kernels_on_cpu, shape):
    """The results may be changed in place as any operation's, what the gradient needs of them is checked,
    and strided inputs get gradients of their own."""
    x, res, w, dy, ds = norm_leaves(shape)
    y, total = torch_ops.rms_norm(x, w, res)
    y.mul_(2)
    y.backward(dy)
    want = x.grad.clone()
    x.grad = None
    torch_ops.rms_norm(x, w, res)[0].backward(2 * dy)
    assert torch.equal(want, x.grad)
    y, total = torch_ops.rms_norm(x, w, res)
    total.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    xt, rt = (t.detach().transpose(0, -1).contiguous().transpose(0, -1).requires_grad_() for t in (x, res))
    assert not xt.is_contiguous()
    torch_ops.rms_norm(xt, w, rt)[0].backward(2 * dy)
    assert torch.equal(xt.grad, want) and torch.equal(rt.grad, want)


@pytest.mark.parametrize("which", ["x", "scale", "residual"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(kernels_on_cpu, which, grad):
    """A dual tensor has no requires_grad of its own; its tangent must not vanish. Without a tangent, a call
    inside a dual level is an ordinary one."""
    from torch.autograd import forward_ad
    x, res, w, _, _ = (t.detach() for t in norm_leaves((2, 3, 64)))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        want = torch_ops.rms_norm(x, w, res)
        args = dict(x=x, scale=w, residual=res)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="jvp|forward"):
            torch_ops.rms_norm(**args)
    assert all(torch.equal(a, b) for a, b in zip(torch_ops.rms_norm(x, w, res), want))


def test_backward_is_refused_under_capture(kernels_on_cpu, monkeypatch):
    """An eager forward whose backward runs into a capture, for each result that may be used; the same graph's
    backward outside of the capture still runs."""
    x, res, w, dy, ds = norm_leaves((2, 3, 64))
    y, total = torch_ops.rms_norm(x, w, res)
    alone = torch_ops.rms_norm(x, w)
    with monkeypatch.context() as m:
        m.setattr(torch_ops, "_capturing", lambda t: True)
        for outs, grads in (((y, total), (dy, ds)), ((y,), (dy,)), ((total,), (ds,)), ((alone,), (dy,))):
            with pytest.raises(H.InvalidArgument, match="cannot be captured"):
                torch.autograd.backward(outs, grads, retain_graph=True)
        with pytest.raises(H.InvalidArgument, match="cannot be captured"):
            torch_ops.rms_norm(x, w, res)
        torch_ops.rms_norm(x.detach(), w.detach())
    assert x.grad is None and res.grad is None and w.grad is None
    torch.autograd.backward((y, total), (dy, ds))
    assert x.grad is not None


def test_residuals_of_another_shape_are_refused():
    """Also where they hold as many values: [3, 2, 64] is not added to [2, 3, 64] by position in memory. Rows [M, C]
    pass to the entry point, which checks them."""
    x, w = torch.zeros((2, 3, 64), dtype=torch.float16), torch.ones(64)
    q, s = torch.zeros((2, 3, 64), dtype=torch.int8), torch.ones((2, 3))
    weights = layouts.q8_blocked(torch.zeros((8, 64), dtype=torch.int8)), torch.ones(8)
    for other in ((3, 2, 64), (1, 6, 64), (2, 3, 32), (2, 3, 65)):
        with pytest.raises(H.InvalidArgument, match="residual must be like x"):
            torch_ops.rms_norm_q8(x, w, torch.zeros(other, dtype=torch.float16))
        with pytest.raises(H.InvalidArgument, match="residual must be like x"):
            torch_ops.q8_transition(x, w, weights, None, weights, None, torch.zeros(other, dtype=torch.float16))
    for other in ((3, 2, 8), (1, 6, 8), (2, 3, 9), (2, 3, 64)):
        with pytest.raises(H.InvalidArgument, match="residual must be like the result"):
            torch_ops.q8_projection(q, s, weights, residual=torch.zeros(other, dtype=torch.float16))


def test_nearest():
    """Against Python's fractions: values on and next to halves, one of the tiniest rows, one too tiny, zeros."""
    from fractions import Fraction
    rng = np.random.default_rng(5)
    a = (rng.uniform(1, 2, (40, 1)) * 2.0 ** rng.integers(-118, 120, (40, 1))).astype(np.float32)
    t = (a.astype(np.float64) * (2 * rng.integers(-127, 127, (40, 50)) + 1) / 254).astype(np.float32)
    t = (t.view(np.int32) + rng.integers(-2, 3, t.shape).astype(np.int32)).view(np.float32)
    t[:, 0], t[:, 1], t[:, 2] = a[:, 0], a[:, 0] / 2, -a[:, 0] / 2
    t[3] *= np.float32(2.0 ** -119) / a[3, 0]
    t[4] *= np.float32(2.0 ** -121) / a[4, 0]
    t[5] = 0
    got = orr.nearest(t)
    for row, q in zip(t, got):
        top = max(Fraction(abs(float(v))) for v in row)
        for v, n in zip(row, q):
            assert n == (round(127 * Fraction(float(v)) / top) if top >= Fraction(2) ** -119 else 0)


def test_inline_assembly_names_the_m0_that_it_writes():
    """m0 is the compiler's too (it holds the LDS address of the direct-to-LDS builtin, and lane indices): a block that
    writes it has to say so."""
    import glob
    import os
    import re
    import build as pkg_build
    writers = 0
    for path in glob.glob(os.path.join(pkg_build.CSRC, "*.h*")):
        for text in re.findall(r"asm(?:\s+volatile)?\s*\((.*?)\);", open(path).read(), re.S):
            code, _, rest = text.partition("::") if "::" in text else text.partition(" :")
            if re.search(r"\bs_\w+ m0\b", code):
                writers += 1
                assert '"m0"' in rest, os.path.basename(path)
    assert writers == 1
