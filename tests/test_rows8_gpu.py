"""RMS norm and 8-bit rows on gfx950 against the float64 oracle, through the C ABI.

Tolerances, counted from the roundings (u: half a step of the result's type, 2^-11 or 2^-8; E = 2^-24):
  y, ds    one rounding to 16 bits, after fp32 operations of relative error E each. A row's sums run over
           at most C / 256 + 32 terms in sequence (a lane's share, then the lanes), so a sum of same-sign
           terms is off by at most (C / 256 + 32) E, a mixed one by that times its terms' magnitudes.
           fp16 results below 2^-14 round to steps of 2^-24: 2^-25 absolute.
  q        the nearest integer to 127 t / a: off by half, plus four roundings of a value up to 127.
  scales   a r / 127: a's rounding, r's sums, two operations.
"""
import numpy as np
import pytest
import torch

from oracle import rows8 as orr

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY16 = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def host(t):
    return t.detach().double().cpu().numpy()


def seq(c):
    return c / 256 + 32


def make(rng, kind, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(DT[kind]).cuda()


def inputs(m, c, kind, residual, seed=0):
    rng = np.random.default_rng(seed + 1000 * m + c)
    spread = np.exp(0.5 * rng.standard_normal(c)).astype(np.float32)
    x = torch.from_numpy(rng.standard_normal((m, c)).astype(np.float32) * spread).to(DT[kind]).cuda()
    res = make(rng, kind, m, c) if residual else None
    w = torch.from_numpy((1 + 0.2 * rng.standard_normal(c)).astype(np.float32)).cuda()
    return x, res, w


def check_sum(got, x, res, kind):
    want = host(x) + host(res)
    assert (np.abs(host(got) - want) <= (U[kind] + E) * np.abs(want) + TINY16[kind]).all()


def check_norm(y, rstd, s, w, eps, kind):
    want, r = orr.rms_norm(s, host(w), eps)
    d = (seq(s.shape[1]) + 8) * E
    assert (np.abs(host(y) - want) <= (U[kind] + d) * np.abs(want) + TINY16[kind]).all()
    if rstd is not None:
        assert (np.abs(host(rstd) - r) <= d * r).all()


def check_q8(q, q_scale, t, r, slack=0.0):
    """8-bit rows of t, whose scale carries r; slack: t's own relative error."""
    m, k = t.shape
    got = q.cpu().numpy().astype(np.float64)
    assert (got[:, k:] == 0).all() and q.shape[1] == (k + 63) // 64 * 64
    quot, scale = orr.quotients(t)
    assert (np.abs(got[:, :k] - quot) <= 0.5 + 127 * (4 * E + 2 * slack)).all()
    want = scale * r
    assert (np.abs(host(q_scale) - want) <= (4 * E + (seq(k) + 8) * E + slack) * want).all()


# every route over the width: one row a lane group, a wave, a workgroup of each size, and longer rows
WIDTHS = [1, 7, 8, 13, 63, 64, 65, 100, 128, 129, 200, 256, 300, 512, 513, 640, 1000, 1024, 1025, 1536, 2048, 2050, 2056,
          4096, 5120, 8192, 8200, 16384, 16392, 20001, 33000, 70001]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("c", WIDTHS)
def test_rms_norm_widths(hip, c, kind):
    for m, residual in ((1, True), (5, False), (37 if c < 9000 else 3, True)):
        x, res, w = inputs(m, c, kind, residual)
        y, total, rstd = hip.rms_norm(x, w, res, 1e-5, want_rstd=True)
        assert (total is None) == (res is None)
        if residual:
            check_sum(total, x, res, kind)
        check_norm(y, rstd, host(x if total is None else total), w, 1e-5, kind)
        q, qs, total8 = hip.rms_norm_q8(x, w, res, 1e-5)
        if residual:
            assert torch.equal(total8, total)
        s = host(x if total is None else total)
        check_q8(q, qs, s * host(w), orr.rms_norm(s, host(w), 1e-5)[1])


@pytest.mark.parametrize("m", [1, 2, 3, 4, 15, 16, 17, 64, 255, 1024, 2049, 9000])
@pytest.mark.parametrize("c", [64, 136, 1024, 1100])
def test_rms_norm_rows(hip, m, c):
    x, res, w = inputs(m, c, "f16", True)
    y, total, rstd = hip.rms_norm(x, w, res, 1e-6, want_rstd=True)
    check_sum(total, x, res, "f16")
    check_norm(y, rstd, host(total), w, 1e-6, "f16")
    q, qs, _ = hip.rms_norm_q8(x, w, res, 1e-6)
    check_q8(q, qs, host(total) * host(w), orr.rms_norm(host(total), host(w), 1e-6)[1])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("c", WIDTHS)
def test_rms_norm_bwd_widths(hip, c, kind):
    for m, with_dsum in ((1, True), (6, False), (45 if c < 9000 else 4, True)):
        check_bwd(hip, m, c, kind, with_dsum)


def check_bwd(hip, m, c, kind, with_dsum):
    s, _, w = inputs(m, c, kind, False, seed=7)
    rng = np.random.default_rng(m + c)
    dy = make(rng, kind, m, c)
    dsum = make(rng, kind, m, c) if with_dsum else None
    _, _, rstd = hip.rms_norm(s, w, None, 1e-5, want_rstd=True)
    ds, dw = hip.rms_norm_bwd(s, w, rstd, dy, dsum)
    want, wantw = orr.rms_norm_bwd(host(s), host(w), host(dy), None if dsum is None else host(dsum), 1e-5)
    r = orr.rms_norm(host(s), host(w), 1e-5)[1][:, None]
    xh, g = host(s) * r, host(dy) * host(w)
    # r's own error reaches xh and the product; the dot's terms are summed as counted above
    n = seq(c) + 16
    terms = r * (np.abs(g) + np.abs(xh) * np.abs(g * xh).mean(1, keepdims=True)) + (0 if dsum is None else np.abs(host(dsum)))
    assert (np.abs(host(ds) - want) <= U[kind] * np.abs(want) + TINY16[kind] + 3 * n * E * terms).all()
    assert (np.abs(host(dw) - wantw) <= (m + n) * E * np.abs(host(dy) * xh).sum(0)).all()
    again = hip.rms_norm_bwd(s, w, rstd, dy, dsum)
    assert torch.equal(again[0], ds) and torch.equal(again[1], dw)


@pytest.mark.parametrize("m,c", [(511, 64), (513, 128), (1531, 1025), (4100, 256), (2100, 2048), (1100, 4096), (700, 8192),
                                 (20000, 64), (530, 33000)])
def test_rms_norm_bwd_rows(hip, m, c):
    check_bwd(hip, m, c, "bf16", True)


def test_rms_norm_bwd_of_no_rows(hip):
    s, w = torch.empty((0, 96), dtype=torch.float16, device="cuda"), torch.ones(96, device="cuda")
    dw = torch.full((96,), 5.0, device="cuda")
    hip.rms_norm_bwd(s, w, torch.empty(0, device="cuda"), s, grads=(torch.empty_like(s), dw))
    assert (dw == 0).all()


@pytest.mark.parametrize("c", [64, 96, 700, 3000, 9000, 40000])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_special_rows(hip, c, kind):
    """Zeros, infinities, NaN, the type's largest values, and (bf16) values whose squares leave fp32: each row
    goes by itself."""
    x, _, w = inputs(8, c, kind, False)
    big = float(torch.finfo(DT[kind]).max)
    x[1] = 0
    x[2, c // 2] = float("inf")
    x[3, c - 1] = float("nan")
    x[4] = torch.where(x[4] > 0, big, -big).to(x.dtype)
    x[5] = x[5] * (1e25 if kind == "bf16" else 1.0)
    x[6] = x[6] * 1e-30 if kind == "bf16" else x[6] * 2.0 ** -12
    y, _, rstd = hip.rms_norm(x, w, None, 1e-5, want_rstd=True)
    q, qs, _ = hip.rms_norm_q8(x, w, None, 1e-5)
    ok = [0, 1, 4, 5, 6, 7]
    check_norm(y[ok], rstd[ok], host(x)[ok], w, 1e-5, kind)
    check_q8(q[ok], qs[ok], (host(x) * host(w))[ok], orr.rms_norm(host(x)[ok], host(w), 1e-5)[1])
    assert (y[1] == 0).all() and (q[1] == 0).all() and qs[1] == 0
    # an infinity: its own place is NaN (inf times 0), the others are 0; a NaN: the row is NaN
    assert torch.isnan(y[2, c // 2]) and (y[2, :c // 2] == 0).all() and rstd[2] == 0
    assert torch.isnan(y[3]).all() and torch.isnan(rstd[3])
    for row in (2, 3):
        assert (q[row] == 0).all() and torch.isnan(qs[row])
    # q8: a scale (or weight) that is not finite makes its rows NaN, whatever x holds there
    w2 = w.clone()
    w2[c // 3] = float("inf")
    q, qs, _ = hip.rms_norm_q8(x, w2, None, 1e-5)
    assert (q == 0).all() and torch.isnan(qs).all()


def test_eps_zero_and_large(hip):
    x, _, w = inputs(9, 128, "f16", False)
    x[3] = 0
    y, _, _ = hip.rms_norm(x, w, None, 0.0)
    assert torch.isnan(y[3]).all()  # 0 / 0, as the formula has it
    live = [0, 1, 2, 4, 5, 6, 7, 8]
    check_norm(y[live], None, host(x)[live], w, 0.0, "f16")
    y, _, rstd = hip.rms_norm(x, w, None, 100.0, want_rstd=True)
    check_norm(y, rstd, host(x), w, 100.0, "f16")


@pytest.mark.parametrize("std,eps", [(2.0 ** -85, 0.0), (2.0 ** -126, 0.0), (2.0 ** -55, 2.0 ** -110),
                                     (2.0 ** -85, 2.0 ** -140), (2.0 ** -45, 1e-5), (2.0 ** 45, 2.0 ** 92)])
@pytest.mark.parametrize("c", [128, 1000, 40000])
def test_squares_out_of_range(hip, c, std, eps):
    """bf16 rows whose squares leave fp32's range below (eps next to nothing) or above, eps of their size too."""
    x, _, w = inputs(5, c, "bf16", False)
    x = (x.double() * std).to(torch.bfloat16)
    y, _, rstd = hip.rms_norm(x, w, None, eps, want_rstd=True)
    check_norm(y, rstd if std > 2.0 ** -120 else None, host(x), w, eps, "bf16")
    q, qs, _ = hip.rms_norm_q8(x, w, None, eps)
    t, r = host(x) * host(w), orr.rms_norm(host(x), host(w), eps)[1]
    check_q8(q, qs, t * 2.0 ** 120 if std < 1 else t, r * (2.0 ** -120 if std < 1 else 1.0), slack=E)


@pytest.mark.parametrize("c", [128, 1000, 9000, 40000])
def test_in_place(hip, c):
    """sum over x or over residual, out over x: the same bits as into buffers of their own."""
    x, res, w = inputs(11, c, "bf16", True)
    y, total, _ = hip.rms_norm(x, w, res)
    for over in ("x", "residual", "out"):
        x2, r2 = x.clone(), res.clone()
        y2, t2, _ = hip.rms_norm(x2, w, r2, sum_out={"x": x2, "residual": r2}.get(over, None),
                                 out=x2 if over == "out" else None)
        assert torch.equal(y2, y) and torch.equal(t2, total)
        x2, r2 = x.clone(), res.clone()
        q, qs, _ = hip.rms_norm_q8(x, w, res)
        q2, qs2, t2 = hip.rms_norm_q8(x2, w, r2, sum_out={"x": x2, "residual": r2}.get(over, None))
        assert torch.equal(q2, q) and torch.equal(qs2, qs) and torch.equal(t2, total)
    y1, _, rstd = hip.rms_norm(x, w, want_rstd=True)
    x2 = x.clone()
    assert torch.equal(hip.rms_norm(x2, w, out=x2)[0], y1)
    ds, dw = hip.rms_norm_bwd(x, w, rstd, res, total)
    for over in ("dout", "dsum"):
        do, dt = res.clone(), total.clone()
        d2, dw2 = hip.rms_norm_bwd(x, w, rstd, do, dt, grads=(do if over == "dout" else dt, torch.empty_like(w)))
        assert torch.equal(d2, ds) and torch.equal(dw2, dw)


def shifted(t, by=1):
    """The same values at an address `by` elements past an allocation's start."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    v = flat[by:].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("c", [64, 129, 1024, 2056, 8192])
def test_odd_addresses(hip, c):
    """16-bit buffers that start on any 2-byte address, fp32 ones on any 4-byte one: the same bits."""
    x, res, w = inputs(9, c, "f16", True)
    y, total, rstd = hip.rms_norm(x, w, res, want_rstd=True)
    y2, t2, _ = hip.rms_norm(shifted(x), shifted(w), shifted(res), out=shifted(y), sum_out=shifted(total))
    assert torch.equal(y2, y) and torch.equal(t2, total)
    for act in (0, 1, 2):
        if act == 2 and c % 2:
            continue
        q, qs = hip.quantize_rows(x, act)
        q2, qs2 = hip.quantize_rows(shifted(x), act)
        assert torch.equal(q2, q) and torch.equal(qs2, qs)
        f = x.float()
        q2, qs2 = hip.quantize_rows(shifted(f), act)
        assert torch.equal(q2, q) and torch.equal(qs2, qs)
    ds, dw = hip.rms_norm_bwd(total, w, rstd, y, x)
    d2, dw2 = hip.rms_norm_bwd(shifted(total), shifted(w), shifted(rstd), shifted(y), shifted(x),
                               grads=(shifted(ds), shifted(dw)))
    assert torch.equal(d2, ds) and torch.equal(dw2, dw)
    q, qs = hip.quantize_rows(x)
    v = hip.dequantize_rows(q, qs, c)
    assert torch.equal(hip.dequantize_rows(q, qs, c, out=shifted(v)), v)


def guarded(shape, dtype, fill):
    """A result buffer with a page of `fill` on either side, and a check that they are untouched."""
    n = int(np.prod(shape))
    flat = torch.full((n + 4096,), fill, dtype=dtype, device="cuda")
    return flat[2048:2048 + n].view(shape), lambda: bool((flat[:2048] == fill).all() and (flat[2048 + n:] == fill).all())


@pytest.mark.parametrize("m,c", [(1, 65), (3, 100), (5, 1025), (7, 4097), (2, 20001), (33, 72)])
def test_nothing_outside_is_written(hip, m, c):
    x, res, w = inputs(m, c, "f16", True)
    bufs = [guarded((m, c), torch.float16, 7.0), guarded((m, c), torch.float16, 7.0), guarded((m,), torch.float32, 7.0),
            guarded((m, hip.padded_k(c)), torch.int8, 7), guarded((m,), torch.float32, 7.0), guarded((m, c), torch.float16, 7.0),
            guarded((c,), torch.float32, 7.0)]
    (y, _), (t, _), (rstd, _), (q, _), (qs, _), (ds, _), (dw, _) = bufs
    hip.rms_norm(x, w, res, out=y, sum_out=t, rstd=rstd)
    hip.rms_norm_q8(x, w, res, q=q, q_scale=qs, sum_out=t)
    hip.rms_norm_bwd(t, w, rstd, y, x, grads=(ds, dw))
    hip.quantize_rows(x, 1, q=q, q_scale=qs)
    hip.dequantize_rows(q, qs, out=y)
    assert all(ok() for _, ok in bufs)


# ---- rows to 8 bits ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize_rows(hip, k, act, kind):
    for m in (1, 6, 35 if k < 9000 else 3):
        x, _, _ = inputs(m, 2 * k if act == 2 else k, kind, False)
        q, qs = hip.quantize_rows(x, act)
        h = orr.hidden(host(x), act)
        # swish: the exponent's argument carries |g| E more than one, twice (log2 e and the product)
        slack = 0.0 if act != 2 else (2 * np.abs(host(x)).max() + 8) * 2 * E
        check_q8(q, qs, h, 1.0, slack)
        for out in ("f16", "bf16", "f32"):
            v = hip.dequantize_rows(q, qs, k, DT[out])
            want = q[:, :k].cpu().numpy().astype(np.float64) * host(qs)[:, None]
            assert (np.abs(host(v) - want) <= (U[out] + E) * np.abs(want) + TINY16[out]).all()


@pytest.mark.parametrize("m", [1, 2, 5, 16, 31, 33, 1000, 5001])
@pytest.mark.parametrize("act", [0, 2])
def test_quantize_many_rows(hip, m, act):
    x, _, _ = inputs(m, 256, "bf16", False)
    q, qs = hip.quantize_rows(x, act)
    check_q8(q, qs, orr.hidden(host(x), act), 1.0, 0.0 if act != 2 else (2 * np.abs(host(x)).max() + 8) * 2 * E)


@pytest.mark.parametrize("k", [3, 64, 700, 5000, 40000])
def test_quantize_special_rows(hip, k):
    x, _, _ = inputs(7, k, "f32", False)
    x[1] = 0
    x[2, k - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] = x[4] * 1e-40      # subnormal
    x[5] = x[5].sign() * 3.4e38
    x[6] = -x[6].abs()
    for act in (0, 1):
        q, qs = hip.quantize_rows(x, act)
        h = orr.hidden(host(x), act)
        ok = [0, 1, 4, 5, 6] + ([2] if act == 1 else [])  # relu takes the -inf away
        check_q8(q[ok], qs[ok], h[ok], 1.0)
        for row in (3,) if act else (2, 3):
            assert (q[row] == 0).all() and torch.isnan(qs[row])
        if act:
            assert (q[6] == 0).all() and qs[6] == 0


def test_halves_go_to_even(hip):
    """127 t / a on exact halves: a = 127 and t = k + 1/2."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]], device="cuda")
    q, qs = hip.quantize_rows(x)
    assert q[0, :8].tolist() == [127, 0, 2, 2, 0, -2, -2, 126] and qs[0] == 1.0


def test_on_another_stream(hip):
    """Calls go to the current stream: their inputs are ready only there."""
    x, res, w = inputs(300, 4096, "f16", True)
    want = hip.rms_norm_q8(x, w, res)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(x)
        for _ in range(20):
            late = late + 0 * x
        got = hip.rms_norm_q8(late + x, w, res)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("m,c", [(300000, 8), (4097, 65)])
def test_more_rows_than_workgroups(hip, m, c):
    x, res, w = inputs(m, c, "bf16", True)
    y, total, rstd = hip.rms_norm(x, w, res, want_rstd=True)
    check_sum(total, x, res, "bf16")
    check_norm(y, rstd, host(total), w, 1e-5, "bf16")
    q, qs = hip.quantize_rows(x)
    check_q8(q, qs, host(x), 1.0)


def test_offsets_past_2_31(hip):
    """Rows whose byte offsets pass 2^32: the last ones against the same rows alone."""
    m, c = 140001, 16384
    x = torch.empty((m, c), dtype=torch.bfloat16, device="cuda")
    x.fill_(1.0)
    tail, _, w = inputs(3, c, "bf16", False)
    x[-3:] = tail
    q, qs, _ = hip.rms_norm_q8(x, w)
    q1, qs1, _ = hip.rms_norm_q8(tail, w)
    assert torch.equal(q[-3:], q1) and torch.equal(qs[-3:], qs1) and torch.equal(q[5], q[m - 5])
    q, qs = hip.quantize_rows(x, 2)
    q1, qs1 = hip.quantize_rows(tail, 2)
    assert torch.equal(q[-3:], q1) and torch.equal(qs[-3:], qs1)
    y, _, rstd = hip.rms_norm(x, w, want_rstd=True, out=x)
    y1, _, rstd1 = hip.rms_norm(tail, w, want_rstd=True)
    assert torch.equal(y[-3:], y1) and torch.equal(rstd[-3:], rstd1)
    ds, _ = hip.rms_norm_bwd(x, w, rstd, x)
    ds1, _ = hip.rms_norm_bwd(y1, w, rstd1, y1)
    assert torch.equal(ds[-3:], ds1)


# ---- the integers themselves, against 127 t / a without a rounding before the nearest ---------------

def check_nearest(q, t):
    """q's first columns are the nearest integers to 127 t / a, bit for bit (t: fp32 values)."""
    assert np.array_equal(q.cpu().numpy()[:, :t.shape[1]].astype(np.float64), orr.nearest(t))


def norm_products(x, w):
    return (x.float().cpu().numpy() * w.cpu().numpy()[None]).astype(np.float64)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("c", [13, 64, 512, 1000, 2050, 8200, 16384, 20001])
def test_nearest_integers(hip, c, kind):
    for m in (3, 4000000 // c // 8):
        x, res, w = inputs(m, c, kind, kind != "f32", seed=11)
        for act in (0, 1):
            check_nearest(hip.quantize_rows(x, act)[0], orr.hidden(host(x), act))
        if kind != "f32":
            check_nearest(hip.rms_norm_q8(x, w)[0], norm_products(x, w))
            q, _, total = hip.rms_norm_q8(x, w, res)
            check_nearest(q, norm_products(total, w))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_half_of_the_largest(hip, kind):
    """t = a / 2, so 127 t / a = 63.5, for every 16-bit a above the type's smallest hundred: 64, whatever 127 / a rounds
    to; and a row of both signs."""
    bits = torch.arange(101 if kind == "f16" else 0x500, int(torch.tensor(float("inf"), dtype=DT[kind]).view(torch.int16)),
                        dtype=torch.int16)
    a = bits.view(DT[kind])
    x = torch.stack([a, a / 2, -a / 2, -a, a / 4, torch.zeros_like(a)], 1).cuda()
    x = x[(x[:, 1] * 2 == x[:, 0]) & (x[:, 0] >= 2.0 ** -119)]
    q, _ = hip.quantize_rows(x)
    assert len(x) > 20000 and (q[:, :4].cpu() == torch.tensor([127, 64, -64, -127])).all()
    check_nearest(q, host(x))
    check_nearest(hip.rms_norm_q8(x, torch.ones(6, device="cuda"))[0], host(x))


@pytest.mark.parametrize("k", [61, 1000, 9000, 40000])
@pytest.mark.parametrize("low,high", [(-10, 10), (-118, -100), (110, 127), (-119, 127)])
def test_next_to_halves(hip, k, low, high):
    """fp32 values on, and up to three steps beside, the halves of a row's scale."""
    rng = np.random.default_rng(k + 300 + low)
    m = 200000 // k + 1
    a = (rng.uniform(1, 2, (m, 1)) * 2.0 ** rng.integers(low, high + 1, (m, 1))).astype(np.float32)
    t = (a.astype(np.float64) * (2 * rng.integers(-127, 127, (m, k)) + 1) / 254).astype(np.float32)
    t = (t.view(np.int32) + rng.integers(-3, 4, (m, k)).astype(np.int32)).view(np.float32)
    t[:, 0] = a[:, 0]
    t[:, k // 2] = -a[:, 0] / 2
    assert np.abs(t).max() < np.inf and (np.abs(t).max(1) == a[:, 0]).all()
    q, _ = hip.quantize_rows(torch.from_numpy(t).cuda())
    check_nearest(q, t)


@pytest.mark.parametrize("c", [13, 128, 1000, 9000, 40000])
@pytest.mark.parametrize("wexp", [-50, -80, -100, -126, -150])
def test_huge_rows_of_tiny_weights(hip, c, wexp):
    """bf16 rows past 2^40 times weights of any size: a row is zeros where its own largest product is under 2^-119, not
    where that of the values as they are taken for their squares is."""
    x, _, w = inputs(6, c, "bf16", False)
    x = x * 2.0 ** 60
    x[1] = x[1] * 2.0 ** 60
    w = w * 2.0 ** (wexp / 2) * 2.0 ** (wexp / 2)
    x[2] = 0
    x[2, 0] = 2.0 ** 41
    q, qs, _ = hip.rms_norm_q8(x, w)
    t = norm_products(x, w)
    check_nearest(q, t)
    quot, scale = orr.quotients(t)
    assert wexp < -126 or (np.abs(quot).max(1) == 127).all()
    want = scale * orr.rms_norm(host(x), host(w), 1e-5)[1]
    # below fp32's normal range a scale is off by half its smallest step
    assert (np.abs(host(qs) - want) <= (12 + seq(c)) * E * want + 2.0 ** -150).all()


@pytest.mark.parametrize("m,c", [((1 << 25) + 5, 1), ((1 << 20) + 3, 1025)])
def test_more_rows_than_a_grid_takes(hip, m, c):
    """A grid has at most 2^20 workgroups (of 32 rows each where rows are shortest): the rows past it are their second
    ones. Every row is compared with the same row in calls that fit a grid."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    x = torch.empty((m, c), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = torch.ones(c, device="cuda").normal_(generator=gen)
    y, total, rstd = hip.rms_norm(x, w, x, want_rstd=True)
    q, qs, _ = hip.rms_norm_q8(x, w)
    h, hs = hip.quantize_rows(x, 1)
    v = hip.dequantize_rows(h, hs, c)
    step = m // 3 + 1
    for lo in range(0, m, step):
        part = x[lo:lo + step]
        y1, total1, rstd1 = hip.rms_norm(part, w, part, want_rstd=True)
        q1, qs1, _ = hip.rms_norm_q8(part, w)
        h1, hs1 = hip.quantize_rows(part, 1)
        v1 = hip.dequantize_rows(h1, hs1, c)
        for whole, alone in ((y, y1), (total, total1), (rstd, rstd1), (q, q1), (qs, qs1), (h, h1), (hs, hs1), (v, v1)):
            assert torch.equal(whole[lo:lo + step], alone)
    last = slice(m - 70, m)
    check_norm(y[last], rstd[last], host(total[last]), w, 1e-5, "bf16")
    check_nearest(q[last], norm_products(x[last], w))


def test_more_long_rows_than_a_grid_takes(hip):
    """The same for the rows of any length, 34 GB of them: the last five against calls of their own."""
    m, c = (1 << 20) + 5, 16385
    x = torch.ones((m, c), dtype=torch.bfloat16, device="cuda")
    tail, _, w = inputs(8, c, "bf16", False)
    x[-8:] = tail
    q, qs = hip.quantize_rows(x)
    q1, qs1 = hip.quantize_rows(tail)
    assert torch.equal(q[-8:], q1) and torch.equal(qs[-8:], qs1) and torch.equal(q[3], q[m - 9])
    hip.rms_norm_q8(x, w, q=q, q_scale=qs)
    q1, qs1, _ = hip.rms_norm_q8(tail, w)
    assert torch.equal(q[-8:], q1) and torch.equal(qs[-8:], qs1) and torch.equal(q[3], q[m - 9])
    del q
    y1, _, rstd1 = hip.rms_norm(tail, w, want_rstd=True)
    _, _, rstd = hip.rms_norm(x, w, want_rstd=True, out=x)
    assert torch.equal(x[-8:], y1) and torch.equal(rstd[-8:], rstd1) and torch.equal(x[3], x[m - 9])
    del x
    torch.cuda.empty_cache()
