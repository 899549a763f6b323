"""Heads' norm and rotation, and the key-value cache written and read, on the GPU against the float64 oracle.

Tolerances. A result of 16 bits is off by half a step of its type, and by fp32's rounding before that: each value of the
forward is a sum of two products, each with about a dozen roundings of 2^-24 (16 values are summed lane by lane, then
over at most 32 lanes), 2^-20 of what it is summed from. Gradients have twice as many, 2^-19, and the weights'
gradients are sums with at most a hundred additions in a row at these sizes, 2^-17 of the sum of the terms' magnitudes.
8-bit rows of fp32 values lie within that, 127 times, of the nearest integer."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import layouts, torch_ops
from oracle import heads as oh
from oracle import rows8 as orr

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def np64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, terms, dtype, part=2.0 ** -20):
    """|got - want| within half a step of the type and `part` of the terms (fp16's steps do not shrink under 2^-24)."""
    got = np64(got)
    half = torch.finfo(dtype).eps / 2 if dtype is not None else 2.0 ** -24
    least = 2.0 ** -25 if dtype is torch.float16 else 0.0
    room = (half * np.abs(want) + part * terms) * 1.001 + least
    bad = ~(np.abs(got - want) <= room)
    assert not bad.any(), (got[bad][:4], want[bad][:4], room[bad][:4], int(bad.sum()))


def inputs(t, hq, hkv, d, r, kind, seed=0, p=200):
    rng = np.random.default_rng([seed, t, hq, d])
    dt = TYPES[kind]
    make = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    x = make(t, hq + 2 * hkv, d).to(dt)
    rope = layouts.rope_table(p, r, 100.0, "cuda")
    pos = torch.from_numpy(rng.integers(0, p, t).astype(np.int32)).cuda()
    return x, 1 + 0.2 * make(d), 1 + 0.2 * make(d), rope, pos, [make(t, h, d).to(dt) for h in (hq, hkv, hkv)]


def want_heads(x, qn, kn, rope, pos, hkv, interleaved, eps=EPS):
    x64, hq = np64(x), x.shape[1] - 2 * hkv
    at = (np64(rope), pos.cpu().numpy())
    return (oh.norm_rope(x64[:, :hq], np64(qn), *at, eps, interleaved), oh.norm_rope(x64[:, hq:hq + hkv], np64(kn), *at, eps, interleaved),
            x[:, hq + hkv:])


SHAPES = [(1, 1, 1, 8, 8), (3, 2, 1, 16, 8), (5, 3, 3, 24, 16), (17, 4, 2, 32, 32), (33, 6, 2, 48, 40), (64, 5, 1, 64, 32), (65, 9, 3, 80, 80),
          (31, 8, 2, 96, 48), (130, 7, 7, 128, 128), (19, 40, 8, 128, 64), (9, 4, 1, 160, 160), (7, 6, 3, 192, 96), (12, 5, 5, 224, 16),
          (21, 2, 2, 256, 256), (700, 33, 11, 128, 128), (6000, 12, 2, 64, 64)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,r", SHAPES)
def test_forward(hip, t, hq, hkv, d, r, kind):
    for interleaved in (False, True):
        x, qn, kn, rope, pos, _ = inputs(t, hq, hkv, d, r, kind)
        q, k, v = hip.qk_norm_rope(x, qn, kn, rope, pos, hkv, EPS, interleaved)
        (wq, tq), (wk, tk), wv = want_heads(x, qn, kn, rope, pos, hkv, interleaved)
        close(q, wq, tq, TYPES[kind])
        close(k, wk, tk, TYPES[kind])
        assert torch.equal(v, wv)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,r", SHAPES)
def test_backward(hip, t, hq, hkv, d, r, kind):
    for interleaved in (False, True):
        x, qn, kn, rope, pos, dy = inputs(t, hq, hkv, d, r, kind)
        got = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, interleaved)
        x64, at = np64(x), (np64(rope), pos.cpu().numpy())
        for w, g, lo, hi, dw in ((qn, dy[0], 0, hq, got[1]), (kn, dy[1], hq, hq + hkv, got[2])):
            dx, terms, want, wterms = oh.norm_rope_bwd(x64[:, lo:hi], np64(w), *at, np64(g), EPS, interleaved)
            close(got[0][:, lo:hi], dx, terms, TYPES[kind], 2.0 ** -19)
            close(dw, want, wterms, None, 2.0 ** -17)
        assert torch.equal(got[0][:, hq + hkv:], dy[2])
        again = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, interleaved)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("t,hq,hkv", [(1, 1, 1), (17, 5, 2), (600, 3, 1)])
def test_backward_without_eps(hip, t, hq, hkv):
    """Tokens and heads that only fill up a workgroup count as zeros also where eps is 0."""
    x, qn, kn, rope, pos, dy = inputs(t, hq, hkv, 96, 48, "f16")
    got = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, 0.0)
    for w, g, lo, hi, dw in ((qn, dy[0], 0, hq, got[1]), (kn, dy[1], hq, hq + hkv, got[2])):
        dx, terms, want, wterms = oh.norm_rope_bwd(np64(x)[:, lo:hi], np64(w), np64(rope), pos.cpu().numpy(), np64(g), 0.0, False)
        close(got[0][:, lo:hi], dx, terms, torch.float16, 2.0 ** -19)
        close(dw, want, wterms, None, 2.0 ** -17)


def test_backward_of_no_tokens(hip):
    x, qn, kn, rope, pos, dy = inputs(0, 4, 2, 64, 32, "f16")
    dx, dq, dk = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy)
    assert dx.shape == x.shape and (dq == 0).all() and (dk == 0).all()
    q, k, v = hip.qk_norm_rope(x, qn, kn, rope, pos, 2)
    assert q.shape == (0, 4, 64) and k.shape == v.shape == (0, 2, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_autograd(hip, interleaved):
    """Batched tokens, shared positions, a query gradient alone, and the sum over the heads that share a norm's weight."""
    x, qn, kn, rope, pos, dy = inputs(2 * 9, 4, 2, 64, 48, "f16")
    xb = x.view(2, 9, 8, 64).clone().requires_grad_()
    qn.requires_grad_(), kn.requires_grad_()
    shared = pos[:9]
    y = torch_ops.qk_norm_rope(xb, qn, kn, rope, shared, 2, EPS, interleaved)
    assert [tuple(t.shape) for t in y] == [(2, 9, 4, 64), (2, 9, 2, 64), (2, 9, 2, 64)]
    at = (np64(rope), np.concatenate([shared.cpu().numpy()] * 2))
    grads = torch.autograd.grad(y, (xb, qn, kn), [g.view(t.shape) for g, t in zip(dy, y)], retain_graph=True)
    flat = hip.qk_norm_rope_bwd(x, qn.detach(), kn.detach(), rope, torch.cat([shared, shared]), *dy, EPS, interleaved)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(grads, flat))
    dx, dq, dk = torch.autograd.grad(y[0], (xb, qn, kn), dy[0].view(y[0].shape))
    want, terms, _, _ = oh.norm_rope_bwd(np64(x)[:, :4], np64(qn), *at, np64(dy[0]), EPS, interleaved)
    close(dx.view(18, 8, 64)[:, :4], want, terms, torch.float16, 2.0 ** -19)
    assert (dx.view(18, 8, 64)[:, 4:] == 0).all() and (dk == 0).all() and torch.equal(dq, flat[1])
    with torch.no_grad():
        z = torch_ops.qk_norm_rope(xb, qn, kn, rope, shared, 2, EPS, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(y, z))
    strided = torch.cat([xb.detach(), xb.detach()], -1)[..., :64]
    assert not strided.is_contiguous()
    z = torch_ops.qk_norm_rope(strided, qn.detach(), kn.detach(), rope, shared, 2, EPS, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(y, z))


def test_gradient_accumulates_in_leaves(hip):
    """Two passes into the same leaves: a leaf keeps a gradient of its own."""
    x, qn, kn, rope, pos, dy = inputs(5, 4, 2, 64, 64, "bf16")
    x.requires_grad_(), qn.requires_grad_(), kn.requires_grad_()
    for n in (1, 2):
        torch.autograd.backward(torch_ops.qk_norm_rope(x, qn, kn, rope, pos, 2, EPS), dy)
        if n == 1:
            first = [t.grad.clone() for t in (x, qn, kn)]
    assert torch.equal(x.grad, (first[0].float() * 2).to(x.dtype)) and torch.equal(qn.grad, first[1] * 2)


def test_duals_and_captures_are_refused(hip):
    from torch.autograd import forward_ad
    x, qn, kn, rope, pos, dy = inputs(5, 4, 2, 64, 64, "f16")
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        torch_ops.qk_norm_rope(forward_ad.make_dual(x, x), qn, kn, rope, pos, 2)
    x.requires_grad_()
    y = torch_ops.qk_norm_rope(x, qn, kn, rope, pos, 2)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        with pytest.raises(hip.InvalidArgument, match="cannot be captured"):
            torch_ops.qk_norm_rope(x, qn, kn, rope, pos, 2)
        keep = torch.zeros(1, device="cuda")
    del keep, y


@pytest.mark.parametrize("kind", TYPES)
def test_special_heads(hip, kind):
    """Zeros, infinities and NaN stay in their heads (and, rotated, in their pairs); positions outside the table give NaN."""
    x, qn, kn, rope, pos, dy = inputs(6, 4, 2, 64, 32, kind)
    x[0, 0] = 0
    x[1, 1, 3] = float("inf")
    x[2, 4, 40] = float("nan")
    pos[4], pos[5] = -1, rope.shape[0]
    q, k, v = hip.qk_norm_rope(x, qn, kn, rope, pos, 2, EPS)
    (wq, tq), (wk, tk), wv = want_heads(x[[0, 3]], qn, kn, rope, pos[[0, 3]], 2, False)
    assert (q[0, 0] == 0).all()
    close(q[[0, 3]], wq, tq, TYPES[kind])
    close(k[[0, 3]], wk, tk, TYPES[kind])
    assert torch.isnan(q[1, 1, [3, 19]]).all() and (q[1, 1, [0, 1, 2, 4, 40, 63]] == 0).all() and torch.isfinite(q[1, [0, 2, 3]]).all()
    assert torch.isnan(k[2, 0]).all() and torch.isfinite(k[2, 1]).all()
    assert torch.isnan(q[4:]).all() and torch.isnan(k[4:]).all() and torch.equal(v, x[:, 6:])
    dx = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS)[0]
    assert torch.isnan(dx[4:, :6]).all() and torch.isfinite(dx[[0, 3]]).all() and torch.equal(dx[:, 6:], dy[2])


@pytest.mark.parametrize("std", (1e25, 1e-25))
def test_squares_out_of_range(hip, std):
    """bf16 heads whose squares leave fp32's range, with an eps of nothing."""
    x, qn, kn, rope, pos, dy = inputs(9, 3, 2, 96, 96, "bf16")
    x = (x.float() * std).to(torch.bfloat16)
    q, k, _ = hip.qk_norm_rope(x, qn, kn, rope, pos, 2, 0.0)
    (wq, tq), (wk, tk), _ = want_heads(x, qn, kn, rope, pos, 2, False, 0.0)
    close(q, wq, tq, torch.bfloat16)
    close(k, wk, tk, torch.bfloat16)
    dx = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, 0.0)[0]
    want, terms, _, _ = oh.norm_rope_bwd(np64(x)[:, :3], np64(qn), np64(rope), pos.cpu().numpy(), np64(dy[0]), 0.0, False)
    close(dx[:, :3], want, terms, torch.bfloat16, 2.0 ** -19)


@pytest.mark.parametrize("kind", TYPES)
def test_every_pattern_passes(hip, kind):
    """What is only moved keeps its 16 bits, whatever they are: values, their gradients, and the cache."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(256, 2, 128).cuda()
    x, qn, kn, rope, pos, dy = inputs(256, 4, 2, 128, 128, kind)
    x[:, 6:] = bits.view(TYPES[kind])
    v = hip.qk_norm_rope(x, qn, kn, rope, pos, 2, EPS)[2]
    assert torch.equal(v.view(torch.int16), bits)
    dx = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, dy[0], dy[1], bits.view(TYPES[kind]), EPS)[0]
    assert torch.equal(dx[:, 6:].contiguous().view(torch.int16), bits)
    slots, cache = run_of(256, 18, 16, 3), hip.kv_cache(18, 2, 16, 128, TYPES[kind])
    hip.kv_cache_write(bits.view(TYPES[kind]), v, slots, cache)
    assert all(torch.equal(t.view(torch.int16), bits) for t in hip.kv_cache_read(cache, slots))
    cache = hip.kv_cache(18, 2, 16, 128, TYPES[kind])
    hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, cache, EPS)
    assert torch.equal(hip.kv_cache_read(cache, slots)[1].view(torch.int16), bits)


@pytest.mark.parametrize("t", (1, 37, 3000))
def test_nothing_outside_is_written(hip, t):
    x, qn, kn, rope, pos, dy = inputs(t, 3, 1, 96, 64, "f16")
    bufs = [torch.full((t + 2, h, 96), 7.0, dtype=torch.float16, device="cuda") for h in (3, 1, 1, 5)]
    hip.qk_norm_rope(x, qn, kn, rope, pos, 1, EPS, out=[b[1:-1] for b in bufs[:3]])
    dw = torch.full((2, 128), 7.0, device="cuda")
    hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, grads=(bufs[3][1:-1], dw[0, :96], dw[1, :96]))
    for b in bufs:
        assert (b[0] == 7).all() and (b[-1] == 7).all() and not (b[1:-1] == 7).all()
    assert (dw[:, 96:] == 7).all()


# ---- the cache ----------------------------------------------------------------------------

def scattered(t, pages, page, seed=0):
    """t distinct slots in any order, every fifth not in the cache."""
    rng = np.random.default_rng(seed)
    s = rng.permutation(pages * page)[:t].astype(np.int32)
    s[::5] = np.resize([-1, pages * page, -2 ** 31, 2 ** 31 - 1], len(s[::5]))
    return torch.from_numpy(s).cuda()


def run_of(t, pages, page, start, seed=0):
    """A prompt's slots from place `start` of its first page on."""
    order = np.random.default_rng(seed).permutation(pages)
    at = start + np.arange(t)
    return torch.from_numpy((order[at // page] * page + at % page).astype(np.int32)).cuda()


def dense(cache):
    """(k, v) [pages, heads, page, d], as the cache's numbers."""
    return layouts.keys_unblocked(cache.k), layouts.values_unblocked(cache.v)


CACHES = [(1, 1, 32, 16), (40, 3, 64, 16), (70, 2, 96, 32), (33, 8, 128, 48), (129, 1, 160, 64), (50, 4, 192, 16), (20, 2, 224, 16),
          (300, 2, 256, 128), (2500, 5, 128, 64), (2500, 3, 96, 32)]


def all_slots(t, page):
    """Slots of each pattern, and the pages they need."""
    pages = -(-(t + page) // page) + 2
    for start in (0, 5, 16 % page):
        yield run_of(t, pages, page, start), pages
    yield scattered(t, 2 * pages, page), 2 * pages
    both = torch.cat([run_of(t, pages, page, 0)[: t // 2], torch.full((t - t // 2,), -1, dtype=torch.int32, device="cuda")])
    yield both, pages


def check_written(cache, slots, page, want):
    """Each token's head where its slot says, zeros everywhere else; want(k or v index) the rows written."""
    live = ((slots >= 0) & (slots < cache.k.shape[0] * page)).cpu().numpy()
    at = slots.cpu().numpy()[live]
    for n, x in enumerate(dense(cache)):
        rows = x.cpu().permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])
        other = torch.ones(len(rows), dtype=torch.bool)
        other[at] = False
        assert (rows[other] == 0).all()
        want(n, rows[at], live)
        scale = cache[2 + n]
        if scale is not None:
            assert (scale.cpu().permute(0, 2, 1).reshape(-1, x.shape[1])[other] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,heads,d,page", CACHES)
def test_write_and_read_16(hip, t, heads, d, page, kind):
    x, *_ = inputs(t, heads, heads, d, 8, kind)
    k, v = x[:, :heads].contiguous(), x[:, heads:2 * heads].contiguous()
    for slots, pages in all_slots(t, page):
        cache = hip.kv_cache(pages, heads, page, d, TYPES[kind])
        hip.kv_cache_write(k, v, slots, cache)
        check_written(cache, slots, page, lambda n, rows, live: None if torch.equal(rows, (k, v)[n].cpu()[live]) else pytest.fail("rows"))
        rk, rv = hip.kv_cache_read(cache, slots)
        live = ((slots >= 0) & (slots < pages * page))[:, None, None]
        assert torch.equal(rk, torch.where(live, k, torch.zeros_like(k))) and torch.equal(rv, torch.where(live, v, torch.zeros_like(v)))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,heads,d,page", CACHES)
def test_write_and_read_8(hip, t, heads, d, page, kind):
    """16-bit values go to the nearest integer, exactly; reading gives integer times scale, rounded once."""
    x, *_ = inputs(t, heads, heads, d, 8, kind)
    x[0, 0] = 0
    k, v = x[:, :heads].contiguous(), x[:, heads:2 * heads].contiguous()
    for slots, pages in all_slots(t, page):
        cache = hip.kv_cache(pages, heads, page, d)
        hip.kv_cache_write(k, v, slots, cache)

        def want(n, rows, live):
            w = np64((k, v)[n]).reshape(-1, d)
            assert np.array_equal(rows.numpy(), orr.nearest(w).reshape(t, heads, d)[live])
            s = cache[2 + n].double().cpu().permute(0, 2, 1).reshape(-1, heads).numpy()[slots.cpu().numpy()[live]]
            a = orr.quotients(w)[1].reshape(t, heads)[live]
            assert (np.abs(s - a) <= 2.0 ** -23 * a).all()
        check_written(cache, slots, page, want)
        ints = [t.cpu().permute(0, 2, 1, 3).reshape(-1, heads, d) for t in dense(cache)]
        scales = [t.cpu().permute(0, 2, 1).reshape(-1, heads) for t in cache[2:]]
        at = slots.cpu().long()
        live = (at >= 0) & (at < pages * page)
        at = torch.where(live, at, torch.zeros_like(at))
        for dt in TYPES.values():
            for got, i, s in zip(hip.kv_cache_read(cache, slots, dt), ints, scales):
                w = (i[at].float() * s[at][..., None]).to(dt)
                assert torch.equal(got.cpu(), torch.where(live[:, None, None], w, torch.zeros_like(w)))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,heads,d,page", CACHES)
def test_norm_rope_into_the_cache(hip, t, heads, d, page, kind):
    """16 bits: what qk_norm_rope gives, to the bit. 8 bits: the rows of the fp32 values before that rounding."""
    hq, r = 2 * heads + 1, d // 2
    x, qn, kn, rope, pos, _ = inputs(t, hq, heads, d, r, kind)
    for interleaved in (False, True):
        q, k, v = hip.qk_norm_rope(x, qn, kn, rope, pos, heads, EPS, interleaved)
        _, (wk, tk), _ = want_heads(x, qn, kn, rope, pos, heads, interleaved)
        for slots, pages in all_slots(t, page):
            cache = hip.kv_cache(pages, heads, page, d, TYPES[kind])
            assert torch.equal(hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, cache, EPS, interleaved), q)
            check_written(cache, slots, page, lambda n, rows, live: None if torch.equal(rows, (k, v)[n].cpu()[live]) else pytest.fail("rows"))
            cache = hip.kv_cache(pages, heads, page, d)
            assert torch.equal(hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, cache, EPS, interleaved), q)

            def want(n, rows, live):
                s = cache[2 + n].double().cpu().permute(0, 2, 1).reshape(-1, heads).numpy()[slots.cpu().numpy()[live]]
                got = rows.double().numpy()
                if n == 1:
                    w = np64(v).reshape(-1, d)
                    assert np.array_equal(got, orr.nearest(w).reshape(t, heads, d)[live])
                    return
                a = np.abs(wk).max(-1)[live]
                room = 2.0 ** -20 * tk.max(-1)[live]
                assert (np.abs(s * 127 - a) <= room + 2.0 ** -22 * a).all()
                off = np.abs(got - wk[live] * (127 / a)[..., None])
                assert (off <= 0.5 + (254 * room / a)[..., None] + 2.0 ** -16).all(), off.max()
            check_written(cache, slots, page, want)


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("t,heads,d,page", ((1100, 9, 128, 32), (2100, 9, 128, 16), (1100, 17, 64, 48), (2500, 5, 256, 16), (4100, 3, 96, 64), (2100, 33, 32, 16)))
def test_long_prompts_as_short_ones(hip, t, heads, d, page, bits):
    """A token's rows do not depend on the call: long ones, whose workgroups take several heads, give what short ones give."""
    x, qn, kn, rope, pos, _ = inputs(t, heads + 1, heads, d, d // 2, "bf16")
    for slots, pages in all_slots(t, page):
        one, many = (hip.kv_cache(pages, heads, page, d, torch.int8 if bits == 8 else torch.bfloat16) for _ in range(2))
        q = hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, one, EPS)
        parts = [hip.qk_norm_rope_cache(x[i:i + 37], qn, kn, rope, pos[i:i + 37].clone(), slots[i:i + 37].clone(), many, EPS)
                 for i in range(0, t, 37)]
        assert torch.equal(q, torch.cat(parts))
        assert all(torch.equal(a, b) for a, b in zip(one, many) if a is not None)


def test_rows_that_are_not_finite(hip):
    x, qn, kn, rope, pos, _ = inputs(20, 2, 1, 64, 64, "bf16")
    x[3, 2, 5] = float("inf")
    x[4, 3, 6] = float("nan")
    pos[5] = -1
    cache = hip.kv_cache(4, 1, 16, 64)
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, cache, EPS)
    ks, vs = cache.k_scale.view(-1), cache.v_scale.view(-1)
    assert torch.isnan(ks[[3, 5]]).all() and torch.isnan(vs[4]) and int(torch.isnan(ks).sum()) == 2 and int(torch.isnan(vs).sum()) == 1
    k, v = hip.kv_cache_read(cache, slots)
    assert torch.isnan(k[[3, 5]]).all() and torch.isnan(v[4]).all() and int(torch.isnan(k).sum()) == 128


def test_read_the_same_slot_often(hip):
    x, *_ = inputs(40, 2, 2, 64, 8, "f16")
    k, v = x[:, :2].contiguous(), x[:, 2:4].contiguous()
    cache = hip.kv_cache(3, 2, 16, 64, torch.float16)
    hip.kv_cache_write(k, v, torch.arange(40, dtype=torch.int32, device="cuda"), cache)
    at = torch.tensor([7] * 50 + [39, 0, 7, 38, 48, 47], dtype=torch.int32, device="cuda")
    rk, rv = torch_ops.kv_cache_read(cache, at.view(2, 28))
    w = torch.cat([k, torch.zeros_like(k[:8])])
    assert rk.shape == (2, 28, 2, 64) and torch.equal(rk.view(56, 2, 64)[:54], w[at[:54].long()]) and (rk.view(56, 2, 64)[54:] == 0).all()


def test_offsets_past_2_31(hip):
    """A cache whose bytes pass 2^32 (and its 16-bit values 2^31): its last page, and nothing near it."""
    pages, heads, page, d = 33000, 4, 128, 128
    x, *_ = inputs(40, heads, heads, d, 8, "f16")
    k, v = x[:, :heads].contiguous(), x[:, heads:2 * heads].contiguous()
    for dt in (torch.float16, torch.int8):
        cache = hip.kv_cache(pages, heads, page, d, dt)
        slots = torch.arange(pages * page - 40, pages * page, dtype=torch.int32, device="cuda")
        hip.kv_cache_write(k, v, slots, cache)
        assert all((c[:-1] == 0).all() for c in cache if c is not None)
        rk, rv = hip.kv_cache_read(cache, slots, torch.float16)
        part = 0.0 if dt is torch.float16 else 1 / 254 + 2.0 ** -10
        assert ((rk - k).abs().float() <= part * k.abs().amax(-1, keepdim=True).float()).all()
        assert ((rv - v).abs().float() <= part * v.abs().amax(-1, keepdim=True).float()).all()
        del cache


def test_on_another_stream(hip):
    x, qn, kn, rope, pos, dy = inputs(2000, 8, 2, 128, 128, "bf16")
    want = hip.qk_norm_rope(x, qn, kn, rope, pos, 2, EPS)
    grads = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        y = x + big[0, 0].to(x.dtype) * 0
        got = hip.qk_norm_rope(y, qn, kn, rope, pos, 2, EPS)
        back = hip.qk_norm_rope_bwd(y, qn, kn, rope, pos, *dy, EPS)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want + grads, got + back))


def test_captured(hip):
    """A step and the gradients replayed from a graph, with the inputs changed and eager calls between the replays."""
    x, qn, kn, rope, pos, dy = inputs(33, 6, 2, 64, 64, "f16")
    slots, cache = scattered(33, 9, 16), hip.kv_cache(9, 2, 16, 64)
    ws = torch.empty(hip.qk_norm_rope_bwd_workspace(x, dy[1]), dtype=torch.uint8, device="cuda")
    grads = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, cache, EPS)
        k, v = hip.kv_cache_read(cache, slots)
        hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, workspace=ws, grads=grads)
    for n in range(4):
        x.copy_(inputs(33, 6, 2, 64, 64, "f16", seed=n)[0])
        g.replay()
        torch.cuda.synchronize()
        other = hip.kv_cache(9, 2, 16, 64)
        assert torch.equal(q, hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, other, EPS))
        assert all(torch.equal(a, b) for a, b in zip((k, v), hip.kv_cache_read(other, slots)))
        assert all(torch.equal(a, b) for a, b in zip(grads, hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS)))
