"""Heads' norm and rotation, its gradients, and the cache in calls so large that workgroups take several heads or go round for
further tokens, on the GPU: to the bit what short calls give, and a sample against the float64 definition."""
import pytest
import torch

from colabfold_legacy_kernels import layouts
from oracle import heads as oh
from test_heads_gpu import close, np64, want_heads

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS, P = 1e-6, 500


def inputs(t, hq, hkv, d, r, kind, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(s, generator=gen, device="cuda", dtype=TYPES[kind])  # noqa: E731
    w = [1 + 0.2 * torch.randn(d, generator=gen, device="cuda") for _ in range(2)]
    pos = torch.randint(0, P, (t,), generator=gen, device="cuda", dtype=torch.int32)
    return make(t, hq + 2 * hkv, d), w[0], w[1], layouts.rope_table(P, r, 100.0, "cuda"), pos, make


def sample(t):
    """Tokens at the ends, at blocks' borders and between."""
    return torch.tensor(sorted({0, 1, 7, 8, 15, 16, 63, 64, t // 3, t // 2, t - 65, t - 17, t - 2, t - 1}), device="cuda")


# (tokens, query heads, key heads, d, r), neither a multiple of what workgroups take: four heads a workgroup, then eight
FOUR = [(4099, 33, 7, 128, 64), (4099, 33, 7, 96, 96), (16387, 33, 7, 32, 32), (2051, 33, 7, 256, 128), (65539, 33, 7, 8, 8)]
EIGHT = [(16385, 51, 6, 128, 128), (16385, 51, 6, 96, 48), (16389, 51, 6, 32, 16), (8195, 51, 6, 160, 160)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,r", FOUR + EIGHT)
def test_forward(hip, t, hq, hkv, d, r, kind):
    x, qn, kn, rope, pos, _ = inputs(t, hq, hkv, d, r, kind)
    for interleaved in (False, True):
        guard = [torch.full((t + 2, h, d), 7.0, dtype=x.dtype, device="cuda") for h in (hq, hkv, hkv)]
        got = hip.qk_norm_rope(x, qn, kn, rope, pos, hkv, EPS, interleaved, out=[b[1:-1] for b in guard])
        assert all((b[0] == 7).all() and (b[-1] == 7).all() for b in guard)
        short = 2 ** 19 // ((hq + 2 * hkv) * d // 4)  # tokens of which a workgroup takes one head
        parts = [hip.qk_norm_rope(x[i:i + short], qn, kn, rope, pos[i:i + short].clone(), hkv, EPS, interleaved)
                 for i in range(0, t, short)]
        assert all(torch.equal(a, torch.cat(b)) for a, b in zip(got, zip(*parts)))
        at = sample(t)
        (wq, tq), (wk, tk), wv = want_heads(x[at], qn, kn, rope, pos[at], hkv, interleaved)
        close(got[0][at], wq, tq, TYPES[kind])
        close(got[1][at], wk, tk, TYPES[kind])
        assert torch.equal(got[2][at], wv)


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,r", [s for s in FOUR if s[3] >= 32] + [(8195, 51, 6, 160, 160)])
def test_step(hip, t, hq, hkv, d, r, kind, bits):
    """Several heads of queries a workgroup beside several of keys and values: what the heads apart and short calls give."""
    x, qn, kn, rope, pos, _ = inputs(t, hq, hkv, d, r, kind)
    page, pages = 48, -(-t // 48) + 2
    slots = torch.randperm(pages, generator=torch.Generator().manual_seed(t)).to(torch.int32)
    at = torch.arange(t, dtype=torch.int32) + 5
    slots = (slots[(at // page).long()] * page + at % page).cuda()
    slots[::1000] = -1
    for interleaved in (False, True):
        q0 = hip.qk_norm_rope(x, qn, kn, rope, pos, hkv, EPS, interleaved)[0]
        one, many = (hip.kv_cache(pages, hkv, page, d, torch.int8 if bits == 8 else TYPES[kind]) for _ in range(2))
        assert torch.equal(hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, one, EPS, interleaved), q0)
        for i in range(0, t, 48):
            s = slice(i, i + 48)
            hip.qk_norm_rope_cache(x[s], qn, kn, rope, pos[s].clone(), slots[s].clone(), many, EPS, interleaved)
        assert all(torch.equal(a, b) for a, b in zip(one, many) if a is not None)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,hq,hkv,d,r,interleaved", [(4099, 48, 6, 128, 128, False), (16387, 33, 7, 32, 16, True), (2051, 33, 7, 256, 64, False),
                                                      (3001, 61, 9, 160, 160, True)])
def test_backward(hip, t, hq, hkv, d, r, interleaved, kind):
    """Workgroups go round for further tokens and carry the weights' sums. Those have at most 4 heads x 16 rounds, 64 rows, and two
    sums of 64 in a row: under 2^8 - 2^5 additions and 2^5 roundings of a term, 2^-16 of the sum of the terms' magnitudes."""
    x, qn, kn, rope, pos, make = inputs(t, hq, hkv, d, r, kind)
    dy = [make(t, h, d) for h in (hq, hkv, hkv)]
    dw = torch.full((2, d + 32), 7.0, device="cuda")
    guard = torch.full((t + 2, hq + 2 * hkv, d), 7.0, dtype=x.dtype, device="cuda")
    got = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, interleaved, grads=(guard[1:-1], dw[0, :d], dw[1, :d]))
    assert (guard[0] == 7).all() and (guard[-1] == 7).all() and (dw[:, d:] == 7).all()
    again = hip.qk_norm_rope_bwd(x, qn, kn, rope, pos, *dy, EPS, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    short = [hip.qk_norm_rope_bwd(x[i:i + 64], qn, kn, rope, pos[i:i + 64].clone(), *[g[i:i + 64] for g in dy], EPS, interleaved)[0]
             for i in range(0, t, 64)]
    assert torch.equal(got[0], torch.cat(short))
    at, angles = sample(t), (np64(rope), pos.cpu().numpy())
    for w, g, lo, hi, dw in ((qn, dy[0], 0, hq, got[1]), (kn, dy[1], hq, hq + hkv, got[2])):
        dx, terms, _, _ = oh.norm_rope_bwd(np64(x[at, lo:hi]), np64(w), angles[0], pos[at].cpu().numpy(), np64(g[at]), EPS, interleaved)
        close(got[0][at, lo:hi], dx, terms, TYPES[kind], 2.0 ** -19)
        want = sums = 0.0
        for i in range(0, t, 512):  # (the whole in 64 bits at once would take gigabytes)
            _, _, a, b = oh.norm_rope_bwd(np64(x[i:i + 512, lo:hi]), np64(w), angles[0], angles[1][i:i + 512], np64(g[i:i + 512]), EPS, interleaved)
            want, sums = want + a, sums + b
        close(dw, want, sums, None, 2.0 ** -16)
    assert torch.equal(got[0][:, hq + hkv:], dy[2])


# ---- more workgroups than a launch takes ---------------------------------------------------

def same_in_parts(whole, part, t, step):
    """whole's tensors [t, ...] to the bit what part(slice) gives, `step` tokens at a time"""
    for i in range(0, t, step):
        s = slice(i, min(i + step, t))
        assert all(torch.equal(a[s], b) for a, b in zip(whole, part(s)))


def test_forward_past_a_launch(hip):
    """2^22 workgroups of three kinds of heads go round: 8 tokens each, and some more."""
    t, d = (2 ** 22 // 3) * 8 + 37, 136
    x, qn, kn, rope, pos, _ = inputs(t, 1, 1, d, 64, "bf16")
    out = [torch.full((t + 1, 1, d), 7.0, dtype=x.dtype, device="cuda") for _ in range(3)]
    got = hip.qk_norm_rope(x, qn, kn, rope, pos, 1, EPS, out=[b[:-1] for b in out])
    assert all((b[-1] == 7).all() for b in out)
    same_in_parts(got, lambda s: hip.qk_norm_rope(x[s], qn, kn, rope, pos[s].clone(), 1, EPS), t, 2 ** 20)
    del x, out, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", (16, 8))
def test_cache_past_a_launch(hip, bits):
    """2^22 windows of 16 tokens, and some more, in and out, from a place in a block and with tokens that have no slot."""
    t, d, page = 2 ** 26 + 37, 32, 2 ** 20
    pages = t // page + 2
    x, qn, kn, rope, pos, make = inputs(t, 1, 1, d, 16, "f16")
    slots = torch.arange(5, t + 5, dtype=torch.int32, device="cuda")
    slots[::1001] = -1
    live = (slots >= 0)[:, None, None]
    dt = torch.int8 if bits == 8 else torch.float16
    one, many = (hip.kv_cache(pages, 1, page, d, dt) for _ in range(2))
    q = hip.qk_norm_rope_cache(x, qn, kn, rope, pos, slots, one, EPS)
    same_in_parts((q,), lambda s: (hip.qk_norm_rope_cache(x[s], qn, kn, rope, pos[s].clone(), slots[s].clone(), many, EPS),), t, 2 ** 23 + 16)
    assert all(torch.equal(a, b) for a, b in zip(one, many) if a is not None)
    del x, q
    k, v = hip.kv_cache_read(one, slots)
    same_in_parts((k, v), lambda s: hip.kv_cache_read(one, slots[s].clone()), t, 2 ** 23 + 16)
    assert not ((k != 0) & ~live).any()
    for c in (one, many):
        for b in c:
            if b is not None:
                b.zero_()
    hip.kv_cache_write(k, v, slots, one)
    for i in range(0, t, 2 ** 23 + 16):
        s = slice(i, i + 2 ** 23 + 16)
        hip.kv_cache_write(k[s], v[s], slots[s].clone(), many)
    assert all(torch.equal(a, b) for a, b in zip(one, many) if a is not None)
    if bits == 16:
        back = hip.kv_cache_read(one, slots)
        assert torch.equal(back[0], k) and torch.equal(back[1], v)
        del back
    del k, v, one, many
    torch.cuda.empty_cache()
