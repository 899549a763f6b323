"""Attention of one new token over a paged cache on the GPU against the float64 oracle.

Tolerances. A score is a sum of D products in fp32, off by 2^-20 of the sum of their magnitudes (at most 2^-24 an addition, 16
of them in a row), which the exponential turns into a relative error of each weight; the weights go to the second
product in two parts, off by 2^-16, and are summed in fp32. So a result is off by half a step of its type and
2 (2^-20 sum |q k| + 2^-16) of the weighted mean of |v|, and lse by 2 (2^-20 sum |q k| + 2^-18) / ln 2."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import layouts, torch_ops
from oracle import heads as oh

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def np64(t):
    return t.double().cpu().numpy()


class Case:
    """A cache with B sequences' tokens on pages in any order; what no sequence holds is NaN, infinities and pages that the
    cache does not have."""

    def __init__(self, lengths, hq, hkv, d, page, bits, kind, seed=0, spare=2, std=1.0):
        rng = np.random.default_rng([seed, len(lengths), d, page])
        self.dt, self.d, self.page, self.hkv, self.lengths = TYPES[kind], d, page, hkv, lengths
        per = [-(-n // page) for n in lengths]
        pages = sum(per) + spare
        order = rng.permutation(pages)
        table = np.full((len(lengths), max(per + [1]) + 1), 2 ** 31 - 1, np.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        make = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        shape = (pages, hkv, page, d)
        if bits == 16:
            raw = [(make(*shape) * std).to(self.dt) for _ in range(2)]
            scales = [None, None]
            self.k, self.v = (np64(t) for t in raw)
        else:
            raw = [(make(*shape) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
            scales = [torch.from_numpy(rng.uniform(0.01, 0.05, shape[:3]).astype(np.float32)) for _ in range(2)]
            self.k, self.v = (np64(t) * np64(s)[..., None] for t, s in zip(raw, scales))
        stale = np.ones((pages, page), bool)
        for b, n in enumerate(lengths):
            for i in range(per[b]):
                stale[table[b, i], :min(page, n - i * page)] = False
        bad = torch.from_numpy(stale)[:, None, :].expand(pages, hkv, page)
        for t, s in zip(raw, scales):
            if bits == 16:
                t[bad] = torch.tensor(float("nan")).to(self.dt)
                t[bad.logical_and(torch.arange(page) % 2 == 0)] = float("inf")
            else:
                t[bad] = 127
                s[bad] = float("nan")
        blocked = [layouts.keys_blocked(raw[0]), layouts.values_blocked(raw[1])]
        self.cache = tuple(t.cuda() for t in blocked) + tuple(None if s is None else s.cuda() for s in scales)
        self.host_table = table
        self.table = torch.from_numpy(table).cuda()
        self.len = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.q = make(len(lengths), hq, d).to(self.dt).cuda()

    def rows(self, b, h):
        n = self.lengths[b]
        pages = self.host_table[b, :-(-n // self.page)]
        return tuple(t[pages, h].reshape(-1, self.d)[:n] for t in (self.k, self.v))

    def check(self, out, lse, scale, only=None):
        g = self.q.shape[1] // self.hkv
        got, q = np64(out), np64(self.q)
        stats = None if lse is None else np64(lse)
        half, least = torch.finfo(self.dt).eps / 2, 2.0 ** -25 if self.dt is torch.float16 else 0.0
        for b in range(len(self.lengths)) if only is None else only:
            for h in range(self.hkv):
                want, wl, mean, dots = oh.attend(q[b, h * g:(h + 1) * g], *self.rows(b, h), scale)
                room = half * np.abs(want) + 2 * (2.0 ** -20 * dots + 2.0 ** -16)[:, None] * mean + least
                off = np.abs(got[b, h * g:(h + 1) * g] - want)
                assert (off <= room).all(), (b, h, off.max(), room[off > room][:3], int((~(off <= room)).sum()))
                if stats is not None:
                    s = stats[b, h * g:(h + 1) * g]
                    if self.lengths[b] == 0:
                        assert (s == -np.inf).all() and (got[b] == 0).all()
                    else:
                        room = 2 * (2.0 ** -20 * dots + 2.0 ** -18) / np.log(2) + 2.0 ** -23 * np.abs(wl)
                        assert (np.abs(s - wl) <= room).all(), (b, h, np.abs(s - wl).max())


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 300]
SHAPES = [(EDGES, 4, 4, 32, 16), (EDGES, 8, 2, 64, 16), (EDGES, 3, 1, 96, 32), (EDGES, 15, 3, 128, 48), (EDGES, 8, 8, 160, 16),
          (EDGES, 16, 1, 192, 64), (EDGES, 34, 2, 224, 32), (EDGES, 33, 1, 256, 128), (EDGES, 142, 2, 64, 16), ([2000, 0, 1, 777], 32, 4, 128, 32),
          ([5003], 8, 1, 128, 64), ([1], 1, 1, 32, 16), ([0], 2, 2, 64, 16), ([9001, 8, 4096], 6, 3, 64, 16)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("lengths,hq,hkv,d,page", SHAPES)
def test_lengths_and_heads(hip, lengths, hq, hkv, d, page, bits, kind):
    c = Case(lengths, hq, hkv, d, page, bits, kind)
    for scale in (d ** -0.5, -0.3):
        out, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, scale, want_lse=True)
        c.check(out, lse, scale)
        again, none = hip.paged_attention(c.q, c.cache, c.table, c.len, scale)
        assert none is None and torch.equal(again, out)
        wide = torch.nn.functional.pad(c.table, (0, 1 + 5000 // page), value=-7)  # room for long sequences: split calls
        out, lse = hip.paged_attention(c.q, c.cache, wide, c.len, scale, want_lse=True)
        c.check(out, lse, scale)
        assert torch.equal(hip.paged_attention(c.q, c.cache, wide, c.len, scale)[0], out)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("b", (1, 3, 70, 300))
def test_batches(hip, b, bits, kind):
    """Ragged batches from one sequence to several hundred, some of them empty."""
    rng = np.random.default_rng(b)
    lengths = [int(n) for n in np.exp(rng.uniform(0, np.log(3000 if b < 100 else 400), b))]
    for i in range(3, b, 7):
        lengths[i] = 0
    c = Case(lengths, 8, 2, 64, 32, bits, kind, seed=b)
    out, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True)
    c.check(out, lse, 64 ** -0.5)


@pytest.mark.parametrize("bits", (16, 8))
def test_many_short_sequences(hip, bits):
    lengths = [i % 5 for i in range(4100)]
    c = Case(lengths, 2, 1, 32, 16, bits, "f16")
    for table in (c.table, torch.nn.functional.pad(c.table, (0, 40), value=-1)):
        out, lse = hip.paged_attention(c.q, c.cache, table, c.len, want_lse=True)
        c.check(out, lse, 32 ** -0.5, only=list(range(0, 4100, 37)) + [4099])


@pytest.mark.parametrize("b,longest,hq,hkv", ((256, 900, 4, 1), (257, 900, 4, 1), (513, 700, 40, 2), (1100, 1200, 3, 3), (700, 30, 2, 1)))
def test_large_ragged_batches(hip, b, longest, hq, hkv):
    """Batches past what a workgroup looks through by itself: a few long sequences in parts among short and empty ones, one that
    says more tokens than its pages hold, and more items than the chip takes at once."""
    rng = np.random.default_rng(b)
    lengths = [int(n) for n in np.exp(rng.uniform(0, np.log(40), b))]
    for i in range(0, b, 5):
        lengths[i] = 0
    for i in (1, 2, b // 2, b - 2, b - 1):
        lengths[i] = longest
    c = Case(lengths, hq, hkv, 32, 16, 8, "f16", seed=b)
    table = torch.nn.functional.pad(c.table, (0, 40), value=-1)
    c.len[3] = table.shape[1] * 16 + 1
    out, lse = hip.paged_attention(c.q, c.cache, table, c.len, want_lse=True)
    assert out[3].isnan().all() and lse[3].isnan().all()
    c.check(out, lse, 32 ** -0.5, only=[i for i in range(b) if i != 3 and (i % 9 == 0 or lengths[i] == longest)])
    again, _ = hip.paged_attention(c.q, c.cache, table, c.len)
    assert torch.equal(again.nan_to_num(7), out.nan_to_num(7))


@pytest.mark.parametrize("kind", TYPES)
def test_large_and_peaked_scores(hip, kind):
    """Scores of some hundreds: one token has all the weight, and the running maximum moves often."""
    c = Case([1000, 77], 8, 2, 128, 16, 16, kind, std=6.0)
    c.q *= 4
    out, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, 0.5, want_lse=True)
    c.check(out, lse, 0.5)


def test_many_small_weights(hip):
    """One token far ahead of 60000 alike: each of the others weighs 2^-18, together a fifth of the result."""
    n, d = 60001, 64
    cache = hip.kv_cache(n // 64 + 1, 1, 64, d, torch.float16)
    k = torch.zeros((n, 1, d), dtype=torch.float16, device="cuda")
    k[12345, 0, 0] = 18 * float(np.log(2))
    v = torch.ones((n, 1, d), dtype=torch.float16, device="cuda")
    v[12345] = -1
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    hip.kv_cache_write(k, v, slots, cache)
    q = torch.zeros((1, 1, d), dtype=torch.float16, device="cuda")
    q[..., 0] = 1
    table = torch.arange(n // 64 + 1, dtype=torch.int32, device="cuda")[None]
    out, _ = hip.paged_attention(q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    w = (n - 1) * np.exp(-float(k[12345, 0, 0]))
    assert (np.abs(np64(out) - (w - 1) / (w + 1)) <= 2.0 ** -11).all()


@pytest.mark.parametrize("bits", (16, 8))
def test_huge_values(hip, bits):
    """bf16 values near the type's largest do not overflow on their way to a mean."""
    c = Case([700, 40], 4, 2, 64, 16, bits, "bf16")
    big = 2.0 ** 120
    if bits == 16:
        v = c.cache[1] * big
        c.cache = (c.cache[0], v, None, None)
    else:
        c.cache = c.cache[:3] + (c.cache[3] * big,)
    c.v = c.v * big
    out, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True)
    assert torch.isfinite(out).all()
    c.check(out, lse, 64 ** -0.5)


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("lengths", ([40, 100, 33, 5], [4000, 100, 2000, 5]))
def test_bad_pages_and_lengths(hip, lengths, bits):
    """A page that the cache does not have, or a length past the table, makes a sequence NaN and no other."""
    c = Case(lengths, 4, 2, 64, 16, bits, "f16")
    good, _ = hip.paged_attention(c.q, c.cache, c.table, c.len)
    c.check(good, None, 64 ** -0.5)
    for bad in (-1, c.cache[0].shape[0], 2 ** 31 - 1, -2 ** 31):
        for b, i in ((1, 0), (1, 6), (0, 2)):
            t = c.table.clone()
            t[b, i] = bad
            out, lse = hip.paged_attention(c.q, c.cache, t, c.len, want_lse=True)
            assert torch.isnan(out[b]).all() and torch.isnan(lse[b]).all()
            rest = [x for x in range(4) if x != b]
            c.check(out, None, 64 ** -0.5, only=rest)
    n = c.len.clone()
    n[2] = c.table.shape[1] * 16 + 1
    n[3] = -5
    out, lse = hip.paged_attention(c.q, c.cache, c.table, n, want_lse=True)
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all() and (out[3] == 0).all() and (lse[3] == -float("inf")).all()
    c.check(out, None, 64 ** -0.5, only=[0, 1])
    n[2] = 2 ** 31 - 1
    assert torch.isnan(hip.paged_attention(c.q, c.cache, c.table, n)[0][2]).all()


def test_values_that_are_not_finite(hip):
    """An infinity or NaN among a sequence's own tokens is seen, and stays with its head of keys and, in values, its channel."""
    c = Case([50, 20], 4, 2, 64, 16, 16, "f16")
    v = layouts.values_unblocked(c.cache[1])
    v[c.host_table[0, 1], 0, 3, 7] = float("nan")
    v[c.host_table[0, 0], 1, 3, 9] = float("inf")
    k = layouts.keys_unblocked(c.cache[0])
    k[c.host_table[1, 0], 1, 4] = float("nan")
    out, _ = hip.paged_attention(c.q, (layouts.keys_blocked(k), layouts.values_blocked(v), None, None), c.table, c.len)
    nan = torch.isnan(out)
    assert nan[0, :2, 7].all() and int(nan[0].sum()) == 2 and (out[0, 2:, 9] == float("inf")).all()
    assert nan[1, 2:].all() and not nan[1, :2].any()


@pytest.mark.parametrize("b,longest", ((1, 60), (5, 3000)))
def test_nothing_outside_is_written(hip, b, longest):
    c = Case([longest] + [7] * (b - 1), 6, 2, 96, 16, 16, "f16")
    out = torch.full((b + 2, 6, 96), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((b + 2, 6), 7.0, device="cuda")
    need = hip.paged_attention_workspace(c.q, c.cache, c.table)
    ws = torch.full((need + 512,), 77, dtype=torch.uint8, device="cuda")
    hip.paged_attention(c.q, c.cache, c.table, c.len, out=out[1:-1], lse=lse[1:-1], workspace=ws[:need] if need else ws)
    c.check(out[1:-1], lse[1:-1], 96 ** -0.5)
    assert (out[[0, -1]] == 7).all() and (lse[[0, -1]] == 7).all() and (ws[need:] == 77).all()


def test_offsets_past_2_31(hip):
    """Sequences on the last pages of a cache of more than 2^32 bytes."""
    pages, hkv, page, d = 33000, 4, 128, 128
    for dt in (torch.float16, torch.int8):
        cache = hip.kv_cache(pages, hkv, page, d, dt)
        rng = np.random.default_rng(3)
        k, v = (torch.from_numpy(rng.standard_normal((300, hkv, d)).astype(np.float32)).half().cuda() for _ in range(2))
        table = torch.tensor([[pages - 1, 16384, pages - 2]], dtype=torch.int32, device="cuda")
        slots = torch_ops.cache_slots(table, torch.arange(300, device="cuda")[None], page)
        torch_ops.kv_cache_write(k[None], v[None], slots, cache)
        q = torch.from_numpy(rng.standard_normal((1, 8, d)).astype(np.float32)).half().cuda()
        out = torch_ops.paged_attention(q, cache, table, torch.tensor([300], dtype=torch.int32, device="cuda"))
        rk, rv = torch_ops.kv_cache_read(cache, slots, torch.float16)
        for h in range(hkv):
            want, _, mean, dots = oh.attend(np64(q)[0, 2 * h:2 * h + 2], np64(rk)[0, :, h], np64(rv)[0, :, h], d ** -0.5)
            # (what is read back of 8 bits is rounded to fp16: 2^-11 of each product and value)
            more = 0.0 if dt is torch.float16 else 2.0 ** -11
            room = 2.0 ** -11 * np.abs(want) + (2 * ((2.0 ** -20 + more) * dots + 2.0 ** -16) + more)[:, None] * mean
            assert (np.abs(np64(out)[0, 2 * h:2 * h + 2] - want) <= room).all()
        del cache


def test_on_another_stream_and_two_at_once(hip):
    """Calls on two streams at once, each with a workspace of its own."""
    cases = [Case([3000, 40, 777], 8, 2, 128, 32, bits, "bf16", seed=bits) for bits in (16, 8)]
    want = [hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.parametrize("bits", (16, 8))
def test_captured_decode_loop(hip, bits):
    """Lengths and pages change between a graph's replays, as in a decode loop, with eager calls in between."""
    c = Case([2000, 900, 1, 0], 8, 2, 64, 16, bits, "f16")
    ws = torch.empty(max(1, hip.paged_attention_workspace(c.q, c.cache, c.table)), dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(c.q), torch.empty((4, 8), device="cuda")
    hip.paged_attention(c.q, c.cache, c.table, c.len, out=out, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hip.paged_attention(c.q, c.cache, c.table, c.len, out=out, lse=lse, workspace=ws)
    for lengths in ([2000, 900, 1, 0], [1, 0, 1, 0], [1999, 17, 0, 0], [0, 0, 0, 0], [64, 899, 1, 0]):
        c.len.copy_(torch.tensor(lengths, dtype=torch.int32))
        c.lengths = lengths
        out.fill_(7)
        lse.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        c.check(out, lse, 64 ** -0.5)
        eager = hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True)
        assert torch.equal(eager[0], out) and torch.equal(eager[1], lse)


def test_captured_large_batch(hip):
    """The same for a batch whose items a launch deals out: two graphs that share a workspace, replayed one after the other, an
    eager call with another between them."""
    b, room = 300, 640
    c = Case([room] * 2 + [1 + i % 40 for i in range(b - 2)], 4, 2, 32, 16, 16, "bf16")
    table = torch.nn.functional.pad(c.table, (0, 5), value=-1)
    ws = torch.empty(hip.paged_attention_workspace(c.q, c.cache, table), dtype=torch.uint8, device="cuda")
    lens = [c.len.clone(), c.len.clone()]
    outs = [torch.empty_like(c.q) for _ in lens]
    for n, out in zip(lens, outs):
        hip.paged_attention(c.q, c.cache, table, n, out=out, workspace=ws)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in lens]
    for g, n, out in zip(graphs, lens, outs):
        with torch.cuda.graph(g):
            hip.paged_attention(c.q, c.cache, table, n, out=out, workspace=ws)
    for seed in range(4):
        gen = torch.Generator().manual_seed(seed)
        for i, n in enumerate(lens):
            share = torch.rand(b, generator=gen) if seed else torch.zeros(b)
            n.copy_((c.len.cpu() * share).int())
            outs[i].fill_(7)
        for i, g in enumerate(graphs):
            g.replay()
            hip.paged_attention(c.q, c.cache, table, c.len)
        torch.cuda.synchronize()
        for n, out in zip(lens, outs):
            assert torch.equal(out, hip.paged_attention(c.q, c.cache, table, n)[0])
            assert (out[n == 0] == 0).all()


@pytest.mark.parametrize("bits", (16, 8))
def test_pages_that_sequences_share(hip, bits):
    """Sequences with the same first pages, one page twice in a sequence, and the same sequence in every row."""
    c = Case([200, 90, 33], 6, 2, 64, 16, bits, "f16")
    c.host_table[1, :3] = c.host_table[0, :3]
    c.host_table[2, :3] = c.host_table[0, [4, 4, 0]]
    table = torch.from_numpy(c.host_table).cuda()
    out, lse = hip.paged_attention(c.q, c.cache, table, c.len, want_lse=True)
    c.check(out, lse, 64 ** -0.5)
    q, rows = c.q[:1].expand(100, 6, 64).contiguous(), table[:1].expand(100, -1).contiguous()
    same, _ = hip.paged_attention(q, c.cache, torch.nn.functional.pad(rows, (0, 60), value=-1), c.len[:1].expand(100).contiguous())
    assert (same == same[:1]).all()


@pytest.mark.parametrize("bits", (16, 8))
def test_a_serving_block(hip, bits):
    """A prompt and then tokens one by one through an attention block of 8-bit projections: norm to 8 bits, one projection for
    all heads, heads' norm with rotation into the cache, attention, output projection with the residual; each step
    against the whole sequence's attention in float64 on what the projections gave."""
    rng = np.random.default_rng(11)
    b, hq, hkv, d, c, page, eps = 3, 8, 2, 64, 256, 16, 1e-6
    dt = torch.bfloat16
    make = lambda *s, std=1.0: (torch.from_numpy(rng.standard_normal(s).astype(np.float32)) * std).cuda()  # noqa: E731
    scale = 1 + 0.1 * make(c)
    qn, kn = 1 + 0.1 * make(d), 1 + 0.1 * make(d)
    wqkv = torch_ops.q8_weights(make(c, (hq + 2 * hkv) * d, std=c ** -0.5).half())
    wo = torch_ops.q8_weights(make(hq * d, c, std=(hq * d) ** -0.5).half())
    rope = layouts.rope_table(256, d, device="cuda")
    cache = hip.kv_cache(40, hkv, page, d, torch.int8 if bits == 8 else dt)
    table = torch.from_numpy(rng.permutation(40)[:33].reshape(b, 11).astype(np.int32)).cuda()
    prompt = torch.tensor([37, 16, 1])
    seen = [[] for _ in range(b)]

    def heads(x):
        q8, qs, s = torch_ops.rms_norm_q8(x, scale, torch.zeros_like(x), eps)
        return torch_ops.q8_projection(q8, qs, wqkv, dtype=dt).reshape(x.shape[:-1] + (hq + 2 * hkv, d)), s

    # the prompts, padded to the longest: rows past a prompt's end have position -1 and so no slot
    x = make(b, 37, c).to(dt)
    at = torch.arange(37)[None].expand(b, 37)
    at = torch.where(at < prompt[:, None], at, torch.full_like(at, -1)).cuda()
    qkv, _ = heads(x)
    torch_ops.qk_norm_rope_cache(qkv, qn, kn, rope, at.clamp(min=0).int(), torch_ops.cache_slots(table, at, page), cache, eps)
    for i in range(b):
        seen[i] += [qkv[i, t] for t in range(int(prompt[i]))]
    for step in range(4):
        x = make(b, c).to(dt)
        qkv, s = heads(x)
        pos = (prompt + step).cuda()
        q = torch_ops.qk_norm_rope_cache(qkv, qn, kn, rope, pos.int(), torch_ops.cache_slots(table, pos, page), cache, eps)
        o = torch_ops.paged_attention(q, cache, table, (pos + 1).int())
        out = torch_ops.q8_projection(*torch_ops.quantize_rows(o.reshape(b, hq * d)), wo, residual=s)
        assert out.shape == (b, c) and torch.isfinite(out).all()
        for i in range(b):
            seen[i].append(qkv[i])
            rows = np64(torch.stack(seen[i]))
            n = np.arange(len(rows))
            wq = oh.norm_rope(rows[-1:, :hq], np64(qn), np64(rope), n[-1:], eps, False)[0][0]
            wk = oh.norm_rope(rows[:, hq:hq + hkv], np64(kn), np64(rope), n, eps, False)[0]
            for h in range(hkv):
                k, v = wk[:, h], rows[:, hq + hkv + h]
                want, _, mean, dots = oh.attend(wq[4 * h:4 * h + 4], k, v, d ** -0.5)
                # queries and keys are off by half a step of theirs, of 2^-8 of the type or of 1 / 254 of a head's largest
                grid = 2.0 ** -9 if bits == 16 else 1 / 254
                dk = grid * (np.abs(k) if bits == 16 else np.abs(k).max(-1, keepdims=True))
                dv = 0.0 if bits == 16 else grid * np.abs(v).max()
                ds = (2.0 ** -9 * dots + (np.abs(wq[4 * h:4 * h + 4]) @ dk.repeat(1 if dk.shape[1] == d else d, 1).T).max(1) * d ** -0.5)
                room = 2.0 ** -9 * np.abs(want) + (np.expm1(2.02 * ds) + 2.0 ** -15)[:, None] * mean + dv
                assert (np.abs(np64(o)[i, 4 * h:4 * h + 4] - want) <= room).all()
