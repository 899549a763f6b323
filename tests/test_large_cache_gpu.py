"""Attention over caches that are read past the caches of the chip (keys and values of 128 MiB and more together), and past 2^31
values, with parts that are joined, on the GPU: where a cache's bytes lie changes no result."""
import numpy as np
import pytest
import torch

from test_paged_attention_gpu import TYPES, Case

pytestmark = pytest.mark.gpu


def spread(c, pages, seed):
    """The case's pages at places of a cache of `pages` pages, the last and the first among them: (cache, table)."""
    n = c.cache[0].shape[0]
    rest = torch.randperm(pages - 2, generator=torch.Generator().manual_seed(seed))[:n - 2] + 1
    where = torch.cat([torch.tensor([pages - 1, 0]), rest])[:n].cuda()
    cache = []
    for t in c.cache:
        if t is None:
            cache.append(None)
            continue
        big = torch.zeros((pages,) + t.shape[1:], dtype=t.dtype, device="cuda")
        big[where] = t
        cache.append(big)
    table = c.table.long()
    known = (table >= 0) & (table < n)
    return tuple(cache), torch.where(known, where[table.clamp(0, n - 1)], table).to(torch.int32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("d", (64, 96, 128, 256))
@pytest.mark.parametrize("hq", (12, 80))
def test_caches_around_the_limit(hip, hq, d, bits, kind):
    """The same pages in caches just under and just over 128 MiB, with room for long sequences: 3 query heads a head of keys,
    and 20, which stay with the chip's caches. Then a batch that a launch deals out."""
    hkv, page = 4, 64
    size = 2 * hkv * page * d * (2 if bits == 16 else 1)
    at = -(-2 ** 27 // size)  # pages of 128 MiB
    lengths = [3000, 0, 1, 777, 64, 5000]
    if hq == 12 and d == 64:
        lengths = lengths + [i % 90 for i in range(200)]
    c = Case(lengths, hq, hkv, d, page, bits, kind)
    small, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True)
    c.check(small, lse, d ** -0.5, only=list(range(6)) + list(range(6, len(lengths), 17)))
    for pages in (at - 1, at, at + 9):
        cache, table = spread(c, pages, pages)
        out, other = hip.paged_attention(c.q, cache, table, c.len, want_lse=True)
        assert torch.equal(out, small) and torch.equal(other, lse)
        assert torch.equal(hip.paged_attention(c.q, cache, table, c.len)[0], small)
        del cache


@pytest.mark.parametrize("bits", (16, 8))
@pytest.mark.parametrize("hq", (8, 72))
def test_parts_past_2_31(hip, hq, bits):
    """Sequences of several thousand tokens on pages all over a cache of more than 2^32 bytes, read in parts."""
    c = Case([4000, 129, 6001], hq, 4, 128, 128, bits, "f16")
    want, lse = hip.paged_attention(c.q, c.cache, c.table, c.len, want_lse=True)
    c.check(want, lse, 128 ** -0.5)
    cache, table = spread(c, 33000, 1)
    assert cache[0].numel() > 2 ** 31 and int(table.max()) >= 32999
    out, other = hip.paged_attention(c.q, cache, table, c.len, want_lse=True)
    assert torch.equal(out, want) and torch.equal(other, lse)
    del cache
    torch.cuda.empty_cache()


def test_bad_pages_in_a_large_cache(hip):
    """A page that a large cache does not have, just behind its last, is not read."""
    c = Case([3000, 700], 8, 4, 128, 64, 8, "bf16")
    cache, table = spread(c, 2100, 2)
    good, _ = hip.paged_attention(c.q, cache, table, c.len)
    table[0, 30] = 2100
    out, _ = hip.paged_attention(c.q, cache, table, c.len)
    assert torch.isnan(out[0]).all() and torch.equal(out[1], good[1]) and np.isfinite(good.float().cpu().numpy()).all()
