"""Attention over a paged cache where values or weights stand at the edge of their type, on the GPU against the float64
definition. Tolerances that are not stated here are those of the attention's other tests."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import layouts
from oracle import heads as oh

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def np64(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("room", (512, 4096))
@pytest.mark.parametrize("d", (32, 64, 96, 128, 160, 192, 224, 256))
@pytest.mark.parametrize("n", (3, 40, 500))
def test_infinities_with_small_weights(hip, n, d, room, kind):
    """A positive weight times an infinite value is that infinity, however small the weight is against the largest (2^-90 here):
    scores are the keys' first channels, the token ahead has 0, one has -gap, all others -1000 (no weight)."""
    dt = TYPES[kind]
    gaps = (2, 15, 26, 27, 28, 40, 62)
    page, b = 16, len(gaps)
    pages = -(-n // page)
    k = torch.zeros((b * pages, 1, page, d))
    v = torch.zeros((b * pages, 1, page, d))
    rows_k, rows_v = k.view(b, pages * page, d), v.view(b, pages * page, d)
    rows_k[:, :, 0] = -1000.0
    rows_v[:, :] = torch.randn(rows_v.shape, generator=torch.Generator().manual_seed(n + d))
    for i, gap in enumerate(gaps):
        ahead, inf = (i, n - 1) if i % 2 else (n - 1, 0)
        rows_k[i, ahead, 0], rows_k[i, inf, 0] = 0.0, -float(gap)
        rows_v[i, inf, 5], rows_v[i, inf, d - 2] = float("inf"), -float("inf")
    q = torch.zeros((b, 3, d))
    q[..., 0] = 1.0
    table = torch.arange(b * pages, dtype=torch.int32).view(b, pages)
    table = torch.nn.functional.pad(table, (0, room // page - pages), value=-1).cuda()
    lengths = torch.full((b,), n, dtype=torch.int32, device="cuda")
    cache = (layouts.keys_blocked(k.to(dt).cuda()), layouts.values_blocked(v.to(dt).cuda()), None, None)
    out, _ = hip.paged_attention(q.to(dt).cuda(), cache, table, lengths, 1.0)
    assert (out[:, :, 5] == float("inf")).all() and (out[:, :, d - 2] == -float("inf")).all()
    other = [c for c in range(d) if c not in (5, d - 2)]
    for i in range(b):
        want, _, mean, dots = oh.attend(np64(q[i]), np64(rows_k[i, :n].to(dt)), np64(rows_v[i, :n].to(dt))[:, other].copy(), 1.0)
        # (the scores are exact: the weights' parts are all that is rounded, and the result; fp16's steps end at 2^-24)
        room_ = torch.finfo(dt).eps / 2 * np.abs(want) + 2.0 ** -14 * mean + (2.0 ** -25 if dt is torch.float16 else 0.0)
        assert (np.abs(np64(out[i])[:, other] - want) <= room_).all()


@pytest.mark.parametrize("room", (1024, 8192))
@pytest.mark.parametrize("d", (64, 128))
@pytest.mark.parametrize("bits", (16, 8))
def test_tiny_values(hip, bits, d, room):
    """bf16 values of 2^-118, or 8-bit rows with scales of 2^-107, are normal numbers of their types, and their mean is one.

    A weight times 2^-10 (700 tokens) and such a scale is 2^-117 and less, in two parts whose steps end at 2^-133; a product with
    a value of 2^-118 is 2^-128 and less, whose steps in fp32 end at 2^-149, as the sums' do. The result's own steps
    end at 2^-133."""
    lengths, page, heads = [700, 1, 40], 16, 2
    gen = torch.Generator().manual_seed(bits + d)
    pages = -(-max(lengths) // page)
    shape = (3 * pages, heads, page, d)
    k = torch.randn(shape, generator=gen).to(torch.bfloat16)
    if bits == 16:
        v = (torch.randn(shape, generator=gen) * 2.0 ** -118).to(torch.bfloat16)
        scales = (None, None)
        v64, k64 = np64(v), np64(k)
    else:
        k, v = ((torch.randn(shape, generator=gen) * 40).round().clamp(-127, 127).to(torch.int8) for _ in range(2))
        ks, vs = torch.rand(shape[:3], generator=gen) * 0.02 + 0.02, (torch.rand(shape[:3], generator=gen) + 1) * 2.0 ** -108
        scales = (ks.cuda(), vs.cuda())
        k64, v64 = np64(k) * np64(ks)[..., None], np64(v) * np64(vs)[..., None]
    q = torch.randn((3, 4, d), generator=gen).to(torch.bfloat16)
    table = torch.nn.functional.pad(torch.arange(3 * pages, dtype=torch.int32).view(3, pages), (0, room // page - pages), value=-1)
    cache = (layouts.keys_blocked(k).cuda(), layouts.values_blocked(v).cuda()) + scales
    out, lse = hip.paged_attention(q.cuda(), cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), want_lse=True)
    out, lse = np64(out), np64(lse)
    for i, n in enumerate(lengths):
        rows_k, rows_v = (t[i * pages:(i + 1) * pages].transpose(0, 2, 1, 3).reshape(-1, heads, d)[:n] for t in (k64, v64))
        for h in range(heads):
            want, wl, mean, dots = oh.attend(np64(q)[i, 2 * h:2 * h + 2], rows_k[:, h], rows_v[:, h], d ** -0.5)
            x = np64(q)[i, 2 * h:2 * h + 2] @ rows_k[:, h].T * d ** -0.5
            total = np.exp(x - x.max(1, keepdims=True)).sum(1) * 2.0 ** -n.bit_length()  # of the weights, as they are held
            # what the ends of the steps cost: of weights, 2^-134 each times the integers; of products' sums, 2^-149 each
            steps = 2.0 ** -134 * 127 * n if bits == 8 else 2.0 ** -149 * n
            room_ = 2.0 ** -8 * np.abs(want) + 2 * (2.0 ** -20 * dots + 2.0 ** -16)[:, None] * mean + (steps / total)[:, None] + 2.0 ** -134
            assert (np.abs(out[i, 2 * h:2 * h + 2] - want) <= room_).all()
            room_ = 2 * (2.0 ** -20 * dots + 2.0 ** -18) / np.log(2) + 2.0 ** -23 * np.abs(wl)
            assert (np.abs(lse[i, 2 * h:2 * h + 2] - wl) <= room_).all()


def test_the_largest_values(hip):
    """The mean of bf16's largest value over many tokens is that value."""
    n, page, d = 5000, 16, 32
    big = torch.finfo(torch.bfloat16).max
    k = torch.zeros((-(-n // page), 1, page, d), dtype=torch.bfloat16, device="cuda")
    v = torch.full_like(k, big)
    table = torch.arange(len(k), dtype=torch.int32, device="cuda")[None]
    q = torch.ones((1, 2, d), dtype=torch.bfloat16, device="cuda")
    out, _ = hip.paged_attention(q, (k, v, None, None), table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    assert (out == big).all()
