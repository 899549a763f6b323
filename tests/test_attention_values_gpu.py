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
@pytest.mark.parametrize("d", (32, 64, 96, 128, 160, 256))
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
