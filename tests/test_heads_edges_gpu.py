"""Heads' norm and rotation, and the cache, at the edges of their arguments, on the GPU. Tolerances are those of the operators'
other tests."""
import pytest
import torch

from colabfold_legacy_kernels import layouts

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("eps", (1e-30, 1e-40, 1e-45))
def test_zeros_with_a_tiny_eps(hip, eps, kind):
    """A head of zeros is zeros with every eps above 0, normal or not, and so is its share of the weights' gradients; others
    are as without one."""
    dt, t, d = TYPES[kind], 5, 64
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((t, 4, d), generator=gen).to(dt)
    x[[1, 3]] = 0
    w, rope = 1 + 0.1 * torch.randn(d, generator=gen), layouts.rope_table(9, d)
    args = [v.cuda() for v in (x, w, w, rope, torch.arange(t, dtype=torch.int32))]
    live = [0, 2, 4]
    some = [args[0][live].contiguous()] + args[1:4] + [args[4][live].contiguous()]
    out = hip.qk_norm_rope(*args, 1, eps)
    assert all((a[[1, 3]] == 0).all() for a in out)
    assert all(torch.equal(a[live], b) for a, b in zip(out, hip.qk_norm_rope(*some, 1, 0.0)))
    dy = [torch.randn((t, h, d), generator=gen).to(dt).cuda() for h in (2, 1, 1)]
    for g in dy:
        g[[1, 3]] = 0  # (another gradient is multiplied by 1 / sqrt(eps), which is past fp16's range)
    dx, dq, dk = hip.qk_norm_rope_bwd(*args, *dy, eps)
    want = hip.qk_norm_rope_bwd(*some, *[g[live].contiguous() for g in dy], 0.0)
    assert (dx[[1, 3]] == 0).all() and torch.equal(dx[live], want[0]) and torch.equal(dq, want[1]) and torch.equal(dk, want[2])
