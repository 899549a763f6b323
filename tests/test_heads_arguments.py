"""Arguments of the heads' and the cache's Python entry points that contradict one another are refused, on the CPU."""
import pytest
import torch

from colabfold_legacy_kernels import hip as H
from colabfold_legacy_kernels import layouts, torch_ops


def test_results_of_other_heads_than_said():
    """Results given for 1 key head and for 3, where 2 are said: taken for what they are, they would be other heads' values."""
    x, w, rope = torch.zeros((4, 8, 64), dtype=torch.float16), torch.ones(64), layouts.rope_table(10, 64)
    pos = torch.zeros(4, dtype=torch.int32)
    for n in (1, 3):
        out = [torch.zeros((4, heads, 64), dtype=torch.float16) for heads in (8 - 2 * n, n, n)]
        with pytest.raises(H.InvalidArgument, match="out has %d key heads, not 2" % n):
            H.qk_norm_rope(x, w, w, rope, pos, 2, out=out)
        with pytest.raises(H.InvalidArgument, match="must be on one GPU"):
            H.qk_norm_rope(x, w, w, rope, pos, n, out=out)


def test_slots_that_tokens_would_share():
    """Slots of one sequence for a batch of two would have each token overwrite the other's; a leading dimension of 1 shares none."""
    x, w, rope = torch.zeros((2, 5, 8, 64), dtype=torch.float16), torch.ones(64), layouts.rope_table(10, 64)
    pos = torch.arange(5, dtype=torch.int32)
    c = H.kv_cache(3, 2, 16, 64, torch.float16, device="cpu")
    k = x[:, :, :2]
    for slots in (pos, pos[None], pos[:1], pos[0], pos[:2, None]):
        for call in (lambda x, k: torch_ops.qk_norm_rope_cache(x, w, w, rope, pos, slots, c), lambda x, k: torch_ops.kv_cache_write(k, k, slots, c)):
            with pytest.raises(H.InvalidArgument, match="slots must be of the tokens' shape"):
                call(x, k)
    for call in (lambda x, k: torch_ops.qk_norm_rope_cache(x, w, w, rope, pos, pos, c), lambda x, k: torch_ops.kv_cache_write(k, k, pos, c)):
        with pytest.raises(H.InvalidArgument, match="must be on one GPU"):
            call(x[:1], k[:1])
