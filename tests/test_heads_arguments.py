"""Arguments of the heads' and the cache's Python entry points that contradict one another are refused, on the CPU."""
import pytest
import torch

from colabfold_legacy_kernels import hip as H
from colabfold_legacy_kernels import layouts


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
