"""The kernels' sources keep the rule that bf16 results are never put into half-precision vectors value by value: the compiler may
pack those with an instruction that quiets fp16's signalling NaNs, which as bf16 are values past 2^121. No kernel runs here."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "colabfold-legacy-kernels_amd", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".hip", ".h")))


@pytest.mark.parametrize("name", SOURCES)
def test_no_raw_pattern_in_a_half_vector(name):
    """A raw pattern (act_cvt) is stored to memory by itself, a.<array>[...], and goes nowhere else."""
    with open(os.path.join(CSRC, name)) as f:
        lines = f.read().split("\n")
    bad = [(i + 1, l.strip()) for i, l in enumerate(lines) if re.search(r"\bact_cvt<", l) and "act_cvt(float v)" not in l
           and not re.search(r"\ba\.\w+\[[^=]*\] = act_cvt<", l)]
    assert not bad, bad
