"""A rule of the serving kernels that no result shows reliably: they are launched early, so what
they read may still be written when they start, and read-only loads are not theirs to use."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustgears_b200", "csrc")
EARLY = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu") and "launch_early(" in open(os.path.join(CSRC, f)).read())


def test_the_kernels_are_found():
    assert {"k_attn_paged.cu", "k_attn_tc.cu", "k_linear_token.cu", "k_rope.cu"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY + ["rg_serving.h", "rg_mma16.cuh", "rg_sm100_pair.cuh"])
def test_early_kernels_load_plainly(name):
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(os.path.join(CSRC, name)).read(), flags=re.S)
    found = re.findall(r"__ldg\b|__restrict__|ld\.global\.nc", code)
    assert not found, f"{name}: {sorted(set(found))}"
