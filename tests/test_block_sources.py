"""Rules of the decoder-block kernels that only their sources can show (no GPU)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onebitsparsemul_b200", "csrc")


def code_of(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", ["norm.cu", "rotary_append.cu", "cache_attend.cu", "cache_attend_sm100.cu"])
def test_kernels_that_start_early_have_no_read_only_loads(name):
    """A kernel that is launched before its predecessor is complete lives while the predecessor writes: nothing that it or a
    helper of its file reads may be promised to be constant."""
    code = code_of(name)
    kernels = re.split(r"(?=template <[^\n]*>\s*__global__|__global__)", code)
    early = [k for k in kernels if "__global__" in k and "follow_previous_kernel()" in k]
    assert early
    for k in early:
        assert not re.search(r"__ldg|ld\.global\.nc|__ldcs|__ldca|__restrict__", k)
    if all("follow_previous_kernel()" in k for k in kernels if "__global__" in k):      # then the helpers are theirs too
        assert not re.search(r"__ldg|ld\.global\.nc|__ldcs|__ldca|__restrict__", code)


@pytest.mark.parametrize("name", ["gemm_decode.cu", "gemm_decode_sm100.cu"])
def test_few_token_products_read_tokens_that_may_just_have_been_written(name):
    """They start before the norm that writes their tokens is complete."""
    code = code_of(name)
    assert "griddepcontrol.wait" in code and not re.search(r"__ldg|ld\.global\.nc|__ldcs|__ldca|__restrict__", code)
