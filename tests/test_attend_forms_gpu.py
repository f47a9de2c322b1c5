"""Forms of few-row attention that only some shapes take, each named by the kernels that the call launches, against the plain form."""
import re

import pytest
import torch

import onebitsparsemul_b200 as ob
from tests.kernels_of import kernels_of
from tests.test_block_ops_gpu import check_attend

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def forms(names):
    """few kernel: (row tiles, line); its join: whole CTAs per row; the prompt kernel."""
    found = set()
    for n in names:
        if m := re.search(r"ob_attend_few_kernelI\w+?Li(?:64|128)ELi(\d)ELb(\d)E", n):
            found.add(("few", int(m[1]), "line" if m[2] == "1" else "clusters"))
        elif m := re.search(r"ob_attend_combine_kernelI\w+?Li(?:64|128)ELb(\d)E", n):
            found.add("join by CTAs" if m[1] == "1" else "join by warps")
        else:
            assert "ob_attend_many_kernel" in n or "ob_attend_join_kernel" in n, n
            found.add("many" if "many" in n else "join of parts")
    return found


@pytest.mark.parametrize("new,kv,heads,kv_heads,dim,dtype,hint,want", [
    # one long sequence with few heads: many parts of a segment, a CTA joins a row
    ([1], [20000], 8, 2, 128, F16, 1, {("few", 1, "line"), "join by CTAs"}), ([2], [33333], 4, 1, 64, BF16, 2, {("few", 1, "line"), "join by CTAs"}),
    ([5], [24001], 16, 4, 64, F16, 5, {("few", 2, "line"), "join by CTAs"}),
    # drafted tokens of ragged sequences: two tiles of rows on the line
    ([4, 3, 4, 1, 0, 4, 2], [9000, 300, 5000, 77, 40, 4, 6400], 30, 10, 64, BF16, 4, {("few", 2, "line"), "join by warps"}),
    ([1] * 12, [6000, 1, 0, 900, 64, 65, 5999, 3000, 10, 4097, 2048, 128], 96, 8, 128, F16, 1, {("few", 2, "line"), "join by warps"}),
    # more rows than the bound says, on the line
    ([40, 1, 9], [20000, 18000, 300], 16, 8, 64, F16, 1, {("few", 1, "line"), "join by warps"}),
    # single tokens on the line beside a prompt in the prompt's kernel, whole and in parts
    ([1] * 39 + [200], [5000, 1, 4200, 90] + [100 + 40 * s for s in range(35)] + [700], 32, 8, 64, F16, 200, {("few", 1, "line"), "join by warps", "many"}),
    ([1] * 30 + [90, 1, 2, 40], [6000, 64, 5000] + [33 * s for s in range(27)] + [5000, 100, 4500, 40], 48, 4, 128, BF16, 90, {("few", 2, "line"), "join by warps", "many"})])
def test_forms(new, kv, heads, kv_heads, dim, dtype, hint, want, tmp_path):
    q, cache, batch, got = check_attend(new, kv, heads, kv_heads, dim, dtype, max_new=hint, seed=kv[0], pad=(1, 2))
    assert forms(kernels_of(lambda: ob.cache_attend(q, cache, batch), tmp_path)) - {"join of parts"} == want
    for _ in range(3):
        assert torch.equal(ob.cache_attend(q, cache, batch)[1:1 + sum(new)], got[1:1 + sum(new)])
