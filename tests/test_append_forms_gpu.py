"""The two append kernels: which sequences each gets, and both against the definition."""
import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib
from tests import block_plain as plain
from tests.kernels_of import kernels_of
from tests.test_block_ops_gpu import equal_pages, gen, i32, paged, starts

pytestmark = pytest.mark.gpu
F16, BF16, DEV = torch.float16, torch.bfloat16, "cuda"


def forms(names):
    assert all("ob_cache_append" in n for n in names), names
    return sorted("warps" if "append_few" in n else "pages" for n in names)


@pytest.mark.parametrize("new,hint,want", [
    ([1] * 64, 1, ["warps"]), ([2] * 9, 2, ["warps"]), ([3, 0, 1], 3, ["warps"]), ([1], None, ["warps"]), ([4], 4, ["pages"]), ([4] * 9, 4, ["pages"]),
    ([100] + [0] * 63, 100, ["pages", "warps"]), ([1] * 255 + [200], 200, ["pages", "warps"]), ([1] * 64, None, ["pages", "warps"]), ([1] * 64 + [512], 512, ["pages"]),
    ([100, 40], None, ["pages"])])
def test_a_page_of_many_tokens_is_no_single_warp_s(new, hint, want, tmp_path):
    """One long range among many single tokens went to the kernel that walks a page token by token (217 us for 255 + 200)."""
    H, dim = 2, 64
    kv = [n + 70 for n in new]
    cache, table = ob.KVCache8.empty(sum(-(-x // 64) for x in kv), H, dim), paged(kv, sum(-(-x // 64) for x in kv), 3)
    k = gen(1)(sum(new), H, dim).to(F16)
    batch = ob.CacheBatch(starts(new), i32(*kv), table, hint)
    assert forms(kernels_of(lambda: ob.cache_append(k, k, cache, batch), tmp_path)) == want


@pytest.mark.parametrize("hint", [None, 1, 3, 130])
@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128)])
def test_long_ranges_among_single_tokens(hint, dtype, dim):
    n = gen(dim)
    new = [1, 1, 0, 70, 1, 2, 3, 4, 1, 1, 0, 1, 130, 1] + [1, 0] * 70
    kv = [a + (37 * s) % 150 for s, a in enumerate(new)]
    pages, H, T = sum(-(-x // 64) for x in kv) + 3, 3, sum(new) + 4
    cache = ob.KVCache8.empty(pages, H, dim)
    cache.k_scale.fill_(2.0 ** -9), cache.v_scale.fill_(2.0 ** -7)     # as if the earlier tokens were there
    cache.k_pages.view(torch.uint8).fill_(0x31), cache.v_pages.view(torch.uint8).fill_(0x52)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    table = paged(kv, pages, 9)
    k, v = n(T, H, dim).to(dtype), n(T, H, dim).to(dtype)
    batch = ob.CacheBatch(starts(new, 2), i32(*kv), table, hint)
    ob.cache_append(k, v, cache, batch)
    want.append(k.double().cpu(), v.double().cpu(), batch.q_start, batch.kv_len, table)
    equal_pages(cache, want)
    assert _lib.load().onebit_check_device_status() == 0
