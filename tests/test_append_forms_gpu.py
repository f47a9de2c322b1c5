"""The two append kernels: which sequences each gets, and both against the definition."""
import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib
from tests import block_plain as plain
from tests.kernels_of import kernels_of
from tests.test_block_ops_gpu import check_rotary, equal_pages, gen, i32, paged, starts

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


def few_steps(dtype, dim, H, aligned, poison):
    """Steps of up to three tokens a sequence, behind prompts that end next to page ends, louder from step to step: batches of
    the warps' kernel, with what the plain form makes of them."""
    n = gen(dim + 7)
    new0, pages = [62, 1, 63, 5, 127, 64, 0], 40
    steps = [[1, 1, 1, 3, 1, 1, 0], [1, 0, 2, 1, 3, 1, 1], [1, 1, 1, 1, 1, 1, 1], [3, 2, 1, 0, 1, 2, 3], [1, 1, 1, 1, 1, 1, 1], [2, 3, 0, 3, 1, 1, 2]]
    total = [sum(x) for x in zip(new0, *steps)]
    cache, table = ob.KVCache8.empty(pages, H, dim), paged(total, pages, 5)
    cache.k_pages.view(torch.uint8).fill_(0x31), cache.v_pages.view(torch.uint8).fill_(0x52)
    kv = [0] * 7
    for i, new in enumerate([new0] + steps):
        kv = [a + b for a, b in zip(kv, new)]
        T = sum(new) + 3
        width = H * dim if aligned else H * dim + 5
        rows = (n(T, 2, width) * (1.0 if i == 0 else 3.0 ** i)).to(dtype)
        k, v = rows[:, 0, : H * dim].view(T, H, dim), rows[:, 1, : H * dim].unflatten(1, (H, dim))
        if poison and i:
            k[2, 0, 5], k[3, 1, 9], v[4, 0, 7], v[2, 1, dim - 1], v[5, 1, 0], k[6, 0, 0] = float("inf"), float("nan"), float("-inf"), float("nan"), float("nan"), float("-inf")
        yield cache, table, k, v, ob.CacheBatch(starts(new, 1), i32(*kv), table, None if i == 0 else 3), kv, new, i


@pytest.mark.parametrize("poison", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype,dim", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
def test_steps_of_few_tokens_are_exact(dtype, dim, aligned, poison, tmp_path):
    """Codes and scales of the warps' kernel equal the definition's bit for bit, re-scaled pages, infinities and NaN included."""
    want = None
    for cache, table, k, v, batch, kv, new, i in few_steps(dtype, dim, 3, aligned, poison):
        want = want or plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
        if i == 1:
            spare = ob.KVCache8.empty(cache.pages, 3, dim)
            assert forms(kernels_of(lambda: ob.cache_append(k, v, spare, batch), tmp_path)) == ["warps"]
        ob.cache_append(k, v, cache, batch)
        want.append(k.double().cpu(), v.double().cpu(), batch.q_start, batch.kv_len, table)
        equal_pages(cache, want)
    assert _lib.load().onebit_check_device_status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dim,rotary,heads,H", [(64, 64, 4, 4), (128, 128, 6, 2), (128, 64, 5, 1), (64, 20, 8, 2), (128, 8, 2, 1)])
def test_steps_of_few_tokens_with_rotation(layout, aligned, dim, rotary, heads, H):
    freq = ob.rotary_frequencies(rotary)[0]
    queries = gen(rotary)
    for cache, table, k, v, batch, kv, new, i in few_steps(F16, dim, H, aligned, False):
        T, live = k.shape[0], sum(new)
        q = queries(T, heads, dim + 3).to(F16)[..., :dim] if not aligned else queries(T, heads, dim).to(F16)
        got = ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq, layout=layout, magnitude=1.1, q_out=torch.full((T, heads, dim), 7.0, dtype=F16, device=DEV))
        assert (got[0] == 7.0).all() and (got[1 + live:] == 7.0).all()
        pos = torch.cat([torch.arange(a - n, a) for a, n in zip(kv, new)])
        check_rotary(got[1:1 + live], q[1:1 + live], pos, freq, layout, 1.1)
        turned, reach = plain.rotate(k[1:1 + live].cpu(), pos, freq.cpu(), layout, 1.1)
        at = 0
        for s, n in enumerate(new):
            gk, gv = (t.cpu().double()[kv[s] - n:] for t in cache.tokens(table[s], kv[s]))
            wk, wv = turned[at:at + n], v[1 + at:1 + at + n].cpu().double()
            # half an e4m3 step: 2^-4 of the value, 2^-10 of the scale among the subnormals (of either neighbouring scale for a largest
            # value within the fp32 error of 448 * 2^e), and the fp32 error of the rotation
            assert ((gk - wk).abs() <= wk.abs() * 2.0 ** -4 * 1.001 + reach[at:at + n].abs() * 2.0 ** -19 + float(cache.k_scale.max()) * 2.0 ** -9).all()
            assert ((gv - wv).abs() <= wv.abs() * 2.0 ** -4 + float(cache.v_scale.max()) * 2.0 ** -10).all()
            at += n
    assert _lib.load().onebit_check_device_status() == 0
