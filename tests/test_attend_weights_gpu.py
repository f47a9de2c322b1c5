"""Attention rows whose weight lies nearly all on one token (a sink) with no value of its own, or in a page that is louder than the
others: what is left of the output comes from thousands of small weights, and they have to survive their 16-bit form."""
import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib
from tests import block_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def sink_batch(new, kv, seqs, H, dim, dtype, loud, seed):
    """Equal scores of all tokens but the first, which is 14 above them (97 to 99.9 % of the weight) and has value 0; positive values
    elsewhere, so that nothing cancels and a bound of the sum of |weight * value| is one of the output. The first token's page
    has `loud` times the others' value scale."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    blocks = -(-kv // 64)
    pages = seqs * blocks
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(seqs, blocks)
    k = torch.zeros(pages, H, 64, dim, device=DEV)
    v = torch.randint(64, 129, (pages, H, dim, 64), generator=g, device=DEV).float()
    ks, vs = torch.full((pages, H), 2.0 ** -5, device=DEV), torch.full((pages, H), 2.0 ** -6, device=DEV)
    first = table[:, 0].long()
    k[first, :, 0, 0] = 448.0                                   # times 2^-5 and a query of 1: 14
    v[first, :, :, 0] = 0.0
    vs[first] *= loud
    cache = ob.KVCache8(k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn), ks, vs)
    q = torch.zeros(seqs * new, H, dim, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    i32 = dict(dtype=torch.int32, device=DEV)
    return q, cache, ob.CacheBatch(torch.arange(seqs + 1, **i32) * new, torch.full((seqs,), kv, **i32), table, new)


@pytest.mark.parametrize("loud", [1, 16, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,kv,seqs,H,dim", [(1, 4096, 40, 8, 64), (1, 16384, 12, 4, 128), (2, 8192, 1, 2, 64), (160, 8192, 1, 2, 64), (100, 4096, 9, 9, 128)])
def test_small_weights_beside_a_sink(new, kv, seqs, H, dim, dtype, loud):
    q, cache, batch = sink_batch(new, kv, seqs, H, dim, dtype, loud, kv + loud)
    rows = torch.arange(0, seqs * new, max(1, seqs * new // 30))                        # of these the plain form
    got = ob.cache_attend(q, cache, batch, scale=1.0).cpu().double()[rows]
    assert _lib.load().onebit_check_device_status() == 0
    want, top = torch.zeros_like(got), torch.zeros(got.shape[:2], dtype=torch.float64)
    for i, r in enumerate(rows.tolist()):
        s, limit = r // new, kv - new + r % new + 1
        page = batch.block_table[s].long()
        k = (cache.k_pages.view(torch.uint8)[page].view(torch.float8_e4m3fn).double() * cache.k_scale[page].double()[..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :limit]
        v = (cache.v_pages.view(torch.uint8)[page].view(torch.float8_e4m3fn).double() * cache.v_scale[page].double()[..., None, None]).permute(1, 0, 3, 2).flatten(1, 2)[:, :limit]
        w = torch.softmax((k @ q[r].double()[..., None])[..., 0], -1)                   # (H, limit)
        want[i] = (w[:, None] @ v)[:, 0].cpu()
        scale = cache.v_scale[page].double().repeat_interleave(64, 0)[:limit].T
        top[i] = (w * scale).amax(-1).cpu()
    # A weight is held in 16 bits as 2^(score + log2 scale - M + shift), shift 15 with few rows and at least 11 with many (M is the
    # row's largest or above it by less than what the shift leaves): 2^-11 of it, or 2^-25 where it is subnormal, which is
    # 2^-25-shift of the largest weight * scale, times codes of up to 448 and every token. The argument of 2^x is at most 40 and
    # rounded twice: 2 * 40 * 2^-24 < 2^-17, in the numerator and in the sum. The products are added 16 tokens at a time, each
    # addition off by at most 2^-23 of the sum.
    shift = 15 if new * (q.shape[1] // H) <= 64 else 11
    tol = want * (2.0 ** -11 + 2 * 2.0 ** -17 + kv / 16 * 2.0 ** -23 + plain.HALF_STEP[dtype] * (1 + 2.0 ** -6)) + (kv * 448 * 2.0 ** -(25 + shift) * top)[..., None] + 1e-7
    err = (got - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), float((err / want).max()))
