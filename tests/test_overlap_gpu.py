"""Outputs that share memory with an input without being it are refused, views into the rows of a fused projection among them, and
views that only interleave are not."""
import pytest
import torch

import onebitsparsemul_b200 as ob

pytestmark = pytest.mark.gpu
DEV, F16 = "cuda", torch.float16


def rows_of(tokens, heads, dim=64):
    g = torch.Generator(device=DEV)
    g.manual_seed(tokens + heads)
    return torch.randn(tokens, heads, dim, generator=g, device=DEV).to(F16)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_rotary_views():
    rows, pos, freq = rows_of(9, 12), torch.arange(9, device=DEV), ob.rotary_frequencies(64)[0]
    square = rows_of(16, 16, 8)
    for x, out in ((rows[:, 0:4], rows[:, 1:5]), (rows[:, 1:5], rows[:, 0:4]), (rows[:, ::3], rows[:, 3:7]), (rows[:-1, :4], rows[1:, :4]), (rows[:, :4, :32], rows[:, :4, 16:48]),
                   (rows[:, :4], torch.as_strided(rows, (9, 4, 64), (12 * 64, 32, 1))), (square, square.transpose(0, 1))):
        t = x.shape[0]
        f = freq[: x.shape[2] // 2]
        with pytest.raises(ValueError):
            ob.rotary_tokens(x, torch.arange(t, device=DEV), f, out=out)
    for first, second in ((slice(0, 4), slice(4, 8)), (slice(0, None, 2), slice(1, None, 2)), (slice(8, 12), slice(0, 4))):
        x, out = rows.clone()[:, first], None
        base = torch.empty_like(rows)
        base[:, first] = x
        x, out = base[:, first], base[:, second]
        want = ob.rotary_tokens(x.clone(), pos, freq)
        assert ob.rotary_tokens(x, pos, freq, out=out) is out
        assert torch.equal(out, want)


def test_norm_views():
    w = rows_of(1, 1, 96).view(96)
    buffer = rows_of(1, 1, 20 * 200).view(20, 200)
    for x, out in ((buffer[::2, :96], buffer.view(-1)[: 960].view(10, 96)),):
        with pytest.raises(ValueError):
            ob.residual_norm(x, w, out=out)
        with pytest.raises(ValueError):
            ob.residual_norm(x, w, residual=torch.zeros_like(x), residual_out=out)
    x = rows_of(1, 1, 96 * 96).view(96, 96)
    with pytest.raises(ValueError):
        ob.residual_norm(x.T, w, out=x)


def test_attention_views():
    cache = ob.KVCache8.empty(1, 1, 64)
    batch = ob.CacheBatch(i32(0, 8), i32(8), i32(0).view(1, 1))
    rows = rows_of(8, 4)
    flat = rows.view(-1)
    for q, out in ((rows[:, :1], flat[:512].view(8, 1, 64)), (rows[:, 1:3], flat[128:128 + 1024].view(8, 2, 64))):
        with pytest.raises(ValueError):
            ob.cache_attend(q, cache, batch, out=out)


def test_append_queries_apart_from_keys_values_and_cache():
    """Queries are turned while other threads read k and v and write the pages: none of them may be where q_out is."""
    cache = ob.KVCache8.empty(2, 4, 64)
    batch = ob.CacheBatch(i32(0, 8), i32(8), i32(0).view(1, 1))
    rows, freq = rows_of(8, 16), ob.rotary_frequencies(64)[0]
    q, k, v = rows[:, :4], rows[:, 4:8], rows[:, 8:12]
    pages = cache.k_pages.view(torch.uint8).view(-1)[: 8 * 4 * 64 * 2].view(F16).view(8, 4, 64)
    for out in (k, v, rows[:, 5:9], rows[:, 3:7], rows[:, 11:15], pages):
        with pytest.raises(ValueError):
            ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq, q_out=out)
    before = rows.clone()
    want = ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq)
    assert torch.equal(rows, before)
    assert torch.equal(ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq, q_out=rows[:, 12:]), want)
    assert torch.equal(ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq, q_out=q), want) and torch.equal(rows[:, 4:12], before[:, 4:12])
    with pytest.raises(ValueError):
        ob.cache_attend(q, cache, batch, out=pages)


def test_norm_outputs_apart_from_the_weights():
    """h is written before the weight is read: a residual_out that is the weight gave the norm a changed one."""
    x, r, w, p = rows_of(1, 1, 96).view(1, 96), rows_of(1, 2, 96)[:, 1], rows_of(3, 1, 96)[:1].view(96).clone(), rows_of(4, 1, 96)[:1].view(96).clone()
    many = rows_of(5, 1, 96).view(5, 96)
    for kw in (dict(residual_out=w.view(1, 96)), dict(out=w.view(1, 96)), dict(residual_out=p.view(1, 96), post_weight=p), dict(out=p.view(1, 96), post_weight=p)):
        with pytest.raises(ValueError):
            ob.residual_norm(x, w, residual=r, **kw)
    with pytest.raises(ValueError):
        ob.residual_norm(many, many[2], out=many)
    want = ob.residual_norm(x, w, residual=r, gate=p.view(1, 96))
    gate = p.clone().view(1, 96)
    got = ob.residual_norm(x, w, residual=r, gate=gate, residual_out=gate)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1] is gate
