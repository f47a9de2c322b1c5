"""Decoder-block operators against plain 64-bit restatements, on the GPU."""
import math

import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib
from tests import block_plain as plain

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DEV = "cuda"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV)


def status_ok():
    return _lib.load().onebit_check_device_status() == 0


# ---- norm ---------------------------------------------------------------------------------------------------------------

def check_norm(y, h, x, weight, residual, gate, scale, post, eps):
    wy, wh, reach_y, reach_h = plain.norm(x, weight, residual, gate, scale, post, eps)
    u = plain.HALF_STEP[x.dtype]
    # fp32: a sum of at most 32 values a thread and 10 tree levels, rsqrt and a handful of products: 64 roundings of 2^-24,
    # of the terms' sizes (they may cancel in h)
    tol = wy.abs() * u * 1.01 + (reach_y + wy.abs()) * 2.0 ** -18 + 1e-7 * u
    if x.dtype == F16:
        tol = tol + 2.0 ** -25                               # half a step among the subnormals
    assert ((y.double() - wy).abs() <= tol).all(), float(((y.double() - wy).abs() / tol).max())
    if residual is not None:
        uh = plain.HALF_STEP[residual.dtype]
        tol = wh.abs() * uh * 1.01 + reach_h * 2.0 ** -20 + (2.0 ** -25 if residual.dtype == F16 else 1e-30)
        assert ((h.double() - wh).abs() <= tol).all(), float(((h.double() - wh).abs() / tol).max())


@pytest.mark.parametrize("rows,hidden", [(1, 4096), (1, 1), (3, 7), (5, 64), (130, 256), (2, 512), (7, 1000), (33, 2047), (9, 4096), (4, 11008), (3, 16384),
                                         (2, 32767), (2, 32768)])
@pytest.mark.parametrize("dtype,wide", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("form", ["norm", "residual", "post", "channel", "full"])
def test_residual_norm(rows, hidden, dtype, wide, form):
    n = gen(rows * 77 + hidden)
    x, weight = (n(rows, hidden) * 3).to(dtype), (1 + 0.2 * n(hidden)).to(dtype)
    if form == "norm":
        if wide:
            pytest.skip("no residual")
        y = ob.residual_norm(x, weight)
        return check_norm(y, None, x, weight, None, None, 1.0, None, 1e-6)
    residual = (n(rows, hidden) * 2).to(F32 if wide else dtype)
    post = (1 + 0.2 * n(hidden)).to(dtype) if form != "residual" else None
    gate = n(hidden).to(dtype) if form == "channel" else n(rows, hidden).to(dtype) if form == "full" else None
    scale = 1.0 if form == "residual" else 0.37
    y, h = ob.residual_norm(x, weight, residual=residual, gate=gate, residual_scale=scale, post_weight=post, eps=1e-5)
    assert y.dtype == dtype and h.dtype == residual.dtype
    check_norm(y, h, x, weight, residual, gate, scale, post, 1e-5)


@pytest.mark.parametrize("rows,hidden", [(300, 64), (259, 1024), (300, 4096), (257, 4104), (300, 2048), (270, 3001), (260, 4097), (600, 40)])
def test_residual_norm_of_many_rows(rows, hidden):
    for form in ("norm", "residual", "post", "full"):
        test_residual_norm(rows, hidden, BF16, False, form)


def test_residual_norm_of_long_unaligned_rows_in_place():
    n = gen(4)
    x, r, w, g = n(3, 9007).to(F16), n(3, 9007), (1 + 0.2 * n(9007)).to(F16), n(3, 9007).to(F16)
    y, h = ob.residual_norm(x, w, residual=r, gate=g, post_weight=w, residual_scale=0.7)
    x2, r2 = x.clone(), r.clone()
    ob.residual_norm(x2, w, residual=r2, gate=g, post_weight=w, residual_scale=0.7, out=x2, residual_out=r2)
    assert torch.equal(y, x2) and torch.equal(h, r2)
    check_norm(y, h, x, w, r, g, 0.7, w, 1e-6)


def test_residual_norm_shapes_strides_and_in_place():
    n = gen(1)
    rows = n(6, 6, 2 * 96 + 8).to(F16)
    weight, gate = n(96).to(F16), n(6, 6, 96).to(F16)
    for x in (rows[..., :96], rows[..., 8:104], rows[..., 3:99], rows.transpose(0, 1)[..., 1:193:2], rows[:1, :1, :96].expand(6, 6, 96)):
        residual = n(6, 6, 96)
        y, h = ob.residual_norm(x, weight, residual=residual, gate=gate, residual_scale=0.5)
        check_norm(y, h, x, weight, residual, gate, 0.5, None, 1e-6)
    x, r = n(30, 96).to(F16), n(30, 96).to(F16)
    y, h = ob.residual_norm(x, weight, residual=r)
    x2, r2 = x.clone(), r.clone()
    y2, h2 = ob.residual_norm(x2, weight, residual=r2, out=x2, residual_out=r2)
    assert y2 is x2 and h2 is r2 and torch.equal(y, x2) and torch.equal(h, r2)
    v = n(96).to(F16)
    check_norm(ob.residual_norm(v, weight), None, v, weight, None, None, 1.0, None, 1e-6)
    assert ob.residual_norm(v.new_zeros(0, 96), weight).shape == (0, 96)
    # rows of zeros, of the type's largest values, with an infinity and with a NaN: only their own row is touched
    x = n(5, 96).to(F16)
    x[0], x[1] = 0, 65504
    x[2, 3], x[3, 4] = math.inf, math.nan
    y = ob.residual_norm(x, weight)
    assert (y[0] == 0).all() and y[1].isfinite().all() and y[2, 3].isnan() and y[3].isnan().all() and y[4].isfinite().all()


def test_residual_norm_refusals():
    n = gen(2)
    x, w = n(4, 64).to(F16), n(64).to(F16)
    bad = [dict(x=x.float(), weight=w), dict(x=x, weight=w[:32]), dict(x=x, weight=w.to(BF16)), dict(x=x, weight=w, gate=w), dict(x=x, weight=w, residual_scale=0.5),
           dict(x=x, weight=w, residual=x[:2]), dict(x=x, weight=w, residual=x.to(BF16)), dict(x=x, weight=w, residual=x, gate=x[:, :1]), dict(x=x, weight=w, eps=-1.0),
           dict(x=x, weight=w, out=x[:2]), dict(x=x, weight=w, residual=x, residual_out=x.float()), dict(x=x, weight=w.cpu()), dict(x=n(1, 32769).to(F16), weight=w),
           dict(x=x, weight=w, residual=x, residual_scale=math.inf), dict(x=x.clone().requires_grad_(), weight=w)]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            ob.residual_norm(**kw)
    with torch.no_grad():
        ob.residual_norm(x.clone().requires_grad_(), w)


# ---- rotary ---------------------------------------------------------------------------------------------------------------

def check_rotary(y, x, positions, freq, layout, magnitude=1.0):
    want, reach = plain.rotate(x.cpu(), positions.cpu(), freq.cpu(), layout, magnitude)
    # cos and sin: phase in turns to 2^-32, its fp32 form to 2^-25 half turns, cosf and sinf of the
    # special function unit to 2^-21.2, products and sum 3 roundings
    tol = want.abs() * plain.HALF_STEP[x.dtype] * 1.01 + reach * 2.0 ** -20 + (2.0 ** -25 if x.dtype == F16 else 0)
    err = (y.double().cpu() - want).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    assert torch.equal(y[..., 2 * freq.numel():], x[..., 2 * freq.numel():])


@pytest.mark.parametrize("tokens,heads,dim,rotary", [(1, 1, 64, 64), (1, 32, 128, 128), (5, 3, 128, 64), (9, 7, 80, 80), (6, 2, 128, 24), (3, 5, 64, 20), (4, 3, 7, 6), (67, 12, 96, 48),
                                                     (2, 2, 512, 512), (3, 2, 64, 0)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rotary(tokens, heads, dim, rotary, layout, dtype):
    n = gen(tokens + heads + dim)
    x = n(tokens, heads, dim).to(dtype)
    freq = ob.rotary_frequencies(rotary)[0] if rotary else torch.empty(0, dtype=torch.float64, device=DEV)
    for positions in (torch.arange(tokens, device=DEV), torch.arange(tokens, device=DEV, dtype=torch.int32) + 1000003, torch.arange(tokens, device=DEV) - 5,
                      torch.full((tokens,), 2 ** 31 - 1, device=DEV, dtype=torch.int32), torch.full((tokens,), 3 * 2 ** 32 + 17, device=DEV)):
        check_rotary(ob.rotary_tokens(x, positions, freq, layout=layout, magnitude=1.25), x, positions, freq, layout, 1.25)


def test_rotary_views_in_place_and_refusals():
    n = gen(4)
    rows = n(9, 12, 64).to(F16)
    freq, pos = ob.rotary_frequencies(64)[0], torch.arange(9, device=DEV) * 7
    for x in (rows[:, 2:6], rows[:, ::3], rows[::2], rows.transpose(0, 1)[:9], n(9, 4, 66).to(F16)[..., 1:65], n(9, 4, 128).to(F16)[..., ::2], rows[:1].expand(9, 12, 64)):
        p = pos[: x.shape[0]]
        check_rotary(ob.rotary_tokens(x, p, freq), x, p, freq, "half")
    y = ob.rotary_tokens(rows[:, 2:6], pos, freq)
    before = rows.clone()
    got = ob.rotary_tokens(rows[:, 2:6], pos, freq, out=rows[:, 2:6])
    assert torch.equal(got, y) and torch.equal(rows[:, 2:6], y)
    assert torch.equal(rows[:, :2], before[:, :2]) and torch.equal(rows[:, 6:], before[:, 6:])
    assert ob.rotary_tokens(rows[:0], pos[:0], freq).shape == (0, 12, 64)
    for kw in (dict(x=rows[0]), dict(positions=pos[:3]), dict(positions=pos.float()), dict(inv_freq=freq.float()), dict(layout="thirds"), dict(x=rows.float()),
               dict(inv_freq=torch.ones(33, dtype=torch.float64, device=DEV)), dict(out=rows[:, :3]), dict(positions=pos.cpu()), dict(x=rows.clone().requires_grad_())):
        with pytest.raises((ValueError, TypeError)):
            ob.rotary_tokens(**{**dict(x=rows, positions=pos, inv_freq=freq), **kw})


# ---- append ---------------------------------------------------------------------------------------------------------------

def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def paged(kv, pages, seed, width=None):
    """A table with the pages of sequences of these lengths in shuffled order, -1 elsewhere."""
    blocks = [max(0, -(-x // 64)) for x in kv]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g)[: sum(blocks)].to(torch.int32)
    table = torch.full((len(kv), width or max(1, max(blocks))), -1, dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    return table.to(DEV)


def starts(lengths, first=0):
    out = [first]
    for x in lengths:
        out.append(out[-1] + x)
    return i32(*out)


def equal_pages(cache, want):
    k, v = cache.k_pages.float().cpu().double(), cache.v_pages.float().cpu().double()
    assert torch.equal(cache.k_scale.cpu().double(), want.ks) and torch.equal(cache.v_scale.cpu().double(), want.vs)
    assert torch.equal(k.nan_to_num(999.0), want.k.nan_to_num(999.0)) and torch.equal(v.nan_to_num(999.0), want.v.nan_to_num(999.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("aligned", [True, False])
def test_append_without_rotation_is_exact(dtype, dim, aligned):
    """Three steps of ragged sequences, one of them without tokens, with louder and louder tokens: codes and scales equal the
    definition's, bit for bit, in the whole pool."""
    n = gen(dim)
    pages, H, steps = 24, 3, [[1, 0, 70, 5, 64], [3, 1, 1, 130, 0], [1, 1, 200, 1, 1]]
    cache = ob.KVCache8.empty(pages, H, dim)
    cache.k_pages.view(torch.uint8).fill_(0x31)              # what a recycled page may hold
    cache.v_pages.view(torch.uint8).fill_(0x52)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    total = [sum(x) for x in zip(*steps)]
    table = paged(total, pages, 5)
    kv = [0] * 5
    for step, new in enumerate(steps):
        kv = [a + b for a, b in zip(kv, new)]
        T = sum(new) + 3                                      # rows before and behind the sequences
        width = H * dim if aligned else H * dim + 5
        rows = (n(T, 2, width) * 5.0 ** step).to(dtype)
        k, v = rows[:, 0, : H * dim].view(T, H, dim), rows[:, 1, : H * dim].unflatten(1, (H, dim))
        batch = ob.CacheBatch(starts(new, 1), i32(*kv), table)
        assert ob.cache_append(k, v, cache, batch) is None
        want.append(k.double().cpu(), v.double().cpu(), batch.q_start, batch.kv_len, table)
        equal_pages(cache, want)
    assert status_ok()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary,heads,kv_heads", [(64, 64, 4, 4), (128, 128, 6, 2), (128, 64, 5, 1), (64, 20, 8, 2)])
def test_append_with_rotation(layout, dim, rotary, heads, kv_heads):
    n = gen(rotary + heads)
    new, kv, pages = [1, 33, 0, 129, 2], [1, 33, 7, 300, 70], 16
    T = sum(new) + 2
    rows = n(T, heads + 2 * kv_heads, dim).to(F16)
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
    cache = ob.KVCache8.empty(pages, kv_heads, dim)
    table = paged(kv, pages, 7)
    batch = ob.CacheBatch(starts(new), i32(*kv), table)
    freq = ob.rotary_frequencies(rotary)[0]
    out = torch.full_like(q, 7.0)
    got = ob.cache_append(k, v, cache, batch, q=q, inv_freq=freq, layout=layout, magnitude=1.1, q_out=out)
    assert got is out and (out[sum(new):] == 7.0).all()       # rows behind the last sequence are left as they were
    at, pos = batch.q_start.tolist(), torch.zeros(T, dtype=torch.long)
    for s in range(len(new)):
        pos[at[s]:at[s + 1]] = torch.arange(kv[s] - new[s], kv[s])
    live = sum(new)
    check_rotary(out[:live], q[:live], pos[:live], freq, layout, 1.1)
    turned, reach = plain.rotate(k.cpu(), pos, freq.cpu(), layout, 1.1)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    want.k.zero_(), want.v.zero_()
    want.append(turned, v.cpu().double(), batch.q_start, batch.kv_len, table)
    for s in range(len(new)):
        if not new[s]:
            continue
        gk, gv = cache.tokens(table[s], kv[s])
        gk, gv = gk.cpu().double()[kv[s] - new[s]:], gv.cpu().double()[kv[s] - new[s]:]
        wk = turned[at[s]:at[s + 1]]
        # a code is half an e4m3 step off: 2^-4 of the value, 2^-10 of the scale among the subnormals; a largest value within
        # the fp32 error of 448 * 2^e may take either neighbouring scale, which this bound covers (2^-10 of twice the scale)
        tol = wk.abs() * 2.0 ** -4 * 1.001 + reach[at[s]:at[s + 1]].abs() * 2.0 ** -19 + float(cache.k_scale.max()) * 2.0 ** -9
        assert ((gk - wk).abs() <= tol).all()
        assert torch.equal(gv, torch.stack([want.v[table[s][(kv[s] - new[s] + i) // 64], :, :, (kv[s] - new[s] + i) % 64]
                                            * want.vs[table[s][(kv[s] - new[s] + i) // 64]][:, None] for i in range(new[s])]))
    assert torch.equal(cache.v_scale.cpu().double(), want.vs)
    in_place = q.clone()
    assert torch.equal(ob.cache_append(k, v, cache, batch, q=in_place, inv_freq=freq, layout=layout, magnitude=1.1, q_out=in_place)[:live], out[:live])
    assert status_ok()


def test_append_of_infinities_nan_and_extremes():
    H, dim = 2, 64
    n = gen(11)
    k, v = n(70, H, dim).to(BF16), n(70, H, dim).to(BF16)
    k[3, 0, 5], k[4, 0, 6], v[5, 0, 7], v[6, 1, 8] = math.inf, math.nan, -math.inf, math.nan
    k[66:, 1], v[66:, 1] = 1e30, 1e-30                       # the scale's ends; the pages' other head stays ordinary
    k[64:66, 1], v[64:66, 1] = 0, 0
    cache = ob.KVCache8.empty(4, H, dim)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    batch = ob.CacheBatch(i32(0, 70), i32(70), i32(2, 1).view(1, 2))
    ob.cache_append(k, v, cache, batch)
    want.append(k.double().cpu(), v.double().cpu(), batch.q_start, batch.kv_len, batch.block_table)
    equal_pages(cache, want)
    assert float(cache.k_scale.max()) == 2.0 ** 32 and not cache.v_pages.float().isnan().any()
    # the queries that see a poisoned token answer NaN, the others do not
    y = ob.cache_attend(n(70, H, dim).to(BF16), cache, batch)
    assert y[4:, 0].isnan().all() and y[6:, 1].isnan().all()
    assert y[:4, 0].isfinite().all() and y[:6, 1].isfinite().all()


def test_bad_pages_and_ranges_are_left_out():
    H, dim, pages = 2, 64, 4
    n = gen(12)
    cache = ob.KVCache8.empty(pages, H, dim)
    k, v, q = n(10, H, dim).to(F16), n(10, H, dim).to(F16), n(10, 4, dim).to(F16)
    table = i32(1, -1, 99, 2).view(2, 2)
    # sequence 0: its second page is unmapped; sequence 1: its first page does not exist; the batch is longer than the table
    for q_start, kv_len in ((i32(0, 5, 10), i32(67, 70)), (i32(0, 5, 11), i32(67, 200)), (i32(-3, 5, 10), i32(-2, 128))):
        batch = ob.CacheBatch(q_start, kv_len, table)
        want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
        if int(q_start[0]) == 0 and int(q_start[-1]) == 10:
            ob.cache_append(k, v, cache, batch)
            want.append(k.double().cpu(), v.double().cpu(), q_start, kv_len, table)
            assert not status_ok() and b"page number" in _lib.load().onebit_last_error() and status_ok()
            equal_pages(cache, want)
            out, spread, delta, least, _ = plain.attend(q, want, q_start, kv_len, table, dim ** -0.5, True)
            got = ob.cache_attend(q, cache, batch)
            assert ((got.cpu().double() - out).abs() <= plain.attend_tolerance(out, spread, delta, least, F16)).all()
            assert not status_ok() and status_ok()
        else:
            ob.cache_append(k, v, cache, batch)
            ob.cache_attend(q, cache, batch)
            torch.cuda.synchronize()
            status_ok()
    assert status_ok()


@pytest.mark.parametrize("new", [1, 80])
def test_a_sequence_longer_than_its_table_is_reported(new):
    cache, table = random_cache([128], 2, 64, 3)
    batch = ob.CacheBatch(i32(0, new), i32(190), table, new)          # two pages for 190 tokens
    q = gen(4)(new, 4, 64).to(F16)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    out, spread, delta, least, _ = plain.attend(q, want, batch.q_start, batch.kv_len, table, 0.125, True)
    got = ob.cache_attend(q, cache, batch)
    assert ((got.cpu().double() - out).abs() <= plain.attend_tolerance(out, spread, delta, least, F16)).all()
    assert not status_ok() and status_ok()
    k = gen(5)(new, 2, 64).to(F16)
    ob.cache_append(k, k, cache, batch)
    assert not status_ok() and status_ok()


@pytest.mark.parametrize("width,hint", [(8, 1), (200, 1), (8, 200)])
def test_ranges_that_run_backwards_are_reported(width, hint):
    cache, table = random_cache([300] * 40, 4, 64, 3)
    wide = torch.zeros(40, width, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = gen(4)(40, 4, 64).to(F16)
    good = ob.CacheBatch(i32(*range(41)), i32(*[300] * 40), wide, hint)
    want = ob.cache_attend(q, cache, good)
    assert status_ok()
    starts_ = list(range(41))
    starts_[7] = 3                                              # sequence 6 runs from 6 back to 3, sequence 7 from 3 to 8
    ob.cache_attend(q, cache, ob.CacheBatch(i32(*starts_), good.kv_len, wide, hint))
    assert not status_ok() and status_ok()
    assert torch.equal(ob.cache_attend(q, cache, good), want)


def test_outputs_that_overlap_are_refused():
    n = gen(9)
    x, w, r = n(8, 64).to(F16), n(64).to(F16), n(8, 64).to(F16)
    y = torch.empty_like(x)
    flat = n(9 * 64).to(F16)
    for kw in (dict(out=y, residual_out=y), dict(x=flat[:512].view(8, 64), out=flat[64:].view(8, 64)), dict(residual=flat[:512].view(8, 64), residual_out=flat[64:].view(8, 64))):
        with pytest.raises(ValueError):
            ob.residual_norm(**{**dict(x=x, weight=w, residual=r), **kw})
    pos, freq = torch.arange(8, device=DEV), ob.rotary_frequencies(64)[0]
    with pytest.raises(ValueError):
        ob.rotary_tokens(x.view(8, 1, 64), pos, freq, out=n(1, 1, 64).to(F16).expand(8, 1, 64))
    with pytest.raises(ValueError):
        ob.rotary_tokens(flat[:512].view(8, 1, 64), pos, freq, out=flat[64:].view(8, 1, 64))
    cache = ob.KVCache8.empty(1, 1, 64)
    batch = ob.CacheBatch(i32(0, 8), i32(8), i32(0).view(1, 1))
    q = x.view(8, 1, 64)
    with pytest.raises(ValueError):
        ob.cache_attend(q, cache, batch, out=q)
    with pytest.raises(ValueError):
        ob.cache_append(q, q, cache, batch, q=q, inv_freq=freq, q_out=n(1, 1, 64).to(F16).expand(8, 1, 64))


def test_append_refusals():
    n = gen(13)
    cache = ob.KVCache8.empty(4, 2, 64)
    batch = ob.CacheBatch(i32(0, 3), i32(3), i32(0).view(1, 1))
    k, q, freq = n(3, 2, 64).to(F16), n(3, 4, 64).to(F16), ob.rotary_frequencies(64)[0]
    ok = dict(k=k, v=k, cache=cache, batch=batch)
    for kw in (dict(k=k[:, :1]), dict(v=k[:2]), dict(v=k.to(BF16)), dict(q=q), dict(q=q[:, :3], inv_freq=freq), dict(q=q.to(BF16), inv_freq=freq), dict(q_out=q),
               dict(q=q, inv_freq=freq.float()), dict(q=q, inv_freq=freq, q_out=q[:, :2]), dict(k=k.clone().requires_grad_()), dict(inv_freq=freq, layout="x"),
               dict(cache=ob.KVCache8.empty(4, 2, 128)), dict(cache=ob.KVCache8.empty(4, 2, 64, device="cpu"))):
        with pytest.raises((ValueError, TypeError)):
            ob.cache_append(**{**ok, **kw})
    for kw in (dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[0]), dict(scale=math.nan), dict(out=q.transpose(0, 1)), dict(q=q.clone().requires_grad_())):
        with pytest.raises((ValueError, TypeError)):
            ob.cache_attend(**{**dict(q=q, cache=cache, batch=batch), **kw})


# ---- attend -----------------------------------------------------------------------------------------------------------------

def random_cache(kv, H, dim, seed, slack=2, loud=True):
    """A filled cache: e4m3 codes of normal values, a scale of its own for each page and head, NaN codes wherever a sequence
    has no token (which nothing may read into a result)."""
    n = gen(seed)
    pages = sum(max(0, -(-x // 64)) for x in kv) + slack
    table = paged(kv, pages, seed)
    k, v = (n(pages, H, 64, dim) * 100).clamp(-448, 448).to(torch.float8_e4m3fn), (n(pages, H, dim, 64) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    ks = 2.0 ** torch.randint(-8, -5, (pages, H), device=DEV).float()
    vs = 2.0 ** torch.randint(-9, -3 if loud else -6, (pages, H), device=DEV).float()
    kb, vb = k.view(torch.uint8), v.view(torch.uint8)
    held = torch.zeros(pages, dtype=torch.long)
    for s, x in enumerate(kv):
        for b in range(max(0, -(-x // 64))):
            held[table[s, b].item()] = min(64, x - 64 * b)
    gone = torch.arange(64)[None] >= held[:, None]
    gone = gone.to(DEV)
    kb.masked_fill_(gone[:, None, :, None], 0x7F)
    vb.masked_fill_(gone[:, None, None, :], 0xFF)
    return ob.KVCache8(k, v, ks, vs), table


def check_attend(new, kv, heads, kv_heads, dim, dtype, causal=True, scale=None, max_new=None, seed=0, q=None, pad=(0, 0), loud=True):
    cache, table = random_cache(kv, kv_heads, dim, seed, loud=loud)
    n = gen(seed + 1)
    T = sum(new) + sum(pad)
    q = n(T, heads, dim).to(dtype) if q is None else q
    batch = ob.CacheBatch(starts(new, pad[0]), i32(*kv), table, max_new)
    plain_cache = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    out, spread, delta, least, written = plain.attend(q, plain_cache, batch.q_start, batch.kv_len, table, dim ** -0.5 if scale is None else scale, causal)
    got = torch.full(q.shape, 9.0, dtype=dtype, device=DEV)
    assert ob.cache_attend(q, cache, batch, scale=scale, causal=causal, out=got) is got
    assert status_ok(), _lib.load().onebit_last_error()
    assert (got[~written.to(DEV)] == 9.0).all()
    err, tol = (got.cpu().double() - out).abs()[written], plain.attend_tolerance(out, spread, delta, least, dtype)[written]
    assert (err <= tol).all(), float((err / tol).max())
    return q, cache, batch, got


FEW = [  # new tokens, cached tokens
    ([1], [1]), ([1], [63]), ([1], [64]), ([1], [65]), ([1], [1000]), ([1, 1, 1], [5, 700, 129]), ([1, 0, 1], [5, 70, 64]), ([4, 1, 3], [4, 200, 66]),
    ([8], [8]), ([8, 2], [530, 2]), ([1] * 40, list(range(1, 400, 10))), ([3, 3], [2, 0]), ([0, 0], [10, 20]), ([5], [3])]


@pytest.mark.parametrize("new,kv", FEW)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 4, 128, F16), (8, 2, 128, BF16), (6, 2, 64, F16), (16, 1, 64, BF16)])
def test_attend_few_rows(new, kv, heads, kv_heads, dim, dtype):
    check_attend(new, kv, heads, kv_heads, dim, dtype, max_new=max(1, max(new)), seed=len(kv) + kv[0])


@pytest.mark.parametrize("new,kv,hint", [  # clusters of every size, more and fewer CTAs than pages, more row tiles than the bound says
    ([1], [2500], 1), ([1], [300], 1), ([3], [700], 1), ([20], [2100], 1), ([1, 1], [4000, 3], 1), ([20, 2], [2100, 130], 2), ([9, 1, 0, 1], [1025, 0, 5, 640], 9),
    ([1] * 5, [0, 1, 600, 1025, 130], 1), ([1] * 12, list(range(60, 1260, 100)), 1), ([17] * 3, [400, 17, 1100], 3), ([1] * 40, [4200] + list(range(1, 391, 10)), 1)])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 8, 128, BF16), (8, 2, 64, F16), (5, 1, 128, F16), (48, 16, 64, BF16)])
def test_attend_few_rows_by_clusters(new, kv, hint, heads, kv_heads, dim, dtype):
    q, cache, batch, got = check_attend(new, kv, heads, kv_heads, dim, dtype, max_new=hint, seed=kv[0], pad=(1, 2))
    for _ in range(3):
        assert torch.equal(ob.cache_attend(q, cache, batch)[1:1 + sum(new)], got[1:1 + sum(new)])


MANY = [([200], [200]), ([130], [1000]), ([64, 1, 65], [64, 600, 65]), ([300, 0, 7, 129], [300, 5, 900, 129]), ([100], [60]), ([128], [128]), ([256], [256]), ([257], [640])]


@pytest.mark.parametrize("new,kv", MANY)
@pytest.mark.parametrize("heads,kv_heads,dim,dtype,causal", [(2, 2, 128, F16, True), (8, 2, 128, BF16, True), (3, 1, 64, F16, True), (4, 4, 64, BF16, False), (5, 1, 128, F16, False)])
def test_attend_many_rows(new, kv, heads, kv_heads, dim, dtype, causal):
    check_attend(new, kv, heads, kv_heads, dim, dtype, causal=causal, seed=sum(new))


@pytest.mark.parametrize("hint", [None, 1, 3, 40, 5000])
def test_attend_hint_and_padding_do_not_change_what_is_right(hint):
    check_attend([1, 30, 2, 90], [100, 230, 2, 90], 8, 2, 128, F16, max_new=hint, seed=3, pad=(3, 5))


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,causal", [(16, 8, 128, F16, True), (32, 32, 64, BF16, True), (40, 10, 64, F16, False), (24, 8, 128, BF16, False)])
def test_attend_prompts_among_single_tokens(heads, kv_heads, dim, dtype, causal):
    """Batches that both kernels share, each its sequences: lengths on either side of the rule, empty ones, padded rows."""
    new = [1, 0, 150, 1, 12, 13, 1, 24, 25, 1, 1, 16, 17, 1, 48, 49, 2, 1, 1, 1]
    kv = [700, 5, 1000, 64, 12, 80, 1, 100, 25, 300, 129, 10, 17, 0, 48, 200, 65, 900, 33, 63]
    q, cache, batch, got = check_attend(new, kv, heads, kv_heads, dim, dtype, causal=causal, max_new=150, seed=dim, pad=(2, 3))
    written = slice(2, 2 + sum(new))
    for _ in range(5):
        assert torch.equal(ob.cache_attend(q, cache, batch, causal=causal)[written], got[written])
    check_attend([1] * 40 + [200], list(range(1, 1601, 40)) + [333], heads, kv_heads, dim, dtype, causal=causal, max_new=200, seed=7)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    out, spread, delta, least, _ = plain.attend(q, want, batch.q_start, batch.kv_len, batch.block_table, dim ** -0.5, causal)
    tol = plain.attend_tolerance(out, spread, delta, least, dtype)
    batch.q_start[3] = -1                                       # bad sequences in the middle: two have no range, the others stay right
    again = torch.full_like(got, 9.0)
    ob.cache_attend(q, cache, batch, causal=causal, out=again)
    assert not status_ok() and status_ok()
    ends = [2 + sum(new[:i]) for i in range(len(new) + 1)]
    assert (again[ends[2]:ends[4]] == 9.0).all()
    # right, not the same bits: the sums are cut into pieces where the whole batch says, each of them within the bound
    for keep in (slice(ends[0], ends[2]), slice(ends[4], ends[-1])):
        assert ((again.cpu().double() - out).abs() <= tol)[keep].all()


@pytest.mark.parametrize("scale,size", [(0.0, 1.0), (-0.1, 1.0), (3.0, 2.0), (1e-3, 300.0), (1e-4, 6e4)])
def test_attend_scales_and_large_queries(scale, size):
    for new, kv in (([1, 2], [300, 90]), ([140], [200])):
        n = gen(8)
        q = (n(sum(new), 4, 64) * size).clamp(-6e4, 6e4)
        for dtype in (F16, BF16):
            check_attend(new, kv, 4, 2, 64, dtype, scale=scale, seed=9, q=q.to(dtype))
    check_attend([1, 2], [300, 90], 4, 2, 64, BF16, scale=1e-30, seed=9, q=(gen(3)(3, 4, 64) * 1e30).to(BF16))


def test_attend_query_views_and_other_streams():
    n = gen(21)
    q, cache, batch, got = check_attend([1, 3, 70], [130, 40, 300], 4, 2, 64, F16, seed=21)
    rows = torch.zeros(74, 7, 80, dtype=F16, device=DEV)
    rows[:, 2:6, 8:72] = q
    assert torch.equal(ob.cache_attend(rows[:, 2:6, 8:72], cache, batch), got)          # strides of 8
    rows[:, 2:6, 3:67] = q
    assert torch.equal(ob.cache_attend(rows[:, 2:6, 3:67], cache, batch), got)          # not aligned: copied
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = [ob.cache_attend(q, cache, batch) for _ in range(3)]
    z = [ob.cache_attend(q, cache, batch) for _ in range(3)]                            # at the same time
    torch.cuda.synchronize()
    for t in y + z:
        assert torch.equal(t, got)


def test_attend_is_the_same_every_time():
    for new, kv in (([1] * 9, [3000, 1, 500, 64, 65, 2000, 7, 900, 1200]), ([150, 40], [800, 2500])):
        q, cache, batch, got = check_attend(new, kv, 8, 2, 128, F16, max_new=max(new), seed=31)
        for _ in range(5):
            assert torch.equal(ob.cache_attend(q, cache, batch), got)


def test_offsets_beyond_32_bits():
    """Pages whose bytes lie beyond 2^32: the last ones of a pool of 4.4e9 bytes a side."""
    H, dim = 16, 128
    pages = (1 << 32) // (64 * H * dim) + 700
    cache = ob.KVCache8.empty(pages, H, dim)
    n = gen(33)
    table = i32(*range(pages - 1, pages - 6, -1)).view(1, 5)
    k, v, q = n(300, H, dim).to(F16), n(300, H, dim).to(F16), n(300, H, dim).to(F16)
    small = ob.KVCache8.empty(5, H, dim)
    for new, kv in ((299, 299), (1, 300)):
        for c, t in ((cache, table), (small, i32(0, 1, 2, 3, 4).view(1, 5))):
            b = ob.CacheBatch(i32(0, new), i32(kv), t, new)
            ob.cache_append(k[kv - new:kv], v[kv - new:kv], c, b)
        a, b = (ob.cache_attend(q[:new], c, ob.CacheBatch(i32(0, new), i32(kv), t, new)) for c, t in ((cache, table), (small, i32(0, 1, 2, 3, 4).view(1, 5))))
        assert torch.equal(a, b) and a.isfinite().all() and float(a.abs().max()) > 0
    assert torch.equal(cache.k_pages.view(torch.uint8)[pages - 5:].flip(0), small.k_pages.view(torch.uint8))
    assert int(cache.k_pages.view(torch.uint8)[:8].sum()) == 0 and status_ok()


# ---- together, as a step uses them ------------------------------------------------------------------------------------------

def test_a_step_captured_twice_and_replayed():
    """norm -> append -> attend for one-token steps, captured in two graphs over one cache and replayed in turn, against the
    same steps run eagerly over a cache of their own."""
    S, heads, H, dim, steps = 3, 8, 2, 64, 70
    n = gen(41)
    freq, weight = ob.rotary_frequencies(dim)[0], (1 + 0.1 * n(heads * dim)).to(F16)
    rows, residual = n(steps, S, heads + 2 * H, dim).to(F16), n(S, heads * dim).to(F16)

    def make():
        return ob.KVCache8.empty(12, H, dim), ob.CacheBatch(i32(0, 1, 2, 3), i32(0, 30, 64), torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4), 1)

    def step(x, cache, batch):
        batch.kv_len.add_(1)
        q = ob.cache_append(x[:, heads:heads + H], x[:, heads + H:], cache, batch, q=x[:, :heads], inv_freq=freq)
        y = ob.cache_attend(q, cache, batch)
        return ob.residual_norm(y.flatten(1), weight, residual=residual)

    cache, batch = make()
    want = [tuple(t.clone() for t in step(x, cache, batch)) for x in rows]
    cache2, batch2 = make()
    x0, x1 = rows[0].clone(), rows[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x0, *make())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g0, g1 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g0):
        y0 = step(x0, cache2, batch2)
    with torch.cuda.graph(g1):
        y1 = step(x1, cache2, batch2)
    for i, x in enumerate(rows):
        buf, g, y = ((x0, g0, y0), (x1, g1, y1))[i % 2]
        buf.copy_(x)
        g.replay()
        assert torch.equal(y[0], want[i][0]) and torch.equal(y[1], want[i][1]), i
    assert torch.equal(cache.k_pages.view(torch.uint8), cache2.k_pages.view(torch.uint8)) and torch.equal(cache.v_scale, cache2.v_scale)
    assert status_ok()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_and_single_steps_agree(dtype):
    """A prompt in one call, in chunks, and token by token: the same tokens reach the same cache up to e4m3's rounding of a
    page's earlier tokens, and each form's attention matches the plain form on the cache that it made."""
    heads, H, dim, T = 6, 2, 64, 150
    n = gen(51)
    rows = n(T, heads + 2 * H, dim).to(dtype)
    freq = ob.rotary_frequencies(dim)[0]
    table = i32(3, 0, 2).view(1, 3)
    for chunks in ([150], [64, 64, 22], [100, 50], [1] * 150):
        cache, at = ob.KVCache8.empty(4, H, dim), 0
        for c in chunks:
            x = rows[at:at + c]
            at += c
            batch = ob.CacheBatch(i32(0, c), i32(at), table, c)
            q = ob.cache_append(x[:, heads:heads + H], x[:, heads + H:], cache, batch, q=x[:, :heads], inv_freq=freq)
            got = ob.cache_attend(q, cache, batch)
            if at == T:
                out, spread, delta, least, _ = plain.attend(q, plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale), batch.q_start, batch.kv_len, table, dim ** -0.5, True)
                assert ((got.cpu().double() - out).abs() <= plain.attend_tolerance(out, spread, delta, least, dtype)).all()
    assert status_ok()


def small_stack(**kw):
    from onebitsparsemul_b200.decode_loop import CachedLlamaStack
    model = CachedLlamaStack(blocks=2, hidden=256, intermediate=512, heads=4, kv_heads=2, head_dim=64, device=DEV, seed=3, **kw)
    for b in model.blocks:
        b.input_norm.copy_(1 + 0.1 * gen(1)(256))
        b.post_norm.copy_(1 + 0.1 * gen(2)(256))
    assert ob.replace_linear_layers(model) == 8
    return model


def test_cached_stack_block_by_block():
    """The packed stack's forward, operator by operator: each output against the plain form of the operator on its own inputs."""
    model = small_stack(rotary=dict(base=5000.0, scaling=("linear", 2.0), layout="interleaved"))
    from onebitsparsemul_b200.decode_loop import CachedDecoder
    dec = CachedDecoder(model, 3, 200)
    new = [70, 1, 33]
    x = gen(4)(sum(new), 256).to(F16)
    seen = []
    keep = {}
    from onebitsparsemul_b200 import block_ops

    def spy(name):
        real = keep[name] = getattr(block_ops, name)

        def call(*args, **kw):
            before = [a.clone() if torch.is_tensor(a) else a for a in args]
            kb = {k: v.clone() if torch.is_tensor(v) else v for k, v in kw.items()}
            cache = plain.Cache(args[2].k_pages, args[2].v_pages, args[2].k_scale, args[2].v_scale) if name == "cache_append" else None
            got = real(*args, **kw)
            seen.append((name, before, kb, [t.clone() if torch.is_tensor(t) else t for t in (got if isinstance(got, tuple) else (got,))], cache, args))
            return got
        setattr(block_ops, name, call)

    for n in ("residual_norm", "cache_append", "cache_attend"):
        spy(n)
    try:
        y = dec.prompt(x, new).clone()
    finally:
        for n, real in keep.items():
            setattr(block_ops, n, real)
    assert [s[0] for s in seen] == ["residual_norm"] + ["cache_append", "cache_attend", "residual_norm", "residual_norm"] * 2
    pos = torch.cat([torch.arange(n) for n in new])
    for name, args, kw, got, cache, live in seen:
        if name == "residual_norm":
            check_norm(got[0], got[1] if len(got) > 1 else None, args[0], args[1], kw.get("residual"), None, 1.0, None, kw["eps"])
        elif name == "cache_append":
            check_rotary(got[0], kw["q"], pos, kw["inv_freq"], "interleaved")
        else:
            c, b = live[1], live[2]
            want = plain.Cache(c.k_pages, c.v_pages, c.k_scale, c.v_scale)
            out, spread, delta, least, _ = plain.attend(args[0], want, b.q_start, b.kv_len, b.block_table, 0.125, True)
            assert ((got[0].cpu().double() - out).abs() <= plain.attend_tolerance(out, spread, delta, least, F16)).all()
    assert torch.equal(y, seen[-1][3][0]) and status_ok()


def test_cached_decoder_prompts_then_graphed_steps():
    """Prompts, graphed steps, another ragged prompt and more steps: the same numbers as the model called eagerly on a cache of
    its own, and refusals when a sequence is full."""
    from onebitsparsemul_b200.decode_loop import CachedDecoder
    model = small_stack()
    a, b = CachedDecoder(model, 3, 150), CachedDecoder(model, 3, 150)
    n = gen(6)

    def eager(x):
        b._grow([1] * 3)
        b.kv_len.add_(1)
        with torch.no_grad():
            return model(x, b.caches, b.step_batch)

    for lengths, steps in (([5, 64, 20], 40), ([30, 0, 3], 5), ([0, 0, 0], 2)):
        x = n(sum(lengths), 256).to(F16)
        assert torch.equal(a.prompt(x, lengths), b.prompt(x, lengths))
        for _ in range(steps):
            x = n(3, 256).to(F16)
            assert torch.equal(a.step(x), eager(x))
    assert a.lengths == b.lengths == a.kv_len.tolist() and status_ok()
    for ca, cb in zip(a.caches, b.caches):
        assert torch.equal(ca.k_pages.view(torch.uint8), cb.k_pages.view(torch.uint8)) and torch.equal(ca.k_scale, cb.k_scale)
    with pytest.raises(ValueError):
        a.prompt(n(100, 256).to(F16), [100, 0, 0])
    with pytest.raises(ValueError):
        a.prompt(n(4, 256).to(F16), [1, 1, 1])
    with pytest.raises(ValueError):
        a.step(n(2, 256).to(F16))
