"""Batches whose ranges are not inside the call's rows, or run backwards: reported, and without an effect on the other sequences."""
import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib
from tests import block_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


def status():
    lib = _lib.load()
    return lib.onebit_check_device_status(), lib.onebit_last_error()


def i32(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def singles(bad):
    q = list(range(201))
    q[150] = bad
    return q, 200, [s for s in range(200) if s not in (149, 150)]


# q_start, rows of the call, the sequences that stand
BATCHES = [([1000, 1005, 1010], 10, []),                        # all of it behind the rows
           ([0, 300, 420, 9000, 9001], 430, [0, 1]),             # behind them from the third sequence on
           ([-5, 300, 420], 420, [1]),
           ([0, 300, -1, 300, 420], 420, [0, 3]),                # the third starts before everything
           ([0, 300, 7, 300, 420], 420, [0, 3]),                 # the second runs backwards; the third, from 7, overlaps the first
           ([0, 300, 2 ** 31 - 1, 300, 420], 420, [0, 3]), ([0, 300, -2 ** 31, 300, 420], 420, [0, 3]),
           singles(-1), singles(100000)]


@pytest.mark.parametrize("which", range(len(BATCHES)))
def test_append_of_ranges_out_of_order(which):
    starts, rows, good = BATCHES[which]
    S, H, dim = len(starts) - 1, 2, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(which)
    k, v, q = (torch.randn(rows, h, dim, generator=g, device=DEV).half() for h in (H, H, 4))
    new = [starts[s + 1] - starts[s] if s in good else 1 for s in range(S)]
    kv = [n + 9 * (s % 3) for s, n in enumerate(new)]
    width = max(-(-x // 64) for x in kv)
    table = torch.randperm(S * width, generator=g, device=DEV).to(torch.int32).view(S, width)
    cache = ob.KVCache8.empty(S * width, H, dim)
    want = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    batch = ob.CacheBatch(i32(starts), i32(kv), table)
    assert status()[0] == 0
    out = torch.full_like(q, 7.0)
    ob.cache_append(k, v, cache, batch, q=q, inv_freq=torch.zeros(dim // 2, dtype=torch.float64, device=DEV), q_out=out)
    code, text = status()
    assert code == 7 and b"page number or a sequence offset" in text and status()[0] == 0
    overlapped = 7 in starts                                    # a row that two sequences claim has no right answer
    if not overlapped:
        for s in good:
            want.append(k.double().cpu(), v.double().cpu(), torch.tensor(([0] * s + [starts[s], starts[s + 1]] + [starts[s + 1]] * S)[:S + 1]),
                        torch.tensor([kv[t] if t == s else 0 for t in range(S)]), table)
        assert torch.equal(cache.k_scale.cpu().double(), want.ks) and torch.equal(cache.v_scale.cpu().double(), want.vs)
        assert torch.equal(cache.k_pages.float().cpu().double(), want.k) and torch.equal(cache.v_pages.float().cpu().double(), want.v)
    else:
        for s in good:
            gk, gv = cache.tokens(table[s], kv[s])
            n = new[s]
            err = (gv[kv[s] - n:] - v[starts[s]:starts[s + 1]].float()).abs()
            # e4m3: 2^-4 of the value, 2^-10 of the scale among the subnormals
            assert (err <= v[starts[s]:starts[s + 1]].float().abs() * 2.0 ** -4 + float(cache.v_scale.max()) * 2.0 ** -9).all()
    written = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for s in good:
        written[starts[s]:starts[s + 1]] = True
    assert torch.equal(out[written], q[written]) and (out[~written] == 7.0).all()       # frequencies of 0: passed on


@pytest.mark.parametrize("hint", [None, 1, 300])
@pytest.mark.parametrize("which", range(len(BATCHES)))
def test_attention_of_ranges_out_of_order(which, hint):
    starts, rows, good = BATCHES[which]
    S, H, dim, heads = len(starts) - 1, 2, 64, 8
    g = torch.Generator(device=DEV)
    g.manual_seed(which + 50)
    new = [starts[s + 1] - starts[s] if s in good else 1 for s in range(S)]
    kv = [n + 9 * (s % 3) + (200 if S < 9 else 0) for s, n in enumerate(new)]
    width = max(-(-x // 64) for x in kv)
    pages = S * width
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(S, width)
    code = lambda *s: (torch.randn(*s, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    cache = ob.KVCache8(code(pages, H, 64, dim), code(pages, H, dim, 64), torch.full((pages, H), 2.0 ** -7, device=DEV), torch.full((pages, H), 2.0 ** -7, device=DEV))
    q = torch.randn(rows, heads, dim, generator=g, device=DEV).half()
    batch = ob.CacheBatch(i32(starts), i32(kv), table, hint)
    assert status()[0] == 0
    out = torch.full_like(q, 9.0)
    ob.cache_attend(q, cache, batch, out=out)
    answer, text = status()
    assert answer == 7 and b"page number or a sequence offset" in text and status()[0] == 0
    pc = plain.Cache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale)
    written = torch.zeros(rows, dtype=torch.bool)
    for s in good[:3] + good[-60:]:
        mine = slice(starts[s], starts[s + 1])
        want, spread, delta, least, _ = plain.attend(q[mine], pc, torch.tensor([0, new[s]]), torch.tensor([kv[s]]), table[s:s + 1], dim ** -0.5, True)
        tol = plain.attend_tolerance(want, spread, delta, least, torch.float16)
        got = out[mine].cpu().double()
        if 7 in starts and s == 0:                              # rows from 7 on are claimed by two sequences
            got, want, tol = got[:7], want[:7], tol[:7]
        assert ((got - want).abs() <= tol).all(), s
    for s in good:
        written[starts[s]:starts[s + 1]] = True
    assert (out.cpu()[~written] == 9.0).all()
