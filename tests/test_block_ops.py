"""Decoder-block operators: refusals and host logic (CPU only; no kernel runs)."""
import ctypes
import math

import pytest
import torch

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import _lib, build
from tests import block_plain as plain


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build_torch_extension()
    return _lib.load()


P = ctypes.c_void_p(256)          # never dereferenced: validation fails first
ODD = ctypes.c_void_p(264)


def test_norm_refusals_on_the_host(lib):
    def call(x=P, res=P, f32=0, gate=None, post=None, w=P, y=P, h=P, rows=4, hidden=64, dtype=0):
        return lib.onebit_residual_norm(x, hidden, res, hidden, f32, gate, 0, post, w, y, hidden, h, hidden, rows, hidden, 1.0, 1e-6, dtype, None)
    assert call(x=None) == 2 and call(w=None) == 2 and call(y=None) == 2 and call(h=None) == 2
    assert call(res=None, gate=P) == 5 and call(res=None, post=P) == 5
    assert call(hidden=0) == 1 and call(hidden=32769) == 1 and call(rows=-1) == 1
    assert call(dtype=2) == 5
    assert call(rows=0) == 0                       # nothing to do


def test_rotary_refusals_on_the_host(lib):
    def call(x=P, pos=P, freq=P, rd=64, tokens=4, heads=2, dim=64, dtype=0):
        return lib.onebit_rotary(x, 128, 64, P, 128, 64, pos, 0, freq, rd, 0, 1.0, tokens, heads, dim, dtype, None)
    assert call(x=None) == 2 and call(pos=None) == 2 and call(freq=None) == 2
    assert call(rd=63) == 1 and call(rd=66) == 1 and call(rd=-2) == 1
    assert call(dim=513, rd=64) == 1 and call(heads=0) == 1 and call(tokens=-1) == 1 and call(dtype=7) == 5
    assert call(tokens=0) == 0


def append_args(k=P, q=P, q_out=P, freq=P, rd=64, k_pages=P, pages=8, q_start=P, width=4, tokens=4, seqs=2, heads=8, kv_heads=2, dim=64, dtype=0):
    return (k, 128, 64, P, 128, 64, q, 512, 64, q_out, 512, 64, freq, rd, 0, 1.0, k_pages, P, P, P, pages, q_start, P, P, width, width,
            tokens, seqs, heads, kv_heads, dim, dtype, None)


def test_append_refusals_on_the_host(lib):
    def call(**kw):
        return lib.onebit_cache_append(*append_args(**kw))
    assert call(k=None) == 2 and call(q_out=None) == 2 and call(freq=None) == 2 and call(q_start=None) == 2
    assert call(dim=96) == 1 and call(heads=7) == 1 and call(kv_heads=0) == 1 and call(rd=65) == 1 and call(rd=128) == 1
    assert call(seqs=0) == 1 and call(pages=0) == 1 and call(width=0) == 1 and call(tokens=(1 << 24) + 1) == 1
    assert call(dtype=9) == 5 and call(k_pages=ODD) == 5
    assert call(tokens=0) == 0


def test_attend_refusals_on_the_host(lib):
    def call(q=P, q_ts=512, k_pages=P, pages=8, width=4, tokens=4, seqs=2, heads=8, kv_heads=2, dim=64, max_new=0, dtype=0, ws=None, ws_bytes=0, kv_len=P):
        return lib.onebit_cache_attend(q, q_ts, 64, P, 512, 64, k_pages, P, P, P, pages, P, kv_len, P, width, width, tokens, seqs, heads, kv_heads, dim,
                                       max_new, 0.125, 1, dtype, ws, ws_bytes, None)
    assert call(q=None) == 2 and call(kv_len=None) == 2
    assert call(dim=32) == 1 and call(heads=9) == 1 and call(seqs=70000) == 1 and call(width=1 << 25) == 1
    assert call(q=ODD) == 5 and call(q_ts=516) == 5 and call(k_pages=ODD) == 5 and call(dtype=3) == 5
    assert call(tokens=1 << 20, heads=4096, kv_heads=4) == 1          # 2^20 tokens of 1024 heads: 2^40
    assert call(tokens=0) == 0
    need = lib.onebit_cache_attend_workspace(4, 4, 2, 8, 2, 64, 0)
    if need:
        assert call() == 4 and b"workspace" in lib.onebit_last_error()
        assert call(ws=P, ws_bytes=need - 1) == 4
        assert call(ws=ODD, ws_bytes=need) == 4


def test_python_layer_refuses_cpu_tensors():
    x, w = torch.zeros(2, 64, dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    with pytest.raises(ob.OneBitError):
        ob.residual_norm(x, w)
    with pytest.raises(ob.OneBitError):
        ob.rotary_tokens(x.view(2, 1, 64), torch.zeros(2, dtype=torch.int32), torch.ones(4, dtype=torch.float64))
    cache = ob.KVCache8.empty(2, 1, 64, device="cpu")
    batch = ob.CacheBatch(torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32))
    with pytest.raises(ob.OneBitError):
        ob.cache_append(x.view(2, 1, 64), x.view(2, 1, 64), cache, batch)
    with pytest.raises(ob.OneBitError):
        ob.cache_attend(x.view(2, 1, 64), cache, batch)
    with pytest.raises(TypeError):
        ob.residual_norm(x.float(), w.float())


def test_cache_and_batch_refuse_wrong_tensors():
    c = ob.KVCache8.empty(3, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        ob.KVCache8.empty(3, 2, 96, device="cpu")
    with pytest.raises(ValueError):
        ob.KVCache8(c.k_pages, c.k_pages.transpose(2, 3)[:, :1], c.k_scale, c.v_scale)
    with pytest.raises(TypeError):
        ob.KVCache8(c.k_pages.view(torch.uint8), c.v_pages, c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        ob.KVCache8(c.k_pages, c.v_pages, c.k_scale[:, :1], c.v_scale)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table = torch.zeros((2, 3), dtype=torch.int32)
    ob.CacheBatch(i(0, 1, 2), i(4, 4), table)
    for bad in ((i(0, 1), i(4, 4), table), (i(0, 1, 2), i(4), table), (i(0, 1, 2), i(4, 4), table[0])):
        with pytest.raises(ValueError):
            ob.CacheBatch(*bad)
    with pytest.raises(TypeError):
        ob.CacheBatch(i(0, 1, 2).long(), i(4, 4), table)
    with pytest.raises(ValueError):
        ob.CacheBatch(i(0, 1, 2), i(4, 4), table, max_new=0)
    with pytest.raises(ValueError):
        ob.CacheBatch(i(0, 1, 2), i(4, 4), torch.zeros((3, 2), dtype=torch.int32).T)


def test_frequencies():
    f, m = ob.rotary_frequencies(128, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0 and f.shape == (64,)
    assert f[0] == 1.0 and abs(float(f[32]) - 0.01) < 1e-15
    lin, _ = ob.rotary_frequencies(128, scaling=("linear", 4), device="cpu")
    assert torch.equal(lin, f / 4)
    base, _ = ob.rotary_frequencies(128, scaling=("base", 8), device="cpu")
    assert base[0] == 1.0 and abs(float(base[-1] / f[-1]) - 1 / 8) < 1e-12
    part, m = ob.rotary_frequencies(128, scaling=("parts", 16, 8192), device="cpu")
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(part[turns > 32], f[turns > 32]) and torch.allclose(part[turns < 1], f[turns < 1] / 16, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (part[mid] < f[mid]).all() and (part[mid] > f[mid] / 16).all()
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    for bad in ((63,), (0,), (128, 10000.0, ("linear", 0.5)), (128, 10000.0, ("none", 2)), (128, -1.0), (2, 10000.0, ("base", 2)), (128, 1e4, ("parts", 2, 0))):
        with pytest.raises(ValueError):
            ob.rotary_frequencies(*bad, device="cpu")


def test_plain_e4m3_rounding_is_torch_s():
    x = torch.cat((torch.linspace(-460, 460, 20001), torch.linspace(-0.04, 0.04, 20001))).double().clamp(-448, 448)
    want = x.float().to(torch.float8_e4m3fn).float().double()
    assert torch.equal(plain.to_e4m3(x.float().double()), want)
    for amax, e in ((448.0, 0), (448.0000001, 1), (224.0, -1), (1e-20, -32), (1e20, 32), (0.0, -32)):
        assert plain.scale_for(amax) == 2.0 ** e
