"""The decoder-block operators have no derivatives: whatever would lose one is refused, before anything else is looked at (no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import onebitsparsemul_b200 as ob
from onebitsparsemul_b200 import build

F16 = torch.float16


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_torch_extension()


def calls(change):
    """Every tensor argument of every operator, one at a time through `change`."""
    x, w, r = torch.ones(2, 64, dtype=F16), torch.ones(64, dtype=F16), torch.ones(2, 64)
    k, pos, freq = torch.ones(2, 1, 64, dtype=F16), torch.arange(2), torch.ones(4, dtype=torch.float64)
    norm = dict(x=x, weight=w, residual=r, gate=w.clone(), post_weight=w.clone(), out=torch.empty_like(x), residual_out=torch.empty_like(r))
    for name in norm:
        yield lambda name=name: ob.residual_norm(**{**norm, name: change(norm[name])})
    rotary = dict(x=k, inv_freq=freq, out=torch.empty_like(k))
    for name in rotary:
        yield lambda name=name: ob.rotary_tokens(**{**rotary, "positions": pos, name: change(rotary[name])})
    batch = ob.CacheBatch(torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))
    cache = ob.KVCache8.empty(1, 1, 64, device="cpu")

    def scaled(which):
        return ob.KVCache8(cache.k_pages, cache.v_pages, *(change(t) if i == which else t for i, t in enumerate((cache.k_scale, cache.v_scale))))
    append = dict(k=k, v=k.clone(), q=k.clone(), inv_freq=freq, q_out=torch.empty_like(k))
    for name in append:
        yield lambda name=name: ob.cache_append(**{**append, "cache": cache, "batch": batch, name: change(append[name])})
    attend = dict(q=k, out=torch.empty_like(k))
    for name in attend:
        yield lambda name=name: ob.cache_attend(**{**attend, "cache": cache, "batch": batch, name: change(attend[name])})
    for which in range(2):
        yield lambda which=which: ob.cache_append(k, k, scaled(which), batch)
        yield lambda which=which: ob.cache_attend(k, scaled(which), batch)


def test_tangents_are_refused():
    with forward_ad.dual_level():
        n = 0
        for call in calls(lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):            # which does not stop forward mode
                call()
            n += 1
        assert n == 21
        for call in calls(lambda t: forward_ad.unpack_dual(forward_ad.make_dual(t, torch.ones_like(t))).primal):
            with pytest.raises(ob.OneBitError):                 # nothing to lose: on to the missing device
                call()


def test_gradients_are_refused():
    for call in calls(lambda t: t.clone().requires_grad_()):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ob.OneBitError):
            call()
