"""`CachedLlamaStack` and `CachedDecoder` on the host (no GPU)."""
import torch
import torch.nn as nn

from onebitsparsemul_b200.decode_loop import CachedLlamaStack


def small(**kw):
    return CachedLlamaStack(blocks=1, hidden=64, intermediate=64, heads=1, head_dim=64, **kw)


def test_frequencies_stay_in_64_bits():
    want = small().inv_freq.clone()
    assert want.dtype == torch.float64
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.float().half(), lambda m: m.to("cpu", torch.bfloat16), lambda m: nn.Sequential(m).half()[0],
                   lambda m: m.to("cpu"), lambda m: m.double()):
        model = small()
        assert change(model) is model
        assert model.inv_freq.dtype == torch.float64 and torch.equal(model.inv_freq, want)
    model = small().to(torch.bfloat16)
    assert model.norm.dtype == model.blocks[0].input_norm.dtype == model.blocks[0].qkv_proj.weight.dtype == torch.bfloat16
    assert list(small().state_dict()) == list(model.state_dict()) and "inv_freq" in model.state_dict()
    other = small(rotary=dict(base=500.0)).half()
    other.load_state_dict(small().half().state_dict())
    assert torch.equal(other.inv_freq, want)
    assert small().to("meta").inv_freq.device.type == "meta"
