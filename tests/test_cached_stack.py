"""`CachedLlamaStack` and `CachedDecoder` on the host (no GPU)."""
import pytest
import torch
import torch.nn as nn

from onebitsparsemul_b200 import build
from onebitsparsemul_b200.decode_loop import CachedDecoder, CachedLlamaStack


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_torch_extension()


class Stub(nn.Module):
    """A model that keeps the batches that it was called with."""

    def __init__(self, hidden=8):
        super().__init__()
        self.hidden, self.batches = hidden, []

    def make_caches(self, pages, device):
        return []

    def forward(self, x, caches, batch):
        self.batches.append((batch, None if x.is_cuda else batch.kv_len.tolist()))
        return x + 0


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


def test_a_prompt_s_table_is_as_wide_as_its_longest_sequence():
    model = Stub()
    dec = CachedDecoder(model, 3, 32768, device="cpu")
    for lengths, width in (([5, 64, 0], 1), ([0, 1, 0], 2), ([3, 0, 2000], 32), ([0, 0, 48], 32), ([1, 1, 1], 33), ([0, 30000, 0], 470)):
        dec.prompt(torch.zeros(sum(lengths), 8), lengths)
        batch, kv_len = model.batches[-1]
        assert (batch.seqs, batch.width) == (3, width) and tuple(batch.block_table.shape) == (3, width)
        assert kv_len == dec.lengths and max(kv_len) <= 64 * width
        assert torch.equal(batch.block_table, dec.table[:, :width])


class Failing(Stub):
    fails = False

    def forward(self, x, caches, batch):
        if self.fails:
            raise RuntimeError("out of memory")
        return super().forward(x, caches, batch)


def test_a_prompt_that_raises_leaves_the_sequences_as_they_were():
    model = Failing()
    dec = CachedDecoder(model, 2, 100, device="cpu")
    dec.prompt(torch.zeros(7, 8), [3, 4])
    model.fails = True
    with pytest.raises(RuntimeError):
        dec.prompt(torch.zeros(2, 8), [1, 1])
    for x, lengths in ((torch.zeros(2, 9), [1, 1]), (torch.zeros(2, 8), [1, 2]), (torch.zeros(2), [1, 1]), (torch.zeros(200, 8), [100, 100]), (torch.zeros(2, 8), [3, -1])):
        with pytest.raises(ValueError):
            dec.prompt(x, lengths)
    assert dec.lengths == dec.kv_len.tolist() == [3, 4]
    model.fails = False
    dec.prompt(torch.zeros(2, 8), [1, 1])
    assert dec.lengths == dec.kv_len.tolist() == model.batches[-1][1] == [4, 5]
    assert dec.prompt(torch.zeros(0, 8), [0, 0]).shape == (0, 8) and dec.lengths == [4, 5]


@pytest.mark.gpu
def test_a_step_that_raises_leaves_the_sequences_as_they_were():
    class Once(Failing):
        calls = 0

        def forward(self, x, caches, batch):
            self.calls += 1
            if self.calls == 2:
                raise RuntimeError("out of memory")
            return x + batch.kv_len[:, None]
    model = Once()
    dec = CachedDecoder(model, 2, 100)
    with pytest.raises(RuntimeError):
        dec.step(torch.zeros(2, 8, device="cuda"))
    assert dec.graph is None and dec.lengths == dec.kv_len.tolist() == [0, 0]
    for i in range(3):
        y = dec.step(torch.full((2, 8), 10.0 * i, device="cuda"))
        assert (y == 10.0 * i + i + 1).all() and dec.lengths == dec.kv_len.tolist() == [i + 1] * 2


@pytest.mark.gpu
def test_a_step_is_captured_on_its_device_s_stream(monkeypatch):
    """Without a stream of its own a capture takes one of the device that was current when the first graph of the process was made."""
    seen, real = [], torch.cuda.graph

    def graph(*args, stream=None, **kw):
        seen.append(stream)
        return real(*args, stream=stream, **kw)
    monkeypatch.setattr(torch.cuda, "graph", graph)
    device = torch.cuda.device_count() - 1
    dec = CachedDecoder(Stub(), 2, 100, device=f"cuda:{device}")
    for i in range(2):
        assert (dec.step(torch.full((2, 8), float(i), device=dec.device)) == i).all()
    assert [s.device.index for s in seen] == [device] and dec.kv_len.tolist() == [2, 2]
