"""A Llama-shaped stack of linear layers and a CUDA-graph decode loop over it.

The reference's model-replace demo (tests/python/test_model_replace.py:22-44) walks a TinyLlama checkpoint and
swaps every ``nn.Linear`` for a ``BinaryLinear_2_4``. The checkpoint is not part of that repository; what the
flow exercises is the set of linear layers of a decoder block -- q/k/v/o (hidden x hidden), gate/up
(intermediate x hidden), down (hidden x intermediate) -- called one token at a time. `LlamaShapedStack` is
exactly that set with random weights; the attention and normalisation arithmetic between the layers, which the
one-bit path does not touch, is replaced by cheap element-wise glue with the same data flow, so that every
linear layer reads the output of an earlier one.

`CachedLlamaStack` is the whole decoder stack: the same linear layers with the operators of `block_ops` between them -- residual
adds with their norms, rotary positions and attention over an 8-bit key/value cache -- and `CachedDecoder` runs it for a
batch of sequences, prompts eagerly and single tokens from a CUDA graph.

`GraphedDecoder` captures one step of the (replaced) stack in a CUDA graph and replays it per token: the
few-token kernels then run back to back without host launches between them, each grid starting while its
predecessor drains (programmatic dependent launch). This is the measurement of the decode regime as a model
sees it: a single call moves 3-9 MB and costs less at HBM speed than a kernel launch.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import block_ops


class LlamaShapedBlock(nn.Module):
    """The seven linear layers of a Llama-style decoder block (no biases, like the original).

    With ``fused=True`` the three projections that read the same input are one layer (``qkv_proj``, 3 * hidden rows) and
    so are gate and up (``gate_up_proj``, 2 * intermediate rows), as serving stacks lay them out: four GEMMs per
    block instead of seven, each with more row blocks to spread over the SMs. The arithmetic is the same."""

    def __init__(self, hidden: int = 4096, intermediate: int = 11008, dtype=torch.float16, device=None, fused: bool = False):
        super().__init__()
        kw = dict(bias=False, dtype=dtype, device=device)
        self.fused, self.hidden, self.intermediate = fused, hidden, intermediate
        if fused:
            self.qkv_proj = nn.Linear(hidden, 3 * hidden, **kw)
            self.gate_up_proj = nn.Linear(hidden, 2 * intermediate, **kw)
        else:
            self.q_proj, self.k_proj = nn.Linear(hidden, hidden, **kw), nn.Linear(hidden, hidden, **kw)
            self.v_proj = nn.Linear(hidden, hidden, **kw)
            self.gate_proj, self.up_proj = nn.Linear(hidden, intermediate, **kw), nn.Linear(hidden, intermediate, **kw)
        self.o_proj = nn.Linear(hidden, hidden, **kw)
        self.down_proj = nn.Linear(intermediate, hidden, **kw)

    def forward(self, x):
        """x: (tokens, hidden). Element-wise glue stands in for attention and normalisation."""
        if self.fused:
            q, k, v = self.qkv_proj(x).split(self.hidden, dim=-1)
        else:
            q, k, v = self.q_proj(x), self.k_proj(x), self.v_proj(x)
        h = x + self.o_proj(torch.tanh(q) * torch.sigmoid(k) + 0.5 * v)
        h = h * torch.rsqrt(h.float().pow(2).mean(-1, keepdim=True) + 1e-5).to(h.dtype)
        if self.fused:
            gate, up = self.gate_up_proj(h).split(self.intermediate, dim=-1)
        else:
            gate, up = self.gate_proj(h), self.up_proj(h)
        return h + self.down_proj(F.silu(gate) * up)


class LlamaShapedStack(nn.Module):
    def __init__(self, blocks: int = 4, hidden: int = 4096, intermediate: int = 11008, dtype=torch.float16, device=None, seed: int = 0,
                 fused: bool = False):
        super().__init__()
        self.hidden, self.intermediate = hidden, intermediate
        self.blocks = nn.ModuleList([LlamaShapedBlock(hidden, intermediate, dtype, device, fused) for _ in range(blocks)])
        g = torch.Generator(device="cpu")
        g.manual_seed(seed)
        with torch.no_grad():
            for p in self.parameters():                          # N(0, 1 / fan_in): activations keep their scale
                p.copy_((torch.randn(p.shape, generator=g) / p.shape[1] ** 0.5).to(p.dtype))

    def forward(self, x):
        for b in self.blocks:
            x = b(x)
        return x

    def linear_layers(self):
        return [m for m in self.modules() if isinstance(m, nn.Linear) or type(m).__name__ == "BinaryLinear_2_4"]


class GraphedDecoder:
    """One decode step of `model` for a fixed number of tokens, captured in a CUDA graph.

    The first calls run eagerly (they make the library allocate its per-device status word and mark the packed
    weights as long-lived); the capture follows. `step(x)` copies x into the graph's input, replays, and returns
    the graph's output tensor (overwritten by the next step)."""

    def __init__(self, model: nn.Module, tokens: int, hidden: int, device="cuda", warmup: int = 3):
        self.model = model
        self.x = torch.zeros((tokens, hidden), dtype=torch.float16, device=device)
        side = torch.cuda.Stream(device=device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side), torch.no_grad():
            for _ in range(warmup):
                self.model(self.x)
        torch.cuda.current_stream(device).wait_stream(side)
        torch.cuda.synchronize(device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph), torch.no_grad():
            self.y = self.model(self.x)

    def step(self, x):
        self.x.copy_(x)
        self.graph.replay()
        return self.y


def measure_decode(model: nn.Module, hidden: int, tokens: int = 1, steps: int = 50, device="cuda"):
    """Device time of one decode step through the graph, per token step and per linear layer."""
    dec = GraphedDecoder(model, tokens, hidden, device)
    x = torch.randn((tokens, hidden), device=device, dtype=torch.float32).to(torch.float16)
    for _ in range(3):
        dec.step(x)
    torch.cuda.synchronize(device)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(steps):
        dec.graph.replay()
    e1.record()
    torch.cuda.synchronize(device)
    us = e0.elapsed_time(e1) * 1e3 / steps
    layers = [m for m in model.modules() if type(m).__name__ == "BinaryLinear_2_4"]
    packed_bytes = sum(m.bits_tile.numel() + m.meta_tile.numel() for m in layers)
    return {"tokens": tokens, "linear_layers": len(layers), "us_per_step": us, "us_per_linear_layer": us / max(1, len(layers)),
            "steps_per_s": 1e6 / us, "tokens_per_s": tokens * 1e6 / us, "packed_weight_bytes": packed_bytes,
            "weight_gbs": packed_bytes / us / 1e3}


# ---- the stack with its attention and norms --------------------------------------------------------------------------------

class CachedLlamaBlock(nn.Module):
    """A Llama-style decoder block that serves: fused q/k/v and gate/up projections (four linear layers, which
    `replace_linear_layers` can pack), two norms, rotary positions, attention over an 8-bit cache. Heads may share keys and
    values (kv_heads < heads)."""

    def __init__(self, hidden: int, intermediate: int, heads: int, kv_heads: int, head_dim: int, eps: float = 1e-6, dtype=torch.float16, device=None):
        super().__init__()
        kw = dict(bias=False, dtype=dtype, device=device)
        self.heads, self.kv_heads, self.head_dim, self.eps, self.intermediate = heads, kv_heads, head_dim, eps, intermediate
        self.qkv_proj = nn.Linear(hidden, (heads + 2 * kv_heads) * head_dim, **kw)
        self.o_proj = nn.Linear(heads * head_dim, hidden, **kw)
        self.gate_up_proj = nn.Linear(hidden, 2 * intermediate, **kw)
        self.down_proj = nn.Linear(intermediate, hidden, **kw)
        self.register_buffer("input_norm", torch.ones(hidden, dtype=dtype, device=device))
        self.register_buffer("post_norm", torch.ones(hidden, dtype=dtype, device=device))

    def forward(self, y, h, cache, batch, inv_freq, next_norm, layout="half", magnitude=1.0):
        """y (tokens, hidden): the normed input; h: the residual stream, updated in place; next_norm: the weight of the norm
        behind the block. Returns y for the next block."""
        H, K = self.heads, self.kv_heads
        qkv = self.qkv_proj(y).view(-1, H + 2 * K, self.head_dim)
        q = qkv[:, :H]
        block_ops.cache_append(qkv[:, H:H + K], qkv[:, H + K:], cache, batch, q=q, inv_freq=inv_freq, layout=layout, magnitude=magnitude, q_out=q)
        a = self.o_proj(block_ops.cache_attend(q, cache, batch).flatten(1))
        y, h = block_ops.residual_norm(a, self.post_norm, residual=h, eps=self.eps, residual_out=h)
        gate, up = self.gate_up_proj(y).split(self.intermediate, dim=-1)
        y, h = block_ops.residual_norm(self.down_proj(F.silu(gate) * up), next_norm, residual=h, eps=self.eps, residual_out=h)
        return y


class CachedLlamaStack(nn.Module):
    """A stack of `CachedLlamaBlock` and its last norm. `rotary`: keyword arguments of `rotary_frequencies` (base, scaling), and
    "layout"."""

    def __init__(self, blocks: int = 4, hidden: int = 4096, intermediate: int = 11008, heads: int = 32, kv_heads: int | None = None, head_dim: int = 128,
                 dtype=torch.float16, device=None, seed: int = 0, rotary: dict | None = None):
        super().__init__()
        self.hidden, self.heads, self.kv_heads, self.head_dim = hidden, heads, kv_heads or heads, head_dim
        self.blocks = nn.ModuleList([CachedLlamaBlock(hidden, intermediate, heads, self.kv_heads, head_dim, dtype=dtype, device=device) for _ in range(blocks)])
        self.register_buffer("norm", torch.ones(hidden, dtype=dtype, device=device))
        rotary = dict(rotary or {})
        self.layout = rotary.pop("layout", "half")
        freq, self.magnitude = block_ops.rotary_frequencies(head_dim, device="cpu" if device is None else device, **rotary)
        self.register_buffer("inv_freq", freq)
        g = torch.Generator(device="cpu")
        g.manual_seed(seed)
        with torch.no_grad():
            for p in self.parameters():                          # N(0, 1 / fan_in): activations keep their scale
                p.copy_((torch.randn(p.shape, generator=g) / p.shape[1] ** 0.5).to(p.dtype))

    def _apply(self, fn, *args, **kw):
        """`half()`, `to(dtype)` and the like: the frequencies move, but stay in 64 bits, which far positions need."""
        freq = self.inv_freq
        super()._apply(fn, *args, **kw)
        if self.inv_freq.dtype != freq.dtype:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self

    def make_caches(self, pages: int, device="cuda"):
        return [block_ops.KVCache8.empty(pages, self.kv_heads, self.head_dim, device=device) for _ in self.blocks]

    def forward(self, x, caches, batch):
        """x (tokens, hidden): the step's token embeddings, laid out as `batch` says. Returns the normed output of every token."""
        h = x.clone()
        y = block_ops.residual_norm(x, self.blocks[0].input_norm, eps=self.blocks[0].eps)
        for i, (block, cache) in enumerate(zip(self.blocks, caches)):
            following = self.blocks[i + 1].input_norm if i + 1 < len(self.blocks) else self.norm
            y = block(y, h, cache, batch, self.inv_freq, following, self.layout, self.magnitude)
        return y


class CachedDecoder:
    """Serves `sequences` sequences of up to `max_len` tokens with a `CachedLlamaStack`: `prompt(x, lengths)` appends that many
    tokens to each sequence (eagerly), `step(x)` one token to every sequence, replayed from a CUDA graph that is captured by the
    first step. Each sequence has pages of its own. The output of `step` is overwritten by the next one."""

    def __init__(self, model: CachedLlamaStack, sequences: int, max_len: int, device="cuda"):
        self.model, self.sequences, self.max_len, self.device = model, sequences, max_len, device
        width = -(-max_len // block_ops.PAGE_TOKENS)
        i32 = dict(dtype=torch.int32, device=device)
        self.caches = model.make_caches(sequences * width, device)
        self.table = torch.arange(sequences * width, **i32).view(sequences, width)
        self.kv_len = torch.zeros(sequences, **i32)
        self.lengths = [0] * sequences                           # the host's copy
        self.step_batch = block_ops.CacheBatch(torch.arange(sequences + 1, **i32), self.kv_len, self.table, max_new=1)
        self.graph = None

    def _grown(self, new):
        """The lengths with `new` tokens more, or a refusal."""
        if len(new) != self.sequences or min(new) < 0 or any(a + b > self.max_len for a, b in zip(self.lengths, new)):
            raise ValueError(f"{new} new tokens do not fit {self.sequences} sequences of at most {self.max_len} that hold {self.lengths}")
        return [a + b for a, b in zip(self.lengths, new)]

    def _grow(self, new):
        self.lengths = self._grown(new)

    def prompt(self, x, lengths):
        """x (sum(lengths), hidden): the sequences' new tokens one after the other. Returns (tokens, hidden). A call that raises
        leaves the sequences as long as they were."""
        lengths = [int(n) for n in lengths]
        if tuple(x.shape) != (sum(lengths), self.model.hidden):
            raise ValueError(f"x of {tuple(x.shape)} for lengths {lengths} and a hidden size of {self.model.hidden}")
        grown = self._grown(lengths)
        if not x.shape[0]:
            return x.new_empty(x.shape)
        start = torch.zeros(self.sequences + 1, dtype=torch.int32)
        start[1:] = torch.tensor(lengths).cumsum(0)
        start = start.to(self.device)
        kv_len = self.kv_len + start.diff()
        # as wide as the longest sequence needs: attention deals out its work, and cuts a long cache into parts, by the table's width
        width = -(-max(grown) // block_ops.PAGE_TOKENS)
        batch = block_ops.CacheBatch(start, kv_len, self.table[:, :width], max_new=max(lengths))
        with torch.no_grad():
            y = self.model(x, self.caches, batch)
        self.kv_len.copy_(kv_len)
        self.lengths = grown
        return y

    def _step(self):
        self.kv_len.add_(1)
        return self.model(self.x, self.caches, self.step_batch)

    def _capture(self, x):
        """The graph of a step. The first calls load kernels and mark the packed weights as long-lived: they run outside the capture, on
        the sequences as they are, and the lengths are put back. What they wrote, the step itself writes again."""
        self.x = x.clone()
        before = self.kv_len.clone()
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        try:
            with torch.cuda.stream(side), torch.no_grad():
                for _ in range(2):
                    self._step()
                    self.kv_len.copy_(before)
        finally:
            torch.cuda.current_stream(self.device).wait_stream(side)
            self.kv_len.copy_(before)
            torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side), torch.no_grad():        # this device's stream, whichever is current
            self.y = self._step()
        self.graph = graph

    def step(self, x):
        """x (sequences, hidden): one token for every sequence. A call that raises leaves the sequences as long as they were."""
        if tuple(x.shape) != (self.sequences, self.model.hidden):
            raise ValueError(f"x must be ({self.sequences}, {self.model.hidden})")
        grown = self._grown([1] * self.sequences)
        if self.graph is None:
            self._capture(x)
        self.x.copy_(x)
        self.graph.replay()
        self.lengths = grown
        return self.y
