"""What stands between the linear layers of a decoder block: the residual add with its norms, rotary positions, an 8-bit
key/value cache and the attention that reads it. Every function is one call into libonebitmul (hand-written sm_100a
kernels); the reference leaves these parts to the model it patches (tests/python/test_model_replace.py:22-44).

Serving only, like the packed layers: no function records a gradient, and one that is handed a tensor that wants a
gradient (with gradients enabled) or carries a forward-mode tangent refuses it. Tensors are float16 or bfloat16 on one CUDA device; work is queued on that
device's current stream, nothing synchronises, and every call can be captured in a CUDA graph.

The cache. `KVCache8` holds pages of 64 tokens: keys (pages, kv_heads, 64, head_dim), values transposed
(pages, kv_heads, head_dim, 64), both float8_e4m3fn, and one power-of-two float32 scale for each page and head of either; a
stored value stands for code * scale. `CacheBatch` says which new tokens a step brings and where each sequence's pages
are; the same batch goes to `cache_append` and then to `cache_attend`:

    cache = KVCache8.empty(pages, kv_heads, head_dim)
    batch = CacheBatch(q_start, kv_len, block_table)       # int32 on the device; kv_len counts the new tokens
    q = cache_append(k, v, cache, batch, q=q, inv_freq=inv_freq)
    y = cache_attend(q, cache, batch)
"""
from __future__ import annotations

import math

import torch

__all__ = ["residual_norm", "rotary_frequencies", "rotary_tokens", "KVCache8", "CacheBatch", "cache_append", "cache_attend"]

PAGE_TOKENS = 64
_extension = None


def _ext():
    """The torch extension, whose C++ side checks the tensors and calls libonebitmul."""
    global _extension
    if _extension is None:
        try:
            import onebit_sparse_cuda
        except ImportError as e:
            raise ImportError("the onebit_sparse_cuda extension is missing: build it with `python -m onebitsparsemul_b200.build --all` "
                              "(or `make torch_ext`)") from e
        _extension = onebit_sparse_cuda
    return _extension


# ---- norms -------------------------------------------------------------------------------------------------------------

def residual_norm(x, weight, residual=None, gate=None, residual_scale=1.0, post_weight=None, eps=1e-6, out=None, residual_out=None):
    """The residual add with the norms around it, in one pass over the rows (``onebit_residual_norm``):

        u = x                                       or, with post_weight, x / sqrt(mean(x^2) + eps) * post_weight
        h = residual + residual_scale * gate * u
        y = h / sqrt(mean(h^2) + eps) * weight

    x: (..., hidden) float16 / bfloat16, hidden <= 32768. weight, post_weight: (hidden,) of x's type. residual: x's shape,
    x's type or float32. gate: (hidden,) or x's shape, x's type. Returns (y, h), y in x's type and h in residual's; without a
    residual only y, the norm of x. `out` / `residual_out` (contiguous) receive y / h and may be x / residual themselves.
    Arithmetic and sums are float32; y is the norm of h before h's own rounding."""
    return _ext().residual_norm(x, weight, residual, gate, residual_scale, post_weight, eps, out, residual_out)


# ---- rotary positions -----------------------------------------------------------------------------------------------------

def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """Angular frequencies of the rotary_dim / 2 pairs, float64 on `device`, and the magnitude that goes with them.
    Pair i turns by base^(-2 i / rotary_dim) per position. `scaling` for contexts longer than the model was trained on:

        None                                  the plain frequencies
        ("linear", factor)                    every frequency / factor
        ("base", factor)                      base * factor^(rotary_dim / (rotary_dim - 2)): the slowest pair / factor, the first unchanged
        ("parts", factor, length[, lo, hi])   pairs that turn fewer than lo (1) times over the original `length` are slowed by
                                              factor, more than hi (32) times are left, in between a linear blend; the
                                              magnitude is 0.1 ln(factor) + 1, else 1
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    kind, factor = (None, 1.0) if scaling is None else (scaling[0], float(scaling[1]))
    if not (base > 0 and factor >= 1.0):
        raise ValueError("base must be positive, the factor at least 1")
    if kind == "base":
        if rotary_dim == 2:
            raise ValueError("scaling the base needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    magnitude = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "parts":
        length = float(scaling[2])
        lo, hi = (float(scaling[3]), float(scaling[4])) if len(scaling) > 3 else (1.0, 32.0)
        if not (length > 0 and hi > lo):
            raise ValueError("parts scaling needs a positive length and hi > lo")
        keep = ((length * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f / factor * (1 - keep) + f * keep
        magnitude = 0.1 * math.log(factor) + 1.0
    elif kind not in (None, "base"):
        raise ValueError(f"unknown scaling {kind!r}")
    return f.to(device), magnitude


def rotary_tokens(x, positions, inv_freq, layout="half", magnitude=1.0, out=None):
    """x (tokens, heads, head_dim <= 512) with the first 2 * len(inv_freq) values of every head turned by its token's position
    (``onebit_rotary``): pairs (i, i + len(inv_freq)) for "half", (2i, 2i + 1) for "interleaved"; the rest is passed on.
    positions: (tokens,) int32 or int64, any sign. inv_freq: float64, see `rotary_frequencies`. x may be a view into the rows
    of a fused projection; `out` may be x itself or any tensor of its shape with contiguous heads that does not overlap x."""
    return _ext().rotary_tokens(x, positions, inv_freq, layout, magnitude, out)


# ---- the cache ----------------------------------------------------------------------------------------------------------------

class KVCache8:
    """The tensors of an 8-bit key/value cache (layout in the module's docstring), checked once here. Bytes that no append
    has written must be finite codes (`empty` makes zeros); a page may be given to another sequence at any time."""

    __slots__ = ("k_pages", "v_pages", "k_scale", "v_scale", "pages", "kv_heads", "head_dim")

    def __init__(self, k_pages, v_pages, k_scale, v_scale):
        self.pages, self.kv_heads, self.head_dim = _ext().check_cache(k_pages, v_pages, k_scale, v_scale)
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale

    @classmethod
    def empty(cls, pages, kv_heads, head_dim, device="cuda"):
        def zeros(*shape, dtype=torch.uint8):
            return torch.zeros(shape, dtype=dtype, device=device)

        return cls(zeros(pages, kv_heads, PAGE_TOKENS, head_dim).view(torch.float8_e4m3fn), zeros(pages, kv_heads, head_dim, PAGE_TOKENS).view(torch.float8_e4m3fn),
                   zeros(pages, kv_heads, dtype=torch.float32), zeros(pages, kv_heads, dtype=torch.float32))

    def tokens(self, block_table_row, count):
        """The first `count` tokens behind one row of a block table as float32 (count, kv_heads, head_dim) keys and values
        (a helper for inspection, in torch)."""
        page = block_table_row[: -(-count // PAGE_TOKENS)].long()

        def values(pages, scale):
            return pages.view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * scale[page][..., None, None]

        k = values(self.k_pages, self.k_scale).permute(0, 2, 1, 3).flatten(0, 1)
        v = values(self.v_pages, self.v_scale).permute(0, 3, 1, 2).flatten(0, 1)
        return k[:count], v[:count]


class CacheBatch:
    """Which new tokens a step brings, and where the sequences' pages are. All int32 on the device:

        q_start      (sequences + 1,)  rows q_start[s] .. q_start[s + 1] of the step's tokens belong to sequence s
        kv_len       (sequences,)      tokens of the sequence in the cache, the new ones included
        block_table  (sequences, width) page of each 64 tokens; entries behind a sequence's length do not matter

    max_new: an upper bound of the sequences' new tokens, if the caller knows one (a decode step: 1). It picks the
    kernels of both, as the table's width does attention's (the narrower, the better short batches are dealt out); results are right whatever it
    says, though sums may be taken in another order. Rows outside q_start's range are padding: what they hold does not matter, and their
    outputs are not written. The values stay on the device and may be rewritten between steps (a captured step reads them anew). A page
    number that lies outside its tensor is left out, and so is a sequence whose range does or that runs backwards;
    the other sequences are not touched by that, and ``onebit_check_device_status`` reports it."""

    __slots__ = ("q_start", "kv_len", "block_table", "max_new", "seqs", "width")

    def __init__(self, q_start, kv_len, block_table, max_new=None):
        if max_new is not None and max_new < 1:
            raise ValueError("max_new must be positive")
        self.seqs, self.width = _ext().check_batch(q_start, kv_len, block_table)
        self.q_start, self.kv_len, self.block_table, self.max_new = q_start, kv_len, block_table, max_new or 0


def cache_append(k, v, cache, batch, q=None, inv_freq=None, layout="half", magnitude=1.0, q_out=None):
    """Store the step's keys and values (tokens, kv_heads, head_dim) in the cache, keys turned by their positions if `inv_freq` is
    given, and turn the queries q (tokens, heads, head_dim) too, in one launch, or two where most sequences bring up to three tokens
    and some more (``onebit_cache_append_ex``). Returns the turned queries (None without q); `q_out` may be q itself.

    The scale of a page and head is the smallest power of two (2^-32 to 2^32) that brings the largest finite |value| of its
    tokens into e4m3's range; when a step's tokens make it grow, the page's earlier tokens are re-scaled. Infinities are
    stored as the largest value of the page's scale. A NaN key stays NaN; a token with a NaN value has it stored as 0 and its key
    made NaN, so that the queries that see the token answer NaN and no others. A page that a step writes must stand once in the
    batch's table: in one sequence, in one place."""
    return _ext().cache_append(k, v, cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale, batch.q_start, batch.kv_len, batch.block_table,
                               batch.max_new, q, inv_freq, layout, magnitude, q_out)


def cache_attend(q, cache, batch, scale=None, causal=True, out=None):
    """softmax(scale * q k^T) v of the step's queries q (tokens, heads, head_dim) over their sequences' cached tokens
    (``onebit_cache_attend``); call it after `cache_append` of the same batch. Query head h reads cache head
    h // (heads // kv_heads). causal: a token sees the positions up to its own (the new tokens are the last ones of the
    sequence), else the whole sequence. scale: head_dim ** -0.5 by default. A row that sees nothing, or nothing but scores of
    minus infinity, is zero. `out`: contiguous, q's shape and type, apart from q and the cache."""
    return _ext().cache_attend(q, cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale, batch.q_start, batch.kv_len, batch.block_table,
                               batch.max_new, scale, causal, out)
