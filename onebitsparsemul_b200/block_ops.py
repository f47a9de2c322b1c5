"""What stands between the linear layers of a decoder block: the residual add with its norms, rotary positions, an 8-bit
key/value cache and the attention that reads it. Every function is one call into libonebitmul (hand-written sm_100a
kernels); the reference leaves these parts to the model it patches (tests/python/test_model_replace.py:22-44).

Serving only, like the packed layers: no function records a gradient, and one that is handed a tensor that wants a
gradient (with gradients enabled) refuses it. Tensors are float16 or bfloat16 on one CUDA device; work is queued on that
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

from . import _lib
from ._lib import OneBitError

__all__ = ["residual_norm", "rotary_frequencies", "rotary_tokens", "KVCache8", "CacheBatch", "cache_append", "cache_attend"]

PAGE_TOKENS = 64
_TYPES = {torch.float16: _lib.DENSE_F16, torch.bfloat16: _lib.DENSE_BF16}
_LAYOUTS = {"half": 0, "interleaved": 1}


def _check(tensors, device):
    """Every tensor on `device`, none of them waiting for a gradient."""
    if device.type != "cuda":
        raise OneBitError("no CUDA tensor: this library has no CPU path")
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"tensors on different devices: {t.device} and {device}")
        if grad and t.requires_grad:
            raise ValueError("a tensor wants a gradient, and this operator has none: call it under torch.no_grad()")


def _call(fn, device, *args):
    """fn(*args, stream) on the current stream of `device`."""
    if device.index == torch.cuda.current_device():
        _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def _type_code(dtype):
    try:
        return _TYPES[dtype]
    except KeyError:
        raise TypeError(f"expected float16 or bfloat16, got {dtype}") from None


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- norms -------------------------------------------------------------------------------------------------------------

def _rows(t, hidden):
    """t as (rows, hidden) with contiguous rows."""
    t = t if t.dim() == 2 else t.reshape(-1, hidden)
    return t if t.stride(1) == 1 or hidden == 1 else t.contiguous()


def residual_norm(x, weight, residual=None, gate=None, residual_scale=1.0, post_weight=None, eps=1e-6, out=None, residual_out=None):
    """The residual add with the norms around it, in one pass over the rows (``onebit_residual_norm``):

        u = x                                       or, with post_weight, x / sqrt(mean(x^2) + eps) * post_weight
        h = residual + residual_scale * gate * u
        y = h / sqrt(mean(h^2) + eps) * weight

    x: (..., hidden) float16 / bfloat16, hidden <= 32768. weight, post_weight: (hidden,) of x's type. residual: x's shape,
    x's type or float32. gate: (hidden,) or x's shape, x's type. Returns (y, h), y in x's type and h in residual's; without a
    residual only y, the norm of x. `out` / `residual_out` (contiguous) receive y / h and may be x / residual themselves.
    Arithmetic and sums are float32; y is the norm of h before h's own rounding."""
    lib = _lib.load()
    code, dev = _type_code(x.dtype), x.device
    _check((x, weight, residual, gate, post_weight, out, residual_out), dev)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 32768:
        raise ValueError("x must be (..., hidden) with 1 <= hidden <= 32768")
    hidden, shape = x.shape[-1], x.shape
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is not None and (w.dtype != x.dtype or w.shape != (hidden,)):
            raise ValueError(f"{name} must be ({hidden},) of x's type")
    if not (eps >= 0 and math.isfinite(eps) and math.isfinite(residual_scale)):
        raise ValueError("eps must be finite and not negative, residual_scale finite")
    if residual is None:
        if gate is not None or post_weight is not None or residual_out is not None or residual_scale != 1.0:
            raise ValueError("gate, post_weight, residual_scale and residual_out need a residual")
    else:
        if residual.shape != shape or residual.dtype not in (x.dtype, torch.float32):
            raise ValueError("residual must have x's shape and x's type or float32")
        if residual_out is None:
            residual_out = torch.empty(shape, dtype=residual.dtype, device=dev)
        elif residual_out.shape != shape or residual_out.dtype != residual.dtype or not residual_out.is_contiguous():
            raise ValueError("residual_out must be contiguous with residual's shape and type")
    gate_stride = 0
    if gate is not None:
        if gate.dtype != x.dtype or gate.shape not in ((hidden,), shape):
            raise ValueError("gate must be (hidden,) or x's shape, of x's type")
        per_row = gate.shape == shape and gate.dim() > 1
        gate = _rows(gate, hidden) if per_row else gate.contiguous()
        gate_stride = gate.stride(0) if per_row else 0
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=dev)
    elif out.shape != shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous with x's shape and type")
    x2 = _rows(x, hidden)
    r2 = None if residual is None else _rows(residual, hidden)
    weight = weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    rows = x2.shape[0]
    if rows:
        _call(lib.onebit_residual_norm, dev, x2.data_ptr(), x2.stride(0), _ptr(r2), 0 if r2 is None else r2.stride(0),
              r2 is not None and r2.dtype == torch.float32, _ptr(gate), gate_stride, _ptr(post_weight), weight.data_ptr(),
              out.data_ptr(), hidden, _ptr(residual_out), hidden, rows, hidden, residual_scale, eps, code)
    return out if residual is None else (out, residual_out)


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


def _heads(t, name, tokens=None, heads=None, dim=None):
    if t.dim() != 3 or any(want is not None and got != want for got, want in zip(t.shape, (tokens, heads, dim))):
        want = ", ".join("?" if w is None else str(w) for w in (tokens, heads, dim))
        raise ValueError(f"{name} must be ({want}), got {tuple(t.shape)}")


def _inner(t):
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _rotation(inv_freq, layout, head_dim):
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 vector (32 bits lose the angles of far positions)")
    if 2 * inv_freq.numel() > head_dim:
        raise ValueError(f"{inv_freq.numel()} pairs do not fit a head of {head_dim}")
    return 2 * inv_freq.numel()


def rotary_tokens(x, positions, inv_freq, layout="half", magnitude=1.0, out=None):
    """x (tokens, heads, head_dim <= 512) with the first 2 * len(inv_freq) values of every head turned by its token's position
    (``onebit_rotary``): pairs (i, i + len(inv_freq)) for "half", (2i, 2i + 1) for "interleaved"; the rest is passed on.
    positions: (tokens,) int32 or int64, any sign. inv_freq: float64, see `rotary_frequencies`. x may be a view into the rows
    of a fused projection; `out` may be x itself or any tensor of its shape with contiguous heads that does not overlap x."""
    lib = _lib.load()
    code, dev = _type_code(x.dtype), x.device
    _check((x, positions, inv_freq, out), dev)
    _heads(x, "x")
    tokens, heads, dim = x.shape
    if not 1 <= dim <= 512 or not 1 <= heads <= 4096 or tokens > 1 << 24:
        raise ValueError("x must be (tokens <= 2^24, heads <= 4096, head_dim <= 512)")
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,):
        raise ValueError("positions must be (tokens,) int32 or int64")
    rotary_dim = _rotation(inv_freq, layout, dim)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    elif out.shape != x.shape or out.dtype != x.dtype or out.stride(2) != 1:
        raise ValueError("out must have x's shape and type and contiguous heads")
    if out.data_ptr() == x.data_ptr() and out.stride() != x.stride():
        raise ValueError("out overlaps x without being x")
    x, positions = _inner(x), positions.contiguous()
    if tokens:
        _call(lib.onebit_rotary, dev, x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
              positions.data_ptr(), positions.dtype == torch.int64, inv_freq.data_ptr(), rotary_dim, _LAYOUTS[layout], magnitude,
              tokens, heads, dim, code)
    return out


# ---- the cache ----------------------------------------------------------------------------------------------------------------

class KVCache8:
    """The tensors of an 8-bit key/value cache (layout in the module's docstring), checked once here. Bytes that no append
    has written must be finite codes (`empty` makes zeros); a page may be given to another sequence at any time."""

    __slots__ = ("k_pages", "v_pages", "k_scale", "v_scale", "pages", "kv_heads", "head_dim", "device")

    def __init__(self, k_pages, v_pages, k_scale, v_scale):
        if k_pages.dim() != 4 or k_pages.shape[2] != PAGE_TOKENS or k_pages.shape[3] not in (64, 128):
            raise ValueError("k_pages must be (pages, kv_heads, 64, 64 or 128)")
        pages, heads, _, dim = k_pages.shape
        if v_pages.shape != (pages, heads, dim, PAGE_TOKENS) or k_scale.shape != (pages, heads) or v_scale.shape != (pages, heads):
            raise ValueError(f"with {pages} pages of {heads} heads of {dim}: v_pages must be ({pages}, {heads}, {dim}, 64), scales ({pages}, {heads})")
        if k_pages.dtype != torch.float8_e4m3fn or v_pages.dtype != torch.float8_e4m3fn or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise TypeError("pages must be float8_e4m3fn, scales float32")
        for t in (k_pages, v_pages, k_scale, v_scale):
            if not t.is_contiguous() or t.device != k_pages.device:
                raise ValueError("pages and scales must be contiguous, on one device")
        if pages < 1 or not 1 <= heads <= 4096:
            raise ValueError("need at least one page and 1 to 4096 heads")
        self.k_pages, self.v_pages, self.k_scale, self.v_scale = k_pages, v_pages, k_scale, v_scale
        self.pages, self.kv_heads, self.head_dim, self.device = pages, heads, dim, k_pages.device

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
        block_table  (sequences, width) page of each 64 tokens; entries behind a sequence's length are never read

    max_new: an upper bound of the sequences' new tokens, if the caller knows one (a decode step: 1). It picks the
    kernel, no result depends on it. Rows outside q_start's range are padding: not read, and their outputs not written. The
    values stay on the device and may be rewritten between steps (a captured step reads them anew). A page number or a range
    that lies outside its tensor is left out, and ``onebit_check_device_status`` reports it."""

    __slots__ = ("q_start", "kv_len", "block_table", "max_new", "seqs", "width", "device")

    def __init__(self, q_start, kv_len, block_table, max_new=None):
        if q_start.dtype != torch.int32 or kv_len.dtype != torch.int32 or block_table.dtype != torch.int32:
            raise TypeError("q_start, kv_len and block_table must be int32")
        if block_table.dim() != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1 or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
            raise ValueError("block_table must be (sequences, width), at least 1 x 1, with contiguous rows")
        seqs, width = block_table.shape
        if q_start.shape != (seqs + 1,) or kv_len.shape != (seqs,) or not q_start.is_contiguous() or not kv_len.is_contiguous():
            raise ValueError(f"with {seqs} sequences: q_start must be ({seqs + 1},), kv_len ({seqs},), both contiguous")
        if q_start.device != block_table.device or kv_len.device != block_table.device:
            raise ValueError("q_start, kv_len and block_table must be on one device")
        if seqs > 1 << 16 or width > 1 << 24:
            raise ValueError("at most 2^16 sequences of 2^24 pages")
        if max_new is not None and max_new < 1:
            raise ValueError("max_new must be positive")
        self.q_start, self.kv_len, self.block_table = q_start, kv_len, block_table
        self.max_new, self.seqs, self.width, self.device = max_new or 0, seqs, width, block_table.device


def cache_append(k, v, cache, batch, q=None, inv_freq=None, layout="half", magnitude=1.0, q_out=None):
    """Store the step's keys and values (tokens, kv_heads, head_dim) in the cache, keys turned by their positions if `inv_freq` is
    given, and turn the queries q (tokens, heads, head_dim) too, all in one launch (``onebit_cache_append``). Returns the turned
    queries (None without q); `q_out` may be q itself.

    The scale of a page and head is the smallest power of two (2^-32 to 2^32) that brings the largest finite |value| of its
    tokens into e4m3's range; when a step's tokens make it grow, the page's earlier tokens are re-scaled. Infinities are
    stored as the largest value of the page's scale. A NaN key stays NaN; a token with a NaN value has it stored as 0 and its key
    made NaN, so that the queries that see the token answer NaN and no others. A page that a step writes must belong to one
    sequence of the batch only."""
    lib = _lib.load()
    code, dev = _type_code(k.dtype), k.device
    _check((k, v, q, inv_freq, q_out), dev)
    if cache.device != dev or batch.device != dev:
        raise ValueError("cache, batch and tensors must be on one device")
    tokens, H, D = k.shape[0], cache.kv_heads, cache.head_dim
    _heads(k, "k", tokens, H, D)
    _heads(v, "v", tokens, H, D)
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise TypeError("q, k and v must have one type")
    if tokens > 1 << 24:
        raise ValueError("at most 2^24 tokens")
    rotary_dim = 0 if inv_freq is None else _rotation(inv_freq, layout, D)
    heads = H
    if q is not None:
        _heads(q, "q", tokens, None, D)
        heads = q.shape[1]
        if inv_freq is None:
            raise ValueError("q is only turned: it needs inv_freq")
        if heads % H or not 1 <= heads <= 4096:
            raise ValueError(f"{heads} query heads are no multiple of {H} cache heads")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(2) != 1:
            raise ValueError("q_out must have q's shape and type and contiguous heads")
        if q_out.data_ptr() == q.data_ptr() and q_out.stride() != q.stride():
            raise ValueError("q_out overlaps q without being q")
        q = _inner(q)
    elif q_out is not None:
        raise ValueError("q_out without q")
    k, v = _inner(k), _inner(v)
    if tokens:
        qs, os_ = ((0, 0), (0, 0)) if q is None else (q.stride(), q_out.stride())
        ks, vs = k.stride(), v.stride()
        _call(lib.onebit_cache_append, dev, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _ptr(q), qs[0], qs[1], _ptr(q_out), os_[0], os_[1],
              _ptr(inv_freq), rotary_dim, _LAYOUTS.get(layout, 0), magnitude, cache.k_pages.data_ptr(), cache.v_pages.data_ptr(),
              cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.pages, batch.q_start.data_ptr(), batch.kv_len.data_ptr(),
              batch.block_table.data_ptr(), batch.block_table.stride(0), batch.width, tokens, batch.seqs, heads, H, D, code)
    return q_out


def _aligned(t):
    """t with 16-byte aligned heads, copied if it has none."""
    if t.stride(2) == 1 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def cache_attend(q, cache, batch, scale=None, causal=True, out=None):
    """softmax(scale * q k^T) v of the step's queries q (tokens, heads, head_dim) over their sequences' cached tokens
    (``onebit_cache_attend``); call it after `cache_append` of the same batch. Query head h reads cache head
    h // (heads // kv_heads). causal: a token sees the positions up to its own (the new tokens are the last ones of the
    sequence), else the whole sequence. scale: head_dim ** -0.5 by default. A row that sees nothing is zero. `out`: contiguous,
    q's shape and type."""
    lib = _lib.load()
    code, dev = _type_code(q.dtype), q.device
    _check((q, out), dev)
    if cache.device != dev or batch.device != dev:
        raise ValueError("cache, batch and tensors must be on one device")
    _heads(q, "q", None, None, cache.head_dim)
    tokens, heads, D = q.shape
    if heads % cache.kv_heads or not 1 <= heads <= 4096:
        raise ValueError(f"{heads} query heads are no multiple of {cache.kv_heads} cache heads")
    if tokens > 1 << 24:
        raise ValueError("at most 2^24 tokens")
    scale = D ** -0.5 if scale is None else scale
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous (and 16-byte aligned) with q's shape and type")
    if tokens:
        q = _aligned(q)
        qs = q.stride()
        need = lib.onebit_cache_attend_workspace(batch.width, tokens, batch.seqs, heads, cache.kv_heads, D, batch.max_new)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _call(lib.onebit_cache_attend, dev, q.data_ptr(), qs[0], qs[1], out.data_ptr(), heads * D, D, cache.k_pages.data_ptr(), cache.v_pages.data_ptr(),
              cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.pages, batch.q_start.data_ptr(), batch.kv_len.data_ptr(),
              batch.block_table.data_ptr(), batch.block_table.stride(0), batch.width, tokens, batch.seqs, heads, cache.kv_heads, D,
              batch.max_new, scale, causal, code, _ptr(ws), need)
    return out
