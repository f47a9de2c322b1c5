"""Cases of the operators around the one-bit linear layers of a decoder block: the residual add with its norms, rotary
positions, the 8-bit key/value cache that a step appends to, and the attention that reads it.

`run` computes each operator in its plain form (elementary torch operations in 32 bits, angles in 64) or, where `own` is
true, through the framework's entry points. The cache is the framework's: pages of 64 tokens, keys (pages, heads, 64, dim)
and values (pages, heads, dim, 64) in e4m3, and one power-of-two scale for each page and head."""
import math
import random

import torch

if torch.cuda.is_available():
    torch.backends.cuda.matmul.allow_tf32 = False

own = False

BLOCK = 64                       # tokens of a cache page
E4M3_MAX = 448.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the norm before the next linear layer of a 4096-wide decode step: latency
        dict(name="norm_token", op="norm", rows=1, hidden=4096, dtype="fp16", residual="fp16", gate="none", post=False, alpha=1.0),
        # a prompt through a block with a norm after it, a channel gate and a scaled residual
        dict(name="norm_prompt", op="norm", rows=8192, hidden=4096, dtype="fp16", residual="fp16", gate="channel", post=True, alpha=0.5),
        # odd width, 32-bit residual stream, a gate for every token and channel
        dict(name="norm_odd", op="norm", rows=1111, hidden=2047, dtype="bf16", residual="fp32", gate="full", post=True, alpha=0.7),
        # queries inside a fused projection's rows (32 heads out of 48), a prompt
        dict(name="rotary_prompt", op="rotary", tokens=4096, heads=32, row_heads=48, dim=128, rotary=128, layout="half", dtype="fp16", far=8192,
             factor=1.0),
        # few tokens at far positions, half of the head, neighbouring pairs, stretched frequencies
        dict(name="rotary_far", op="rotary", tokens=37, heads=20, row_heads=20, dim=128, rotary=64, layout="interleaved", dtype="bf16", far=1000000,
             factor=16.0),
        # a decode step of 64 sequences writes its tokens
        dict(name="append_step", op="append", seqs=64, new=1, ragged=True, kv=2048, heads=32, kv_heads=8, dim=128, rotary=128, layout="half",
             dtype="fp16", lens=1),
        # ragged prompts on top of earlier turns
        dict(name="append_prompt", op="append", seqs=8, new=2048, ragged=True, kv=4096, heads=32, kv_heads=8, dim=128, rotary=64, layout="interleaved",
             dtype="bf16", lens=2),
        # one sequence, one token, 32 heads of its own each: the 4096-wide stack's step
        dict(name="attend_one", op="attend", seqs=1, new=1, ragged=False, kv=4096, heads=32, kv_heads=32, dim=128, dtype="fp16", causal=True, lens=3),
        # a serving batch with ragged contexts and shared heads
        dict(name="attend_batch", op="attend", seqs=64, new=1, ragged=True, kv=8192, heads=32, kv_heads=8, dim=128, dtype="fp16", causal=True, lens=4),
        # a few drafted tokens for each sequence, narrow heads, an odd group
        dict(name="attend_draft", op="attend", seqs=7, new=4, ragged=True, kv=5000, heads=30, kv_heads=10, dim=64, dtype="bf16", causal=True, lens=5),
        # a whole prompt
        dict(name="attend_prompt", op="attend", seqs=1, new=8192, ragged=False, kv=8192, heads=32, kv_heads=8, dim=128, dtype="fp16", causal=True, lens=6),
        # chunks of prompts over long contexts
        dict(name="attend_chunk", op="attend", seqs=3, new=512, ragged=True, kv=16384, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lens=7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "append", "attend", "attend"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "norm":
        hidden = _log(rng, 64, 16384)
        hidden = hidden // 8 * 8 if rng.random() < 0.7 else hidden
        return dict(op=op, rows=_log(rng, 1, max(1, 8192 * 4096 // hidden)), hidden=hidden, dtype=dtype, residual=rng.choice((dtype, dtype, "fp32")),
                    gate=rng.choice(("none", "channel", "full")), post=rng.random() < 0.5, alpha=round(rng.uniform(0.1, 1.5), 3))
    dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 8, 10, 16))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 8))
    if heads * dim == 3 << 10:
        heads += kv_heads
    rotary = rng.choice((dim, dim, dim // 2, dim // 4))
    layout = rng.choice(("half", "interleaved"))
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, max(1, 4096 * 32 * 128 // (heads * dim))), heads=heads, row_heads=heads + rng.choice((0, 2)) * kv_heads, dim=dim,
                    rotary=rotary, layout=layout, dtype=dtype, far=_log(rng, 8192, 1000000), factor=rng.choice((1.0, 4.0, 16.0)))
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = rng.choice((1, _log(rng, 1, max(1, 8192 // seqs))))
        return dict(op=op, seqs=seqs, new=new, ragged=rng.random() < 0.8, kv=new + _log(rng, 1, 2048), heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                    layout=layout, dtype=dtype, lens=rng.randrange(1 << 20))
    kind = rng.choice(("step", "draft", "prompt"))
    if kind == "prompt":
        seqs = _log(rng, 1, 8)
        new = _log(rng, 9, 4096 // seqs)
        kv = new + rng.choice((0, _log(rng, 1, 8192 // seqs)))
    else:
        seqs = _log(rng, 1, 64)
        new = 1 if kind == "step" else rng.randrange(2, 9)
        kv = new + _log(rng, 1, 8192)
    return dict(op=op, seqs=seqs, new=new, ragged=rng.random() < 0.8, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                causal=rng.random() < 0.9, lens=rng.randrange(1 << 20))


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence: the first has the full lengths, the others go down to one token."""
    r = random.Random(case["lens"])
    n, kv = [case["new"]], [case["kv"]]
    for _ in range(case["seqs"] - 1):
        n.append(_log(r, 1, case["new"]) if case["ragged"] else case["new"])
        kv.append(n[-1] + r.randint(0, case["kv"] - case["new"]) if case["ragged"] else case["kv"])
    return n, kv


def work(case):
    """Bytes: every input once and every output once. Flops: those of the matrix products, or of the arithmetic of a value."""
    op = case["op"]
    if op == "norm":
        values = case["rows"] * case["hidden"]
        wide = 4 if case["residual"] == "fp32" else 2
        return {"bytes": values * (2 + wide + wide + 2 + (2 if case["gate"] == "full" else 0)), "flops": values * 12}
    if op == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": values * 4 + case["tokens"] * 8, "flops": values * 3}
    n, kv = _lengths(case)
    token = case["kv_heads"] * case["dim"]
    if op == "append":
        tokens = sum(n)
        return {"bytes": tokens * (case["heads"] * case["dim"] * 4 + token * 2 * 3), "flops": tokens * (case["heads"] * case["dim"] + token) * 4}
    pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(n, kv))
    return {"bytes": sum(kv) * token * 2 + sum(n) * case["heads"] * case["dim"] * 4, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _frequencies(rotary, base, factor, original, device):
    """Angular frequency of each pair, in 64 bits. Stretched contexts: a pair that turns fewer than once over the original
    length is slowed down by `factor`, one that turns over 32 times is left, and between them the two are blended."""
    f = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    if factor == 1.0:
        return f
    keep = ((original * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f / factor * (1 - keep) + f * keep


def _pow2_scale(amax):
    """The smallest power of two, from 2^-32 to 2^32, that brings amax to e4m3's range."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -32)).clamp(-32, 32)
    return torch.ldexp(torch.ones_like(amax), e)


def _paged(case, g, dev):
    """A cache with the tokens of earlier steps (and, for attention, of this one), and the step's batch."""
    n, kv = _lengths(case)
    S, H, D = case["seqs"], case["kv_heads"], case["dim"]
    blocks = [-(-x // BLOCK) for x in kv]
    width, used = max(blocks), sum(blocks)
    pool = used + 3
    order = torch.randperm(pool, generator=g, device=dev)[:used].to(torch.int32)
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev)[None] < torch.tensor(blocks, device=dev)[:, None]] = order
    # which tokens of each page are there
    filled = torch.tensor(kv, device=dev) if case["op"] == "attend" else torch.tensor(kv, device=dev) - torch.tensor(n, device=dev)
    held = (filled[:, None] - BLOCK * torch.arange(width, device=dev)[None]).clamp(0, BLOCK)
    page_held = torch.zeros(pool, dtype=torch.int64, device=dev)
    page_held[table[table >= 0].long()] = held[table >= 0]
    live = torch.arange(BLOCK, device=dev)[None] < page_held[:, None]                       # (pool, 64)
    channel = torch.where(torch.rand(H, 1, D, generator=g, device=dev) < 0.03, 4.0, 1.0)    # a few loud key channels
    k = torch.randn(pool, H, BLOCK, D, generator=g, device=dev) * channel * live[:, None, :, None]
    k_scale = _pow2_scale(k.abs().amax((2, 3)))
    k_pages = (k / k_scale[..., None, None]).to(torch.float8_e4m3fn)
    del k
    v = torch.randn(pool, H, D, BLOCK, generator=g, device=dev) * live[:, None, None, :]
    v_scale = _pow2_scale(v.abs().amax((2, 3)))
    v_pages = (v / v_scale[..., None, None]).to(torch.float8_e4m3fn)
    del v
    start = torch.tensor([sum(n[:i]) for i in range(S + 1)], dtype=torch.int32, device=dev)
    return dict(k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale, q_start=start,
                kv_len=torch.tensor(kv, dtype=torch.int32, device=dev), table=table, tokens=sum(n), max_new=max(n), channel=channel)


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = dict(op=case["op"])
    if case["op"] == "norm":
        R, N = case["rows"], case["hidden"]
        s.update(x=normal(R, N).to(dt), residual=(2 * normal(R, N)).to(DTYPES[case["residual"]]), weight=(1 + 0.1 * normal(N)).to(dt),
                 post=(1 + 0.1 * normal(N)).to(dt) if case["post"] else None,
                 gate=None if case["gate"] == "none" else torch.sigmoid(normal(N) if case["gate"] == "channel" else normal(R, N)).to(dt),
                 alpha=case["alpha"], eps=1e-6)
        return s
    if case["op"] == "rotary":
        rows = normal(case["tokens"], case["row_heads"], case["dim"]).to(dt)
        first = torch.randint(0, case["far"] - case["tokens"] + 1, (1,), generator=g, device=dev)
        s.update(x=rows[:, : case["heads"]], positions=first + torch.arange(case["tokens"], device=dev),
                 freq=_frequencies(case["rotary"], 10000.0, case["factor"], 8192, dev), layout=case["layout"],
                 magnitude=1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0)
        return s
    s.update(_paged(case, g, dev))
    T, Hq, H, D = s["tokens"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        rows = normal(T, Hq + 2 * H, D)                   # one row of the fused q, k, v projection for each token
        rows[:, Hq:Hq + H] *= s["channel"][:, 0]
        rows = rows.to(dt)
        s.update(q=rows[:, :Hq], k=rows[:, Hq:Hq + H], v=rows[:, Hq + H:], freq=_frequencies(case["rotary"], 10000.0, 1.0, 8192, dev), layout=case["layout"])
    else:
        s.update(q=normal(T, Hq, D).to(dt), scale=D ** -0.5, causal=case["causal"])
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"norm": _norm, "rotary": _rotary, "append": _append, "attend": _attend}[s["op"]](s)


def _own(s):
    import onebitsparsemul_b200 as ob
    if s["op"] == "norm":
        return ob.residual_norm(s["x"], s["weight"], residual=s["residual"], gate=s["gate"], residual_scale=s["alpha"], post_weight=s["post"], eps=s["eps"])
    if s["op"] == "rotary":
        return ob.rotary_tokens(s["x"], s["positions"], s["freq"], layout=s["layout"], magnitude=s["magnitude"])
    cache = ob.KVCache8(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    batch = ob.CacheBatch(s["q_start"], s["kv_len"], s["table"], s["max_new"])
    if s["op"] == "append":
        q = ob.cache_append(s["k"], s["v"], cache, batch, q=s["q"], inv_freq=s["freq"], layout=s["layout"])
        return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]
    return ob.cache_attend(s["q"], cache, batch, scale=s["scale"], causal=s["causal"])


def _norm(s):
    u = s["x"].float()
    if s["post"] is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + s["eps"]) * s["post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = s["residual"].float() + s["alpha"] * u
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    return y.to(s["x"].dtype), h.to(s["residual"].dtype)


def _turned(x, positions, freq, layout, magnitude):
    """x (tokens, heads, dim) in 32 bits with its first 2 * len(freq) values turned."""
    angle = positions.double()[:, None, None] * freq
    c, s = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    half = freq.numel()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _rotary(s):
    return _turned(s["x"].float(), s["positions"], s["freq"], s["layout"], s["magnitude"]).to(s["x"].dtype)


def _tokens(s):
    """Sequence, place among the new tokens and position of every new token."""
    t = torch.arange(s["tokens"], device=s["q_start"].device)
    seq = (t[:, None] >= s["q_start"][None, 1:]).sum(1)
    place = t - s["q_start"][seq]
    n = s["q_start"][1:] - s["q_start"][:-1]
    return seq, place, s["kv_len"][seq] - n[seq] + place, n


def _append(s):
    seq, place, pos, n = _tokens(s)
    q = _turned(s["q"].float(), pos, s["freq"], s["layout"], 1.0).to(s["q"].dtype)
    k = _turned(s["k"].float(), pos, s["freq"], s["layout"], 1.0)
    v = s["v"].float()
    block = (pos // BLOCK).long()
    page, slot = s["table"][seq, block].long(), (pos % BLOCK).long()
    pool, H, D = s["k_pages"].shape[0], s["k_pages"].shape[1], s["k_pages"].shape[3]
    fresh = block * BLOCK >= (s["kv_len"] - n)[seq]                       # the block holds no token of an earlier call
    touched = torch.zeros(pool, dtype=torch.bool, device=k.device)
    touched[page] = True
    new_page = torch.zeros(pool, dtype=torch.bool, device=k.device)
    new_page[page] = fresh

    def quantise(x, pages, scale, transposed):
        amax = torch.zeros(pool, H, device=x.device).scatter_reduce(0, page[:, None].expand(-1, H), x.abs().amax(-1), "amax")
        want = _pow2_scale(amax)
        to = torch.where(touched[:, None], torch.where(new_page[:, None], want, torch.maximum(scale, want)), scale)
        ratio = torch.where(new_page[:, None], torch.zeros_like(to), scale / to)
        old = pages.float() * ratio[..., None, None]
        old = torch.where(touched[:, None, None, None], old, pages.float()).to(torch.float8_e4m3fn)
        code = (x / to[page][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        old = old.view(torch.uint8)
        if transposed:
            old[page, :, :, slot] = code
        else:
            old[page, :, slot] = code
        pages.view(torch.uint8).copy_(old)
        scale.copy_(to)

    quantise(k, s["k_pages"], s["k_scale"], False)
    quantise(v, s["v_pages"], s["v_scale"], True)
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _attend(s):
    seq, place, pos, n = _tokens(s)
    S, P = s["table"].shape
    H, D = s["k_pages"].shape[1], s["k_pages"].shape[3]
    Hq, Q, L = s["q"].shape[1], s["max_new"], P * BLOCK
    page = s["table"].clamp(min=0).long()
    k = s["k_pages"].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * s["k_scale"][page][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(S, H, L, D)
    rows = torch.zeros(S, Q, Hq, D, device=k.device)
    rows[seq, place] = s["q"].float()
    rows = rows.view(S, Q, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(S, H, -1, D)       # (S, H, group * Q, D)
    score = (rows @ k.transpose(-1, -2)).mul_(s["scale"]).view(S, H, Hq // H, Q, L)
    del k
    last = (s["kv_len"] - n)[:, None] + torch.arange(Q, device=n.device) if s["causal"] else (s["kv_len"] - 1)[:, None].expand(S, Q)
    hidden = torch.arange(L, device=n.device) > last[:, None, None, :, None]
    score.masked_fill_(hidden, -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    v = s["v_pages"].view(torch.uint8)[page].view(torch.float8_e4m3fn).float() * s["v_scale"][page][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(S, H, L, D)
    o = (score.view(S, H, -1, L) @ v).view(S, H, Hq // H, Q, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(S, Q, Hq, D)[seq, place].to(s["q"].dtype)


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)


def _exact_norm(s):
    x, r = s["x"].double(), s["residual"].double()
    n = x.shape[1]
    if s["post"] is not None:
        x = x / (x.pow(2).sum(1, keepdim=True) / n + s["eps"]).sqrt() * s["post"].double()
    h = r + (x if s["gate"] is None else x * s["gate"].double()) * s["alpha"]
    return h / (h.pow(2).sum(1, keepdim=True) / n + s["eps"]).sqrt() * s["weight"].double(), h


def _complex_turn(x, positions, freq, layout):
    """Each pair as a complex number, times e^(i angle)."""
    x = x.double().clone()
    half = freq.numel()
    first = torch.arange(half, device=x.device) if layout == "half" else 2 * torch.arange(half, device=x.device)
    second = first + half if layout == "half" else first + 1
    turn = torch.polar(torch.ones(len(positions), half, dtype=torch.float64, device=x.device), torch.outer(positions.double(), freq))
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x, torch.cat((first, second))


def _exact_rotary(s):
    y, turned = _complex_turn(s["x"], s["positions"], s["freq"], s["layout"])
    y[..., turned] *= s["magnitude"]
    return y


def _exact_append(s):
    start, kv, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    pos = torch.cat([torch.arange(kv[i] - (start[i + 1] - start[i]), kv[i], device=s["q"].device) for i in range(len(kv))])
    q, _ = _complex_turn(s["q"], pos, s["freq"], s["layout"])
    k, _ = _complex_turn(s["k"], pos, s["freq"], s["layout"])
    v = s["v"].double()
    out = [q, s["k_pages"].double(), s["v_pages"].double(), s["k_scale"].double(), s["v_scale"].double()]
    for i in range(len(kv)):
        n = start[i + 1] - start[i]
        before = kv[i] - n
        for b in range(before // BLOCK, (kv[i] - 1) // BLOCK + 1):
            page, lo, hi = table[i][b], max(before, b * BLOCK), min(kv[i], (b + 1) * BLOCK)
            rows = slice(start[i] + lo - before, start[i] + hi - before)
            for x, pages, scales, swap in ((k, out[1], out[3], False), (v, out[2], out[4], True)):
                new = x[rows].transpose(0, 1)                                                # (heads, tokens, dim)
                size = new.abs().amax((1, 2))
                need = torch.exp2(torch.ceil(torch.log2(size / E4M3_MAX)).clamp(-32, 32))
                held = pages[page].transpose(1, 2) if swap else pages[page]
                if lo == b * BLOCK:
                    held.zero_()
                    scale = need
                else:
                    scale = torch.maximum(need, scales[page])
                    held *= (scales[page] / scale)[:, None, None]
                held[:, lo - b * BLOCK:hi - b * BLOCK] = new / scale[:, None, None]
                scales[page] = scale
    return tuple(out)


def _exact_attend(s):
    start, kv, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    H, D = s["k_pages"].shape[1], s["k_pages"].shape[3]
    group = s["q"].shape[1] // H
    for i in range(len(kv)):
        n = start[i + 1] - start[i]
        pages = torch.tensor(table[i][: -(-kv[i] // BLOCK)], device=out.device)
        k = s["k_pages"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s["k_scale"].double()[pages][..., None, None]
        v = s["v_pages"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * s["v_scale"].double()[pages][..., None, None]
        sees = torch.arange(kv[i] - n, kv[i], device=out.device) if s["causal"] else torch.full((n,), kv[i] - 1, device=out.device)
        for h in range(H):
            kh, vh = k[:, h].reshape(-1, D)[: kv[i]], v[:, h].transpose(1, 2).reshape(-1, D)[: kv[i]]
            for j in range(h * group, (h + 1) * group):
                w = s["q"][start[i]:start[i + 1], j].double() @ kh.T * s["scale"]
                w[torch.arange(kv[i], device=out.device)[None] > sees[:, None]] = -math.inf
                out[start[i]:start[i + 1], j] = torch.softmax(w, -1) @ vh
    return out
