"""Plain 64-bit restatements of the decoder-block operators, straight from their definitions, for the tests."""
from __future__ import annotations

import math

import torch

PAGE = 64
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def norm(x, weight, residual, gate, residual_scale, post, eps):
    """(y, h, reach): `reach` is the size of the terms that h is summed from, for the tolerance."""
    u = x.double()
    if post is not None:
        u = u / (u.pow(2).mean(-1, keepdim=True) + eps).sqrt() * post.double()
    if gate is not None:
        u = u * gate.double()
    h = u if residual is None else residual.double() + residual_scale * u
    reach = h.abs() if residual is None else residual.double().abs() + (residual_scale * u).abs()
    f = 1 / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return h * f * weight.double(), h, reach * f * weight.double().abs(), reach


def rotate(x, positions, freq, layout, magnitude=1.0):
    """(turned, reach) of x (tokens, heads, dim)."""
    y, reach = x.double().clone(), x.double().abs()
    n = freq.numel()
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        angle = positions.double() * freq[i]
        c, s = (angle.cos() * magnitude)[:, None], (angle.sin() * magnitude)[:, None]
        va, vb = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = va * c - vb * s, vb * c + va * s
        reach[..., a] = reach[..., b] = (va.abs() + vb.abs()) * abs(magnitude)
    return y, reach


def e4m3_values():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return codes


def scale_for(amax):
    if not amax > 0:
        return 2.0 ** -32
    e = math.ceil(math.log2(amax / 448.0))
    while amax > 448.0 * 2.0 ** e:
        e += 1
    while amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** min(max(e, -32), 32)


def to_e4m3(x):
    """Nearest e4m3 value of doubles, ties to the even code, saturating; NaN stays."""
    table = e4m3_values()
    mag = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(table, mag.nan_to_num(0.0)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = table[hi] - mag, mag - table[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    out = torch.copysign(table[pick], x)
    return torch.where(x.isnan(), x, out)


class Cache:
    """The cache as dicts of doubles: code values and scales, written token by token."""

    def __init__(self, k_pages, v_pages, k_scale, v_scale):
        self.k, self.v = k_pages.float().cpu().double(), v_pages.float().cpu().double()
        self.ks, self.vs = k_scale.cpu().double(), v_scale.cpu().double()

    def append(self, k, v, q_start, kv_len, table):
        """k (turned already), v: doubles (tokens, heads, dim). Codes follow the definition; returns the unrounded values where
        new tokens were written, to measure against."""
        q_start, kv_len, table = q_start.tolist(), kv_len.tolist(), table.tolist()
        pages = self.k.shape[0]
        for s in range(len(kv_len)):
            q0, n, kv = q_start[s], q_start[s + 1] - q_start[s], kv_len[s]
            if n <= 0 or kv <= 0:
                continue
            before = kv - n
            for b in range(max(before, 0) // PAGE, (kv - 1) // PAGE + 1):
                page = table[s][b] if b < len(table[s]) else -1
                if not 0 <= page < pages:
                    continue
                lo, hi = max(before, b * PAGE, 0), min(kv, (b + 1) * PAGE)
                for h in range(k.shape[1]):
                    kn, vn = k[q0 + lo - before:q0 + hi - before, h], v[q0 + lo - before:q0 + hi - before, h]
                    bad = vn.isnan().any(1)
                    for new, pool, scale, swap in ((kn, self.k, self.ks, False), (vn, self.v, self.vs, True)):
                        fin = new[new.isfinite()].abs()
                        want = scale_for(float(fin.max()) if fin.numel() else 0.0)
                        view = pool[page, h].T if swap else pool[page, h]
                        if before <= b * PAGE:
                            view.zero_()
                        else:
                            old = float(scale[page, h])
                            want = max(want, old)
                            if want != old:
                                view[: lo - b * PAGE] = to_e4m3(view[: lo - b * PAGE] * (old / want))
                        scale[page, h] = want
                        code = to_e4m3((new.nan_to_num(0.0, math.inf, -math.inf) if swap else new) / want)
                        if not swap:
                            code[bad, 0] = math.nan
                        view[lo - b * PAGE:hi - b * PAGE] = code


def attend(q, cache, q_start, kv_len, table, scale, causal):
    """(out, spread, seen, touched): out in doubles; `spread` = sum of weight * |value|, `delta` = bound of the score error in
    units of 2^-23, `least` = length * largest value scale; `written` marks the rows that belong to a sequence."""
    q_start, kv_len, table = q_start.tolist(), kv_len.tolist(), table.tolist()
    out = torch.zeros(q.shape, dtype=torch.float64)
    spread, delta, least = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    written = torch.zeros(q.shape[0], dtype=torch.bool)
    qd = q.cpu().double()
    H, D = cache.k.shape[1], cache.k.shape[3]
    group = q.shape[1] // H
    for s in range(len(kv_len)):
        q0, n, kv = q_start[s], q_start[s + 1] - q_start[s], kv_len[s]
        if n <= 0:
            continue
        written[q0:q0 + n] = True
        blocks = min(max(0, -(-kv // PAGE)), len(table[s]))
        pages = table[s][:blocks]
        ok = torch.tensor([0 <= p < cache.k.shape[0] for p in pages], dtype=torch.bool).repeat_interleave(PAGE)[:max(kv, 0)]
        idx = torch.tensor([p if 0 <= p < cache.k.shape[0] else 0 for p in pages], dtype=torch.long)
        kv_seen = min(max(kv, 0), blocks * PAGE)
        for h in range(H):
            k = (cache.k[idx, h] * cache.ks[idx, h][:, None, None]).reshape(-1, D)[:kv_seen]
            v = (cache.v[idx, h] * cache.vs[idx, h][:, None, None]).transpose(1, 2).reshape(-1, D)[:kv_seen]
            for i in range(n):
                limit = kv - n + i + 1 if causal else kv
                see = (torch.arange(kv_seen) < limit) & ok[:kv_seen]
                if not see.any():
                    continue
                rows = qd[q0 + i, h * group:(h + 1) * group]
                sc = rows @ k[see].T * scale
                w = torch.softmax(sc, -1)
                out[q0 + i, h * group:(h + 1) * group] = w @ v[see]
                spread[q0 + i, h * group:(h + 1) * group] = w @ v[see].abs()
                delta[q0 + i, h * group:(h + 1) * group] = (rows.abs() @ k[see].abs().T * abs(scale)).amax(-1) * D
                least[q0 + i, h * group:(h + 1) * group] = float(see.sum()) * float(cache.vs[idx, h].max())
    return out, spread, delta, least, written


def attend_tolerance(out, spread, delta, least, dtype):
    """Weights are rounded to 16 bits (2^-11 of each, 2^-25 of the largest for the small ones, times codes up to 448); a score's
    fp32 sum of D products is off by at most D * 2^-23 of the products' sizes, exp2 and its argument by 2^-21, which move a
    weight by that share, once in the numerator and once in the sum; then the output's own rounding."""
    share = 2.0 ** -11 + 2 * (delta * 2.0 ** -23 + 2.0 ** -21)
    return spread * share[..., None] + (least * 448 * 2.0 ** -25)[..., None] + out.abs() * HALF_STEP[dtype] * (1 + 2.0 ** -6) + 1e-7
