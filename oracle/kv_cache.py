"""Float64 restatements of the operators on rotary positions and an 8-bit
key/value cache, from their definitions (test oracle; CPU, plain loops)."""

from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rope(x, positions, freqs, interleaved=False, scale=1.0, backward=False):
    x, r = x.double(), 2 * freqs.numel()
    a = positions.double()[:, None] * freqs.double()
    c, s = (scale * torch.cos(a))[:, None], (scale * torch.sin(a))[:, None]
    if backward:
        s = -s
    y = x.clone()
    u = x[..., 0:r:2] if interleaved else x[..., : r // 2]
    w = x[..., 1:r:2] if interleaved else x[..., r // 2 : r]
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = u * c - w * s, w * c + u * s
    else:
        y[..., : r // 2], y[..., r // 2 : r] = u * c - w * s, w * c + u * s
    return y


def spans(lengths, starts, tokens):
    """(first packed token, number) of each sequence's new tokens."""
    if starts is None:
        return [(b, 1) for b in range(len(lengths))]
    out = []
    for b in range(len(lengths)):
        lo = min(max(int(starts[b]), 0), tokens)
        out.append((lo, max(0, min(int(starts[b + 1]), tokens) - lo)))
    return out


def place(table, b, pos, page, pages):
    """(page, slot) of a position, or None."""
    if pos < 0 or pos >= table.shape[1] * page:
        return None
    p = int(table[b, pos // page])
    return (p, pos % page) if 0 <= p < pages else None


def scale_for(largest: float, dtype) -> float:
    if not math.isfinite(largest):
        return math.nan
    if largest == 0:
        return 2.0 ** -126
    e = math.ceil(math.log2(largest / TOP[dtype]))
    while TOP[dtype] * 2.0 ** e < largest:
        e += 1
    while TOP[dtype] * 2.0 ** (e - 1) >= largest:
        e -= 1
    return max(2.0 ** e, 2.0 ** -126)


def to_code(x, dtype):
    """x (float64, at most the largest code) rounded to a code, half to even."""
    if dtype == torch.int8:
        return torch.round(x).to(torch.int8)
    unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / unit) * unit).to(torch.float32).to(dtype)


def write(k, v, k_cache, v_cache, k_scale, v_scale, table, lengths, starts=None):
    """Updates the caches and scales in place."""
    pages, heads, page, _ = k_cache.shape
    for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        for b, (first, n) in enumerate(spans(lengths, starts, k.shape[0])):
            begin = int(lengths[b]) - n
            runs = {}  # page -> [(slot, token)]
            for i in range(n):
                at = place(table, b, begin + i, page, pages)
                if at is not None:
                    runs.setdefault(at[0], []).append((at[1], first + i))
            for p, run in runs.items():
                for h in range(heads):
                    rows = torch.stack([x[t, h] for _, t in run]).double()
                    s = scale_for(float(rows.abs().max()) if not rows.isnan().any() else math.nan,
                                  codes.dtype)
                    if run[0][0] > 0 and begin > 0:  # the page holds earlier tokens
                        old = float(scales[p, h])
                        s = max(old, s) if 0 <= old < math.inf and math.isfinite(s) else math.nan
                        if s > old:
                            slot = run[0][0]
                            codes[p, h, :slot] = to_code(
                                codes[p, h, :slot].double() * (old / s), codes.dtype)
                    scales[p, h] = s
                    for (slot, _), row in zip(run, rows):
                        codes[p, h, slot] = to_code(
                            row / s if math.isfinite(s) else torch.zeros_like(row), codes.dtype)


def sound(scale):
    """A page's scale; one that is negative or not finite makes NaN of the page."""
    s = scale.double()
    return torch.where((s >= 0) & s.isfinite(), s, torch.full_like(s, math.nan))


def attention(q, k_cache, v_cache, k_scale, v_scale, table, lengths, scale, starts=None,
              window=0, softcap=0.0):
    """(o, size, reach): o float64, NaN in rows of no sequence; per element the sum
    of p |v| that o's cancels from; per (token, head) the largest sum of |q k| scale
    of its scores."""
    pages, heads, page, dim = k_cache.shape
    tokens, q_heads, _ = q.shape
    group = q_heads // heads
    o = torch.full((tokens, q_heads, dim), math.nan, dtype=torch.float64)
    size, reach = torch.zeros_like(o), torch.zeros(tokens, q_heads, 1, dtype=torch.float64)
    for b, (first, n) in enumerate(spans(lengths, starts, tokens)):
        at = [(j, *pl) for j in range(max(0, min(int(lengths[b]), table.shape[1] * page)))
              if (pl := place(table, b, j, page, pages)) is not None]
        pos = torch.tensor([a[0] for a in at], dtype=torch.long)
        pg = torch.tensor([a[1] for a in at], dtype=torch.long)
        slot = torch.tensor([a[2] for a in at], dtype=torch.long)
        for h in range(heads):
            ks = k_cache[pg, h, slot].double() * sound(k_scale[pg, h])[:, None]
            vs = v_cache[pg, h, slot].double() * sound(v_scale[pg, h])[:, None]
            for i in range(n):
                p = int(lengths[b]) - n + i
                sees = (pos <= p) & ((pos > p - window) if window else (pos >= 0))
                kk, vv = ks[sees], vs[sees]
                for g in range(group):
                    t, hq = first + i, h * group + g
                    if not len(kk):
                        o[t, hq] = 0
                        continue
                    x = q[t, hq].double()
                    s = (kk * x).sum(1) * scale
                    reach[t, hq] = float(((kk * x).abs().sum(1) * abs(scale)).max())
                    if softcap:
                        s = softcap * torch.tanh(s / softcap)
                    w = torch.softmax(s, 0)
                    o[t, hq], size[t, hq] = w @ vv, w @ vv.abs()
    return o, size, reach
