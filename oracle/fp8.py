"""Float64 restatements of the operators of linear layers in 8-bit floating point, from
their definitions (test oracle; CPU)."""

from __future__ import annotations

import math

import torch

GROUP, TOP, LEAST = 128, 448.0, 2.0 ** -126


def e4m3(v):
    """v, at most 448 in magnitude, rounded to a code's value, ties to even."""
    unit = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / unit) * unit


def scale_for(largest: float) -> float:
    """The smallest 2^e, e from -126 on, with largest <= 448 2^e; NaN where it is not finite."""
    if not math.isfinite(largest):
        return math.nan
    m, e = math.frexp(largest)
    return max(math.ldexp(1.0, e - 9 + (m > TOP / 512)), LEAST) if largest else LEAST


def scales(y):
    """[rows, dim] -> the scales of its groups, [rows, groups]."""
    rows, dim = y.shape
    groups = -(-dim // GROUP)
    s = torch.empty(rows, groups, dtype=torch.float64)
    for g in range(groups):
        for r, big in enumerate(y[:, g * GROUP:(g + 1) * GROUP].abs().amax(1).tolist()):
            s[r, g] = scale_for(big)
    return s


def each(s, dim):
    """[rows, groups] -> [rows, dim]"""
    return s.repeat_interleave(GROUP, 1)[:, :dim]


def by_row(laid_out, groups):
    """Scales as the operators lay them out -> [rows, groups]."""
    return laid_out.double().transpose(0, 1).reshape(laid_out.shape[1], -1)[:, :groups]


def rms_norm(x, weight, eps, residual=None):
    t = x.double() + (residual.double() if residual is not None else 0.0)
    return t, t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * weight.double()


def glu(gate, up, act):
    g = gate.double()
    y = g / (1 + torch.exp(-g)) if act == "silu" else 0.5 * g * torch.special.erfc(-g * math.sqrt(0.5))
    return y * up.double()


def values(codes, laid_out, rows=1):
    """Codes times their scales; `rows` rows of codes share one of scales."""
    s = by_row(laid_out, -(-codes.shape[1] // GROUP)).repeat_interleave(rows, 0)[:codes.shape[0]]
    return codes.double() * each(s, codes.shape[1])
