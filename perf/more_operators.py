"""The operators of linear layers in 8-bit floating point, with the calls that stand
for their use: their inputs, their work and what they compute.

quant_fp8     values into e4m3 codes with a scale for each 128 of a row
rms_norm_fp8  the root-mean-square norm of a residual sum into such codes
glu_fp8       a gated activation into such codes
matmul_fp8    the product of such codes with weights that have a scale for each
              128 x 128 block

A scale is a power of two in 8 bits (e8m0).  Scales are laid out [groups / 4, rows, 4]:
a row's groups 4 i .. 4 i + 3 are one 32-bit word.

`own` false: `run` computes them with elementary torch operations in 32 bits (the
largest value of a group, which lies next to a power of two's border now and then, in
64); true: it calls the framework.  Both get the same tensors.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GROUP, TOP = 128, 448.0  # values that share a scale, the largest code
EPS = 1e-6

_kernels = None


def _own_kernels():
    global _kernels
    if _kernels is None:
        pkg = os.path.join(os.getcwd(), "tt-lang_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from ttlhip import kernels

        _kernels = kernels
    return _kernels


# --- cases --------------------------------------------------------------------
# rows: tokens in the call.  quant, norm, glu: dim values of each become codes;
# matmul: k values of each meet the weights of n outputs.


def listed():
    return [
        # one token of a chat: the attention's output on its way into a projection
        {"name": "quant one token", "op": "quant", "rows": 1, "dim": 4096, "dtype": "bf16"},
        # the same of a long prompt
        {"name": "quant prompt", "op": "quant", "rows": 8192, "dim": 4096, "dtype": "bf16"},
        # the norm in front of a layer, one token
        {"name": "norm one token", "op": "norm", "rows": 1, "dim": 4096, "dtype": "bf16",
         "residual": True},
        # the same of a long prompt
        {"name": "norm prompt", "op": "norm", "rows": 8192, "dim": 4096, "dtype": "bf16",
         "residual": True},
        # a norm alone, in fp32, of rows that end inside a group
        {"name": "norm odd f32", "op": "norm", "rows": 2017, "dim": 2890, "dtype": "f32",
         "residual": False},
        # a step of 64 answers at once, gate and up beside each other as their product leaves them
        {"name": "glu step", "op": "glu", "rows": 64, "dim": 11008, "dtype": "bf16", "act": "silu"},
        # a prompt
        {"name": "glu prompt", "op": "glu", "rows": 4099, "dim": 11008, "dtype": "bf16",
         "act": "gelu"},
        # one token through the widest projection: the weights are all there is to read
        {"name": "matmul one token", "op": "matmul", "rows": 1, "n": 22016, "k": 4096,
         "dtype": "bf16"},
        # a step of a busy server, a long inner dimension and few outputs
        {"name": "matmul step", "op": "matmul", "rows": 32, "n": 4096, "k": 11008, "dtype": "bf16"},
        # short prompts packed together through the projections of q, k and v
        {"name": "matmul batch", "op": "matmul", "rows": 300, "n": 6144, "k": 4096, "dtype": "bf16"},
        # sizes off every tile, the last group short, results in fp32
        {"name": "matmul odd f32", "op": "matmul", "rows": 1057, "n": 1507, "k": 2896,
         "dtype": "f32"},
        # a long prompt through the widest projection: the largest product
        {"name": "matmul prompt", "op": "matmul", "rows": 8192, "n": 22016, "k": 4096,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "norm", "glu", "matmul", "matmul"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "matmul":
        k, n = 16 * _log(rng, 4, 1024), _log(rng, 64, 22016)
        most = min(8192, 8192 * 22016 * 4096 // (n * k))
        rows = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 1, most)
        return {"op": op, "rows": rows, "n": n if rng.random() < 0.3 else -(-n // 128) * 128,
                "k": k, "dtype": dtype}
    dim = _log(rng, 64, 16384)
    if rng.random() < 0.6:
        dim = -(-dim // 128) * 128
    rows = _log(rng, 1, min(8192, 8192 * 4096 // dim))
    if op == "quant":
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype}
    if op == "norm":
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "residual": rng.random() < 0.7}
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "act": rng.choice(["silu", "gelu"])}


# --- codes and scales ---------------------------------------------------------


def _exponents(largest):
    """e8m0 codes (biased exponents) of the scales of groups whose largest magnitudes
    are given in 64 bits: the smallest s = 2^e, e >= -126, with largest <= 448 s."""
    m, e = torch.frexp(largest)  # largest = m 2^e, m from 0.5 on; 448 = 0.875 2^9
    e = torch.where(largest > 0, e - 9 + (m > TOP / 512).int(), torch.full_like(e, -126))
    return (e.clamp(min=-126) + 127).to(torch.uint8)


def _laid_out(exps):
    """[rows, groups] -> e8m0 [ceil(groups / 4), rows, 4]; groups past the last one
    have the scale of zeros."""
    rows, groups = exps.shape
    words = -(-groups // 4)
    full = torch.ones(rows, 4 * words, dtype=torch.uint8, device=exps.device)
    full[:, :groups] = exps
    return full.view(rows, words, 4).transpose(0, 1).contiguous().view(torch.float8_e8m0fnu)


def _by_row(scales, groups):
    """The scales as numbers, [rows, groups]."""
    bits = scales.view(torch.uint8).transpose(0, 1).reshape(scales.shape[1], -1)[:, :groups]
    return torch.exp2(bits.float() - 127)


def _grouped(y, fill=0.0):
    """[rows, dim] -> [rows, groups, 128], the last group filled up."""
    rows, dim = y.shape
    groups = -(-dim // GROUP)
    if dim != groups * GROUP:
        y = torch.cat((y, y.new_full((rows, groups * GROUP - dim), fill)), 1)
    return y.view(rows, groups, GROUP)


def _coded(y, largest):
    """(codes, scales) of y with each group's largest magnitude given."""
    exps = _exponents(largest)
    inv = torch.exp2(127.0 - exps.to(y.dtype))
    codes = (_grouped(y) * inv[..., None]).flatten(1)[:, :y.shape[1]]
    return codes.clamp(-TOP, TOP).to(torch.float8_e4m3fn).contiguous(), _laid_out(exps)


# --- inputs -------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dt, rows, st = DTYPES[case["dtype"]], case["rows"], {"case": case}
    if case["op"] == "matmul":
        n, k = case["n"], case["k"]
        groups = -(-k // GROUP)
        # a few channels of the activations are much larger than the others, and rows
        # differ in size
        loud = 1.0 + 15.0 * (torch.rand(k, generator=gen, device="cuda") > 0.99).float()
        x = rnd(rows, k) * loud * torch.exp(0.5 * rnd(rows, 1))
        st["x"], st["x_scale"] = _coded(x, _grouped(x).abs().amax(-1).double())
        blocks = -(-n // GROUP)
        w = rnd(n, k) * (0.02 * torch.exp(0.3 * rnd(blocks, 1))).repeat_interleave(GROUP, 0)[:n]
        largest = _grouped(w).abs().amax(-1)  # [n, groups]
        largest = _grouped(largest.t().contiguous()).amax(-1).t().double()  # [blocks, groups]
        exps = _exponents(largest)
        inv = torch.exp2(127.0 - exps.float()).repeat_interleave(GROUP, 0)[:n]
        st["w"] = (_grouped(w) * inv[..., None]).flatten(1)[:, :k].to(torch.float8_e4m3fn).contiguous()
        st["w_scale"] = _laid_out(exps)
        st["c"] = torch.empty(rows, n, dtype=dt, device="cuda")
        return st
    dim = case["dim"]
    words = -(-dim // (4 * GROUP))
    st["codes"] = torch.empty(rows, dim, dtype=torch.float8_e4m3fn, device="cuda")
    st["scales"] = torch.empty(words, rows, 4, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    if case["op"] == "glu":
        x = rnd(rows, 2 * dim)
        x[:, :dim] *= 2.0
        st["x"] = x.to(dt)
        return st
    loud = 1.0 + 15.0 * (torch.rand(dim, generator=gen, device="cuda") > 0.99).float()
    st["x"] = (rnd(rows, dim) * loud).to(dt)
    if case["op"] == "norm":
        st["weight"] = (1.0 + 0.2 * rnd(dim)).to(dt)
        if case["residual"]:
            st["residual"] = (3.0 * rnd(rows, dim) * loud).to(dt)
            st["total"] = torch.empty_like(st["residual"])
    return st


# --- the plain forms ----------------------------------------------------------


def _norm(st, x, number):
    """(sum, norm) in the type `number`."""
    t = x.to(number)
    if "residual" in st:
        t = t + st["residual"].to(number)
    return t, t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * st["weight"].to(number)


def _glu(st, number):
    dim = st["case"]["dim"]
    g, u = st["x"][:, :dim].to(number), st["x"][:, dim:].to(number)
    if st["case"]["act"] == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    return 0.5 * g * torch.special.erfc(-g * math.sqrt(0.5)) * u


def _largest(y):
    return _grouped(y).abs().amax(-1)


def _plain(st):
    op = st["case"]["op"]
    if op == "quant":
        y = st["x"].float()
        return list(_coded(y, _largest(y).double()))
    if op == "glu":
        return list(_coded(_glu(st, torch.float32), _largest(_glu(st, torch.float64))))
    total, y = _norm(st, st["x"], torch.float32)
    out = list(_coded(y, _largest(_norm(st, st["x"], torch.float64)[1])))
    return out + [total.to(st["x"].dtype)] if "residual" in st else out


def _values(codes, scales, rows):
    """Codes times their scales, in 32 bits; `rows` rows of codes share one of scales."""
    s = _by_row(scales, -(-codes.shape[1] // GROUP))
    if rows > 1:
        s = s.repeat_interleave(rows, 0)[:codes.shape[0]]
    return (_grouped(codes.float()) * s[..., None]).flatten(1)[:, :codes.shape[1]]


def _product(st):
    x, w = _values(st["x"], st["x_scale"], 1), _values(st["w"], st["w_scale"], GROUP)
    return torch.matmul(x, w.t()).to(st["c"].dtype)


# --- one pass -----------------------------------------------------------------


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return _product(st) if op == "matmul" else _plain(st)
    K = _own_kernels()
    if op == "matmul":
        K.matmul_fp8(st["x"], st["x_scale"], st["w"], st["w_scale"], st["c"])
        return st["c"]
    if op == "quant":
        K.quant_fp8(st["x"], st["codes"], st["scales"])
    elif op == "glu":
        dim = case["dim"]
        K.glu_fp8(st["x"][:, :dim], st["x"][:, dim:], st["codes"], st["scales"], act=case["act"])
    elif case["residual"]:
        K.rms_norm_fp8(st["x"], st["weight"], st["codes"], st["scales"], eps=EPS,
                       residual=st["residual"], total=st["total"])
        return [st["codes"], st["scales"], st["total"]]
    else:
        K.rms_norm_fp8(st["x"], st["weight"], st["codes"], st["scales"], eps=EPS)
    return [st["codes"], st["scales"]]


# --- work and exact values ----------------------------------------------------


def work(case):
    rows, size = case["rows"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "matmul":
        n, k = case["n"], case["k"]
        groups = -(-k // GROUP)
        return {"bytes": (rows + n) * k + (rows + -(-n // GROUP)) * groups + rows * n * size,
                "flops": 2 * rows * n * k}
    dim = case["dim"]
    values = rows * dim
    out = values + rows * -(-dim // GROUP)
    if case["op"] == "quant":
        return {"bytes": values * size + out, "flops": 2 * values}
    if case["op"] == "norm":
        times = 3 if case["residual"] else 1
        return {"bytes": times * values * size + dim * size + out, "flops": 6 * values}
    return {"bytes": 2 * values * size + out, "flops": 8 * values}


def _exact_codes(y):
    """The values of the codes and scales of y (64 bits), as run() lays them out."""
    rows, dim = y.shape
    groups = -(-dim // GROUP)
    scale = torch.full((-(-groups // 4), rows, 4), 2.0 ** -126, dtype=torch.float64, device=y.device)
    codes = torch.empty_like(y)
    for g in range(groups):
        part = y[:, g * GROUP:(g + 1) * GROUP]
        largest = part.abs().amax(1)
        e = torch.ceil(torch.log2(largest / TOP)).clamp(min=-126.0)
        e = e + (TOP * torch.exp2(e) < largest).double()
        e = torch.where((TOP * torch.exp2(e - 1) >= largest) & (e > -126), e - 1, e)
        s = torch.exp2(e)
        scale[g // 4, :, g % 4] = s
        v = part / s[:, None]
        # four significant bits, the last of them no smaller than 2^-9
        unit = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        codes[:, g * GROUP:(g + 1) * GROUP] = torch.round(v / unit) * unit
    return codes, scale


def _exact_product(st):
    k, out = st["x"].shape[1], 0.0
    for g in range(-(-k // GROUP)):
        at = slice(g * GROUP, min(k, (g + 1) * GROUP))
        x = st["x"][:, at].double() * st["x_scale"][g // 4, :, g % 4].double()[:, None]
        block = st["w_scale"][g // 4, :, g % 4].double()
        n = torch.arange(st["w"].shape[0], device=block.device) // GROUP
        out = out + x @ (st["w"][:, at].double() * block[n, None]).t().contiguous()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "matmul":
        return _exact_product(st)
    x = st["x"].double()
    if case["op"] == "quant":
        return list(_exact_codes(x))
    if case["op"] == "glu":
        g, u = x[:, :case["dim"]], x[:, case["dim"]:]
        gate = torch.sigmoid(g) if case["act"] == "silu" else torch.special.ndtr(g)
        return list(_exact_codes(g * gate * u))
    total = x + st["residual"].double() if case["residual"] else x
    rms = torch.sqrt((total * total).sum(1) / case["dim"] + EPS)
    out = list(_exact_codes(total / rms[:, None] * st["weight"].double()))
    return out + [total] if case["residual"] else out
