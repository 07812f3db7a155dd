"""The operators of serving from an 8-bit key/value cache, with the calls that
stand for their use: their inputs, their work and what they compute.

rope            rotary positions on the heads of packed tokens
kv_cache_write  new tokens' keys and values into pages of 8-bit codes
sdpa_cached     attention of new tokens over such a cache

`own` false: `run` computes them with elementary torch operations in 32 bits
(angles in 64); true: it calls the framework.  Both get the same tensors.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32,
          "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code

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
# q heads / kv heads 32 / 8 of 128 unless said otherwise.  seqs: sequences in the
# call; most: the longest one's tokens in the cache after the call (the others
# have from a quarter of it on); new: the most new tokens a sequence has (with
# `ragged`, others have fewer); page: tokens that share a page and its scales.


def listed():
    return [
        # one token of a chat: q and k rotated by one call
        {"name": "rope one token", "op": "rope", "tokens": 1, "heads": 40, "dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "backward": False, "far": 30000},
        # a prompt's tokens, far into a long context
        {"name": "rope prompt", "op": "rope", "tokens": 8192, "heads": 40, "dim": 128, "rot": 128,
         "dtype": "bf16", "interleaved": False, "backward": False, "far": 1000000},
        # the gradient of interleaved positions on part of the head, an odd batch in fp32
        {"name": "rope gradient f32", "op": "rope", "tokens": 4099, "heads": 33, "dim": 96,
         "rot": 64, "dtype": "f32", "interleaved": True, "backward": True, "far": 5000},
        # a step of 64 answers at once: one token each into partly filled pages
        {"name": "write a step", "op": "write", "seqs": 64, "most": 4096, "new": 1, "ragged": False,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "cache": "int8"},
        # prompts of different lengths, some of them continued
        {"name": "write prompts", "op": "write", "seqs": 5, "most": 8191, "new": 8000,
         "ragged": True, "kv_heads": 8, "dim": 128, "page": 32, "dtype": "bf16", "cache": "e4m3"},
        # one user, a short context: latency
        {"name": "decode short", "op": "attn", "seqs": 1, "most": 501, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "int8", "window": 0,
         "softcap": 0.0},
        # a step of a busy server
        {"name": "decode batch", "op": "attn", "seqs": 32, "most": 8192, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "int8", "window": 0,
         "softcap": 0.0},
        # long documents: the largest cache
        {"name": "decode long", "op": "attn", "seqs": 16, "most": 65537, "new": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "cache": "e4m3", "window": 0,
         "softcap": 0.0},
        # a layer with a window and capped scores, every head its own keys, small pages
        {"name": "decode window cap", "op": "attn", "seqs": 24, "most": 4096, "new": 1,
         "ragged": False, "heads": 32, "kv_heads": 32, "dim": 64, "page": 16, "cache": "int8",
         "window": 1024, "softcap": 50.0},
        # drafted tokens checked at once, many heads to a key
        {"name": "several tokens", "op": "attn", "seqs": 16, "most": 16384, "new": 5,
         "ragged": True, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "cache": "int8",
         "window": 0, "softcap": 0.0},
        # a chunk of a long prompt
        {"name": "chunk", "op": "attn", "seqs": 1, "most": 18000, "new": 2048, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "int8", "window": 0,
         "softcap": 0.0},
        # whole prompts of different lengths
        {"name": "prompts", "op": "attn", "seqs": 4, "most": 2049, "new": 2049, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "cache": "e4m3", "window": 0,
         "softcap": 30.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "attn", "attn"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": _log(rng, 1, 40), "dim": dim,
                "rot": rng.choice([dim, dim // 2, 32]), "dtype": rng.choice(["bf16", "f32"]),
                "interleaved": rng.random() < 0.5, "backward": rng.random() < 0.5,
                "far": _log(rng, 100, 1000000)}
    page, dim = rng.choice([16, 32, 64, 128]), rng.choice([64, 128])
    cache, seqs = rng.choice(["int8", "e4m3"]), _log(rng, 1, 64)
    if op == "write":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 32000 // seqs)
        return {"op": op, "seqs": seqs, "most": new + _log(rng, 1, 8192), "new": new,
                "ragged": rng.random() < 0.5, "kv_heads": rng.choice([1, 2, 4, 8, 16]), "dim": dim,
                "page": page, "dtype": rng.choice(["bf16", "f32"]), "cache": cache}
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    form = rng.random()
    if form < 0.5:
        new, most = 1, _log(rng, 1, 500000 // seqs)
    elif form < 0.75:
        new = rng.randint(2, 9)
        most = new + _log(rng, 1, 200000 // seqs)
    else:  # no more scores than the listed chunk has
        new, scores = _log(rng, 10, 2048), 1000000000
        seqs = min(seqs, 8)
        if seqs * kv_heads * group * new * new > scores:
            seqs = 1
        most = new + _log(rng, 1, 16384)
        most = min(most, scores // (seqs * kv_heads * group * new))
    return {"op": op, "seqs": seqs, "most": most, "new": new,
            "ragged": rng.random() < 0.5, "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": dim, "page": page, "cache": cache,
            "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
            "softcap": rng.choice([0.0, 0.0, 30.0])}


def _sizes(case):
    """([tokens in the cache after the call], [new tokens]) of the sequences."""
    lens, news = [], []
    for b in range(case["seqs"]):
        f = (0.25 + 0.75 * ((b * 0.6180339887) % 1.0)) if b else 1.0
        n = case["new"] if not (case["ragged"] and b) else 1 + int((case["new"] - 1) * ((b * 0.3819) % 1.0))
        lens.append(max(n, int(case["most"] * f)))
        news.append(n)
    return lens, news


# --- inputs -------------------------------------------------------------------


def _frequencies(rot):
    return 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)


def _codes(shape, kind, gen):
    """Codes like those of normal values under their largest one."""
    if kind == "int8":
        return (torch.randn(shape, generator=gen, device="cuda").mul_(40.0).round_()
                .clamp_(-127, 127).to(torch.int8))
    return torch.randn(shape, generator=gen, device="cuda").mul_(100.0).clamp_(-448, 448).to(
        torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    st = {"case": case}
    if case["op"] == "rope":
        t = case["tokens"]
        st["x"] = rnd(t, case["heads"], case["dim"]).to(DTYPES[case["dtype"]])
        st["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda",
                                        dtype=torch.int32)
        st["freqs"] = _frequencies(case["rot"]).cuda()
        st["scale"] = 1.25  # as contexts stretched beyond their training have it
        st["out"] = torch.empty_like(st["x"])
        return st
    lens, news = _sizes(case)
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    flat = order.cpu()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = flat[at:at + n]
        at += n
    st["table"] = table.cuda()
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    # None: one new token of every sequence
    st["starts"] = (None if max(news) == 1
                    else torch.tensor(starts, dtype=torch.int32, device="cuda"))
    pages = order.numel()
    for n in ("k_cache", "v_cache"):
        st[n] = _codes((pages, hk, page, d), case["cache"], gen)
    unit = (1.25 / 40) if case["cache"] == "int8" else (1.25 / 100)
    for n in ("k_scale", "v_scale"):
        e = torch.randint(-1, 2, (pages, hk), generator=gen, device="cuda").float()
        st[n] = torch.exp2(torch.floor(torch.log2(torch.tensor(unit, device="cuda"))) + e)
    if case["op"] == "write":
        dt = DTYPES[case["dtype"]]
        # a few channels of keys are much larger than the others
        loud = 1.0 + 5.0 * (torch.rand(d, generator=gen, device="cuda") > 0.95).float()
        st["k"] = (rnd(starts[-1], hk, d) * loud).to(dt)
        st["v"] = rnd(starts[-1], hk, d).to(dt)
    else:
        st["q"] = (1.5 * rnd(starts[-1], case["heads"], d)).to(torch.bfloat16)
        st["o"] = torch.empty_like(st["q"])
        st["scale"] = 1.0 / math.sqrt(d)
    return st


# --- the plain forms ----------------------------------------------------------


def _rope(st):
    c = st["case"]
    x, r = st["x"].float(), c["rot"]
    a = st["positions"].double()[:, None] * st["freqs"][None, :]
    cos = (torch.cos(a) * st["scale"]).float()[:, None, :]
    sin = (torch.sin(a) * st["scale"]).float()[:, None, :]
    if c["backward"]:
        sin = -sin
    if c["interleaved"]:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((u * cos - w * sin, w * cos + u * sin), -1).flatten(-2)
    else:
        u, w = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((u * cos - w * sin, w * cos + u * sin), -1)
    return torch.cat((y, x[..., r:]), -1).to(st["x"].dtype)


def _tokens(st):
    """Per new token its sequence and its position, and per sequence its new tokens."""
    case, lengths = st["case"], st["lengths"].long()
    if st["starts"] is None:
        seq = torch.arange(case["seqs"], device="cuda")
        new = torch.ones_like(seq)
        first = seq
    else:
        starts = st["starts"].long()
        new = starts[1:] - starts[:-1]
        seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), new)
        first = starts[:-1]
    i = torch.arange(seq.numel(), device="cuda") - first[seq]
    return seq, lengths[seq] - new[seq] + i, i, first, new


def _scale_for(largest, top):
    """The smallest power of two s with largest <= top s, from 2^-126 on."""
    m, e = torch.frexp(largest)
    mt, et = math.frexp(top)
    e = e - et + (m > mt).int()
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), e.clamp(min=-126)),
                       torch.full_like(largest, 2.0 ** -126))


def _round_to(x, dtype):
    return x.round().to(dtype) if dtype == torch.int8 else x.to(dtype)


def _write(st):
    case = st["case"]
    page, top = case["page"], TOP[case["cache"]]
    seq, pos, _, _, new = _tokens(st)
    at = st["table"].long()[seq, pos // page]
    slot = pos % page
    begin = st["lengths"].long() - new
    cut = begin % page > 0  # the page that holds earlier tokens
    old_page = st["table"].long()[torch.arange(case["seqs"], device="cuda"), begin // page][cut]
    earlier = (begin % page)[cut]
    out = []
    for x, codes, scales in ((st["k"], st["k_cache"], st["k_scale"]),
                             (st["v"], st["v_cache"], st["v_scale"])):
        x = x.float()
        # the largest value of each page and head that gets tokens
        largest = torch.full_like(scales, -1.0)
        largest = largest.index_reduce(0, at, x.abs().amax(-1), "amax")
        need = _scale_for(largest, top)
        need[old_page] = torch.maximum(need[old_page], scales[old_page])
        was = codes[old_page].float()
        again = _round_to(was * (scales[old_page] / need[old_page])[:, :, None, None], codes.dtype)
        kept = torch.arange(page, device="cuda")[None, :] < earlier[:, None]
        again = torch.where(kept[:, None, :, None], again.float(), was).to(codes.dtype)
        codes[old_page] = again
        scales.copy_(torch.where(largest >= 0, need, scales))
        codes[at, :, slot] = _round_to(x / scales[at][:, :, None], codes.dtype)
        out += [codes, scales]
    return out


def _attention(st):
    case = st["case"]
    b, hk, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    g, n = case["heads"] // hk, case["new"]
    seq, pos, i, first, new = _tokens(st)
    table = st["table"].long().clamp(min=0)
    length = table.shape[1] * page

    def values(codes, scales):
        x = codes[table].float() * scales[table][..., None, None]  # [b, pages, hk, page, d]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, length, d)

    # the sequences' queries side by side, [b, hk, n g, d]
    pick = (first[:, None] + torch.arange(n, device="cuda")).clamp(max=seq.numel() - 1)
    q = st["q"].float()[pick].view(b, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, d)
    s = torch.matmul(q, values(st["k_cache"], st["k_scale"]).transpose(-1, -2)) * st["scale"]
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    qpos = ((st["lengths"].long() - new)[:, None] + torch.arange(n, device="cuda")).repeat_interleave(g, 1)
    j = torch.arange(length, device="cuda")
    hidden = j[None, None, :] > qpos[:, :, None]
    if case["window"]:
        hidden = hidden | (j[None, None, :] <= qpos[:, :, None] - case["window"])
    s.masked_fill_(hidden[:, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(s, values(st["v_cache"], st["v_scale"])) / s.sum(-1, keepdim=True)
    o = o.view(b, hk, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hk * g, d)
    return o[seq, i].to(torch.bfloat16)


# --- one pass -----------------------------------------------------------------


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"rope": _rope, "write": _write, "attn": _attention}[op](st)
    K = _own_kernels()
    if op == "rope":
        K.rope(st["x"], st["positions"], st["freqs"], st["out"], interleaved=case["interleaved"],
               scale=st["scale"], backward=case["backward"])
        return st["out"]
    cache = (st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if op == "write":
        K.kv_cache_write(st["k"], st["v"], *cache, st["table"], st["lengths"], starts=st["starts"])
        return [cache[0], cache[2], cache[1], cache[3]]
    K.sdpa_cached(st["q"], *cache, st["table"], st["lengths"], st["o"], st["scale"],
                  starts=st["starts"], window=case["window"], softcap=case["softcap"])
    return st["o"]


# --- work and exact values ----------------------------------------------------


def _visible(length, new, window):
    """Pairs of a new token and a position that it sees."""
    first = length - new + 1
    if not window or window >= length:
        return new * first + new * (new - 1) // 2
    short = max(0, min(new, window - first))  # tokens that the window leaves whole
    return short * first + short * (short - 1) // 2 + (new - short) * window


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4), "flops": 3 * n}
    lens, news = _sizes(case)
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "write":
        n = 2 * sum(news) * hk * d
        touched = sum(-(-a // page) - (a - b) // page for a, b in zip(lens, news))
        return {"bytes": n * ((2 if case["dtype"] == "bf16" else 4) + 1) + 8 * touched * hk,
                "flops": 2 * n}
    w = case["window"]
    seen = [min(a, b + w - 1) if w else a for a, b in zip(lens, news)]
    codes = 2 * sum(seen) * hk * d + 8 * hk * sum(-(-a // page) for a in seen)
    pairs = sum(_visible(a, b, w) for a, b in zip(lens, news)) * case["heads"]
    return {"bytes": codes + 4 * sum(news) * case["heads"] * d, "flops": 4 * d * pairs}


def _exact_codes(x, kind):
    """x, at most the largest code, rounded to a code."""
    if kind == "int8":
        return torch.round(x)
    # four significant bits, the last of them no smaller than 2^-9
    unit = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / unit) * unit


def _exact_write(case, st):
    """Sequence by sequence.  The codes of int8 are whole numbers (which both
    forms have to give alike) and have no place here."""
    lens, news = _sizes(case)
    page, top, kind = case["page"], TOP[case["cache"]], case["cache"]
    out = []
    for x, codes, scales in ((st["k"], st["k_cache"], st["k_scale"]),
                             (st["v"], st["v_cache"], st["v_scale"])):
        x, codes, scales, t = x.double(), codes.double(), scales.double(), 0
        for b, (length, new) in enumerate(zip(lens, news)):
            lo, hi = (length - new) // page, -(-length // page)
            at = st["table"][b, lo:hi].long()
            head = length - new - lo * page  # earlier tokens of the first page
            rows = torch.zeros((hi - lo) * page, *x.shape[1:], dtype=x.dtype, device=x.device)
            rows[head:head + new] = x[t:t + new]
            t += new
            rows = rows.view(hi - lo, page, *x.shape[1:]).transpose(1, 2)  # [pages, heads, page, d]
            largest = rows.abs().amax((2, 3))
            e = torch.ceil(torch.log2(largest / top))
            e = e + (top * torch.exp2(e) < largest).double()
            e = e - (top * torch.exp2(e - 1) >= largest).double()
            s = torch.exp2(e)
            if head:
                s[0] = torch.maximum(s[0], scales[at[0]])
                codes[at[0], :, :head] = _exact_codes(
                    codes[at[0], :, :head] * (scales[at[0]] / s[0])[:, None, None], kind)
            scales[at] = s
            new_codes = _exact_codes(rows / s[:, :, None, None], kind)
            end = length - (hi - 1) * page
            for i in range(hi - lo):
                u, w = (head if i == 0 else 0), (end if i == hi - lo - 1 else page)
                codes[at[i], :, u:w] = new_codes[i, :, u:w]
        out += [None if kind == "int8" else codes, scales]
    return out


def _exact_attention(case, st):
    lens, news = _sizes(case)
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    g, t = case["heads"] // hk, 0
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, (length, new) in enumerate(zip(lens, news)):
        at = st["table"][b, :-(-length // page)].long()
        qpos = torch.arange(length - new, length, device="cuda")
        j = torch.arange(length, device="cuda")
        seen = j[None, :] <= qpos[:, None]
        if case["window"]:
            seen &= j[None, :] > qpos[:, None] - case["window"]
        for h in range(hk):
            k, v = ((c[at, h].double() * s[at, h].double()[:, None, None]).reshape(-1, d)[:length]
                    for c, s in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])))
            for i in range(g):
                q = st["q"][t:t + new, h * g + i].double()
                x = (q @ k.t().contiguous()) * st["scale"]
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                out[t:t + new, h * g + i] = torch.softmax(x.masked_fill(~seen, -math.inf), 1) @ v
        t += new
    return out


def _exact_rope(case, st):
    r = case["rot"]
    x = st["x"].double()
    a = st["positions"].double()[:, None] * st["freqs"]
    turn = torch.polar(torch.full_like(a, st["scale"]), -a if case["backward"] else a)[:, None]
    at = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous()) * turn
    y = x.clone()
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "attn": _exact_attention}[case["op"]](case, st)
