"""Rotary positions and the 8-bit key/value cache on the MI355X against float64
restatements (oracle/kv_cache.py).

Tolerances, derived:
* rope: a c - b s with c and s one rounding of scale times an fp32 rounding of the
  exact cosine, two products and a sum: (|a| + |b|) scale 5 * 2^-24, and for bf16 a
  rounding of the result, 2^-8 of it.
* kv_cache_write: codes and scales are equal: scales are powers of two, so every
  quotient is exact and each code one rounding of an exact value.
* sdpa_cached: p v sums run over bf16 roundings of p (2^-8 each: 2^-8 sum p |v|),
  the result is rounded to bf16 (2^-8 of it).  Scores are fp32 sums of dim products
  and a few factors, off by at most (dim + 16) 2^-24 of the sum of |q k| scale (and by
  2^-21 softcap where capped), which moves p, in numerator and denominator, by twice
  that; n terms in fp32 sums add (n + 64) 2^-24, exponentials 2^-21.
"""

import math
import threading
import time

import pytest
import torch

from oracle import kv_cache as R
from ttlhip import expr as X
from ttlhip import kernels as K

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# --- rope ---------------------------------------------------------------------


def _check_rope(out, x, positions, freqs, interleaved, scale, backward):
    ref = R.rope(x, positions, freqs, interleaved, scale, backward)
    r = 2 * freqs.numel()
    big = x.double().abs()
    both = big.clone()  # |a| + |b| of an element's plane
    if interleaved:
        pair = big[..., 0:r:2] + big[..., 1:r:2]
        both[..., 0:r:2], both[..., 1:r:2] = pair, pair
    else:
        pair = big[..., : r // 2] + big[..., r // 2 : r]
        both[..., :r] = torch.cat((pair, pair), -1)
    tol = both * abs(scale) * 5 * 2.0 ** -24
    tol[..., r:] = 0
    if out.dtype == BF16:
        tol = tol + 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -20) + (tol * 2.0 ** -8)
        tol[..., r:] = 0
    bad = (out.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((out.double() - ref).abs() - tol).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [
    (1, 1, 64, 64), (1, 40, 128, 128), (3, 5, 80, 32), (7, 3, 96, 64), (130, 2, 10, 6),
    (2, 2, 7, 2), (5, 1, 128, 0), (2, 70, 128, 128), (1, 3, 2048, 1024), (9, 1, 3, 0),
    (4100, 2, 32, 16)])
def test_rope(dtype, interleaved, tokens, heads, dim, rot):
    g = _gen(tokens + heads + dim)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (tokens,), generator=g, dtype=torch.int32)
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    for backward in (False, True):
        out = torch.full_like(x, 7.0).cuda()
        K.rope(x.cuda(), pos.cuda(), f.cuda(), out, interleaved, 1.25, backward)
        _check_rope(out.cpu(), x, pos, f, interleaved, 1.25, backward)


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 24 + 3, 2 ** 31 - 64])
def test_rope_far_positions_keep_their_angles(far):
    g = _gen(3)
    x = torch.randn(64, 2, 128, generator=g)
    pos = far + torch.arange(64)
    f = K.rope_freqs(128, device="cpu")
    out = torch.empty_like(x, device="cuda")
    K.rope(x.cuda(), pos.cuda(), f.cuda(), out)
    _check_rope(out.cpu(), x, pos, f, False, 1.0, False)
    neg = torch.empty_like(x, device="cuda")
    K.rope(x.cuda(), -pos.cuda(), f.cuda(), neg)
    _check_rope(neg.cpu(), x, -pos, f, False, 1.0, False)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_in_place_in_a_projection(offset, interleaved):
    """q and k of one buffer in one call, in place; v beside them stays.  offset 1:
    addresses that vectors cannot have."""
    g = _gen(5)
    buf = torch.randn(33, 12 * 64 + 8, generator=g).to(BF16).cuda()
    qk = buf[:, offset:offset + 8 * 64].unflatten(1, (8, 64))
    before = buf.clone()
    pos = torch.arange(33, dtype=torch.int32)
    f = K.rope_freqs(64, device="cpu")
    K.rope(qk, pos.cuda(), f.cuda(), qk, interleaved)
    old = before[:, offset:offset + 512].unflatten(1, (8, 64)).cpu()
    _check_rope(qk.cpu(), old, pos, f, interleaved, 1.0, False)
    assert torch.equal(buf[:, offset + 512:], before[:, offset + 512:])
    assert torch.equal(buf[:, :offset], before[:, :offset])


def test_rope_heads_before_tokens():
    g = _gen(6)
    x = torch.randn(4, 50, 64, generator=g).to(BF16)  # [heads, tokens, dim]
    pos = torch.arange(50, dtype=torch.int64) * 7
    f = K.rope_freqs(64, device="cpu")
    out = torch.empty_like(x, device="cuda")
    K.rope(x.cuda().transpose(0, 1), pos.cuda(), f.cuda(), out.transpose(0, 1))
    _check_rope(out.cpu().transpose(0, 1), x.transpose(0, 1), pos, f, False, 1.0, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    """backward against the formula's gradient (autograd of the float64 form) and
    against differences of the forward kernel."""
    g = _gen(7)
    x, dy = torch.randn(5, 3, 32, generator=g), torch.randn(5, 3, 32, generator=g)
    pos = torch.tensor([0, 1, 17, 999, 123456], dtype=torch.int32)
    f = K.rope_freqs(16, device="cpu")
    dx = torch.empty_like(x, device="cuda")
    K.rope(dy.cuda(), pos.cuda(), f.cuda(), dx, interleaved, 1.5, backward=True)
    xd = x.double().requires_grad_()
    a = pos.double()[:, None] * f
    c, s = 1.5 * torch.cos(a)[:, None], 1.5 * torch.sin(a)[:, None]
    u, w = (xd[..., 0:16:2], xd[..., 1:16:2]) if interleaved else (xd[..., :8], xd[..., 8:16])
    yu, yw = u * c - w * s, w * c + u * s
    du, dw = (dy[..., 0:16:2], dy[..., 1:16:2]) if interleaved else (dy[..., :8], dy[..., 8:16])
    ((yu * du).sum() + (yw * dw).sum() + (xd[..., 16:] * dy[..., 16:]).sum()).backward()
    # |dy| <= 6 here: both elements of a plane, 5 roundings of 2^-24
    assert float((dx.cpu().double() - xd.grad).abs().max()) <= 2 * 6 * 1.5 * 5 * 2.0 ** -24
    # the map is linear: differences of step 2 around x = 0 are its columns, exactly
    # rounded like the outputs (|x| = 1: 1.5 * 5 * 2^-24 each, times 32 of dy)
    for i in (0, 3, 9, 15, 16, 31):
        e = torch.zeros_like(x)
        e[..., i] = 1.0
        up, down = torch.empty_like(dx), torch.empty_like(dx)
        K.rope(e.cuda(), pos.cuda(), f.cuda(), up, interleaved, 1.5)
        K.rope(-e.cuda(), pos.cuda(), f.cuda(), down, interleaved, 1.5)
        diff = (((up - down) / 2).cpu().double() * dy.double()).sum(-1)
        assert float((diff - dx[..., i].cpu().double()).abs().max()) <= 32 * 6 * 1.5 * 6 * 2.0 ** -24


# --- the cache: writes ----------------------------------------------------------------


def _cache(pages, heads, page, dim, dtype, seed):
    """Pages filled with something: codes of every kind (NaN's too, in e4m3)."""
    g = _gen(seed)
    raw = [torch.randint(0, 256, (pages, heads, page, dim), generator=g, dtype=torch.uint8)
           for _ in range(2)]
    sc = [torch.exp2(torch.randint(-6, 3, (pages, heads), generator=g).float()) for _ in range(2)]
    return [raw[0].view(dtype), raw[1].view(dtype), sc[0], sc[1]]


def _table(need, width, pages, seed):
    order = torch.randperm(pages, generator=_gen(seed)).to(torch.int32)
    t = torch.full((len(need), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def _same(a, b):
    return torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a,
                       b.view(torch.uint8) if b.dtype == E4M3 else b)


def _run_write(k, v, cache, table, lengths, starts=None):
    """The kernel on copies against the oracle on copies; returns the kernel's."""
    ref, dev = [c.clone() for c in cache], [c.cuda() for c in cache]
    R.write(k, v, *ref, table, lengths, starts)
    K.kv_cache_write(k.cuda(), v.cuda(), *dev, table.cuda(), lengths.cuda(),
                     starts=None if starts is None else starts.cuda())
    got = [c.cpu() for c in dev]
    for name, x, y in zip(("k", "v", "k_scale", "v_scale"), got, ref):
        if x.dtype == F32:
            assert torch.equal(x.isnan(), y.isnan()), name
            x, y = x.nan_to_num(), y.nan_to_num()
        if x.dtype == E4M3:  # -0 and 0 are one value
            x, y = x.float().nan_to_num(500.0), y.float().nan_to_num(500.0)
        assert torch.equal(x, y), (name, int((x != y).sum()))
    return got


def _random_call(lens, news, heads, dim, page, dtype, cdtype, seed, one=False):
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    table = _table(need, max(need) + 1, pages, seed)
    cache = _cache(pages, heads, page, dim, cdtype, seed + 1)
    g = _gen(seed + 2)
    t = sum(news)
    k = (torch.randn(t, heads, dim, generator=g) * torch.exp2(4 * torch.randn(t, heads, 1, generator=g)))
    v = torch.randn(t, heads, dim, generator=g) * 0.01
    starts = None if one else torch.tensor([sum(news[:i]) for i in range(len(news) + 1)],
                                           dtype=torch.int32)
    return k.to(dtype), v.to(dtype), cache, table, torch.tensor(lens, dtype=torch.int32), starts


def _valid_codes(cache, table, lengths, news, page):
    """Earlier tokens' codes as a write leaves them: no NaN."""
    if cache[0].dtype != E4M3:
        return
    for c in cache[:2]:
        raw = c.view(torch.uint8)
        raw[(raw & 0x7f) == 0x7f] = 0x12


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,dim", [(16, 64), (16, 128), (32, 128), (64, 64), (64, 128), (128, 128)])
def test_write_ragged(cdtype, dtype, page, dim):
    lens, news = [1, 17, 200, 128, 129, 65, 64, 300], [1, 17, 1, 128, 2, 0, 5, 299]
    call = _random_call(lens, news, 3, dim, page, dtype, cdtype, page + dim)
    _valid_codes(call[2], call[3], lens, news, page)
    _run_write(*call)


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("seqs,heads,dim", [(1, 1, 64), (1, 8, 128), (70, 3, 128), (5, 17, 64)])
def test_write_one_token_each(cdtype, seqs, heads, dim):
    lens = [1 + (37 * b) % 150 for b in range(seqs)]
    call = _random_call(lens, [1] * seqs, heads, dim, 32, BF16, cdtype, seqs, one=True)
    _valid_codes(call[2], call[3], lens, None, 32)
    _run_write(*call)


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
def test_write_token_by_token_follows_the_definition(cdtype):
    """40 calls of one token, magnitudes growing: every growth rounds again."""
    cache = _cache(4, 2, 16, 64, cdtype, 9)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    g = _gen(10)
    for i in range(40):
        k = torch.randn(1, 2, 64, generator=g) * 1.1 ** i
        v = torch.randn(1, 2, 64, generator=g)
        cache = _run_write(k, v, cache, table, torch.tensor([i + 1], dtype=torch.int32))
    # every key is within the last rounding and those before it, each at half the step
    # of the one before: less than one step of the final scale (int8)
    if cdtype == INT8:
        assert float(cache[0][2].float().abs().max()) <= 127


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("value", [0.0, -0.0, 1e-45, 2.0 ** -126, 127.0, 127.00001, 448.0, 449.0, 254.0,
                                   3.4028234e38, math.inf, -math.inf, math.nan])
def test_write_special_values(cdtype, value):
    cache = _cache(2, 1, 16, 64, cdtype, 11)
    _valid_codes(cache, None, None, None, 16)
    k = torch.zeros(2, 1, 64)
    k[1, 0, 5] = value
    v = torch.randn(2, 1, 64, generator=_gen(1))
    table = torch.tensor([[1]], dtype=torch.int32)
    for length in (2, 5):  # a new page; one that holds tokens
        _run_write(k, v, cache, table, torch.tensor([length], dtype=torch.int32),
                   torch.tensor([0, 2], dtype=torch.int32))


def test_write_after_nan_stays_nan_until_the_page_begins_anew():
    cache = _cache(1, 1, 16, 64, INT8, 12)
    table = torch.zeros(1, 1, dtype=torch.int32)
    k = torch.full((1, 1, 64), math.nan)
    one = torch.ones(1, 1, 64)
    cache = _run_write(k, one, cache, table, torch.tensor([1], dtype=torch.int32))
    cache = _run_write(one, one, cache, table, torch.tensor([2], dtype=torch.int32))
    assert math.isnan(cache[2][0, 0])
    cache = _run_write(one, one, cache, table, torch.tensor([1], dtype=torch.int32))
    assert float(cache[2][0, 0]) == 2.0 ** -6


@pytest.mark.parametrize("lens,starts,table", [
    ([40, 20], [0, 10, 20], [[-1, 1, 99], [0, -7, 2]]),         # pages that do not exist
    ([500, 3], [0, 10, 20], [[0, 1, 2], [3, 4, 5]]),            # past the table, before position 0
    ([-5, 0], [0, 10, 20], [[0, 1, 2], [3, 4, 5]]),             # no tokens
    ([20, 20], [-3, 12, 500], [[0, 1, 2], [3, 4, 5]]),          # starts outside the packed rows
    ([20, 20], [15, 5, 20], [[0, 1, 2], [3, 4, 5]]),            # starts that go back
    ([2 ** 31 - 1, -2 ** 31], [0, 10, 20], [[0, 1, 2], [3, 4, 5]]),
])
@pytest.mark.parametrize("cdtype", [INT8, E4M3])
def test_tables_lengths_and_starts_out_of_range_touch_nothing(cdtype, lens, starts, table):
    cache = _cache(6, 2, 16, 64, cdtype, 13)
    _valid_codes(cache, None, None, None, 16)
    g = _gen(14)
    k, v = torch.randn(20, 2, 64, generator=g), torch.randn(20, 2, 64, generator=g)
    t, n, s = (torch.tensor(x, dtype=torch.int32) for x in (table, lens, starts))
    got = _run_write(k, v, cache, t, n, s)
    q = torch.randn(20, 4, 64, generator=g).to(BF16)
    _check_attention(q, got, t, n, s, 0.125)


def test_write_strided_views():
    g = _gen(15)
    qkv = torch.randn(50, 12, 128, generator=g).to(BF16)
    lens = torch.tensor([50], dtype=torch.int32)
    starts = torch.tensor([0, 50], dtype=torch.int32)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    cache = _cache(2, 2, 32, 128, INT8, 16)
    ref = [c.clone() for c in cache]
    R.write(qkv[:, 8:10], qkv[:, 10:12], *ref, table, lens, starts)
    dev, d = [c.cuda() for c in cache], qkv.cuda()
    wide = torch.full((1, 5), -1, dtype=torch.int32)
    wide[:, :2] = table
    K.kv_cache_write(d[:, 8:10], d[:, 10:12], *dev, wide.cuda()[:, :2], lens.cuda(), starts.cuda())
    for x, y in zip(dev, ref):
        assert _same(x.cpu(), y)
    # off every vector's address: bf16 one element on, f32 with heads before tokens
    odd = torch.randn(50, 4 * 128 + 3, generator=g).to(BF16)
    ref, dev = [c.clone() for c in cache], [c.cuda() for c in cache]
    kv = odd[:, 1:513].unflatten(1, (4, 128))
    R.write(kv[:, :2], kv[:, 2:], *ref, table, lens, starts)
    kv = odd.cuda()[:, 1:513].unflatten(1, (4, 128))
    K.kv_cache_write(kv[:, :2], kv[:, 2:], *dev, table.cuda(), lens.cuda(), starts.cuda())
    for a, b in zip(dev, ref):
        assert _same(a.cpu(), b)
    flat = torch.randn(1 + 2 * 50 * 128, generator=g)
    x = flat[1:].view(2, 50, 128).transpose(0, 1)
    ref, dev = [c.clone() for c in cache], [c.cuda() for c in cache]
    R.write(x, x, *ref, table, lens, starts)
    xd = flat.cuda()[1:].view(2, 50, 128).transpose(0, 1)
    K.kv_cache_write(xd, xd, *dev, table.cuda(), lens.cuda(), starts.cuda())
    for a, b in zip(dev, ref):
        assert _same(a.cpu(), b)


# --- attention ----------------------------------------------------------------


def _tolerance(ref, size, reach, dim, n, softcap):
    off = (dim + 16) * 2.0 ** -24 * reach + 2.0 ** -21 * softcap
    share = 2.0 ** -8 + 2 * off + 2 * (n + 64) * 2.0 ** -24 + 2 * 2.0 ** -21
    # (and p v is below fp32's ordinary range where V is below 2^-118)
    return size * share + 2.0 ** -8 * (ref.abs() + size * share) + 2.0 ** -118


def _check_attention(q, cache, table, lengths, starts, scale, window=0, softcap=0.0, o=None):
    ref, size, reach = R.attention(q, *cache, table, lengths, scale, starts, window, softcap)
    out = torch.full_like(q, 7.0).cuda() if o is None else o
    K.sdpa_cached(q.cuda() if not q.is_cuda else q, *[c.cuda() for c in cache], table.cuda(),
                  lengths.cuda(), out, scale,
                  starts=None if starts is None else starts.cuda(), window=window, softcap=softcap)
    got = out.cpu()
    n = max([1] + [min(int(x), table.shape[1] * cache[0].shape[2]) for x in lengths])
    tol = _tolerance(ref, size, reach, q.shape[2], n, softcap)
    owned = torch.zeros(q.shape[0], dtype=torch.bool)
    for first, m in R.spans(lengths, starts, q.shape[0]):
        owned[first:first + m] = True
    assert (got[~owned] == 7.0).all(), "rows of no sequence"
    got, ref, tol = got[owned].double(), ref[owned], tol[owned]
    assert torch.equal(got.isnan(), ref.isnan())
    err = (got - ref).abs().nan_to_num()
    assert (err <= tol.nan_to_num(1.0)).all(), (float((err - tol).max()), float(err.max()))
    return got


def _attention_call(lens, news, heads, group, dim, page, cdtype, seed, one=False, loud=1.5):
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + 2
    table = _table(need, max(need) + 1, pages, seed)
    cache = _cache(pages, heads, page, dim, cdtype, seed + 1)
    # what a write leaves in the tokens' slots; the others keep any code
    g = _gen(seed + 2)
    codes = []
    for c in cache[:2]:
        x = (torch.randn(c.shape, generator=g) * 40).clamp(-127, 127)
        x = x.round().to(torch.int8) if cdtype == INT8 else x.to(E4M3)
        raw = x.view(torch.uint8)
        keep = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                keep[table[b, j // page], j % page] = True
        raw = torch.where(keep[:, None, :, None], raw, c.view(torch.uint8))
        codes.append(raw.view(cdtype))
    sc = [torch.exp2(torch.randint(-7, -3, (pages, heads), generator=g).float()) for _ in range(2)]
    q = (torch.randn(sum(news), heads * group, dim, generator=g) * loud).to(BF16)
    starts = None if one else torch.tensor([sum(news[:i]) for i in range(len(news) + 1)],
                                           dtype=torch.int32)
    return q, codes + sc, table, torch.tensor(lens, dtype=torch.int32), starts


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attention_one_token_each(cdtype, dim, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 130, 200]
    q, cache, table, n, _ = _attention_call(lens, [1] * len(lens), 2, 4, dim, page, cdtype, 21, True)
    _check_attention(q, cache, table, n, None, dim ** -0.5)


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 2), (3, 3), (2, 7), (1, 8), (1, 16), (2, 17),
                                         (1, 32), (1, 40), (5, 1)])
@pytest.mark.parametrize("news", [[1, 1], [2, 3], [9, 1], [40, 33], [0, 5]])
def test_attention_groups_and_tokens(heads, group, news):
    lens = [150, 75]
    q, cache, table, n, starts = _attention_call(lens, news, heads, group, 64, 32, INT8, 22)
    _check_attention(q, cache, table, n, starts, 0.125)


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (64, 128)])
@pytest.mark.parametrize("lens,news", [
    ([130, 1, 33], [130, 1, 33]),           # whole prompts
    ([257], [257]),
    ([300, 128, 64, 190], [100, 128, 1, 7]),
    ([513], [65]),
])
def test_attention_chunks(cdtype, dim, page, lens, news):
    q, cache, table, n, starts = _attention_call(lens, news, 2, 2, dim, page, cdtype, 23)
    _check_attention(q, cache, table, n, starts, dim ** -0.5)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 1000, 2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("news", [[1, 1], [130, 40]])
def test_attention_window(window, news):
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 128, 32, INT8, 24)
    _check_attention(q, cache, table, n, starts, 0.09, window=window)


@pytest.mark.parametrize("softcap", [0.5, 30.0, 1e4])
@pytest.mark.parametrize("news", [[1, 1], [130, 40]])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_softcap(softcap, news, window):
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 128, 32, E4M3, 25, loud=4.0)
    _check_attention(q, cache, table, n, starts, 0.09, window=window, softcap=softcap)


@pytest.mark.parametrize("scale", [0.0, -0.09, 1.0])
@pytest.mark.parametrize("news", [[1, 1], [70, 40]])
def test_attention_scales(scale, news):
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 128, 32, INT8, 26)
    _check_attention(q, cache, table, n, starts, scale)


@pytest.mark.parametrize("news", [[1, 1, 1], [130, 20, 40]])
def test_attention_missing_pages_and_rows_that_see_nothing(news):
    q, cache, table, n, starts = _attention_call([300, 55, 90], news, 2, 4, 128, 32, E4M3, 27)
    table[0, 2] = -1
    table[0, 5] = 10 ** 6
    table[1] = -1  # nothing to see: zeros
    got = _check_attention(q, cache, table, n, starts, 0.09)
    assert (got[news[0]:news[0] + news[1]] == 0).all()
    _check_attention(q, cache, table, n, starts, 0.09, window=20)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("news", [[1, 1], [130, 55]])
def test_attention_nan_reaches_only_the_tokens_that_see_it(which, news):
    """A page's NaN scale: the tokens that see any of it, in its head."""
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 128, 32, INT8, 28)
    cache[which][table[0, 7], 1] = math.nan  # positions 224 .. 255
    cache[which][table[1, 1], 0] = math.nan  # positions 32 .. 54
    got = _check_attention(q, cache, table, n, starts, 0.09)
    assert got.isnan().any() and not got.isnan().all()
    got = _check_attention(q, cache, table, n, starts, 0.09, window=20)
    if news[0] > 1:
        assert got.isnan().any() and not got.isnan().all()


@pytest.mark.parametrize("news", [[1, 1], [70, 40]])
def test_attention_of_queries_that_are_not_finite(news):
    q, cache, table, n, starts = _attention_call([300, 55], news, 1, 4, 64, 32, INT8, 29)
    q[0, 1, 3] = math.nan
    q[1, 2, 5] = math.nan
    got = _check_attention(q, cache, table, n, starts, 0.125)
    assert int(got.isnan().any(-1).sum()) == 2


@pytest.mark.parametrize("news", [[1, 1], [130, 55]])
def test_attention_large_scores(news):
    """Scores that differ by thousands: exponentials of 0 beside one of 1."""
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 2, 64, 16, INT8, 30, loud=3000.0)
    ref, size, reach = R.attention(q, *cache, table, n, 0.125, starts)
    out = torch.empty_like(q, device="cuda")
    K.sdpa_cached(q.cuda(), *[c.cuda() for c in cache], table.cuda(), n.cuda(), out, 0.125,
                  starts=starts.cuda())
    assert torch.isfinite(out).all()
    tol = _tolerance(ref, size, reach, 64, 300, 0.0)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


def test_attention_strided_views():
    q, cache, table, n, starts = _attention_call([100, 55], [37, 20], 2, 4, 64, 32, INT8, 31)
    buf = torch.zeros(57, 20, 64, dtype=BF16, device="cuda")
    buf[:, 4:12] = q.cuda()
    o = torch.full((8, 57, 64), 7.0, dtype=BF16, device="cuda").transpose(0, 1)
    ref = torch.full((57, 8, 64), 7.0, dtype=BF16, device="cuda")
    dev = [c.cuda() for c in cache]
    K.sdpa_cached(buf[:, 4:12], *dev, table.cuda(), n.cuda(), o, 0.125, starts=starts.cuda())
    K.sdpa_cached(q.cuda(), *dev, table.cuda(), n.cuda(), ref, 0.125, starts=starts.cuda())
    assert torch.equal(o, ref)


def test_rows_behind_the_last_sequence_stay():
    q, cache, table, n, starts = _attention_call([100, 55], [37, 20], 2, 4, 64, 32, INT8, 32)
    q = torch.cat((q, torch.ones(9, 8, 64, dtype=BF16)))
    _check_attention(q, cache, table, n, starts, 0.125)


def test_empty_calls():
    cache = [c.cuda() for c in _cache(2, 2, 16, 64, INT8, 33)]
    none = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    before = [c.clone() for c in cache]
    for seqs, starts in ((0, None), (0, torch.zeros(1, dtype=torch.int32, device="cuda")),
                         (3, torch.zeros(4, dtype=torch.int32, device="cuda"))):
        table = torch.zeros(seqs, 2, dtype=torch.int32, device="cuda")
        n = torch.ones(seqs, dtype=torch.int32, device="cuda")
        K.kv_cache_write(none[:, :2], none[:, :2], *cache, table, n, starts=starts)
        K.sdpa_cached(none, *cache, table, n, torch.empty_like(none), 0.1, starts=starts)
    K.rope(none, torch.zeros(0, dtype=torch.int32, device="cuda"), K.rope_freqs(64), none)
    # a table without columns: nothing to write to, nothing to see
    one = torch.ones(1, 4, 64, dtype=BF16, device="cuda")
    o = torch.full_like(one, 7.0)
    table = torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    K.kv_cache_write(one[:, :2], one[:, :2], *cache, table, n)
    K.sdpa_cached(one, *cache, table, n, o, 0.1)
    assert (o == 0).all()
    assert all(_same(a, b) for a, b in zip(cache, before))


# --- long sequences, many of them, divided ones -------------------------------


def _check_heads(q, cache, table, n, starts, scale, heads, window=0, softcap=0.0):
    """The whole call; the cache heads `heads` of it against the oracle."""
    group = q.shape[1] // cache[0].shape[1]
    out = torch.full_like(q, 7.0).cuda()
    K.sdpa_cached(q.cuda(), *[c.cuda() for c in cache], table.cuda(), n.cuda(), out, scale,
                  starts=None if starts is None else starts.cuda(), window=window, softcap=softcap)
    out = out.cpu()
    for h in heads:
        part = [c[:, h:h + 1] for c in cache]
        qs = slice(h * group, (h + 1) * group)
        ref, size, reach = R.attention(q[:, qs], *part, table, n, scale, starts, window, softcap)
        tol = _tolerance(ref, size, reach, q.shape[2], int(n.max()), softcap)
        got = out[:, qs].double()
        assert torch.equal(got.isnan(), ref.isnan()), h
        err = (got - ref).abs().nan_to_num()
        assert (err <= tol.nan_to_num(1.0)).all(), (h, float((err - tol).max()))
    return out


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,news", [(4, [1, 1, 1]), (9, [2, 3, 1]), (16, [2, 2, 2]), (3, [40, 11, 90])])
def test_attention_divided_into_parts(cdtype, dim, group, news):
    """Every tile size with sequences of several parts, of one and of none."""
    lens = [4001, 90, 1777]
    q, cache, table, n, starts = _attention_call(lens, news, 2, group, dim, 64, cdtype, 70)
    _check_attention(q, cache, table, n, starts, dim ** -0.5)
    _check_attention(q, cache, table, n, starts, dim ** -0.5, window=1500, softcap=20.0)


@pytest.mark.parametrize("dim,cdtype", [(64, E4M3), (128, INT8)])
@pytest.mark.parametrize("group,news", [(2, [1] * 6), (8, [20, 9, 1, 3, 0, 2]), (8, [40, 24, 9]),
                                        (8, [100, 60, 9, 0, 0, 70])])
def test_attention_parts_that_fill_the_chip(dim, cdtype, group, news):
    """More parts than places, were they as short as parts may be: their lengths come from
    all sequences', for few tiles, for half as many as there are places, and for more."""
    lens = [9000, 5000, 1503, 700, 0, 4100][:len(news)]
    q, cache, table, n, starts = _attention_call(lens, news, 64, group, dim, 64, cdtype, 77)
    _check_heads(q, cache, table, n, starts, dim ** -0.5, (0, 63))


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dim,cdtype", [(64, INT8), (128, E4M3)])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_attention_long_undivided_tiles(page, dim, cdtype, softcap):
    """Tiles that walk more than 2 x 16 blocks, some pages missing and some NaN where
    the sixteens meet."""
    q, cache, table, n, starts = _attention_call([2300, 1100], [260, 130], 128, 2, dim, page, cdtype, 71)
    _check_heads(q, cache, table, n, starts, dim ** -0.5, (0, 127), softcap=softcap)
    table[0, 1024 // page] = -1
    table[0, 2047 // page] = 10 ** 7
    cache[2][table[1, 1023 // page], 0] = math.nan
    out = _check_heads(q, cache, table, n, starts, dim ** -0.5, (0, 127), softcap=softcap)
    # (of head 0's, those from the bad page's first position on)
    sees = torch.arange(970, 1100) >= 1023 // page * page
    assert torch.equal(out[260:, :2].isnan().all(-1).all(-1), sees)
    assert not out[260:, 2:].isnan().any()


def _check_tokens(q, cache, table, n, starts, scale, heads, tokens, window=0, softcap=0.0):
    """The whole call; tokens (sequence, new token) of the cache heads `heads` against the
    oracle, each as the one new token of a sequence that ends with it."""
    group = q.shape[1] // cache[0].shape[1]
    out = torch.full_like(q, 7.0).cuda()
    K.sdpa_cached(q.cuda(), *[c.cuda() for c in cache], table.cuda(), n.cuda(), out, scale,
                  starts=starts.cuda(), window=window, softcap=softcap)
    out = out.cpu()
    assert not (out == 7.0).all(-1).any()
    for b, i in tokens:
        t, news = int(starts[b]) + i, int(starts[b + 1] - starts[b])
        m = n[b:b + 1] - (news - 1 - i)
        for h in heads:
            part = [c[:, h:h + 1] for c in cache]
            qs = slice(h * group, (h + 1) * group)
            ref, size, reach = R.attention(q[t:t + 1, qs], *part, table[b:b + 1], m, scale, None,
                                           window, softcap)
            tol = _tolerance(ref, size, reach, q.shape[2], int(m[0]), softcap)
            got = out[t:t + 1, qs].double()
            assert torch.equal(got.isnan(), ref.isnan()), (b, i, h)
            err = (got - ref).abs().nan_to_num()
            assert (err <= tol.nan_to_num(1.0)).all(), (b, i, h, float((err - tol).max()))


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (3900, 0.0), (0, 20.0)])
@pytest.mark.parametrize("heads,group,lens,news", [
    (64, 8, [4097], [201]),         # one chunk, its tiles alike
    (16, 8, [4100, 2000], [601, 500]),
    (8, 32, [33000], [49])])        # and divided into parts
def test_attention_tiles_of_256_rows(cdtype, window, softcap, heads, group, lens, news):
    """Calls whose rows go in tiles of eight waves, some pages missing, some bad, some with
    scales that V's codes are multiplied by."""
    q, cache, table, n, starts = _attention_call(lens, news, heads, group, 128, 32, cdtype, 78)
    tokens = [(b, i) for b, m in enumerate(news) for i in (0, 7, 8, 31, 32, m - 1)]
    _check_tokens(q, cache, table, n, starts, 0.09, (0, heads - 1), tokens, window, softcap)
    last = lens[0] - news[0]
    table[0, 5], table[0, 1024 // 32] = -1, 10 ** 7
    cache[3][table[0, 70], 0], cache[3][table[0, 71], 0] = 2.0 ** -110, 2.0 ** 70
    cache[2][table[0, (last + 8) // 32], 0] = math.nan
    cache[3][table[0, (last + 8) // 32], heads - 1] = math.inf
    _check_tokens(q, cache, table, n, starts, 0.09, (0, heads - 1), tokens, window, softcap)


def test_attention_rows_of_more_than_4096_positions():
    """One part of a wave's more than 32 steps."""
    q, cache, table, n, _ = _attention_call([17000], [1], 256, 1, 64, 128, INT8, 72, True)
    _check_heads(q, cache, table, n, None, 0.125, (0, 100, 255))


@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("group", [2, 30])
def test_attention_of_150_sequences(one, group):
    g = _gen(73)
    lens = [int(x) for x in torch.randint(1, 90, (150,), generator=g)]
    lens[3], lens[80], lens[149] = 2000, 1300, 700
    news = [1] * 150 if one else [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 4, (150,), generator=g))]
    q, cache, table, n, starts = _attention_call(lens, news, 1, group, 64, 32, INT8, 74, one)
    _check_attention(q, cache, table, n, starts, 0.125)


def test_write_of_150_sequences():
    lens = [1 + (37 * b) % 150 for b in range(150)]
    news = [min(n, b % 5) for b, n in enumerate(lens)]
    call = _random_call(lens, news, 2, 64, 16, BF16, INT8, 75)
    _run_write(*call)


@pytest.mark.parametrize("news", [[1, 1], [130, 55]])
@pytest.mark.parametrize("cdtype", [INT8, E4M3])
def test_attention_extreme_scales(news, cdtype):
    """V scales down to those of pages of zeros and up to 2^80, K scales of zero and
    2^-126; a negative scale is NaN."""
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 64, 16, cdtype, 76)
    ks, vs = cache[2], cache[3]
    vs[table[0, 1], 0], vs[table[0, 2], 0], vs[table[0, 3], 1] = 2.0 ** -126, 2.0 ** -100, 2.0 ** 80
    vs[table[1, 0], 1], vs[table[1, 1], 1], vs[table[1, 2], 1] = 2.0 ** -90, 2.0 ** -80, 2.0 ** -85
    ks[table[0, 4], 0], ks[table[0, 5], 0] = 0.0, 2.0 ** -126
    _check_attention(q, cache, table, n, starts, 0.125)
    zero = vs.clone()
    zero[table[0, 6]] = 0.0
    _check_attention(q, [*cache[:3], zero], table, n, starts, 0.125)
    for i in (2, 3):
        bad = [c.clone() for c in cache]
        bad[i][table[0, 4], 1] = -1.0
        o = torch.empty_like(q, device="cuda")
        K.sdpa_cached(q.cuda(), *[c.cuda() for c in bad], table.cuda(), n.cuda(), o, 0.125,
                      starts=starts.cuda())
        pos = [n[0] - news[0] + i for i in range(news[0])]
        sees = torch.tensor([p >= 64 for p in pos])
        assert torch.equal(o[:news[0], 4:].isnan().all(-1).all(-1).cpu(), sees)
        assert not o[:, :4].isnan().any() and not o[news[0]:].isnan().any()


@pytest.mark.parametrize("news", [[1, 1], [130, 55]])
def test_attention_into_its_queries(news):
    q, cache, table, n, starts = _attention_call([900, 555], news, 2, 4, 128, 32, INT8, 77)
    dev = [c.cuda() for c in cache]
    o, x = torch.empty_like(q, device="cuda"), q.cuda()
    K.sdpa_cached(x, *dev, table.cuda(), n.cuda(), o, 0.09, starts=starts.cuda())
    K.sdpa_cached(x, *dev, table.cuda(), n.cuda(), x, 0.09, starts=starts.cuda())
    assert torch.equal(o, x)


def test_caches_past_32_bits():
    """Codes more than 4 GiB into a cache."""
    heads, page, dim = 8, 128, 128
    pages = (5 << 30) // (heads * page * dim)
    k, v = (torch.zeros(pages, heads, page, dim, dtype=INT8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 3], [pages - 2, pages - 3]], dtype=torch.int32)
    lens, starts = torch.tensor([200, 250], dtype=torch.int32), torch.tensor([0, 200, 450], dtype=torch.int32)
    g = _gen(78)
    x = [torch.randn(450, heads, dim, generator=g).to(BF16) for _ in range(2)]
    K.kv_cache_write(x[0].cuda(), x[1].cuda(), k, v, ks, vs, table.cuda(), lens.cuda(), starts.cuda())
    at = [3, pages - 3, pages - 2, pages - 1]
    small = [c[at].cpu() for c in (k, v, ks, vs)]
    local = torch.tensor([[3, 0], [2, 1]], dtype=torch.int32)
    ref = [torch.zeros_like(c) for c in small]
    R.write(*x, *ref, local, lens, starts)
    assert all(_same(a, b) for a, b in zip(small, ref))
    for news in ([1, 1], [60, 50]):
        st = torch.tensor([0, news[0], sum(news)], dtype=torch.int32)
        q = torch.randn(sum(news), heads, dim, generator=g).to(BF16)
        o = torch.empty_like(q, device="cuda")
        K.sdpa_cached(q.cuda(), k, v, ks, vs, table.cuda(), lens.cuda(), o, 0.09, starts=st.cuda())
        out, size, reach = R.attention(q, *ref, local, lens, 0.09, st)
        assert ((o.cpu().double() - out).abs() <= _tolerance(out, size, reach, dim, 250, 0.0)).all()


def test_long_and_short_sequences_in_one_call():
    """A prompt of many tiles beside single tokens far into their sequences: the tiles fill
    the chip, the long sequences are divided all the same."""
    lens, news = [700, 9000, 400, 5000], [700, 1, 1, 1]
    q, cache, table, n, starts = _attention_call(lens, news, 64, 2, 64, 64, INT8, 79)
    _check_heads(q, cache, table, n, starts, 0.125, (0, 63))


# --- together -----------------------------------------------------------------


def _step(qkv, pos, freqs, cache, table, lengths, o, starts=None, window=0):
    """One layer's attention of a step: 4 q heads, 2 k heads, 2 v heads of 64."""
    K.rope(qkv[:, :6], pos, freqs, qkv[:, :6])
    K.kv_cache_write(qkv[:, 4:6], qkv[:, 6:], *cache, table, lengths, starts=starts)
    K.sdpa_cached(qkv[:, :4], *cache, table, lengths, o, 0.125, starts=starts, window=window)


def _oracle_step(qkv, pos, freqs, cache, table, lengths, starts=None, window=0):
    qk = R.rope(qkv[:, :6], pos, freqs).to(BF16)
    R.write(qk[:, 4:6], qkv[:, 6:], *cache, table, lengths, starts)
    return R.attention(qk[:, :4], *cache, table, lengths, 0.125, starts, window)


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
def test_prompts_then_tokens(cdtype):
    """Two prompts, then ten tokens each, as a program serves them; the oracle follows
    with the kernel's rotated values (a rounding of rope may fall either way)."""
    g = _gen(40)
    freqs = K.rope_freqs(64, scaling="parts", factor=4.0, original=64, device="cpu")
    lens = [45, 9]
    dev = [c.cuda() for c in _cache(16, 2, 16, 64, cdtype, 41)]
    table = _table([5, 5], 5, 16, 42)
    ref = [c.cpu().clone() for c in dev]
    starts = torch.tensor([0, 45, 54], dtype=torch.int32)
    for step in range(11):
        if step == 0:
            pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32)
            s = starts
        else:
            lens = [n + 1 for n in lens]
            pos, s = torch.tensor([n - 1 for n in lens], dtype=torch.int32), None
        n = torch.tensor(lens, dtype=torch.int32)
        qkv = torch.randn(len(pos), 8, 64, generator=g).to(BF16)
        d = qkv.cuda()
        o = torch.full((len(pos), 4, 64), 7.0, dtype=BF16, device="cuda")
        _step(d, pos.cuda(), freqs.cuda(), dev, table.cuda(), n.cuda(), o,
              None if s is None else s.cuda())
        turned = d.cpu()
        _check_rope(turned[:, :6], qkv[:, :6], pos, freqs, False, 1.0, False)
        R.write(turned[:, 4:6], turned[:, 6:], *ref, table, n, s)
        for a, b in zip(dev, ref):
            assert torch.equal(a.float().cpu().nan_to_num(500.0), b.float().nan_to_num(500.0)), step
        out, size, reach = R.attention(turned[:, :4], *ref, table, n, 0.125, s)
        err = (o.cpu().double() - out).abs()
        assert (err <= _tolerance(out, size, reach, 64, 60, 0.0)).all(), (step, float(err.max()))


def test_captured_steps_follow_the_lengths():
    """Steps captured into two graphs replay on lengths that grow on the device, with
    eager calls between them, and equal the eager steps bit for bit."""
    g = _gen(43)
    seqs, width = 5, 20
    table = _table([width] * seqs, width, seqs * width, 44).cuda()
    freqs = K.rope_freqs(64)
    first = [c.cuda() for c in _cache(seqs * width, 2, 16, 64, INT8, 45)]
    lens0 = torch.tensor([1, 70, 16, 200, 33], dtype=torch.int32, device="cuda")
    qkvs = [torch.randn(seqs, 8, 64, generator=g).to(BF16).cuda() for _ in range(12)]

    def eager():
        cache, lens, outs = [c.clone() for c in first], lens0.clone(), []
        for x in qkvs:
            x, o = x.clone(), torch.empty(seqs, 4, 64, dtype=BF16, device="cuda")
            _step(x, lens - 1, freqs, cache, table, lens, o)
            outs.append(o)
            lens += 1
        return outs, cache

    want, want_cache = eager()
    cache, lens = [c.clone() for c in first], lens0.clone()
    x = [torch.empty_like(qkvs[0]) for _ in range(2)]
    o = [torch.empty(seqs, 4, 64, dtype=BF16, device="cuda") for _ in range(2)]
    graphs = []
    saved = [c.clone() for c in cache], lens.clone()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _step(x[i], lens - 1, freqs, cache, table, lens, o[i])
            lens.add_(1)
        graphs.append(graph)
    for c, s in zip(cache, saved[0]):
        c.copy_(s)
    lens.copy_(saved[1])
    for j, q in enumerate(qkvs):
        x[j % 2].copy_(q)
        graphs[j % 2].replay()
        if j % 3 == 0:
            again, _ = eager()
            torch.cuda.synchronize()
        assert torch.equal(o[j % 2], want[j]), j
    assert all(_same(a, b) for a, b in zip(cache, want_cache))


@pytest.mark.parametrize("tokens", [1, 40])
def test_captured_parts_grow_with_the_lengths(tokens):
    """Divided attention in two graphs, each with its own workspace, replayed in turns while
    eager calls with other, larger workspaces run between: as many parts as the
    lengths of each replay ask for, and the eager call's bits."""
    seqs, width = 3, 130
    q, cache, table, n, starts = _attention_call([2000, 1000, 400], [tokens] * seqs, 2, 4, 64, 16, INT8, 80)
    table = torch.cat((table, table[:, :width - table.shape[1]]), 1) if table.shape[1] < width else table
    dev, table, n = [c.cuda() for c in cache], table.cuda(), n.cuda()
    starts = None if tokens == 1 else starts.cuda()
    qs = [q.cuda(), q.flip(0).contiguous().cuda()]
    lens = torch.full((seqs,), 60, dtype=torch.int32, device="cuda")
    outs = [torch.empty_like(x) for x in qs]
    big, bcache, btable, bn, bstarts = _attention_call([3000, 900], [90, 70], 2, 8, 128, 64, INT8, 81)
    bdev = [big.cuda(), *[c.cuda() for c in bcache], btable.cuda(), bn.cuda()]

    def eager(i, n):
        o = torch.empty_like(qs[i])
        K.sdpa_cached(qs[i], *dev, table, n, o, 0.125, starts=starts)
        return o

    eager(0, lens)
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.sdpa_cached(qs[i], *dev, table, lens, outs[i], 0.125, starts=starts)
        graphs.append(graph)
    for j in range(8):
        now = (n * (j + 1) // 8).clamp(min=tokens)
        lens.copy_(now)
        graphs[0].replay()
        graphs[1].replay()
        o = torch.empty_like(bdev[0])
        K.sdpa_cached(*bdev, o, 0.09, starts=bstarts.cuda())
        for i in range(2):
            assert torch.equal(outs[i], eager(i, now)), (j, i)
        torch.cuda.synchronize()


def test_two_streams_at_once():
    calls = [_attention_call([4000, 1333, 90], [1, 1, 1], 2, 4, 128, 32, INT8, 50 + i, True)
             for i in range(2)]
    dev = [[q.cuda(), [c.cuda() for c in cache], t.cuda(), n.cuda()] for q, cache, t, n, _ in calls]
    want = []
    for q, cache, t, n in dev:
        o = torch.empty_like(q)
        K.sdpa_cached(q, *cache, t, n, o, 0.09)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.full_like(d[0], 7.0) for _ in range(20)] for d in dev]
    torch.cuda.synchronize()
    for j in range(20):
        for s, (q, cache, t, n), o in zip(streams, dev, outs):
            K.sdpa_cached(q, *cache, t, n, o[j], 0.09, stream=s)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


def test_same_call_same_bits():
    q, cache, table, n, starts = _attention_call([1500, 700], [3, 2], 2, 4, 128, 64, INT8, 60)
    dev = [c.cuda() for c in cache]
    outs = []
    for _ in range(5):
        o = torch.empty_like(q, device="cuda")
        K.sdpa_cached(q.cuda(), *dev, table.cuda(), n.cuda(), o, 0.09, starts=starts.cuda())
        outs.append(o)
    assert all(torch.equal(outs[0], o) for o in outs)


# --- pages that are not there, values at the ends of the range ---------------------------


def _free_page_0(cache, table):
    """The same call with a page 0 that no sequence has."""
    free = next(p for p in range(cache[0].shape[0]) if p > 0 and not (table == p).any())
    for c in cache:
        raw = c.view(torch.uint8) if c.dtype == E4M3 else c
        raw[free] = raw[0]
    table[table == 0] = free


@pytest.mark.parametrize("scale0", [0.0, 2.0 ** 70, 2.0 ** -3])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("dim,heads,group,lens,news,holes", [
    (64, 2, 4, [300, 155], [130, 40], (0, 3, 8)),        # tiles of 128 rows
    (128, 2, 4, [300, 155], [130, 40], (0, 3, 8)),
    (128, 64, 8, [4097], [201], (0, 5, 31, 32, 64)),     # tiles of 256 rows
    (128, 2, 4, [300, 155], [1, 1], (0, 3, 8))])         # few rows
def test_attention_missing_pages_beside_a_page_0_of_nan_codes(dim, heads, group, lens, news, holes,
                                                              softcap, scale0):
    """What is not in the table is not there, whatever is in page 0: here codes that are NaN
    under a scale that was never written, or one so large that V is multiplied by it."""
    q, cache, table, n, starts = _attention_call(lens, news, heads, group, dim, 32, E4M3, 82)
    _free_page_0(cache, table)
    for c in cache[:2]:
        c.view(torch.uint8)[0] = 0x7f
    cache[2][0], cache[3][0] = scale0, scale0
    for i, p in enumerate(holes):
        table[0, p] = -1 if i % 2 else 10 ** 6
    if heads == 2:
        _check_attention(q, cache, table, n, starts, 0.09, softcap=softcap)
    else:
        tokens = [(0, i) for i in (0, 31, 32, 200)]
        _check_tokens(q, cache, table, n, starts, 0.09, (0, heads - 1), tokens, 0, softcap)


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("dim,heads,group,length,tokens", [
    (64, 2, 4, 300, 130), (128, 2, 4, 300, 130), (128, 64, 8, 4117, 201), (64, 2, 4, 300, 2)])
def test_attention_of_tokens_before_the_largest_value(dim, heads, group, length, tokens, cdtype):
    """V's last token holds bf16's largest value, whose code times its scale is 2^128: the
    tokens before it do not see it, in tiles of 128 and 256 rows and in those of few rows."""
    pages = -(-length // 32)
    g = _gen(83)
    cache = [torch.zeros(pages, heads, 32, dim, dtype=cdtype) for _ in range(2)]
    cache += [torch.zeros(pages, heads) for _ in range(2)]
    k, v = (torch.randn(length, heads, dim, generator=g).to(BF16) for _ in range(2))
    v[-1] = torch.finfo(BF16).max
    table = torch.randperm(pages, generator=g).to(torch.int32)[None]
    n = torch.tensor([length], dtype=torch.int32)
    dev = [c.cuda() for c in cache]
    K.kv_cache_write(k.cuda(), v.cuda(), *dev, table.cuda(), n.cuda(),
                     torch.tensor([0, length], dtype=torch.int32).cuda())
    cache = [c.cpu() for c in dev]
    last = cache[0][table[0, -1].long(), 0, (length - 1) % 32], cache[1][table[0, -1].long(), 0, (length - 1) % 32]
    assert float(last[1].float()[0]) * float(cache[3][table[0, -1].long(), 0]) == 2.0 ** 128
    q = torch.randn(tokens, heads * group, dim, generator=g).to(BF16)
    starts = torch.tensor([0, tokens], dtype=torch.int32)
    o = torch.full_like(q, 7.0).cuda()
    K.sdpa_cached(q.cuda(), *dev, table.cuda(), n.cuda(), o, 0.09, starts=starts.cuda())
    o = o.cpu()
    for i in {0, tokens // 2, tokens - 2}:
        for h in (0, heads - 1):
            qs = slice(h * group, (h + 1) * group)
            ref, size, reach = R.attention(q[i:i + 1, qs], *[c[:, h:h + 1] for c in cache], table,
                                           n - (tokens - 1 - i), 0.09)
            err = (o[i:i + 1, qs].double() - ref).abs()
            assert (err <= _tolerance(ref, size, reach, dim, length, 0.0)).all(), (i, h, float(err.max()))


@pytest.mark.parametrize("dim,group,length", [
    (64, 4, 524900), (64, 4, 525100), (128, 4, 393800), (128, 16, 442980), (64, 4, 524800)])
def test_attention_parts_of_one_long_sequence(dim, group, length):
    """One cache head and a sequence whose parts are a little longer than a multiple of 64
    when shared out evenly: the last positions, which weigh the most, are in some part."""
    page = 128
    pages = -(-length // page)
    g = _gen(84)
    cache = [torch.randint(-40, 41, (pages, 1, page, dim), generator=g, dtype=torch.int8) for _ in range(2)]
    cache += [torch.full((pages, 1), 2.0 ** -5) for _ in range(2)]
    last = length - 1
    table = torch.randperm(pages, generator=g).to(torch.int32)[None]
    for j in range(last - 9, last + 1):
        cache[0][table[0, j // page].long(), 0, j % page] = 40
        cache[1][table[0, j // page].long(), 0, j % page] = 100
    q = torch.ones(1, group, dim).to(BF16)
    n = torch.tensor([length], dtype=torch.int32)
    got = _check_attention(q, cache, table, n, None, dim ** -0.5 * (128 / dim) ** 0.5 * 2)
    assert (got > 2.5).all()  # (most of the weight is on V = 100 / 32)


def test_two_threads_on_one_stream():
    """Divided calls and column sums of two threads on one stream, some with larger
    workspaces than others, while a third gives the workspaces back: the bits of calls by
    themselves."""
    calls = [_attention_call([4000, 1333, 90], [1, 1, 1], 2, 4, 128, 32, INT8, 89, True),
             _attention_call([3000, 2333, 190], [1, 1, 1], 8, 8, 64, 32, E4M3, 90, True)]
    dev = [[q.cuda(), *[c.cuda() for c in cache], t.cuda(), n.cuda()] for q, cache, t, n, _ in calls]
    rows = torch.randn(4096, 512, generator=_gen(91)).cuda()
    prog = X.compile_expr(X.Leaf(0, F32))

    def once(i):
        o = torch.empty_like(dev[i][0])
        s = torch.empty(1, 512, device="cuda")
        K.sdpa_cached(*dev[i], o, 0.09)
        K.reduce(prog, [K.OperandMap(rows)], "sum", [0], s, (0, 0, 4096, 512))
        return o, s

    want = [once(i) for i in range(2)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(i):
        try:
            for _ in range(60):
                got[i].append(once(i))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    while any(t.is_alive() for t in threads):
        K.release_workspaces()
        time.sleep(0.001)
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for w, g in zip(want, got):
        assert len(g) == 60 and all(torch.equal(a, b) for x in g for a, b in zip(w, x))


def test_workspace_of_another_stream():
    """A call on a stream that is not the current one, while the current one has still to
    fill memory that it has given back: the call's workspace is not that memory."""
    q, cache, t, n, _ = _attention_call([4000, 1333, 90], [1, 1, 1], 2, 4, 128, 32, INT8, 92, True)
    dev = [q.cuda(), *[c.cuda() for c in cache], t.cuda(), n.cuda()]
    want = torch.empty_like(dev[0])
    K.sdpa_cached(*dev, want, 0.09)
    side = torch.cuda.Stream()
    out = [torch.empty_like(want) for _ in range(4)]
    torch.cuda.synchronize()
    for o in out:
        K.release_workspaces()
        blocks = [torch.empty(k << 20, dtype=torch.uint8, device="cuda") for k in (1, 2, 4, 8, 16, 32)]
        torch.cuda._sleep(2_000_000)  # (about a millisecond)
        for b in blocks:
            b.fill_(255)
        del b, blocks
        K.sdpa_cached(*dev, o, 0.09, stream=side)
        side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in out)


def test_captured_reductions_have_memory_of_their_own():
    """Column sums in two graphs, replayed while eager ones, some larger, run between."""
    prog = X.compile_expr(X.Leaf(0, F32))
    g = _gen(93)
    small, large = torch.randn(4096, 512, generator=g).cuda(), torch.randn(8192, 2048, generator=g).cuda()

    def sums(x, o):
        K.reduce(prog, [K.OperandMap(x)], "sum", [0], o, (0, 0) + tuple(x.shape))
        return o

    want, want_large = (sums(x, torch.empty(1, x.shape[1], device="cuda")) for x in (small, large))
    K.release_workspaces()
    xs = [torch.zeros_like(small) for _ in range(2)]
    outs = [torch.empty(1, 512, device="cuda") for _ in range(2)]
    graphs = []
    for x, o in zip(xs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            sums(x, o)
        graphs.append(graph)
    for j in range(6):
        for x, o, graph in zip(xs, outs, graphs):
            x.copy_(small if j % 2 else -small)
            graph.replay()
        assert torch.equal(sums(large, torch.empty_like(want_large)), want_large)
        junk = torch.full((8 << 20,), float("nan"), device="cuda")
        for o in outs:
            assert torch.equal(o, want if j % 2 else -want), j
        del junk
        torch.cuda.synchronize()
    K.release_workspaces()


@pytest.mark.parametrize("cdtype", [INT8, E4M3])
@pytest.mark.parametrize("old", [-1.0, -1000.0, -math.inf, math.inf, -0.0])
def test_write_behind_tokens_of_a_bad_scale(cdtype, old):
    """A page that is NaN for its readers stays so while tokens are appended to it."""
    for one in (True, False):
        cache = _cache(2, 2, 16, 64, cdtype, 85)
        _valid_codes(cache, None, None, None, 16)
        cache[2][1, 0], cache[3][1, 1] = old, old
        k = torch.randn(1, 2, 64, generator=_gen(86))
        table = torch.tensor([[1]], dtype=torch.int32)
        n = torch.tensor([5], dtype=torch.int32)
        starts = None if one else torch.tensor([0, 1], dtype=torch.int32)
        got = _run_write(k, k, cache, table, n, starts)
        assert math.isnan(got[2][1, 0]) == (old != 0.0) and not math.isnan(got[2][1, 1])
        q = torch.randn(1, 4, 64, generator=_gen(87)).to(BF16)
        _check_attention(q, got, table, n, None, 0.125)
        _run_write(k, k, got, table, torch.tensor([1], dtype=torch.int32), starts)


@pytest.mark.parametrize("dim,group,tokens", [(64, 4, 1), (128, 4, 1), (128, 20, 1), (64, 30, 1), (64, 4, 40),
                                              (128, 4, 40), (128, 8, 300)])
@pytest.mark.parametrize("softcap", [100.0, 129.0, 1000.0, 1e4, 65536.0])
def test_attention_of_close_scores_under_a_large_cap(softcap, dim, group, tokens):
    """Two positions whose scores, up to 192, differ by so little that o is the difference of
    two probabilities: p = 1 and p = 1 - i / 256, V = 1 and -1.  Both are numbers of bf16, and
    scores that are right to 2^-10 leave them so (a step of bf16 below 1 is 2^-8): o = (1 - p)
    / (1 + p) up to its rounding, 2^-8 of it, p's own error in the sum 1 + p, less than 2^-10
    of it, and fp32's (64 + n) 2^-24.

    The scores: sums of dim products that fp32 holds exactly, a few factors and the cap: 16
    roundings of numbers up to 192 log2 e < 512, 2^-12.  softcap tanh(s / softcap) is flatter
    than s, so i is whole only for large caps; where p is not near a number of bf16, its
    rounding may go either way."""
    heads, length = 8, 310
    page = 32
    pages = -(-length // page)
    k = torch.full((pages, heads, page, dim), -127, dtype=torch.int8)
    v = torch.zeros(pages, heads, page, dim, dtype=torch.int8)
    k[0, :, :2] = 127
    v[0, :, 0], v[0, :, 1] = 1, -1
    ks, vs = torch.empty(pages, heads), torch.ones(pages, heads)
    for h in range(heads):
        k[0, h, 1, 3 * h] = 126  # one less in the sum
        i = 1 + h % 3
        ks[:, h] = -math.log(1 - i / 256) * 128 / dim
    cache = [k, v, ks, vs]
    q = torch.full((tokens, heads * group, dim), 1.0).to(BF16)
    table = torch.arange(pages, dtype=torch.int32)[None]
    n, starts = torch.tensor([length], dtype=torch.int32), torch.tensor([0, tokens], dtype=torch.int32)
    scale = dim / 128
    out = torch.full_like(q, 7.0).cuda()
    K.sdpa_cached(q.cuda(), *[c.cuda() for c in cache], table.cuda(), n.cuda(), out, scale,
                  starts=starts.cuda(), softcap=softcap)
    got = out.cpu().double()
    for h in range(heads):
        s = torch.tensor([127.0 * dim, 127.0 * dim - 1], dtype=torch.float64) * float(ks[0, h]) * scale
        assert float(s[0]) < 192
        s = softcap * torch.tanh(s / softcap)
        p = float(torch.exp(s[1] - s[0]))
        near = round(p * 256) / 256
        ref = (1 - near) / (1 + p)
        off = 2.0 ** -10
        tol = 2.0 ** -8 * ref + 2 * off * ref + 400 * 2.0 ** -24
        if abs(near - p) > 2.0 ** -9 - off:  # (either neighbour)
            tol += 2.0 ** -8
        err = (got[:, h * group:(h + 1) * group] - ref).abs().max()
        assert float(err) <= tol, (h, p, ref, float(err), tol)


@pytest.mark.parametrize("news", [[1, 1], [130, 40]])
@pytest.mark.parametrize("softcap,loud", [(129.0, 100.0), (1000.0, 300.0), (1000.0, 3000.0), (65536.0, 4.0)])
def test_attention_large_caps(softcap, loud, news):
    """Scores far below, about and far above the cap."""
    q, cache, table, n, starts = _attention_call([300, 55], news, 2, 4, 128, 32, INT8, 88, loud=loud)
    _check_attention(q, cache, table, n, starts, 0.09, softcap=softcap)
    _check_attention(q, cache, table, n, starts, -0.09, window=50, softcap=softcap)
    table[0, 2] = -1
    cache[2][table[0, 7], 1] = math.nan
    _check_attention(q, cache, table, n, starts, 0.09, softcap=softcap)
