"""Rotary positions and the 8-bit key/value cache without a GPU: what the wrappers
and the library refuse, the frequencies, and the header's rules for positions and
scales, compiled for the host."""

import contextlib
import ctypes
import math
import os
import shutil
import subprocess
import threading
import time
import weakref

import pytest
import torch

from oracle import kv_cache as R
from ttlhip import _lib as L
from ttlhip import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


def _call(**change):
    """A valid call's arguments on the CPU, some of them changed."""
    a = dict(k_cache=torch.zeros(6, 2, 16, 64, dtype=INT8), v_cache=torch.zeros(6, 2, 16, 64, dtype=INT8),
             k_scale=torch.ones(6, 2), v_scale=torch.ones(6, 2),
             table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.ones(3, dtype=torch.int32),
             starts=torch.tensor([0, 2, 3, 5], dtype=torch.int32))
    a.update(change)
    return a


X = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
Q = torch.zeros(5, 6, 64, dtype=torch.bfloat16)

BAD_CACHES = [
    dict(k_cache=torch.zeros(6, 2, 16, 64)),
    dict(k_cache=torch.zeros(6, 2, 16, 64, dtype=E4M3)),
    dict(k_cache=torch.zeros(6, 2, 16, 64, dtype=INT8).transpose(1, 2)),
    dict(k_cache=torch.zeros(6, 2, 16 * 64, dtype=INT8)),
    dict(v_cache=torch.zeros(7, 2, 16, 64, dtype=INT8)),
    dict(k_scale=torch.ones(6, 2, dtype=torch.float64)),
    dict(v_scale=torch.ones(6, 3)),
    dict(k_scale=torch.ones(6, 4)[:, ::2]),
    dict(table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]),
    dict(table=torch.zeros(3, dtype=torch.int32)),
    dict(lengths=torch.ones(2, dtype=torch.int32)),
    dict(lengths=torch.ones(3, dtype=torch.int64)),
    dict(starts=torch.zeros(3, dtype=torch.int32)),
    dict(starts=torch.zeros(4, dtype=torch.int64)),
    dict(starts=None),  # 5 tokens, 3 sequences
]


@pytest.mark.parametrize("change", BAD_CACHES)
def test_bad_caches_are_refused(change):
    with pytest.raises(ValueError):
        K.kv_cache_write(X, X, **_call(**change))
    with pytest.raises(ValueError):
        K.sdpa_cached(Q, o=Q.clone(), scale=0.1, **_call(**change))


@pytest.mark.parametrize("k,v", [
    (X[0], X[0]), (X, X[:4]), (X, X.float()), (torch.zeros(5, 3, 64), torch.zeros(5, 3, 64)),
    (torch.zeros(5, 2, 128), torch.zeros(5, 2, 128)), (torch.zeros(5, 2, 128)[..., ::2],) * 2])
def test_bad_tokens_are_refused(k, v):
    with pytest.raises(ValueError):
        K.kv_cache_write(k, v, **_call())


def test_half_precision_is_refused():
    with pytest.raises(TypeError):
        K.kv_cache_write(X.half(), X.half(), **_call())


@pytest.mark.parametrize("q,o", [
    (Q[0], Q[0]), (Q, Q[:4]), (Q.float(), Q.float()), (Q, Q.float()), (Q[:, :3], Q[:, :3].clone()),
    (torch.zeros(5, 4, 128, dtype=torch.bfloat16),) * 2,
    (Q, torch.zeros(5, 1, 64, dtype=torch.bfloat16).expand(5, 6, 64)),
    (Q, torch.zeros(1, 6, 64, dtype=torch.bfloat16).expand(5, 6, 64)),
    (torch.zeros(5, 6, 68, dtype=torch.bfloat16)[..., :64], Q),
    (torch.zeros(5 * 6 * 64 + 1, dtype=torch.bfloat16)[1:].view(5, 6, 64), Q)])
def test_bad_queries_are_refused(q, o):
    with pytest.raises(ValueError):
        K.sdpa_cached(q, o=o, scale=0.1, **_call())


def test_device_tensors_only():
    for f in (lambda: K.kv_cache_write(X, X, **_call()),
              lambda: K.sdpa_cached(Q, o=Q.clone(), scale=0.1, **_call()),
              lambda: K.rope(X, torch.zeros(5, dtype=torch.int32), K.rope_freqs(64, device="cpu"), X)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


class _On:
    """A tensor of another device, as far as the check looks at it."""

    is_cuda = True

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


def test_tensors_of_other_devices_are_refused(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    K._check_on_one_device("f", (_On(0), _On(0)), None)
    for tensors in ((_On(1), _On(1)), (_On(0), _On(1))):
        with pytest.raises(ValueError, match="device 1"):
            K._check_on_one_device("f", tensors, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K._check_on_one_device("f", (_On(0), X), None)
    stream = type("S", (), {"device": torch.device("cuda", 1)})()
    K._check_on_one_device("f", (_On(1), _On(1)), stream)
    with pytest.raises(ValueError, match="device 0, the launch on 1"):
        K._check_on_one_device("f", (_On(0),), stream)


def test_one_cache_for_k_and_v_is_refused():
    a = _call()
    a["v_cache"] = a["k_cache"]
    with pytest.raises(ValueError, match="one memory"):
        K.kv_cache_write(X, X, **a)


POS, FREQS = torch.zeros(5, dtype=torch.int32), torch.ones(32, dtype=torch.float64)


@pytest.mark.parametrize("change", [
    dict(x=X[0]), dict(out=X[:4]), dict(out=X.float()), dict(positions=POS[:4]),
    dict(positions=POS.float()), dict(positions=torch.zeros(10, dtype=torch.int32)[::2]),
    dict(freqs=FREQS.float()), dict(freqs=torch.ones(33, dtype=torch.float64)),
    dict(freqs=torch.ones(64, dtype=torch.float64)[::2]), dict(freqs=FREQS[None]),
    dict(x=torch.zeros(5, 2, 128, dtype=torch.bfloat16)[..., ::2]),
    dict(out=torch.zeros(5, 1, 64, dtype=torch.bfloat16).expand(5, 2, 64)),
    dict(out=X.view(2, 5, 64).transpose(0, 1))])
def test_bad_rope_calls_are_refused(change):
    a = dict(x=X, positions=POS, freqs=FREQS, out=torch.zeros_like(X))
    a.update(change)
    with pytest.raises(ValueError):
        K.rope(**a)


# --- the C ABI ----------------------------------------------------------------


def _c_cache(**change):
    c = L.KVCache(k=4096, v=8192, k_scale=256, v_scale=512, table=1024, lengths=2048, starts=3000,
                  table_ld=2, pages=6, width=2, heads=2, seqs=3, tokens=5, page=16, dim=64,
                  format=0, pad=0)
    for n, x in change.items():
        setattr(c, n, x)
    return ctypes.byref(c)


@pytest.mark.parametrize("change,status", [
    (dict(page=24), L.TTLH_EUNSUPPORTED), (dict(page=256), L.TTLH_EUNSUPPORTED),
    (dict(dim=96), L.TTLH_EUNSUPPORTED), (dict(format=2), L.TTLH_EINVAL),
    (dict(heads=0), L.TTLH_EINVAL), (dict(pages=-1), L.TTLH_EINVAL), (dict(seqs=-1), L.TTLH_EINVAL),
    (dict(table_ld=1), L.TTLH_EINVAL), (dict(starts=None), L.TTLH_EINVAL),
    (dict(k=None), L.TTLH_EINVAL), (dict(k=4100), L.TTLH_EINVAL), (dict(lengths=None), L.TTLH_EINVAL),
    (dict(table=None), L.TTLH_EINVAL), (dict(v_scale=None), L.TTLH_EINVAL),
    (dict(width=2 ** 26 + 1), L.TTLH_EINVAL),
    (dict(width=2 ** 26 + 1, table_ld=2 ** 27), L.TTLH_EUNSUPPORTED),
    (dict(tokens=2 ** 28), L.TTLH_EUNSUPPORTED), (dict(pages=2 ** 31), L.TTLH_EUNSUPPORTED)])
def test_library_refuses_bad_caches(change, status):
    lib = L.load()
    assert lib.ttlh_kv_cache_write(_c_cache(**change), 16, 16, 0, 128, 64, 128, 64, None) == status
    assert lib.ttlh_last_error()
    assert lib.ttlh_sdpa_cached(_c_cache(**change), 16, 16, 4, 256, 64, 256, 64, 0.1, 0, 0.0, None, 0,
                                None) == status


def test_library_refuses_bad_calls():
    lib = L.load()
    E = L.TTLH_EINVAL
    # a workspace that is not there, too small or off its alignment
    long = _c_cache(width=200, table_ld=200)
    need = lib.ttlh_sdpa_cached_workspace_bytes(long, 4)
    assert need > 0
    for ws, size in ((None, need), (4096, need - 1), (4104, need)):
        assert lib.ttlh_sdpa_cached(long, 16, 16, 4, 256, 64, 256, 64, 0.1, 0, 0.0, ws, size, None) == E
    assert b"workspace" in lib.ttlh_last_error()
    assert lib.ttlh_sdpa_cached_workspace_bytes(_c_cache(), 4) == 0
    assert lib.ttlh_kv_cache_write(None, 16, 16, 0, 128, 64, 128, 64, None) == E
    assert lib.ttlh_kv_cache_write(_c_cache(), 16, 16, 2, 128, 64, 128, 64, None) == E
    assert lib.ttlh_kv_cache_write(_c_cache(), None, 16, 0, 128, 64, 128, 64, None) == E

    def attention(q=16, o=16, heads=4, strides=(256, 64, 256, 64), scale=0.1, window=0, cap=0.0):
        return lib.ttlh_sdpa_cached(_c_cache(), q, o, heads, *strides, scale, window, cap, None, 0, None)

    for bad in (dict(q=None), dict(q=8), dict(o=8), dict(heads=3), dict(heads=0), dict(window=-1),
                dict(strides=(252, 64, 256, 64)), dict(strides=(256, 64, 256, 4)),
                dict(scale=math.inf), dict(scale=math.nan), dict(cap=-1.0), dict(cap=math.nan),
                dict(cap=math.inf), dict(cap=1e-6), dict(cap=1e6), dict(scale=1e31)):
        assert attention(**bad) == E, bad

    def rope(x=16, dtype=0, pos=16, pb=4, freqs=16, sizes=(5, 2, 64, 64), scale=1.0):
        return lib.ttlh_rope(x, x, dtype, pos, pb, freqs, *sizes, 128, 64, 128, 64, 0, scale, 0, None)

    for bad in (dict(x=None), dict(dtype=3), dict(pos=None), dict(pb=2), dict(freqs=None),
                dict(sizes=(5, 2, 64, 63)), dict(sizes=(5, 2, 64, 66)), dict(sizes=(-1, 2, 64, 64)),
                dict(sizes=(5, 2, 0, 0)), dict(scale=math.nan)):
        assert rope(**bad) == E, bad
    assert rope(sizes=(5, 2, 4096, 2048)) == L.TTLH_EUNSUPPORTED
    assert rope(sizes=(2 ** 31, 2, 64, 64)) == L.TTLH_EUNSUPPORTED


def test_nothing_to_do_is_no_error():
    lib = L.load()
    assert lib.ttlh_rope(None, None, 0, None, 4, None, 0, 2, 64, 64, 0, 0, 0, 0, 0, 1.0, 0, None) == 0
    empty = _c_cache(tokens=0)
    assert lib.ttlh_kv_cache_write(empty, None, None, 0, 0, 0, 0, 0, None) == 0
    assert lib.ttlh_sdpa_cached(empty, None, None, 4, 0, 0, 0, 0, 0.1, 0, 0.0, None, 0, None) == 0


# --- frequencies --------------------------------------------------------------


def test_rope_freqs():
    f = K.rope_freqs(8, base=10000.0, device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(K.rope_freqs(8, scaling="linear", factor=4.0, device="cpu"), f / 4, rtol=1e-14)
    b = K.rope_freqs(8, scaling="base", factor=4.0, device="cpu")
    assert abs(float(b[0]) - 1) < 1e-14 and abs(float(b[-1]) / float(f[-1]) - 0.25) < 1e-14
    # turns over 4096: 652, 65, 6.5, 0.65: two kept, one blended, one divided
    p = K.rope_freqs(8, scaling="parts", factor=4.0, original=4096, device="cpu")
    assert torch.equal(p[:2], f[:2]) and abs(float(p[3] / f[3]) - 0.25) < 1e-14
    keep = (4096 * 0.01 / (2 * math.pi) - 1) / 31
    assert abs(float(p[2]) - 0.01 * (keep + (1 - keep) / 4)) < 1e-16


@pytest.mark.parametrize("bad", [dict(rot=3), dict(rot=0), dict(rot=8, base=0.0), dict(rot=8, factor=0.5),
                                 dict(rot=8, scaling="other"), dict(rot=8, scaling="parts", factor=2.0),
                                 dict(rot=8, scaling="parts", original=10, fast=1.0, slow=1.0)])
def test_bad_frequencies_are_refused(bad):
    with pytest.raises(ValueError):
        K.rope_freqs(device="cpu", **bad)


# --- the header's rules, on the host ------------------------------------------

SOURCE = r"""
#include "ttlh_kvcache.h"
extern "C" float scale_for(float a, int f) { return ttlh::scale_for(a, f); }
extern "C" float joined(float a, float b) { return ttlh::joined_scale(a, b); }
extern "C" float sound(float a) { return ttlh::sound_scale(a); }
static ttlh::CacheArgs args(const int32_t* t, int ld, int width, int pages, int shift, const int32_t* starts,
                            int tokens) {
  ttlh::CacheArgs c = {};
  c.table = t; c.table_ld = ld; c.width = width; c.pages = pages; c.shift = shift; c.starts = starts;
  c.tokens = tokens; c.heads = 8; c.dim = 128;
  return c;
}
extern "C" int page_at(const int32_t* t, int ld, int width, int pages, int shift, int b, int pos) {
  return ttlh::page_at(args(t, ld, width, pages, shift, nullptr, 0), b, pos);
}
extern "C" void tokens_of(const int32_t* s, int tokens, int b, int* out) {
  ttlh::seq_tokens(args(nullptr, 0, 0, 0, 4, s, tokens), b, out[0], out[1]);
}
extern "C" void seen(int width, int len, int n, int i, int window, int* out) {
  ttlh::seen_by(args(nullptr, 0, width, 0, 4, nullptr, 0), len, n, i, window, out[0], out[1]);
}
extern "C" int64_t offset(int page, int head, int slot) {
  return ttlh::slot_offset(args(nullptr, 0, 0, 0, 7, nullptr, 0), page, head, slot);
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "tt-lang_amd", "csrc"), str(d / "rules.cpp"), "-o",
                    str(d / "rules.so")], check=True)
    lib = ctypes.CDLL(str(d / "rules.so"))
    lib.scale_for.restype = lib.joined.restype = ctypes.c_float
    lib.scale_for.argtypes = [ctypes.c_float, ctypes.c_int]
    lib.joined.argtypes = [ctypes.c_float, ctypes.c_float]
    lib.sound.restype, lib.sound.argtypes = ctypes.c_float, [ctypes.c_float]
    lib.offset.restype = ctypes.c_int64
    return lib


@pytest.mark.parametrize("fmt,dtype", [(0, INT8), (1, E4M3)])
def test_scales_are_the_smallest_powers_of_two(rules, fmt, dtype):
    vals = [0.0, 1e-45, 1e-38, 2.0 ** -126, 2.0 ** -120, 1.0, 126.9, 127.0, 127.00001, 254.0, 254.1, 448.0,
            448.1, 3.4028234e38, 1e-30, 0.3]
    vals += [float(v) for v in torch.randn(200, generator=torch.Generator().manual_seed(1)).abs()]
    for a in vals:
        a = ctypes.c_float(a).value
        s = rules.scale_for(a, fmt)
        assert s == R.scale_for(a, dtype), a
        assert R.TOP[dtype] * s >= a
    assert math.isnan(rules.scale_for(math.inf, fmt)) and math.isnan(rules.scale_for(math.nan, fmt))


def test_joined_scales(rules):
    nan, inf = math.nan, math.inf
    assert rules.joined(1.0, 2.0) == 2.0 and rules.joined(2.0, 1.0) == 2.0
    assert rules.joined(0.0, 1.0) == 1.0 and rules.joined(-1.0, 1.0) == 1.0
    for a, b in ((nan, 1.0), (1.0, nan), (inf, 1.0)):
        assert math.isnan(rules.joined(a, b))


def test_positions_outside_have_no_page(rules):
    t = (ctypes.c_int32 * 8)(0, 5, -1, 6, 2, 2 ** 31 - 1, -2 ** 31, 3)
    at = lambda b, pos: rules.page_at(t, 4, 4, 6, 4, b, pos)  # noqa: E731
    assert [at(0, p) for p in (0, 15, 16, 31, 32, 48, 63)] == [0, 0, 5, 5, -1, -1, -1]
    assert [at(1, p) for p in (0, 16, 32, 48)] == [2, -1, -1, 3]
    for pos in (-1, -2 ** 31, 64, 2 ** 31 - 1):
        assert at(0, pos) == -1
    assert rules.page_at(t, 4, 0, 6, 4, 0, 0) == -1


def test_tokens_outside_the_packed_rows_do_not_exist(rules):
    def of(starts, tokens):
        s, out = (ctypes.c_int32 * len(starts))(*starts), (ctypes.c_int * 2)()
        res = []
        for b in range(len(starts) - 1):
            rules.tokens_of(s, tokens, b, out)
            res.append((out[0], out[1]))
        return res
    assert of([0, 2, 2, 5], 5) == [(0, 2), (2, 0), (2, 3)]
    for starts in ([-3, 12, 500], [15, 5, 20], [2 ** 31 - 1, -2 ** 31, 7], [30, 31, 32]):
        for first, n in of(starts, 20):
            assert 0 <= first <= first + n <= 20


def test_what_a_token_sees(rules):
    def seen(*a):
        out = (ctypes.c_int * 2)()
        rules.seen(*a, out)
        return range(out[0], out[1])
    big = 2 ** 31 - 1
    for width in (0, 3, 2 ** 26):
        for length in (0, 1, 20, 48, 60, big, -1, -big - 1):
            for n in (1, 7, 2 ** 28 - 1):
                for i in {0, n // 2, n - 1}:
                    for window in (0, 1, 5, big):
                        end = length - n + i + 1
                        want = range(max(0, end - window) if window else 0, max(0, end))
                        want = range(min(want.start, 16 * width), min(want.stop, 16 * width))
                        got = seen(width, length, n, i, window)
                        assert list(got[:3]) == list(want[:3]) and len(got) == len(want)


def test_offsets_pass_32_bits(rules):
    assert rules.offset(2 ** 20, 7, 127) == ((2 ** 20 * 8 + 7) * 128 + 127) * 128


# --- workspaces, on the host ------------------------------------------------------


class _Library:
    """Stands for the library where a call needs a workspace: notes where each launch's is
    and whether its memory is alive, and lets other threads run while it launches."""

    def __init__(self, monkeypatch):
        self.alive, self.inside, self.overlaps, self.dead = {}, {}, [], []
        empty = torch.empty

        def noted(*a, **k):
            t = empty(*a, **k)
            self.alive[t.data_ptr()] = t.numel()
            weakref.finalize(t, self.alive.pop, t.data_ptr(), None)
            return t

        monkeypatch.setattr(K.torch, "empty", noted)
        monkeypatch.setattr(K.L, "call", self.call)
        monkeypatch.setattr(K.L, "stream_ptr", lambda stream=None: 1234)
        monkeypatch.setattr(K, "_check_on_one_device", lambda *a: None)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        K.release_workspaces()

    def call(self, fn, *args):
        assert fn == "ttlh_sdpa_cached"
        ws, nbytes = args[-3], args[-2]
        if ws in self.inside:
            self.overlaps.append(ws)
        self.inside[ws] = True
        time.sleep(0.002)
        if self.alive.get(ws, 0) < nbytes:
            self.dead.append(ws)
        self.inside.pop(ws, None)


def _long_call(width):
    return _call(table=torch.zeros(3, width, dtype=torch.int32))


def test_threads_take_turns_at_a_streams_workspace(monkeypatch):
    """A call has two launches: nobody else's on the same memory may come between them, and
    the memory lives until they are done, also where another thread asks for more of it or
    gives the workspaces back."""
    lib = _Library(monkeypatch)
    errors = []

    def work(i):
        try:
            for j in range(12):
                q = torch.zeros(5, 2 * (1 + (i + j) % 4), 64, dtype=torch.bfloat16)
                K.sdpa_cached(q, o=q.clone(), scale=0.1, **_long_call(200))
                if i == 0 and j % 4 == 3:
                    K.release_workspaces()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    K.release_workspaces()
    assert not errors and not lib.overlaps and not lib.dead


def test_other_streams_do_not_wait(monkeypatch):
    """The workspaces of two streams are two."""
    lib = _Library(monkeypatch)
    seen = []
    monkeypatch.setattr(K.L, "call", lambda fn, *a: seen.append(a[-3]))
    for sp in (1, 2, 1):
        monkeypatch.setattr(K.L, "stream_ptr", lambda stream=None, sp=sp: sp)
        K.sdpa_cached(Q, o=Q.clone(), scale=0.1, **_long_call(200))
    assert seen[0] == seen[2] != seen[1] and not lib.overlaps
    K.release_workspaces()


class _Stream:
    device = torch.device("cuda", 0)
    cuda_stream = 77


def _current(monkeypatch, pointers, capturing=()):
    """The current stream is pointers[-1] (a list that torch.cuda.stream() pushes to);
    streams in `capturing` are being captured."""

    @contextlib.contextmanager
    def stream(s):
        pointers.append(s.cuda_stream)
        yield
        pointers.pop()

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None, raising=False)
    monkeypatch.setattr(K.L, "stream_ptr", lambda s=None: pointers[-1] if s is None else s.cuda_stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: pointers[-1] in capturing)


@pytest.mark.parametrize("captured", [None, 5, 77])
def test_workspaces_come_from_the_launch_stream(monkeypatch, captured):
    """Memory for stream 77 is asked for on stream 77, and it is 77's capture that counts:
    captured calls have memory of their own, which a later eager call does not get."""
    lib = _Library(monkeypatch)
    streams = [5]
    capturing = {captured}
    _current(monkeypatch, streams, capturing)
    asked, used = [], []
    empty = torch.empty  # (the library's)
    monkeypatch.setattr(K.torch, "empty", lambda *a, **k: (asked.append(streams[-1]), empty(*a, **k))[1])
    kept = []

    def call(fn, *a):
        assert lib.alive.get(a[-3], 0) >= a[-2]
        used.append(a[-3])
        kept.append(empty(a[-2], dtype=torch.uint8))  # (nothing else gets this address)

    monkeypatch.setattr(K.L, "call", call)
    q, o = Q, Q.clone()
    for _ in range(2):
        K.sdpa_cached(q, o=o, scale=0.1, stream=_Stream(), **_long_call(200))
    assert streams == [5]
    assert asked == ([77, 77] if captured == 77 else [77])
    if captured == 77:
        assert not K._WORKSPACES
        capturing.clear()
        K.sdpa_cached(q, o=o, scale=0.1, stream=_Stream(), **_long_call(200))
        assert asked == [77, 77, 77]
    else:
        assert used[0] == used[1]
    K.release_workspaces()


def test_scales_that_readers_take_as_nan(rules):
    for s in (-1.0, -1e-45, -math.inf, math.inf, math.nan):
        assert math.isnan(rules.sound(s)) and math.isnan(rules.joined(rules.sound(s), 1.0))
    for s in (0.0, -0.0, 1e-45, 2.0 ** -126, 3.0, 3.4028234e38):
        s = ctypes.c_float(s).value
        assert rules.sound(s) == s


def test_caches_and_scales_that_overlap_are_refused():
    """K's and V's codes or scales in one memory, whole or in part, would be written by both."""
    both = torch.zeros(7, 2, 16, 64, dtype=INT8)
    scales = torch.ones(7, 2)
    for change in (dict(k_cache=both[:6], v_cache=both[1:]), dict(k_cache=both[1:], v_cache=both[:6]),
                   dict(k_scale=scales[:6], v_scale=scales[:6]), dict(k_scale=scales[:6], v_scale=scales[1:])):
        with pytest.raises(ValueError, match="one memory"):
            K.kv_cache_write(X, X, **_call(**change))
    two, sc = torch.zeros(12, 2, 16, 64, dtype=INT8), torch.ones(12, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):  # halves of one buffer are two
        K.kv_cache_write(X, X, **_call(k_cache=two[:6], v_cache=two[6:], k_scale=sc[:6], v_scale=sc[6:]))
    none, ns = torch.zeros(0, 2, 16, 64, dtype=INT8), torch.ones(0, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):  # and nothing has no memory
        K.kv_cache_write(X, X, **_call(k_cache=none, v_cache=none.clone(), k_scale=ns, v_scale=ns.clone()))


def test_results_over_other_views_of_the_queries_are_refused():
    """o may be q itself: with other strides, rows that others still read would be written."""
    square = torch.zeros(6, 6, 64, dtype=torch.bfloat16)
    a = _call(starts=torch.tensor([0, 2, 3, 6], dtype=torch.int32))
    with pytest.raises(ValueError, match="another view"):
        K.sdpa_cached(square, o=square.transpose(0, 1), scale=0.1, **a)
    with pytest.raises(RuntimeError, match="no CPU path"):
        K.sdpa_cached(square, o=square, scale=0.1, **a)


def test_library_refuses_rows_past_31_bits():
    """The rows of a sequence, new tokens x q heads of a cache head, are rounded up to a tile
    in 32 bits."""
    lib = L.load()
    cache = _c_cache(heads=1, tokens=2 ** 28 - 1)
    for q_heads in (8, 9):  # (2 ** 31 - 8 rows; more)
        assert lib.ttlh_sdpa_cached(cache, 16, 16, q_heads, 512, 64, 512, 64, 0.1, 0, 0.0, None, 0,
                                    None) == L.TTLH_EUNSUPPORTED


def test_library_refuses_grids_past_32_bits_of_threads():
    lib = L.load()
    cache = _c_cache(heads=4, seqs=2 ** 22, tokens=2 ** 22, starts=None, width=200, table_ld=200)
    need = lib.ttlh_sdpa_cached_workspace_bytes(cache, 4)
    assert lib.ttlh_sdpa_cached(cache, 16, 16, 4, 256, 64, 256, 64, 0.1, 0, 0.0, 4096, need,
                                None) == L.TTLH_EUNSUPPORTED
