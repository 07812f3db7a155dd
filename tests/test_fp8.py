"""Linear layers in 8-bit floating point without a GPU: what the wrappers and the library
refuse, the weights' codes, and the header's rules for scales, compiled for the host."""

import ctypes
import os
import subprocess

import pytest
import torch

from oracle import fp8 as R
from ttlhip import _lib as L
from ttlhip import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, E4M3, E8M0 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _scales(rows, dim):
    return K.fp8_scales(rows, dim, device="cpu")


def _codes(rows, dim):
    return torch.zeros(rows, dim, dtype=E4M3)


X = torch.zeros(6, 640, dtype=BF16)
BUF = torch.zeros(6, 1280, dtype=BF16)
W = torch.ones(640)

BAD_OUT = [
    dict(codes=_codes(5, 640)),
    dict(codes=_codes(6, 639)),
    dict(codes=torch.zeros(6, 640, dtype=torch.int8)),
    dict(codes=torch.zeros(6, 640, dtype=torch.float8_e5m2)),
    dict(codes=_codes(6, 1280)[:, ::2]),
    dict(codes=_codes(1, 640).expand(6, 640)),
    dict(codes=torch.zeros(6 * 640, dtype=E4M3)),
    dict(codes=torch.empty_strided((6, 640), (320, 1), dtype=E4M3)),
    dict(scales=_scales(6, 512)),
    dict(scales=_scales(5, 640)),
    dict(scales=torch.ones(2, 6, 4)),
    dict(scales=torch.ones(2, 6, 4, dtype=torch.uint8)),
    dict(scales=torch.ones(2, 12, 4, dtype=torch.uint8).view(E8M0)[:, ::2]),
    dict(scales=torch.ones(2, 4, 6, dtype=torch.uint8).view(E8M0).transpose(1, 2)),
    dict(scales=torch.ones(50, dtype=torch.uint8)[1:49].view(2, 6, 4).view(E8M0)),
    dict(scales=_scales(6, 512).expand(2, 6, 4)),
    dict(codes=BUF.view(E4M3)[:, :640], x=BUF[:, 100:740]),
]


@pytest.mark.parametrize("change", BAD_OUT)
def test_bad_outputs_are_refused(change):
    a = dict(x=X, codes=_codes(6, 640), scales=_scales(6, 640))
    a.update(change)
    with pytest.raises(ValueError):
        K.quant_fp8(**a)
    with pytest.raises(ValueError):
        K.rms_norm_fp8(a["x"], W, a["codes"], a["scales"])
    with pytest.raises(ValueError):
        K.glu_fp8(a["x"], X, a["codes"], a["scales"])


def test_codes_and_scales_of_one_memory_are_refused():
    m = torch.zeros(2, 6, 1280, dtype=torch.uint8)
    with pytest.raises(ValueError, match="memory in common"):
        K.quant_fp8(X, m.view(E4M3)[0, :, :640], m.view(-1)[:48].view(2, 6, 4).view(E8M0))


@pytest.mark.parametrize("x", [X[0], X[None], BUF[:, ::2], torch.zeros(6, 0, dtype=BF16)])
def test_bad_values_are_refused(x):
    with pytest.raises(ValueError):
        K.quant_fp8(x, _codes(6, 640), _scales(6, 640))


def test_empty_rows_are_refused():
    with pytest.raises(ValueError):
        K.quant_fp8(torch.zeros(6, 0), torch.zeros(6, 0, dtype=E4M3), torch.zeros(0, 6, 4, dtype=torch.uint8).view(E8M0))
    with pytest.raises(ValueError):
        K.fp8_scales(6, 0)


def test_half_precision_is_refused():
    with pytest.raises(TypeError):
        K.quant_fp8(X.half(), _codes(6, 640), _scales(6, 640))
    with pytest.raises(TypeError):
        K.rms_norm_fp8(X, W.half(), _codes(6, 640), _scales(6, 640))
    with pytest.raises(TypeError):
        K.glu_fp8(X.half(), X.half(), _codes(6, 640), _scales(6, 640))


@pytest.mark.parametrize("change", [
    dict(weight=torch.ones(639)), dict(weight=torch.ones(1, 640)), dict(weight=torch.ones(1280)[::2]),
    dict(residual=X[:5]), dict(residual=X.float()), dict(residual=BUF[:, ::2]),
    dict(total=X.float()), dict(total=X[:, :639]),
    dict(total=torch.zeros(1, 640, dtype=BF16).expand(6, 640)),
    dict(x=BUF[:, :640], total=BUF[:, 8:648]),
    dict(residual=BUF[:, :640], total=BUF[:, 8:648]),
    dict(residual=BUF[:, :640], total=BUF.view(-1)[:3840].view(6, 640))])
def test_bad_norms_are_refused(change):
    a = dict(x=X, weight=W, codes=_codes(6, 640), scales=_scales(6, 640))
    a.update(change)
    with pytest.raises(ValueError):
        K.rms_norm_fp8(**a)


@pytest.mark.parametrize("eps", [-1e-6, 0.0, 1e-50, float("nan"), float("inf")])
def test_the_library_refuses_a_bad_eps(eps):
    lib = L.load()
    st = lib.ttlh_fp8_rms_norm(16, 640, 0, 0, 0, 0, 0, 16, 0, eps, 16, 640, 16, 6, 6, 640, None)
    assert st == L.TTLH_EINVAL and b"eps" in lib.ttlh_last_error()


@pytest.mark.parametrize("change", [dict(up=X[:5]), dict(up=X.float()), dict(act="relu"), dict(act=0),
                                    dict(gate=X[0])])
def test_bad_gates_are_refused(change):
    a = dict(gate=X, up=X, codes=_codes(6, 640), scales=_scales(6, 640))
    a.update(change)
    with pytest.raises(ValueError):
        K.glu_fp8(**a)


def _product(**change):
    a = dict(x=_codes(6, 640), x_scale=_scales(6, 640), w=_codes(300, 640), w_scale=_scales(3, 640),
             c=torch.zeros(6, 300, dtype=BF16))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(x=_codes(6, 656)), dict(x=_codes(5, 640)), dict(x=_codes(6, 640)[0]), dict(x=X),
    dict(x=_codes(6, 648)[:, :640]), dict(x=_codes(6, 656)[:, 8:648]), dict(x=_codes(6, 1280)[:, ::2]),
    dict(x_scale=_scales(5, 640)), dict(x_scale=_scales(6, 512)), dict(x_scale=torch.ones(2, 6, 4)),
    dict(w=_codes(299, 640)), dict(w=torch.zeros(300, 640, dtype=torch.int8)),
    dict(w=_codes(300, 648)[:, :640]), dict(w_scale=_scales(2, 640)), dict(w_scale=_scales(300, 640)),
    dict(c=torch.zeros(6, 299)), dict(c=torch.zeros(6, 600)[:, ::2]), dict(c=torch.zeros(1, 300).expand(6, 300)),
    dict(x=_codes(6, 632), w=_codes(300, 632)),
    dict(x=_codes(6, 0), w=_codes(300, 0))])
def test_bad_products_are_refused(change):
    with pytest.raises(ValueError):
        K.matmul_fp8(**_product(**change))


def test_products_into_half_precision_or_their_operands_are_refused():
    with pytest.raises(TypeError):
        K.matmul_fp8(**_product(c=torch.zeros(6, 300, dtype=torch.half)))
    m = torch.zeros(6, 640, dtype=torch.uint8)
    with pytest.raises(ValueError, match="memory in common"):
        K.matmul_fp8(**_product(x=m.view(E4M3), c=m.view(BF16)[:, 10:310]))


def test_device_tensors_only():
    o = (_codes(6, 640), _scales(6, 640))
    for f in (lambda: K.quant_fp8(X, *o), lambda: K.rms_norm_fp8(X, W, *o), lambda: K.glu_fp8(X, X, *o),
              lambda: K.matmul_fp8(**_product())):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


def test_rows_of_one_buffer_may_lie_beside_each_other():
    """The check that refuses common memory knows rows that lie between others."""
    assert K._apart(BUF[:, :640], BUF[:, 640:])
    assert not K._apart(BUF[:, :641], BUF[:, 640:])
    assert not K._apart(BUF[:, 640:], BUF[:, :641])
    assert K._apart(BUF[:3], BUF[3:]) and not K._apart(BUF[:4], BUF[3:])
    assert K._apart(BUF[:0], BUF)
    assert not K._apart(BUF[:, :640], BUF.view(-1)[:3840].view(6, 640))
    assert not K._apart(BUF[1:2, :4], BUF[:, 4:])  # (one row: by its ends alone)


def test_the_library_refuses_what_it_cannot_run():
    lib = L.load()

    def quant(dtype=0, codes=16, scales=16, rows=6, dim=640, x=16, ld=1 << 40, sl=1 << 40):
        return lib.ttlh_fp8_quant(x, ld, dtype, codes, ld, scales, sl, rows, dim, None)

    assert quant(dim=0) == quant(rows=-1) == quant(dtype=2) == L.TTLH_EINVAL
    assert quant(x=None) == quant(codes=None) == quant(scales=None) == quant(scales=18) == L.TTLH_EINVAL
    assert quant(rows=1 << 31) == quant(dim=1 << 31) == L.TTLH_EUNSUPPORTED
    assert quant(rows=(1 << 31) - 1, dim=4096) == L.TTLH_EUNSUPPORTED
    assert quant(sl=5) == quant(ld=639) == L.TTLH_EINVAL
    # more threads than a launch has
    assert quant(rows=1 << 26, dim=512, ld=512) == quant(rows=1 << 22, dim=8192, ld=8192, sl=1 << 22) == L.TTLH_EUNSUPPORTED

    def norm(rows=6, dim=640, ld=640, tl=640, sl=6):
        return lib.ttlh_fp8_rms_norm(16, ld, 0, 0, 16, tl, 0, 16, 0, 1e-6, 16, ld, 16, sl, rows, dim, None)

    assert norm(tl=639) == norm(ld=639) == norm(sl=5) == L.TTLH_EINVAL
    assert norm(rows=1 << 26, sl=1 << 26) == norm(rows=1 << 23, dim=4096, ld=4096, tl=4096, sl=1 << 23) == L.TTLH_EUNSUPPORTED
    assert quant(rows=0, x=None) == L.TTLH_OK
    assert lib.ttlh_fp8_glu(16, 640, 16, 640, 0, 2, 16, 640, 16, 6, 6, 640, None) == L.TTLH_EINVAL

    def product(x=16, xl=640, w=16, wl=640, c=16, cd=0, M=6, N=300, K=640, xs=16, cl=1 << 30):
        return lib.ttlh_matmul_fp8(x, xl, xs, 6, w, wl, 16, 3, c, cd, cl, M, N, K, None)

    assert product(K=632) == product(K=0) == product(x=24) == product(xl=648) == L.TTLH_EINVAL
    assert product(wl=632) == product(cd=5) == product(c=17) == product(xs=18) == L.TTLH_EINVAL
    assert product(x=None) == product(w=None) == product(c=None) == product(xs=None) == L.TTLH_EINVAL
    assert product(M=1 << 28) == product(K=1 << 29) == L.TTLH_EUNSUPPORTED
    assert product(cl=299) == L.TTLH_EINVAL
    assert product(M=1, N=1 << 27, K=16) == product(M=1 << 27, N=1 << 27) == L.TTLH_EUNSUPPORTED  # blocks
    assert product(M=0, x=None) == product(N=0, c=None) == L.TTLH_OK


# --- weights ------------------------------------------------------------------


@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 640), (300, 130), (5, 16)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_weights(n, k, dtype):
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(n + k)) * 0.05).to(dtype)
    w[0, 0] = 3.0
    codes, scales = K.fp8_weights(w)
    blocks, groups = -(-n // 128), -(-k // 128)
    assert codes.dtype == E4M3 and codes.shape == (n, k) and codes.is_contiguous()
    assert scales.dtype == E8M0 and scales.shape == (-(-groups // 4), blocks, 4)
    s = R.by_row(scales, 4 * scales.shape[0])
    for b in range(blocks):
        for g in range(groups):
            part = w[b * 128:(b + 1) * 128, g * 128:(g + 1) * 128].double()
            assert s[b, g] == R.scale_for(float(part.abs().max()))
            assert torch.equal(codes[b * 128:(b + 1) * 128, g * 128:(g + 1) * 128].double(),
                               R.e4m3(part / s[b, g]))
    assert (s[:, groups:] == 2.0 ** -126).all()


def test_weights_of_zeros_tiny_and_large_blocks():
    w = torch.zeros(128, 512)
    w[3, 130], w[5, 260] = 2.0 ** -140, 448.0 * 2.0 ** 100
    w[6, 400] = 448.0 * (1 + 2.0 ** -23)
    codes, scales = K.fp8_weights(w)
    assert R.by_row(scales, 4).tolist() == [[2.0 ** -126, 2.0 ** -126, 2.0 ** 100, 2.0]]
    assert codes[5, 260].float() == 448.0 and codes[6, 400].float() == 224.0


@pytest.mark.parametrize("w", [torch.zeros(3), torch.zeros(3, 0), torch.zeros(3, 4, dtype=torch.int32),
                               torch.tensor([[1.0, float("nan")]]), torch.tensor([[1.0, float("inf")]])])
def test_bad_weights_are_refused(w):
    with pytest.raises(ValueError):
        K.fp8_weights(w)


# --- the header's rules ---------------------------------------------------------


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp8")
    src = d / "r.cpp"
    src.write_text('#include "ttlh_fp8.h"\n#include <string.h>\nusing namespace ttlh;\nextern "C" {\n'
                   'int code32(float a) { uint32_t u; memcpy(&u, &a, 4); return scale_code(u); }\n'
                   'int open32(float a) { uint32_t u; memcpy(&u, &a, 4); return scale_open(u); }\n'
                   'int code64(double a) { uint64_t u; memcpy(&u, &a, 8); return scale_code64(u); }\n'
                   'float inverse(int c) { uint32_t u = inverse_scale_bits(c); float f; memcpy(&f, &u, 4); return f; }\n}\n')
    so = d / "r.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tt-lang_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for n, a in (("code32", ctypes.c_float), ("open32", ctypes.c_float), ("code64", ctypes.c_double)):
        getattr(lib, n).argtypes = [a]
    lib.inverse.restype = ctypes.c_float
    return lib


def _edges():
    for n in (-149, -140, -127, -126, -125, -30, 0, 1, 60, 127):
        for m in (1.0, 1.25, 1.75 * (1 - 2.0 ** -24), 1.75, 1.75 * (1 + 2.0 ** -23), 1.999):
            yield m * 2.0 ** n
    yield 0.0


def test_scales_of_the_header(rules):
    for a in _edges():
        f = ctypes.c_float(a).value
        s = R.scale_for(f)
        assert 2.0 ** (rules.code32(f) - 127) == s, f
        assert 2.0 ** (rules.code64(f) - 127) == s, f
        assert rules.inverse(rules.code32(f)) == 1 / s
    assert rules.code32(float("inf")) == rules.code32(float("nan")) == 255
    # fp64 tells what fp32 cannot
    assert rules.code64(448.0 * (1 + 2.0 ** -50)) == 128 and rules.code64(448.0) == 127


def test_open_scales_are_those_near_a_border(rules):
    for n in (-100, 0, 100):
        b = 1.75 * 2.0 ** n
        ulp = 2.0 ** (n - 23)
        for d in range(-40, 41):
            assert rules.open32(b + d * ulp) == (abs(d) <= 32), (n, d)
