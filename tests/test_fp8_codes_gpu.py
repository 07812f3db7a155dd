"""Codes and scales of norms and gated activations on the MI355X are, each of them, those of the values
computed in 64 bits (oracle/fp8.py): equality, at the sizes and over the ranges of tests/test_fp8_gpu.py.

The kernels compute in fp32 and decide in fp64 what lies within 2^-20 of a border.  Their fp32 values are off by
less: a norm's by 5 x 2^-24 (sum, root, two products and what the second look multiplies by), silu's by 4.1 x 2^-24
and gelu's by 7.6 x 2^-24 (the largest of all fp32 gates whose integral is 2^-126 and more, measured), and
2^-24 for the product."""

import pytest
import torch

from oracle import fp8 as R
from test_fp8_gpu import SHAPES, _check_exact, _gen, _out, _untouched, _values
from ttlhip import kernels as K

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (BF16, F32), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_norms(rows, dim, dtype, wdtype):
    g = _gen(rows + dim + 21)
    x, r = _values(rows, dim, g, dtype), _values(rows, dim, g, dtype)
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(wdtype)
    for residual in (None, r):
        wide, codes, s, scales = _out(rows, dim)
        K.rms_norm_fp8(x.cuda(), w.cuda(), codes, scales, eps=2.0 ** -10,
                       residual=None if residual is None else r.cuda())
        _check_exact(R.rms_norm(x, w, 2.0 ** -10, residual)[1], codes.cpu(), scales.cpu())
        _untouched(wide, s, dim)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_gates(rows, dim, dtype, act):
    g = _gen(rows + dim + 22)
    gate, up = (2 * torch.randn(rows, dim, generator=g)).to(dtype), _values(rows, dim, g, dtype)
    wide, codes, s, scales = _out(rows, dim)
    K.glu_fp8(gate.cuda(), up.cuda(), codes, scales, act=act)
    _check_exact(R.glu(gate, up, act), codes.cpu(), scales.cpu())
    _untouched(wide, s, dim)


@pytest.mark.parametrize("act,lo", [("silu", -85.0), ("gelu", -12.8)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gates_over_their_range(act, lo, dtype):
    """Rows of one gate each, from where its factor is next to fp32's smallest, with values so large that
    the products are not."""
    gate = torch.cat((torch.linspace(lo, 30, 2000), torch.tensor([0.0, -0.0, 2.0 ** -100, 1000.0, 3e4])))
    gate = gate[:, None].expand(-1, 512).contiguous().to(dtype)
    up = (torch.randn(gate.shape, generator=_gen(23)) * 2.0 ** 40).to(dtype)
    _, codes, _, scales = _out(*gate.shape)
    K.glu_fp8(gate.cuda(), up.cuda(), codes, scales, act=act)
    _check_exact(R.glu(gate, up, act), codes.cpu(), scales.cpu())
