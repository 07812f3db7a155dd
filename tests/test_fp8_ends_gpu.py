"""Scales of rows of 8-bit codes past the row's end, on the MI355X: 2^-126 whatever the row holds."""

import math

import pytest
import torch

from test_fp8_gpu import _gen, _values
from ttlhip import kernels as K

pytestmark = pytest.mark.gpu

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [1, 100, 128, 300, 640, 2890, 4099, 9000, 20000])
def test_scales_past_a_row_s_end_are_those_of_zeros(dim, dtype):
    x = _values(6, dim, _gen(dim), dtype, 0.5)
    r = torch.zeros_like(x)
    x[0, dim // 2] = math.nan
    x[1, 0], r[1, 0] = math.inf, -math.inf
    x[2, -1] = -math.inf
    groups = -(-dim // 128)
    codes, scales = torch.empty(6, dim, dtype=E4M3, device="cuda"), K.fp8_scales(6, dim)
    ways = {
        "norm": lambda: K.rms_norm_fp8(x.cuda(), torch.ones(dim, device="cuda"), codes, scales),
        "norm of a sum": lambda: K.rms_norm_fp8(x.cuda(), torch.ones(dim, device="cuda"), codes, scales,
                                                residual=r.cuda()),
        "quant": lambda: K.quant_fp8(x.cuda(), codes, scales),
        "glu": lambda: K.glu_fp8(x.cuda(), x.cuda(), codes, scales, act="gelu"),
    }
    for name, way in ways.items():
        scales.view(torch.uint8).fill_(0x5A)
        way()
        s = scales.cpu().view(torch.uint8).transpose(0, 1).reshape(6, -1)
        assert (s[:, groups:] == 1).all(), name
        if "norm" in name:
            assert (s[0, :groups] == 255).all(), name
            assert (codes.cpu().float()[0] == 0).all(), name
        assert s[2, groups - 1] == 255, name
        assert not (s[3:] == 255).any(), name
