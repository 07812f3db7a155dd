"""Weights into 8-bit codes: 64-bit weights are rounded once, and the same codes come of any device."""

import pytest
import torch

from oracle import fp8 as R
from ttlhip import kernels as K

F64, E4M3 = torch.float64, torch.float8_e4m3fn


def _check(w):
    codes, scales = K.fp8_weights(w)
    s = R.by_row(scales, 4 * scales.shape[0])
    for b in range(-(-w.shape[0] // 128)):
        for g in range(-(-w.shape[1] // 128)):
            at = (slice(b * 128, (b + 1) * 128), slice(g * 128, (g + 1) * 128))
            assert s[b, g] == R.scale_for(float(w[at].abs().max())), (b, g)
            assert torch.equal(codes[at].double(), R.e4m3(w[at] / s[b, g])), (b, g)


def test_weights_of_64_bits_next_to_a_border_of_the_scales():
    w = torch.zeros(1, 384, dtype=F64)
    w[0, 0] = 448 * (1 + 2.0 ** -40)  # fp32 takes it for 448
    w[0, 128] = -448 * (1 - 2.0 ** -40)
    w[0, 256] = 448
    _check(w)
    assert R.by_row(K.fp8_weights(w)[1], 3).tolist() == [[2.0, 1.0, 1.0]]


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -30, 2.0 ** -130])
def test_weights_of_64_bits_next_to_the_middle_between_two_codes(scale):
    """Every middle, and values on either side of it that fp32 takes for it."""
    c = torch.arange(0, 0x7F, dtype=torch.uint8).view(E4M3).double()
    mid = (c[1:] + c[:-1]) / 2
    v = torch.cat([mid * (1 + d) for d in (0.0, 2.0 ** -40, -2.0 ** -40, 2.0 ** -30, -2.0 ** -30)])
    v = torch.cat((v, -v))
    w = torch.zeros(10, 128, dtype=F64)
    w[:, :127] = v[:1260].view(10, 126).repeat(1, 2)[:, :127]
    w[:, 127] = 448
    _check(w * scale)


def test_random_weights_of_64_bits():
    g = torch.Generator().manual_seed(0)
    _check(torch.randn(300, 400, generator=g, dtype=F64) * torch.exp(3 * torch.randn(300, 400, generator=g, dtype=F64)))


def test_weights_of_64_bits_that_fp32_does_not_hold_are_refused():
    with pytest.raises(ValueError, match="finite"):
        K.fp8_weights(torch.full((2, 2), 1e39, dtype=F64))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, F64])
def test_no_outputs(dtype):
    codes, scales = K.fp8_weights(torch.empty(0, 640, dtype=dtype))
    assert codes.shape == (0, 640) and codes.dtype == E4M3
    assert scales.shape == (2, 0, 4) and scales.dtype == K.fp8_scales(0, 640, "cpu").dtype


@pytest.mark.gpu
def test_a_product_with_no_outputs():
    c = torch.empty(3, 640, dtype=E4M3, device="cuda")
    K.matmul_fp8(c, K.fp8_scales(3, 640), *K.fp8_weights(torch.empty(0, 640, device="cuda")),
                 torch.empty(3, 0, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, F64])
def test_weights_on_the_device_are_those_on_the_host(dtype):
    """Blocks of all sizes: every exponent that a scale has, and many values in the middle between two codes."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(260, 128 * 250, generator=g) * torch.exp2(torch.arange(-129, 121).float()).repeat_interleave(128)
    w = w.to(dtype)
    w[:, ::7] = 1.0625 * w[:, ::7].sign() * torch.exp2(torch.floor(torch.log2(w[:, ::7].abs().double()))).to(dtype)
    (a, b), (c, d) = K.fp8_weights(w), K.fp8_weights(w.cuda())
    for x, y in ((a, c), (b, d)):
        assert torch.equal(x.view(torch.uint8), y.cpu().view(torch.uint8))
