"""Weights into 8-bit codes: the same codes come of any device."""

import pytest
import torch

from ttlhip import kernels as K


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_on_the_device_are_those_on_the_host(dtype):
    """Blocks of all sizes: every exponent that a scale has, and many values in the middle between two codes."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(260, 128 * 250, generator=g) * torch.exp2(torch.arange(-129, 121).float()).repeat_interleave(128)
    w = w.to(dtype)
    w[:, ::7] = 1.0625 * w[:, ::7].sign() * torch.exp2(torch.floor(torch.log2(w[:, ::7].abs().double()))).to(dtype)
    (a, b), (c, d) = K.fp8_weights(w), K.fp8_weights(w.cuda())
    for x, y in ((a, c), (b, d)):
        assert torch.equal(x.view(torch.uint8), y.cpu().view(torch.uint8))
