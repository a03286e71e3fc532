"""Calls of the dense 8-bit operators and of the combine beside them that the documentation
allows, at the edges of what is allowed."""

import pytest
import torch

import megamoe

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_finalize_takes_a_longer_buffer_of_shared_rows():
    g = torch.Generator().manual_seed(3)
    rows, shared = (torch.randn((n, 256), generator=g).to(BF).cuda() for n in (24, 9))
    weights = torch.rand((5, 4), generator=g).cuda()
    permuted = torch.randint(-1, 24, (5, 4), generator=g).int().cuda()
    got = megamoe.finalize(rows, weights, permuted, shared)
    assert torch.equal(got, megamoe.finalize(rows, weights, permuted, shared[:5].clone()))
    assert not torch.equal(got, megamoe.finalize(rows, weights, permuted))


@pytest.mark.parametrize("width", [100, 1, 250, 1990])
def test_empty_batches_of_any_width(width):
    """No tokens: nothing is launched and nothing refused, whatever the depth."""
    x = torch.empty((0, width), dtype=BF, device="cuda")
    gamma = torch.ones(width, dtype=BF, device="cuda")
    none = torch.empty(0, device="cuda")
    held = torch.zeros((2 * width, (width + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    w, w13 = held[:width, :width], held[:, :width]
    s, s13 = torch.ones(width, device="cuda"), torch.ones(2 * width, device="cuda")
    quantized = megamoe.quantize_int8(x)
    normed = megamoe.rms_norm(x, gamma, quant="int8")
    plain = torch.empty((0, width), dtype=torch.int8, device="cuda")
    for codes, scales in (quantized, (normed.codes, normed.scales), (plain, none)):
        assert megamoe.int8_linear(codes, scales, w, s).shape == (0, width)
        assert megamoe.int8_ffn(codes, scales, w13, s13, w, s).shape == (0, width)
