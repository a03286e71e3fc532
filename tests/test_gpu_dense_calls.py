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
