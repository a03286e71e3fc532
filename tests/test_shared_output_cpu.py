"""What the combine adds to the routed sum: rows that its kernel would misread, or read past
their end, are refused in Python before anything reaches the device (so CPU tensors do)."""

import pytest
import torch

import megamoe

BF = torch.bfloat16
T, K, H, ROWS = 4, 2, 64, 16


def triple():
    return torch.zeros((ROWS, H), dtype=BF), torch.ones((T, K)), torch.zeros((T, K), dtype=torch.int32)


BAD = [
    torch.zeros((T, H), dtype=torch.float16),
    torch.zeros((T, H)),
    torch.zeros((T, 2 * H), dtype=BF)[:, :H],     # a strided out=
    torch.zeros((H, T), dtype=BF).t(),
    torch.zeros((T - 1, H), dtype=BF),            # would be read past its end
    torch.zeros((T, H - 8), dtype=BF),
    torch.zeros((T * H,), dtype=BF),
    torch.zeros((T, H), dtype=BF, device="meta"),
]


@pytest.mark.parametrize("bad", BAD)
def test_finalize_refuses_rows_it_would_misread(bad):
    with pytest.raises(ValueError, match="shared_output"):
        megamoe.finalize(*triple(), shared_output=bad)
    with pytest.raises(ValueError, match="shared_output"):
        megamoe.finalize(*triple(), shared_output=bad, partial=True)


@pytest.mark.parametrize("bad", BAD)
def test_layer_finalize_refuses_rows_it_would_misread(bad):
    layer = object.__new__(megamoe.RoutedMoE)
    with pytest.raises(ValueError, match="shared_output"):
        layer.finalize(*triple(), shared_output=bad)


@pytest.mark.parametrize("bad", BAD)
def test_peer_finalize_refuses_rows_it_would_misread(bad):
    comm = object.__new__(megamoe.PeerAllReduce)
    comm.handle, comm.hidden = 1, H  # never used: the check comes first
    rows, weights, permuted = triple()
    try:
        with pytest.raises(ValueError, match="shared_output"):
            comm.finalize(rows, weights, permuted, bad)
        with pytest.raises(ValueError, match="shared_output"):
            comm.moe_finalize_all_reduce_rms_norm(routed_output=rows, expert_weights=weights, permuted_indices=permuted,
                                                  gated_shared_output=bad, residual=rows[:T], gamma=None)
    finally:
        comm.handle = None
