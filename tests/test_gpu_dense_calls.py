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


def test_rows_beside_each_other_in_one_buffer():
    """Columns of one buffer interleave in memory and share none of it."""
    g = torch.Generator().manual_seed(4)
    hidden, gamma = 512, torch.ones(512, dtype=BF, device="cuda")
    for tokens in (1, 2, 9):
        room = torch.randn((tokens, 4 * hidden), generator=g).to(BF).cuda()
        x, res, out, other = room.split(hidden, 1)
        want = megamoe.rms_norm(x.clone(), gamma, residual=res.clone(), quant="int8", with_norm=True)
        kept = x.clone(), other.clone()
        got = megamoe.rms_norm(x, gamma, residual=res, quant="int8", with_norm=True, out=out, residual_out=res)
        for u, v in zip(got, want):
            assert torch.equal(u, v)
        assert torch.equal(x, kept[0]) and torch.equal(other, kept[1])


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_product_rows_beside_their_codes(tokens):
    g = torch.Generator().manual_seed(tokens)
    room = torch.zeros((tokens, 2048), dtype=torch.uint8, device="cuda")
    x, out = room.view(torch.int8)[:, :512], room.view(BF)[:, 256:512]
    x.copy_(torch.randint(-127, 128, (tokens, 512), generator=g))
    w13 = torch.randint(-127, 128, (512, 512), dtype=torch.int8, generator=g).cuda()
    w2 = torch.randint(-127, 128, (256, 256), dtype=torch.int8, generator=g).cuda()
    xs, s13, s2 = (torch.rand(n, generator=g).cuda() * 1e-2 for n in (tokens, 512, 256))
    codes = x.clone()
    assert torch.equal(megamoe.int8_linear(x, xs, w13[:256], s13[:256], out=out), megamoe.int8_linear(codes, xs, w13[:256], s13[:256]))
    # of the block: w2 [512, 256] gives 512 values a token
    wide = room.view(BF)[:, 512:1024]
    w2 = torch.randint(-127, 128, (512, 256), dtype=torch.int8, generator=g).cuda()
    s2 = torch.rand(512, generator=g).cuda() * 1e-2
    assert torch.equal(megamoe.int8_ffn(x, xs, w13, s13, w2, s2, out=wide), megamoe.int8_ffn(codes, xs, w13, s13, w2, s2))
    assert torch.equal(x, codes)


@pytest.mark.parametrize("first", [1, 511, 768])
def test_columns_that_meet_are_refused(first):
    room = torch.zeros(6 * 1024, dtype=BF, device="cuda")
    x, out = (room[at:].as_strided((4, 512), (1024, 1)) for at in (0, first))
    with pytest.raises(ValueError, match="overlaps"):
        megamoe.rms_norm(x, torch.ones(512, dtype=BF, device="cuda"), out=out)


def test_an_error_in_an_argument_reaches_the_caller():
    class Undecided:
        def __bool__(self):
            raise KeyError("undecided")

    x, gamma = torch.ones((2, 64), dtype=BF, device="cuda"), torch.ones(64, dtype=BF, device="cuda")
    with pytest.raises(KeyError, match="undecided"):
        megamoe.rms_norm(x, gamma, quant="int8", with_norm=Undecided())
