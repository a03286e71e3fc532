"""The dense 8-bit operators at sizes on either side of the choices between their kernels' forms:
how many chunks of a row a thread holds, and how a cluster's CTAs add the parts of a product."""

import pytest
import torch

import megamoe
from test_gpu_dense import BF, D, F32, FH, check_norm, gen, randn, weights

pytestmark = pytest.mark.gpu


# rows that fit in the SMs at once with one, two or four chunks a thread; more rows; rows whose
# starts share no alignment; rows of more chunks than the denser form's threads hold
@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("quant", [None, "mxfp8", "int8"])
@pytest.mark.parametrize("tokens,hidden,residual", [
    (148, 7168, False), (149, 7168, True), (296, 7168, False), (297, 7168, True), (741, 7168, False), (600, 2048, True), (889, 2048, False),
    (160, 16384, True), (700, 9216, False), (700, 9224, False), (1037, 5120, True), (520, 6147, True), (1021, 6147, False),
])
def test_norm_forms(tokens, hidden, residual, quant, dtype):
    if quant == "mxfp8":
        hidden = hidden // 32 * 32
    g = gen(tokens, hidden, residual, 3)
    x = randn((tokens, hidden), g, dtype) * 3
    res = randn((tokens, hidden), g, dtype) if residual else None
    gamma = (1 + 0.2 * randn((hidden,), g)).to(dtype)
    check_norm(megamoe.rms_norm(x, gamma, 1e-6, residual=res, quant=quant, with_norm=True), x, gamma, 1e-6, res, quant, True)


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("tokens,hidden", [(149, 7168), (700, 7168), (1500, 5120), (300, 1990), (592, 6147), (160, 40000)])
def test_quantize_forms(tokens, hidden, dtype):
    # a code is within half a step of x / s, and the largest value of a row has code 127: s is exact
    # to one rounding (2^-24), the quotient to two
    g = gen(tokens, hidden, 5)
    x = randn((tokens, hidden), g, dtype)
    codes, s = megamoe.quantize_int8(x)
    top = x.to(D).abs().amax(-1)
    assert bool(((s.to(D) * 127 - top).abs() <= top * 2.0 ** -23).all())
    assert bool(((codes.to(D) - x.to(D) / s.to(D)[:, None]).abs() <= 0.5 + 127 * 2.0 ** -22).all())
    assert bool((codes.abs().amax(-1) == 127).all())


# one to 128 tokens of the last token tile; two and eight CTAs a cluster, and one
@pytest.mark.parametrize("tokens", [2, 15, 31, 32, 34, 47, 63, 66, 81, 96, 97, 112, 127])
@pytest.mark.parametrize("features,depth", [(70, 4096), (1500, 1100), (130, 256), (20000, 300)])
def test_linear_parts(tokens, features, depth):
    g = gen(tokens, features, depth, 7)
    x, xs = weights(tokens, depth, g)
    w, ws = weights(features, depth, g)
    exact = x.to(D) @ w.to(D).T
    one_x, one_w = torch.ones_like(xs), torch.ones_like(ws)
    # the sums are exact and below 2^24 here, so fp32 outputs with scales of one are exact too
    assert float(exact.abs().max()) < 2 ** 24
    assert torch.equal(megamoe.int8_linear(x, one_x, w, one_w, out_dtype=F32).to(D), exact)
    megamoe.int8_check()


@pytest.mark.parametrize("tokens", [17, 33, 50, 64, 65, 90, 128])
def test_ffn_parts(tokens):
    # a batch's rows have the bits of its rows one at a time
    g = gen(tokens, 11)
    hidden, inter = 1100, 700
    x, xs = weights(tokens, hidden, g)
    xs = xs * hidden ** 0.5 * 2
    w13, s13 = weights(2 * inter, hidden, g)
    w2, s2 = weights(hidden, inter, g)
    got = megamoe.int8_ffn(x, xs, w13, s13, w2, s2, clamp=2.0)
    for t in (0, tokens // 2, tokens - 1):
        assert torch.equal(got[t:t + 1], megamoe.int8_ffn(x[t:t + 1], xs[t:t + 1], w13, s13, w2, s2, clamp=2.0))
