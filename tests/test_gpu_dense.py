"""The dense 8-bit operators on the GPU against their definitions in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, fp32's half step; e = eps / 2, the output type's):
  norm    the sum of squares adds at most 64 + 10 + 5 terms in a chain, so it is within 2^-17
          of its value, its root within 2^-18, and four more roundings: y within 2^-17.
  mxfp8   E4M3 is off by at most 2^-4 of the value, or half its smallest step 2^-10 (in units
          of the block's scale).
  int8    half a step, plus what y itself is off by.
  linear  the integer sum is exact; its conversion, two products and the bias: 3u of the
          product, u + e of the result.
  ffn     gate and up within 4u; silu's exponential within 4u of its value, and |gate| < 30
          here multiplies gate's own error: h within 2^-17. A code can then differ by one step
          where h / s is within 2 * 127 * 2^-17 of a tie; each such code moves the output by at
          most s * |w2| * w2_scale.
"""

import math
import os
import subprocess
import sys

import pytest
import torch

import megamoe

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
D = torch.float64


def gen(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(sum((i + 1) * 7919 * int(k) for i, k in enumerate(key)) % (1 << 31))
    return g


def randn(shape, g, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def int8_rows(q):
    n, k = q.shape
    held = torch.full((n, (k + 15) // 16 * 16), 77, dtype=torch.int8, device=q.device)  # pads are never read
    held[:, :k] = q
    return held[:, :k]


def weights(n, k, g):
    q = (torch.randn((n, k), generator=g, device="cuda") * 40).round().clamp(-128, 127).to(torch.int8)
    return int8_rows(q), torch.rand((n,), generator=g, device="cuda") * (0.5 / (40 * math.sqrt(k))) + 0.5 / (40 * math.sqrt(k))


def norm_exact(x, gamma, eps, residual):
    y = x.to(D)
    if residual is not None:
        y = (x.float() + residual.float()).to(x.dtype).to(D)
    r = y
    return r, y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * gamma.to(D)


def check_norm(got, x, gamma, eps, residual, quant, with_norm):
    r, y = norm_exact(x, gamma, eps, residual)
    if residual is None:
        assert got.residual is None
    else:
        assert got.residual.dtype == x.dtype and torch.equal(got.residual.to(D), r)
    if with_norm:
        tol = (torch.finfo(x.dtype).eps / 2 + 2.0 ** -17) * y.abs() + torch.finfo(x.dtype).smallest_normal
        assert got.norm.dtype == x.dtype and bool(((got.norm.to(D) - y).abs() <= tol).all())
    else:
        assert got.norm is None
    if quant == "mxfp8":
        b = y.view(y.size(0), -1, 32)
        amax = b.abs().amax(-1)
        s = got.scales.to(F32).to(D)
        assert bool((torch.frexp(s)[0] == 0.5).all())  # powers of two
        assert bool((amax <= s * 448 * (1 + 2.0 ** -16)).all())           # nothing saturates
        tight = (amax * (1 + 2.0 ** -16) >= s * 224) | (amax == 0)        # the least power of two that holds it
        assert bool(tight.all()) and bool((s[amax == 0] == 1).all())
        v = got.codes.to(F32).to(D).view_as(b) * s[..., None]
        assert bool(((v - b).abs() <= b.abs() * (2.0 ** -4 + 2.0 ** -17) + s[..., None] * 2.0 ** -10).all())
    elif quant == "int8":
        amax = y.abs().amax(-1)
        s = got.scales.to(D)
        assert bool(((s * 127 - amax).abs() <= amax * 2.0 ** -17 + 127 * 2.0 ** -149).all())
        v = got.codes.to(D) * s[:, None]
        assert bool(((v - y).abs() <= 0.5 * s[:, None] + y.abs() * 2.0 ** -16 + 2.0 ** -149).all())
        assert bool((got.codes.abs().amax(-1)[amax > 1e-30] == 127).all())
    else:
        assert got.codes is None and got.scales is None


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("quant", [None, "mxfp8", "int8"])
@pytest.mark.parametrize("tokens,hidden,residual", [
    (1, 7168, True), (1, 32, False), (3, 1024, True), (48, 5120, False), (297, 6144, True), (300, 96, True),
    (2, 16384, True), (300, 16384, False), (2, 40000, True), (300, 40032, False), (2501, 512, True), (4801, 1024, True),
])
def test_norm(tokens, hidden, residual, quant, dtype):
    if quant == "mxfp8":
        hidden = hidden // 32 * 32
    g = gen(tokens, hidden, residual)
    x = randn((tokens, hidden), g, dtype) * 3
    res = randn((tokens, hidden), g, dtype) if residual else None
    gamma = (1 + 0.2 * randn((hidden,), g)).to(dtype)
    for with_norm in ((True,) if quant is None else (True, False)):
        got = megamoe.rms_norm(x, gamma, 1e-5, residual=res, quant=quant, with_norm=with_norm)
        check_norm(got, x, gamma, 1e-5, res, quant, with_norm)


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("quant", [None, "int8"])
@pytest.mark.parametrize("tokens,hidden", [(1, 1), (2, 7), (5, 33), (3, 1001), (299, 4099), (2, 16383), (1, 50001), (2499, 505), (4803, 1017)])
def test_norm_odd_rows(tokens, hidden, quant, dtype):
    g = gen(tokens, hidden, 5)
    x, res = randn((tokens, hidden), g, dtype), randn((tokens, hidden), g, dtype)
    gamma = (1 + 0.2 * randn((hidden,), g)).to(dtype)
    check_norm(megamoe.rms_norm(x, gamma, 1e-6, residual=res, quant=quant, with_norm=True), x, gamma, 1e-6, res, quant, True)


@pytest.mark.parametrize("quant", [None, "mxfp8", "int8"])
@pytest.mark.parametrize("dtype,offset,pitch", [(BF, 1, 1031), (BF, 8, 1040), (FH, 3, 1024 + 3), (F32, 2, 1030), (BF, 0, 2048)])
def test_norm_strided_views(dtype, offset, pitch, quant):
    g = gen(offset, pitch)
    room = randn((9, pitch + 16), g, dtype)
    x = room.flatten()[offset:offset + 8 * pitch + 1024].as_strided((9, 1024), (pitch, 1))
    res = randn((9, 1024 + 8), g, dtype)[:, 8:]
    gamma = (1 + 0.2 * randn((1024 + 1,), g)).to(dtype)[1:]
    out = torch.full((9, 1100), 5.0, dtype=dtype, device="cuda")
    got = megamoe.rms_norm(x, gamma, 1e-6, residual=res, quant=quant, with_norm=True, out=out[:, 3:1027])
    check_norm(got, x, gamma, 1e-6, res, quant, True)
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 1027:] == 5).all())  # nothing beside the rows


@pytest.mark.parametrize("dtype", [BF, FH])
def test_norm_fp32_gamma(dtype):
    g = gen(3)
    x, gamma = randn((5, 2048), g, dtype), 1 + 0.2 * randn((2048,), g)
    check_norm(megamoe.rms_norm(x, gamma, 1e-6, quant="mxfp8", with_norm=True), x, gamma, 1e-6, None, "mxfp8", True)


@pytest.mark.parametrize("hidden,tokens", [(4096, 3), (4096, 300), (40000, 2), (1001, 4)])
@pytest.mark.parametrize("quant", [None, "int8"])
def test_norm_residual_in_place(hidden, tokens, quant):
    g = gen(hidden, 9)
    x, res = randn((tokens, hidden), g, BF), randn((tokens, hidden), g, BF)
    gamma = (1 + 0.2 * randn((hidden,), g)).to(BF)
    want = megamoe.rms_norm(x, gamma, residual=res, quant=quant, with_norm=True)
    for place in ("residual", "x"):
        a, b = x.clone(), res.clone()
        got = megamoe.rms_norm(a, gamma, residual=b, quant=quant, with_norm=True, residual_out=b if place == "residual" else a)
        assert got.residual.data_ptr() == (b if place == "residual" else a).data_ptr()
        for u, v in zip(got, want):
            assert (u is None and v is None) or torch.equal(u.view(torch.uint8) if u.element_size() == 1 else u,
                                                            v.view(torch.uint8) if v.element_size() == 1 else v)


def test_norm_values_that_are_not_finite():
    x = torch.ones((4, 256), dtype=BF, device="cuda")
    x[0] = 0.0
    x[1, 40] = float("nan")
    x[2, 50] = float("inf")
    gamma = torch.ones((256,), dtype=BF, device="cuda")
    got = megamoe.rms_norm(x, gamma, 1e-6, quant="int8", with_norm=True)
    assert got.scales[0] == 0 and not got.codes[0].any() and not got.norm[0].any()
    assert got.scales[1:3].isnan().all() and not got.codes[1:3].any()
    assert got.norm[1].isnan().all()
    assert (got.codes[3] == 127).all() and got.norm[3].isfinite().all()
    mx = megamoe.rms_norm(x, gamma, 1e-6, quant="mxfp8")
    s = mx.scales.view(torch.uint8)
    assert (s[0] == 127).all() and not mx.codes[0].view(torch.uint8).any()
    assert (s[1] == 255).all()                                    # inv is NaN: every block
    assert (s[2] == torch.tensor([127, 255] + [127] * 6, device="cuda", dtype=torch.uint8)).all()  # 1 / inf = 0, 0 * inf


def test_norm_zero_row_and_zero_eps():
    x = torch.zeros((2, 64), dtype=F32, device="cuda")
    x[1] = 2.0
    got = megamoe.rms_norm(x, torch.ones(64, device="cuda"), 1e-6).norm
    assert not got[0].any()
    assert torch.allclose(got[1], torch.ones_like(got[1]), rtol=1e-6)


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("tokens,hidden", [(1, 1), (1, 7168), (8, 7168), (3, 1001), (300, 2048), (301, 999), (2, 18432), (5, 70001), (5001, 1024), (2999, 77)])
def test_quantize_bit_exact(tokens, hidden, dtype):
    g = gen(tokens, hidden, 3)
    x = (randn((tokens, hidden), g) * torch.exp(4 * randn((tokens, 1), g))).to(dtype)
    codes, scales = megamoe.quantize_int8(x)
    v = x.float().cpu()
    top = v.abs().amax(-1)
    fine = top.isfinite()  # a few fp16 rows overflow: scale NaN, codes 0
    s = torch.where(fine, top / 127, torch.full_like(top, float("nan")))
    assert torch.allclose(scales.cpu(), s, rtol=0.0, atol=0.0, equal_nan=True)
    want = torch.where(fine[:, None], torch.round(v / s[:, None]), torch.zeros_like(v))
    assert torch.equal(codes.cpu(), want.to(torch.int8))
    assert codes.data_ptr() % 16 == 0 and (codes.size(0) == 1 or codes.stride(0) % 16 == 0)


def test_quantize_extremes():
    big = torch.finfo(F32).max
    x = torch.zeros((7, 64), device="cuda")
    x[1, :3] = torch.tensor([big, -big, big / 254], device="cuda")
    x[2, :3] = torch.tensor([2.0 ** -149, -(2.0 ** -149), 0.0], device="cuda")  # amax / 127 rounds to zero
    x[3, :2] = torch.tensor([190 * 2.0 ** -149, 2.0 ** -149], device="cuda")    # a scale of one subnormal step
    x[4, :2] = torch.tensor([2.0 ** -126, 2.0 ** -130], device="cuda")
    x[5, 3] = float("-inf")
    x[6, 3] = float("nan")
    codes, s = megamoe.quantize_int8(x)
    codes = codes.cpu()
    assert s[0] == 0 and not codes[0].any()
    assert codes[1, :3].tolist() in ([127, -127, 0], [127, -127, 1])  # the third sits at a tie of rounded numbers
    assert s[2] == 0 and not codes[2].any()
    assert codes[3, 0] == 127 and codes[3, 1] == 1
    assert codes[4, 0] == 127 and codes[4, 1] == 8
    assert s[5:].isnan().all() and not codes[5:].any()


LINEAR = [(1, 128, 128), (1, 4096, 7168), (1, 1, 1), (2, 7, 16), (5, 129, 130), (16, 300, 1000), (17, 256, 2048), (33, 1000, 512),
          (64, 2311, 5104), (65, 100, 640), (128, 512, 1024), (129, 640, 384), (255, 130, 4096), (256, 384, 256),
          (257, 384, 256), (300, 1000, 777), (512, 512, 512), (1000, 1100, 1300), (2049, 513, 129), (4096, 2048, 1024),
          # few features of great depth: the stream form by tiles of 128 tokens
          (200, 70, 12000), (513, 64, 20000), (1000, 300, 8000), (131, 1, 131071)]


@pytest.mark.parametrize("tokens,features,depth", LINEAR)
@pytest.mark.parametrize("dtype", [BF, FH, F32])
def test_linear(tokens, features, depth, dtype):
    g = gen(tokens, features, depth)
    x, xs = weights(tokens, depth, g)
    w, ws = weights(features, depth, g)
    bias = randn((features,), g) if (tokens + features) % 2 else None
    got = megamoe.int8_linear(x, xs, w, ws, bias, out_dtype=dtype)
    prod = (x.to(D) @ w.to(D).T) * xs.to(D)[:, None] * ws.to(D)
    want = prod if bias is None else prod + bias.to(D)
    e = torch.finfo(dtype).eps / 2
    tol = 3 * 2.0 ** -24 * prod.abs() + (e + 2.0 ** -24) * want.abs() + torch.finfo(dtype).smallest_normal * e
    assert got.dtype == dtype and got.shape == (tokens, features)
    assert bool(((got.to(D) - want).abs() <= tol).all())
    assert torch.equal(got, megamoe.int8_linear(x, xs, w, ws, bias, out_dtype=dtype))
    megamoe.int8_check()


def test_linear_extreme_sums():
    # the largest sum the depth limit allows: 131056 products of 128 * 128 is 2^31 - 2^18
    for tokens in (1, 300):
        k = 131056
        x = torch.full((tokens, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((130, k), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(tokens, device="cuda")
        got = megamoe.int8_linear(x, one, w, torch.ones(130, device="cuda"), out_dtype=F32)
        assert bool((got == float(k * 16384)).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens", [3, 40, 700])
def test_linear_strided_operands_and_output(tokens, dtype):
    g = gen(tokens, 17)
    n, k = 333, 700
    held_x = (torch.randn((tokens, 1024), generator=g, device="cuda") * 40).to(torch.int8)
    held_w = (torch.randn((n, 720), generator=g, device="cuda") * 40).to(torch.int8)
    x, w = held_x[:, 32:32 + k], held_w[:, 16:16 + k]
    xs, ws = torch.rand(tokens, 1, device="cuda", generator=g), torch.rand(n, 1, device="cuda", generator=g)
    for first, pitch in ((0, n + 3), (5, 400), (8, 352)):
        held = torch.full((tokens, pitch), 9.0, dtype=dtype, device="cuda")
        if first + n > pitch:
            held = torch.full((tokens, first + n + 2), 9.0, dtype=dtype, device="cuda")
        out = held[:, first:first + n]
        assert megamoe.int8_linear(x, xs, w, ws, out_dtype=dtype, out=out) is out
        want = megamoe.int8_linear(int8_rows(x), xs.flatten(), int8_rows(w), ws.flatten(), out_dtype=dtype)
        assert torch.equal(out, want)
        assert bool((held[:, :first] == 9).all()) and bool((held[:, first + n:] == 9).all())
    exact = (x.to(D) @ w.to(D).T) * xs.to(D) * ws.to(D).T
    assert float((want.to(D) - exact).abs().max() / exact.abs().max()) < torch.finfo(dtype).eps


def test_linear_large_offsets():
    # outputs past 2^31 elements and 2^32 bytes: rows at the far end
    tokens, n, k = 140000, 16000, 128
    g = gen(6)
    x, xs = weights(tokens, k, g)
    w, ws = weights(n, k, g)
    got = megamoe.int8_linear(x, xs, w, ws)
    for rows in (slice(0, 3), slice(tokens - 3, tokens), slice(134217, 134220)):
        want = (x[rows].to(D) @ w.to(D).T) * xs[rows].to(D)[:, None] * ws.to(D)
        assert bool(((got[rows].to(D) - want).abs() <= 2.0 ** -7.9 * want.abs()).all())


def ffn_reference(x, xs, w13, s13, w2, s2, clamp):
    inter = w13.size(0) // 2
    both = (x.to(D) @ w13.to(D).T) * xs.to(D)[:, None] * s13.to(D)
    gate, up = both[:, :inter], both[:, inter:]
    assert float(gate.abs().max()) < 30
    if clamp:
        gate, up = gate.clamp(max=clamp), up.clamp(-clamp, clamp)
    h = gate / (1 + torch.exp(-gate)) * up
    s = h.abs().amax(-1) / 127
    t = h / s[:, None]
    codes = t.round()
    near = ((t - t.floor() - 0.5).abs() <= 2 * 127 * 2.0 ** -17).to(D)
    scale = s[:, None] * s2.to(D)
    return (codes @ w2.to(D).T) * scale, (near @ w2.to(D).abs().T) * scale


@pytest.mark.parametrize("tokens,hidden,inter,clamp", [
    (1, 7168, 2048, None), (1, 128, 64, 2.0), (3, 250, 130, None), (8, 1024, 512, 1.0), (16, 512, 1990, None), (40, 640, 300, 2.5),
    (80, 512, 1000, None), (128, 384, 256, 2.0), (200, 520, 264, None), (257, 256, 384, 1.5), (600, 1000, 700, None), (1024, 2048, 1024, None),
    (200, 6000, 100, 1.0), (200, 256, 16000, None),  # one product in either form
])
@pytest.mark.parametrize("dtype", [BF, FH, F32])
def test_ffn(tokens, hidden, inter, clamp, dtype):
    g = gen(tokens, hidden, inter)
    x, xs = weights(tokens, hidden, g)
    xs = xs * math.sqrt(hidden) * 2  # activations of order one
    w13, s13 = weights(2 * inter, hidden, g)
    w2, s2 = weights(hidden, inter, g)
    got = megamoe.int8_ffn(x, xs, w13, s13, w2, s2, clamp=clamp, out_dtype=dtype)
    want, flips = ffn_reference(x, xs, w13, s13, w2, s2, clamp)
    tol = flips + (torch.finfo(dtype).eps / 2 + 2.0 ** -16) * want.abs() + torch.finfo(dtype).smallest_normal
    assert got.dtype == dtype and got.shape == (tokens, hidden)
    assert bool(((got.to(D) - want).abs() <= tol).all())
    assert torch.equal(got, megamoe.int8_ffn(x, xs, w13, s13, w2, s2, clamp=clamp, out_dtype=dtype))
    megamoe.int8_check()


def test_ffn_zero_and_not_finite_rows():
    g = gen(77)
    x, xs = weights(5, 256, g)
    w13, s13 = weights(512, 256, g)
    w2, s2 = weights(256, 256, g)
    xs[1] = 0.0            # a zero row of the quantizer
    xs[3] = float("nan")   # a row that was not finite
    got = megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
    assert not got[1].any() and got[3].isnan().all()
    keep = [0, 2, 4]
    assert torch.equal(got[keep], megamoe.int8_ffn(int8_rows(x[keep]), xs[keep], w13, s13, w2, s2))


@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_rows_do_not_depend_on_their_batch(tokens):
    """A token's row is the same bits whatever stands beside it within one form of the kernels'
    sums: integer sums have one value, and what follows is per element."""
    g = gen(tokens, 31)
    x, xs = weights(tokens, 900, g)
    w, ws = weights(333, 900, g)
    whole = megamoe.int8_linear(x, xs, w, ws)
    for t in (0, tokens // 2, tokens - 1):
        assert torch.equal(whole[t:t + 1], megamoe.int8_linear(int8_rows(x[t:t + 1]), xs[t:t + 1], w, ws))


@pytest.mark.parametrize("hidden,inter", [(512, 1990), (1000, 77), (256, 4096)])
def test_ffn_rows_do_not_depend_on_their_batch(hidden, inter):
    """One token, the largest batch that makes h's codes inside the down product, the first that
    makes them in a launch of their own, and many tokens: the same bits a row."""
    g = gen(hidden, inter, 4)
    x, xs = weights(300, hidden, g)
    w13, s13 = weights(2 * inter, hidden, g)
    w2, s2 = weights(hidden, inter, g)
    xs = xs * math.sqrt(hidden)
    whole = megamoe.int8_ffn(x, xs, w13, s13, w2, s2, clamp=3.0)
    for t in (1, 5, 16, 17, 64, 65, 128, 129):
        assert torch.equal(whole[:t], megamoe.int8_ffn(x[:t], xs[:t], w13, s13, w2, s2, clamp=3.0)), t


def test_weights_written_just_before_the_call():
    """The launches start early and fetch weights early: never before they are written."""
    g = gen(12)
    w13a, s13 = weights(2 * 2048, 1024, g)
    w2a, s2 = weights(1024, 2048, g)
    w13b, w2b = w13a.flip(0).contiguous(), w2a.flip(0).contiguous()
    x, xs = weights(4, 1024, g)
    want = [megamoe.int8_ffn(x, xs, a, s13, b, s2) for a, b in ((w13a, w2a), (w13b, w2b))]
    w13, w2 = w13a.clone(), w2a.clone()
    got = []
    for k in range(40):
        w13.copy_(w13b if k % 2 else w13a)
        w2.copy_(w2b if k % 2 else w2a)
        got.append(megamoe.int8_ffn(x, xs, w13, s13, w2, s2))
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 2]), k
    # a gated product of many tokens before a down product that loads early
    x, xs = weights(200, 256, g)
    w13, s13 = weights(2 * 8192, 256, g)
    w2a, s2 = weights(256, 8192, g)
    w2b = w2a.flip(0).contiguous()
    want = [megamoe.int8_ffn(x, xs, w13, s13, b, s2) for b in (w2a, w2b)]
    w2 = w2a.clone()
    for k in range(20):
        w2.copy_(w2b if k % 2 else w2a)
        y = megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
        torch.cuda.synchronize()
        assert torch.equal(y, want[k % 2]), k
    x, xs = weights(4, 1024, g)
    # and by an operator of this library that lets its successor start early
    f = randn((4096, 1024), g)
    for k in range(20):
        f.mul_(-1)
        q, qs = megamoe.quantize_int8(f)
        y = megamoe.int8_linear(x, xs, q, qs)
        torch.cuda.synchronize()
        assert torch.equal(y, megamoe.int8_linear(x, xs, q, qs)), k


def test_empty_batches():
    e = torch.empty
    x = e((0, 64), dtype=torch.int8, device="cuda")
    w, ws = weights(32, 64, gen(1))
    assert megamoe.int8_linear(x, e(0, device="cuda"), w, ws).shape == (0, 32)
    w13, s13 = weights(64, 64, gen(2))
    w2, s2 = weights(64, 32, gen(3))
    assert megamoe.int8_ffn(x, e(0, device="cuda"), w13, s13, w2, s2).shape == (0, 64)
    out = megamoe.rms_norm(e((0, 64), dtype=BF, device="cuda"), torch.ones(64, dtype=BF, device="cuda"), quant="int8")
    assert out.codes.shape == (0, 64) and out.scales.shape == (0,)
    assert megamoe.quantize_int8(e((0, 64), device="cuda"))[0].shape == (0, 64)


def test_refusals():
    x = torch.zeros((4, 64), dtype=BF, device="cuda")
    gamma = torch.ones(64, dtype=BF, device="cuda")
    q, s = torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    bad = [
        lambda: megamoe.rms_norm(x.double(), gamma.double()),
        lambda: megamoe.rms_norm(x.flatten(), gamma),
        lambda: megamoe.rms_norm(x.t(), gamma[:4]),
        lambda: megamoe.rms_norm(x, gamma[:32]),
        lambda: megamoe.rms_norm(x, gamma.half()),
        lambda: megamoe.rms_norm(x, gamma.cpu()),
        lambda: megamoe.rms_norm(x, gamma, residual=x[:2]),
        lambda: megamoe.rms_norm(x, gamma, residual=x.half()),
        lambda: megamoe.rms_norm(x, gamma, residual_out=x),
        lambda: megamoe.rms_norm(x, gamma, out=x),
        lambda: megamoe.rms_norm(x, gamma, quant="fp8"),
        lambda: megamoe.rms_norm(x, gamma, with_norm=False),
        lambda: megamoe.rms_norm(x[:, :40], gamma[:40], quant="mxfp8"),
        lambda: megamoe.quantize_int8(q),
        lambda: megamoe.int8_linear(x, s, q, s),
        lambda: megamoe.int8_linear(q, s, q[:, :32], s),
        lambda: megamoe.int8_linear(q, s[:3], q, s),
        lambda: megamoe.int8_linear(q, s, q, s.double()),
        lambda: megamoe.int8_linear(q, s, q, s, s.half()),
        lambda: megamoe.int8_linear(q, s, q, s, out_dtype=torch.float64),
        lambda: megamoe.int8_linear(q, s, q, s, out=torch.empty((4, 5), dtype=BF, device="cuda")),
        lambda: megamoe.int8_linear(q[:, 8:], s, q[:, 8:], s),
        lambda: megamoe.int8_linear(torch.zeros((4, 72), dtype=torch.int8, device="cuda")[:, :64], s, q, s),
        lambda: megamoe.int8_ffn(q, s, q[:3], s[:3], q, s),
        lambda: megamoe.int8_ffn(q, s, q, s, q, s),
        lambda: megamoe.int8_ffn(q, s, q, s, torch.zeros((64, 16), dtype=torch.int8, device="cuda")[:, :2], gamma.float(), clamp=0.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_refusals_name_types_as_torch_does():
    q, s = torch.zeros((4, 64), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match=r"weight: expected a int8 \[T, 64\] tensor on cuda:0, got \[4, 64\] float32 on cuda:0"):
        megamoe.int8_linear(q, s, q.float(), s)


def test_streams_and_graphs():
    """Captured twice, replayed in turn and beside an eager call on another stream: no shared state."""
    g = gen(55)
    gamma = torch.ones(512, dtype=BF, device="cuda")
    w13, s13 = weights(2 * 320, 512, g)
    w2, s2 = weights(512, 320, g)

    def step(x):
        n = megamoe.rms_norm(x, gamma, quant="int8")
        return megamoe.int8_ffn(n.codes, n.scales, w13, s13, w2, s2)

    xs = [randn((t, 512), g, BF) for t in (3, 300, 40)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    graphs, outs, ins = [], [], []
    for x in xs:
        held = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(held)
        graphs.append(graph), outs.append(out), ins.append(held)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for turn in range(3):
        for k in (0, 1, 2, 1, 0):
            outs[k].zero_()
            graphs[k].replay()
            with torch.cuda.stream(side):
                eager = step(xs[k])
            torch.cuda.synchronize()
            assert torch.equal(outs[k], want[k]) and torch.equal(eager, want[k])
    ins[0].mul_(-1)
    graphs[0].replay()
    assert torch.equal(outs[0], step(-xs[0]))


@pytest.mark.parametrize("tokens", [1, 64, 300])
def test_first_call_of_a_process_is_captured(tokens):
    """Nothing that a first call sets up is closed to a capture."""
    code = f"""
import torch, megamoe
x, g = torch.randn(({tokens}, 512), device="cuda").bfloat16(), torch.ones(512, device="cuda").bfloat16()
w13, w2 = (torch.randint(-127, 127, s, dtype=torch.int8, device="cuda") for s in ((1024, 512), (512, 512)))
s13, s2 = torch.full((1024,), 1e-3, device="cuda"), torch.full((512,), 1e-3, device="cuda")
def step():
    n = megamoe.rms_norm(x, g, quant="int8")
    return megamoe.int8_ffn(n.codes, n.scales, w13, s13, w2, s2)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = step()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, step()) and y.isfinite().all()
"""
    path = os.pathsep.join(p for p in sys.path if p)
    done = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=path), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_back_to_back_chain_reads_finished_inputs():
    """Launches overlap their predecessors: a long chain without a wait gives the waited one's bits."""
    g = gen(8)
    gamma = torch.ones(1024, dtype=BF, device="cuda")
    w13, s13 = weights(2 * 512, 1024, g)
    w2, s2 = weights(1024, 512, g)

    def chain(x, wait):
        r = torch.zeros_like(x)
        for _ in range(12):
            n = megamoe.rms_norm(x, gamma, residual=r, quant="int8")
            x, r = megamoe.int8_ffn(n.codes, n.scales, w13, s13, w2, s2), n.residual
            if wait:
                torch.cuda.synchronize()
        return x, r

    for tokens in (1, 48, 300):
        x = randn((tokens, 1024), g, BF)
        for u, v in zip(chain(x, True), chain(x, False)):
            assert torch.equal(u, v)
