"""The dense 8-bit operators run together with the routed-MoE chain, as a decoder step uses
them: norm -> int8 dense layer -> norm with MXFP8 -> routed experts beside an int8 shared
expert -> combine. Each hand-over is held bit for bit to the same step taken apart."""

import math

import pytest
import torch

import megamoe
import oracle.oracle as O

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
H, I, E, K, TMAX = 1024, 512, 16, 4, 16


def ffn_weights(hidden, inter, g):
    def q(n, k):
        return (torch.randn((n, k), generator=g) * 40).round().clamp(-127, 127).to(torch.int8).cuda(), \
            (torch.rand(n, generator=g) + 0.5).cuda() / (40 * math.sqrt(k))
    return (*q(2 * inter, hidden), *q(hidden, inter))


def setup(seed):
    g = torch.Generator().manual_seed(seed)
    layer = O.make_layer(H, I, E, shared=False, seed=seed)
    moe = megamoe.RoutedMoE(*(layer[k].cuda() for k in ("w13", "w13_scale", "w2", "w2_scale")), K, TMAX)
    _, wr, bias = O.make_inputs(1, H, E, seed=seed)
    gammas = [(1 + 0.1 * torch.randn(H, generator=g)).to(BF).cuda() for _ in range(3)]
    return g, layer, moe, wr.cuda(), bias.cuda(), gammas, ffn_weights(H, 768, g), ffn_weights(H, I, g)


def step(x, r, moe, wr, bias, gammas, dense, shared, buffers=None):
    n = megamoe.rms_norm(x, gammas[0], residual=r, quant="int8")
    y = megamoe.int8_ffn(n.codes, n.scales, *dense)
    m = megamoe.rms_norm(y, gammas[1], residual=n.residual, quant="mxfp8", with_norm=True)
    q, s = megamoe.quantize_int8(m.norm)
    shared_rows = megamoe.int8_ffn(q, s, *shared, clamp=7.0)
    logits = megamoe.router_gemv(m.norm, wr)
    rows, w, perm, ids = moe.gate_topk_and_gemms(m.codes, m.scales, logits, bias, 2.5)
    out = moe.finalize(rows, w, perm, shared_rows)
    f = megamoe.rms_norm(out, gammas[2], residual=m.residual)
    return dict(y=y, m=m, shared=shared_rows, ids=ids, w=w, perm=perm, rows=rows, out=out, norm=f.norm, residual=f.residual)


@pytest.mark.parametrize("T", [1, 5, 16])
def test_decoder_step(T):
    g, layer, moe, wr, bias, gammas, dense, shared = setup(40 + T)
    x, r = (torch.randn((T, H), generator=g).to(BF).cuda() for _ in range(2))
    a = step(x, r, moe, wr, bias, gammas, dense, shared)
    moe.check()
    megamoe.int8_check()
    m = a["m"]
    # the codes are the norm's MXFP8: fed back as the bf16 values that they stand for, the experts
    # compute the same rows
    values = (m.codes.float().view(T, -1, 32) * m.scales.float()[..., None]).view(T, H)
    assert torch.equal(values.to(BF).float(), values)
    rows, _, perm = moe(values.to(BF), None, a["ids"], a["w"])
    used = a["perm"][a["perm"] >= 0].long()
    assert torch.equal(perm, a["perm"]) and torch.equal(rows[used], a["rows"][used])
    # and the step is the fp32 layer of those values, with the int8 block added
    want, _, _ = O.moe_layer(values.to(BF).cpu(), a["ids"].cpu().numpy(), a["w"].cpu().numpy(), layer, numerics="exact")
    want = want + a["shared"].float().cpu()
    assert O.max_abs_rel(a["out"].float().cpu().numpy(), want.numpy()) <= 2e-2
    # the norm's rule: what the next layer reads is out + residual in bf16
    assert torch.equal(a["residual"], (a["out"].float() + m.residual.float()).to(BF))


def test_forward_takes_a_shared_output():
    T = 7
    g, layer, moe, wr, bias, gammas, dense, shared = setup(51)
    x = torch.randn((T, H), generator=g).to(BF).cuda()
    q, s = megamoe.quantize_int8(x)
    rows = megamoe.int8_ffn(q, s, *shared)
    call = dict(router_weight=wr, bias=bias, routed_scaling_factor=2.5)
    b = {}
    got = moe.forward(x, **call, shared_output=rows, buffers=b)
    want = megamoe.finalize(b["rows"], b["weights"], b["permuted"], rows)
    assert torch.equal(got, want) and not torch.equal(got, moe.forward(x, **call))
    part = moe.forward(x, **call, shared_output=rows, partial=True)
    assert torch.equal(megamoe.finalize_partial(part), want) and torch.equal(part[1], rows.float())
    comm = megamoe.PeerAllReduce(TMAX, H, eps=1e-6)
    assert torch.equal(moe.forward(x, **call, shared_output=rows, comm=comm), want)
    res = torch.randn((T, H), generator=g).to(BF).cuda()
    norm, new = moe.forward(x, **call, shared_output=rows, comm=comm, residual=res, gamma=gammas[0])
    single = megamoe.rms_norm(want, gammas[0], 1e-6, residual=res)
    assert torch.equal(new, single.residual)
    # the hop's fold of the sum of squares is its own: one bf16 step apart at most
    assert bool(((norm.float() - single.norm.float()).abs() <= 2.0 ** -7 * single.norm.float().abs()).all())
    none, new = moe.forward(x, **call, shared_output=rows, comm=comm, residual=res)
    assert none is None and torch.equal(new, single.residual)
    comm.check()


def test_forward_refuses_a_wrong_shared_output():
    g, layer, moe, wr, bias, gammas, dense, shared = setup(52)
    x = torch.randn((3, H), generator=g).to(BF).cuda()
    for bad in (x[:2], x.half(), x.cpu(), x.t().contiguous().t()):
        with pytest.raises(ValueError, match="shared_output"):
            moe.forward(x, router_weight=wr, bias=bias, shared_output=bad)
    full = O.make_layer(H, I, E, shared=True, seed=3)
    own = megamoe.RoutedMoE(*(full[k].cuda() for k in ("w13", "w13_scale", "w2", "w2_scale")), K, TMAX,
                            shared=[t.cuda() for t in full["shared"]])
    with pytest.raises(ValueError, match="shared_output"):
        own.forward(x, router_weight=wr, bias=bias, shared_output=x)


def test_decoder_step_in_a_graph():
    g, layer, moe, wr, bias, gammas, dense, shared = setup(60)
    T = 6
    x, r = (torch.randn((T, H), generator=g).to(BF).cuda() for _ in range(2))
    want = step(x, r, moe, wr, bias, gammas, dense, shared)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, r, moe, wr, bias, gammas, dense, shared)
    for _ in range(3):
        for k in ("out", "norm", "residual", "shared", "y"):
            got[k].zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k in ("out", "norm", "residual", "shared", "y"):
            assert torch.equal(got[k], want[k]), k
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    again = step(x, r, moe, wr, bias, gammas, dense, shared)
    assert torch.equal(got["norm"], again["norm"]) and not torch.equal(got["norm"], want["norm"])
