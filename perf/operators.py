"""The dense 8-bit operators that stand beside the routed-MoE chain, as cases to measure.

  norm    megamoe.rms_norm: the residual's addition, the RMSNorm and its 8-bit output with scales
  quant   megamoe.quantize_int8: rows of activations to int8 with one scale a token
  linear  megamoe.int8_linear: a product in int8 with scales for each token and each channel
  ffn     megamoe.int8_ffn: the gated feed-forward block over int8 weights (the dense layers, and the
          shared expert whose output megamoe.finalize adds to the routed experts' sum)

Every case is one pass through one of them on data that a serving step has in hand: activations of the
model's type, int8 weights with a scale a channel, fp32 scales.
"""

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sgl-nvidia-mega_b200")
if _PACKAGE not in sys.path:
    sys.path.append(_PACKAGE)

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6

# the work of the largest listed case (flops) and its bytes: a drawn case stays below
_MOST_FLOPS = 6 * 4096 * 7168 * 18432
_MOST_BYTES = 8192 * 7168 * 10


def listed():
    return [
        # one token's step into an MoE layer: the router reads the norm, the experts its MXFP8 codes
        {"name": "norm 1 token mxfp8", "op": "norm", "tokens": 1, "hidden": 7168, "type": "bf16", "quant": "mxfp8", "norm": True, "residual": True},
        # a verify step into a dense layer: int8 codes alone
        {"name": "norm 48 tokens int8", "op": "norm", "tokens": 48, "hidden": 5120, "type": "bf16", "quant": "int8", "norm": False, "residual": True},
        # a ragged prompt at an odd width: no row starts on a 16-byte boundary but the first
        {"name": "norm 1021 tokens odd", "op": "norm", "tokens": 1021, "hidden": 6147, "type": "fp16", "quant": "", "norm": True, "residual": False},
        # a long prompt into an MoE layer
        {"name": "norm 8192 tokens mxfp8", "op": "norm", "tokens": 8192, "hidden": 7168, "type": "bf16", "quant": "mxfp8", "norm": True, "residual": True},
        # a decode step's attention output before its projection
        {"name": "quant 8 tokens", "op": "quant", "tokens": 8, "hidden": 7168, "type": "bf16"},
        # a prompt's activations at a dense layer's full width
        {"name": "quant 4093 tokens", "op": "quant", "tokens": 4093, "hidden": 18432, "type": "fp16"},
        # one token's projection: the weights' stream
        {"name": "linear 1 token", "op": "linear", "tokens": 1, "features": 4096, "depth": 7168, "type": "bf16", "bias": False},
        # a ragged batch, an odd number of features, a depth that ends inside a tile
        {"name": "linear 77 tokens odd", "op": "linear", "tokens": 77, "features": 2311, "depth": 5104, "type": "fp16", "bias": True},
        # a long prompt's projection: the tensor cores' rate
        {"name": "linear 8192 tokens", "op": "linear", "tokens": 8192, "features": 7168, "depth": 7168, "type": "bf16", "bias": False},
        # the shared expert of one token's step
        {"name": "ffn 1 token", "op": "ffn", "tokens": 1, "hidden": 7168, "inter": 2048, "type": "bf16", "clamp": 0.0},
        # the shared expert of a verify step, clamped, at a width that fills no tile
        {"name": "ffn 80 tokens clamped", "op": "ffn", "tokens": 80, "hidden": 6144, "inter": 1990, "type": "bf16", "clamp": 7.0},
        # a prompt through a dense layer as wide as nine experts
        {"name": "ffn 4096 tokens", "op": "ffn", "tokens": 4096, "hidden": 7168, "inter": 18432, "type": "bf16", "clamp": 0.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "quant", "linear", "ffn"])
        tokens = _log(rng, 1, 8192)
        if op == "norm":
            quant = rng.choice(["", "mxfp8", "int8"])
            kind = rng.choice(["bf16", "bf16", "fp16"] if quant == "int8" else ["bf16", "fp16", "fp32"])
            hidden = 32 * _log(rng, 4, 512) if quant == "mxfp8" else _log(rng, 100, 16384)
            case = {"op": op, "tokens": tokens, "hidden": hidden, "type": kind, "quant": quant, "norm": quant == "" or rng.random() < 0.5, "residual": rng.random() < 0.7}
        elif op == "quant":
            case = {"op": op, "tokens": tokens, "hidden": _log(rng, 100, 20000), "type": rng.choice(["bf16", "fp16"])}
        elif op == "linear":
            case = {"op": op, "tokens": tokens, "features": _log(rng, 64, 20000), "depth": _log(rng, 64, 20000), "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "bias": rng.random() < 0.3}
        else:
            case = {"op": op, "tokens": tokens, "hidden": _log(rng, 256, 8192), "inter": _log(rng, 64, 18432), "type": rng.choice(["bf16", "fp16"]), "clamp": rng.choice([0.0, 7.0])}
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return case


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(tokens, width, kind, g):
    """A residual stream's rows: normal values, each row of its own size, a few channels far larger than the rest."""
    x = _randn((tokens, width), g) * torch.exp(0.5 * _randn((tokens, 1), g))
    x *= 1.0 + 20.0 * (torch.rand((width,), generator=g, device="cuda") < 0.004)
    return x.to(_TYPES[kind])


def _rows(q):
    """int8 rows that start on 16-byte boundaries."""
    n, k = q.shape
    held = torch.zeros((n, (k + 15) // 16 * 16), dtype=torch.int8, device=q.device)
    held[:, :k] = q
    return held[:, :k]


def _codes(x):
    s = x.abs().amax(-1) / 127.0
    return _rows(torch.round(x / s.clamp_min(1e-30)[:, None]).to(torch.int8)), s


def _weights(n, k, g):
    """A checkpoint's channels: normal weights at their channel's own scale."""
    q = torch.empty((n, k), dtype=torch.float32, device="cuda").normal_(0.0, 32.0, generator=g).round_().clamp_(-127, 127)
    return _rows(q.to(torch.int8)), torch.exp(0.3 * _randn((n,), g)) / (32.0 * math.sqrt(k))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    state = dict(case)
    t = case["tokens"]
    if case["op"] in ("norm", "quant"):
        state["x"] = _activations(t, case["hidden"], case["type"], g)
    if case["op"] == "norm":
        if case["residual"]:
            state["r"] = _activations(t, case["hidden"], case["type"], g)
        state["gamma"] = (1.0 + 0.2 * _randn((case["hidden"],), g)).to(_TYPES[case["type"]])
    elif case["op"] == "linear":
        state["x"], state["xs"] = _codes(_activations(t, case["depth"], "fp32", g))
        state["w"], state["ws"] = _weights(case["features"], case["depth"], g)
        state["b"] = _randn((case["features"],), g) if case["bias"] else None
    elif case["op"] == "ffn":
        state["x"], state["xs"] = _codes(_activations(t, case["hidden"], "fp32", g))
        state["w13"], state["s13"] = _weights(2 * case["inter"], case["hidden"], g)
        state["w2"], state["s2"] = _weights(case["hidden"], case["inter"], g)
    return state


def _values(codes, scales, kind):
    """int8 codes as the values that they stand for, in the activations' type."""
    return torch.mul(codes, scales[:, None], out=torch.empty(codes.shape, dtype=kind, device=codes.device))


def _quantise(y):
    """int8 codes (as numbers) and scales of the rows of y: amax / 127, to the nearest even; a zero row's scale is zero."""
    s = y.abs().amax(-1) / 127.0
    q = torch.round(y / torch.where(s == 0, torch.ones_like(s), s)[:, None])
    return q.clamp(-127, 127), s


def _mx(y):
    """MXFP8 of the rows of y: an E8M0 scale, amax / 448 rounded up to a power of two, for each 32 values, and E4M3 codes."""
    b = y.reshape(y.shape[0], -1, 32)
    amax = b.abs().amax(-1).double()
    m, e = torch.frexp(torch.where(amax == 0, torch.full_like(amax, 448.0), amax) / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(-127, 127)
    return torch.ldexp(b.double(), -e[..., None]).float().reshape(y.shape), torch.ldexp(torch.ones_like(amax), e).float()


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _run_own(s):
    import megamoe

    kind = _TYPES[s["type"]]
    if s["op"] == "norm":
        out = megamoe.rms_norm(s["x"], s["gamma"], _EPS, residual=s.get("r"), quant=s["quant"] or None, with_norm=s["norm"])
        got = {"norm": out.norm, "residual": out.residual}
        if s["quant"] == "mxfp8":
            got["codes"], got["scales"] = out.codes, out.scales
        elif s["quant"] == "int8":
            got["values"], got["scales"] = _values(out.codes, out.scales, kind), out.scales
        return got
    if s["op"] == "quant":
        codes, scales = megamoe.quantize_int8(s["x"])
        return {"values": _values(codes, scales, kind), "scales": scales}
    if s["op"] == "linear":
        return megamoe.int8_linear(s["x"], s["xs"], s["w"], s["ws"], s["b"], out_dtype=kind)
    return megamoe.int8_ffn(s["x"], s["xs"], s["w13"], s["s13"], s["w2"], s["s2"], clamp=s["clamp"] or None, out_dtype=kind)


def run(s):
    if own:
        return _run_own(s)
    kind = _TYPES[s["type"]]
    if s["op"] == "norm":
        v, r = s["x"].float(), None
        if s["residual"]:
            r = (v + s["r"].float()).to(kind)
            v = r.float()
        y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * s["gamma"].float()
        got = {"norm": y.to(kind) if s["norm"] else None, "residual": r}
        if s["quant"] == "mxfp8":
            q, e = _mx(y)
            got["codes"], got["scales"] = q.to(torch.float8_e4m3fn), e.to(torch.float8_e8m0fnu)
        elif s["quant"] == "int8":
            q, scale = _quantise(y)
            got["values"], got["scales"] = (q * scale[:, None]).to(kind), scale
        return got
    if s["op"] == "quant":
        q, scale = _quantise(s["x"].float())
        return {"values": (q * scale[:, None]).to(kind), "scales": scale}
    if s["op"] == "linear":
        y = (s["x"].float() @ s["w"].float().t()) * s["xs"][:, None] * s["ws"]
        return (y if s["b"] is None else y + s["b"]).to(kind)
    y = (s["x"].float() @ s["w13"].float().t()) * s["xs"][:, None] * s["s13"]
    gate, up = y[:, : s["inter"]], y[:, s["inter"]:]
    if s["clamp"]:
        gate, up = gate.clamp(max=s["clamp"]), up.clamp(-s["clamp"], s["clamp"])
    q, scale = _quantise(_silu(gate) * up)
    return ((q @ s["w2"].float().t()) * scale[:, None] * s["s2"]).to(kind)


def work(case):
    t, e = case["tokens"], _BYTES[case["type"]]
    if case["op"] == "norm":
        h = case["hidden"]
        b = t * h * e * (1 + 2 * case["residual"] + case["norm"]) + h * e
        b += {"": 0, "mxfp8": t * h + t * h // 32, "int8": t * h * e + t * 4}[case["quant"]]
        return {"bytes": b, "flops": 8 * t * h}
    if case["op"] == "quant":
        h = case["hidden"]
        return {"bytes": t * h * (e + e) + t * 4, "flops": 4 * t * h}
    if case["op"] == "linear":
        n, k = case["features"], case["depth"]
        return {"bytes": t * k + 4 * t + n * k + 4 * n + 4 * n * case["bias"] + t * n * e, "flops": 2 * t * n * k}
    h, i = case["hidden"], case["inter"]
    return {"bytes": t * h + 4 * t + 3 * h * i + 8 * i + 4 * h + t * h * e, "flops": 6 * t * h * i}


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] in ("norm", "quant"):
        y, got = s["x"].to(d), {"norm": None, "residual": None}
        if case["op"] == "norm":
            if case["residual"]:
                # the stream that goes on, and that the norm reads, is held in the activations' type
                got["residual"] = y = (y + s["r"].to(d)).to(_TYPES[case["type"]]).to(d)
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / case["hidden"] + _EPS) * s["gamma"].to(d)
            if case["norm"]:
                got["norm"] = y
        quant = case.get("quant", "int8")
        if quant == "mxfp8":
            blocks = y.view(case["tokens"], -1, 32)
            top = blocks.abs().max(-1).values
            scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(-127, 127))
            scale = torch.where(top > 0, scale, torch.ones_like(scale))
            v = blocks / scale[..., None]
            # the nearest E4M3 number: 4 significant bits, and steps of 2^-9 below 2^-6; ties to even
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
            got["codes"], got["scales"] = (torch.round(v / step) * step).view(y.shape), scale
        elif quant == "int8":
            scale = y.abs().max(-1).values / 127
            codes = torch.where(scale[:, None] > 0, torch.round(y / scale[:, None]), torch.zeros_like(y))
            got["values"], got["scales"] = codes * scale[:, None], scale
        return got if case["op"] == "norm" else {"values": got["values"], "scales": got["scales"]}
    if case["op"] == "linear":
        out = torch.mm(s["x"].to(d), s["w"].to(d).T).mul_(s["xs"].to(d).unsqueeze(1)).mul_(s["ws"].to(d))
        return out if s["b"] is None else out.add_(s["b"].to(d))
    both = torch.mm(s["x"].to(d), s["w13"].to(d).T).mul_(s["xs"].to(d).unsqueeze(1)).mul_(s["s13"].to(d))
    gate, up = both.split(case["inter"], 1)
    if case["clamp"]:
        gate, up = torch.minimum(gate, torch.full_like(gate, case["clamp"])), up.clip(-case["clamp"], case["clamp"])
    h = gate * torch.sigmoid(gate) * up
    scale = h.abs().max(1).values / 127
    codes = torch.where(scale[:, None] > 0, torch.round(h / scale[:, None]), torch.zeros_like(h))
    return torch.mm(codes, s["w2"].to(d).T).mul_(scale[:, None]).mul_(s["s2"].to(d))
