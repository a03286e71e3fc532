"""The dense 8-bit operators beside the routed-MoE chain.

  * ``rms_norm``: the residual's addition, the RMSNorm and its output in bf16 /
    fp16 / fp32 and in 8 bits (MXFP8, the routed input of ``RoutedMoE``, or int8)
    in one launch; what the reference's hop fuses behind its all-reduce
    (deepseek_v41/sm103/all_reduce_mhc.py:665-1190), for one GPU's rows;
  * ``quantize_int8``: rows to int8 with one scale a token;
  * ``int8_linear``: a product in int8 with scales for each token and channel;
  * ``int8_ffn``: the gated feed-forward block over int8 weights: dense layers, and
    the shared expert (deepseek_v41/moe/shared_ll.py:1-20 keeps it at 8 bits beside
    FP4 routed experts), whose output ``finalize(..., shared_output=)`` takes.

Every call runs on the current stream of the tensors' device, allocates its
outputs and its workspace from torch's allocator (so calls on several streams,
and captured graphs, share none) and never synchronizes. Tensors are 2-D with
their last dimension contiguous; rows may be strided. Violations raise ValueError.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check, lib

_DTYPES = {torch.bfloat16: _lib.MM_DTYPE_BF16, torch.float16: _lib.MM_DTYPE_FP16, torch.float32: _lib.MM_DTYPE_FP32}
_QUANTS = {None: _lib.MM_QUANT_NONE, "mxfp8": _lib.MM_QUANT_MXFP8, "int8": _lib.MM_QUANT_INT8}


class NormOutput(NamedTuple):
    """What ``rms_norm`` made; None for what was not asked for."""

    norm: Optional[torch.Tensor]      # x's type [T, H]
    codes: Optional[torch.Tensor]     # float8_e4m3fn or int8 [T, H]
    scales: Optional[torch.Tensor]    # float8_e8m0fnu [T, H / 32] or fp32 [T]
    residual: Optional[torch.Tensor]  # x + residual, x's type [T, H]


class _on:
    """The tensors' device as the current one for a call, and its current stream."""

    def __init__(self, device: torch.device):
        self.index = device.index
        self.before = torch._C._cuda_getDevice()

    def __enter__(self) -> int:
        if self.index != self.before:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.index != self.before:
            torch.cuda.set_device(self.before)


def _rows(t: torch.Tensor, name: str, device: torch.device, dtype=None, cols: Optional[int] = None,
          rows: Optional[int] = None) -> int:
    """Checks a [rows, cols] tensor with contiguous rows; its row stride."""
    if t.dim() != 2 or (dtype is not None and t.dtype != dtype) or t.device != device or t.layout != torch.strided \
            or (cols is not None and t.size(1) != cols) or (rows is not None and t.size(0) != rows):
        want = f"[{'T' if rows is None else rows}, {'K' if cols is None else cols}]"
        raise ValueError(f"{name}: expected a {dtype or ''} {want} tensor on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t.size(1) > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: rows must be contiguous (stride 1 along the last dimension)")
    return t.stride(0) if t.size(0) > 1 else max(t.size(1), 1)


def _vector(t: torch.Tensor, name: str, n: int, device: torch.device, dtype=torch.float32) -> int:
    """Checks n contiguous values ([n] or [n, 1]); their address."""
    if t.dtype != dtype or t.numel() != n or t.device != device or t.size(0) != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous {dtype} values on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _code_rows(t: torch.Tensor, name: str, device: torch.device, cols: Optional[int] = None, rows: Optional[int] = None) -> int:
    ld = _rows(t, name, device, torch.int8, cols, rows)
    if t.size(0) == 1:  # one row needs no stride of its own
        ld = (ld + 15) // 16 * 16
    if t.data_ptr() % 16 or ld % 16:
        raise ValueError(f"{name}: int8 rows must start on 16-byte boundaries (row stride {ld}); rms_norm and "
                         "quantize_int8 return them so, weights are laid out once with a padded row stride")
    return ld


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.device


def _int8_rows(rows: int, cols: int, device: torch.device) -> torch.Tensor:
    """int8 [rows, cols] whose rows start on 16-byte boundaries."""
    if cols % 16 == 0:
        return torch.empty((rows, cols), dtype=torch.int8, device=device)
    return torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :cols]


def _out(out: Optional[torch.Tensor], name: str, rows: int, cols: int, dtype, device: torch.device):
    if out is None:
        return torch.empty((rows, cols), dtype=dtype, device=device), cols
    return out, _rows(out, name, device, dtype, cols, rows)


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, *, residual: Optional[torch.Tensor] = None,
             quant: Optional[str] = None, with_norm: Optional[bool] = None, out: Optional[torch.Tensor] = None,
             residual_out: Optional[torch.Tensor] = None) -> NormOutput:
    """RMSNorm of x (+ residual), bf16, fp16 or fp32 [T, H], in one launch:
    r = x + residual rounded to x's type (``residual`` of the result),
    y = r / sqrt(mean(r^2) + eps) * gamma in fp32, ``norm`` = y in x's type.
    ``quant="mxfp8"``: also y's E4M3 codes and E8M0 scales per 32 values
    (H a multiple of 32), what ``RoutedMoE(x_quant, x_scale, ...)`` takes;
    ``quant="int8"``: y's int8 codes and fp32 scale per token, what
    ``int8_linear`` and ``int8_ffn`` take. The 8-bit forms return no norm
    unless ``with_norm`` (a router reads it). ``gamma``: [H] of x's type or
    fp32. ``out`` / ``residual_out`` take the norm and the sum where given
    (``residual_out`` may be ``residual`` or ``x`` itself)."""
    device = _cuda(x, "x")
    ld_x = _rows(x, "x", device)
    tokens, hidden = x.shape
    if x.dtype not in _DTYPES:
        raise ValueError(f"x: bf16, fp16 or fp32, not {x.dtype}")
    if quant not in _QUANTS:
        raise ValueError(f"quant {quant!r}: None, 'mxfp8' or 'int8'")
    if hidden < 1 or (quant == "mxfp8" and hidden % 32):
        raise ValueError(f"rows of {hidden} values (mxfp8: a multiple of 32)")
    if gamma.dtype != x.dtype and gamma.dtype != torch.float32:
        raise ValueError(f"gamma: {x.dtype} or fp32, not {gamma.dtype}")
    a = _lib.MMNormArgs()
    a.gamma = _vector(gamma, "gamma", hidden, device, gamma.dtype)
    a.gamma_dtype = _DTYPES[gamma.dtype]
    a.x, a.ld_x = x.data_ptr(), ld_x
    r = norm = codes = scales = None
    if residual is not None:
        a.ld_residual = _rows(residual, "residual", device, x.dtype, hidden, tokens)
        a.residual = residual.data_ptr()
        r, a.ld_residual_out = _out(residual_out, "residual_out", tokens, hidden, x.dtype, device)
        a.residual_out = r.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    if quant is None or with_norm or out is not None:
        if with_norm is False:
            raise ValueError("with_norm=False needs quant and no out")
        norm, a.ld_norm = _out(out, "out", tokens, hidden, x.dtype, device)
        a.norm_out = norm.data_ptr()
    if quant == "mxfp8":
        codes = torch.empty((tokens, hidden), dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty((tokens, hidden // 32), dtype=torch.float8_e8m0fnu, device=device)
    elif quant == "int8":
        codes = _int8_rows(tokens, hidden, device)
        scales = torch.empty((tokens,), dtype=torch.float32, device=device)
    if quant is not None:
        a.codes, a.scales, a.ld_codes = codes.data_ptr(), scales.data_ptr(), (hidden + 15) // 16 * 16
    a.tokens, a.hidden, a.dtype, a.quant, a.eps = tokens, hidden, _DTYPES[x.dtype], _QUANTS[quant], eps
    with _on(device) as stream:
        check(lib().mm_rms_norm(ctypes.byref(a), stream), "rms_norm")
    return NormOutput(norm, codes, scales, r)


def quantize_int8(x: torch.Tensor):
    """(codes int8 [T, H], scales fp32 [T]) of the rows of x (bf16, fp16 or fp32):
    scale = max |x| / 127, codes = rint(x / scale). A zero row has scale 0, a row
    with a value that is not finite scale NaN; both have codes 0. Code rows start
    on 16-byte boundaries (for other H, codes is a view of padded rows)."""
    device = _cuda(x, "x")
    ld = _rows(x, "x", device)
    tokens, hidden = x.shape
    if x.dtype not in _DTYPES or hidden < 1:
        raise ValueError(f"x: bf16, fp16 or fp32 [T, H], not {tuple(x.shape)} {x.dtype}")
    codes = _int8_rows(tokens, hidden, device)
    scales = torch.empty((tokens,), dtype=torch.float32, device=device)
    with _on(device) as stream:
        check(lib().mm_quantize_int8(x.data_ptr(), ld, _DTYPES[x.dtype], codes.data_ptr(), (hidden + 15) // 16 * 16,
                                     scales.data_ptr(), tokens, hidden, stream), "quantize_int8")
    return codes, scales


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, out_dtype: torch.dtype = torch.bfloat16,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t, n] = (sum_k x[t, k] weight[n, k]) * x_scale[t] * weight_scale[n] + bias[n],
    one rounding to ``out_dtype`` (bf16, fp16 or fp32) from an exact integer sum:
    x int8 [T, K] (``rms_norm`` / ``quantize_int8`` codes), weight int8 [N, K], both with
    rows on 16-byte boundaries, scales fp32 [T] and [N] (or [.., 1]), bias fp32 [N].
    K < 131072."""
    device = _cuda(x, "x")
    ld_x = _code_rows(x, "x", device)
    tokens, depth = x.shape
    ld_w = _code_rows(weight, "weight", device, depth)
    features = weight.size(0)
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype: bf16, fp16 or fp32, not {out_dtype}")
    if features < 1 or not 1 <= depth < 1 << 17:
        raise ValueError(f"weight: {features} features of depth {depth} (1..131071)")
    xs, ws = _vector(x_scale, "x_scale", tokens, device), _vector(weight_scale, "weight_scale", features, device)
    b = None if bias is None else _vector(bias, "bias", features, device)
    out, ld_out = _out(out, "out", tokens, features, out_dtype, device)
    with _on(device) as stream:
        check(lib().mm_int8_linear(x.data_ptr(), ld_x, xs, weight.data_ptr(), ld_w, ws, b, out.data_ptr(), ld_out,
                                   _DTYPES[out_dtype], tokens, features, depth, stream), "int8_linear")
    return out


def int8_ffn(x: torch.Tensor, x_scale: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
             w2_scale: torch.Tensor, *, clamp: Optional[float] = None, out_dtype: torch.dtype = torch.bfloat16,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gated feed-forward block over int8 weights: x int8 [T, H] with fp32 [T] scales,
    w13 int8 [2I, H] (rows [0, I) gate, [I, 2I) up, as RoutedMoE's) and w2 int8 [H, I] with
    fp32 scales per row. gate, up = x's products with w13 (gate at most ``clamp``, up within
    +-``clamp``); h = silu(gate) * up in fp32; h's rows in int8 with a scale per token; out =
    their product with w2 in ``out_dtype``. As the shared expert of a layer, out is
    ``finalize``'s and ``RoutedMoE.forward``'s ``shared_output``."""
    device = _cuda(x, "x")
    a = _lib.MMInt8FFNArgs()
    a.ld_x = _code_rows(x, "x", device)
    tokens, hidden = x.shape
    a.ld_w13 = _code_rows(w13, "w13", device, hidden)
    inter = w13.size(0) // 2
    if w13.size(0) != 2 * inter or not 1 <= inter < 1 << 17 or not 1 <= hidden < 1 << 17:
        raise ValueError(f"w13: expected int8 [2I, H] with I and H in 1..131071, got {tuple(w13.shape)}")
    a.ld_w2 = _code_rows(w2, "w2", device, inter, hidden)
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype: bf16, fp16 or fp32, not {out_dtype}")
    if clamp is not None and not 0.0 < clamp < float("inf"):
        raise ValueError(f"clamp {clamp}: a positive number or None")
    a.x_scale = _vector(x_scale, "x_scale", tokens, device)
    a.w13_scale = _vector(w13_scale, "w13_scale", 2 * inter, device)
    a.w2_scale = _vector(w2_scale, "w2_scale", hidden, device)
    out, a.ld_out = _out(out, "out", tokens, hidden, out_dtype, device)
    size = lib().mm_int8_ffn_workspace(tokens, inter)
    space = torch.empty((size,), dtype=torch.uint8, device=device)
    a.x, a.w13, a.w2, a.out = x.data_ptr(), w13.data_ptr(), w2.data_ptr(), out.data_ptr()
    a.workspace, a.workspace_bytes = space.data_ptr(), size
    a.tokens, a.hidden, a.inter, a.out_dtype = tokens, hidden, inter, _DTYPES[out_dtype]
    a.clamp = 0.0 if clamp is None else clamp
    with _on(device) as stream:
        check(lib().mm_int8_ffn(ctypes.byref(a), stream), "int8_ffn")
    return out


def int8_check(device: Optional[torch.device] = None) -> None:
    """Synchronize and raise (DeviceTimeoutError) if a bounded device wait of
    ``int8_linear`` or ``int8_ffn`` gave up on this device (default: the current one)."""
    index = torch._C._cuda_getDevice() if device is None else torch.device(device).index
    with _on(torch.device("cuda", index)):
        check(lib().mm_int8_check(), "int8_check")
