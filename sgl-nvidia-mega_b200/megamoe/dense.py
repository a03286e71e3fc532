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
and captured graphs, share none) and never synchronizes. What calls share is one
word a device, set when a bounded wait of an int8 product runs out and read by
``int8_check``. Tensors are 2-D with
their last dimension contiguous; rows may be strided. An output given as ``out=``
may not share memory with an input (``rms_norm``'s ``residual_out`` may; columns beside
each other of one buffer's rows share none). Outputs of
one call of up to 1 MiB together are parts of one allocation, which lives as long as
any of them. The operators are for inference: outputs carry no gradient. Violations
raise ValueError.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import check, lib

_dense = None


def _load():
    """The native calls (csrc/mm_dense_torch.cpp); raises if they have not been built."""
    global _dense
    if _dense is None:
        lib()
        try:
            from . import _dense as native
        except ImportError as e:
            raise RuntimeError(f"megamoe/_dense.so does not load ({e}): build it with `python __graft_entry__.py build` "
                               "(or megamoe._build.build())") from e
        _dense = native
    return _dense


class NormOutput(NamedTuple):
    """What ``rms_norm`` made; None for what was not asked for."""

    norm: Optional[torch.Tensor]      # x's type [T, H]
    codes: Optional[torch.Tensor]     # float8_e4m3fn or int8 [T, H]
    scales: Optional[torch.Tensor]    # float8_e8m0fnu [T, H / 32] or fp32 [T]
    residual: Optional[torch.Tensor]  # x + residual, x's type [T, H]


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
    return tuple.__new__(NormOutput, (_dense or _load()).rms_norm(x, gamma, eps, residual, quant, with_norm, out, residual_out))


def quantize_int8(x: torch.Tensor):
    """(codes int8 [T, H], scales fp32 [T]) of the rows of x (bf16, fp16 or fp32):
    scale = max |x| / 127, codes = rint(x / scale). A zero row has scale 0, a row
    with a value that is not finite scale NaN; both have codes 0. Code rows start
    on 16-byte boundaries (for other H, codes is a view of padded rows)."""
    return (_dense or _load()).quantize_int8(x)


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, out_dtype: torch.dtype = torch.bfloat16,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t, n] = (sum_k x[t, k] weight[n, k]) * x_scale[t] * weight_scale[n] + bias[n]:
    the sum is an exact integer, its conversion, the product with x_scale and the last
    product with the bias (fused) round in fp32, and the result to ``out_dtype`` (bf16,
    fp16 or fp32). x int8 [T, K] (``rms_norm`` / ``quantize_int8`` codes), weight int8 [N, K], both with
    rows on 16-byte boundaries, scales fp32 [T] and [N] (or [.., 1]), bias fp32 [N].
    K < 131072."""
    return (_dense or _load()).int8_linear(x, x_scale, weight, weight_scale, bias, out_dtype, out)


def int8_ffn(x: torch.Tensor, x_scale: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
             w2_scale: torch.Tensor, *, clamp: Optional[float] = None, out_dtype: torch.dtype = torch.bfloat16,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gated feed-forward block over int8 weights: x int8 [T, H] with fp32 [T] scales,
    w13 int8 [2I, H] (rows [0, I) gate, [I, 2I) up, as RoutedMoE's) and w2 int8 [H, I] with
    fp32 scales per row. gate, up = x's products with w13 (gate at most ``clamp``, up within
    +-``clamp``); h = silu(gate) * up in fp32; h's rows in int8 with a scale per token; out =
    their product with w2 in ``out_dtype``. As the shared expert of a layer, out is
    ``finalize``'s and ``RoutedMoE.forward``'s ``shared_output``."""
    return (_dense or _load()).int8_ffn(x, x_scale, w13, w13_scale, w2, w2_scale, clamp, out_dtype, out)


def int8_check(device: Optional[torch.device] = None) -> None:
    """Synchronize and raise (DeviceTimeoutError) if a bounded device wait of
    ``int8_linear`` or ``int8_ffn`` gave up on this device (default: the current one) since
    the last call. What such a call could not finish is NaN."""
    with torch.cuda.device(device):
        check(lib().mm_int8_check(), "int8_check")


def int8_set_wait_budget(microseconds: int) -> None:
    """Budget of every bounded device wait of the int8 products that this process launches or
    captures from now on (default 1.5 s)."""
    check(lib().mm_int8_set_wait_budget(int(microseconds)), "int8_set_wait_budget")
