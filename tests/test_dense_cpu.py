"""The dense 8-bit operators without a GPU: every refusal comes back as a status (C) or a
ValueError (Python) before anything reaches the device, and empty calls launch nothing."""

import ctypes
import os

import pytest
import torch

import megamoe
from megamoe import _lib
from test_kernel_resources import NVCC, _ptxas_info

BUF = (ctypes.c_uint8 * (1 << 16))()
BASE = (ctypes.addressof(BUF) + 255) & ~255  # a 256-byte aligned host address that is never read


def norm_args(**kw):
    a = _lib.MMNormArgs()
    a.x, a.gamma, a.norm_out, a.codes, a.scales = BASE, BASE + 4096, BASE + 8192, BASE + 12288, BASE + 16384
    a.residual, a.residual_out = BASE + 20480, BASE + 24576
    for f in ("ld_x", "ld_residual", "ld_residual_out", "ld_norm", "ld_codes"):
        setattr(a, f, 64)
    a.tokens, a.hidden, a.eps = 2, 64, 1e-6
    a.dtype = a.gamma_dtype = _lib.MM_DTYPE_BF16
    a.quant = _lib.MM_QUANT_INT8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,word", [
    (dict(x=None), b"null"),
    (dict(gamma=None), b"gamma"),
    (dict(gamma_dtype=_lib.MM_DTYPE_FP16), b"gamma"),
    (dict(gamma=BASE + 4097), b"gamma"),
    (dict(codes=None), b"null"),
    (dict(scales=None), b"null"),
    (dict(scales=BASE + 16386), b"scales"),
    (dict(quant=_lib.MM_QUANT_NONE, norm_out=None), b"null"),
    (dict(residual_out=None), b"residual_out"),
    (dict(dtype=3, gamma_dtype=3), b"type"),
    (dict(quant=3), b"format"),
    (dict(tokens=-1), b"tokens"),
    (dict(hidden=0), b"values"),
    (dict(hidden=48, quant=_lib.MM_QUANT_MXFP8), b"32"),
    (dict(ld_x=63), b"stride"),
    (dict(ld_residual=63), b"stride"),
    (dict(ld_residual_out=63), b"stride"),
    (dict(ld_norm=63), b"stride"),
    (dict(ld_codes=63), b"stride"),
    (dict(x=BASE + 1), b"misaligned"),
    (dict(norm_out=BASE), b"overlaps"),
    (dict(norm_out=BASE + 20480 + 64), b"overlaps"),
    (dict(residual_out=BASE + 2), b"overlaps"),
    (dict(residual_out=BASE, ld_residual_out=128), b"overlaps"),
    (dict(norm_out=BASE + 24576), b"overlaps"),
])
def test_norm_refusals(bad, word):
    L = _lib.lib()
    assert L.mm_rms_norm(ctypes.byref(norm_args(**bad)), None) == _lib.MM_ERR_INVALID
    assert word in L.mm_last_error(), L.mm_last_error()


@pytest.mark.parametrize("bad", [
    dict(norm_out=BASE + 4096 - 64), dict(codes=BASE + 64), dict(codes=BASE + 4096), dict(scales=BASE + 12288 + 32),
    dict(codes=BASE + 20480), dict(residual_out=BASE + 4096), dict(scales=BASE + 8192),
    dict(codes=BASE + 24576 + 192), dict(gamma=BASE + 12288 - 124, gamma_dtype=_lib.MM_DTYPE_FP32),
])
def test_norm_outputs_share_no_memory(bad):
    L = _lib.lib()
    assert L.mm_rms_norm(ctypes.byref(norm_args(**bad)), None) == _lib.MM_ERR_INVALID
    assert b"overlaps" in L.mm_last_error(), L.mm_last_error()


MOST = 1 << 30


@pytest.mark.parametrize("tokens,hidden", [(1, MOST + 1), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (0, MOST + 1)])
def test_row_kernels_sizes(tokens, hidden):
    L = _lib.lib()
    big = dict(tokens=tokens, hidden=hidden, **{f: hidden for f in ("ld_x", "ld_residual", "ld_residual_out", "ld_norm", "ld_codes")})
    assert L.mm_rms_norm(ctypes.byref(norm_args(**big)), None) == _lib.MM_ERR_UNSUPPORTED
    assert L.mm_quantize_int8(BASE, hidden, 0, BASE, hidden, BASE, tokens, hidden, None) == _lib.MM_ERR_UNSUPPORTED


def test_empty_calls_launch_nothing():
    L = _lib.lib()
    assert L.mm_rms_norm(ctypes.byref(norm_args(tokens=0)), None) == _lib.MM_OK
    assert L.mm_quantize_int8(BASE, 64, 0, BASE, 64, BASE, 0, 64, None) == _lib.MM_OK
    assert L.mm_int8_linear(BASE, 64, BASE, BASE, 64, BASE, None, BASE, 64, 0, 0, 64, 64, None) == _lib.MM_OK
    assert L.mm_int8_ffn(ctypes.byref(ffn_args(tokens=0)), None) == _lib.MM_OK
    assert L.mm_int8_ffn_workspace(0, 64) == 0


def linear(**kw):
    a = dict(x=BASE, ld_x=64, xs=BASE, w=BASE + 8192, ld_w=64, ws=BASE, bias=None, out=BASE + 16384, ld_out=32, dtype=0, tokens=2,
             features=32, depth=64)
    a.update(kw)
    return _lib.lib().mm_int8_linear(a["x"], a["ld_x"], a["xs"], a["w"], a["ld_w"], a["ws"], a["bias"], a["out"],
                                     a["ld_out"], a["dtype"], a["tokens"], a["features"], a["depth"], None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), 1), (dict(xs=None), 1), (dict(w=None), 1), (dict(ws=None), 1), (dict(out=None), 1),
    (dict(x=BASE + 8), 1), (dict(w=BASE + 8), 1), (dict(ld_x=72), 1), (dict(ld_w=72), 1),
    (dict(ld_x=48), 1), (dict(ld_w=48), 1), (dict(ld_out=31), 1), (dict(out=BASE + 16385), 1),
    (dict(out=BASE + 2, dtype=2), 1), (dict(xs=BASE + 2), 1), (dict(bias=BASE + 2), 1), (dict(dtype=5), 1),
    (dict(tokens=-1), 1), (dict(features=0), 1), (dict(depth=0), 1),
    (dict(out=BASE + 126), 1), (dict(out=BASE + 8192 + 2046), 1), (dict(out=BASE + 8192 - 126), 1),
    (dict(depth=1 << 17, ld_x=1 << 17, ld_w=1 << 17), 2), (dict(tokens=1 << 23), 2),
])
def test_linear_refusals(bad, status):
    assert linear(**bad) == status
    assert b"mm_int8_linear" in _lib.lib().mm_last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(out=BASE + 40960, xs=BASE + 40960 + 124), 1), (dict(out=BASE + 40960, ws=BASE + 40960 - 124), 1),
    (dict(out=BASE + 40960, bias=BASE + 40960), 1), (dict(features=MOST + 1, ld_out=MOST + 1), 2),
])
def test_linear_output_and_sizes(bad, status):
    assert linear(**bad) == status


@pytest.mark.parametrize("name,at", [("x", 0), ("w13", 256), ("w2", 256), ("x_scale", 300), ("w13_scale", 300), ("w2_scale", 300), ("out", 256)])
def test_ffn_workspace_overlaps(name, at):
    L = _lib.lib()
    assert L.mm_int8_ffn(ctypes.byref(ffn_args(**{name: BASE + 4096 * 7 + at})), None) == _lib.MM_ERR_INVALID
    assert b"overlaps" in L.mm_last_error(), L.mm_last_error()


@pytest.mark.parametrize("name", ["x", "x_scale", "w13", "w13_scale", "w2", "w2_scale"])
def test_ffn_output_overlaps(name):
    L = _lib.lib()
    assert L.mm_int8_ffn(ctypes.byref(ffn_args(**{name: BASE + 4096 * 6})), None) == _lib.MM_ERR_INVALID
    assert b"overlaps an input" in L.mm_last_error(), L.mm_last_error()


def ffn_args(**kw):
    a = _lib.MMInt8FFNArgs()
    for i, f in enumerate(("x", "x_scale", "w13", "w13_scale", "w2", "w2_scale", "out", "workspace")):
        setattr(a, f, BASE + 4096 * i)
    a.ld_x = a.ld_w13 = a.ld_out = 64
    a.ld_w2 = 32
    a.tokens, a.hidden, a.inter, a.out_dtype = 2, 64, 32, 0
    a.workspace_bytes = _lib.lib().mm_int8_ffn_workspace(2, 32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,word", [
    (dict(workspace=None), b"workspace"), (dict(workspace=BASE + 16), b"workspace"), (dict(workspace_bytes=8), b"workspace"),
    (dict(clamp=-1.0), b"clamp"), (dict(clamp=float("nan")), b"clamp"), (dict(clamp=float("inf")), b"clamp"),
    (dict(x=None), b"null"), (dict(w13_scale=None), b"null"), (dict(w2=None), b"null"), (dict(out=None), b"null"),
    (dict(ld_w2=24), b"stride"), (dict(ld_w13=72), b"16-byte"), (dict(w2=BASE + 4), b"16-byte"), (dict(inter=0), b"inter"),
    (dict(tokens=-1), b"tokens"), (dict(out_dtype=9), b"type"),
])
def test_ffn_refusals(bad, word):
    L = _lib.lib()
    assert L.mm_int8_ffn(ctypes.byref(ffn_args(**bad)), None) == _lib.MM_ERR_INVALID
    assert word in L.mm_last_error(), L.mm_last_error()


def test_null_arguments():
    L = _lib.lib()
    assert L.mm_rms_norm(None, None) == _lib.MM_ERR_INVALID
    assert L.mm_int8_ffn(None, None) == _lib.MM_ERR_INVALID


def test_there_is_no_cpu_path():
    x, q = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.int8)
    s = torch.ones(2)
    with pytest.raises(ValueError, match="CUDA"):
        megamoe.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="CUDA"):
        megamoe.quantize_int8(x)
    with pytest.raises(ValueError, match="CUDA"):
        megamoe.int8_linear(q, s, q, s)
    with pytest.raises(ValueError, match="CUDA"):
        megamoe.int8_ffn(q, s, q, s, q, s)


@pytest.mark.skipif(not os.path.exists(NVCC), reason="nvcc not found")
@pytest.mark.parametrize("source,spills", [("mm_int8.cu", {}), ("mm_norm.cu", {"norm_rows_kernelIfLi8ELi2ELb0E": 300})])
def test_no_kernel_spills(source, spills):
    """Only the fp32 row form that keeps two CTAs on an SM trades a few registers for them."""
    kernels = _ptxas_info(source)
    assert len(kernels) >= 8
    for name, info in kernels.items():
        most = next((v for k, v in spills.items() if k in name), 0)
        assert info.get("spill", 0) <= most, (name, info)
        if "int8_stream_kernel" in name:  # two CTAs an SM
            assert info["regs"] <= 128


def test_workspace_size():
    ws = _lib.lib().mm_int8_ffn_workspace
    assert ws(3, 100) == 1280 + 512 + 12  # fp32 rows, code rows of 112 bytes, scales
    assert ws(1 << 20, 1 << 14) > 1 << 36
