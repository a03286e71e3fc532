"""fp32 gamma beside 16-bit rows, in each form of the row kernels: few and many rows, one to
eight chunks a thread, rows that share a CTA, rows too long to hold, rows and gamma off the
16-byte grid. Against the norm in 64 bits; tolerances as tests/test_gpu_dense.py derives them."""

import pytest
import torch

import megamoe
from test_gpu_dense import check_norm, gen, randn

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("quant", [None, "int8", "mxfp8"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("tokens,hidden", [(1, 7168), (3, 1001), (5, 2048), (40, 6147), (300, 7168), (700, 6147), (2, 40032), (301, 40032),
                                           (2500, 512), (5000, 1001), (2, 33000)])
def test_norm_with_fp32_gamma(tokens, hidden, offset, quant, dtype):
    if quant == "mxfp8":
        hidden = hidden // 32 * 32
    g = gen(tokens, hidden, offset, 21)
    x, res = randn((tokens, hidden), g, dtype), randn((tokens, hidden), g, dtype)
    gamma = (1 + 0.2 * randn((hidden + offset,), g))[offset:]
    got = megamoe.rms_norm(x, gamma, 1e-6, residual=res, quant=quant, with_norm=True)
    check_norm(got, x, gamma, 1e-6, res, quant, True)
    # x's type and fp32 that hold the same values give the same bits
    same = gamma.to(dtype)
    a = megamoe.rms_norm(x, same, 1e-6, residual=res, quant=quant, with_norm=True)
    b = megamoe.rms_norm(x, same.float(), 1e-6, residual=res, quant=quant, with_norm=True)
    for u, v in zip(a, b):
        assert (u is None and v is None) or torch.equal(u.view(torch.uint8) if u.element_size() == 1 else u,
                                                        v.view(torch.uint8) if v.element_size() == 1 else v)
