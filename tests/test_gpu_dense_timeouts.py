"""Bounded waits of the int8 products that run out: the launch ends within its budget,
int8_check raises, and the next call is right again. Each test makes a wait run out on a load
that is left out (mm_int8_withhold), with a short budget; no kernel waits without a bound."""

import time

import pytest
import torch

import megamoe
from megamoe import _lib

pytestmark = pytest.mark.gpu

BUDGET_US = 5000
# (tokens, features, depth, ranks): one CTA a tile; parts sent to, and read by, eight CTAs; pairs
FORMS = [(3, 40000, 1024, (0,)), (4, 300, 7168, (0, 1, 7)), (30, 130, 4096, (0, 3)), (80, 300, 7168, (0, 5)), (128, 256, 4096, (7,)),
         (600, 1000, 2048, (0, 1)), (4096, 4096, 512, (0, 1))]


def operands(tokens, features, depth):
    g = torch.Generator(device="cuda").manual_seed(tokens + features)
    x, w = (torch.randint(-127, 128, (n, depth), dtype=torch.int8, device="cuda", generator=g) for n in (tokens, features))
    return x, torch.full((tokens,), 2.0 ** -8, device="cuda"), w, torch.full((features,), 2.0 ** -8, device="cuda")


@pytest.fixture(autouse=True)
def settings():
    megamoe.int8_check()
    megamoe.int8_set_wait_budget(BUDGET_US)
    yield
    _lib.lib().mm_int8_withhold(0, 0)
    megamoe.int8_set_wait_budget(1_500_000)
    torch.cuda.synchronize()
    try:
        megamoe.int8_check()
    except _lib.DeviceTimeoutError:
        pass


@pytest.mark.parametrize("tokens,features,depth,ranks", FORMS)
def test_a_wait_runs_out_and_the_next_call_is_right(tokens, features, depth, ranks):
    call = operands(tokens, features, depth)
    want = megamoe.int8_linear(*call)
    megamoe.int8_check()
    for rank in ranks:
        _lib.lib().mm_int8_withhold(rank, 1)
        t0 = time.perf_counter()
        megamoe.int8_linear(*call)
        with pytest.raises(_lib.DeviceTimeoutError):
            megamoe.int8_check()
        # the budget and the teardown's drains (20 ms at most each), far below the default of 1.5 s
        assert time.perf_counter() - t0 < 1.0
        got = megamoe.int8_linear(*call)
        megamoe.int8_check()
        assert torch.equal(got, want)


def test_a_wait_of_the_block_runs_out():
    x, xs, w13, s13 = operands(20, 1024, 512)
    _, _, w2, s2 = operands(1, 512, 512)
    want = megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
    for launches in (1, 2):
        _lib.lib().mm_int8_withhold(0, launches)
        megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
        with pytest.raises(_lib.DeviceTimeoutError):
            megamoe.int8_check()
        assert torch.equal(megamoe.int8_ffn(x, xs, w13, s13, w2, s2), want)
        megamoe.int8_check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,features,depth,ranks", FORMS)
def test_what_a_failed_launch_could_not_finish_is_nan(tokens, features, depth, ranks, dtype):
    """No value of a launch whose wait ran out looks valid without being right: the CTAs that
    share a tile's depth all know of it, and what none of them could finish is NaN."""
    call = operands(tokens, features, depth)
    want = megamoe.int8_linear(*call, out_dtype=dtype)
    for rank in ranks:
        got = torch.full_like(want, 7.0)
        _lib.lib().mm_int8_withhold(rank, 1)
        megamoe.int8_linear(*call, out_dtype=dtype, out=got)
        with pytest.raises(_lib.DeviceTimeoutError):
            megamoe.int8_check()
        assert bool(got.isnan().any())
        assert bool((got.isnan() | (got == want)).all()), int((~(got.isnan() | (got == want))).sum())


@pytest.mark.parametrize("tokens", [3, 20, 100, 600])
def test_a_failed_product_of_the_block_reaches_its_rows(tokens):
    """The gated product's rows are a workspace: what it could not finish is not taken from the
    call before."""
    x, xs, w13, s13 = operands(tokens, 1024, 2048)
    _, _, w2, s2 = operands(1, 2048, 512)
    want = megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
    megamoe.int8_ffn(x.flip(0).contiguous(), xs * 0.5, w13, s13, w2, s2)
    _lib.lib().mm_int8_withhold(0, 1)
    got = megamoe.int8_ffn(x, xs, w13, s13, w2, s2)
    with pytest.raises(_lib.DeviceTimeoutError):
        megamoe.int8_check()
    assert bool(got.isnan().any()) and bool((got.isnan() | (got == want)).all())


@pytest.mark.parametrize("tokens,features,depth", [(4, 300, 7168), (100, 300, 7168), (600, 1000, 2048)])
def test_a_launch_keeps_its_budget_after_another_failed(tokens, features, depth):
    """The word that int8_check reads belongs to the device: a wait that ran out in one launch,
    unread, is no reason for another launch's waits to give up."""
    call = operands(tokens, features, depth)
    want = megamoe.int8_linear(*call)
    _lib.lib().mm_int8_withhold(0, 1)
    megamoe.int8_linear(*operands(4, 300, 7168))
    torch.cuda.synchronize()
    megamoe.int8_set_wait_budget(400_000)
    _lib.lib().mm_int8_withhold(0, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    t0 = time.perf_counter()
    with torch.cuda.stream(side):
        megamoe.int8_linear(*call)
    torch.cuda.synchronize()
    assert 0.4 <= time.perf_counter() - t0 < 2.0
    assert torch.equal(megamoe.int8_linear(*call), want)
    with pytest.raises(_lib.DeviceTimeoutError):
        megamoe.int8_check()
    megamoe.int8_check()
