"""The strict checks fail on one planted NaN, infinity or wrong value, and pass on what is right."""
import pytest
import torch

import fp8_block_ref as R
import fp8_strict


def _product():
    g = torch.Generator().manual_seed(0)
    x, xs = R.quantise(torch.randn(4, 200, generator=g))
    w, ws = R.quantise(torch.randn(150, 200, generator=g), 128)
    return R.product(x, xs, w, ws)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_outputs(dtype):
    want, S = _product()
    good = want.to(dtype)
    fp8_strict.check_out(good, want, S, 2, dtype)
    for value in (float("nan"), float("inf"), float("-inf"), float(good[2, 7]) + 1.0):
        bad = good.clone()
        bad[2, 7] = value
        with pytest.raises(AssertionError):
            fp8_strict.check_out(bad, want, S, 2, dtype)
    R.check_out(torch.full_like(good, float("nan")), want, S, 2, dtype)  # the hole that this closes


def test_outputs_past_the_largest():
    want, S = _product()
    want = want.clone()
    want[1, 3], want[1, 4] = 70000.0, -70000.0
    fp8_strict.check_out(want.half(), want, S, 2, torch.float16)
    for a, b in ((float("nan"), float("-inf")), (float("-inf"), float("-inf")), (float("inf"), 65504.0)):
        bad = want.half()
        bad[1, 3], bad[1, 4] = a, b
        with pytest.raises(AssertionError):
            fp8_strict.check_out(bad, want, S, 2, torch.float16)


def test_quantised():
    y = torch.randn(3, 300, generator=torch.Generator().manual_seed(1)).double()
    q, s = R.quantise(y.float())
    zero = torch.zeros_like(y)
    fp8_strict.check_quant(q, s, y, zero)
    bad = q.clone()
    bad.view(torch.uint8)[1, 200] = 0x7F
    with pytest.raises(AssertionError):
        fp8_strict.check_quant(bad, s, y, zero)
    R.check_quant(bad, s, y, zero)  # the hole that this closes
    for value in (float("nan"), float("inf")):
        off = s.clone()
        off[2, 1] = value
        with pytest.raises(AssertionError):
            fp8_strict.check_quant(q, off, y, zero)
