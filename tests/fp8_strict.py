"""fp8_block_ref's checks in a form that a NaN cannot pass.

fp8_block_ref collects `(got - want).abs() > tol`, which is False for a NaN: an output that is not a
number counts as near. Here an output has to be shown near. What may round to an infinity (the definition
within its bound of the type's largest value) may be one, of the right sign."""
from __future__ import annotations

import torch

import fp8_block_ref as R

_check_quant = R.check_quant  # a test may put the one below in its place


def check_out(got, want, S, G, dtype):
    err = R.sum_error(G) * S
    tol = err + R.HALF[dtype] * (want.abs() + err) + R.TINY[dtype]
    near = (got.double() - want).abs() <= tol
    over = (want.abs() + tol >= torch.finfo(dtype).max) & got.isinf() & (torch.signbit(got) == torch.signbit(want))
    ok = near | over
    assert bool(ok.all()), f"{int((~ok).sum())} outputs not within the derived bound"


def check_quant(q, s, y, dy):
    _check_quant(q, s, y, dy)
    c = y.shape[1]
    f = R.spread_cols(s.double(), c)
    tol = torch.clamp_min((y / f).abs() * 2.0 ** -4, 2.0 ** -10) * (1 + 2.0 ** -9) * f + dy * 1.0625 + 2.0 ** -22 * y.abs()
    ok = (q.double() * f - y).abs() <= tol
    assert bool(ok.all()), f"{int((~ok).sum())} quantised values not within the derived bound"
