"""Zeros of the norm that quantises its output keep their sign, in the vectorised kernel (H a multiple
of 8, aligned rows) as in the general one: the byte is e4m3(y / scale), and y may be -0."""
import pytest
import torch

import fp8_block_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,off", [(8, 0), (128, 0), (128, 1), (1000, 0), (1001, 0), (2048, 0), (5120, 0), (16392, 0)])
def test_zeros_keep_their_sign(H, off, dtype):
    import w4a8_fp8_wmma as w4
    g = torch.Generator(device="cuda").manual_seed(H + off)
    x = torch.randn(5, H, generator=g, device="cuda")
    x[torch.rand(5, H, generator=g, device="cuda") < 0.2] = -0.0
    x[torch.rand(5, H, generator=g, device="cuda") < 0.2] = 0.0
    x[3] = -0.0
    w = torch.randn(H, generator=g, device="cuda")
    w[torch.rand(H, generator=g, device="cuda") < 0.2] = 0.0
    w[torch.rand(H, generator=g, device="cuda") < 0.1] = -0.0
    base = torch.empty(5 * H + off, dtype=dtype, device="cuda")
    rows = base[off:].view(5, H)
    rows.copy_(x.to(dtype))
    w = w.to(dtype)
    q, s, _, n = w4.rms_norm_quant_fp8(rows, w, 1e-6, with_normed=True)
    y = rows.float() * w.float()  # the norm's factor is positive
    bits = q.view(torch.uint8)
    zero = y == 0
    assert bool(zero.any()) and bool((~zero).any())
    assert bool(((bits[zero] & 0x7F) == 0).all())
    assert torch.equal((bits >> 7).bool(), torch.signbit(y))
    assert torch.equal(torch.signbit(n), torch.signbit(y))
    assert bool((s[3] == (torch.tensor(R.FLOOR) / 448.0).cuda()).all())
