"""The gate_up product's SiLU at gates far from zero, where silu(g) * u lives by up alone, and at gates
that are not numbers. Gates and ups are exact products (one value a row, scales that are powers of two),
so all of a result's error is the epilogue's.

Bound: exp(-|g|) 4 units of 2^-24 and 1.25 |g| (its argument's rounding, and log2(e)'s), the sum, the
reciprocal of two sums' product, and four products, 12 units: (16 + 1.25 |g|) 2^-24 of the value. Where
exp(-|g|) or silu is subnormal, each of them loses up to 2^-149: (|g| + 1) |u| 2^-149, with |g| up to
110, from where on exp(-|g|) is 0 and so is every result."""
import pytest
import torch

import fp8_block_ref as R

pytestmark = pytest.mark.gpu

# (e4m3 value, power of two of its block scale)
GATES = [(-5.5, 0), (-14, 0), (-30, 0), (-44, 0), (-52, 0), (-80, 0), (-88, 0), (-96, 0), (-104, 0), (-120, 0),
         (-240, 12), (-256, 54), (-448, 100), (5.5, 0), (30, 0), (88, 0), (104, 0), (448, 12)]


@pytest.fixture(scope="module")
def w4():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import w4a8_fp8_wmma
    return w4a8_fp8_wmma


def _inputs(K, up_pow, gates):
    """x (3, K) with 1, 0.5 and -0.25 in the first column, one 128-output block per gate."""
    gen = torch.Generator().manual_seed(K + up_pow)
    inter = 128 * len(gates)
    x = torch.zeros(3, K)
    x[:, 0] = torch.tensor([1.0, 0.5, -0.25])
    w = torch.zeros(1, 2 * inter, K)
    ups = torch.randint(8, 57, (inter,), generator=gen) * 8.0  # 64 to 448, some of them rounded by e4m3
    w[0, inter:, 0] = torch.where(torch.rand(inter, generator=gen) < 0.5, -ups, ups)
    ws = torch.ones(1, 2 * len(gates), R.blocks(K))
    for b, (v, p) in enumerate(gates):
        w[0, b * 128:(b + 1) * 128, 0] = v
        ws[0, b] = 2.0 ** p
        ws[0, len(gates) + b] = 2.0 ** up_pow
    as8 = lambda t: t.to(torch.float8_e4m3fn).cuda()  # noqa: E731
    return as8(x), torch.ones(3, R.blocks(K)).cuda(), as8(w), ws.cuda()


def _routing(bm):
    s = torch.full((bm,), 3, dtype=torch.int32)
    s[:3] = torch.tensor([2, 0, 1])
    return s.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), torch.tensor([bm], dtype=torch.int32).cuda()


@pytest.mark.parametrize("up_pow", [0, 24, 90, 100])
@pytest.mark.parametrize("bm", [16, 64, 128])
@pytest.mark.parametrize("K", [128, 512, 1024, 100])
def test_far_gates(w4, K, bm, up_pow):
    # the blocks whose results fp32 holds (a token may turn a gate's sign and quarter it)
    gates = [(v, p) for v, p in GATES if abs(v) * 2.0 ** p * 448 * 2.0 ** up_pow < 2.0 ** 126 or
             (v < 0 and p < 13)]
    x, xs, w, ws = _inputs(K, up_pow, gates)
    s, e, n = _routing(bm)
    q, qs = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, 1, bm)
    inter = 128 * len(gates)
    first = x[s[:3].long(), 0].double()
    full = first[:, None] * w[0, :, 0].double() * ws[0, :, 0].double().repeat_interleave(128)
    g, u = full[:, :inter], full[:, inter:]
    h = g / (1 + torch.exp(-g)) * u
    dh = (16 + 1.25 * g.abs()) * 2.0 ** -24 * h.abs() + (g.abs().clamp_max(110) + 1) * u.abs() * 2.0 ** -149
    assert bool(q.float().isfinite().all()) and bool(qs.isfinite().all())
    R.check_quant(q[:3], qs[:3], h, dh)
    assert bool((q[3:].view(torch.uint8) == 0).all())


@pytest.mark.parametrize("bm", [16, 128])
@pytest.mark.parametrize("K", [128, 1024, 100])
def test_a_nan_gate_stays_where_it_is(w4, K, bm):
    x, xs, w, ws = _inputs(K, 0, [(5.5, 0), (-14, 0)])
    s, e, n = _routing(bm)
    col = torch.tensor([0, 1, 66, 127, 130, 255])
    w.view(torch.uint8)[0, 256 + col, 0] = 0  # their up values: nothing there enters a maximum
    q0, s0 = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, 1, bm)
    w.view(torch.uint8)[0, col, 0] = 0x7F
    q1, s1 = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, 1, bm)
    b0, b1 = q0.view(torch.uint8)[:3], q1.view(torch.uint8)[:3]
    nan = torch.zeros(256, dtype=torch.bool, device="cuda")
    nan[col] = True
    assert bool(((b1[:, nan] & 0x7F) == 0x7F).all())
    assert torch.equal(b1[:, ~nan], b0[:, ~nan]) and torch.equal(s1, s0)


@pytest.mark.parametrize("bm", [16, 128])
@pytest.mark.parametrize("K", [128, 100])
def test_infinite_gates(w4, K, bm):
    """silu(-inf) is -inf / inf, not a number, and silu(inf) infinite, in every kernel."""
    x, xs, w, ws = _inputs(K, 0, [(-1, 0), (1, 0), (5.5, 0)])
    s, e, n = _routing(bm)
    ws[0, :2] = float("inf")
    q, qs = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, 1, bm)
    bits = q.view(torch.uint8) & 0x7F
    row = (s[:3] == 0).nonzero().item()  # the token of x = 1
    assert bool((bits[row, :256] == 0x7F).all()) and bool((bits[row, 256:] != 0x7F).all())
    assert bool(qs[row, 0].isfinite()) and bool(qs[row, 1].isinf()) and bool(qs[row, 2].isfinite())
