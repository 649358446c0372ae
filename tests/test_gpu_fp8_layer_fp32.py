"""The block-scaled MoE layer asked for an fp32 result: no step between may hold less than fp32 holds,
in range or in bits. Against 64 bits (tests/fp8_block_ref.py derives the bounds)."""
import pytest
import torch

import fp8_block_ref as R

pytestmark = pytest.mark.gpu
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def w4():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import w4a8_fp8_wmma
    return w4a8_fp8_wmma


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _layer(g, E, H, I, loud):
    w1, s1 = R.quantise(_randn(g, E, 2 * I, H) * H ** -0.5, 128)
    w2, s2 = R.quantise(_randn(g, E, H, I) * I ** -0.5, 128)
    return w1, w2, s1, s2 * loud


def _definition(q, s, w1, w2, s1, s2, ids, tw, k):
    """The layer in 64 bits, and how far fp32 steps and the quantisation before down may be off."""
    T, E, H, I = q.shape[0], w1.shape[0], w2.shape[1], w2.shape[2]
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    tol, size = torch.zeros_like(want), torch.zeros_like(want)
    for j in range(k):
        for e in range(E):
            at = (ids[:, j] == e).nonzero().reshape(-1)
            if not at.numel():
                continue
            o, S = R.product(q[at], s[at], w1[e], s1[e])
            h, dh = R.silu_mul(o, S, R.sum_error(R.blocks(q.shape[1])))
            f = R.spread_cols(h.reshape(len(at), -1, 128).abs().amax(2).clamp_min(R.FLOOR) / 448.0, I)
            dh = dh + torch.maximum(h.abs() * 2.0 ** -4, f * 2.0 ** -10) * 1.01
            b = w2[e].double() * R.spread_w(s2[e].double(), H, I)
            d = h @ b.T
            dd = dh @ b.abs().T + R.sum_error(R.blocks(I)) * (h.abs() @ b.abs().T)
            w = tw[at, j, None].double()
            want[at] += w * d
            tol[at] += w * dd
            size[at] += w * (d.abs() + dd)
    return want, tol * (1 + 1e-6) + (k + 1) * 2.0 ** -24 * size


@pytest.mark.parametrize("loud", [1.0, 1e7, 1e-9])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 256, 128), (32, 16, 4, 512, 256), (700, 8, 2, 384, 256),
                                       (4100, 4, 1, 256, 128)])
def test_fp32_layer(w4, T, E, k, H, I, loud):
    """Down rows past fp16's range (1e7), in it, and below it (1e-9)."""
    from w4a8_fp8_wmma.fp8_block import run_fp8_block_moe
    g = torch.Generator(device="cuda").manual_seed(T + H)
    x = _randn(g, T, H)
    w1, w2, s1, s2 = _layer(g, E, H, I, loud)
    ids, tw, _ = w4.route_topk(_randn(g, T, E), k)
    y = run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids)
    assert y.dtype == FP32 and y.shape == (T, H)
    q, s = w4.act_quant_fp8_block(x)
    want, tol = _definition(q, s, w1, w2, s1, s2, ids, tw, k)
    assert bool(((y.double() - want).abs() <= tol).all())
    if loud == 1e7:
        assert float(want.abs().max()) > 65504
    # from bf16 rows with an fp32 result, and as 64 bits
    z = run_fp8_block_moe(x.bfloat16(), w1, w2, s1, s2, tw, ids, out_dtype=FP32)
    assert z.dtype == FP32 and bool(z.isfinite().all())
    assert torch.equal(run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids, out_dtype=torch.float64), y.double())


def test_fp32_rows_keep_their_bits(w4):
    """One expert with weight 1: the layer's result is the down product, bit for bit."""
    from w4a8_fp8_wmma.fp8_block import fp8_block_m, run_fp8_block_moe
    g = torch.Generator(device="cuda").manual_seed(3)
    T, H, I = 40, 256, 256
    w1, w2, s1, s2 = _layer(g, 1, H, I, 1.0)
    x = _randn(g, T, H)
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    y = run_fp8_block_moe(x, w1, w2, s1, s2, torch.ones(T, 1, device="cuda"), ids)
    bm = fp8_block_m(T, 1)
    s, e, n = w4.moe_align_block_size(ids, bm, 1)
    h, hs = w4.fp8_block_moe_gemm1_silu(*w4.act_quant_fp8_block(x), w1, s1, s, e, n, 1, bm)
    rows = w4.fp8_block_moe_gemm(h, hs, w2, s2, None, e, n, 1, bm, out_dtype=FP32)
    assert torch.equal(y, rows[:T])


def test_layer_of_one_chunk_past_65535_tokens(w4, monkeypatch):
    """With chunking switched off; the first and the last tokens against the definition."""
    from w4a8_fp8_wmma import fp8_block
    monkeypatch.setattr(fp8_block, "APPLY_CHUNK", 0)
    g = torch.Generator(device="cuda").manual_seed(8)
    T, E, k, H, I = 70000, 4, 2, 128, 128
    x = _randn(g, T, H)
    w1, w2, s1, s2 = _layer(g, E, H, I, 1.0)
    ids, tw, _ = w4.route_topk(_randn(g, T, E), k)
    y = fp8_block.run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids)
    assert bool(y.isfinite().all())
    some = torch.cat([torch.arange(60), torch.arange(T - 60, T)]).cuda()
    q, s = w4.act_quant_fp8_block(x[some])
    want, tol = _definition(q, s, w1, w2, s1, s2, ids[some], tw[some], k)
    assert bool(((y[some].double() - want).abs() <= tol).all())
