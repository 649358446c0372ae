"""The block-scaled FP8 tests that compare with a definition, run again with checks that a NaN cannot
pass (fp8_strict) and on operands of which some scale blocks are zero."""
import pytest
import torch

import fp8_block_ref as R
import fp8_strict
import test_gpu_fp8_block as base

pytestmark = pytest.mark.gpu
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


def _matrix(gen, *shape, row_block):
    """base's random values and scales, a tenth of the scales zero."""
    q = R.e4m3(shape, gen, "cuda")
    rows = (shape[-2] + row_block - 1) // row_block
    size = shape[:-2] + (rows, R.blocks(shape[-1]))
    s = torch.rand(size, generator=gen, device="cuda") * 2e-3 + 1e-5
    return q, torch.where(torch.rand(size, generator=gen, device="cuda") < 0.1, 0.0, s)


@pytest.fixture
def w4(monkeypatch):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import w4a8_fp8_wmma
    monkeypatch.setattr(R, "check_out", fp8_strict.check_out)
    monkeypatch.setattr(R, "check_quant", fp8_strict.check_quant)
    monkeypatch.setattr(base, "_matrix", _matrix)
    return w4a8_fp8_wmma


def test_the_matrices_have_zero_scales(w4):
    _, s = base._matrix(base._gen(1), 4, 256, 512, row_block=128)
    assert bool((s == 0).any()) and bool((s > 0).any())


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("M,N,K", base.GEMMS)
def test_dense(w4, M, N, K, dtype):
    base.test_fp8_block_gemm(w4, M, N, K, dtype)


@pytest.mark.parametrize("off", [1, 8, 16])
def test_dense_misaligned_views(w4, off):
    base.test_fp8_block_gemm_misaligned_views(w4, off)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("T,E,k,N,K,bm", base.MOES)
def test_grouped(w4, T, E, k, N, K, bm, dtype):
    base.test_fp8_block_moe_gemm(w4, T, E, k, N, K, bm, dtype)


@pytest.mark.parametrize("T,E,k,N,K,bm", [(1, 4, 2, 256, 128, 16), (5, 8, 3, 512, 272, 16), (40, 8, 2, 256, 512, 32),
                                          (100, 6, 4, 1280, 144, 64), (300, 5, 3, 768, 1024, 128),
                                          (2, 64, 8, 1024, 2048, 16), (33, 16, 5, 512, 100, 32)])
def test_gate_up(w4, T, E, k, N, K, bm):
    base.test_fp8_block_moe_gemm1_silu(w4, T, E, k, N, K, bm)


@pytest.mark.parametrize("bm,T", [(16, 6), (128, 150)])
def test_rows_past_the_last(w4, bm, T):
    base.test_rows_past_the_last_are_left(w4, bm, T)


def test_many_tiles(w4):
    base.test_many_tiles_with_a_short_last_block(w4)


def test_offsets_past_32_bits(w4):
    base.test_offsets_past_32_bits(w4)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("M,K", base.SHAPES)
def test_quantisation(w4, M, K, dtype):
    base.test_act_quant_block_bit_exact(w4, M, K, dtype)


@pytest.mark.parametrize("dtype,wdtype", [(FP16, FP16), (BF16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("residual,normed", [(False, False), (True, True)])
@pytest.mark.parametrize("M,H", [(1, 128), (3, 127), (5, 1000), (33, 2048), (2, 40000)])
def test_norm(w4, M, H, residual, normed, dtype, wdtype):
    base.test_rms_norm_quant(w4, M, H, residual, normed, dtype, wdtype)


@pytest.mark.parametrize("K", [128, 512, 1024, 200])
@pytest.mark.parametrize("M,N", [(1, 256), (33, 300), (300, 2048), (2500, 2100)])
def test_zero_scales_give_zeros(w4, M, N, K):
    """Rows, and blocks of weight rows, all of whose scales are zero are zeros; so are the SiLU form's."""
    g = base._gen(M + N + K)
    x, xs = base._matrix(g, M, K, row_block=1)
    w, ws = base._matrix(g, N, K, row_block=128)
    xs[M // 2], ws[1] = 0.0, 0.0
    out = w4.fp8_block_gemm(x, xs, w, ws, out_dtype=FP32)
    want, S = R.product(x, xs, w, ws)
    R.check_out(out, want, S, R.blocks(K), FP32)
    assert bool((out[M // 2] == 0).all()) and bool((out[:, 128:256] == 0).all())
