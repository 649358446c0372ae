"""Block-scaled FP8 operators without a GPU: what the C entries refuse, the fakes' shapes, and
the 64-bit definitions against a loop over elements."""
import ctypes

import pytest
import torch

import fp8_block_ref as R
from helpers import load_lib

vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float


def _fn(name, args):
    f = getattr(load_lib(), name)
    f.restype, f.argtypes = ctypes.c_int, args
    return f


def _err():
    lib = load_lib()
    lib.w4a8_last_error.restype = ctypes.c_char_p
    return lib.w4a8_last_error().decode()


def test_act_quant_block_refusals():
    f = _fn("w4a8_act_quant_fp8_block", [vp, i32, i64, i64, vp, vp, vp])
    for a, msg in [((1, 3, 4, 128, 1, 1, None), "x_dtype"), ((1, 0, -1, 128, 1, 1, None), "bad sizes"),
                   ((1, 0, 4, 0, 1, 1, None), "bad sizes"), ((None, 0, 4, 128, 1, 1, None), "null")]:
        assert f(*a) == -1 and msg in _err()
    assert f(None, 0, 0, 128, None, None, None) == 0


def test_rms_norm_quant_refusals():
    f = _fn("w4a8_rms_norm_quant_fp8", [vp, vp, vp, i32, i32, f32, i64, i64, vp, vp, vp, vp, vp])
    ok = dict(x=1, r=None, w=1, xd=1, wd=1, eps=1e-6, M=4, H=128, q=1, s=1, ro=None, n=None, st=None)
    for change, msg in [(dict(xd=3), "x_dtype"), (dict(wd=2), "weight must have"), (dict(eps=-1.0), "eps"),
                        (dict(eps=float("nan")), "eps"), (dict(M=-1), "bad sizes"), (dict(H=0), "bad sizes"),
                        (dict(r=1), "go together"), (dict(ro=1), "go together"), (dict(x=None), "null")]:
        assert f(*{**ok, **change}.values()) == -1 and msg in _err()
    assert f(*{**ok, "M": 0}.values()) == 0


def test_fp8_gemm_refusals():
    f = _fn("w4a8_fp8_block_gemm", [vp] * 5 + [i32] + [i64] * 3 + [vp])
    for a, msg in [((1, 1, 1, 1, 1, 3, 4, 64, 128), "out_dtype"), ((1, 1, 1, 1, 1, 1, -4, 64, 128), "bad sizes"),
                   ((1, 1, 1, 1, 1, 1, 4, 0, 128), "bad sizes"), ((1, 1, 1, 1, 1, 1, 4, 64, 0), "bad sizes"),
                   ((1, 1, 1, 1, 1, 1, 1 << 31, 64, 128), "bad sizes"), ((1, None, 1, 1, 1, 1, 4, 64, 128), "null")]:
        assert f(*a, None) == -1 and msg in _err()
    assert f(None, None, None, None, None, 1, 0, 64, 128, None) == 0


@pytest.mark.parametrize("silu", [False, True])
def test_fp8_moe_refusals(silu):
    if silu:
        f = _fn("w4a8_fp8_block_moe_gemm1_silu", [vp] * 9 + [i64] * 7 + [vp])
        call = lambda p, T=8, E=2, N=128, K=128, P=32, k=2, bm=16: f(*p, *([1] * 2), T, E, N, K, P, k, bm, None)  # noqa: E731
    else:
        f = _fn("w4a8_fp8_block_moe_gemm", [vp] * 8 + [i32] + [i64] * 7 + [vp])
        call = lambda p, T=8, E=2, N=128, K=128, P=32, k=2, bm=16: f(*p, 1, 1, T, E, N, K, P, k, bm, None)  # noqa: E731
    p = [1] * 7
    for kw, msg in [(dict(bm=8), "block_m"), (dict(bm=48), "block_m"), (dict(bm=0), "block_m"), (dict(bm=192), "block_m"),
                    (dict(P=24), "divisible"), (dict(k=0), "top_k"), (dict(E=0), "bad sizes"), (dict(K=0), "bad sizes"),
                    (dict(T=-1), "bad sizes"), (dict(T=1 << 30, k=4), "top_k"), (dict(E=1 << 24, N=1 << 9), "2^31")]:
        assert call(p, **kw) == -1 and msg in _err(), kw
    assert call([1, 1, 1, 1, None, 1, 1]) == -1 and "P rows" in _err()  # T = 8 rows, P = 32
    assert call([1, 1, 1, 1, 1, None, 1]) == -1 and "null" in _err()
    assert call([None] * 7, T=0, P=0) == 0
    if silu:
        assert call(p, N=64) == -1 and "multiple of 128" in _err()


def test_fake_shapes():
    import w4a8_fp8_wmma as w4
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 300, dtype=torch.bfloat16, device="cuda")
        q, s = w4.act_quant_fp8_block(x)
        assert (q.shape, q.dtype, s.shape, s.dtype) == ((5, 300), torch.float8_e4m3fn, (5, 3), torch.float32)
        q, s, r, n = w4.rms_norm_quant_fp8(x, x[0], residual=x, with_normed=True)
        assert r.shape == n.shape == (5, 300) and r.dtype == n.dtype == torch.bfloat16
        assert w4.rms_norm_quant_fp8(x, x[0])[2:] == (None, None)
        w = torch.empty(4, 512, 300, dtype=torch.float8_e4m3fn, device="cuda")
        ws = torch.empty(4, 4, 3, device="cuda")
        o = w4.fp8_block_gemm(q, s, w[0], ws[0], out_dtype=torch.bfloat16)
        assert o.shape == (5, 512) and o.dtype == torch.bfloat16
        ids = torch.empty(48, dtype=torch.int32, device="cuda")
        o = w4.fp8_block_moe_gemm(q, s, w, ws, ids, ids[:3], ids[:1], 2, 16)
        assert o.shape == (48, 512) and o.dtype == torch.float16
        q, s = w4.fp8_block_moe_gemm1_silu(q, s, w, ws, ids, ids[:3], ids[:1], 2, 16)
        assert q.shape == (48, 256) and s.shape == (48, 2)


def test_cpu_tensors_refused():
    import w4a8_fp8_wmma as w4
    with pytest.raises((RuntimeError, NotImplementedError)):
        w4.act_quant_fp8_block(torch.zeros(2, 128))
    with pytest.raises((RuntimeError, NotImplementedError)):
        w4.fp8_block_gemm(torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(2, 1),
                          torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(1, 1))


def test_layer_needs_out_dtype_for_quantised_rows():
    from w4a8_fp8_wmma.fp8_block import fp8_block_m, run_fp8_block_moe
    z = torch.zeros(1)
    with pytest.raises(ValueError):
        run_fp8_block_moe(z, z, z, z, z, z, z, x_scales=z)
    assert [fp8_block_m(r, 256) for r in (8, 256, 2048, 2049, 8192, 8193, 1 << 20)] == [16, 16, 16, 32, 64, 128, 128]


def test_definitions_against_a_loop():
    g = torch.Generator().manual_seed(0)
    x, xs = R.quantise(torch.randn(3, 200, generator=g))
    w, ws = R.quantise(torch.randn(150, 200, generator=g), 128)
    out, S = R.product(x, xs, w, ws)
    for m, n in [(0, 0), (2, 149), (1, 127), (1, 128)]:
        t = sum(float(x[m, k]) * float(xs[m, k // 128]) * float(w[n, k]) * float(ws[n // 128, k // 128])
                for k in range(200))
        assert abs(t - float(out[m, n])) <= 1e-12 * float(S[m, n])
    ids = torch.tensor([[0, 2], [2, 3], [2, 0]])
    s, e, n = R.align(ids, 4, 16, spare=1)
    assert int(n) == 48 and e.tolist() == [0, 2, 3, -1] and s[:2].tolist() == [0, 5] and s[16:19].tolist() == [1, 2, 4]
    # a planted mistake in the scales of one block falls outside the derived bound
    wrong, _ = R.product(x, xs, w, ws * torch.tensor([[1.0, 1.01], [1.0, 1.0]]))
    with pytest.raises(AssertionError):
        R.check_out(wrong, out, S, 2, torch.float32)
