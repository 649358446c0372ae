"""The block-scaled FP8 operators on the GPU against their 64-bit definitions
(tests/fp8_block_ref.py, which also derives the bounds)."""
import ctypes

import pytest
import torch

import fp8_block_ref as R
from helpers import load_lib

pytestmark = pytest.mark.gpu
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def w4():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import w4a8_fp8_wmma
    return w4a8_fp8_wmma


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=FP32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _matrix(gen, *shape, row_block):
    """Random e4m3 values with random positive scales, and some all-zero scale blocks."""
    q = R.e4m3(shape, gen, "cuda")
    rows = (shape[-2] + row_block - 1) // row_block
    s = torch.rand(shape[:-2] + (rows, R.blocks(shape[-1])), generator=gen, device="cuda") * 2e-3 + 1e-5
    return q, s


# ------------------------------------------------------------------ quantisation ------------
SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (2, 1000), (33, 1024), (7, 2056), (64, 4096),
          (257, 640), (1, 8192), (2, 20000)]


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("M,K", SHAPES)
def test_act_quant_block_bit_exact(w4, M, K, dtype):
    x = _randn(_gen(M * 7 + K), M, K, dtype=dtype) * 3
    if M > 1:
        x[0] = 0
        x[1, : K // 2] *= 1e-5
        x[-1, K - 1] = 60000.0
    q, s = w4.act_quant_fp8_block(x)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (M, K) and s.shape == (M, R.blocks(K))
    rq, rs = R.quantise(x.float())  # IEEE divides: equal to the last bit
    assert torch.equal(s, rs)
    assert torch.equal(q.view(torch.uint8), rq.view(torch.uint8))
    R.check_quant(q, s, x.double(), torch.zeros_like(x, dtype=torch.float64))


def test_act_quant_block_nan_and_inf(w4):
    x = _randn(_gen(1), 4, 384, dtype=FP16)
    clean = x.clone()
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    q, s = w4.act_quant_fp8_block(x)
    q0, s0 = w4.act_quant_fp8_block(clean)
    bits, bits0 = q.view(torch.uint8), q0.view(torch.uint8)
    assert torch.equal(bits[0], bits0[0]) and torch.equal(bits[3], bits0[3])
    assert int(bits[1, 5]) & 0x7F == 0x7F and torch.isfinite(s[1]).all()
    assert torch.isfinite(q[1, 128:].float()).all()
    assert torch.isinf(s[2, 1]) and torch.equal(s[2, [0, 2]], s0[2, [0, 2]])


def test_act_quant_block_misaligned_view(w4):
    base = _randn(_gen(2), 9 * 256 + 1, dtype=FP16)
    x = base[1:].view(9, 256)  # rows start 2 bytes off a 16-byte boundary
    q, s = w4.act_quant_fp8_block(x)
    rq, rs = R.quantise(x.float())
    assert torch.equal(s, rs) and torch.equal(q.view(torch.uint8), rq.view(torch.uint8))


@pytest.mark.parametrize("dtype,wdtype", [(FP16, FP16), (BF16, BF16), (BF16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("residual,normed", [(False, False), (True, True), (True, False)])
@pytest.mark.parametrize("M,H", [(1, 128), (3, 127), (5, 1000), (33, 2048), (4, 4096), (2, 5120),
                                 (3, 8192), (1, 1), (2, 40000), (130, 1536)])
def test_rms_norm_quant(w4, M, H, residual, normed, dtype, wdtype):
    g = _gen(M * 31 + H)
    x = _randn(g, M, H, dtype=dtype)
    w = (1 + 0.3 * _randn(g, H)).to(wdtype)
    r = _randn(g, M, H, dtype=dtype) * 4 if residual else None
    eps = 1e-5
    q, s, res, n = w4.rms_norm_quant_fp8(x, w, eps, residual=r, with_normed=normed)
    h = x if r is None else (x.float() + r.float()).to(dtype)
    if residual:
        assert torch.equal(res, h)
    else:
        assert res is None
    d = h.double()
    y = d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * w.double()
    # sum of H squares in chains of at most H / 32 + 16 additions (halved by the root), the
    # reciprocal root 4 units of 2^-24, three products
    rel = ((H / 32 + 16) / 2 + 8) * 2.0 ** -24
    dy = rel * y.abs()
    R.check_quant(q, s, y, dy)
    if normed:
        tol = dy + R.HALF[dtype] * (y.abs() + dy) + R.TINY[dtype]
        assert bool(((n.double() - y).abs() <= tol).all())
    else:
        assert n is None


def test_rms_norm_quant_edges(w4):
    x = torch.zeros(3, 256, device="cuda", dtype=BF16)
    w = torch.ones(256, device="cuda", dtype=BF16)
    x[1] = 3.0
    x[2, 7] = float("nan")
    q, s, _, n = w4.rms_norm_quant_fp8(x, w, 1e-6, with_normed=True)
    assert bool((q[0].float() == 0).all()) and bool((n[0] == 0).all())
    assert torch.equal(n[1].float(), torch.ones(256, device="cuda"))
    assert bool(((q[2].view(torch.uint8) & 0x7F) == 0x7F).all()) and bool(n[2].isnan().all())
    q, s, res, n = w4.rms_norm_quant_fp8(x[:0], w, 1e-6, residual=x[:0], with_normed=True)
    assert q.shape == (0, 256) and s.shape == (0, 2) and res.shape == (0, 256) and n.shape == (0, 256)


def test_quantisers_take_strided_rows(w4):
    g = _gen(10)
    wide = _randn(g, 6, 3 * 256, dtype=BF16)
    x, r, w = wide[:, 256:512], wide[:, 512:], _randn(g, 512, dtype=BF16)[::2]
    for a, b in zip(w4.act_quant_fp8_block(x), w4.act_quant_fp8_block(x.contiguous())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    ours = w4.rms_norm_quant_fp8(x, w, 1e-6, residual=r, with_normed=True)
    ref = w4.rms_norm_quant_fp8(x.contiguous(), w.contiguous(), 1e-6, residual=r.contiguous(), with_normed=True)
    for a, b in zip(ours, ref):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_rms_norm_quant_residual_in_place(w4):
    """The C entry may be given the residual itself as the new residual."""
    g = _gen(9)
    for H in (2048, 1000, 1001):
        x, r = _randn(g, 17, H, dtype=BF16), _randn(g, 17, H, dtype=BF16)
        w = _randn(g, H, dtype=BF16)
        q, s, res, _ = w4.rms_norm_quant_fp8(x, w, 1e-6, residual=r)
        q2, s2 = torch.empty_like(q), torch.empty_like(s)
        f = load_lib().w4a8_rms_norm_quant_fp8
        f.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int32] * 2 + [ctypes.c_float] + \
            [ctypes.c_int64] * 2 + [ctypes.c_void_p] * 5
        assert f(x.data_ptr(), r.data_ptr(), w.data_ptr(), 2, 2, 1e-6, 17, H, q2.data_ptr(),
                 s2.data_ptr(), r.data_ptr(), None, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(r, res) and torch.equal(s, s2)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))


# ------------------------------------------------------------------ dense product -----------
GEMMS = [(1, 1, 16), (1, 128, 128), (3, 129, 144), (16, 256, 512), (17, 33, 7), (128, 256, 384),
         (129, 257, 1040), (200, 1000, 656), (64, 512, 2048), (1, 4096, 2048), (300, 384, 200),
         (2, 8192, 128), (1000, 640, 1152), (513, 2048, 272), (5, 136, 8192), (33, 2048, 4096),
         (260, 260, 2064), (2500, 2100, 400), (2432, 2048, 256), (1281, 4001, 144),
         (130, 19000, 256), (100, 38000, 128), (385, 12800, 384)]


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("M,N,K", GEMMS)
def test_fp8_block_gemm(w4, M, N, K, dtype):
    g = _gen(M + N + K)
    x, xs = _matrix(g, M, K, row_block=1)
    w, ws = _matrix(g, N, K, row_block=128)
    out = w4.fp8_block_gemm(x, xs, w, ws, out_dtype=dtype)
    assert out.shape == (M, N) and out.dtype == dtype
    want, S = R.product(x, xs, w, ws)
    R.check_out(out, want, S, R.blocks(K), dtype)
    again = w4.fp8_block_gemm(x.view(torch.uint8), xs, w.view(torch.uint8), ws, out_dtype=dtype)
    assert torch.equal(out, again)  # same bytes, same order of sums


@pytest.mark.parametrize("K", [256, 200])
def test_fp8_block_gemm_nan_stays_in_its_row(w4, K):
    g = _gen(3)
    x, xs = _matrix(g, 40, K, row_block=1)
    w, ws = _matrix(g, 200, K, row_block=128)
    clean = w4.fp8_block_gemm(x, xs, w, ws)
    x.view(torch.uint8)[7, 3] = 0x7F
    xs[21, 0] = float("inf")
    out = w4.fp8_block_gemm(x, xs, w, ws)
    keep = [r for r in range(40) if r not in (7, 21)]
    assert torch.equal(out[keep], clean[keep])
    assert bool(out[7].isnan().all()) and not bool(out[21].isfinite().any())


@pytest.mark.parametrize("off", [1, 8, 16])
def test_fp8_block_gemm_misaligned_views(w4, off):
    g = _gen(4)
    M, N, K = 70, 300, 256
    xb, wb = R.e4m3((M * K + 64,), g, "cuda"), R.e4m3((N * K + 64,), g, "cuda")
    x, w = xb[off:off + M * K].view(M, K), wb[off:off + N * K].view(N, K)
    _, xs = _matrix(g, M, K, row_block=1)
    _, ws = _matrix(g, N, K, row_block=128)
    want, S = R.product(x, xs, w, ws)
    R.check_out(w4.fp8_block_gemm(x, xs, w, ws), want, S, 2, FP16)


def test_fp8_block_gemm_empty(w4):
    x = torch.empty(0, 256, dtype=torch.float8_e4m3fn, device="cuda")
    w = torch.zeros(64, 256, dtype=torch.uint8, device="cuda")
    out = w4.fp8_block_gemm(x, torch.empty(0, 2, device="cuda"), w, torch.zeros(1, 2, device="cuda"))
    assert out.shape == (0, 64)


# ------------------------------------------------------------------ grouped products --------
# (T, E, top_k, N, K, block_m)
MOES = [(1, 4, 2, 256, 128, 16), (5, 8, 3, 264, 272, 16), (40, 8, 2, 384, 512, 32),
        (100, 6, 4, 1000, 144, 64), (300, 5, 3, 256, 1024, 128), (64, 3, 2, 128, 256, 256),
        (2, 64, 8, 512, 2048, 16), (700, 4, 2, 640, 384, 128), (33, 16, 5, 31, 100, 32)]


def _routing(T, E, k, bm, seed, spare=2, skip=None):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)])
    if skip is not None:  # one expert gets no rows
        ids = torch.where(ids == skip, (skip + 1) % E, ids)
    s, e, n = R.align(ids, E, bm, spare)
    return s.cuda(), e.cuda(), n.cuda()


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32])
@pytest.mark.parametrize("T,E,k,N,K,bm", MOES)
def test_fp8_block_moe_gemm(w4, T, E, k, N, K, bm, dtype):
    g = _gen(T + N + K)
    x, xs = _matrix(g, T, K, row_block=1)
    w, ws = _matrix(g, E, N, K, row_block=128)
    s, e, n = _routing(T, E, k, bm, T, skip=1)
    rows = int(n)
    want, S, live = R.grouped(x, xs, w, ws, s, e, rows, k, bm)
    out = w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, k, bm, out_dtype=dtype)
    assert out.shape == (s.numel(), N) and out.dtype == dtype
    R.check_out(out[:rows], want, S, R.blocks(K), dtype)
    assert bool((out[:rows][~live] == 0).all())
    # the same rows, gathered beforehand
    src = torch.where(s < T * k, s // k, 0).long()
    xr, xsr = x.view(torch.uint8)[src], xs[src]
    xr[s >= T * k] = 0
    direct = w4.fp8_block_moe_gemm(xr, xsr, w, ws, None, e, n, 1, bm, out_dtype=dtype)
    assert torch.equal(direct[:rows], out[:rows])


@pytest.mark.parametrize("T,E,k,N,K,bm", [(1, 4, 2, 256, 128, 16), (5, 8, 3, 512, 272, 16),
                                          (40, 8, 2, 256, 512, 32), (100, 6, 4, 1280, 144, 64),
                                          (300, 5, 3, 768, 1024, 128), (64, 3, 2, 256, 256, 256),
                                          (2, 64, 8, 1024, 2048, 16), (33, 16, 5, 512, 100, 32)])
def test_fp8_block_moe_gemm1_silu(w4, T, E, k, N, K, bm):
    g = _gen(T + N + K)
    x, xs = R.quantise(_randn(g, T, K))
    w, ws = R.quantise(_randn(g, E, N, K) * K ** -0.5, 128)
    s, e, n = _routing(T, E, k, bm, T, skip=2)
    rows = int(n)
    q, qs = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, k, bm)
    assert q.shape == (s.numel(), N // 2) and qs.shape == (s.numel(), N // 256)
    out, S, live = R.grouped(x, xs, w, ws, s, e, rows, k, bm)
    h, dh = R.silu_mul(out, S, R.sum_error(R.blocks(K)))
    R.check_quant(q[:rows], qs[:rows], h, dh)
    assert bool((q[:rows].view(torch.uint8)[~live] == 0).all())
    zero_scale = (torch.tensor(R.FLOOR) / 448.0).cuda()
    assert bool((qs[:rows][~live] == zero_scale).all())


def test_grouped_absent_experts_and_bad_slots_give_zeros(w4):
    g = _gen(12)
    T, E, k, N, K, bm = 24, 4, 2, 256, 256, 16
    x, xs = _matrix(g, T, K, row_block=1)
    w, ws = _matrix(g, E, N, K, row_block=128)
    w.view(torch.uint8)[:, :, 0] = 0x7F  # NaN weights: a zero row must not pick them up
    s, e, n = _routing(T, E, k, bm, 5, spare=0)
    e[0] = -1
    e[1] = E
    s[-1] = -3
    rows = int(n)
    out = w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, k, bm)
    dead = torch.zeros(rows, dtype=torch.bool, device="cuda")
    dead[: 2 * bm] = True
    dead |= (s < 0) | (s >= T * k)
    assert bool((out[dead] == 0).all()) and bool(out[~dead].isnan().all())
    q, qs = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, k, bm)
    assert bool((q.view(torch.uint8)[dead] == 0).all()) and bool(qs[dead].isfinite().all())


@pytest.mark.parametrize("bm,T", [(16, 6), (128, 150)])
def test_rows_past_the_last_are_left(w4, bm, T):
    """Through the C entries, with prefilled outputs: rows at or past num_tokens_post_padded keep
    what they held, also where it ends inside a block, and 0 writes nothing."""
    g = _gen(13)
    E, k, N, K = 3, 2, 256, 384
    x, xs = _matrix(g, T, K, row_block=1)
    w, ws = _matrix(g, E, N, K, row_block=128)
    s, e, n = _routing(T, E, k, bm, 6, spare=3)
    P, rows = s.numel(), int(n)
    lib = load_lib()
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    st = torch.cuda.current_stream().cuda_stream
    for count in (rows, rows - 5, rows - 70 if rows > 128 else 1, 0):
        n.fill_(count)
        out = torch.full((P, N), 7.0, dtype=FP16, device="cuda")
        f = lib.w4a8_fp8_block_moe_gemm
        f.argtypes = [vp] * 8 + [i32] + [i64] * 7 + [vp]
        assert f(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), s.data_ptr(), e.data_ptr(),
                 n.data_ptr(), out.data_ptr(), 1, T, E, N, K, P, k, bm, st) == 0
        assert bool((out[count:] == 7).all())
        q = torch.full((P, N // 2), 9, dtype=torch.uint8, device="cuda")
        qs = torch.full((P, N // 256), 5.0, device="cuda")
        f = lib.w4a8_fp8_block_moe_gemm1_silu
        f.argtypes = [vp] * 9 + [i64] * 7 + [vp]
        assert f(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), s.data_ptr(), e.data_ptr(),
                 n.data_ptr(), q.data_ptr(), qs.data_ptr(), T, E, N // 2, K, P, k, bm, st) == 0
        assert bool((q[count:] == 9).all()) and bool((qs[count:] == 5).all())
        if count:
            want, S, _ = R.grouped(x, xs, w, ws, s, e, rows, k, bm)
            R.check_out(out[:count], want[:count], S[:count], 3, FP16)


def test_no_activations_give_zero_rows(w4):
    """T = 0 with row blocks that hold padding only."""
    w, ws = _matrix(_gen(14), 2, 256, 256, row_block=128)
    x, xs = torch.empty(0, 256, dtype=torch.uint8, device="cuda"), torch.empty(0, 2, device="cuda")
    s = torch.zeros(32, dtype=torch.int32, device="cuda")
    e = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    n = torch.tensor([32], dtype=torch.int32, device="cuda")
    assert bool((w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, 2, 16) == 0).all())
    q, _ = w4.fp8_block_moe_gemm1_silu(x, xs, w, ws, s, e, n, 2, 16)
    assert bool((q.view(torch.uint8) == 0).all())


def test_many_tiles_with_a_short_last_block(w4):
    """More tiles than the GPU holds, outputs that leave by copies of 128 rows, and a count that ends
    inside the last block: the short tile follows copies that are still being read."""
    g = _gen(15)
    T, E, k, N, K, bm = 3000, 2, 1, 2048, 128, 128
    x, xs = _matrix(g, T, K, row_block=1)
    w, ws = _matrix(g, E, N, K, row_block=128)
    s, e, n = _routing(T, E, k, bm, 3, spare=0)
    rows = int(n) - 60
    n.fill_(rows)
    for dtype in (FP16, FP32):
        out = w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, k, bm, out_dtype=dtype)
        want, S, _ = R.grouped(x, xs, w, ws, s, e, rows, k, bm)
        R.check_out(out[:rows], want, S, 1, dtype)


def test_offsets_past_32_bits(w4):
    """Quantisation over, and products into, more than 2^31 elements; the last rows are checked."""
    g = _gen(16)
    M, K = 270000, 8192
    x = torch.zeros(M, K, dtype=BF16, device="cuda")
    x[-3:] = _randn(g, 3, K, dtype=BF16)
    q, s, _, n = w4.rms_norm_quant_fp8(x, torch.ones(K, dtype=BF16, device="cuda"), 1e-5, with_normed=True)
    q2, s2, _, n2 = w4.rms_norm_quant_fp8(x[-3:], torch.ones(K, dtype=BF16, device="cuda"), 1e-5, with_normed=True)
    assert torch.equal(q[-3:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-3:], s2) and torch.equal(n[-3:], n2)
    del n, n2
    q, s = w4.act_quant_fp8_block(x)
    rq, rs = R.quantise(x[-3:].float())
    assert torch.equal(q[-3:].view(torch.uint8), rq.view(torch.uint8)) and torch.equal(s[-3:], rs)
    del x
    w, ws = _matrix(g, 8320, 128, row_block=128)
    out = w4.fp8_block_gemm(q[:, :128].contiguous(), s[:, :1].contiguous(), w, ws)
    assert out.numel() > 1 << 31
    want, S = R.product(q[-3:, :128], s[-3:, :1], w, ws)
    R.check_out(out[-3:], want, S, 1, FP16)
    del out
    # activation rows past 2^31 bytes, through the routing, in both forms of the kernel
    xw, wsw = _matrix(g, 2, 256, K, row_block=128)
    for bm in (16, 128):
        src = torch.tensor([M - 1, M - 2, M - 3, 5] + [M] * (bm - 4), dtype=torch.int32, device="cuda")
        one = torch.ones(1, dtype=torch.int32, device="cuda")
        got = w4.fp8_block_moe_gemm(q, s, xw, wsw, src, one, one * bm, 1, bm, out_dtype=FP32)
        want, S = R.product(q[src[:4].long()], s[src[:4].long()], xw[1], wsw[1])
        R.check_out(got[:4], want, S, R.blocks(K), FP32)
        assert bool((got[4:] == 0).all())


def test_two_streams_at_once(w4):
    """Calls of both kernel forms that overlap on the GPU."""
    g = _gen(17)
    cases = []
    for M, N, K in ((700, 4096, 1024), (8, 4096, 2048)):
        x, xs = _matrix(g, M, K, row_block=1)
        w, ws = _matrix(g, N, K, row_block=128)
        cases.append((x, xs, w, ws, w4.fp8_block_gemm(x, xs, w, ws)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for i in range(24):
        x, xs, w, ws, ref = cases[i % 2]
        with torch.cuda.stream(streams[i % 4]):
            outs.append((w4.fp8_block_gemm(x, xs, w, ws), ref))
    torch.cuda.synchronize()
    for out, ref in outs:
        assert torch.equal(out, ref)


# ------------------------------------------------------------------ together ----------------
def _layer(g, T, E, H, I):
    w1, s1 = R.quantise(_randn(g, E, 2 * I, H) * H ** -0.5, 128)
    w2, s2 = R.quantise(_randn(g, E, H, I) * I ** -0.5, 128)
    return w1, w2, s1, s2


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 256, 128), (32, 16, 4, 512, 256),
                                       (700, 8, 2, 384, 256), (4100, 4, 1, 256, 128)])
def test_norm_router_moe_together(w4, T, E, k, H, I, dtype):
    """norm + residual -> router -> the layer, as a model's MoE block chains them; the result
    against 64 bits on the operands that the layer quantised itself."""
    from w4a8_fp8_wmma.fp8_block import fp8_block_m, run_fp8_block_moe
    g = _gen(T + H)
    x, r = _randn(g, T, H, dtype=dtype), _randn(g, T, H, dtype=dtype)
    nw = (1 + 0.1 * _randn(g, H)).to(dtype)
    q, s, res, normed = w4.rms_norm_quant_fp8(x, nw, 1e-6, residual=r, with_normed=True)
    gate = _randn(g, E, H, dtype=dtype) * H ** -0.5
    ids, tw, _ = w4.route_topk((normed @ gate.t()).float(), k)
    w1, w2, s1, s2 = _layer(g, T, E, H, I)
    y = run_fp8_block_moe(q, w1, w2, s1, s2, tw, ids, x_scales=s, out_dtype=dtype)
    assert y.shape == (T, H) and y.dtype == dtype and bool(y.isfinite().all())
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    row_t = BF16 if dtype == BF16 else FP16
    for j in range(k):
        for e in range(E):
            at = (ids[:, j] == e).nonzero().reshape(-1)
            if not at.numel():
                continue
            o, S = R.product(q[at], s[at], w1[e], s1[e])
            h, dh = R.silu_mul(o, S, R.sum_error(R.blocks(H)))
            # h enters the down product quantised: half a step of e4m3, at least 2^-10 of a scale
            f = R.spread_cols(torch.nn.functional.pad(h, (0, 0)).reshape(len(at), -1, 128).abs()
                              .amax(2).clamp_min(R.FLOOR) / 448.0, I)
            dh = dh + (torch.maximum(h.abs() * 2.0 ** -4, f * 2.0 ** -10) * 1.01)
            b = w2[e].double() * R.spread_w(s2[e].double(), H, I)
            d = h @ b.T
            dd = dh @ b.abs().T + R.sum_error(R.blocks(I)) * (h.abs() @ b.abs().T)
            dd = dd + R.HALF[row_t] * (d.abs() + dd)
            want[at] += tw[at, j, None].double() * d
            tol[at] += tw[at, j, None].double() * dd
    tol = tol * (1 + 1e-6) + (R.HALF[dtype] + k * 2.0 ** -24) * (want.abs() + tol)
    assert bool(((y.double() - want).abs() <= tol).all())
    # from unquantised rows the layer quantises them itself
    q2, s2x = w4.act_quant_fp8_block(normed)
    a = run_fp8_block_moe(normed, w1, w2, s1, s2, tw, ids)
    b = run_fp8_block_moe(q2, w1, w2, s1, s2, tw, ids, x_scales=s2x, out_dtype=dtype)
    assert torch.equal(a, b)
    assert fp8_block_m(T * k, E) in (16, 32, 64, 128)


def test_layer_with_expert_map(w4):
    """Two halves of the experts, each with the other's slots mapped to -1, sum to the layer."""
    from w4a8_fp8_wmma.fp8_block import run_fp8_block_moe
    g = _gen(77)
    T, E, k, H, I = 50, 8, 3, 256, 128
    x = _randn(g, T, H, dtype=FP16)
    w1, w2, s1, s2 = _layer(g, T, E, H, I)
    ids, tw, _ = w4.route_topk(_randn(g, T, E), k)
    whole = run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids, out_dtype=FP32)
    parts = torch.zeros_like(whole)
    for lo in (0, 4):
        m = torch.full((E,), -1, dtype=torch.int32, device="cuda")
        m[lo:lo + 4] = torch.arange(4, dtype=torch.int32, device="cuda")
        sl = slice(lo, lo + 4)
        parts += run_fp8_block_moe(x, w1[sl], w2[sl], s1[sl], s2[sl], tw, ids,
                                   global_num_experts=E, expert_map=m, out_dtype=FP32)
    # the same fp16 rows, added in another order: k fp32 roundings of sums of |w * row|
    bound = 2 * k * 2.0 ** -24 * (whole.abs().amax() * k + 1)
    assert float((parts - whole).abs().max()) <= float(bound)


def test_gather_reduce_bf16_rows(w4):
    g = _gen(5)
    for N in (64, 20):
        rows = _randn(g, 48, N, dtype=BF16)
        s = torch.randperm(48, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        n = torch.tensor([48], dtype=torch.int32, device="cuda")
        tw = torch.rand(24, 2, generator=g, device="cuda")
        got = w4.mmq_fp8_moe_gather_reduce(rows, s, tw.reshape(-1), n, 2)
        back = torch.empty(48, dtype=torch.long, device="cuda")
        back[s.long()] = torch.arange(48, device="cuda")
        r = rows.float()[back].reshape(24, 2, N)
        assert torch.equal(got, tw[:, 0, None] * r[:, 0] + tw[:, 1, None] * r[:, 1])


def test_side_stream_and_graphs(w4):
    """The layer on another stream, and two captured graphs replayed in turn on new inputs."""
    from w4a8_fp8_wmma.fp8_block import run_fp8_block_moe
    g = _gen(21)
    T, E, k, H, I = 32, 16, 4, 512, 256
    w1, w2, s1, s2 = _layer(g, T, E, H, I)
    xs = [_randn(g, T, H, dtype=BF16) for _ in range(4)]
    routes = [w4.route_topk(_randn(g, T, E), k)[:2] for _ in range(4)]
    nw = torch.ones(H, device="cuda", dtype=BF16)

    def step(x, tw, ids):
        q, s, res, _ = w4.rms_norm_quant_fp8(x, nw, 1e-6, residual=x)
        y = run_fp8_block_moe(q, w1, w2, s1, s2, tw, ids, x_scales=s, out_dtype=BF16)
        a, b = w4.act_quant_fp8_block(y)
        return res, y, w4.fp8_block_gemm(a, b, w1[0], s1[0], out_dtype=BF16)

    eager = [step(x, tw, ids) for x, (ids, tw) in zip(xs, routes)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, (ids, tw), ref in zip(xs, routes, eager):
            for a, b in zip(step(x, tw, ids), ref):
                assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        bx, bi, bw = xs[0].clone(), routes[0][0].clone(), routes[0][1].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(bx, bw, bi)
        graphs.append((gr, bx, bi, bw, out))
    for i in (1, 2, 3, 0, 2):
        gr, bx, bi, bw, out = graphs[i % 2]
        bx.copy_(xs[i]), bi.copy_(routes[i][0]), bw.copy_(routes[i][1])
        gr.replay()
        for a, b in zip(out, eager[i]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,E,k,H,I", [(8, 4, 2, 512, 256), (32, 16, 4, 1024, 512), (24, 64, 8, 2048, 128)])
def test_launches_that_follow_one_another(w4, T, E, k, H, I):
    """Chains in which each call reads what the one before wrote, into the same buffers every time and
    without a wait between, eager and captured, against the same calls waited for one by one."""
    g = _gen(T + E)
    w1, w2, s1, s2 = _layer(g, T, E, H, I)
    w3, s3 = w2[0].view(torch.uint8).repeat(1, 2), s2[0].repeat(1, 2)
    bm = 16
    inputs = []
    for i in range(6):
        q, sc = _matrix(g, T, H, row_block=1)
        inputs.append((q, sc) + _routing(T, E, k, bm, i + 2))
    size = max(t[2].numel() for t in inputs)
    s = torch.empty(size, dtype=torch.int32, device="cuda")
    e = torch.empty(size // bm, dtype=torch.int32, device="cuda")
    x, xs, n = inputs[0][0].clone(), inputs[0][1].clone(), inputs[0][4].clone()

    def load(i):
        q, sc, si, ei, ni = inputs[i]
        x.copy_(q), xs.copy_(sc), n.copy_(ni)
        s.fill_(T * k), e.fill_(-1)
        s[:si.numel()].copy_(si), e[:ei.numel()].copy_(ei)

    def chain(wait=lambda: None):
        h, hs = w4.fp8_block_moe_gemm1_silu(x, xs, w1, s1, s, e, n, k, bm)
        wait()
        y = w4.fp8_block_moe_gemm(h, hs, w2, s2, None, e, n, 1, bm, BF16)
        wait()
        a, b = w4.act_quant_fp8_block(y[:T])  # the first rows: below every count here
        wait()
        z = w4.fp8_block_gemm(a, b, w1[0], s1[0], BF16)
        wait()
        a, b = w4.act_quant_fp8_block(z)
        wait()
        return w4.fp8_block_gemm(a, b, w3, s3, FP32)

    assert all(int(t[4]) >= T for t in inputs)
    want = []
    for i in range(6):
        load(i)
        want.append(chain(torch.cuda.synchronize))
        torch.cuda.synchronize()
    got = []
    for i in [0, 1, 2, 3, 4, 5] * 8:
        load(i)
        got.append((i, chain()))
    for i, z in got:
        assert torch.equal(z, want[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = chain()
    for i in [3, 0, 5, 1, 4, 2] * 4:
        load(i)
        graph.replay()
        assert torch.equal(z, want[i])


def test_capture_with_a_fork(w4):
    """Two captured branches that join in front of a third product; outputs of both are read."""
    g = _gen(5)
    x1, s1 = _matrix(g, 16, 512, row_block=1)
    x2, s2 = _matrix(g, 16, 512, row_block=1)
    w, ws = _matrix(g, 512, 512, row_block=128)

    def joined(fork):
        main = torch.cuda.current_stream()
        side = torch.cuda.Stream() if fork else main
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b, bs = w4.act_quant_fp8_block(w4.fp8_block_gemm(x2, s2, w, ws))
            b = w4.fp8_block_gemm(b, bs, w, ws, FP32)
        a, as_ = w4.act_quant_fp8_block(w4.fp8_block_gemm(x1, s1, w, ws))
        z = w4.fp8_block_gemm(a, as_, w, ws, FP32)
        main.wait_stream(side)
        q, s = w4.act_quant_fp8_block(z + b)
        return w4.fp8_block_gemm(q, s, w, ws), w4.fp8_block_gemm(x2, s2, w, ws), b

    want = [t.clone() for t in joined(False)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = joined(True)
    for _ in range(20):
        for t in got:
            t.zero_()
        graph.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals(w4):
    x = torch.zeros(16, 256, dtype=torch.uint8, device="cuda")
    xs = torch.zeros(16, 2, device="cuda")
    w = torch.zeros(2, 256, 256, dtype=torch.uint8, device="cuda")
    ws = torch.zeros(2, 2, 2, device="cuda")
    e = torch.zeros(1, dtype=torch.int32, device="cuda")
    n = torch.tensor([16], dtype=torch.int32, device="cuda")
    s = torch.arange(16, dtype=torch.int32, device="cuda")
    bad = [
        lambda: w4.fp8_block_gemm(x.float(), xs, w[0], ws[0]),
        lambda: w4.fp8_block_gemm(x, xs.half(), w[0], ws[0]),
        lambda: w4.fp8_block_gemm(x, xs[:, :1], w[0], ws[0]),
        lambda: w4.fp8_block_gemm(x, xs, w[0, :, :128], ws[0]),
        lambda: w4.fp8_block_gemm(x, xs, w[0].t(), ws[0]),
        lambda: w4.fp8_block_gemm(x, xs, w[0], ws[0, :1]),
        lambda: w4.fp8_block_gemm(x, xs, w[0].cpu(), ws[0]),
        lambda: w4.fp8_block_gemm(x, xs, w[0], ws[0], out_dtype=torch.float64),
        lambda: w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, 1, 8),
        lambda: w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, 1, 48),
        lambda: w4.fp8_block_moe_gemm(x, xs, w, ws, s, e, n, 0, 16),
        lambda: w4.fp8_block_moe_gemm(x, xs, w, ws, s.long(), e, n, 1, 16),
        lambda: w4.fp8_block_moe_gemm(x, xs, w, ws, s, torch.cat([e, e]), n, 1, 16),
        lambda: w4.fp8_block_moe_gemm(x, xs, w[0], ws[0], s, e, n, 1, 16),
        lambda: w4.fp8_block_moe_gemm1_silu(x, xs, w[:, :128], ws[:, :1], s, e, n, 1, 16),
        lambda: w4.act_quant_fp8_block(x),
        lambda: w4.act_quant_fp8_block(xs[0]),
        lambda: w4.rms_norm_quant_fp8(xs, xs[0, :1]),
        lambda: w4.rms_norm_quant_fp8(xs.half(), xs[0].bfloat16()),
        lambda: w4.rms_norm_quant_fp8(xs, xs[0], residual=xs[:8]),
        lambda: w4.rms_norm_quant_fp8(xs, xs[0], eps=-1.0),
    ]
    for f in bad:
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()
