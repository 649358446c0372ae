"""Topk-weighted gather-reduce on rows that are not what the allocator gives: views off their
alignment, more tokens than one grid dimension holds, and the types that the MoE layers write."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def w4():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import w4a8_fp8_wmma
    return w4a8_fp8_wmma


def _case(M, N, top_k, dtype, seed):
    """Rows in a shuffled order, their slots, the count and the weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    P = M * top_k
    rows = torch.randn(P, N, generator=g, device="cuda").to(dtype)
    s = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    n = torch.tensor([P], dtype=torch.int32, device="cuda")
    return rows, s, n, torch.rand(P, generator=g, device="cuda")


def _expected(rows, s, tw, top_k):
    """The same fp32 products, added in the same order."""
    back = torch.empty_like(s, dtype=torch.long)
    back[s.long()] = torch.arange(s.numel(), device="cuda")
    r = rows.float()[back].reshape(-1, top_k, rows.shape[1])
    w = tw.reshape(-1, top_k, 1)
    out = torch.zeros_like(r[:, 0])
    for j in range(top_k):
        out = out + w[:, j] * r[:, j]
    return out


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("N", [2, 20, 21, 64, 1000])
@pytest.mark.parametrize("off", [1, 2, 3, 8])
def test_views_off_their_alignment(w4, N, off, dtype):
    rows, s, n, tw = _case(11, N, 3, dtype, N + off)
    base = torch.empty(rows.numel() + off, dtype=dtype, device="cuda")
    view = base[off:].view_as(rows)
    view.copy_(rows)
    got = w4.mmq_fp8_moe_gather_reduce(view, s, tw, n, 3)
    assert torch.equal(got, w4.mmq_fp8_moe_gather_reduce(rows, s, tw, n, 3))
    assert torch.equal(got, _expected(rows, s, tw, 3))


@pytest.mark.parametrize("M,N,top_k", [(65535, 8, 1), (65536, 8, 1), (70000, 16, 2), (70000, 6, 2),
                                       (140000, 8, 3), (140001, 5, 1)])
def test_more_tokens_than_a_grid_dimension_holds(w4, M, N, top_k):
    """Above 65535 tokens, through the vectorised kernel (N a multiple of 8) and the generic one."""
    rows, s, n, tw = _case(M, N, top_k, FP16, M + N)
    assert torch.equal(w4.mmq_fp8_moe_gather_reduce(rows, s, tw, n, top_k), _expected(rows, s, tw, top_k))


def test_refusals(w4):
    """Operands that the kernel could not read, or would read in another order."""
    rows, s, n, tw = _case(4, 16, 2, FP16, 1)
    twice = s.repeat_interleave(2)
    bad = [(rows, s.cpu(), tw, n), (rows, s, tw.cpu(), n), (rows, s, tw, n.cpu()), (rows, twice[::2], tw, n),
           (rows, s.reshape(2, 4), tw, n), (rows, s, tw, n[:0]), (rows, s.long(), tw, n),
           (rows, s, tw.half(), n), (rows.t(), s, tw, n), (rows, twice, tw, n), (rows.int(), s, tw, n)]
    for args in bad:
        with pytest.raises((RuntimeError, NotImplementedError)):
            w4.mmq_fp8_moe_gather_reduce(*args, 2)
    for ids in (s, s[:, None]):  # a column of ids is the ids
        assert torch.equal(w4.mmq_fp8_moe_gather_reduce(rows, ids, tw, n, 2), _expected(rows, s, tw, 2))


def test_layer_refuses_weights_of_another_device(w4):
    from w4a8_fp8_wmma.fp8_block import run_fp8_block_moe
    x = torch.ones(2, 128, dtype=BF16, device="cuda")
    w1 = torch.zeros(2, 256, 128, dtype=torch.uint8, device="cuda")
    w2 = torch.zeros(2, 128, 128, dtype=torch.uint8, device="cuda")
    s1, s2 = torch.ones(2, 2, 1, device="cuda"), torch.ones(2, 1, 1, device="cuda")
    ids = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    tw = torch.ones(2, 1, device="cuda")
    assert bool((run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids) == 0).all())
    assert bool((run_fp8_block_moe(x, w1, w2, s1, s2, tw, ids.long()) == 0).all())  # converted on the way
    for change in (dict(topk_weights=tw.cpu()), dict(topk_ids=ids.cpu())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            run_fp8_block_moe(x, w1, w2, s1, s2, **{"topk_weights": tw, "topk_ids": ids, **change})


@pytest.mark.parametrize("M,N,top_k", [(1, 4, 1), (7, 12, 2), (33, 1000, 8), (5, 1001, 3), (9, 6, 2), (4, 64, 17),
                                       (700, 2048, 4), (70000, 4, 1), (70000, 3, 1)])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_fp32_rows(w4, M, N, top_k, off):
    """Through the vectorised kernel (N a multiple of 4, rows on 16 bytes) and the generic one; values
    that fp16 does not hold."""
    rows, s, n, tw = _case(M, N, top_k, FP32, M + N)
    rows = rows * 1e6
    base = torch.empty(rows.numel() + off, device="cuda")
    view = base[off:].view_as(rows)
    view.copy_(rows)
    got = w4.mmq_fp8_moe_gather_reduce(view, s, tw, n, top_k)
    assert got.dtype == FP32 and torch.equal(got, _expected(rows, s, tw, top_k))


def test_fp32_rows_absent_slots(w4):
    """Slots that no row holds (remote experts) add nothing; a token without any is zero."""
    rows, s, _, tw = _case(6, 16, 2, FP32, 3)
    n = torch.tensor([7], dtype=torch.int32, device="cuda")
    here = torch.zeros(12, dtype=torch.bool, device="cuda")
    here[s[:7].long()] = True
    got = w4.mmq_fp8_moe_gather_reduce(rows, s, tw, n, 2)
    kept = torch.where(here, tw, 0.0)
    assert torch.equal(got, _expected(rows, s, kept, 2))
