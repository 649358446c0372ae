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
