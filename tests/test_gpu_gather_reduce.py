"""Topk-weighted gather-reduce at widths and slot counts outside the vectorised path: N not a
multiple of 8 and top_k above 16 take the generic kernel, which must write every output."""
import numpy as np
import pytest
import torch

import w4a8_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,top_k,E", [(5, 20, 2, 8), (9, 1001, 4, 8), (3, 64, 17, 32),
                                         (1, 1, 1, 4)])
def test_gather_reduce_generic_widths(M, N, top_k, E):
    import w4a8_fp8_wmma as w4
    rng = np.random.default_rng(M * 131 + N)
    ids = np.stack([rng.permutation(E)[:top_k] for _ in range(M)]).astype(np.int32)
    s, _, n = w4.moe_align_block_size(torch.from_numpy(ids).cuda(), 16, E)
    out2 = rng.standard_normal((s.numel(), N), dtype=np.float32).astype(np.float16)
    tw = rng.random((M, top_k), dtype=np.float32)
    # NaN-fill what the allocator hands out next, so an output left unwritten cannot pass
    torch.full((M, N), float("nan"), device="cuda")
    got = w4.mmq_fp8_moe_gather_reduce(torch.from_numpy(out2).cuda(), s,
                                       torch.from_numpy(tw.reshape(-1)).cuda(), n, top_k)
    ref = O.gather_reduce(out2, s.cpu().numpy(), tw, int(n), top_k)
    # the same fp32 products and the same order of addition
    np.testing.assert_array_equal(got.cpu().numpy(), ref.astype(np.float32))
