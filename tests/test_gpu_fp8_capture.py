"""Captured block-scaled products whose predecessor in the stream is no kernel: a fill, a copy on the
device, or work of another stream that they wait for. The kernel of short row blocks is launched to start
early, an edge that exists between kernels only."""
import pytest
import torch

import fp8_block_ref as R

pytestmark = pytest.mark.gpu


def _operands(M, N, K):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    x, xs = R.quantise(torch.randn(M, K, generator=g, device="cuda"))
    w, ws = R.quantise(torch.randn(N, K, generator=g, device="cuda"), 128)
    return x, xs, w, ws


@pytest.mark.parametrize("M,N,K", [(1, 512, 512), (16, 4096, 256), (700, 2048, 256)])
@pytest.mark.parametrize("ahead", ["fill", "copy", "both", "event", "side fill"])
def test_after_what_is_no_kernel(M, N, K, ahead):
    import w4a8_fp8_wmma as w4
    x, xs, w, ws = _operands(M, N, K)
    want = w4.fp8_block_gemm(x, xs, w, ws)
    zero = torch.zeros_like(want)
    bx, bs = x.view(torch.uint8).clone(), xs.clone()
    torch.cuda.synchronize()

    def step():
        main = torch.cuda.current_stream()
        if ahead in ("copy", "both"):
            bx.copy_(x.view(torch.uint8)), bs.copy_(xs)
        if ahead in ("fill", "both"):
            bs.zero_()
        if ahead in ("event", "side fill"):
            side = torch.cuda.Stream()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                bs.zero_() if ahead == "side fill" else bs.copy_(xs)
            main.wait_stream(side)
        a = w4.fp8_block_gemm(bx, bs, w, ws)
        bs.copy_(xs)
        return a, w4.fp8_block_gemm(bx, bs, w, ws)

    first = zero if ahead in ("fill", "both", "side fill") else want
    for a, b in (step(), step()):
        assert torch.equal(a, first) and torch.equal(b, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step()
    for _ in range(5):
        a.fill_(7), b.fill_(7)
        graph.replay()
        assert torch.equal(a, first) and torch.equal(b, want)
