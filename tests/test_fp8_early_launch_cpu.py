"""What the sources say about the kernel that starts before the work ahead of it in the stream has
ended (gemm_fp8_swap.cu). It reads buffers that the launch before may still be writing when it
starts. Loads on the read-only path (ld.global.nc, __ldg) are defined only for memory that nothing
writes during the kernel's life, so it may use none, however late they stand."""
import os
import re

from helpers import ROOT

CSRC = os.path.join(ROOT, "rdna4-vllm_b200", "csrc")


def _code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def _included(name, seen):
    if name in seen or not os.path.exists(os.path.join(CSRC, name)):
        return seen
    seen[name] = _code(name)
    for other in re.findall(r'#include "([^"]+)"', seen[name]):
        _included(other, seen)
    return seen


def _early_sources():
    return [n for n in sorted(os.listdir(CSRC)) if n.endswith(".cu") and
            re.search(r"launch_persistent<[^;(]*,\s*true>", _code(n))]


def test_early_kernel_uses_no_read_only_loads():
    assert _early_sources() == ["gemm_fp8_swap.cu"]
    used = _included("gemm_fp8_swap.cu", {})
    assert "fp8_tc.cuh" in used
    # one helper of the shared headers is on the read-only path; the two files that make the kernel
    # use neither it nor such a load of their own
    others = {n: t for n, t in used.items() if n not in ("gemm_fp8_swap.cu", "fp8_tc.cuh")}
    assert [n for n, t in others.items() if "ld.global.nc" in t or "__ldg" in t] == ["common.cuh"]
    assert others["common.cuh"].count("ld.global.nc") == 1 and "ldg_stream" in others["common.cuh"]
    for name in ("gemm_fp8_swap.cu", "fp8_tc.cuh"):
        assert not re.search(r"ld\.global\.nc|__ldg|ldg_stream|__restrict__", used[name]), name


def test_early_kernel_waits_before_it_reads():
    """Up to follow_launch() the kernel sets up barriers and tensor memory: no fetch, copy or count."""
    body = _code("gemm_fp8_swap.cu").split("fp8_swap_kernel(", 1)[1]
    ahead, behind = body.split("follow_launch();", 1)
    lambdas = re.sub(r"auto expert_of = .*?;\s*};", "", ahead, flags=re.S)
    for read in ("fetch(", "ntp[0]", "tma_load", "tma_gather4", "ld_cluster", "finish_row"):
        assert read not in lambdas, read
    assert "fetch(a.ntp)" in behind and "ntp[0]" not in behind
