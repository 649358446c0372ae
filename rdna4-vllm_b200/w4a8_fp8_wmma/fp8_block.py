"""The gated MoE layer on block-scaled FP8 weights, the 8-bit sibling of moe_experts.run_grouped_moe.

A mixed checkpoint keeps some layers in e4m3 with a scale per 128 x 128 block beside the 4-bit
ones; this composition runs such a layer on the same routing tensors and the same reduce.
"""
from __future__ import annotations

import torch

from . import (act_quant_fp8_block, fp8_block_moe_gemm, fp8_block_moe_gemm1_silu,
               mmq_fp8_moe_gather_reduce, moe_align_block_size)
from .moe_experts import APPLY_CHUNK


def fp8_block_m(rows: int, num_experts: int) -> int:
    """Row-block size of the block-scaled composition for `rows` routed rows: the smallest of
    16, 32, 64, 128 that holds twice the average expert's rows. A block costs one pass over its
    expert's weights, so an expert should fit one; block_m rows are written per block, so the
    padding should stay small.

    gate_up + down of 256 experts, top 8, 2048 -> 2 x 512 -> 2048, in us by block size:
    32 tokens 94 (16), 106 (32), 154 (64), 119 (128); 512 tokens 149, 147, 211, 171;
    1024 tokens 202, 177, 196, 173; 4096 tokens 605, 471, 414, 228. With skewed routing
    (rank^-1.1) the padding is less and 128 gains sooner: 512 tokens 108, 104, 114, 90;
    1024 tokens 177, 160, 158, 105. So the rule is off its best by 13 % (uniform) to 50 % (skewed)
    around 1024 tokens, where it takes 64, and by 16 % at 512 skewed.
    """
    return next((b for b in (16, 32, 64) if b * num_experts >= 2 * rows), 128)


def run_fp8_block_moe(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w1_s: torch.Tensor,
                      w2_s: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor,
                      x_scales: torch.Tensor | None = None,
                      global_num_experts: int | None = None,
                      expert_map: torch.Tensor | None = None,
                      out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Whole gated MoE on block-scaled FP8 weights; (M, K), topk-weighted and reduced.

    x (M, K) fp16/bf16/fp32, quantised here; or already quantised (rms_norm_quant_fp8) as e4m3
    with x_scales (M, ceil(K/128)), and out_dtype given. w1 (E, 2*inter, K) e4m3 [gate | up],
    w2 (E, K, inter) e4m3, w1_s / w2_s (E, ceil(N/128), ceil(K/128)) fp32, inter a multiple of
    128. ``expert_map`` maps global expert ids to local ones (-1 = remote); remote slots
    contribute nothing. The steps are run_grouped_moe's: align, gate_up with SiLU (here also the
    quantisation that down reads), down, gather-reduce; down's rows are fp16 or bf16 when
    out_dtype is, else fp32. Longer batches run in the same 4096-token chunks.
    """
    if (x_scales is not None) and out_dtype is None:
        raise ValueError("run_fp8_block_moe: quantised x needs out_dtype")
    out_dtype = out_dtype or x.dtype
    M = x.size(0)
    if M == 0:
        return torch.empty((0, w2.size(1)), dtype=out_dtype, device=x.device)
    top_k = topk_ids.size(1)
    E_local = w1.size(0)
    E_global = int(global_num_experts) if global_num_experts is not None else E_local
    if APPLY_CHUNK and M > APPLY_CHUNK:
        out = torch.empty((M, w2.size(1)), dtype=out_dtype, device=x.device)
        for lo in range(0, M, APPLY_CHUNK):
            hi = min(lo + APPLY_CHUNK, M)
            out[lo:hi] = run_fp8_block_moe(
                x[lo:hi], w1, w2, w1_s, w2_s, topk_weights[lo:hi], topk_ids[lo:hi],
                None if x_scales is None else x_scales[lo:hi], global_num_experts, expert_map,
                out_dtype)
        return out
    if x_scales is None:
        x, x_scales = act_quant_fp8_block(x)
    block_m = fp8_block_m(M * top_k, E_global)
    sorted_ids, expert_ids, ntp = moe_align_block_size(topk_ids, block_m, E_global, expert_map,
                                                       E_local)
    h, h_scales = fp8_block_moe_gemm1_silu(x, x_scales, w1, w1_s, sorted_ids, expert_ids, ntp,
                                           top_k, block_m)
    row_dtype = out_dtype if out_dtype in (torch.float16, torch.bfloat16) else torch.float32
    rows = fp8_block_moe_gemm(h, h_scales, w2, w2_s, None, expert_ids, ntp, 1, block_m, row_dtype)
    tw = topk_weights.reshape(-1).to(torch.float32).contiguous()
    return mmq_fp8_moe_gather_reduce(rows, sorted_ids, tw, ntp, top_k).to(out_dtype)
