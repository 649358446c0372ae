"""w4a8_fp8_wmma — B200 (sm_100a) build of the W4A8 FP8 GEMM / MoE op library.

Drop-in for the reference package of the same name (w4a8_fp8_wmma/w4a8_fp8_wmma/__init__.py):
same Python wrappers, kernel-name maps, torch op namespace and schemas, and fake (meta) impls.
The ops run hand-written CUDA kernels from ``libw4a8_b200.so`` through the ``_C.so`` torch shim;
there is no CPU or Triton fallback. Importing the package without the built libraries raises.
"""
from __future__ import annotations

import os

import torch  # must come before loading _C so libtorch is already resident

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libw4a8_b200.so")
SHIM_PATH = os.path.join(_HERE, "_C.so")

if not (os.path.exists(LIB_PATH) and os.path.exists(SHIM_PATH)):
    raise ImportError(
        "w4a8_fp8_wmma: native libraries are not built "
        f"({LIB_PATH}, {SHIM_PATH}); run `python rdna4-vllm_b200/build.py`")
torch.ops.load_library(SHIM_PATH)

# Descriptive kernel names -> the opaque ids carried over the op ABI
# (reference: w4a8_fp8_wmma/w4a8_fp8_wmma/__init__.py:10-22, kernel_names.h:18-46).
_MOE_KERNELS = {"scalar": 0, "wmma": 6, "gemv": 7}
_DENSE_KERNELS = {
    "reference_scalar": 0, "rocwmma_v1": 1, "rocwmma_tiled": 2, "rocwmma_pipe": 4,
    "prefill_wmma": 5, "prefill_wmma_b128": 6, "wmma_tiled_tuned": 7, "wmma_dbuf": 8,
    "wmma_dbuf2": 9, "prefill_wmma_ashuffle": 10, "decode_gemv": 11,
    "splitk_smallm": 12, "regdirect_shuffle": 13, "nsplit_smallm": 14,
}
# Names served by this build; the rest are gfx1201 research kernels and raise in the op.
SERVED_DENSE_KERNELS = ("reference_scalar", "prefill_wmma", "prefill_wmma_ashuffle",
                        "decode_gemv")


def _resolve_dense_kernel(kernel) -> int:
    """Map a dense kernel name to its op id; unknown names and bare ints are rejected."""
    if isinstance(kernel, str):
        try:
            return _DENSE_KERNELS[kernel]
        except KeyError:
            raise ValueError(
                f"unknown dense kernel {kernel!r}; known: {sorted(_DENSE_KERNELS)}") from None
    raise TypeError(
        f"dense kernel must be a name in {sorted(_DENSE_KERNELS)} (the integer "
        f"'version' was removed); got {kernel!r}")


def _resolve_moe_kernel(kernel) -> int:
    """Map a MoE kernel name to its op id; unknown names and bare ints are rejected."""
    if isinstance(kernel, str):
        try:
            return _MOE_KERNELS[kernel]
        except KeyError:
            raise ValueError(
                f"unknown moe kernel {kernel!r}; known: {sorted(_MOE_KERNELS)}") from None
    raise TypeError(
        f"moe kernel must be a name in {sorted(_MOE_KERNELS)} (the integer 'version' was "
        f"removed); got {kernel!r}")


def _empty_zeros(dev) -> torch.Tensor:
    return torch.empty(0, dtype=torch.int32, device=dev)


def mmq_fp8_gemm(x: torch.Tensor, w_packed: torch.Tensor, scales: torch.Tensor,
                 kernel: str = "reference_scalar", w_zeros: torch.Tensor | None = None,
                 weight_is_e2m1: bool = False) -> torch.Tensor:
    """Dense W4A8 GEMM: (M, K) fp16 x (N, K/8) int32 codes -> (M, N) fp16.

    scales (N, K/g) fp16; w_zeros (N/8, K/g) int32 packed zero points or None (zp = 8).
    Every served kernel name computes the same function; "decode_gemv" forces the
    small-M register GEMV, "prefill_wmma*" the tile path, "reference_scalar" the scalar kernel.
    """
    if w_zeros is None:
        w_zeros = _empty_zeros(x.device)
    return torch.ops.w4a8_fp8_wmma.mmq_fp8_gemm(
        x, w_packed, scales, w_zeros, _resolve_dense_kernel(kernel), weight_is_e2m1)


def mmq_fp8_moe_gemm(x, w_packed, scales, sorted_token_ids, expert_ids,
                     num_tokens_post_padded, top_k: int, block_m: int, kernel: str = "wmma",
                     w_zeros=None, weight_is_e2m1: bool = False) -> torch.Tensor:
    """Grouped MoE GEMM: out[r] = x[sorted_token_ids[r] // top_k] @ W[expert(r)]^T.

    x (T, K) fp16; w_packed (E, N, K/8) int32; scales (E, N, K/g) fp16; routing tensors in the
    moe_align_block_size layout. Returns (P, N) fp16; padding rows are zero.
    """
    if w_zeros is None:
        w_zeros = _empty_zeros(x.device)
    return torch.ops.w4a8_fp8_wmma.mmq_fp8_moe_gemm(
        x, w_packed, scales, w_zeros, sorted_token_ids, expert_ids, num_tokens_post_padded,
        top_k, block_m, _resolve_moe_kernel(kernel), weight_is_e2m1)


def mmq_fp8_moe_gemm1_silu(x, w_packed, scales, sorted_token_ids, expert_ids,
                           num_tokens_post_padded, top_k: int, block_m: int,
                           kernel: str = "wmma", w_zeros=None,
                           weight_is_e2m1: bool = False) -> torch.Tensor:
    """Fused gate_up GEMM + silu_and_mul: w_packed (E, 2*inter, K/8) = [gate | up].

    Returns (P, inter) fp16, bit-identical to mmq_fp8_moe_gemm followed by vLLM silu_and_mul
    (fp16 gate/up stores, silu in fp32 rounded to fp16, half*half product).
    """
    if w_zeros is None:
        w_zeros = _empty_zeros(x.device)
    return torch.ops.w4a8_fp8_wmma.mmq_fp8_moe_gemm1_silu(
        x, w_packed, scales, w_zeros, sorted_token_ids, expert_ids, num_tokens_post_padded,
        top_k, block_m, _resolve_moe_kernel(kernel), weight_is_e2m1)


def mmq_fp8_moe_gemm_scatter(x, w_packed, scales, sorted_token_ids, expert_ids,
                             num_tokens_post_padded, topk_weights, output, top_k: int,
                             block_m: int, kernel: str = "wmma", w_zeros=None,
                             weight_is_e2m1: bool = False) -> None:
    """Down GEMM + topk-weighted atomic scatter into the pre-zeroed (M, N) fp32 ``output``.

    x (P, K) fp16 is the post-activation buffer, gathered by row identity; row r adds
    topk_weights[s] * (x[r] @ W[e]^T) into output[s // top_k] with s = sorted_token_ids[r].
    """
    if w_zeros is None:
        w_zeros = _empty_zeros(x.device)
    torch.ops.w4a8_fp8_wmma.mmq_fp8_moe_gemm_scatter(
        x, w_packed, scales, w_zeros, sorted_token_ids, expert_ids, num_tokens_post_padded,
        topk_weights, output, top_k, block_m, _resolve_moe_kernel(kernel), weight_is_e2m1)


def mmq_fp8_moe_gather_reduce(out2, sorted_token_ids, topk_weights, num_tokens_post_padded,
                              top_k):
    """Topk-weighted gather-reduce: (P, N) fp16, bf16 or fp32 rows -> (M, N) fp32,
    M = numel(w) // top_k."""
    return torch.ops.w4a8_fp8_wmma.mmq_fp8_moe_gather_reduce(
        out2, sorted_token_ids, topk_weights, num_tokens_post_padded, top_k)


# ---- B200-build extras: the two kernels the reference takes from vLLM / runs implicitly ----

def act_quant_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-token e4m3 quantisation: (M, K) fp16 -> (uint8 e4m3 bytes (M, K), fp32 scales (M,))."""
    q, s = torch.ops.w4a8_b200.act_quant_fp8(x)
    return q, s


def moe_align_block_size(topk_ids: torch.Tensor, block_m: int, num_experts: int,
                         expert_map: torch.Tensor | None = None,
                         num_local_experts: int | None = None):
    """Deterministic moe_align_block_size -> (sorted_token_ids, expert_ids, ntp).

    Order: experts ascending, slot ids ascending inside an expert, runs padded to block_m with
    the sentinel topk_ids.numel(). With ``expert_map`` (global -> local id, -1 = remote) only
    local slots are kept and expert_ids hold local ids. Capacity is
    round_up(numel + E_local * (block_m - 1), block_m); entries past ntp hold the sentinel / -1.
    """
    ids = topk_ids.to(torch.int32).contiguous()
    n_local = int(num_local_experts) if num_local_experts is not None else int(num_experts)
    s, e, n = torch.ops.w4a8_b200.moe_align_block_size(ids, int(block_m), int(num_experts),
                                                       expert_map, n_local)
    return s, e, n


def silu_and_mul(x: torch.Tensor) -> torch.Tensor:
    """(M, 2*inter) fp16 [gate | up] -> (M, inter): fp16(g / (1 + exp(-g))) * up, the unfused
    activation step between gate_up and down (the fused gate_up op applies the same epilogue)."""
    return torch.ops.w4a8_b200.silu_and_mul(x.contiguous())


def route_topk(logits: torch.Tensor, top_k: int, renormalize: bool = True):
    """The MoE router in one launch: (T, E) fp32/fp16/bf16 logits -> topk_ids (T, top_k) int32,
    topk_weights (T, top_k) fp32 (softmax, the top_k largest with ties to the lower expert,
    renormalised) and expert_counts (E,) int32, the slots routed to each expert. It produces the
    inputs vLLM's router hands to the reference's moe_align call (moe_experts.py:587-589)."""
    ids, w, counts = torch.ops.w4a8_b200.route_topk(logits.contiguous(), int(top_k),
                                                    bool(renormalize))
    return ids, w, counts


# ---- Block-scaled FP8: the layers that a mixed checkpoint keeps in 8 bits ----
# e4m3 values (float8_e4m3fn, or their uint8 bytes) with one fp32 scale per 128 columns of an
# activation row and per 128 x 128 block of a weight; the last block of a side may be short.

# the overloads themselves: looking them up at each call costs as much as a decode-size kernel
_act_quant_fp8_block_op = torch.ops.w4a8_b200.act_quant_fp8_block.default
_rms_norm_quant_fp8_op = torch.ops.w4a8_b200.rms_norm_quant_fp8.default
_fp8_block_gemm_op = torch.ops.w4a8_b200.fp8_block_gemm.default
_fp8_block_moe_gemm_op = torch.ops.w4a8_b200.fp8_block_moe_gemm.default
_fp8_block_moe_gemm1_silu_op = torch.ops.w4a8_b200.fp8_block_moe_gemm1_silu.default


def act_quant_fp8_block(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(M, K) fp16/bf16/fp32 -> (q (M, K) float8_e4m3fn, scales (M, ceil(K/128)) fp32): the rule
    of act_quant_fp8 applied to each 128 columns of a row."""
    return tuple(_act_quant_fp8_block_op(x))


def rms_norm_quant_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                       residual: torch.Tensor | None = None, with_normed: bool = False):
    """RMS norm with the residual's addition and a block-scaled e4m3 output, in one pass.

    h = x + residual (rounded to x's type; h = x without one), y = h * rsqrt(mean(h^2) + eps) *
    weight in fp32. Returns (q (M, H) float8_e4m3fn, scales (M, ceil(H/128)) fp32, h as the new
    residual or None, y in x's type if with_normed else None). x and residual fp16, bf16 or
    fp32; weight in x's type or fp32.
    """
    q, s, res, normed = _rms_norm_quant_fp8_op(x, weight, eps, residual, with_normed)
    return q, s, (res if residual is not None else None), (normed if with_normed else None)


def fp8_block_gemm(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor,
                   w_scales: torch.Tensor, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Dense block-scaled FP8 GEMM: (M, K) e4m3 x (N, K) e4m3 -> (M, N) fp16, bf16 or fp32.

    x_scales (M, ceil(K/128)), w_scales (ceil(N/128), ceil(K/128)), fp32. Sums are held in fp32
    and rounded once. K a multiple of 16 takes the tensor cores; any other K is served by a
    plain kernel.
    """
    return _fp8_block_gemm_op(x, x_scales, w, w_scales, out_dtype)


def fp8_block_moe_gemm(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                       num_tokens_post_padded, top_k: int, block_m: int,
                       out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Grouped block-scaled FP8 GEMM: out[r] = x[sorted_token_ids[r] // top_k] @ W[expert(r)]^T.

    x (T, K) e4m3, w (E, N, K) e4m3, w_scales (E, ceil(N/128), ceil(K/128)); routing tensors in
    the moe_align_block_size layout, block_m 16, 32, 64 or a multiple of 128. sorted_token_ids
    None: x has P rows that are already in sorted order. Returns (P, N); padding rows and rows of
    an expert id outside [0, E) are zero, rows past num_tokens_post_padded are not written.
    """
    return _fp8_block_moe_gemm_op(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                                  num_tokens_post_padded, top_k, block_m, out_dtype)


def fp8_block_moe_gemm1_silu(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                             num_tokens_post_padded, top_k: int, block_m: int):
    """Grouped gate_up GEMM + silu_and_mul + block quantisation: w (E, 2*inter, K) = [gate | up].

    Returns (q (P, inter) float8_e4m3fn, scales (P, inter/128) fp32), what fp8_block_moe_gemm
    reads for the down product. silu(gate) * up is evaluated in fp32 and rounded once, to e4m3.
    inter must be a multiple of 128; the rest as fp8_block_moe_gemm.
    """
    return tuple(_fp8_block_moe_gemm1_silu_op(x, x_scales, w, w_scales, sorted_token_ids,
                                              expert_ids, num_tokens_post_padded, top_k, block_m))


# ---- Fake / meta impls (output contracts of the CUDA impls, reference __init__.py:240-297) ----
_register_fake = getattr(getattr(torch, "library", None), "register_fake", None)
if _register_fake is not None:
    @_register_fake("w4a8_fp8_wmma::mmq_fp8_gemm")
    def _fake_mmq_fp8_gemm(x, w_packed, scales, w_zeros, kernel, weight_is_e2m1=False):
        return x.new_empty((x.shape[0], w_packed.shape[0]), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_regdirect_fp8")
    def _fake_mmq_regdirect_fp8(x, w_rep, scales, w_zeros, N):
        return x.new_empty((x.shape[0], N), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_regdirect_f16")
    def _fake_mmq_regdirect_f16(x, w_rep, scales, w_zeros, N):
        return x.new_empty((x.shape[0], N), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_regdirect_w4a16")
    def _fake_mmq_regdirect_w4a16(x, w_rep, scales, w_zeros, N):
        return x.new_empty((x.shape[0], N), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_fp8_moe_gemm")
    def _fake_mmq_fp8_moe_gemm(x, w_packed, scales, w_zeros, sorted_token_ids, expert_ids,
                               num_tokens_post_padded, top_k, block_m, kernel,
                               weight_is_e2m1=False):
        return x.new_empty((sorted_token_ids.shape[0], w_packed.shape[1]), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_fp8_moe_gemm1_silu")
    def _fake_mmq_fp8_moe_gemm1_silu(x, w_packed, scales, w_zeros, sorted_token_ids,
                                     expert_ids, num_tokens_post_padded, top_k, block_m, kernel,
                                     weight_is_e2m1=False):
        return x.new_empty((sorted_token_ids.shape[0], w_packed.shape[1] // 2),
                           dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_fp8_moe_gemm_scatter")
    def _fake_mmq_fp8_moe_gemm_scatter(x, w_packed, scales, w_zeros, sorted_token_ids,
                                       expert_ids, num_tokens_post_padded, topk_weights, output,
                                       top_k, block_m, kernel, weight_is_e2m1=False):
        return None

    @_register_fake("w4a8_b200::route_topk")
    def _fake_route_topk(logits, top_k, renormalize):
        T, E = logits.shape
        return [logits.new_empty((T, top_k), dtype=torch.int32),
                logits.new_empty((T, top_k), dtype=torch.float32),
                logits.new_empty((E,), dtype=torch.int32)]

    @_register_fake("w4a8_b200::silu_and_mul")
    def _fake_silu_and_mul(x):
        return x.new_empty((x.shape[0], x.shape[1] // 2), dtype=torch.float16)

    @_register_fake("w4a8_fp8_wmma::mmq_fp8_moe_gather_reduce")
    def _fake_mmq_fp8_moe_gather_reduce(out2, sorted_token_ids, topk_weights,
                                        num_tokens_post_padded, top_k):
        return out2.new_empty((topk_weights.shape[0] // top_k, out2.shape[1]),
                              dtype=torch.float32)

    def _blocks(n):
        return (n + 127) // 128

    @_register_fake("w4a8_b200::act_quant_fp8_block")
    def _fake_act_quant_fp8_block(x):
        M, K = x.shape
        return [x.new_empty((M, K), dtype=torch.float8_e4m3fn),
                x.new_empty((M, _blocks(K)), dtype=torch.float32)]

    @_register_fake("w4a8_b200::rms_norm_quant_fp8")
    def _fake_rms_norm_quant_fp8(x, weight, eps, residual, with_normed):
        M, H = x.shape
        return [x.new_empty((M, H), dtype=torch.float8_e4m3fn),
                x.new_empty((M, _blocks(H)), dtype=torch.float32),
                x.new_empty((M if residual is not None else 0, H)),
                x.new_empty((M if with_normed else 0, H))]

    @_register_fake("w4a8_b200::fp8_block_gemm")
    def _fake_fp8_block_gemm(x, x_scales, w, w_scales, out_dtype):
        return x.new_empty((x.shape[0], w.shape[0]), dtype=out_dtype)

    @_register_fake("w4a8_b200::fp8_block_moe_gemm")
    def _fake_fp8_block_moe_gemm(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                                 num_tokens_post_padded, top_k, block_m, out_dtype):
        P = (x if sorted_token_ids is None else sorted_token_ids).shape[0]
        return x.new_empty((P, w.shape[1]), dtype=out_dtype)

    @_register_fake("w4a8_b200::fp8_block_moe_gemm1_silu")
    def _fake_fp8_block_moe_gemm1_silu(x, x_scales, w, w_scales, sorted_token_ids, expert_ids,
                                       num_tokens_post_padded, top_k, block_m):
        P = (x if sorted_token_ids is None else sorted_token_ids).shape[0]
        inter = w.shape[1] // 2
        return [x.new_empty((P, inter), dtype=torch.float8_e4m3fn),
                x.new_empty((P, _blocks(inter)), dtype=torch.float32)]
