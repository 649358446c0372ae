"""The FP8 block-scaled operators, case by case: what each one computes and what it costs.

Block-scaled FP8 holds a matrix as e4m3 values with one fp32 scale per block: activations per
(row, 128 columns), weights per (128 rows, 128 columns), the last block of a side may be short.
The operators are the activation quantisation, the RMS norm that quantises its output, the dense
product, the product grouped by expert, and the grouped gate_up product fused with SiLU-and-mul
and the quantisation that the down product reads.

``own`` selects what ``run`` does: False computes the plain form in elementary torch operations,
True calls this package's operators.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 4.48e-6  # the package's clamp: a block of zeros gets the scale 1e-8
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
DEV = "cuda"


def listed():
    return [
        # one decoding token's attention output on its way to the output projection
        {"name": "quant-decode", "op": "quant", "M": 1, "K": 2048, "dtype": "fp16"},
        # a prefill batch's attention output, bf16 model
        {"name": "quant-prefill", "op": "quant", "M": 8192, "K": 4096, "dtype": "bf16"},
        # the norm before an MoE layer at decode batch 32: residual added, the normed rows kept
        # for the router
        {"name": "norm-decode", "op": "norm", "M": 32, "K": 2048, "dtype": "fp16",
         "residual": True, "normed": True},
        # the same norm over a long ragged prefill batch, before a dense projection
        {"name": "norm-prefill", "op": "norm", "M": 16381, "K": 2048, "dtype": "bf16",
         "residual": True, "normed": False},
        # attention input projection of one decoding token
        {"name": "gemm-decode", "op": "gemm", "M": 1, "N": 4096, "K": 2048, "dtype": "fp16"},
        # output projection of a decode batch of 128
        {"name": "gemm-batch", "op": "gemm", "M": 128, "N": 2048, "K": 4096, "dtype": "bf16"},
        # a short prompt through a layer whose sizes fill no tile: short blocks on both sides
        {"name": "gemm-ragged", "op": "gemm", "M": 333, "N": 1001, "K": 1424, "dtype": "fp16"},
        # a long prefill through the widest projection of the dense sweep
        {"name": "gemm-prefill", "op": "gemm", "M": 8192, "N": 8192, "K": 2048, "dtype": "bf16"},
        # the 256-expert top-8 layer, decode batch 32: gate_up with SiLU and quantised output
        {"name": "gateup-decode", "op": "gateup", "T": 32, "E": 256, "top_k": 8, "H": 2048,
         "I": 512, "zipf": False},
        # the same layer on a 4096-token prefill with skewed routing
        {"name": "gateup-prefill", "op": "gateup", "T": 4096, "E": 256, "top_k": 8, "H": 2048,
         "I": 512, "zipf": True},
        # the down product of that layer, decode and prefill
        {"name": "down-decode", "op": "down", "T": 32, "E": 256, "top_k": 8, "H": 2048, "I": 512,
         "zipf": False, "dtype": "fp16"},
        {"name": "down-prefill", "op": "down", "T": 4096, "E": 256, "top_k": 8, "H": 2048,
         "I": 512, "zipf": True, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["quant", "norm", "gemm", "gemm", "gateup", "down"])
    if op in ("quant", "norm"):
        k = log(128, 8192)
        k = k if rng.random() < 0.3 else k // 8 * 8 if rng.random() < 0.4 else k // 128 * 128
        m = min(log(1, 32768), 8192 * 4096 // k)
        case = {"op": op, "M": m, "K": k, "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"])}
        if case["dtype"] == "fp32":
            case["M"] = max(1, m // 2)
        if op == "norm":
            case["residual"] = rng.random() < 0.7
            case["normed"] = rng.random() < 0.5
        return case
    if op == "gemm":
        n, k = log(128, 8192), log(256, 8192) // 16 * 16
        n, k = (n if rng.random() < 0.2 else n // 64 * 64), (k if rng.random() < 0.2 else k // 128 * 128)
        m = min(log(1, 8192), 8192 * 8192 * 2048 // (n * k))
        return {"op": op, "M": m, "N": n, "K": k, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    e, top_k = log(8, 256), rng.randint(1, 8)
    h = log(256, 4096) // 128 * 128
    i = 128 * rng.randint(1, max(1, min(12, 2048 * 1024 // (2 * 128 * h))))
    t = min(log(1, 4096), 32768 // top_k)
    case = {"op": op, "T": t, "E": e, "top_k": top_k, "H": h, "I": i, "zipf": rng.random() < 0.5}
    if op == "down":
        case["dtype"] = rng.choice(["fp16", "bf16"])
    return case


# ---- inputs --------------------------------------------------------------------------------

def _up(n, m):
    return (n + m - 1) // m


def _spread(scales, rows, cols, row_block):
    """Block scales (..., ceil(rows/rb), ceil(cols/128)) as one factor per element."""
    s = scales.repeat_interleave(BLOCK, -1)[..., :cols]
    return s if row_block == 1 else s.repeat_interleave(row_block, -2)[..., :rows, :]


def _quantised(x, row_block):
    """fp32 (..., R, C) -> e4m3 values and block scales, as a checkpoint or a quantiser holds
    them."""
    r, c = x.shape[-2:]
    pr, pc = _up(r, row_block) * row_block - r, _up(c, BLOCK) * BLOCK - c
    p = torch.nn.functional.pad(x, (0, pc, 0, pr))
    b = p.reshape(p.shape[:-2] + (p.shape[-2] // row_block, row_block, p.shape[-1] // BLOCK, BLOCK))
    s = b.abs().amax(dim=(-3, -1)).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (x / _spread(s, r, c, row_block)).to(torch.float8_e4m3fn)
    return q, s


def _activations(gen, m, k, dtype):
    """Rows as a transformer has them: near normal, a few channels an order larger."""
    x = torch.randn(m, k, generator=gen, device=DEV)
    loud = torch.rand(k, generator=gen, device=DEV) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _weights(gen, *shape):
    """Weights ~ N(0, 1/K) with rows of different size, as e4m3 with 128 x 128 block scales."""
    w = torch.randn(*shape, generator=gen, device=DEV)
    w *= torch.rand(shape[:-1] + (1,), generator=gen, device=DEV) + 0.5
    w *= shape[-1] ** -0.5
    return _quantised(w, BLOCK)


def _expert_ids(case):
    """(T, top_k) experts from N(0, 1) router logits; zipf adds the prior rank^-1.1. The loads
    belong to the case; prepare() deals them to other experts and tokens for each seed."""
    gen = torch.Generator().manual_seed(0)
    logits = torch.randn(case["T"], case["E"], generator=gen)
    if case["zipf"]:
        logits -= 1.1 * torch.log(torch.arange(1, case["E"] + 1).float())
    return logits.topk(case["top_k"], dim=1).indices


def _block_m(case):
    """Row-block size of the grouped products: the smallest of 16..128 that holds twice the
    average expert's rows."""
    avg = case["T"] * case["top_k"] / case["E"]
    return next((b for b in (16, 32, 64) if b >= 2 * avg), 128)


def _routing(ids, num_experts, block_m):
    """(T, k) expert ids -> sorted slots, one expert per row block, the padded row count: slots
    ascending by expert, each expert's run padded to block_m with the sentinel T * k."""
    slots = ids.numel()
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=num_experts)
    padded = (counts + block_m - 1) // block_m * block_m
    start = torch.cumsum(padded, 0) - padded
    first = torch.cumsum(counts, 0) - counts
    total = int(padded.sum())
    sorted_ids = torch.full((total,), slots, dtype=torch.int32, device=ids.device)
    by = flat[order]
    at = start[by] + torch.arange(slots, device=ids.device) - first[by]
    sorted_ids[at] = order.to(torch.int32)
    experts = torch.repeat_interleave(torch.arange(num_experts, device=ids.device), padded // block_m)
    ntp = torch.tensor([total], dtype=torch.int32, device=ids.device)
    return sorted_ids, experts.to(torch.int32), ntp


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, s = case["op"], {"case": case}
    if op in ("quant", "norm"):
        dtype = DTYPES[case["dtype"]]
        s["x"] = _activations(gen, case["M"], case["K"], dtype)
        if op == "norm":
            s["weight"] = (1 + 0.2 * torch.randn(case["K"], generator=gen, device=DEV)).to(dtype)
            if case["residual"]:
                s["residual"] = _activations(gen, case["M"], case["K"], dtype) * 2
        return s
    if op == "gemm":
        s["x"], s["xs"] = _quantised(_activations(gen, case["M"], case["K"], torch.float32), 1)
        s["w"], s["ws"] = _weights(gen, case["N"], case["K"])
        return s
    deal = torch.randperm(case["E"], generator=gen, device=DEV)
    ids = deal[_expert_ids(case).to(DEV)][torch.randperm(case["T"], generator=gen, device=DEV)]
    s["block_m"], s["top_k"] = _block_m(case), ids.shape[1]
    s["sorted"], s["experts"], s["ntp"] = _routing(ids, case["E"], s["block_m"])
    if op == "gateup":
        s["x"], s["xs"] = _quantised(_activations(gen, case["T"], case["H"], torch.float32), 1)
        s["w"], s["ws"] = _weights(gen, case["E"], 2 * case["I"], case["H"])
    else:  # the down product reads rows that gate_up left in sorted order, padding rows zero
        rows = _activations(gen, s["sorted"].numel(), case["I"], torch.float32)
        rows *= (s["sorted"] < ids.numel())[:, None]
        s["x"], s["xs"] = _quantised(rows, 1)
        s["w"], s["ws"] = _weights(gen, case["E"], case["H"], case["I"])
    return s


# ---- one pass ------------------------------------------------------------------------------

def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-vllm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import w4a8_fp8_wmma
    return w4a8_fp8_wmma


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    w4, case = _package(), s["case"]
    op = case["op"]
    if op == "quant":
        q, scales = w4.act_quant_fp8_block(s["x"])
        return {"q": q, "scales": scales}
    if op == "norm":
        q, scales, res, normed = w4.rms_norm_quant_fp8(
            s["x"], s["weight"], 1e-6, residual=s.get("residual"), with_normed=case["normed"])
        return {"q": q, "scales": scales, "residual": res, "normed": normed}
    if op == "gemm":
        return w4.fp8_block_gemm(s["x"], s["xs"], s["w"], s["ws"], out_dtype=DTYPES[case["dtype"]])
    if op == "gateup":
        q, scales = w4.fp8_block_moe_gemm1_silu(s["x"], s["xs"], s["w"], s["ws"], s["sorted"],
                                                s["experts"], s["ntp"], s["top_k"], s["block_m"])
        return {"q": q, "scales": scales}
    return w4.fp8_block_moe_gemm(s["x"], s["xs"], s["w"], s["ws"], None, s["experts"], s["ntp"], 1,
                                 s["block_m"], out_dtype=DTYPES[case["dtype"]])


def _plain_quant(y):
    """fp32 (R, C) -> e4m3 values, (R, ceil(C/128)) scales: amax / 448 over each 128 columns."""
    r, c = y.shape
    g = _up(c, BLOCK)
    b = torch.nn.functional.pad(y, (0, g * BLOCK - c)).reshape(r, g, BLOCK)
    scales = b.abs().amax(dim=2).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (b / scales[:, :, None]).reshape(r, g * BLOCK)[:, :c].to(torch.float8_e4m3fn)
    return q, scales


def _plain_grouped(s):
    """(blocks, block_m, N) fp32 products of each row block with its expert's matrix."""
    k = s["x"].shape[1]
    x = s["x"].float() * _spread(s["xs"], 0, k, 1)
    if s["case"]["op"] == "gateup":
        real = s["sorted"] < s["x"].shape[0] * s["top_k"]
        x = x[(s["sorted"] // s["top_k"]).clamp_max(x.shape[0] - 1)] * real[:, None]
    w = s["w"].float() * _spread(s["ws"], s["w"].shape[1], k, BLOCK)
    return torch.bmm(x.reshape(-1, s["block_m"], k), w[s["experts"]].transpose(1, 2))


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quant":
        q, scales = _plain_quant(s["x"].float())
        return {"q": q, "scales": scales}
    if op == "norm":
        h = s["x"].float()
        if case["residual"]:
            h = (h + s["residual"].float()).to(s["x"].dtype)
            res, h = h, h.float()
        y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-6) * s["weight"].float()
        q, scales = _plain_quant(y)
        return {"q": q, "scales": scales, "residual": res if case["residual"] else None,
                "normed": y.to(s["x"].dtype) if case["normed"] else None}
    if op == "gemm":
        x = s["x"].float() * _spread(s["xs"], 0, case["K"], 1)
        w = s["w"].float() * _spread(s["ws"], case["N"], case["K"], BLOCK)
        return (x @ w.t()).to(DTYPES[case["dtype"]])
    y = _plain_grouped(s)
    y = y.reshape(-1, y.shape[2])
    if op == "down":
        return y.to(DTYPES[case["dtype"]])
    gate, up = y[:, :case["I"]], y[:, case["I"]:]
    q, scales = _plain_quant(gate / (1 + torch.exp(-gate)) * up)
    return {"q": q, "scales": scales}


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("quant", "norm"):
        m, k, b = case["M"], case["K"], SIZE[case["dtype"]]
        moved = m * k * b + m * k + m * _up(k, BLOCK) * 4
        if op == "norm":
            moved += k * b + m * k * b * (2 * case["residual"] + case["normed"])
        return {"bytes": moved, "flops": m * k * (8 if op == "norm" else 3)}
    if op == "gemm":
        m, n, k = case["M"], case["N"], case["K"]
        g = _up(k, BLOCK)
        return {"bytes": m * k + 4 * m * g + n * k + 4 * _up(n, BLOCK) * g + m * n * SIZE[case["dtype"]],
                "flops": 2 * m * n * k}
    ids = _expert_ids(case)
    touched, rows = int(torch.unique(ids).numel()), ids.numel()
    k, n = (case["H"], 2 * case["I"]) if op == "gateup" else (case["I"], case["H"])
    weights = touched * (n * k + 4 * _up(n, BLOCK) * _up(k, BLOCK))
    if op == "gateup":
        acts = case["T"] * (k + 4 * _up(k, BLOCK)) + rows * (case["I"] + 4 * _up(case["I"], BLOCK))
    else:
        acts = rows * (k + 4 * _up(k, BLOCK)) + rows * n * SIZE[case["dtype"]]
    return {"bytes": weights + acts, "flops": 2 * rows * n * k}


# ---- the definitions in 64 bits --------------------------------------------------------------

def _round_e4m3(v):
    """Nearest e4m3 value, ties to the even mantissa: 3 mantissa bits, exponents from 2^-6,
    below that steps of 2^-9, at most 448."""
    exponent = torch.frexp(v.abs()).exponent.double() - 1
    step = torch.exp2(exponent.clamp_min(-6.0) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quant(y):
    cols, scales = [], []
    for lo in range(0, y.shape[1], BLOCK):
        part = y[:, lo:lo + BLOCK]
        sc = torch.clamp(part.abs().max(dim=1).values, min=AMAX_FLOOR) / E4M3_MAX
        scales.append(sc)
        cols.append(_round_e4m3(part / sc[:, None]))
    return torch.cat(cols, 1), torch.stack(scales, 1)


def _exact_product(x, xs, w, ws):
    """sum over blocks g of xs[:, g] ws[:, g] (x_g @ w_g^T), in 64 bits."""
    out = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    rows = torch.arange(w.shape[0], device=x.device) // BLOCK
    for g, lo in enumerate(range(0, x.shape[1], BLOCK)):
        part = x[:, lo:lo + BLOCK].double() @ w[:, lo:lo + BLOCK].double().t()
        out += part * xs[:, g, None].double() * ws[rows, g].double()
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quant":
        q, scales = _exact_quant(s["x"].double())
        return {"q": q, "scales": scales}
    if op == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = (h + s["residual"].double()).to(s["x"].dtype).double()
        size = (torch.sum(h * h, dim=1, keepdim=True) / case["K"] + 1e-6) ** 0.5
        y = h / size * s["weight"].double()
        q, scales = _exact_quant(y)
        return {"q": q, "scales": scales, "residual": h if case["residual"] else None,
                "normed": y if case["normed"] else None}
    if op == "gemm":
        return _exact_product(s["x"], s["xs"], s["w"], s["ws"])
    bm, blocks = s["block_m"], s["experts"].tolist()
    outs = []
    for b, e in enumerate(blocks):
        if op == "gateup":
            ids = s["sorted"][b * bm:(b + 1) * bm].long()
            real = ids < s["x"].shape[0] * s["top_k"]
            src = torch.where(real, ids // s["top_k"], 0)
            y = _exact_product(s["x"][src], s["xs"][src], s["w"][e], s["ws"][e])
            gate, up = torch.split(torch.where(real[:, None], y, 0.0), case["I"], dim=1)
            outs.append(gate * torch.sigmoid(gate) * up)
        else:
            at = slice(b * bm, (b + 1) * bm)
            outs.append(_exact_product(s["x"][at], s["xs"][at], s["w"][e], s["ws"][e]))
    y = torch.cat(outs)
    if op == "down":
        return y
    q, scales = _exact_quant(y)
    return {"q": q, "scales": scales}
