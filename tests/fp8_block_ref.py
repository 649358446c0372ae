"""Block-scaled FP8 operators from their definitions in 64 bits, with the error each fp32 kernel
result may have; shared by the CPU and the GPU tests.

Error model. e4m3 x e4m3 products are exact in fp32. A tensor-core step adds 32 of them and the
accumulator, each aligned to the largest and cut at fp32's 24 bits, so it is off by at most
33 * 2^-23 of the sum of the absolute values; a block of 128 takes 4 such steps. Folding G scaled
block sums adds one rounding each (2^-24), the two scales' product one more. With S = sum_g xs ws
sum_k |x w| the fp32 result is within SUM(G) * S of the exact one. A rounding to a type of relative
step eps adds eps / 2 of the value; e4m3's half step is 2^-4 of the value, at least 2^-10."""
from __future__ import annotations

import torch

BLOCK = 128
FLOOR = 4.48e-6
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def sum_error(G: int) -> float:
    return 4 * 33 * 2.0 ** -23 + (G + 3) * 2.0 ** -24


def blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def spread_cols(s, cols):
    return s.repeat_interleave(BLOCK, -1)[..., :cols]


def spread_w(s, rows, cols):
    return spread_cols(s, cols).repeat_interleave(BLOCK, -2)[..., :rows, :]


def e4m3(shape, gen, device="cpu"):
    """Random finite e4m3 values of every exponent, both signs."""
    b = torch.randint(0, 256, shape, generator=gen, device=device, dtype=torch.int32)
    b = torch.where((b & 0x7F) == 0x7F, b - 1, b)
    return b.to(torch.uint8).view(torch.float8_e4m3fn)


def quantise(y, row_block=1):
    """(..., R, C) -> e4m3 values and scales per row_block x 128."""
    r, c = y.shape[-2:]
    rb, cb = (r + row_block - 1) // row_block, blocks(c)
    p = torch.nn.functional.pad(y, (0, cb * BLOCK - c, 0, rb * row_block - r))
    s = p.reshape(p.shape[:-2] + (rb, row_block, cb, BLOCK)).abs().amax((-3, -1))
    s = s.float().clamp_min(FLOOR)
    s = s / torch.full_like(s, 448.0)  # a true divide: by a Python number it is a multiplication
    f = spread_cols(s, c).repeat_interleave(row_block, -2)[..., :r, :]
    return (y / f).to(torch.float8_e4m3fn), s


def product(x, xs, w, ws):
    """(out, S): the scaled product and the sum of absolute terms, fp64."""
    k = x.shape[-1]
    a = x.double() * spread_cols(xs.double(), k)
    b = w.double() * spread_w(ws.double(), w.shape[-2], k)
    return a @ b.T, a.abs() @ b.abs().T


def grouped(x, xs, w, ws, sorted_ids, expert_ids, rows, top_k, block_m):
    """(out, S) of the first `rows` rows of the grouped product; zero rows are exact zeros."""
    E, N, T = w.shape[0], w.shape[1], x.shape[0]
    out = torch.zeros(rows, N, dtype=torch.float64, device=x.device)
    S = torch.zeros_like(out)
    live = torch.zeros(rows, dtype=torch.bool, device=x.device)
    for b in range((rows + block_m - 1) // block_m):
        lo, hi = b * block_m, min(rows, (b + 1) * block_m)
        e = int(expert_ids[b])
        if e < 0 or e >= E:
            continue
        if sorted_ids is None:
            ok, src = torch.ones(hi - lo, dtype=torch.bool, device=x.device), torch.arange(lo, hi, device=x.device)
        else:
            slot = sorted_ids[lo:hi].long()
            ok = (slot >= 0) & (slot < T * top_k)
            src = torch.where(ok, slot // top_k, 0)
        o, s = product(x[src], xs[src], w[e], ws[e])
        out[lo:hi] = torch.where(ok[:, None], o, 0.0)
        S[lo:hi] = torch.where(ok[:, None], s, 0.0)
        live[lo:hi] = ok
    return out, S, live


def silu_mul(out, S, err):
    """h = silu(gate) * up and how far the fp32 kernel's may be off, from the product and err * S."""
    inter = out.shape[1] // 2
    g, u = out[:, :inter], out[:, inter:]
    dg, du = err * S[:, :inter], err * S[:, inter:]
    sil = g * torch.sigmoid(g)
    h = sil * u
    # |silu'| <= 1.1; exp, divide and the two products: 8 units of 2^-24, and exp's argument
    # error |g| 2^-24
    rel = (8 + g.abs()) * 2.0 ** -24
    return h, 1.1 * dg * (u.abs() + du) + sil.abs() * du + rel * h.abs()


def check_out(got, want, S, G, dtype):
    tol = sum_error(G) * S
    tol = tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype]
    over = want.abs() + tol >= torch.finfo(dtype).max  # may round to an infinity
    bad = ((got.double() - want).abs() > tol) & ~over
    assert not bool(bad.any()), f"{int(bad.sum())} outputs outside the derived bound"


def check_quant(q, s, y, dy):
    """q, s (values, scales) against y (fp64) that the kernel knows within dy."""
    c = y.shape[1]
    pad = blocks(c) * BLOCK - c
    shape = (y.shape[0], blocks(c), BLOCK)
    p = torch.nn.functional.pad(y, (0, pad)).reshape(shape)
    d = torch.nn.functional.pad(dy, (0, pad)).reshape(shape)
    want = p.abs().amax(2).clamp_min(FLOOR) / 448.0
    assert bool(((s.double() - want).abs() <= d.amax(2) / 448.0 + 2.0 ** -23 * want).all()), "scales"
    f = spread_cols(s.double(), c)
    v = (y / f).abs()
    tol = torch.clamp_min(v * 2.0 ** -4, 2.0 ** -10) * (1 + 2.0 ** -9) * f + dy * 1.0625 + 2.0 ** -22 * y.abs()
    bad = (q.double() * f - y).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} quantised values outside the derived bound"


def align(ids, num_experts, block_m, spare=0):
    """moe_align_block_size on the host: sorted ids and expert ids with `spare` blocks behind the
    last used one (sentinel / -1), and the padded row count."""
    slots = ids.numel()
    flat = ids.reshape(-1).tolist()
    rows, experts = [], []
    for e in range(num_experts):
        mine = [i for i, v in enumerate(flat) if v == e]
        mine += [slots] * (-len(mine) % block_m)
        rows += mine
        experts += [e] * (len(mine) // block_m)
    n = len(rows)
    rows += [slots] * (spare * block_m)
    experts += [-1] * spare
    as_i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return as_i32(rows), as_i32(experts), as_i32([n])
