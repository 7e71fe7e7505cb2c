"""Plain 64-bit forms of the block-scaled linear, the head norms with rotation, and attention over pages (CPU), with
bounds on how far a kernel of the stated precision may be from them."""

from __future__ import annotations

import math

import torch

BLOCK = 128
STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}    # half a unit in the last place, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half of the smallest subnormal


def block_quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [M, K] e4m3fn, scale [M, ceil(K / 128)]) of bf16 x: fp32 arithmetic as defined, bit for bit."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    padded = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    amax = padded.abs().amax(-1)
    scale = torch.where(amax < 1e-12, torch.tensor(1e-12), amax) / torch.tensor(448.0)
    codes = (padded / scale[..., None]).view(m, -1)[:, :k].contiguous()
    return codes.to(torch.float8_e4m3fn), scale


def block_gemm(codes, scale, weight, weight_scale, bias=None):
    """(y [M, N], bound) in 64 bits.  Bound: half a step of bf16; of the sum of the products' magnitudes 2^-16 (128 fp32
    additions of 2^-23 at worst inside a block) and 2^-23 for each block's scaling and addition; and what the fp8 matrix
    instruction of this hardware leaves out.  It adds the products of eight neighbouring k at the granularity of 2^(e - 13), e
    the largest sum of two factors' exponents among them, cutting off toward zero (probed with 448 * 448 - 448 * 448 + v: v = 8 is kept,
    15 becomes 8, 4 becomes 0, for v among the same eight k and for no other).  The largest product p >= 2^e is kept whole, so
    each of the seven others loses less than 2^-13 p."""
    m, k = codes.shape
    n, blocks = weight.shape[0], -(-k // BLOCK)
    y, mass, cut = (torch.zeros(m, n, dtype=torch.float64) for _ in range(3))
    for g in range(blocks):
        part = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
        f = scale[:, g if scale.shape[1] > 1 else 0].double()[:, None] * weight_scale[:, g].double().repeat_interleave(BLOCK)[:n][None, :]
        a, w = codes[:, part].float(), weight[:, part].float()
        y += f * (a.double() @ w.double().t())
        a, w = a.abs(), w.abs()
        mass += f * (a.double() @ w.double().t())
        largest = torch.zeros(m, n)
        for i in range(0, a.shape[1], 8):
            largest += (a[:, None, i: i + 8] * w[None, :, i: i + 8]).amax(-1)
        cut += f * largest.double()
    if bias is not None:
        y += bias.double()
        mass += bias.double().abs()
    return y, 2.0 ** -8 * y.abs() + (2.0 ** -16 + (blocks + 2) * 2.0 ** -23) * mass + 7 * 2.0 ** -13 * cut + 2.0 ** -134


def block_weight(n: int, k: int, gen) -> tuple[torch.Tensor, torch.Tensor]:
    blocks = (-(-n // BLOCK), -(-k // BLOCK))
    codes = (torch.randn(n, k, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, torch.rand(*blocks, generator=gen) * 2e-4 + 1e-5


def head_rope(x, weight, cos_sin, positions, eps, gemma, interleaved):
    """(heads [T, H, D] in 64 bits, bound) of x [T, H, D].  Bound: half a step of the type, and 2^-18 of the turned pair's
    magnitudes (a few fp32 roundings each of the sum of squares of up to 512 terms, the root, the products and the sum)."""
    x64 = x.double()
    if weight is not None:
        x64 = x64 / torch.sqrt(x64.square().mean(-1, keepdim=True) + eps) * (weight.double() + (1.0 if gemma else 0.0))
    rot = cos_sin.shape[1]
    angles = cos_sin[positions].double()[:, None]
    cos, sin = angles[..., : rot // 2], angles[..., rot // 2:]
    y, mass = x64.clone(), x64.abs()
    a = torch.arange(rot // 2) * 2 if interleaved else torch.arange(rot // 2)
    b = a + (1 if interleaved else rot // 2)
    if rot:
        y[..., a], y[..., b] = x64[..., a] * cos - x64[..., b] * sin, x64[..., b] * cos + x64[..., a] * sin
        both = x64[..., a].abs() + x64[..., b].abs()
        mass[..., a], mass[..., b] = both, both
    return y, STEP[x.dtype] * y.abs() + 2.0 ** -18 * mass + TINY[x.dtype]


def paged_attention(q, k_pages, v_pages, page_table, q_offsets, kv_lens, *, scale=None, causal=True, window=None):
    """(out [T, H, D] in 64 bits with NaN in rows of no sequence, bound).  Bound: half a step of the type for the result, and of
    sum_j p_j |v_j| half a step for the rounding of each probability plus 2^-9 of what the scores' own errors move it: D
    products and sums of at most 2^-23 of sum_d |q_d k_d| scale < 2^7 in these tests, at D <= 256: 2^-8 would be the worst
    case, with the products' errors all of one sign; half of it is allowed."""
    T, H, D = q.shape
    page, kv_heads = k_pages.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), math.nan, dtype=torch.float64)
    bound = torch.full((T, H, D), math.nan, dtype=torch.float64)
    for b in range(kv_lens.numel()):
        q0, q1 = int(q_offsets[b]), int(q_offsets[b + 1])
        n = q1 - q0
        kv = min(int(kv_lens[b]), page_table.shape[1] * page)
        ids = page_table[b, : -(-kv // page)].long()
        k = k_pages[ids].reshape(-1, kv_heads, D)[:kv].double()
        v = v_pages[ids].reshape(-1, kv_heads, D)[:kv].double()
        for i in range(n):
            position = kv - n + i
            last = min(kv, position + 1) if causal else kv
            first = max(0, position - window + 1) if window else 0
            if last <= first:
                out[q0 + i], bound[q0 + i] = 0.0, 0.0
                continue
            for h in range(H):
                kh, vh = k[first:last, h // (H // kv_heads)], v[first:last, h // (H // kv_heads)]
                p = torch.softmax(kh @ q[q0 + i, h].double() * scale, dim=0)
                o, mass = p @ vh, p @ vh.abs()
                out[q0 + i, h] = o
                bound[q0 + i, h] = STEP[q.dtype] * o.abs() + (STEP[q.dtype] + 2.0 ** -9) * mass + TINY[q.dtype]
    return out, bound
