"""Plain 64-bit forms (CPU) of the residual's norm with its quantizer, of a cache in 8 bits, and of attention with capped scores,
prompts that are seen whole and such a cache; with bounds on how far a kernel of the stated precision may be from them."""

from __future__ import annotations

import math

import torch

from layer_oracle import STEP, TINY

BLOCK = 128
E4M3_HALF, E4M3_SMALL = 2.0 ** -4, 2.0 ** -10     # half a step of e4m3: of a normal value, of the subnormal ones


def codes_as_values(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).float().double()


def widen(codes: torch.Tensor, power: torch.Tensor) -> torch.Tensor:
    """What codes [..., D] with the bytes power [...] stand for."""
    by = torch.exp2(power.view(torch.uint8).double() - 127)
    return codes_as_values(codes) * torch.where(power.view(torch.uint8) == 255, math.nan, by)[..., None]


def to_cache(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, bytes) of heads x [..., D] in fp32 (values of the element type as they are): bit for bit."""
    x = x.float()
    if x.dtype != torch.float32:
        raise TypeError
    amax = x.abs().amax(-1)
    part, exponent = torch.frexp(amax)                       # amax = part 2^exponent, part in [0.5, 1)
    byte = torch.where(part <= 0.875, exponent - 9, exponent - 8) + 127
    byte = torch.where(amax > 0, byte.clamp_min(1), 1)
    known = torch.isfinite(x).all(-1)
    byte = torch.where(known, byte, 127)
    codes = (x.double() * torch.exp2(127.0 - byte.double())[..., None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(known[..., None], codes, 0x7F).to(torch.uint8), byte.to(torch.uint8)


def check_cache(codes, power, x, slack, what=""):
    """Codes and bytes of heads whose values are x [..., D] in 64 bits, known to +- slack (the fp32 arithmetic before): the byte is the smallest that
    keeps the largest magnitude within 448, each value half a step of its code off at most."""
    byte = power.cpu().view(torch.uint8).double()
    unit = torch.exp2(byte - 127)
    amax, wide = x.abs().amax(-1), slack.amax(-1)
    assert bool((amax - wide <= 448 * unit).all()), f"{what}: a power is too small"
    assert bool(((byte == 1) | (amax + wide > 224 * unit)).all()), f"{what}: a power is too large"
    off = (codes_as_values(codes.cpu()) * unit[..., None] - x).abs()
    bound = torch.maximum(E4M3_HALF * (x.abs() + slack), E4M3_SMALL * unit[..., None]) + slack
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} values outside, worst {(off - bound)[bad].max():.3e}"


def add_norm(x, residual, weight, eps, gemma):
    """(total as bf16, n in 64 bits)."""
    total = (x.double() + residual.double()).to(torch.bfloat16)
    t = total.double()
    return total, t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * (weight.double() + (1.0 if gemma else 0.0))


def check_norm_codes(codes, scale, n, per_block):
    """A scale is fp32 of the largest magnitude over 448; a code's value is half a step off at most.  Before that: the sum of D
    squares, in which no term passes more than 64 additions of fp32 (each 2^-24), its root (half of that), a division, two products and a sum
    of 2^-24 each: 2^-18 in all."""
    m, d = n.shape
    width = BLOCK if per_block else d
    groups = -(-d // width)
    padded = torch.nn.functional.pad(n, (0, groups * width - d)).view(m, groups, width)
    want = padded.abs().amax(-1).clamp_min(1e-12) / 448.0
    got = scale.cpu().double()
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= 2.0 ** -18 * want).all()), float(((got - want).abs() / want).max())
    per = got.repeat_interleave(width, 1)[:, :d]
    off = (codes_as_values(codes.cpu()) * per - n).abs()
    bound = torch.maximum(E4M3_HALF * n.abs() * (1 + 2.0 ** -17), E4M3_SMALL * per * (1 + 2.0 ** -17)) + 2.0 ** -17 * n.abs()
    bad = ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), float((off - bound)[bad].max()))


def attention(q, k_pages, v_pages, page_table, q_offsets, kv_lens, *, scale=None, causal=True, window=None, k_scales=None, v_scales=None,
              softcap=None, prefix_lens=None, shared_prefix=0):
    """(out [T, H, D] in 64 bits with NaN in rows of no sequence, bound).  Bound: half a step of the type for the result, and of
    sum_j p_j |v_j| half a step for the rounding of each probability plus 2^-9 of what the scores' own errors move it: D
    products and sums of at most 2^-23 of sum_d |q_d k_d| scale < 2^7 in these tests, at D <= 256: 2^-8 would be the worst case, with
    the products' errors all of one sign; half of it is allowed.  A cap makes score errors smaller (its slope is at most one) and
    adds 2^-21 of itself: cap 50 in base 2, 2^-15, which is nothing beside 2^-9."""
    T, H, D = q.shape
    page, kv_heads = k_pages.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    if k_scales is not None:
        k_pages, v_pages = (widen(p, s).to(q.dtype).double() for p, s in ((k_pages, k_scales), (v_pages, v_scales)))
    out = torch.full((T, H, D), math.nan, dtype=torch.float64)
    bound = torch.full((T, H, D), math.nan, dtype=torch.float64)
    for b in range(kv_lens.numel()):
        q0, q1 = int(q_offsets[b]), int(q_offsets[b + 1])
        n, length = q1 - q0, max(0, int(kv_lens[b]))
        kv = min(length, page_table.shape[1] * page)
        ids = page_table[b, : -(-kv // page)].long()
        k = k_pages[ids].reshape(-1, kv_heads, D)[:kv].double().repeat_interleave(H // kv_heads, 1)
        v = v_pages[ids].reshape(-1, kv_heads, D)[:kv].double().repeat_interleave(H // kv_heads, 1)
        prompt = min(kv, int(prefix_lens[b])) if prefix_lens is not None else 0
        for i in range(n):
            position = length - n + i
            last = min(kv, max(position + 1, prompt)) if causal else kv
            first = max(0, position - window + 1) if window else 0
            if last <= first:
                out[q0 + i], bound[q0 + i] = 0.0, 0.0
                continue
            s = torch.einsum("jhd,hd->hj", k[first:last], q[q0 + i].double()) * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            p = torch.softmax(s, dim=1)
            o, mass = (torch.einsum("hj,jhd->hd", p, x) for x in (v[first:last], v[first:last].abs()))
            out[q0 + i] = o
            bound[q0 + i] = STEP[q.dtype] * o.abs() + (STEP[q.dtype] + 2.0 ** -9) * mass + TINY[q.dtype]
    return out, bound
