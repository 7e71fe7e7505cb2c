"""Attention over pages against the text of its interface: where a token stands, what it sees, and every single key."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import seeded
from layer_oracle import STEP, TINY
from test_gpu_layer_ops import cache

pytestmark = pytest.mark.gpu


def ops():
    from phyai_amd import ops as o

    return o


def attend(dev, *tensors, **kw):
    return ops().paged_attention(*(t.to(dev) for t in tensors), **kw).cpu().double()


def by_the_text(q, k_pages, v_pages, table, offsets, lens, *, causal=True, window=None):
    """(out, bound) in 64 bits.  Token i of n new ones stands at p = lens[b] - n + i and sees the keys j < lens[b] that the
    table has room for, with j <= p (causal) and j > p - window.  Bound: half a step of the type for the result; of the
    weighted magnitudes half a step for a probability's rounding, twice (the sum is rounded as well) what D + 2 fp32 additions and
    products of 2^-23 do to a score, and 2^-21 for the exponential and for the score's product with log2(e)."""
    T, H, D = q.shape
    page, kv_heads = k_pages.shape[1:3]
    out, bound = (torch.full((T, H, D), math.nan, dtype=torch.float64) for _ in range(2))
    for b in range(lens.numel()):
        q0, n = int(offsets[b]), int(offsets[b + 1] - offsets[b])
        there = max(0, min(int(lens[b]), table.shape[1] * page))
        ids = table[b, : -(-there // page)].long()
        k, v = (t[ids].reshape(-1, kv_heads, D)[:there].double() for t in (k_pages, v_pages))
        j = torch.arange(there)
        for i in range(n):
            p = int(lens[b]) - n + i
            sees = torch.ones(there, dtype=torch.bool)
            if causal:
                sees &= j <= p
            if window is not None:
                sees &= j > p - window
            if not sees.any():
                out[q0 + i], bound[q0 + i] = 0.0, 0.0
                continue
            for h in range(H):
                g = h // (H // kv_heads)
                products = k[sees, g] * q[q0 + i, h].double() * D ** -0.5
                w = torch.softmax(products.sum(-1), dim=0)
                o, mass = w @ v[sees, g], w @ v[sees, g].abs()
                moved = 2 * (D + 2) * 2.0 ** -23 * products.abs().sum(-1).max() + 2.0 ** -21 * (1 + products.sum(-1).abs().max())
                out[q0 + i, h], bound[q0 + i, h] = o, STEP[q.dtype] * o.abs() + (STEP[q.dtype] + moved) * mass + TINY[q.dtype]
    return out, bound


def within(got, want, bound, what):
    off = (got - want).abs()
    bad = ~((off <= bound) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("plan", ["0", "1", "3"])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 9), (True, 40), (False, 21), (False, None)])
def test_a_token_stands_where_the_stated_length_puts_it(dev, monkeypatch, plan, causal, window):
    """Lengths beyond the keys that the table has room for: by a few tokens, by more than the window, by far."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    k, v, table = cache([64] * 6, 16, 2, 64, torch.bfloat16, 3)
    table = table[:, :4].contiguous()
    lens = torch.tensor([64, 65, 69, 84, 100, 2 ** 31 - 1], dtype=torch.int32)
    offsets = torch.arange(7, dtype=torch.int32) * 10
    q = seeded((60, 4, 64), 4)
    want, bound = by_the_text(q, k, v, table, offsets, lens, causal=causal, window=window)
    within(attend(dev, q, k, v, table, offsets, lens, causal=causal, window=window), want, bound, f"{causal} {window}")


@pytest.mark.parametrize("plan", ["0", "1", "3", "64"])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256)])
def test_a_row_that_sees_only_infinitely_low_scores_has_no_softmax(dev, monkeypatch, plan, dtype, d):
    """The softmax of scores that are all -inf is NaN, in 64 bits as here; one finite score makes theirs weightless.  Only a row
    that sees no key is zero."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    k, v, table = cache([200, 3, 0], 16, 1, d, dtype, 5)
    for b, low in ((0, 140), (1, 3)):
        for j in range(low):
            k[table[b, j // 16].long(), j % 16] = -math.inf
    lens = torch.tensor([200, 3, 0], dtype=torch.int32)
    offsets = torch.tensor([0, 200, 205, 207], dtype=torch.int32)   # the second sequence's first two tokens stand in front of its keys
    q = (seeded((207, 2, d), 6).abs() + 0.1).to(dtype)
    want, bound = by_the_text(q, k, v, table, offsets, lens)
    assert want[:140].isnan().all() and want[202:205].isnan().all() and not want[200:202].any() and not want[140:200].isnan().any()
    within(attend(dev, q, k, v, table, offsets, lens), want, bound, "rows")
