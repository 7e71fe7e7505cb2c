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


# ---- every key counts, once ---------------------------------------------------------------------------------------------

# (bounds that leave room for rounding errors of many keys hide a single one that is lost, doubled or taken from elsewhere)
PLANS = ["0", "1", "7", "64"]


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("page", [3, 16, 200])
@pytest.mark.parametrize("d", [64, 72, 128, 200, 256])
def test_each_value_is_added_once(dev, monkeypatch, plan, page, d):
    """Queries of zero: every score is 0, every weight 1 / n, and sums of small whole numbers are exact.  Key j adds a number from
    1 to 4 to dim j % d and nothing to the others.  A sum is of at most 24 keys, so at most 96: one key more or less changes it by
    a 96th at least, twice the 256th less and the 256th more that one rounding to 8 bits allows (and 2^-22 for the quotient)."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    for dtype in (torch.bfloat16, torch.float16):
        kvs, counts = [1501, 40, 1090], [3, 40, 33]
        k, v, table = cache(kvs, page, 1, d, dtype, 7)
        numbers = torch.randint(1, 5, (3, 1501), generator=torch.Generator().manual_seed(8))
        v[~v.isnan()] = 0
        for b, n in enumerate(kvs):
            j = torch.arange(n)
            v[table[b, j // page].long(), j % page, 0, j % d] = numbers[b, :n].to(dtype)
        offsets = torch.tensor([0] + counts).cumsum(0).int()
        lens = torch.tensor(kvs, dtype=torch.int32)
        q = torch.zeros(sum(counts), 2, d, dtype=dtype)
        for causal, window in ((True, None), (True, 1000), (False, 300)):
            out = attend(dev, q, k, v, table, offsets, lens, causal=causal, window=window)
            for b, n in enumerate(kvs):
                for i in range(counts[b]):
                    p = n - counts[b] + i
                    seen = torch.arange(max(0, p - window + 1) if window else 0, p + 1 if causal else n)
                    sums = torch.zeros(d, dtype=torch.float64).index_add_(0, seen % d, numbers[b, seen].double()) / len(seen)
                    off = (out[offsets[b] + i] - sums).abs()
                    assert bool((off <= (STEP[dtype] + 2.0 ** -22) * sums + TINY[dtype]).all()), (dtype, causal, window, b, i)


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("page", [3, 16, 200])
@pytest.mark.parametrize("d", [64, 72, 128, 200, 256])
def test_each_key_finds_its_value(dev, monkeypatch, plan, page, d):
    """Keys of random signs, and queries that each single one out, at every border of pages, blocks, steps, look-ups and splits.
    All others together have less than 2^-52 of its weight, so that values of up to 5 add less than 2^-24 of one of 2^-25 or more;
    the weight's rounding is in the sum that it is divided by too, and what fp32 makes of the quotient, 2^-22, is less than half
    a step of the type: the result is the value, bit for bit."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    for dtype in (torch.bfloat16, torch.float16):
        n = 1501
        k, v, table = cache([n], page, 1, d, dtype, 9)
        filled = ~k.isnan()
        signs = torch.randint(0, 2, (n, d), generator=torch.Generator().manual_seed(10)) * 2 - 1
        j = torch.arange(n)
        k[table[0, j // page].long(), j % page, 0] = signs.to(dtype)
        assert torch.equal(~k.isnan(), filled) and float(v[~v.isnan()].abs().max()) <= 5
        borders = sorted({x for step in (8, 32, 64, 128, 256, 512, page) for e in range(0, n, step) for x in (e - 1, e)} & set(range(n)) | {n - 1})
        wanted = torch.tensor(borders)
        q = (signs[wanted] * 16).to(dtype)[:, None]
        scores = (q[:, 0].double() @ signs.double().t()) * d ** -0.5
        own = scores.gather(1, wanted[:, None])
        others = scores.scatter(1, wanted[:, None], -math.inf).amax(1, keepdim=True)
        assert bool((own - others > math.log(n * 2.0 ** 52)).all())
        offsets, lens = torch.tensor([0, len(borders)], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
        out = attend(dev, q, k, v, table, offsets, lens, causal=False)
        want = v[table[0, wanted // page].long(), wanted % page, 0].double()
        assert torch.equal(out[:, 0], want), (dtype, [borders[i] for i in (out[:, 0] != want).any(1).nonzero()[:8, 0].tolist()])
