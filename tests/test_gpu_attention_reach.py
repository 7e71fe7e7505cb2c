"""Caches whose places lie beyond 32-bit offsets from one base, and calls that hold prompts and single tokens."""

from __future__ import annotations

import pytest
import torch

from conftest import seeded
from test_gpu_attention_rules import attend, by_the_text, within
from test_gpu_layer_ops import cache

pytestmark = pytest.mark.gpu


def ops():
    from phyai_amd import ops as o

    return o


@pytest.mark.parametrize("plan", ["0", "1"])
@pytest.mark.parametrize("d,page", [(128, 16), (80, 16), (64, 20)])
def test_offsets_beyond_32_bits_from_one_base(dev, monkeypatch, plan, d, page):
    """Keys and values of a page side by side in one pool: the last pages' elements lie past 2^31 from the base of keys, their
    bytes past 2^32.  The page that an offset cut to 32 bits (of elements or of bytes) would reach holds other values."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    heads, kv_heads, t = 4, 2, 3 * page - 5
    size = 2 * page * kv_heads * d                       # elements from page to page
    pages = 2 ** 32 // size + 20
    pool = torch.empty(pages, 2, page, kv_heads, d, dtype=torch.bfloat16, device=dev)
    k_pages, v_pages = pool[:, 0], pool[:, 1]
    assert k_pages.stride(0) == size and (pages - 12) * size > 2 ** 32
    ids = torch.tensor([pages - 1, 2, pages - 9], dtype=torch.int32, device=dev)
    for page_id in ids.tolist():
        for cut in (2 ** 31, 2 ** 32):                   # (2^32 bytes are 2^31 elements; signed words wrap at these too)
            wrong = (page_id * size) % cut // size
            pool[wrong].fill_(100.0)
            pool[wrong + 1].fill_(100.0)
    qkv = seeded((t, (heads + 2 * kv_heads) * d), 3).to(dev)
    slots = (ids.long()[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[:t].contiguous()
    table = ops().rope_table(64, d)
    position = torch.arange(t, device=dev)
    q, _ = ops().qk_norm_rope(qkv, table, position, heads, kv_heads, d, k_pages=k_pages, v_pages=v_pages, slots=slots)
    small = torch.zeros(2, 3, page, kv_heads, d, dtype=torch.bfloat16, device=dev)
    q_small, _ = ops().qk_norm_rope(qkv, table, position, heads, kv_heads, d, k_pages=small[0], v_pages=small[1], slots=position)
    assert torch.equal(q, q_small)
    written = torch.arange(t, device=dev)
    for far, near in ((k_pages, small[0]), (v_pages, small[1])):
        assert torch.equal(far[ids.long()].reshape(-1, kv_heads, d)[written], near.reshape(-1, kv_heads, d)[written])
    offsets, lens = torch.tensor([0, t], dtype=torch.int32, device=dev), torch.tensor([t], dtype=torch.int32, device=dev)
    want = ops().paged_attention(q, small[0], small[1], torch.arange(3, dtype=torch.int32, device=dev)[None], offsets, lens)
    assert torch.equal(ops().paged_attention(q, k_pages, v_pages, ids[None], offsets, lens), want)
    assert float(want.float().abs().max()) < 10


@pytest.mark.parametrize("plan", [None, "0", "1", "2"])
@pytest.mark.parametrize("kv_heads", [1, 4])
@pytest.mark.parametrize("order", [1, -1])
def test_a_prompt_and_single_tokens_in_one_call(dev, monkeypatch, plan, kv_heads, order):
    """The plan is one for the whole call: tiles of many rows that hold one, and a prompt in tiles of few."""
    if plan is not None:
        monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    counts = [700, 1, 1, 0, 1, 5][::order]
    kvs = [740, 1, 333, 17, 64, 5][::order]
    k, v, table = cache(kvs, 16, kv_heads, 64, torch.bfloat16, 11)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    lens = torch.tensor(kvs, dtype=torch.int32)
    q = seeded((int(offsets[-1]), 4, 64), 12)
    out = attend(dev, q, k, v, table, offsets, lens, window=100)
    for b, n in enumerate(counts):
        rows = torch.arange(int(offsets[b]), int(offsets[b]) + n)
        pick = rows[torch.linspace(0, n - 1, min(n, 40)).long()] if n else rows     # (of the prompt, forty rows)
        for i in pick.tolist():
            end = kvs[b] - n + i - int(offsets[b]) + 1                             # a call with this token as the last
            want, bound = by_the_text(q[i:i + 1], k, v, table[b:b + 1], torch.tensor([0, 1]), torch.tensor([end]), window=100)
            within(out[i:i + 1], want, bound, f"sequence {b}, row {i}")
