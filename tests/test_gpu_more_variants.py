"""Forms of the operators around a cache in 8 bits that only large calls or forced choices reach, against plain forms in 64 bits: chunks a
thread of the residual's norm, groups of two heads, the ends of the powers' range."""

from __future__ import annotations

import pytest
import torch

import layer_oracle
import more_oracle as oracle
from conftest import seeded

pytestmark = pytest.mark.gpu


def ops():
    from phyai_amd import ops as o

    return o


def check_norm(dev, m, d, per_block, gemma):
    x, residual, weight = seeded((m, d), 1), seeded((m, d), 2, 4.0), seeded((d,), 3, 0.3)
    residual[:, ::37] *= 20
    weight[::11] = -1.0 if gemma else 0.0                # (columns whose norm is zero)
    codes, scale, total = ops().add_rmsnorm_fp8(x.to(dev), residual.to(dev), weight.to(dev), 1e-6, gemma=gemma, per_block=per_block)
    want, n = oracle.add_norm(x, residual, weight, 1e-6, gemma)
    assert torch.equal(total.cpu(), want)
    oracle.check_norm_codes(codes, scale, n, per_block)


# (as many chunks as a row needs are taken where fewer are forced; 24584 and 32768 need four, 520 ends in the second of 64 threads)
@pytest.mark.parametrize("m,d", [(3, 8), (3, 136), (17, 520), (5, 4304), (2, 8192), (3, 12296), (2, 24584), (2, 32768)])
@pytest.mark.parametrize("chunks", ["1", "2", "3", "4"])
@pytest.mark.parametrize("per_block", [True, False])
def test_add_rmsnorm_of_every_number_of_chunks(dev, monkeypatch, chunks, m, d, per_block):
    monkeypatch.setenv("PHYAI_LAYER_ADD_NORM", chunks)
    check_norm(dev, m, d, per_block, gemma=d % 16 == 0)


@pytest.mark.parametrize("m,d", [(777, 4304), (4200, 520), (3000, 1160), (2100, 2048), (2, 24584), (2, 32768), (2, 32776)])
@pytest.mark.parametrize("per_block,gemma", [(True, True), (False, False)])
def test_add_rmsnorm_of_many_rows_and_the_longest(dev, m, d, per_block, gemma):
    """Rows enough for two or three chunks a thread by the rule itself, the last of them filled in part or not at all; rows of four chunks."""
    check_norm(dev, m, d, per_block, gemma)


@pytest.mark.parametrize("value", ["0", "x", "-3", "9"])
def test_what_is_no_number_of_chunks_changes_nothing(dev, monkeypatch, value):
    monkeypatch.setenv("PHYAI_LAYER_ADD_NORM", value)
    check_norm(dev, 5, 4304, True, False)


# ---- heads into a cache in 8 bits ------------------------------------------------------------------------------------

def raw(t):
    return t.view(torch.uint8) if t.dtype != torch.uint8 else t


def check_heads(dev, t, heads, kv_heads, d, rot, dtype, interleaved, gemma, norm=True, page=8):
    qkv = seeded((t, (heads + 2 * kv_heads) * d), 1, 2.0, dtype)
    weights = [seeded((d,), s, 0.3, dtype) + (0 if gemma else 1) for s in (3, 4)] if norm else [None, None]
    gen = torch.Generator().manual_seed(5)
    positions, table = torch.randint(0, 256, (t,), generator=gen), ops().rope_table(256, rot, device="cpu")
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=gen)[:t]
    slots[t // 3::97] = -1
    pool = list(ops().fp8_cache(pages, page, kv_heads, d, device=dev))
    for p in pool:
        raw(p).fill_(0x55)
    q, none = ops().qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, q_weight=weights[0].to(dev) if norm else None,
                                 k_weight=weights[1].to(dev) if norm else None, gemma=gemma, interleaved=interleaved, k_pages=pool[0], v_pages=pool[1],
                                 slots=slots.to(dev), k_scales=pool[2], v_scales=pool[3])
    assert none is None
    k, v, ks, vs = (raw(p).cpu() for p in pool)
    rows = qkv.view(t, -1, d)
    want, bound = layer_oracle.head_rope(rows[:, :heads], weights[0], table, positions, 1e-6, gemma, interleaved)
    bad = ~((q.cpu().double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[0].tolist())
    written = slots >= 0
    at = (slots[written] // page, slots[written] % page)
    want, bound = layer_oracle.head_rope(rows[:, heads: heads + kv_heads], weights[1], table, positions, 1e-6, gemma, interleaved)
    slack = bound - layer_oracle.STEP[dtype] * want.abs()                        # (what comes before the rounding)
    oracle.check_cache(k[at], ks[at], want[written], slack[written], "k")
    codes, byte = oracle.to_cache(rows[:, heads + kv_heads:])
    assert torch.equal(v[at], codes[written]) and torch.equal(vs[at], byte[written])
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[at] = False
    assert all(bool((x[rest] == 0x55).all()) for x in (k, v, ks, vs))


# (more than 2^19 threads with a head each: two heads a group then.  Of odd numbers of query heads one group has the last query and the first key, of
# odd numbers of both one has the last key and the first value; (1, 1) has no group of queries alone)
LARGE = [(4100, 8, 1, 256, 256), (4800, 5, 1, 256, 128), (4800, 3, 2, 256, 256), (11000, 1, 1, 256, 256), (6600, 8, 1, 128, 64), (3400, 8, 6, 80, 48),
         (25000, 5, 3, 16, 8)]


@pytest.mark.parametrize("t,heads,kv_heads,d,rot", LARGE)
@pytest.mark.parametrize("dtype,interleaved,gemma,norm", [(torch.bfloat16, False, False, True), (torch.float16, True, True, True),
                                                          (torch.bfloat16, True, False, False)])
def test_many_heads_into_a_cache_in_8_bits(dev, t, heads, kv_heads, d, rot, dtype, interleaved, gemma, norm):
    lanes = 1
    while lanes * (16 if rot % 16 == 0 else 8) < d:
        lanes *= 2
    assert t * (heads + 2 * kv_heads) * lanes > 1 << 19
    check_heads(dev, t, heads, kv_heads, d, rot, dtype, interleaved, gemma, norm)


@pytest.mark.parametrize("t,heads,kv_heads,d,rot", [(1, 8, 1, 256, 256), (50, 8, 1, 256, 128), (17, 6, 3, 80, 48), (130, 8, 2, 128, 128), (9, 2, 1, 16, 8),
                                                    (5, 3, 1, 512, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gemma_heads_into_a_cache_in_8_bits(dev, t, heads, kv_heads, d, rot, dtype, interleaved):
    check_heads(dev, t, heads, kv_heads, d, rot, dtype, interleaved, gemma=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_power_reads_back_rounded_once(dev, dtype):
    """All 256 codes times all 255 powers: exact where the type holds the product, elsewhere rounded to nearest even, once; 255: NaN."""
    k, v, ks, vs = ops().fp8_cache(256, 1, 1, 256, device=dev)
    codes = torch.arange(256, dtype=torch.uint8)
    raw(k)[:], raw(v)[:] = codes.to(dev), codes.flip(0).to(dev)
    raw(ks)[:], raw(vs)[:] = codes.to(dev).view(256, 1, 1), codes.flip(0).to(dev).view(256, 1, 1)
    got = ops().read_fp8_cache(k, v, ks, vs, torch.arange(256, device=dev), dtype=dtype)
    for name, out, p, s in (("k", got[0], k, ks), ("v", got[1], v, vs)):
        want = oracle.widen(raw(p).cpu(), raw(s).cpu()).reshape(256, 256).to(dtype)
        out, power = out.cpu().reshape(256, 256), raw(s).cpu().reshape(256)
        same = (out == want) | (out.isnan() & want.isnan())
        bad = ~same
        some = [(name, int(power[i]), int(raw(p).cpu().view(256, 256)[i, j]), float(out[i, j]), float(want[i, j]))
                for i, j in bad.nonzero()[:: max(1, int(bad.sum()) // 24)].tolist()]
        assert not some, (int(bad.sum()), some)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("plan", ["0", "1", "2"])
def test_attention_sees_what_is_read_back(dev, monkeypatch, plan, dtype, d):
    """256 sequences of one key, with each power one of them: probabilities are one, so the result is the value, bit for bit, the smallest,
    infinite ones and NaNs among them."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    k, v, ks, vs = ops().fp8_cache(256, 1, 1, d, device=dev)
    for part in range(0, 256, d):
        raw(v)[:] = torch.arange(part, part + d, dtype=torch.uint8, device=dev)
        raw(vs)[:] = torch.arange(256, dtype=torch.uint8, device=dev).view(256, 1, 1)
        raw(ks).fill_(127)
        want = ops().read_fp8_cache(k, v, ks, vs, torch.arange(256, device=dev), dtype=dtype)[1]
        q = torch.ones(256, 1, d, dtype=dtype, device=dev)
        steps = torch.arange(257, dtype=torch.int32, device=dev)
        out = ops().paged_attention(q, k, v, steps[:256].view(256, 1).contiguous(), steps, torch.ones(256, dtype=torch.int32, device=dev), k_scales=ks, v_scales=vs)
        off = ~((out == want) | (out.isnan() & want.isnan()))
        assert not off.any(), (int(off.sum()), [(i, part + j, float(out[i, 0, j]), float(want[i, 0, j])) for i, _, j in off.nonzero()[:8].tolist()])


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("bits,dtype", [(8, torch.bfloat16), (16, torch.bfloat16), (16, torch.float16)])
@pytest.mark.parametrize("plan", ["0 2 0 0 3", "0 2 1 0 2", "0 2 1 1 3", "1 2 0 1 3", "1 1 0 0 0", "0 1 0 0 0"])
def test_unknown_values_of_shared_and_own_keys(dev, monkeypatch, plan, bits, dtype, d):
    """NaNs and infinities among shared values and a sequence's own, tokens that stand inside the prefix: they reach the rows that see their key
    and no other, whichever kernels share the work."""
    from test_gpu_more_ops import attend, attend_case, within

    monkeypatch.setenv("PHYAI_LAYER_ATTEND_MORE", plan)
    qs, kvs = [20, 30, 10], [64, 70, 66]
    tensors, kw = attend_case((qs, kvs, 16, 4, 2, d, True, None, [0, 45, 0], None), dtype, bits, shared=64)
    want, bound = oracle.attention(*tensors.values(), **kw)
    table, values = tensors["page_table"], tensors["v_pages"]
    planted = [(None, 42, 3), (None, 50, d - 1), (1, 66, 17), (2, 64, 40)]     # (whose, key, value dim): the first two of all sequences
    position = torch.cat([torch.arange(kv - q, kv) for q, kv in zip(qs, kvs)])
    sequence = torch.repeat_interleave(torch.arange(3), torch.tensor(qs))
    hit = torch.zeros(60, 4, d, dtype=torch.bool)
    for n, (b, key, at) in enumerate(planted):
        values[table[b or 0, key // 16].long(), key % 16, 1, at] = 0x7F if bits == 8 else (float("nan"), float("inf"))[n % 2]
        rows = (position >= key) | ((sequence == 1) & (key < 45)) if b is None else (position >= key) & (sequence == b)
        hit[rows, 2:, at] = True                                              # (key head 1: query heads 2 and 3)
    for shared in (64, 0):
        out = attend(dev, tensors, kw | dict(shared_prefix=shared)).cpu().double()
        assert not out[hit].isfinite().any(), shared
        within(torch.where(hit, 0.0, out), torch.where(hit, 0.0, want), torch.where(hit, 0.0, bound), f"shared {shared}")
