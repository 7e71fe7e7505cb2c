"""Residual and norm into fp8, a cache in 8 bits written, read and attended over, capped scores, prompts seen whole, shared prefixes:
against plain forms in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import layer_oracle
import more_oracle as oracle
from conftest import seeded

pytestmark = pytest.mark.gpu


def ops():
    from phyai_amd import ops as o

    return o


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, bound, what=""):
    off = (got.cpu().double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {((off - bound)[bad]).max():.3e} at {bad.nonzero()[0].tolist()}"


# ---- residual and norm -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,d", [(1, 8), (1, 2048), (3, 136), (50, 1024), (17, 520), (5, 4304), (2, 8192), (3, 16384), (2, 16392), (130, 2048), (2, 40000)])
@pytest.mark.parametrize("per_block", [True, False])
@pytest.mark.parametrize("gemma", [True, False])
def test_add_rmsnorm_fp8(dev, m, d, per_block, gemma):
    x, residual, weight = seeded((m, d), 1), seeded((m, d), 2, 4.0), seeded((d,), 3, 0.3)
    residual[:, ::37] *= 20
    weight[::11] = -1.0 if gemma else 0.0                # (columns whose norm is zero)
    codes, scale, total = ops().add_rmsnorm_fp8(x.to(dev), residual.to(dev), weight.to(dev), 1e-6, gemma=gemma, per_block=per_block)
    want, n = oracle.add_norm(x, residual, weight, 1e-6, gemma)
    assert codes.dtype == torch.float8_e4m3fn and torch.equal(total.cpu(), want)
    oracle.check_norm_codes(codes, scale, n, per_block)


@pytest.mark.parametrize("per_block", [True, False])
def test_add_rmsnorm_of_nothing_and_of_special_rows(dev, per_block):
    """A row of zeros has the least scale and zero codes; an infinity or a NaN spoils its own row."""
    x, residual, weight = seeded((6, 300 * 8), 1), seeded((6, 300 * 8), 2), seeded((300 * 8,), 3, 0.2) + 1
    x[1], residual[1] = 0, 0
    x[2], residual[2] = 1.0, -1.0                        # the sum is nothing
    x[3, 5], x[4, 700] = math.inf, math.nan
    codes, scale, total = ops().add_rmsnorm_fp8(x.to(dev), residual.to(dev), weight.to(dev), 1e-6, per_block=per_block)
    want, n = oracle.add_norm(x, residual, weight, 1e-6, False)
    assert torch.equal(total.cpu().isnan(), want.isnan()) and torch.equal(total.cpu().nan_to_num(), want.nan_to_num())
    for row in (1, 2):
        assert bool((codes[row].view(torch.uint8).cpu() & 0x7F == 0).all()) and bool((scale[row].cpu() == torch.tensor(1e-12) / torch.tensor(448.0)).all())
    values = codes.cpu().float()
    assert values[4].isnan().all() and values[3, 5].isnan() and not values[[0, 1, 2, 5]].isnan().any()
    keep = [0, 5]
    oracle.check_norm_codes(codes[keep], scale[keep], n[keep], per_block)
    empty = ops().add_rmsnorm_fp8(x[:0].to(dev), residual[:0].to(dev), weight.to(dev))
    assert empty[0].shape == (0, 2400) and empty[1].shape == (0, 19) and empty[2].shape == (0, 2400)


@pytest.mark.parametrize("d", [512, 2048, 20000])
def test_add_rmsnorm_in_place_and_strided(dev, d):
    m = 7
    weight = seeded((d,), 3, 0.2).to(dev)
    wide_x, wide_r = seeded((m, d + 24), 1).to(dev), seeded((m, d + 64), 2).to(dev)
    x, residual = wide_x[:, 16: 16 + d], wide_r[:, 8: 8 + d]
    want = ops().add_rmsnorm_fp8(x.contiguous(), residual.contiguous(), weight, gemma=True)
    got = ops().add_rmsnorm_fp8(x, residual, weight, gemma=True)
    odd = ops().add_rmsnorm_fp8(wide_x[:, 3: 3 + d], wide_r[:, 1: 1 + d], weight, gemma=True)   # (rows that have to be copied first)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    odd_want = ops().add_rmsnorm_fp8(wide_x[:, 3: 3 + d].contiguous(), wide_r[:, 1: 1 + d].contiguous(), weight, gemma=True)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(odd, odd_want))
    for which in (0, 1):
        pair = [x.contiguous(), residual.contiguous()]
        again = ops().add_rmsnorm_fp8(*pair, weight, gemma=True, out=pair[which])
        assert again[2].data_ptr() == pair[which].data_ptr()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(again, want))
    same = x.contiguous()
    for one in (ops().add_rmsnorm_fp8(same[:1].expand(m, d), residual, weight, gemma=True), ops().add_rmsnorm_fp8(residual, same[:1].expand(m, d), weight, gemma=True)):
        repeated = ops().add_rmsnorm_fp8(same[:1].repeat(m, 1), residual.contiguous(), weight, gemma=True)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, repeated))
    twice = same.clone()
    both = ops().add_rmsnorm_fp8(twice, twice, weight, gemma=True, out=twice)
    assert torch.equal(both[2], same + same)
    three = ops().add_rmsnorm_fp8(x.contiguous().view(1, m, d), residual.contiguous().view(1, m, d), weight, gemma=True)
    assert three[0].shape == (1, m, d) and three[1].shape == (1, m, -(-d // 128)) and torch.equal(three[1][0], want[1])


# ---- a cache in 8 bits -------------------------------------------------------------------------------------------

def fp8_pool(dev, pages, page, kv_heads, d, layout):
    """Zeroed codes and scales; their order in memory: as fp8_cache makes them, or heads outermost and scales token by token."""
    if layout == "made":
        return list(ops().fp8_cache(pages, page, kv_heads, d, device=dev))
    codes = [torch.zeros(pages, kv_heads, page, d + 16, dtype=torch.uint8, device=dev).transpose(1, 2)[..., :d].view(torch.float8_e4m3fn) for _ in range(2)]
    return codes + [torch.zeros(pages, page, kv_heads, dtype=torch.uint8, device=dev) for _ in range(2)]


def raw(t):
    return t.view(torch.uint8) if t.dtype != torch.uint8 else t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_code_reads_back_exactly(dev, dtype):
    """All 256 codes times powers: exact in bf16; in half precision rounded once where it ends (only numbers of its range here)."""
    powers = [3, 60, 120, 126, 127, 128, 134, 200, 247] if dtype == torch.bfloat16 else [112, 120, 127, 134]
    page = 4
    k, v, ks, vs = fp8_pool(dev, len(powers), page, 2, 256, "made")
    codes = torch.arange(256, dtype=torch.uint8)
    raw(k)[:], raw(v)[:] = codes.to(dev), codes.flip(0).to(dev)
    raw(ks)[:] = torch.tensor(powers, dtype=torch.uint8, device=dev)[:, None, None]
    raw(vs)[:] = torch.tensor(powers[::-1], dtype=torch.uint8, device=dev)[:, None, None]
    slots = torch.arange(len(powers) * page, device=dev)
    got_k, got_v = ops().read_fp8_cache(k, v, ks, vs, slots, dtype=dtype)
    for got, p, s in ((got_k, k, ks), (got_v, v, vs)):
        want = oracle.widen(raw(p).cpu(), raw(s).cpu()).reshape(len(powers) * page, 2, 256)
        exact = want.to(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(), exact.nan_to_num())
        if dtype == torch.bfloat16:   # (448 * 2^120 lies beyond the type: infinite, like any value rounded to it)
            inside = want.abs() <= torch.finfo(dtype).max
            assert torch.equal(exact.double()[inside], want[inside]) and int(inside.sum()) > 0.9 * want.numel()


def test_unknown_scales_and_slots(dev):
    k, v, ks, vs = fp8_pool(dev, 3, 4, 2, 64, "other")
    raw(k).random_(1, 100)
    raw(v).random_(1, 100)
    ks.fill_(127)
    vs.fill_(130)
    ks[1, 2, 1] = 255
    slots = torch.tensor([6, -1, 12, 2 ** 62, 11, 6], device=dev)
    a, b = ops().read_fp8_cache(k, v, ks, vs, slots)
    assert a[0, 1].isnan().all() and a[5, 1].isnan().all() and not a[0, 0].isnan().any()
    assert bool((a[1:4] == 0).all()) and bool((b[1:4] == 0).all())
    assert torch.equal(b[4].float(), raw(v)[2, 3].contiguous().view(torch.float8_e4m3fn).float() * 8)
    assert ops().read_fp8_cache(k, v, ks, vs, slots[:0])[0].shape == (0, 2, 64)


CACHE = [(1, 8, 1, 256, 256), (3, 1, 1, 64, 64), (50, 8, 1, 256, 128), (17, 6, 3, 80, 48), (40, 4, 4, 96, 64), (130, 8, 2, 128, 128), (9, 2, 1, 16, 8),
         (5, 3, 1, 512, 512)]


@pytest.mark.parametrize("t,heads,kv_heads,d,rot", CACHE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved,norm,layout", [(False, True, "made"), (True, False, "other"), (False, False, "made"), (True, True, "other")])
def test_heads_into_a_cache_in_8_bits(dev, t, heads, kv_heads, d, rot, dtype, interleaved, norm, layout):
    page = 8
    qkv = seeded((t, (heads + 2 * kv_heads) * d), 1, 2.0, dtype)
    qkv[0, heads * d: heads * d + d] = 0                                         # a key of nothing
    qkv[t - 1, -d:] *= 2.0 ** -9                                                 # a small value head
    weights = [seeded((d,), s, 0.3, dtype) + 1 for s in (3, 4)] if norm else [None, None]
    positions = torch.randperm(200, generator=gen(5))[:t]
    table = ops().rope_table(256, rot, device="cpu")
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=gen(6))[:t]
    if t > 2:
        slots[1] = -1
    k, v, ks, vs = fp8_pool(dev, pages, page, kv_heads, d, layout)
    marks = [raw(x).fill_(0x55) for x in (k, v, ks, vs)]
    q, none = ops().qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, q_weight=weights[0].to(dev) if norm else None,
                                 k_weight=weights[1].to(dev) if norm else None, gemma=False, interleaved=interleaved, k_pages=k, v_pages=v,
                                 slots=slots.to(dev), k_scales=ks, v_scales=vs)
    assert none is None
    rows = qkv.view(t, -1, d)
    want, bound = layer_oracle.head_rope(rows[:, :heads], weights[0], table, positions, 1e-6, False, interleaved)
    within(q, want, bound, "q")
    written = slots >= 0
    at = (slots[written] // page, slots[written] % page)
    want, bound = layer_oracle.head_rope(rows[:, heads: heads + kv_heads], weights[1], table, positions, 1e-6, False, interleaved)
    slack = bound - layer_oracle.STEP[dtype] * want.abs()                        # (what comes before the rounding)
    oracle.check_cache(raw(k).cpu()[at], raw(ks).cpu()[at], want[written], slack[written], "k")
    codes, byte = oracle.to_cache(rows[:, heads + kv_heads:])
    assert torch.equal(raw(v).cpu()[at], codes[written]) and torch.equal(raw(vs).cpu()[at], byte[written])
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[at] = False
    assert all(bool((m.cpu()[rest] == 0x55).all()) for m in marks)
    # read back: what attention will see
    a, b = ops().read_fp8_cache(k, v, ks, vs, slots.to(dev), dtype=dtype)
    want = oracle.widen(raw(v).cpu()[at], raw(vs).cpu()[at]).to(dtype)
    assert torch.equal(b.cpu()[written], want) and bool((a.cpu()[~written] == 0).all())


def test_heads_of_special_values_and_borders(dev):
    """Largest magnitudes at each mantissa around the border 448, both types' ends, infinities and NaNs."""
    d = 64
    for dtype in (torch.bfloat16, torch.float16):
        steps = torch.arange(64, dtype=torch.float64) / 32
        tops = [float(x) for x in (1 + steps[:32]) * 256] + [448.0, 450.0, 446.0, 1.75, 1.7578125, 65504.0, 61440.0, 2.0 ** -14, 2.0 ** -24, 0.0]
        if dtype == torch.bfloat16:
            tops += [3.38e38, 1e-38, 9.2e-41, 448 * 2.0 ** -126, 2.0 ** 120]
        values = torch.tensor(tops, dtype=torch.float64).to(dtype)
        n = len(tops)
        x = (torch.rand(n, d, generator=gen(1), dtype=torch.float64) * 2 - 1)[...] * values.double()[:, None]
        x = x.to(dtype)
        x[:, 7] = -values
        special = torch.zeros(3, d, dtype=dtype)
        special[0, 3], special[1, 60], special[2, 0] = math.inf, math.nan, -math.inf
        x = torch.cat([x, special])
        t = x.shape[0]
        qkv = torch.cat([x, x, x], 1)
        k, v, ks, vs = fp8_pool(dev, t, 1, 1, d, "made")
        ops().qk_norm_rope(qkv.to(dev), torch.zeros(1, 0, device=dev), torch.zeros(t, dtype=torch.int64, device=dev), 1, 1, d, k_pages=k, v_pages=v,
                           slots=torch.arange(t, device=dev), k_scales=ks, v_scales=vs)
        end = 1.875 * 2.0 ** (127 if dtype == torch.bfloat16 else 15)
        clamped = torch.where(x.isfinite(), x.float().clamp(-end, end), x.float())
        codes, byte = oracle.to_cache(clamped)
        for p, s in ((k, ks), (v, vs)):
            assert torch.equal(raw(s).cpu().view(-1), byte) and torch.equal(raw(p).cpu().view(t, d), codes), dtype
        a, _ = ops().read_fp8_cache(k, v, ks, vs, torch.arange(t, device=dev), dtype=dtype)
        assert a[:n].isfinite().all() and a[n:].isnan().all()


# ---- attention -----------------------------------------------------------------------------------------------------

def cache16(kvs, page, kv_heads, d, dtype, seed, shared=0, spare=3):
    """Pages of sequences in random order, places of no sequence full of NaN; the first shared // page pages are everybody's."""
    g = gen(seed)
    same = shared // page
    counts = [max(0, -(-kv // page) - same) for kv in kvs]
    pages = same + sum(counts) + spare
    order = torch.randperm(pages, generator=g).int()
    width = same + max(counts) + 1
    table = torch.full((len(kvs), width), -5, dtype=torch.int32)
    table[:, :same] = order[:same]
    k = torch.full((pages, page, kv_heads, d), math.nan, dtype=dtype)
    v = k.clone()
    for i in order[:same].long():
        k[i], v[i] = (torch.randn(page, kv_heads, d, generator=g).to(dtype) for _ in range(2))
    at = same
    for b, (kv, n) in enumerate(zip(kvs, counts)):
        ids = order[at: at + n]
        at += n
        table[b, same: same + n] = ids
        for j in range(n):
            fill = min(page, kv - (same + j) * page)
            for x in (k, v):
                x[ids[j].long(), :fill] = torch.randn(fill, kv_heads, d, generator=g).to(dtype)
    return k, v, table


def in_8_bits(pages):
    """16-bit pages as codes and bytes; places of NaN as codes of NaN, or as an unknown scale."""
    codes, byte = oracle.to_cache(pages)
    hole = pages.isnan().all(-1)
    byte[hole] = torch.where(torch.arange(int(hole.sum())) % 2 == 0, 255, 127).to(torch.uint8)
    return codes, byte


# new tokens and keys per sequence, page, heads, key heads, head_dim, causal, window, prompts, cap
ATTEND = [
    ([1], [1], 16, 8, 1, 256, True, None, None, None),
    ([1], [33], 16, 1, 1, 64, True, None, None, 5.0),
    ([1, 1, 1], [70, 1, 129], 16, 8, 2, 128, True, None, None, None),
    ([1, 0, 2, 0], [5, 9, 40, 0], 1, 4, 4, 64, True, None, [2, 3, 39, 5], 30.0),
    ([5, 3], [3, 0], 16, 2, 1, 64, True, None, [2, 4], None),
    ([50], [130], 16, 8, 1, 256, False, None, None, None),
    ([37, 64], [37, 100], 24, 5, 1, 80, True, None, [20, 0], 50.0),
    ([40], [40], 3, 6, 3, 96, True, 7, [33], None),
    ([33, 1], [200, 90], 64, 4, 2, 128, True, 33, None, 50.0),
    ([20], [90], 16, 4, 1, 64, False, 12, [50], 10.0),
    ([100], [170], 16, 3, 3, 16, True, 1, None, None),
    ([130, 70], [300, 70], 32, 8, 2, 256, True, None, [290, 64], 50.0),
    ([70], [90], 256, 2, 2, 208, True, None, [10 ** 9], None),
    ([1] * 70, list(range(1, 71)), 8, 2, 1, 64, True, None, [-3] * 70, None),
]


def attend_case(case, dtype, bits, seed=0, shared=0, q_scale=1.0):
    qs, kvs, page, heads, kv_heads, d, causal, window, prompts, cap = case
    k, v, table = cache16(kvs, page, kv_heads, d, dtype, seed + 1, shared)
    offsets = torch.tensor([0] + qs).cumsum(0).int()
    q = seeded((int(offsets[-1]), heads, d), seed + 2, q_scale, dtype)
    tensors = dict(q=q, k_pages=k, v_pages=v, page_table=table, q_offsets=offsets, kv_lens=torch.tensor(kvs, dtype=torch.int32))
    kw = dict(causal=causal, window=window, softcap=cap, prefix_lens=None if prompts is None else torch.tensor(prompts).clamp(max=2 ** 31 - 1).int())
    if bits == 8:
        (tensors["k_pages"], kw["k_scales"]), (tensors["v_pages"], kw["v_scales"]) = in_8_bits(k), in_8_bits(v)
    return tensors, kw


def attend(dev, tensors, kw, layout="token", out=None):
    def on(t, name):
        if not isinstance(t, torch.Tensor):
            return t
        if name in ("k_pages", "v_pages"):
            t = t.view(torch.float8_e4m3fn) if t.dtype == torch.uint8 else t
            if layout == "head":
                return raw(t).transpose(1, 2).contiguous().to(dev).transpose(1, 2).view(t.dtype) if t.itemsize == 1 else \
                    t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
        if name in ("k_scales", "v_scales") and layout == "head":
            return t.transpose(1, 2).contiguous().to(dev).transpose(1, 2).view(torch.float8_e8m0fnu)
        return t.to(dev)

    args = [on(t, n) for n, t in tensors.items()]
    return ops().paged_attention(*args, out=out, **{n: on(t, n) for n, t in kw.items()})


def name_of(c):
    return f"q{max(c[0])}kv{max(c[1])}p{c[2]}h{c[3]}k{c[4]}d{c[5]}{'c' if c[6] else 'f'}{c[7] or ''}"


@pytest.mark.parametrize("case", ATTEND, ids=name_of)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 8), (torch.bfloat16, 16), (torch.float16, 16)])
@pytest.mark.parametrize("plan", [None, "0", "1", "3"])
def test_attention(dev, monkeypatch, case, dtype, bits, plan):
    if plan is not None:
        monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    tensors, kw = attend_case(case, dtype, bits, q_scale=4.0 if case[9] else 1.0)
    want, bound = oracle.attention(*tensors.values(), **kw)
    out = attend(dev, tensors, kw, "head" if plan == "1" else "token")
    within(out, want, bound, "attention")


@pytest.mark.parametrize("case", ATTEND, ids=name_of)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 16)])
@pytest.mark.parametrize("plan", ["1 3 0", "1 1 0", "0 3 1", "0 1 1"])
def test_attention_of_other_splits(dev, monkeypatch, case, dtype, bits, plan):
    """Many rows with the keys split (1 3), few rows with half the wavefronts a workgroup (0 n 1)."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND_MORE", plan)
    tensors, kw = attend_case(case, dtype, bits, q_scale=4.0 if case[9] else 1.0)
    want, bound = oracle.attention(*tensors.values(), **kw)
    within(attend(dev, tensors, kw | dict(shared_prefix=0, prefix_lens=kw["prefix_lens"] if kw["prefix_lens"] is not None else
                                          torch.zeros(len(case[0]), dtype=torch.int32))), want, bound, "attention")


# new tokens and keys per sequence, page, heads, key heads, head_dim, causal, window, prompts, cap, shared
SHARED = [
    ([1, 1], [20, 18], 16, 8, 1, 256, True, None, None, None, 16),
    ([1] * 9, [70 + i for i in range(9)], 16, 4, 1, 128, True, None, None, None, 69),          # not whole pages: 64 are shared
    ([2, 1, 3, 1, 2], [300, 290, 310, 289, 400], 32, 6, 2, 80, True, None, None, 30.0, 288),
    ([1] * 70, [513 + i % 5 for i in range(70)], 64, 2, 1, 64, False, None, None, None, 512),
    ([7, 5, 9], [160, 150, 200], 8, 5, 1, 256, False, None, None, None, 144),
    ([1] * 12, [200 + 3 * i for i in range(12)], 16, 8, 2, 128, True, 100, None, None, 192),     # a window that leaves the prefix to some
    ([1] * 6, [100, 10, 0, 97, 64, 96], 16, 4, 1, 64, True, None, None, None, 96),             # shorter than the prefix, and without keys
    ([3, 2, 4, 0, 1], [120, 118, 130, 112, 115], 8, 4, 4, 64, True, None, [20, 130, 115, 3, 0], 20.0, 112),
    ([20, 30, 10], [64, 70, 66], 16, 2, 1, 64, True, None, None, None, 64),                    # tokens that stand inside the prefix
]


@pytest.mark.parametrize("case", SHARED, ids=name_of)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 16), (torch.bfloat16, 16)])
def test_shared_prefix(dev, case, dtype, bits):
    tensors, kw = attend_case(case[:-1], dtype, bits, shared=case[-1])
    want, bound = oracle.attention(*tensors.values(), **kw)
    within(attend(dev, tensors, kw | dict(shared_prefix=case[-1])), want, bound, "shared")
    within(attend(dev, tensors, kw), want, bound, "each by itself")
    one = tensors | dict(page_table=tensors["page_table"][:1].expand(len(case[0]), -1)) if max(case[1]) <= case[-1] else None
    if one is not None:
        within(attend(dev, one, kw | dict(shared_prefix=case[-1])), want, bound, "one row for all")


@pytest.mark.parametrize("case", SHARED, ids=name_of)
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 16)])
@pytest.mark.parametrize("plan", ["0 2 0 0 3", "0 2 1 1 3", "1 2 0 1 3", "1 1 0 0 2", "0 1 0 1 1"])
def test_shared_prefix_of_other_splits(dev, monkeypatch, case, dtype, bits, plan):
    """Many or few rows a workgroup for the shared keys and for the sequences' own, each with splits of their own."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND_MORE", plan)
    tensors, kw = attend_case(case[:-1], dtype, bits, shared=case[-1])
    want, bound = oracle.attention(*tensors.values(), **kw)
    within(attend(dev, tensors, kw | dict(shared_prefix=case[-1])), want, bound, "shared")


def test_shared_prefix_beyond_the_table_and_of_one_sequence(dev):
    tensors, kw = attend_case(([1, 2], [64, 64], 16, 4, 1, 64, True, None, None, None), torch.bfloat16, 16, shared=64)
    want, bound = oracle.attention(*tensors.values(), **kw)
    tensors["page_table"] = tensors["page_table"][:, :4].contiguous()
    within(attend(dev, tensors, kw | dict(shared_prefix=10 ** 9)), want, bound)
    tensors, kw = attend_case(([1], [64], 16, 4, 1, 64, True, None, None, None), torch.bfloat16, 16, shared=48)
    want, bound = oracle.attention(*tensors.values(), **kw)
    within(attend(dev, tensors, kw | dict(shared_prefix=48)), want, bound)


@pytest.mark.parametrize("shared", [0, 64])
@pytest.mark.parametrize("bits", [8, 16])
def test_rows_of_no_sequence_stay(dev, bits, shared):
    tensors, kw = attend_case(([1, 2, 1], [70, 80, 90], 16, 4, 2, 64, True, None, None, None), torch.bfloat16, bits, shared=shared)
    tensors["q"] = seeded((12, 4, 64), 2)
    tensors["q_offsets"] = torch.tensor([3, 4, 6, 7], dtype=torch.int32)
    want, bound = oracle.attention(*tensors.values(), **kw)
    out = torch.full((12, 4, 64), 7.0, dtype=torch.bfloat16, device=dev)
    attend(dev, tensors, kw | dict(shared_prefix=shared), out=out)
    within(out[3:7], want[3:7], bound[3:7])
    assert bool((out[:3] == 7).all()) and bool((out[7:] == 7).all())


@pytest.mark.parametrize("plan", [None, "0", "2"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_unknown_values_reach_only_the_rows_that_see_them(dev, monkeypatch, plan, dtype):
    """Codes of NaN and unknown scales of values: 64, 128 and 256 dims, causal."""
    if plan is not None:
        monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    for d in (64, 128, 256):
        tensors, kw = attend_case(([70], [100], 16, 2, 1, d, True, None, None, None), dtype, 8)
        want, bound = oracle.attention(*tensors.values(), **kw)
        table = tensors["page_table"][0]
        tensors["v_pages"][table[60 // 16].long(), 60 % 16, 0, 3] = 0x7F
        tensors["v_pages"][table[75 // 16].long(), 75 % 16, 0, d - 1] = 0xFF
        kw["v_scales"][table[98 // 16].long(), 98 % 16, 0] = 255
        out = attend(dev, tensors, kw).cpu().double()
        hit = torch.zeros(70, 2, d, dtype=torch.bool)
        hit[30:, :, 3], hit[45:, :, d - 1], hit[68:] = True, True, True
        assert bool(out[hit].isnan().all()) and bool((((out - want).abs() <= bound) | hit).all()), d
        kw["k_scales"][table[99 // 16].long(), 99 % 16, 0] = 255
        out = attend(dev, tensors, kw).cpu().double()
        assert out[69].isnan().all() and not out[:30].isnan().any()


@pytest.mark.parametrize("shared", [0, 64])
def test_pages_that_do_not_exist(dev, shared):
    for bits in (8, 16):
        for bad in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
            tensors, kw = attend_case(([1, 3, 2], [70, 90, 100], 16, 2, 1, 64, True, None, None, None), torch.bfloat16, bits, shared=64)
            want, bound = oracle.attention(*tensors.values(), **kw)
            tensors["page_table"][1, 5] = bad                     # keys 80 .. 89 of the second sequence, whose tokens stand at 87 .. 89
            out = attend(dev, tensors, kw | dict(shared_prefix=shared)).cpu().double()
            assert out[1:4].isnan().all() and bool(((out - want).abs() <= bound)[[0, 4, 5]].all())


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("case,shared", [(([1] * 9, [70 + i for i in range(9)], 16, 4, 1, 128, True, None, None, 30.0), 64), (([260, 40], [300, 200], 16, 4, 2, 64, True, None, [50, 0], None), 0),
                                         (([1, 2], [900, 1000], 16, 4, 2, 256, True, None, None, None), 0)])
def test_results_in_the_place_of_the_queries(dev, case, shared, bits):
    tensors, kw = attend_case(case, torch.bfloat16, bits, shared=shared)
    want = attend(dev, tensors, kw | dict(shared_prefix=shared))
    q = tensors["q"].to(dev)
    again = attend(dev, tensors | dict(q=q), kw | dict(shared_prefix=shared), out=q)
    assert again.data_ptr() == q.data_ptr() and torch.equal(again, want)


@pytest.mark.parametrize("bits", [8, 16])
def test_one_table_row_for_a_whole_batch(dev, bits):
    """Sequences that have everything in common, their table one row expanded, queries a slice of a fused projection, and a prefix
    length given as a numpy integer."""
    import numpy

    tensors, kw = attend_case(([2] * 5, [96] * 5, 16, 4, 2, 128, True, None, None, None), torch.bfloat16, bits, shared=96)
    table = tensors["page_table"][:1].to(dev)
    want = attend(dev, tensors | dict(page_table=table.repeat(5, 1)), kw | dict(shared_prefix=96))
    wide = torch.zeros(10, 8, 128, dtype=torch.bfloat16, device=dev)
    wide[:, 2:6] = tensors["q"].to(dev)
    got = attend(dev, tensors | dict(page_table=table.expand(5, -1), q=wide[:, 2:6]), kw | dict(shared_prefix=numpy.int64(96)))
    assert torch.equal(got, want)
    expected, bound = oracle.attention(*(tensors | dict(page_table=tensors["page_table"][:1].repeat(5, 1))).values(), **kw)
    within(got, expected, bound)


def test_a_cache_without_pages(dev):
    """Nothing is there: rows without keys are zero, those that should see some NaN, slots are all outside."""
    pool = ops().fp8_cache(0, 16, 2, 64, device=dev)
    k, v = ops().read_fp8_cache(*pool, torch.tensor([0, -1, 5], device=dev))
    assert k.shape == (3, 2, 64) and not k.any() and not v.any()
    q = seeded((3, 4, 64), 1).to(dev)
    offsets, lens = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1, 3], [0, 5]))
    table = torch.full((2, 1), -1, dtype=torch.int32, device=dev)
    out = ops().paged_attention(q, pool[0], pool[1], table, offsets, lens, k_scales=pool[2], v_scales=pool[3])
    assert not out[0].any() and bool(out[1:].isnan().all())


def test_lengths_out_of_range(dev):
    for shared in (0, 32):
        tensors, kw = attend_case(([10, 6], [64, 64], 16, 2, 1, 64, False, None, None, 20.0), torch.bfloat16, 8, shared=64)
        tensors["page_table"] = tensors["page_table"][:, :2].contiguous()
        tensors["kv_lens"] = torch.tensor([10 ** 6, -4], dtype=torch.int32)
        want, bound = oracle.attention(*tensors.values(), **kw)
        for last in (16, 10 ** 6):
            tensors["q_offsets"] = torch.tensor([0, 10, last], dtype=torch.int32)
            within(attend(dev, tensors, kw | dict(shared_prefix=shared)), want, bound)


def test_capped_scores_of_any_size(dev):
    """Scores from far below the cap to far beyond it, infinite ones among them: cap tanh is finite."""
    tensors, kw = attend_case(([3, 40], [200, 90], 16, 4, 1, 128, True, None, None, 30.0), torch.bfloat16, 16)
    q = tensors["q"]
    q[0] *= 1e-3
    q[1] *= 100
    q[2] *= 1e30
    q[3, 0, 0] = math.inf
    want, bound = oracle.attention(*tensors.values(), **kw)
    out = attend(dev, tensors, kw)
    # (a score beyond fp32 is infinite, and its tanh 1 as well; with an infinite q some are inf - inf)
    keep = torch.ones(43, dtype=torch.bool)
    keep[3] = False
    within(out[keep.to(dev)], want[keep], bound[keep], "capped")
    # scores of a cap that does nothing are those of no cap, up to the cap's own rounding
    tensors, kw = attend_case(([5], [50], 16, 2, 1, 64, True, None, None, 1e4), torch.float16, 16)
    want, bound = oracle.attention(*tensors.values(), **(kw | dict(softcap=None)))
    within(attend(dev, tensors, kw), want, bound + 2.0 ** -7, "a high cap")


WIDE = [
    ([3, 40], [200, 90], 16, 4, 1, 64, True, None, None),
    ([300], [700], 16, 8, 2, 64, True, 130, [500]),
    ([1] * 9, [300 + 7 * i for i in range(9)], 16, 4, 2, 64, True, None, None),
    ([5, 0, 33], [70, 20, 100], 8, 2, 2, 80, False, None, None),
    ([20], [150], 16, 3, 1, 256, True, None, [60]),
]


@pytest.mark.parametrize("case", WIDE, ids=name_of)
@pytest.mark.parametrize("cap", [257.0, 3e4, 1e6, 1e20, 2.3e38])
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 16), (torch.bfloat16, 16), (torch.float16, 8)])
def test_caps_that_scores_are_far_below(dev, case, cap, dtype, bits):
    """Scores far below a cap are as exact as without one, those about it as its tanh, whatever their number.  The first token's are eight times
    as large: 64 products and sums of at most 2^-23 / 2 of sum_d |q_d k_d| scale < 2^9 move a probability by 2^-8 at most, and the tanh by less
    than 2^-10; the oracle's bound is at least 2^-9 of the same values, so three times that holds both."""
    d = case[5]
    tensors, kw = attend_case((*case, cap), dtype, bits, q_scale=8.0 if d == 64 else 1.0, shared=16 * 16 if len(case[0]) == 9 else 0)
    if d == 64:
        tensors["q"][0] *= 8
    want, bound = oracle.attention(*tensors.values(), **kw)
    within(attend(dev, tensors, kw), want, 3 * bound, f"cap {cap}")
    if len(case[0]) == 9:
        within(attend(dev, tensors, kw | dict(shared_prefix=256)), want, 3 * bound, f"cap {cap}, shared")


def test_plain_calls_are_the_same_bits(dev):
    """What asks for nothing more is the plain kernel; a prompt of nothing and a prefix of nothing change no bit either."""
    tensors, kw = attend_case(([5, 1, 40], [60, 33, 90], 16, 4, 2, 128, True, None, None, None), torch.bfloat16, 16)
    plain = attend(dev, tensors, dict(causal=True))
    assert torch.equal(attend(dev, tensors, dict(causal=True, prefix_lens=torch.zeros(3, dtype=torch.int32))), plain)
    assert torch.equal(attend(dev, tensors, dict(causal=True, shared_prefix=15)), plain)


def test_cache_beyond_32_bit_offsets(dev):
    """Codes past 2^32 bytes and scales past 2^31, written, read back and attended over."""
    pages, page, heads, kv_heads, d = 300_000, 64, 4, 2, 128
    k, v, ks, vs = ops().fp8_cache(pages, page, kv_heads, d, device=dev)
    assert k.numel() > 2 ** 32
    t = 100
    qkv = seeded((t, (heads + 2 * kv_heads) * d), 3).to(dev)
    ids = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32, device=dev)
    slots = (ids.long()[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[:t].contiguous()
    table, positions = ops().rope_table(128, d), torch.arange(t, device=dev)
    small = ops().fp8_cache(3, page, kv_heads, d, device=dev)
    args = (qkv, table, positions, heads, kv_heads, d)
    q, _ = ops().qk_norm_rope(*args, k_pages=k, v_pages=v, slots=slots, k_scales=ks, v_scales=vs)
    ops().qk_norm_rope(*args, k_pages=small[0], v_pages=small[1], slots=positions, k_scales=small[2], v_scales=small[3])
    for a, b in zip(ops().read_fp8_cache(k, v, ks, vs, slots), ops().read_fp8_cache(*small, positions)):
        assert torch.equal(a, b) and bool((a != 0).any())
    offsets, lens = torch.tensor([0, t], dtype=torch.int32, device=dev), torch.tensor([t], dtype=torch.int32, device=dev)
    a = ops().paged_attention(q, k, v, ids[None], offsets, lens, k_scales=ks, v_scales=vs)
    b = ops().paged_attention(q, small[0], small[1], torch.arange(3, dtype=torch.int32, device=dev)[None], offsets, lens, k_scales=small[2], v_scales=small[3])
    assert torch.equal(a, b)
