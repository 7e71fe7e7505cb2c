"""Block-scaled linear, head norms with rotation and cache write, attention over pages: against plain forms in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import layer_oracle as oracle
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


# ---- block-scaled linear -------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,k", [(1, 8), (1, 128), (3, 136), (17, 1024), (5, 4304), (130, 2040)])
def test_block_quant_is_exact(dev, m, k):
    x = seeded((m, k), 1, 3.0)
    x[:, ::37] *= 50
    x[0, : min(k, 128)] = 0                       # a block of zeros
    if m > 2:
        x[1, 0], x[2, -1] = 1e-30, 3e38           # far below the floor; the largest
    codes, scale = ops().fp8_block_quant(x.to(dev))
    want, want_scale = oracle.block_quant(x)
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))


def test_block_quant_of_every_ratio(dev):
    """Codes on rounding borders: each finite bf16 magnitude class against blocks of every maximum's mantissa."""
    mantissas = torch.arange(128, dtype=torch.int32)
    tops = ((127 + 3) << 7 | mantissas).to(torch.int16).view(torch.bfloat16)
    rows = []
    for shift in range(0, 12):
        values = ((127 + 3 - shift) << 7 | mantissas).to(torch.int16).view(torch.bfloat16)
        x = values[None, :].repeat(128, 1)
        x = torch.where(x.float() > tops.float()[:, None], tops[:, None], x)
        x[:, 0] = tops
        rows.append(x)
    x = torch.cat(rows)
    codes, scale = ops().fp8_block_quant(x.to(dev))
    want, want_scale = oracle.block_quant(x)
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(codes.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_block_quant_special_values_stay_in_their_block(dev, value):
    x = seeded((2, 384), 2)
    x[0, 130] = value
    codes, scale = ops().fp8_block_quant(x.to(dev))
    codes, scale = codes.cpu().float(), scale.cpu()
    assert math.isnan(codes[0, 130]) and not torch.isfinite(scale[0, 1])
    clean, clean_scale = oracle.block_quant(x)
    rest = torch.ones(2, 384, dtype=torch.bool)
    rest[0, 128:256] = False
    assert torch.equal(codes[rest], clean.float()[rest]) and torch.equal(scale[1], clean_scale[1])


SHAPES = [(1, 16, 16), (2, 144, 4224), (8, 272, 8304), (4, 64, 1072), (1, 256, 128), (3, 144, 272), (16, 128, 1024), (17, 2560, 1024), (33, 272, 4304), (50, 1024, 512), (64, 160, 1168),
          (65, 144, 144), (100, 400, 256), (129, 272, 1040), (200, 528, 2064), (300, 256, 128), (257, 784, 384)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("shape", [None, "few 1", "few 2", "few 4", "few 11", "few 12", "few 14", "few 31", "few 32", "1", "2", "3", "4"])
def test_block_linear(dev, monkeypatch, m, n, k, shape):
    if shape is not None:
        few, _, small = shape.partition(" ")
        monkeypatch.setenv("PHYAI_LAYER_BLOCK", "0" if small else few)
        if small:
            monkeypatch.setenv("PHYAI_LAYER_SMALL", small)
    x = seeded((m, k), m + n, 1.0)
    x[:, :: max(1, k // 7)] *= 20
    w, ws = oracle.block_weight(n, k, gen(k))
    bias = seeded((n,), 5) if (m + n) % 3 else None
    codes, scale = oracle.block_quant(x)
    want, bound = oracle.block_gemm(codes, scale, w, ws, bias)
    args = [t.to(dev) if t is not None else None for t in (w, ws, bias)]
    y = ops().fp8_block_linear(x.to(dev), *args)
    within(y, want, bound, "linear")
    z = ops().fp8_block_gemm(codes.to(dev), scale.to(dev), *args)
    within(z, want, bound, "gemm")
    # one scale per token row, as the norms fused with a quantizer leave it
    rows = scale[:, :1].contiguous()
    want, bound = oracle.block_gemm(codes, rows, w, ws, bias)
    within(ops().fp8_block_gemm(codes.to(dev), rows.to(dev), *args), want, bound, "gemm, scale per row")


@pytest.mark.parametrize("m", [3, 70])
def test_block_linear_of_strided_rows_and_leading_dims(dev, m):
    n, k = 144, 272
    wide = seeded((m, 400), 9).to(dev)
    w, ws = (t.to(dev) for t in oracle.block_weight(n, k, gen(1)))
    want = ops().fp8_block_linear(wide[:, 8: 8 + k].contiguous(), w, ws)
    assert torch.equal(ops().fp8_block_linear(wide[:, 8: 8 + k], w, ws), want)
    assert torch.equal(ops().fp8_block_linear(wide[:, 5: 5 + k], w, ws), ops().fp8_block_linear(wide[:, 5: 5 + k].contiguous(), w, ws))
    x3 = wide[:, 8: 8 + k].reshape(1, m, k)
    out = torch.full((1, m, n), 7.0, dtype=torch.bfloat16, device=dev)
    assert ops().fp8_block_linear(x3, w, ws, out=out) is out and torch.equal(out[0], want)
    assert ops().fp8_block_linear(x3[:, :0], w, ws).shape == (1, 0, n)


def test_block_linear_nan_stays_in_its_row(dev):
    for m in (5, 200):
        x = seeded((m, 256), 3)
        w, ws = (t.to(dev) for t in oracle.block_weight(256, 256, gen(3)))
        clean = ops().fp8_block_linear(x.to(dev), w, ws)
        x[2, 200] = math.nan
        y = ops().fp8_block_linear(x.to(dev), w, ws)
        keep = torch.arange(m) != 2
        assert y[2].isnan().all() and torch.equal(y[keep], clean[keep])


# ---- head norms, rotation, cache write -----------------------------------------------------------------------------

HEADS = [(1, 1, 1, 8, 8), (5, 8, 1, 256, 256), (3, 4, 2, 64, 32), (7, 12, 3, 72, 48), (2, 5, 5, 80, 80), (4, 6, 2, 96, 64), (9, 2, 1, 128, 0),
         (3, 3, 1, 512, 512), (6, 2, 2, 24, 8), (65, 16, 4, 128, 128), (2, 40, 8, 112, 104)]


@pytest.mark.parametrize("t,heads,kv_heads,d,rot", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [None, "plain", "gemma"])
def test_qk_norm_rope(dev, t, heads, kv_heads, d, rot, dtype, interleaved, norm):
    qkv = seeded((t, (heads + 2 * kv_heads) * d), t + d, 2.0, dtype)
    qkv[t // 2, :d] = 0                                        # a head of zeros: eps decides
    table = ops().rope_table(4096, rot, device="cpu") if rot else torch.zeros(4096, 0)
    positions = torch.randint(0, 4096, (t,), generator=gen(t))
    positions[0] = 4095
    weights = [seeded((d,), s, 0.5, dtype) for s in (1, 2)] if norm else [None, None]
    rows = qkv.view(t, -1, d)
    want_q, bound_q = oracle.head_rope(rows[:, :heads], weights[0], table, positions, 1e-6, norm == "gemma", interleaved)
    want_k, bound_k = oracle.head_rope(rows[:, heads: heads + kv_heads], weights[1], table, positions, 1e-6, norm == "gemma", interleaved)
    on = [w.to(dev) if w is not None else None for w in weights]
    kw = dict(q_weight=on[0], k_weight=on[1], gemma=norm == "gemma", interleaved=interleaved)
    q, k = ops().qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, **kw)
    within(q, want_q, bound_q, "q")
    within(k, want_k, bound_k, "k")
    # the same into pages that lie head by head, with padding in the batch
    page = 3
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=gen(3))[:t]
    slots[-1] = -1 if t > 1 else pages * page
    k_pages = torch.full((pages, kv_heads, page, d), 7.0, dtype=dtype, device=dev).transpose(1, 2)
    v_pages = torch.full((pages, page, kv_heads, d), 7.0, dtype=dtype, device=dev)
    q2, none = ops().qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, k_pages=k_pages, v_pages=v_pages,
                                  slots=slots.to(dev), **kw)
    assert none is None and torch.equal(q2, q)
    want = torch.full((pages * page, kv_heads, d), 7.0, dtype=dtype)
    want_v = want.clone()
    want[slots[:-1]] = k.cpu()[:-1]
    want_v[slots[:-1]] = rows[:-1, heads + kv_heads:]
    assert torch.equal(k_pages.cpu().reshape(-1, kv_heads, d), want) and torch.equal(v_pages.cpu().reshape(-1, kv_heads, d), want_v)


def test_qk_norm_rope_positions_outside_the_table(dev):
    qkv = seeded((4, 3 * 64), 1).to(dev)
    table = ops().rope_table(8, 32)
    q, k = ops().qk_norm_rope(qkv, table, torch.tensor([7, 8, -1, 0], device=dev), 1, 1, 64)
    assert q[0].isfinite().all() and q[3].isfinite().all()
    for t in (1, 2):
        assert q[t, :, :32].isnan().all() and k[t, :, :32].isnan().all() and torch.equal(q[t, 0, 32:], qkv[t, 32:64])


def test_qk_norm_rope_of_strided_rows(dev):
    wide = seeded((6, 800), 4).to(dev)
    table, pos = ops().rope_table(16, 64), torch.arange(6, device=dev)
    part = wide[:, 16: 16 + 6 * 64]
    a = ops().qk_norm_rope(part, table, pos, 4, 1, 64)
    b = ops().qk_norm_rope(part.contiguous(), table, pos, 4, 1, 64)
    c = ops().qk_norm_rope(wide[:, 3: 3 + 6 * 64], table, pos, 4, 1, 64)
    d = ops().qk_norm_rope(wide[:, 3: 3 + 6 * 64].contiguous(), table, pos, 4, 1, 64)
    assert all(torch.equal(x, y) for x, y in zip(a + c, b + d))
    q, k = ops().qk_norm_rope(part[:0], table, pos[:0], 4, 1, 64)
    assert q.shape == (0, 4, 64) and k.shape == (0, 1, 64)


# ---- attention over pages ---------------------------------------------------------------------------------------

def cache(kvs, page, kv_heads, d, dtype, seed, spare=3, layout="token"):
    """Pages of sequences of kvs keys in random order, unused places full of NaN; (k_pages, v_pages, page_table) on the CPU."""
    g = gen(seed)
    counts = [-(-kv // page) for kv in kvs]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g).int()
    width = max(counts) + 1
    table = torch.full((len(kvs), width), -5, dtype=torch.int32)
    k = torch.full((pages, page, kv_heads, d), math.nan, dtype=dtype)
    v = k.clone()
    at = 0
    for b, (kv, n) in enumerate(zip(kvs, counts)):
        ids = order[at: at + n]
        at += n
        table[b, :n] = ids
        for j in range(n):
            fill = min(page, kv - j * page)
            k[ids[j].long(), :fill] = torch.randn(fill, kv_heads, d, generator=g).to(dtype)
            v[ids[j].long(), :fill] = torch.randn(fill, kv_heads, d, generator=g).to(dtype)
    return k, v, table


def to_gpu(t, dev, layout):
    return t.to(dev) if layout == "token" else t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)


# new tokens and keys per sequence, page, heads, key heads, head_dim, causal, window
ATTEND = [
    ([1], [1], 16, 8, 1, 256, True, None),
    ([1], [33], 16, 1, 1, 64, True, None),
    ([1, 1, 1], [70, 1, 129], 16, 8, 2, 128, True, None),
    ([1, 0, 2, 0], [5, 9, 40, 0], 1, 4, 4, 64, True, None),
    ([5, 3], [3, 0], 16, 2, 1, 64, True, None),              # rows before the first key, and a sequence without keys
    ([50], [130], 16, 8, 1, 256, False, None),
    ([37, 64], [37, 100], 24, 5, 1, 80, True, None),
    ([40], [40], 3, 6, 3, 72, True, 7),
    ([33, 1], [200, 90], 64, 4, 2, 128, True, 33),
    ([20], [90], 16, 4, 1, 64, False, 12),
    ([100], [170], 16, 3, 3, 8, True, 1),
    ([130], [300], 32, 8, 2, 256, True, 64),
    ([70], [90], 256, 2, 2, 200, True, None),
    ([1] * 70, list(range(1, 71)), 8, 2, 1, 64, True, None),  # more sequences than a wavefront looks at together
]


def attend_case(case, dtype, dev, layout="token", seed=0, q_scale=1.0):
    qs, kvs, page, heads, kv_heads, d, causal, window = case
    k, v, table = cache(kvs, page, kv_heads, d, dtype, seed + 1)
    offsets = torch.tensor([0] + qs).cumsum(0).int()
    q = seeded((int(offsets[-1]), heads, d), seed + 2, q_scale, dtype)
    lens = torch.tensor(kvs, dtype=torch.int32)
    return q, k, v, table, offsets, lens, dict(causal=causal, window=window)


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"q{max(c[0])}kv{max(c[1])}p{c[2]}h{c[3]}k{c[4]}d{c[5]}{'c' if c[6] else 'f'}{c[7] or ''}")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("plan", [None, "0", "1", "3"])
def test_paged_attention(dev, monkeypatch, case, dtype, plan):
    if plan is not None:
        monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(case, dtype, dev)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    layout = "head" if plan == "1" else "token"
    out = ops().paged_attention(q.to(dev), to_gpu(k, dev, layout), to_gpu(v, dev, layout), table.to(dev), offsets.to(dev), lens.to(dev), **kw)
    within(out, want, bound, "attention")


@pytest.mark.parametrize("plan", ["0", "2"])
def test_paged_attention_leaves_other_rows_alone(dev, monkeypatch, plan):
    """Rows in front of the first sequence, between sequences (a gap in the offsets is a sequence without keys here) and behind
    the last one."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, _, lens, kw = attend_case(([4, 30], [9, 50], 16, 4, 2, 64, True, None), torch.bfloat16, dev)
    q = seeded((50, 4, 64), 2)
    offsets = torch.tensor([3, 7, 37], dtype=torch.int32)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    out = torch.full((50, 4, 64), 7.0, dtype=torch.bfloat16, device=dev)
    ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), offsets.to(dev), lens.to(dev), out=out, **kw)
    within(out[3:37], want[3:37], bound[3:37])
    assert bool((out[:3] == 7).all()) and bool((out[37:] == 7).all())


@pytest.mark.parametrize("plan", ["0", "1", "2"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 20), (False, 25)])
def test_special_values_reach_only_the_rows_that_see_them(dev, monkeypatch, plan, value, causal, window):
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)):
        q, k, v, table, offsets, lens, kw = attend_case(([70], [100], 16, 2, 1, d, causal, window), dtype, dev)
        clean, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
        at = {60: 3, 75: 5, 99: d - 1}
        for j, dim in at.items():
            v[table[0, j // 16].long(), j % 16, 0, dim] = value
        out = ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), offsets.to(dev), lens.to(dev), **kw).cpu().double()
        hit = torch.zeros(70, 2, d, dtype=torch.bool)
        for i in range(70):
            position = 30 + i
            for j, dim in at.items():
                if (j <= position or not causal) and (window is None or j > position - window):
                    hit[i, :, dim] = True
        same = out.isnan() if math.isnan(value) else out == value
        assert bool(same[hit].all()) and bool((((out - clean).abs() <= bound) | hit).all()), (d, dtype)


@pytest.mark.parametrize("plan", ["0", "1"])
def test_special_keys_in_masked_places(dev, monkeypatch, plan):
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(([40], [70], 16, 2, 1, 128, True, None), torch.bfloat16, dev)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    k[table[0, 60 // 16].long(), 60 % 16] = math.nan
    out = ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), offsets.to(dev), lens.to(dev), **kw).cpu().double()
    assert bool(((out - want).abs() <= bound)[:30].all()) and out[30:].isnan().all()


@pytest.mark.parametrize("plan", ["0", "1", "4"])
def test_pages_that_do_not_exist(dev, monkeypatch, plan):
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(([60, 3], [90, 20], 16, 2, 1, 64, True, None), torch.bfloat16, dev)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 4] = bad                             # keys 64 .. 79, seen from position 64 = token 34 on
        out = ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), t.to(dev), offsets.to(dev), lens.to(dev), **kw).cpu().double()
        good = torch.ones(63, dtype=torch.bool)
        good[34:60] = False
        assert out[~good].isnan().all() and bool(((out - want).abs() <= bound)[good].all())


@pytest.mark.parametrize("plan", ["0", "2"])
def test_lengths_and_offsets_out_of_range_stay_in_bounds(dev, monkeypatch, plan):
    """More keys than the table has pages for: what exists is seen.  Negative lengths are none; offsets are held inside q."""
    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(([10, 6], [64, 32], 16, 2, 1, 64, False, None), torch.bfloat16, dev)
    table = table[:, :2].contiguous()
    lens = torch.tensor([10 ** 6, -4], dtype=torch.int32)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, torch.tensor([32, 0]), **kw)
    far = torch.tensor([0, 10, 10 ** 6], dtype=torch.int32)
    for o in (offsets, far):
        out = ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), o.to(dev), lens.to(dev), **kw)
        within(out, want, bound)


def test_large_scores(dev):
    """Scores of hundreds: one key takes nearly all; the running maximum moves by more than the rescaling threshold."""
    for plan_rows, d in ((1, 128), (40, 256)):
        q, k, v, table, offsets, lens, kw = attend_case(([plan_rows], [300], 16, 4, 1, d, True, None), torch.bfloat16, dev, q_scale=1.0)
        k = (k.float() * torch.linspace(0.05, 1.0, 16)[None, :, None, None]).bfloat16()
        q = (q.float() * 4).bfloat16()
        want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
        out = ops().paged_attention(q.to(dev), k.to(dev), v.to(dev), table.to(dev), offsets.to(dev), lens.to(dev), **kw)
        within(out, want, bound)


def test_cache_beyond_32_bit_offsets(dev):
    """Pages whose elements lie past 2^31 (and bytes past 2^32), written by qk_norm_rope and read by paged_attention."""
    pages, page, heads, kv_heads, d = 140_000, 16, 4, 2, 512 // 2
    pool = torch.empty(2, pages, page, kv_heads, d, dtype=torch.bfloat16, device=dev)     # 2 x 1.15e9 elements: the values' end past 2^31
    assert pool.numel() > 2 ** 31
    k_pages, v_pages = pool[0], pool[1]
    t = 40
    qkv = seeded((t, (heads + 2 * kv_heads) * d), 3).to(dev)
    ids = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32, device=dev)
    slots = (ids.long()[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[:t].contiguous()
    table = ops().rope_table(64, d)
    q, _ = ops().qk_norm_rope(qkv, table, torch.arange(t, device=dev), heads, kv_heads, d, k_pages=k_pages, v_pages=v_pages, slots=slots)
    small_k, small_v = (torch.zeros(3, page, kv_heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops().qk_norm_rope(qkv, table, torch.arange(t, device=dev), heads, kv_heads, d, k_pages=small_k, v_pages=small_v,
                       slots=torch.arange(t, device=dev))
    offsets, lens = torch.tensor([0, t], dtype=torch.int32, device=dev), torch.tensor([t], dtype=torch.int32, device=dev)
    a = ops().paged_attention(q, k_pages, v_pages, ids[None], offsets, lens)
    b = ops().paged_attention(q, small_k, small_v, torch.arange(3, dtype=torch.int32, device=dev)[None], offsets, lens)
    assert torch.equal(a, b)


# ---- together, and in graphs ------------------------------------------------------------------------------------

def test_the_attention_half_of_a_layer(dev):
    """Block-scaled projection, head norms with rotation into pages, attention, block-scaled output projection - prefill, a chunk, a
    single token - against the same in 64 bits with the roundings between the steps."""
    hidden, heads, kv_heads, d, page = 256, 4, 2, 64, 8
    w, ws = oracle.block_weight((heads + 2 * kv_heads) * d, hidden, gen(1))
    wo, wos = oracle.block_weight(hidden, heads * d, gen(2))
    weights = [seeded((d,), s, 0.3) + 1 for s in (3, 4)]
    table = ops().rope_table(64, d, device="cpu")
    pages = torch.tensor([[4, 1, 6, 0]], dtype=torch.int32)
    k_pages, v_pages = (torch.zeros(7, page, kv_heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    on = lambda t: t.to(dev)   # noqa: E731
    done = 0
    for n in (17, 5, 1):
        x = seeded((n, hidden), 10 + n)
        slots = (pages[0].long()[:, None] * page + torch.arange(page)).reshape(-1)[done: done + n]
        qkv = ops().fp8_block_linear(on(x), on(w), on(ws))
        want, bound = oracle.block_gemm(*oracle.block_quant(x), w, ws)
        within(qkv, want, bound, "projection")
        positions = torch.arange(done, done + n)
        q, _ = ops().qk_norm_rope(qkv, on(table), on(positions), heads, kv_heads, d, q_weight=on(weights[0]), k_weight=on(weights[1]),
                                  k_pages=k_pages, v_pages=v_pages, slots=on(slots))
        rows = qkv.cpu().view(n, -1, d)
        want, bound = oracle.head_rope(rows[:, :heads], weights[0], table, positions, 1e-6, False, False)
        within(q, want, bound, "q")
        want, bound = oracle.head_rope(rows[:, heads: heads + kv_heads], weights[1], table, positions, 1e-6, False, False)
        within(k_pages.view(-1, kv_heads, d)[on(slots)], want, bound, "k")
        assert torch.equal(v_pages.cpu().view(-1, kv_heads, d)[slots], rows[:, heads + kv_heads:])
        done += n
        offsets, lens = torch.tensor([0, n], dtype=torch.int32), torch.tensor([done], dtype=torch.int32)
        a = ops().paged_attention(q, k_pages, v_pages, on(pages), on(offsets), on(lens))
        want, bound = oracle.paged_attention(q.cpu(), k_pages.cpu(), v_pages.cpu(), pages, offsets, lens)
        within(a, want, bound, "attention")
        y = ops().fp8_block_linear(a.view(n, heads * d), on(wo), on(wos))
        want, bound = oracle.block_gemm(*oracle.block_quant(a.cpu().view(n, heads * d)), wo, wos)
        within(y, want, bound, "output")


@pytest.mark.parametrize("n", [3, 90])
def test_replayed_from_a_graph(dev, n):
    """Two graphs of the same calls with other eager work between their replays; lengths, slots and pages change in place."""
    from phyai_amd.runtime import HipGraph

    heads, kv_heads, d, page, hidden = 8, 1, 256, 16, 512
    w, ws = (t.to(dev) for t in oracle.block_weight((heads + 2 * kv_heads) * d, hidden, gen(5)))
    table = ops().rope_table(1024, d)
    k_pages, v_pages = (torch.zeros(60, page, kv_heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    pages = torch.randperm(60, generator=gen(6)).int().to(dev)[None].contiguous()
    offsets = torch.tensor([0, n], dtype=torch.int32, device=dev)

    def step(x, lens, positions, slots):
        qkv = ops().fp8_block_linear(x, w, ws)
        q, _ = ops().qk_norm_rope(qkv, table, positions, heads, kv_heads, d, k_pages=k_pages, v_pages=v_pages, slots=slots)
        return ops().paged_attention(q, k_pages, v_pages, pages, offsets, lens)

    def inputs(done, seed):
        places = (pages[0].long()[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[done: done + n].contiguous()
        return dict(x=seeded((n, hidden), seed).to(dev), lens=torch.tensor([done + n], dtype=torch.int32, device=dev),
                    positions=torch.arange(done, done + n, device=dev), slots=places)

    graphs = [HipGraph(), HipGraph()]
    for g in graphs:
        g.capture(step, inputs(0, 0))
    done = 0
    for i in range(6):
        args = inputs(done, i)
        want = step(**args).clone()
        for g in graphs:
            got = g.replay(args)
            ops().fp8_block_linear(seeded((n + 70, hidden), 99).to(dev), w, ws)
            torch.cuda.synchronize()
            assert torch.equal(got, want), i
        done += n


def test_two_streams_at_once(dev):
    q, k, v, table, offsets, lens, kw = attend_case(([3, 2], [900, 700], 16, 8, 1, 256, True, None), torch.bfloat16, dev)
    args = [t.to(dev) for t in (q, k, v, table, offsets, lens)]
    x = seeded((200, 512), 1).to(dev)
    w, ws = (t.to(dev) for t in oracle.block_weight(512, 512, gen(5)))
    want, want_y = ops().paged_attention(*args, **kw), ops().fp8_block_linear(x, w, ws)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                results.append((ops().paged_attention(*args, **kw), ops().fp8_block_linear(x, w, ws)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(y, want_y) for a, y in results)
