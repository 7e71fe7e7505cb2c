"""Block-scaled layers, attention over pages in the denoise loop, and the refusals of the operators' Python entry points."""

from __future__ import annotations

import pytest
import torch

import layer_oracle as oracle
from conftest import seeded

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(got, want, bound, what=""):
    off = (got.cpu().double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {((off - bound)[bad]).max():.3e} at {bad.nonzero()[0].tolist()}"


def bf16_equal(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.fixture(scope="module")
def L(dev):
    import phyai_amd.linear as linear

    torch.cuda.set_device(dev)
    linear.init()
    yield linear
    linear._reset_for_test()


def block_spec(L):
    return L.Fp8Spec(granularity=L.Granularity.BLOCK, block_shape=(128, 128))


def fill(layer, seed):
    w, ws = oracle.block_weight(*layer.weight.shape, gen(seed))
    layer.weight.data.copy_(w)
    layer.weight_scale.data.copy_(ws * 100 * layer.weight.shape[1] ** -0.5)
    return layer.weight.cpu(), layer.weight_scale.cpu()


# ---- layers ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [0, 1, 5, 50, 300])
@pytest.mark.parametrize("bias", [False, True])
def test_block_layer(L, dev, m, bias):
    layer = L.ReplicatedLinear(384, 256, bias=bias, params_dtype=torch.bfloat16, spec=block_spec(L))
    w, ws = fill(layer, m)
    if bias:
        layer.bias.data.copy_(seeded((256,), 3))
    b = layer.bias.cpu() if bias else None
    x = seeded((m, 384), 4)
    y, rest = layer(x.to(dev))
    assert rest is None and y.shape == (m, 256)
    if m == 0:
        return
    want, bound = oracle.block_gemm(*oracle.block_quant(x), w, ws, b)
    within(y, want, bound, "bf16 rows")
    # codes with one scale per token, from the spec's own quantizer, and a norm's with the quantizer in it
    view = layer.spec.quantize_activation(x.to(dev), layer)
    y, _ = layer(view)
    want, bound = oracle.block_gemm(view.x.cpu(), view.x_scale.cpu().reshape(m, 1), w, ws, b)
    within(y, want, bound, "codes")
    from phyai_amd.norm import RMSNorm

    view = RMSNorm(384).to(dev).forward_fp8(x.to(dev))
    want, bound = oracle.block_gemm(view.x.cpu(), view.x_scale.cpu().reshape(m, 1), w, ws, b)
    within(layer(view)[0], want, bound, "a norm's codes")


def test_block_layer_adds_a_gated_residual_and_leaves_its_bias_to_the_caller(L, dev):
    layer = L.RowParallelLinear(256, 128, bias=False, params_dtype=torch.bfloat16, spec=block_spec(L))
    fill(layer, 1)
    x, residual, gate = seeded((7, 256), 2).to(dev), seeded((7, 128), 3).to(dev), seeded((1, 128), 4).to(dev)
    y, _ = layer(x)
    assert bf16_equal(layer.forward_addcmul(x, residual, gate), torch.addcmul(residual, y, gate))
    other = L.ColumnParallelLinear(256, 128, bias=True, skip_bias_add=True, params_dtype=torch.bfloat16, spec=block_spec(L))
    other.weight.data.copy_(layer.weight)
    other.weight_scale.data.copy_(layer.weight_scale)
    other.bias.data.fill_(1.0)
    z, b = other(x)
    assert b is other.bias and bf16_equal(z, y)


def test_block_mlp(L, dev):
    from phyai_amd.mlp import DenseMLP

    mlp = DenseMLP(256, 384, activation="gelu_tanh", params_dtype=torch.bfloat16, spec_in=block_spec(L), spec_out=block_spec(L)).to(dev)
    w1, s1 = fill(mlp.gate_up_proj, 1)
    w2, s2 = fill(mlp.down_proj, 2)
    x = seeded((9, 256), 3)
    h, _ = mlp.gate_up_proj(x.to(dev))
    want, bound = oracle.block_gemm(*oracle.block_quant(x), w1, s1)
    within(h, want, bound, "first")
    a = mlp._unfused_act(h).cpu()
    want, bound = oracle.block_gemm(*oracle.block_quant(a), w2, s2)
    within(mlp(x.to(dev)), want, bound, "both")


# ---- the denoise loop over a paged cache ---------------------------------------------------------------------------

HIDDEN, LAYERS, STEPS, CHUNK, PREFIX, HEADS, HD = 256, 3, 2, 10, 37, 4, 64


def loop_of(L, dev, attend, spec, variant, use_graph):
    from phyai_amd.runtime.expert_loop import ExpertDenoiseLoop, ExpertLayer

    layers = []
    for i in range(LAYERS):
        lay = ExpertLayer(HIDDEN, HD, HEADS, 1, 512, HIDDEN, spec=spec).to(dev)
        for j, lin in enumerate((lay.qkv_proj, lay.o_proj, lay.mlp.gate_up_proj, lay.mlp.down_proj)):
            if spec is None:
                lin.spec.quantize_weight_(lin, seeded(tuple(lin.weight.shape), 10 * i + j, 0.05).to(dev))
            else:
                fill(lin, 10 * i + j)
        for j, norm in enumerate((lay.input_layernorm, lay.post_attention_layernorm)):
            norm.dense.weight.data.copy_(seeded(tuple(norm.dense.weight.shape), 100 + 10 * i + j, 0.02))
            norm.dense.bias.data.copy_(seeded(tuple(norm.dense.bias.shape), 200 + 10 * i + j, 0.1))
        layers.append(lay)
    lp = ExpertDenoiseLoop(layers, attend, chunk_size=CHUNK, action_dim=8, hidden_size=HIDDEN, cond_dim=HIDDEN, variant=variant, use_graph=use_graph)
    lp.embed_action.weight.data.copy_(seeded((HIDDEN, 8), 11, 0.3))
    lp.project_action.weight.data.copy_(seeded((8, HIDDEN), 12, 0.1))
    for lin in (lp.embed_action, lp.project_action):
        lin.bias.data.zero_()
    lp.final_norm.dense.weight.data.copy_(seeded((3 * HIDDEN, HIDDEN), 13, 0.02))
    lp.bind_euler_schedule(seeded((STEPS, HIDDEN), 7).to(dev), -1.0 / STEPS, STEPS)
    lp.setup()
    return lp


def paged(dev, **kw):
    from phyai_amd.runtime import PagedPrefixAttention

    attend = PagedPrefixAttention(LAYERS, CHUNK, PREFIX, HEADS, HD, device=dev, page_size=8, **kw)
    for i in range(LAYERS):
        attend.prefill(seeded((PREFIX, (HEADS + 2) * HD), 300 + i).to(dev), i)
    return attend


@pytest.mark.parametrize("blocks", [False, True])
def test_denoise_loop_over_pages_in_a_graph(L, dev, blocks):
    """Eager and replayed, fused and unfused: the same bits; the chunk's keys lie behind the prefix's."""
    spec = block_spec(L) if blocks else None
    results = []
    for variant, graph in (("fused", False), ("unfused", False), ("fused", True)):
        attend = paged(dev)
        lp = loop_of(L, dev, attend, spec, variant, graph)
        runs = []
        for seed in (1, 2, 1):
            runs.append(lp.run(seeded((CHUNK, 8), seed).to(dev)).clone())
            torch.cuda.synchronize()
        assert bool(torch.isfinite(runs[0].float()).all()) and bf16_equal(runs[0], runs[2]) and not bf16_equal(runs[0], runs[1])
        results.append((runs, [t.clone() for t in attend.k_pages]))
    for runs, pages in results[1:]:
        assert all(bf16_equal(a, b) for a, b in zip(runs, results[0][0]))
        assert all(bf16_equal(a, b) for a, b in zip(pages, results[0][1]))


@pytest.mark.parametrize("norms", [False, True])
def test_paged_prefix_attention_of_several_sequences(L, dev, norms):
    """Prefill and a chunk of sequences of unequal lengths (one without a prefix), against 64 bits."""
    from phyai_amd.runtime import PagedPrefixAttention

    lens, heads, kv_heads, d, chunk = [21, 0, 40], 4, 2, 64, 6
    weights = [(seeded((d,), 1, 0.3) + 1, seeded((d,), 2, 0.3) + 1)]
    attend = PagedPrefixAttention(1, chunk, lens, heads, d, kv_heads, device=dev, page_size=16,
                                  norms=[tuple(w.to(dev) for w in weights[0])] if norms else None)
    table = attend.cos_sin.cpu()
    for name, counts, start in (("prefill", lens, [0, 0, 0]), ("chunk", [chunk] * 3, lens)):
        n = sum(counts)
        qkv = seeded((n, (heads + 2 * kv_heads) * d), 5 + n)
        got = (attend.prefill if name == "prefill" else attend)(qkv.to(dev), 0)
        positions = torch.cat([torch.arange(s, s + c) for s, c in zip(start, counts)])
        rows = qkv.view(n, -1, d)
        keys, key_bound = oracle.head_rope(rows[:, heads: heads + kv_heads], weights[0][1] if norms else None, table, positions, 1e-6, False, False)
        q, bound = oracle.head_rope(rows[:, :heads], weights[0][0] if norms else None, table, positions, 1e-6, False, False)
        # what lies in the pages is within the rotation's bound of the oracle's keys; attention is checked on what lies there
        from phyai_amd import ops

        k_pages, v_pages = attend.k_pages[0].cpu(), attend.v_pages[0].cpu()
        slots = (attend._prefix if name == "prefill" else attend._chunk)[1].cpu()
        assert torch.equal(v_pages.view(-1, kv_heads, d)[slots], rows[:, heads + kv_heads:])
        within(k_pages.view(-1, kv_heads, d)[slots], keys, key_bound, "keys")
        q_gpu, _ = ops.qk_norm_rope(qkv.to(dev), attend.cos_sin, positions.to(dev), heads, kv_heads, d,
                                    **(dict(q_weight=weights[0][0].to(dev), k_weight=weights[0][1].to(dev)) if norms else {}))
        within(q_gpu, q, bound, "q")
        offsets = torch.tensor([sum(counts[:b]) for b in range(4)], dtype=torch.int32)
        kv = torch.tensor([s + c for s, c in zip(start, counts)], dtype=torch.int32)
        want, bound = oracle.paged_attention(q_gpu.cpu(), k_pages, v_pages, attend.page_table.cpu(), offsets, kv, causal=False)
        within(got.view(n, heads, d), want, bound, name)


# ---- refusals -----------------------------------------------------------------------------------------------------

def refuses(fn, *args, **kw):
    with pytest.raises((RuntimeError, ValueError)):
        fn(*args, **kw)


def test_block_ops_refuse(dev):
    from phyai_amd import ops

    x = seeded((4, 256), 1).to(dev)
    w, ws = (t.to(dev) for t in oracle.block_weight(128, 256, gen(1)))
    bias = seeded((128,), 1).to(dev)
    for a in ((x.float(), w, ws), (x.cpu(), w, ws), (x, w.cpu(), ws), (x, w, ws.cpu()), (x, w.float(), ws), (x, w[:, :240], ws), (x, w[:120], ws), (x, w.t(), ws),
              (x, w, ws.double()), (x, w, ws[:, :1]), (x, w, ws.t()), (x, w, ws, bias.float()), (x, w, ws, bias[:64]), (x, w, ws, bias.cpu()), (x[:, :128], w, ws),
              (x, None, ws), (x, w, None), (None, w, ws)):
        refuses(ops.fp8_block_linear, *a)
    for out in (torch.empty(4, 128, device=dev), torch.empty(4, 128, dtype=torch.bfloat16), torch.empty(4, 64, dtype=torch.bfloat16, device=dev),
                torch.empty(128, 4, dtype=torch.bfloat16, device=dev).t()):
        refuses(ops.fp8_block_linear, x, w, ws, out=out)
    codes, scale = ops.fp8_block_quant(x)
    for a in ((codes.cpu(), scale, w, ws), (codes, scale.cpu(), w, ws), (codes, scale[:3], w, ws), (codes, scale.t(), w, ws), (codes, scale.double(), w, ws),
              (x, scale, w, ws), (codes, None, w, ws), (codes, scale.reshape(-1), w, ws)):
        refuses(ops.fp8_block_gemm, *a)
    refuses(ops.fp8_block_quant, x.float())
    refuses(ops.fp8_block_quant, seeded((4, 60), 1).to(dev))
    refuses(ops.fp8_block_quant, x, out=torch.empty(4, 256, dtype=torch.uint8, device=dev))
    refuses(ops.fp8_block_quant, x, scale_out=torch.empty(4, 1, device=dev))


def test_qk_norm_rope_refuses(dev):
    from phyai_amd import ops

    heads, kv_heads, d, t = 4, 2, 64, 3
    qkv = seeded((t, 8 * d), 1).to(dev)
    table = ops.rope_table(16, d)
    pos = torch.arange(t, device=dev)
    w = seeded((d,), 2).to(dev)
    pages = [torch.zeros(4, 8, kv_heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    slots = torch.arange(t, device=dev)
    good = dict(qkv=qkv, cos_sin=table, positions=pos, num_heads=heads, num_kv_heads=kv_heads, head_dim=d)
    ops.qk_norm_rope(**good)
    for over in (dict(qkv=qkv.float()), dict(qkv=qkv.cpu()), dict(qkv=qkv[None]), dict(num_heads=5), dict(num_heads=0), dict(num_kv_heads=-2), dict(head_dim=60),
                 dict(head_dim=1024, num_heads=1, num_kv_heads=1), dict(cos_sin=table.double()), dict(cos_sin=table.cpu()), dict(cos_sin=table[:, :60]),
                 dict(cos_sin=ops.rope_table(16, 128)), dict(cos_sin=table[:0]), dict(positions=pos.int()), dict(positions=pos[:2]), dict(positions=pos.cpu()),
                 dict(q_weight=w), dict(q_weight=w, k_weight=w[:32]), dict(q_weight=w.float(), k_weight=w.float()), dict(q_weight=w.cpu(), k_weight=w.cpu()),
                 dict(k_pages=pages[0]), dict(k_pages=pages[0], v_pages=pages[1]), dict(slots=slots),
                 dict(k_pages=pages[0], v_pages=pages[1], slots=slots.int()), dict(k_pages=pages[0], v_pages=pages[1][:2], slots=slots),
                 dict(k_pages=pages[0].half(), v_pages=pages[1].half(), slots=slots), dict(k_pages=pages[0].cpu(), v_pages=pages[1], slots=slots),
                 dict(k_pages=pages[0][:, :, :1].expand(4, 8, 2, d), v_pages=pages[1], slots=slots),
                 dict(k_pages=pages[0], v_pages=pages[1][:1].expand(4, 8, 2, d), slots=slots),
                 dict(k_pages=pages[0][:, :, :1], v_pages=pages[1][:, :, :1], slots=slots), dict(out=torch.empty(t, heads, d, device=dev)),
                 dict(out=torch.empty(t, heads + 1, d, dtype=torch.bfloat16, device=dev))):
        refuses(ops.qk_norm_rope, **(good | over))


def test_paged_attention_refuses(dev):
    from phyai_amd import ops

    d = 64
    q = seeded((3, 4, d), 1).to(dev)
    k, v = (torch.zeros(6, 8, 2, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=dev)   # noqa: E731
    good = dict(q=q, k_pages=k, v_pages=v, page_table=i32(*range(6)).view(2, 3), q_offsets=i32(0, 1, 3), kv_lens=i32(9, 20))
    ops.paged_attention(**good)
    for over in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(q=q[:, :3]), dict(q=seeded((3, 4, 60), 1).to(dev)), dict(k_pages=k.half()), dict(v_pages=v.cpu()),
                 dict(k_pages=k[:3]), dict(k_pages=k[..., :32], v_pages=v[..., :32]), dict(v_pages=v.transpose(1, 2).contiguous().transpose(1, 2)),
                 dict(page_table=good["page_table"].long()), dict(page_table=good["page_table"][:1]), dict(page_table=good["page_table"].cpu()),
                 dict(page_table=good["page_table"][0]), dict(q_offsets=i32(0, 3)), dict(q_offsets=i32(0, 1, 3).long()), dict(kv_lens=i32(9)), dict(kv_lens=i32(9, 20).cpu()),
                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(window=0), dict(window=-3), dict(out=torch.empty_like(q, dtype=torch.float32)),
                 dict(out=torch.empty(3, 4, 32, dtype=torch.bfloat16, device=dev)), dict(out=torch.empty(4, 3, d, dtype=torch.bfloat16, device=dev).transpose(0, 1))):
        refuses(ops.paged_attention, **(good | over))


@pytest.mark.parametrize("plan", ["0", "2", "64"])
@pytest.mark.parametrize("page", [3, 16, 200])
def test_long_sequences_of_any_page_size(dev, monkeypatch, plan, page):
    """Keys beyond those whose places are looked up at once, pages that end inside every copy, more splits than blocks."""
    from test_gpu_layer_ops import attend_case

    from phyai_amd import ops

    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    for causal, window in ((True, None), (False, 700)):
        q, k, v, table, offsets, lens, kw = attend_case(([3, 40], [1501, 1090], page, 2, 1, 64, causal, window), torch.bfloat16, dev, seed=page)
        want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
        within(ops.paged_attention(*(t.to(dev) for t in (q, k, v, table, offsets, lens)), **kw), want, bound, f"{causal} {window}")


@pytest.mark.parametrize("plan", ["0", "1", "2"])
@pytest.mark.parametrize("d", [72, 128, 200])
@pytest.mark.parametrize("page", [16, 3])
def test_a_missing_page_reaches_only_the_rows_that_see_it(dev, monkeypatch, plan, d, page):
    """Its NaNs stay out of the keys that take its place in shared memory, whatever part of a buffer a key fills."""
    from test_gpu_layer_ops import attend_case

    from phyai_amd import ops

    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(([200], [500], page, 2, 1, d, True, 100), torch.bfloat16, dev, seed=d)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    gone = table.clone()
    at = 210 // page
    gone[0, at] = k.shape[0]
    out = ops.paged_attention(*(t.to(dev) for t in (q, k, v, gone, offsets, lens)), **kw).cpu()
    position = torch.arange(300, 500)
    sees = (position >= at * page) & (position - 99 < (at + 1) * page)
    assert bool(sees.any()) and bool((~sees).any())
    assert bool(torch.isnan(out[sees]).all())
    within(out[~sees], want[~sees], bound[~sees], "rows that do not see it")


@pytest.mark.parametrize("plan", ["0", "1"])
def test_uninitialised_places_of_a_cache_cost_and_change_nothing(dev, monkeypatch, plan):
    """Infinities behind the last key of a page, in the places whose copies are made all the same."""
    from test_gpu_layer_ops import attend_case

    from phyai_amd import ops

    monkeypatch.setenv("PHYAI_LAYER_ATTEND", plan)
    q, k, v, table, offsets, lens, kw = attend_case(([3, 50], [17, 129], 32, 4, 2, 128, False, None), torch.bfloat16, dev)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    for fill in (float("inf"), float("-inf"), float("nan"), 3e38):
        kk, vv = (torch.where(torch.isnan(t), torch.full_like(t, fill), t).to(dev) for t in (k, v))
        within(ops.paged_attention(q.to(dev), kk, vv, *(t.to(dev) for t in (table, offsets, lens)), **kw), want, bound, str(fill))


def test_a_cache_without_pages(dev):
    from phyai_amd import ops

    q = seeded((3, 4, 64), 1).to(dev)
    none = torch.zeros(0, 16, 2, 64, dtype=torch.bfloat16, device=dev)
    table, offsets = torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.tensor([0, 1, 3], dtype=torch.int32, device=dev)
    lens = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    out = ops.paged_attention(q, none, none, table, offsets, lens)
    assert not out[0].any() and bool(torch.isnan(out[1:]).all())
    assert not ops.paged_attention(q, none, none, table[:, :0], offsets, lens).any()   # a table of no pages: no keys
    assert ops.paged_attention(q[:0], none, none, table, offsets * 0, lens).shape == (0, 4, 64)


@pytest.mark.parametrize("heads", [1, 8])
def test_many_sequences_of_unequal_lengths(dev, heads):
    """More sequences than are looked at together, some without tokens or keys, in front of and behind rows of no sequence."""
    from test_gpu_layer_ops import cache

    from phyai_amd import ops

    g = gen(3)
    counts = torch.randint(0, 4, (300,), generator=g)
    kvs = [int(n) + int(x) for n, x in zip(counts, torch.randint(0, 50, (300,), generator=g))]
    k, v, table = cache(kvs, 8, 1, 64, torch.bfloat16, 4)
    first = 5
    offsets = (torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]) + first).int()
    total = int(offsets[-1]) + 7
    q = seeded((total, heads, 64), 5)
    lens = torch.tensor(kvs, dtype=torch.int32)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens)
    out = torch.full((total, heads, 64), 7.0, dtype=torch.bfloat16, device=dev)
    ops.paged_attention(*(t.to(dev) for t in (q, k, v, table, offsets, lens)), out=out)
    inside = slice(first, int(offsets[-1]))
    within(out[inside], want[inside], bound[inside], "rows")
    assert bool((out[:first] == 7).all()) and bool((out[int(offsets[-1]):] == 7).all())


def test_one_token_of_a_padded_batch_leaves_the_padding_alone(dev):
    """Split over many workgroups, with rows behind the last sequence."""
    from test_gpu_layer_ops import attend_case

    from phyai_amd import ops

    q, k, v, table, offsets, lens, kw = attend_case(([1, 1], [3000, 17], 16, 4, 1, 128, True, None), torch.bfloat16, dev)
    want, bound = oracle.paged_attention(q, k, v, table, offsets, lens, **kw)
    padded = torch.cat([q, seeded((6, 4, 128), 9)]).to(dev)
    out = torch.full((8, 4, 128), 7.0, dtype=torch.bfloat16, device=dev)
    ops.paged_attention(padded, *(t.to(dev) for t in (k, v, table, offsets, lens)), out=out, **kw)
    within(out[:2], want, bound, "rows")
    assert bool((out[2:] == 7).all())
    replaced = padded.clone()
    ops.paged_attention(replaced, *(t.to(dev) for t in (k, v, table, offsets, lens)), out=replaced, **kw)   # q's own place
    assert bf16_equal(replaced[:2], out[:2]) and bf16_equal(replaced[2:], padded[2:])


@pytest.mark.parametrize("t,heads,kv_heads,d,rot", [(2200, 12, 3, 72, 48), (9000, 4, 1, 128, 128)])
def test_head_norms_and_rotation_of_many_tokens(dev, t, heads, kv_heads, d, rot):
    """More heads than fit the chip at once: an odd number of them, query, key and value heads in one group."""
    from phyai_amd import ops

    qkv = seeded((t, (heads + 2 * kv_heads) * d), 1)
    table = ops.rope_table(t, rot, device="cpu")
    positions = torch.randperm(t, generator=gen(2))
    weights = [seeded((d,), s, 0.3) + 1 for s in (3, 4)]
    k_pages, v_pages = (torch.zeros(-(-t // 16), 16, kv_heads, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    slots = torch.randperm(t, generator=gen(3))
    q, _ = ops.qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, q_weight=weights[0].to(dev), k_weight=weights[1].to(dev),
                            k_pages=k_pages, v_pages=v_pages, slots=slots.to(dev))
    rows = qkv.view(t, -1, d)
    within(q, *oracle.head_rope(rows[:, :heads], weights[0], table, positions, 1e-6, False, False), "q")
    within(k_pages.cpu().view(-1, kv_heads, d)[slots], *oracle.head_rope(rows[:, heads: heads + kv_heads], weights[1], table, positions, 1e-6, False, False), "k")
    assert torch.equal(v_pages.cpu().view(-1, kv_heads, d)[slots], rows[:, heads + kv_heads:])
    q2, k2 = ops.qk_norm_rope(qkv.to(dev), table.to(dev), positions.to(dev), heads, kv_heads, d, q_weight=weights[0].to(dev), k_weight=weights[1].to(dev))
    assert bf16_equal(q2, q) and bf16_equal(k2.cpu(), k_pages.cpu().view(-1, kv_heads, d)[slots])


def test_sequences_that_share_a_row_of_the_table(dev):
    """An expanded table, and one of a single column that lies across another."""
    from test_gpu_layer_ops import attend_case

    from phyai_amd import ops

    q, k, v, table, offsets, lens, kw = attend_case(([2, 3, 1], [40, 40, 40], 16, 2, 1, 64, True, None), torch.bfloat16, dev)
    one = table[:1].to(dev)
    rest = [t.to(dev) for t in (offsets, lens)]
    want = ops.paged_attention(q.to(dev), k.to(dev), v.to(dev), one.repeat(3, 1), *rest, **kw)
    assert bf16_equal(ops.paged_attention(q.to(dev), k.to(dev), v.to(dev), one.expand(3, -1), *rest, **kw), want)
    lens = torch.tensor([16, 9, 3], dtype=torch.int32, device=dev)
    column = table[:, :1].to(dev)
    want = ops.paged_attention(q.to(dev), k.to(dev), v.to(dev), column.contiguous(), rest[0], lens, **kw)
    across = column.t().contiguous().t()
    assert across.stride(0) == 1 and bf16_equal(ops.paged_attention(q.to(dev), k.to(dev), v.to(dev), across, rest[0], lens, **kw), want)
