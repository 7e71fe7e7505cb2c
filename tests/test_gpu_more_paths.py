"""The operators around a cache in 8 bits together, as a decoder layer uses them: in turn, from graphs, on two streams, through the
modules that call them; and the calls that are refused."""

from __future__ import annotations

import pytest
import torch

import layer_oracle
import more_oracle as oracle
from conftest import seeded
from test_gpu_more_ops import attend, attend_case, gen, ops, raw, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L(dev):
    import phyai_amd.linear as linear

    torch.cuda.set_device(dev)
    linear.init()
    yield linear
    linear._reset_for_test()


def test_the_attention_half_of_a_layer(dev):
    """A prompt whose first tokens see each other, then three sequences that go on from it with one and two tokens: residual and norm,
    projection, heads into the cache in 8 bits, capped attention, output projection - each step against 64 bits on what the one before
    left."""
    hidden, heads, kv_heads, d, page, prompt, cap = 256, 4, 2, 64, 8, 24, 20.0
    w, ws = layer_oracle.block_weight((heads + 2 * kv_heads) * d, hidden, gen(1))
    wo, wos = layer_oracle.block_weight(hidden, heads * d, gen(2))
    norm = seeded((hidden,), 5, 0.2) + 1
    table = ops().rope_table(64, d, device="cpu")
    on = lambda t: t.to(dev)   # noqa: E731
    k, v, ks, vs = ops().fp8_cache(12, page, kv_heads, d, device=dev)
    pages = torch.tensor([[4, 1, 6, 0, 9], [4, 1, 6, 2, 10], [4, 1, 6, 3, 11]], dtype=torch.int32)
    stages = [(pages[:1], [prompt], [prompt], torch.tensor([10]), 0), (pages, [1, 2, 1], [25, 26, 25], None, prompt), (pages, [1, 1, 2], [26, 27, 27], None, prompt)]
    for n, (ids, counts, lens, prompts, shared) in enumerate(stages):
        t = sum(counts)
        x, residual = seeded((t, hidden), 10 + n), seeded((t, hidden), 20 + n, 2.0)
        codes, scale, total = ops().add_rmsnorm_fp8(on(x), on(residual), on(norm))
        want, n64 = oracle.add_norm(x, residual, norm, 1e-6, False)
        assert torch.equal(total.cpu(), want)
        oracle.check_norm_codes(codes, scale, n64, True)
        qkv = ops().fp8_block_gemm(codes, scale, on(w), on(ws))
        want, bound = layer_oracle.block_gemm(codes.cpu(), scale.cpu(), w, ws)
        within(qkv, want, bound, "projection")
        positions = torch.cat([torch.arange(kv - c, kv) for c, kv in zip(counts, lens)])
        slots = torch.cat([(ids[b].long()[:, None] * page + torch.arange(page)).reshape(-1)[kv - c: kv] for b, (c, kv) in enumerate(zip(counts, lens))])
        q, _ = ops().qk_norm_rope(qkv, on(table), on(positions), heads, kv_heads, d, k_pages=k, v_pages=v, slots=on(slots), k_scales=ks, v_scales=vs)
        rows = qkv.cpu().view(t, -1, d)
        want, bound = layer_oracle.head_rope(rows[:, :heads], None, table, positions, 1e-6, False, False)
        within(q, want, bound, "q")
        at = (slots // page, slots % page)
        want, bound = layer_oracle.head_rope(rows[:, heads: heads + kv_heads], None, table, positions, 1e-6, False, False)
        oracle.check_cache(raw(k).cpu()[at], raw(ks).cpu()[at], want, bound - layer_oracle.STEP[torch.bfloat16] * want.abs(), "k")
        assert torch.equal(raw(v).cpu()[at], oracle.to_cache(rows[:, heads + kv_heads:])[0])
        offsets = torch.tensor([0] + counts).cumsum(0).int()
        kw = dict(softcap=cap, prefix_lens=prompts.int() if prompts is not None else None)
        a = ops().paged_attention(q, k, v, on(ids), on(offsets), on(torch.tensor(lens, dtype=torch.int32)), k_scales=ks, v_scales=vs, softcap=cap,
                                  prefix_lens=on(kw["prefix_lens"]) if prompts is not None else None, shared_prefix=shared)
        want, bound = oracle.attention(q.cpu(), raw(k).cpu(), raw(v).cpu(), ids, offsets, torch.tensor(lens), k_scales=raw(ks).cpu(), v_scales=raw(vs).cpu(), **kw)
        within(a, want, bound, "attention")
        y = ops().fp8_block_linear(a.view(t, heads * d), on(wo), on(wos))
        want, bound = layer_oracle.block_gemm(*layer_oracle.block_quant(a.cpu().view(t, heads * d)), wo, wos)
        within(y, want, bound, "output")


@pytest.mark.parametrize("batch,n", [(3, 1), (40, 1), (2, 70)])
def test_replayed_from_graphs(dev, batch, n):
    """Two graphs of the same calls with other eager work between their replays; lengths, slots and pages change in place."""
    from phyai_amd.runtime import HipGraph

    heads, kv_heads, d, page, hidden, shared = 8, 1, 128, 16, 512, 256
    w, ws = (t.to(dev) for t in layer_oracle.block_weight((heads + 2 * kv_heads) * d, hidden, gen(5)))
    table, norm = ops().rope_table(1024, d), (seeded((hidden,), 4, 0.2) + 1).to(dev)
    each = 40
    k, v, ks, vs = ops().fp8_cache(shared // page + batch * each, page, kv_heads, d, device=dev)
    first = torch.arange(shared // page, dtype=torch.int32)
    pages = torch.stack([torch.cat([first, shared // page + b * each + torch.randperm(each, generator=gen(b)).int()]) for b in range(batch)]).to(dev)
    raw(k).copy_(oracle.to_cache(seeded(tuple(k.shape), 7))[0])
    raw(v).copy_(oracle.to_cache(seeded(tuple(v.shape), 8))[0])
    raw(ks).fill_(120)
    raw(vs).fill_(119)
    offsets = (torch.arange(batch + 1) * n).int().to(dev)

    def step(x, residual, lens, positions, slots):
        codes, scale, total = ops().add_rmsnorm_fp8(x, residual, norm)
        qkv = ops().fp8_block_gemm(codes, scale, w, ws)
        q, _ = ops().qk_norm_rope(qkv, table, positions, heads, kv_heads, d, k_pages=k, v_pages=v, slots=slots, k_scales=ks, v_scales=vs)
        a = ops().paged_attention(q, k, v, pages, offsets, lens, k_scales=ks, v_scales=vs, softcap=30.0, shared_prefix=shared)
        return torch.cat([a.flatten(1).float(), total.float()], 1)

    def inputs(done, seed):
        spots = torch.cat([(pages[b].long()[:, None] * page + torch.arange(page, device=dev)).reshape(-1)[shared + done: shared + done + n] for b in range(batch)])
        return dict(x=seeded((batch * n, hidden), seed).to(dev), residual=seeded((batch * n, hidden), seed + 50).to(dev),
                    lens=torch.full((batch,), shared + done + n, dtype=torch.int32, device=dev),
                    positions=(torch.arange(shared + done, shared + done + n, device=dev)).repeat(batch), slots=spots.contiguous())

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
    split, kw = attend_case(([3, 2, 1], [900, 700, 800], 16, 8, 1, 256, True, None, None, 30.0), torch.bfloat16, 8, shared=640)
    many, kw_many = attend_case(([100, 90], [300, 200], 16, 8, 2, 64, True, None, [64, 0], None), torch.float16, 16)
    x, r, w = seeded((200, 512), 1).to(dev), seeded((200, 512), 2).to(dev), seeded((512,), 3).to(dev)

    def both():
        return [attend(dev, split, kw | dict(shared_prefix=640)), attend(dev, many, kw_many), *ops().add_rmsnorm_fp8(x, r, w)]

    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(both())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(raw(a) if a.itemsize == 1 else a, raw(b) if b.itemsize == 1 else b) for a, b in zip(got, want))


def test_a_norm_module_feeds_both_kinds_of_layer(L, dev):
    from phyai_amd.norm import GemmaRMSNorm

    norm = GemmaRMSNorm(256, device=dev)
    norm.weight.data.copy_(seeded((256,), 1, 0.3))
    x, residual = seeded((2, 9, 256), 2).to(dev), seeded((2, 9, 256), 3).to(dev)
    for per_block in (False, True):
        spec = L.Fp8Spec(granularity=L.Granularity.BLOCK, block_shape=(128, 128)) if per_block else L.Fp8Spec(granularity=L.Granularity.PER_CHANNEL)
        layer = L.ReplicatedLinear(256, 384, bias=False, params_dtype=torch.bfloat16, spec=spec, device=dev)
        if per_block:
            weight, scale = layer_oracle.block_weight(384, 256, gen(4))
            layer.weight.data.copy_(weight.to(dev))
            layer.weight_scale.data.copy_(scale.to(dev))
        else:
            spec.quantize_weight_(layer, seeded((384, 256), 5, 0.05).to(dev))
        view, total = norm.forward_add_fp8(x, residual, per_block=per_block)
        want, n = oracle.add_norm(x.cpu().view(18, 256), residual.cpu().view(18, 256), norm.weight.cpu(), norm.variance_epsilon, True)
        assert torch.equal(total.cpu().view(18, 256), want)
        oracle.check_norm_codes(view.x.view(18, 256), view.x_scale.view(18, -1), n, per_block)
        y, _ = layer(view)
        assert y.shape == (2, 9, 384)
        if per_block:
            want, bound = layer_oracle.block_gemm(view.x.cpu().view(18, 256), view.x_scale.cpu().view(18, 2), weight, scale)
            within(y.view(18, 384), want, bound)
        else:
            assert torch.equal(y, ops().fp8_gemm(view.x, view.x_scale, layer.weight, layer.weight_scale))


@pytest.mark.parametrize("fp8,softcap,samples", [(True, None, 1), (False, 10.0, 1), (True, None, 5), (False, None, 3), (True, 10.0, 40)])
def test_prefix_attention_with_a_cache_in_8_bits_and_with_samples(dev, fp8, softcap, samples):
    from phyai_amd.runtime import PagedPrefixAttention

    chunk, prefix, heads, kv_heads, d, page = 6, 48, 4, 2, 64, 16
    a = PagedPrefixAttention(2, chunk, prefix, heads, d, kv_heads, device=dev, page_size=page, fp8=fp8, softcap=softcap, samples=samples)
    width = (heads + 2 * kv_heads) * d
    table = ops().rope_table(prefix + chunk, d, device="cpu")
    for layer in (0, 1):
        before, fused = seeded((prefix, width), 1 + layer), seeded((samples * chunk, width), 5 + layer)
        first = a.prefill(before.to(dev), layer)
        out = a(fused.to(dev), layer)
        caches = [p.cpu() if p.itemsize > 1 else raw(p).cpu() for p in (a.k_pages[layer], a.v_pages[layer])]
        scales = [raw(s).cpu() for s in (a.k_scales[layer], a.v_scales[layer])] if fp8 else [None, None]
        # keys: what the cache holds is what was written there (values bit for bit)
        rows = fused.view(samples, chunk, -1, d)
        for b in range(samples):
            spots = (a.page_table[b].cpu().long()[:, None] * page + torch.arange(page)).reshape(-1)[prefix: prefix + chunk]
            at = (spots // page, spots % page)
            value = rows[b][:, heads + kv_heads:]
            assert torch.equal(caches[1][at], oracle.to_cache(value)[0] if fp8 else value)
        q, _ = ops().qk_norm_rope(fused.to(dev), table.to(dev), torch.arange(prefix, prefix + chunk, device=dev).repeat(samples), heads, kv_heads, d)
        offsets, lens = (torch.arange(samples + 1) * chunk).int(), torch.full((samples,), prefix + chunk, dtype=torch.int32)
        want, bound = oracle.attention(q.cpu(), *caches, a.page_table.cpu(), offsets, lens, causal=False, softcap=softcap, k_scales=scales[0], v_scales=scales[1])
        within(out.view(-1, heads, d), want, bound, "chunks")
        q, _ = ops().qk_norm_rope(before.to(dev), table.to(dev), torch.arange(prefix, device=dev), heads, kv_heads, d)
        want, bound = oracle.attention(q.cpu(), *caches, a.page_table[:1].cpu(), torch.tensor([0, prefix]), torch.tensor([prefix]), causal=False, softcap=softcap,
                                       k_scales=scales[0], v_scales=scales[1])
        within(first.view(-1, heads, d), want, bound, "prefix")


def test_the_same_call_gives_the_same_bits(dev):
    for case, shared in ((([1] * 30, [700 + i for i in range(30)], 16, 8, 2, 128, True, None, None, None), 640), (([90, 70], [500, 400], 16, 8, 2, 128, True, None, [100, 50], 20.0), 0)):
        for bits in (8, 16):
            tensors, kw = attend_case(case, torch.bfloat16, bits, shared=shared)
            want = attend(dev, tensors, kw | dict(shared_prefix=shared))
            assert all(torch.equal(attend(dev, tensors, kw | dict(shared_prefix=shared)), want) for _ in range(5))


def test_refused_calls(dev):
    x, w = seeded((4, 64), 1).to(dev), seeded((64,), 2).to(dev)
    add = ops().add_rmsnorm_fp8
    for bad in (dict(residual=x[:2]), dict(residual=x.float()), dict(residual=x.cpu()), dict(weight=w[:32]), dict(weight=w.float()), dict(out=x.float()),
                dict(out=torch.empty(4, 72, dtype=x.dtype, device=dev)[:, :64]), dict(x=x.cpu()), dict(x=x.half())):
        with pytest.raises(RuntimeError):
            add(**(dict(x=x, residual=x, weight=w) | bad))
    wide = torch.zeros(8, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="overlaps"):
        add(wide[:4], wide[4:], w, out=wide[1:5])
    k, v, ks, vs = ops().fp8_cache(4, 8, 2, 64, device=dev)
    qkv, cs, pos, slots = seeded((3, 6 * 64), 1).to(dev), ops().rope_table(16, 64), torch.arange(3, device=dev), torch.arange(3, device=dev)
    rope = dict(k_pages=k, v_pages=v, slots=slots, k_scales=ks, v_scales=vs)
    ops().qk_norm_rope(qkv, cs, pos, 2, 2, 64, **rope)
    bf = torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16, device=dev)
    for bad in (dict(k_scales=None), dict(v_scales=None), dict(k_pages=bf, v_pages=bf), dict(k_scales=ks.float()), dict(k_scales=ks[:2]), dict(slots=None),
                dict(k_pages=None, v_pages=None), dict(k_scales=raw(ks)[:, :1].expand(4, 8, 2)), dict(k_scales=None, v_scales=None)):
        with pytest.raises(RuntimeError):
            ops().qk_norm_rope(qkv, cs, pos, 2, 2, 64, **(rope | bad))
    odd = ops().fp8_cache(4, 8, 2, 72, device=dev)
    with pytest.raises(RuntimeError, match="16"):
        ops().qk_norm_rope(seeded((3, 6 * 72), 1).to(dev), cs, pos, 2, 2, 72, k_pages=odd[0], v_pages=odd[1], slots=slots, k_scales=odd[2], v_scales=odd[3])
    for bad in (dict(dtype=torch.float32), dict(slots=slots.int()), dict(slots=slots.cpu()), dict(k_pages=bf), dict(v_scales=None), dict(k_scales=ks[1:])):
        with pytest.raises(RuntimeError):
            ops().read_fp8_cache(**(dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs, slots=slots) | bad))
    q, table = seeded((2, 4, 64), 1).to(dev), torch.zeros(2, 3, dtype=torch.int32, device=dev)
    offsets, lens = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev), torch.tensor([5, 6], dtype=torch.int32, device=dev)
    good = dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs)
    ops().paged_attention(q, page_table=table, q_offsets=offsets, kv_lens=lens, **good)
    for bad in (dict(k_scales=None), dict(k_scales=None, v_scales=None), dict(k_pages=bf, v_pages=bf), dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=1e-60), dict(softcap=1e39),
                dict(softcap=float("inf")), dict(shared_prefix=-1), dict(prefix_lens=lens.long()), dict(prefix_lens=lens[:1]), dict(prefix_lens=lens.cpu()),
                dict(k_scales=raw(ks).contiguous())):
        with pytest.raises(RuntimeError):
            ops().paged_attention(q, page_table=table, q_offsets=offsets, kv_lens=lens, **(good | bad))
