"""Operators for serving over a key / value cache in 8 bits, and for batches that share a prefix, at sizes from the smallest
call to the largest, for timing them and for checking them against plain forms.

A case is a dict of plain values.  ``listed()`` names the standing ones, ``draw(rng)`` gives one more of the same
ranges, ``prepare(case, seed)`` builds what a program holds before the call, ``run(state)`` makes one pass - through
the package's entry points where ``own`` is set, else in plain tensor operations - ``work(case)`` counts the bytes and
operations that pass cannot do without and ``exact(case, seed)`` computes the same in 64 bits.

Kinds of case:

``norm``    the residual's addition, the root-mean-square norm of the sum and its quantization to fp8 with a scale per 128
            elements or per row
``cache``   norms of the query and key heads of a fused projection, the position rotation, the write of keys and values into
            a paged cache in 8 bits with a power of two per token and head, and the reading back of what was written
``attend``  attention of each sequence's new tokens over its pages, in 16 or 8 bits, with scores capped by a tanh and a mask
            that shows a causal row the whole of its prompt
``shared``  attention of a batch whose sequences begin with the same pages
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
MAX_NORM = 13056 * 2048                      # elements of the largest listed norm
MAX_CACHE_WRITE = 13056 * 10 * 256           # elements of the largest listed projection
MAX_ATTEND = 4.0 * 2048 * 8192 * 32 * 128    # flops of the largest listed attention, masks not counted
MAX_KEYS = 64 * 8704 * 8 * 128               # elements of the keys of the largest listed batch, shared ones counted for every sequence


def listed() -> list[dict]:
    return [
        # One decoded token in front of the backbone's projections: all latency.
        dict(name="norm_m1", kind="norm", m=1, d=2048, per_block=True, gemma=True),
        # An odd number of rows of a width that ends inside a block of 128, one scale a row.
        dict(name="norm_ragged_m777", kind="norm", m=777, d=4304, per_block=False, gemma=False),
        # Prefill of 16 samples.
        dict(name="norm_m13056", kind="norm", m=13056, d=2048, per_block=True, gemma=True),
        # One decoded token's heads into the cache and back: two launches.
        dict(name="cache_m1", kind="cache", t=1, heads=8, kv_heads=1, d=256, rot=256, interleaved=False, norm=True, gemma=False,
             page=16, dtype="bfloat16"),
        # Prefill of 16 samples.
        dict(name="cache_m13056", kind="cache", t=13056, heads=8, kv_heads=1, d=256, rot=256, interleaved=False, norm=True, gemma=False,
             page=16, dtype="bfloat16"),
        # The action chunk over its prefix and itself, every token sees every other: called in each layer of each Euler step.
        dict(name="attend_chunk_m50", kind="attend", batch=1, q=50, kv=866, heads=8, kv_heads=1, d=256, causal=False, window=0, prefix=0,
             cap=0.0, bits=8, page=16, dtype="bfloat16"),
        # A serving batch that decodes one token each over caches of different lengths, in half the bytes.
        dict(name="attend_decode_b64", kind="attend", batch=64, q=1, kv=8192, heads=32, kv_heads=8, d=128, causal=True, window=0, prefix=0,
             cap=0.0, bits=8, page=64, dtype="bfloat16"),
        # Prefill of image and text: the images' tokens see each other, the text is causal behind them, scores are capped.
        dict(name="attend_prefix_b16", kind="attend", batch=16, q=816, kv=816, heads=8, kv_heads=1, d=256, causal=True, window=0, prefix=768,
             cap=50.0, bits=16, page=16, dtype="bfloat16"),
        # A chunk of a long prompt behind what the cache holds of it: the most arithmetic.
        dict(name="attend_chunk_m2048", kind="attend", batch=1, q=2048, kv=8192, heads=32, kv_heads=8, d=128, causal=True, window=0, prefix=0,
             cap=50.0, bits=8, page=64, dtype="bfloat16"),
        # A few requests decode behind one observation's prefix, in half precision: a small call.
        dict(name="shared_b5", kind="shared", batch=5, q=1, shared=816, kv=866, heads=8, kv_heads=1, d=256, causal=True, cap=0.0, bits=16, page=16,
             dtype="float16"),
        # Sixteen samples of an action chunk from one observation, all rows of a sample see all of it.
        dict(name="shared_chunk_b16", kind="shared", batch=16, q=50, shared=816, kv=866, heads=8, kv_heads=1, d=256, causal=False, cap=0.0, bits=8,
             page=16, dtype="bfloat16"),
        # A serving batch behind one long system prompt.
        dict(name="shared_decode_b64", kind="shared", batch=64, q=1, shared=8192, kv=8704, heads=32, kv_heads=8, d=128, causal=True, cap=0.0, bits=16,
             page=64, dtype="bfloat16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "cache", "attend", "attend", "attend", "shared", "shared"])
    if kind == "norm":
        step = 128 if rng.random() < 0.6 else 8
        d = max(step, round(_log_int(rng, 128, 16384) / step) * step)
        m = max(1, min(_log_int(rng, 1, 13056), MAX_NORM // d))
        return dict(kind=kind, m=m, d=d, per_block=rng.random() < 0.6, gemma=rng.random() < 0.5)
    kv_heads = rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    page = rng.choice([1, 16, 16, 24, 64, 256])
    if kind == "cache":
        d = rng.choice([64, 80, 96, 128, 128, 256, 256])
        rot = d if rng.random() < 0.7 else {64: 32, 80: 48, 96: 64, 128: 64, 256: 128}[d]
        t = max(1, min(_log_int(rng, 1, 13056), MAX_CACHE_WRITE // ((heads + 2 * kv_heads) * d)))
        return dict(kind=kind, t=t, heads=heads, kv_heads=kv_heads, d=d, rot=rot, interleaved=rng.random() < 0.3, norm=rng.random() < 0.8,
                    gemma=rng.random() < 0.4, page=page, dtype=dtype)
    d = rng.choice([64, 80, 128, 128, 256, 256])
    bits = rng.choice([8, 8, 16])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    if kind == "shared":
        batch, shared = _log_int(rng, 2, 256), _log_int(rng, 256, 16384)
        q = 1 if rng.random() < 0.6 else _log_int(rng, 2, 64)
        kv = shared + q + _log_int(rng, 1, 1024)
        limit = min(MAX_KEYS // (batch * kv_heads * d), int(MAX_ATTEND / (4.0 * batch * q * heads * d)))
        kv = max(q + 2, min(kv, limit))
        shared = min(shared, kv - q)
        return dict(kind=kind, batch=batch, q=q, shared=shared, kv=kv, heads=heads, kv_heads=kv_heads, d=d, causal=rng.random() < 0.7, cap=cap,
                    bits=bits, page=page, dtype=dtype)
    if rng.random() < 0.5:
        batch, q, kv = _log_int(rng, 1, 256), 1, _log_int(rng, 1, 32768)
    else:
        batch, q = _log_int(rng, 1, 16), _log_int(rng, 2, 2048)
        kv = q + (_log_int(rng, 1, 8192) if rng.random() < 0.67 else 0)
    kv = max(q, min(kv, MAX_KEYS // (batch * kv_heads * d), int(MAX_ATTEND / (4.0 * batch * q * heads * d))))
    q = max(1, min(q, int(MAX_ATTEND / (4.0 * batch * kv * heads * d))))
    causal = rng.random() < 0.75
    return dict(kind=kind, batch=batch, q=q, kv=kv, heads=heads, kv_heads=kv_heads, d=d, causal=causal,
                window=_log_int(rng, 16, 4096) if rng.random() < 0.2 else 0, prefix=rng.randint(1, kv) if causal and rng.random() < 0.5 else 0,
                cap=cap, bits=bits, page=page, dtype=dtype)


# ---- building what a program holds ---------------------------------------------------------------------------

def _lengths(case: dict) -> tuple[list[int], list[int], list[int]]:
    """New tokens, cached keys (the new ones among them) and prompt of each sequence: the first has the case's, the others
    from a quarter of them upward.  Behind a shared prefix the keys of a sequence's own are counted so."""
    shared = case.get("shared", 0)
    rng = random.Random(case["batch"] * 1000003 + case["kv"])
    qs, kvs, prompts = [case["q"]], [case["kv"]], [case.get("prefix", 0)]
    for _ in range(case["batch"] - 1):
        rest = case["kv"] - shared
        kv = shared + rng.randint(max(1, rest // 4), rest)
        kvs.append(kv)
        qs.append(min(kv - shared, rng.randint(max(1, case["q"] // 4), case["q"])))
        prompts.append(min(kv, rng.randint(case.get("prefix", 0) // 4, case.get("prefix", 0))))
    return qs, kvs, prompts


class _Maker:
    def __init__(self, seed: int) -> None:
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(device=self.dev).manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.bfloat16, scale: float = 1.0):
        return (torch.randn(*shape, generator=self.gen, device=self.dev) * scale).to(dtype)

    def permutation(self, n: int):
        return torch.randperm(n, generator=self.gen, device=self.dev)


def _to_8_bits(x):
    """Codes of x[..., head_dim] (e4m3fn) and the bytes of a power of two per head: the smallest with which nothing leaves the
    type's range (byte b stands for 2 ** (b - 127))."""
    most = x.abs().amax(-1)
    part, exponent = torch.frexp(most)
    byte = (torch.where(part <= E4M3_MAX / 512.0, exponent - 9, exponent - 8) + 127).clamp(1, 254).to(torch.int32)
    byte = torch.where(most > 0, byte, torch.ones_like(byte))
    return torch.ldexp(x, (127 - byte)[..., None]).to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _powers(byte, dtype=torch.float32):
    return (byte.view(torch.uint8).to(torch.int32) << 23).view(torch.float32).to(dtype)


def _eight_bit_pages(make: _Maker, pages: int, page: int, kv_heads: int, d: int):
    """A cache of normal values in 8 bits, filled piece by piece; scales of a page lie head by head."""
    codes = torch.empty(pages, page, kv_heads, d, dtype=torch.float8_e4m3fn, device=make.dev)
    scales = torch.empty(pages, kv_heads, page, dtype=torch.uint8, device=make.dev).transpose(1, 2)
    step = max(1, (1 << 26) // (page * kv_heads * d))
    for first in range(0, pages, step):
        c, s = _to_8_bits(make.normal(min(step, pages - first), page, kv_heads, d, dtype=torch.float32))
        codes[first: first + step], scales[first: first + step] = c, s
    return codes, scales.view(torch.float8_e8m0fnu)


def prepare(case: dict, seed: int) -> dict:
    make = _Maker(seed)
    state = dict(case)
    if case["kind"] == "norm":
        m, d = case["m"], case["d"]
        x, residual = make.normal(m, d), make.normal(m, d, scale=4.0)
        residual[:, make.permutation(d)[: max(1, d // 100)]] *= 20.0     # the outlier channels of a residual stream
        state |= dict(x=x, residual=residual, weight=make.normal(d, scale=0.3) + (0.0 if case["gemma"] else 1.0))
        return state
    dtype = getattr(torch, case["dtype"])
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    if case["kind"] == "cache":
        t, rot = case["t"], case["rot"]
        inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=make.dev) / rot)
        angle = torch.arange(2 * t + 64, dtype=torch.float64, device=make.dev)[:, None] * inv
        pages = -(-t // page) + 2
        state |= dict(qkv=make.normal(t, (heads + 2 * kv_heads) * d, dtype=dtype),
                      cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous(),
                      positions=(torch.arange(t, device=make.dev) + int(seed) % 64),
                      q_weight=make.normal(d, dtype=dtype, scale=0.3) + (0.0 if case["gemma"] else 1.0) if case["norm"] else None,
                      k_weight=make.normal(d, dtype=dtype, scale=0.3) + (0.0 if case["gemma"] else 1.0) if case["norm"] else None,
                      # the tokens' pages in any order, inside a page one after another
                      slots=(make.permutation(pages)[:, None] * page + torch.arange(page, device=make.dev)).reshape(-1)[:t].contiguous())
        for name in ("k", "v"):
            state[name + "_pages"] = torch.zeros(pages, page, kv_heads, d, dtype=torch.float8_e4m3fn, device=make.dev)
            scales = torch.zeros(pages, kv_heads, page, dtype=torch.uint8, device=make.dev).transpose(1, 2)
            state[name + "_scales"] = scales.view(torch.float8_e8m0fnu)
        return state
    qs, kvs, prompts = _lengths(case)
    same = case.get("shared", 0) // page      # pages that every sequence begins with
    counts = torch.tensor([-(-kv // page) - same for kv in kvs], device=make.dev)
    per = same + int(counts.max())
    pages = same + int(counts.sum()) + 1
    order = make.permutation(pages).to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    at = torch.arange(per, device=make.dev)[None, :]
    index = torch.where(at < same, at, first[:, None] + at)
    table = torch.where(at - same < counts[:, None], order[index.clamp_max(pages - 1)], torch.zeros((), dtype=torch.int32, device=make.dev))
    offsets = [0]
    for q in qs:
        offsets.append(offsets[-1] + q)
    # (capped scores are large ones: the cap has to be felt)
    state |= dict(query=make.normal(offsets[-1], heads, d, dtype=dtype, scale=8.0 if case["cap"] else 2.0), page_table=table.contiguous(),
                  q_offsets=torch.tensor(offsets, dtype=torch.int32, device=make.dev), kv_lens=torch.tensor(kvs, dtype=torch.int32, device=make.dev),
                  prefix_lens=torch.tensor(prompts, dtype=torch.int32, device=make.dev) if case.get("prefix", 0) else None, max_q=max(qs),
                  k_scales=None, v_scales=None)
    for name in ("k", "v"):
        if case["bits"] == 8:
            state[name + "_pages"], state[name + "_scales"] = _eight_bit_pages(make, pages, page, kv_heads, d)
        else:
            state[name + "_pages"] = make.normal(pages, page, kv_heads, d, dtype=dtype)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------

def _plain_norm(s: dict):
    m, d = s["x"].shape
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    h = total.float()
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * (s["weight"].float() + (1.0 if s["gemma"] else 0.0))
    width = BLOCK if s["per_block"] else d
    groups = -(-d // width)
    n = torch.nn.functional.pad(n, (0, groups * width - d)).view(m, groups, width)
    # (a division by a number would be a product with its rounded reciprocal, which moves codes on a rounding border)
    scale = n.abs().amax(2).clamp_min(1e-12) / torch.full((), E4M3_MAX, device=n.device)
    codes = (n / scale[..., None]).to(torch.float8_e4m3fn).view(m, groups * width)[:, :d].contiguous()
    return [codes, scale, total]


def _plain_rotate(x, cos, sin, rot: int, interleaved: bool):
    """x [t, heads, d], cos and sin [t, 1, rot / 2]."""
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_cache(s: dict):
    t, heads, kv_heads, d, rot = s["t"], s["heads"], s["kv_heads"], s["d"], s["rot"]
    rows = s["qkv"].view(t, heads + 2 * kv_heads, d)
    q, k, v = rows[:, :heads].float(), rows[:, heads: heads + kv_heads].float(), rows[:, heads + kv_heads:].float()
    if s["norm"]:
        more = 1.0 if s["gemma"] else 0.0
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * (s["q_weight"].float() + more)
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * (s["k_weight"].float() + more)
    cos, sin = s["cos_sin"][s["positions"]][:, None, :].split(rot // 2, dim=-1)
    q, k = (_plain_rotate(x, cos, sin, rot, s["interleaved"]) for x in (q, k))
    page, place = s["slots"] // s["page"], s["slots"] % s["page"]
    back = []
    for x, name in ((k, "k"), (v, "v")):
        codes, byte = _to_8_bits(x)
        # (bytes of both: the copy kernels of 8-bit floats do not all exist)
        s[name + "_pages"].view(torch.uint8)[page, place] = codes.view(torch.uint8)
        s[name + "_scales"].view(torch.uint8)[page, place] = byte
        read = s[name + "_pages"].view(torch.uint8)[page, place].view(torch.float8_e4m3fn).float()
        back.append((read * _powers(s[name + "_scales"].view(torch.uint8)[page, place])[..., None]).to(rows.dtype))
    return [q.to(rows.dtype), *back]


def _plain_attend(s: dict):
    heads, kv_heads, d, batch, q_max = s["heads"], s["kv_heads"], s["d"], s["batch"], s["max_q"]
    q, dev = s["query"], s["query"].device
    begin, lens = s["q_offsets"][:-1].long(), s["kv_lens"].long()
    counts = s["q_offsets"][1:].long() - begin
    at = torch.arange(q_max, device=dev)
    rows = (begin[:, None] + at).clamp_max(q.shape[0] - 1)                                    # [batch, q_max]
    q = q[rows].float().view(batch, q_max, kv_heads, -1, d).permute(0, 2, 3, 1, 4)             # [batch, kv_heads, group, q_max, d]
    group = q.shape[2]

    def gathered(pages, scales):
        table = s["page_table"].long()
        if scales is None:
            x = pages[table].float()
        else:
            x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * _powers(scales.view(torch.uint8)[table])[..., None]
        return x.flatten(1, 2).permute(0, 2, 1, 3).contiguous()                               # [batch, kv_heads, keys, d]

    k = gathered(s["k_pages"], s["k_scales"])
    scores = q.reshape(batch, kv_heads, group * q_max, d) @ k.transpose(-1, -2).contiguous() * d ** -0.5
    keys = k.shape[2]
    del k
    if s["cap"]:
        scores = torch.tanh(scores / s["cap"]) * s["cap"]
    j = torch.arange(keys, device=dev)
    position = (lens - counts)[:, None] + at                                                  # [batch, q_max]
    seen = (j < lens[:, None])[:, None, :].expand(batch, q_max, -1)
    if s["causal"]:
        before = j <= position[..., None]
        if s.get("prefix"):
            before = before | (j < s["prefix_lens"].long()[:, None])[:, None, :]
        seen = seen & before
    if s.get("window"):
        seen = seen & (j > position[..., None] - s["window"])
    scores = scores.view(batch, kv_heads, group, q_max, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.exp(scores - top)
    del scores
    total = p.sum(-1, keepdim=True)
    o = (p.view(batch, kv_heads, group * q_max, -1) @ gathered(s["v_pages"], s["v_scales"])).view(batch, kv_heads, group, q_max, d) / total.clamp_min(1e-38)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * q_max, heads, d).to(s["query"].dtype)
    sequence = torch.searchsorted(s["q_offsets"].long(), torch.arange(s["query"].shape[0], device=dev), right=True) - 1
    return o[sequence * q_max + torch.arange(s["query"].shape[0], device=dev) - begin[sequence]]


def run(state: dict):
    s = state
    if own:
        from phyai_amd import ops

        if s["kind"] == "norm":
            return list(ops.add_rmsnorm_fp8(s["x"], s["residual"], s["weight"], 1e-6, gemma=s["gemma"], per_block=s["per_block"]))
        if s["kind"] == "cache":
            q, _ = ops.qk_norm_rope(s["qkv"], s["cos_sin"], s["positions"], s["heads"], s["kv_heads"], s["d"], q_weight=s["q_weight"],
                                    k_weight=s["k_weight"], eps=1e-6, gemma=s["gemma"], interleaved=s["interleaved"], k_pages=s["k_pages"],
                                    v_pages=s["v_pages"], slots=s["slots"], k_scales=s["k_scales"], v_scales=s["v_scales"])
            return [q, *ops.read_fp8_cache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["slots"], dtype=s["qkv"].dtype)]
        if s["kind"] == "shared":
            return ops.paged_attention(s["query"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"], causal=s["causal"],
                                       k_scales=s["k_scales"], v_scales=s["v_scales"], softcap=s["cap"] or None, shared_prefix=s["shared"])
        return ops.paged_attention(s["query"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"], causal=s["causal"],
                                   window=s["window"] or None, k_scales=s["k_scales"], v_scales=s["v_scales"], softcap=s["cap"] or None,
                                   prefix_lens=s["prefix_lens"])
    return {"norm": _plain_norm, "cache": _plain_cache, "attend": _plain_attend, "shared": _plain_attend}[s["kind"]](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def _span(case: dict, q: int, kv: int, prompt: int, i: int) -> tuple[int, int]:
    """The keys that new token i of a sequence sees, from and to."""
    position = kv - q + i
    last = min(kv, max(position + 1, prompt)) if case["causal"] else kv
    return (max(0, position - case["window"] + 1) if case.get("window") else 0), last


def work(case: dict) -> dict:
    if case["kind"] == "norm":
        m, d = case["m"], case["d"]
        scales = m * (-(-d // BLOCK) if case["per_block"] else 1)
        return {"bytes": 7.0 * m * d + 2.0 * d + 4.0 * scales, "flops": 8.0 * m * d}
    if case["kind"] == "cache":
        t, d = case["t"], case["d"]
        kept = 2 * t * case["kv_heads"]           # key and value heads: written in 8 bits, read, returned in 16
        return {"bytes": 2.0 * t * (case["heads"] + 2 * case["kv_heads"]) * d + 2.0 * t * case["heads"] * d + kept * (2.0 * (d + 1) + 2.0 * d)
                + t * (4.0 * case["rot"] + 16.0), "flops": 8.0 * t * (case["heads"] + case["kv_heads"]) * d}
    qs, kvs, prompts = _lengths(case)
    shared = case.get("shared", 0) // case["page"] * case["page"]
    keys, pairs = shared, 0
    for q, kv, prompt in zip(qs, kvs, prompts):
        spans = [_span(case, q, kv, prompt, i) for i in range(q)]
        pairs += sum(max(0, hi - lo) for lo, hi in spans)
        keys += max(0, max(hi for _, hi in spans) - max(shared, min(lo for lo, _ in spans)))
    per_key = 2.0 * case["kv_heads"] * (case["d"] + 1 if case["bits"] == 8 else 2 * case["d"])
    return {"bytes": 4.0 * sum(qs) * case["heads"] * case["d"] + keys * per_key + 4.0 * keys / case["page"],
            "flops": 4.0 * pairs * case["heads"] * case["d"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def _exact_8_bits(x):
    """What x[..., head_dim] stands for in the cache: multiples of a power of two that go by each value's own size."""
    most = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(most.clamp_min(1e-300) / E4M3_MAX)).clamp(-126, 127))
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-300))).clamp_min(-6) - 3)
    return torch.round(y / step) * step * unit       # (ties go to even)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = (s["x"].double() + s["residual"].double()).to(torch.bfloat16)
        n = h.double()
        n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + 1e-6) * (s["weight"].double() + (1.0 if case["gemma"] else 0.0))
        codes, scales = torch.empty_like(n), []
        width = BLOCK if case["per_block"] else case["d"]
        for first in range(0, case["d"], width):
            part = n[:, first: first + width]
            scale = part.abs().amax(1).clamp_min(1e-12) / E4M3_MAX
            codes[:, first: first + width] = (part / scale[:, None]).float().to(torch.float8_e4m3fn).double()
            scales.append(scale)
        return [codes, torch.stack(scales, 1), h.double()]
    if case["kind"] == "cache":
        t, heads, kv_heads, d, rot = (case[x] for x in ("t", "heads", "kv_heads", "d", "rot"))
        rows = s["qkv"].double().view(t, heads + 2 * kv_heads, d)
        parts = []
        for x, weight in ((rows[:, :heads], s["q_weight"]), (rows[:, heads: heads + kv_heads], s["k_weight"])):
            if weight is not None:
                x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (weight.double() + (1.0 if case["gemma"] else 0.0))
            c = torch.view_as_complex(torch.stack([s["cos_sin"][s["positions"], : rot // 2], s["cos_sin"][s["positions"], rot // 2:]], -1).double())
            first = torch.arange(rot // 2, device=x.device) * 2 if case["interleaved"] else torch.arange(rot // 2, device=x.device)
            second = first + (1 if case["interleaved"] else rot // 2)
            turned = torch.complex(x[..., first], x[..., second]) * c[:, None, :]
            x = x.clone()
            x[..., first], x[..., second] = turned.real, turned.imag
            parts.append(x)
        return [parts[0], _exact_8_bits(parts[1]), _exact_8_bits(rows[:, heads + kv_heads:])]
    qs, kvs, prompts = _lengths(case)
    out, begin = [], 0
    for b, (q, kv, prompt) in enumerate(zip(qs, kvs, prompts)):
        ids = s["page_table"][b, : -(-kv // case["page"])].long()
        both = []
        for name in ("k", "v"):
            x = s[name + "_pages"]
            if case["bits"] == 8:
                power = torch.exp2(s[name + "_scales"].view(torch.uint8)[ids].double() - 127.0)
                x = x.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * power[..., None]
            else:
                x = x[ids].double()
            both.append(x.reshape(-1, case["kv_heads"], case["d"])[:kv])
        k, v = both
        position = torch.arange(kv - q, kv, device=k.device)[:, None]
        j = torch.arange(kv, device=k.device)[None, :]
        hidden = torch.zeros(q, kv, dtype=torch.bool, device=k.device)
        if case["causal"]:
            hidden |= j > torch.clamp_min(position, prompt - 1)
        if case.get("window"):
            hidden |= j <= position - case["window"]
        o = torch.empty(q, case["heads"], case["d"], dtype=torch.float64, device=k.device)
        group = case["heads"] // case["kv_heads"]
        for h in range(case["heads"]):
            scores = (s["query"][begin: begin + q, h].double() @ k[:, h // group].t()) / math.sqrt(case["d"])
            if case["cap"]:
                scores = case["cap"] * torch.tanh(scores / case["cap"])
            o[:, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // group]
        out.append(o)
        begin += q
    return torch.cat(out)
