"""The operators of a decoder layer's attention half, at sizes from the smallest call to the largest, for timing them
and for checking them against plain forms.

A case is a dict of plain values.  ``listed()`` names the standing ones, ``draw(rng)`` gives one more of the same
ranges, ``prepare(case, seed)`` builds what a program holds before the call, ``run(state)`` makes one pass - through
the package's entry points where ``own`` is set, else in plain tensor operations - ``work(case)`` counts the bytes and
operations that pass cannot do without and ``exact(case, seed)`` computes the same in 64 bits.

Kinds of case:

``linear``  the quantized linear whose weights have one scale per block of 128 x 128 and whose activations get one per
            128 elements of a token row
``rope``    norms of the query and key heads of a fused projection, the position rotation, and the write of keys and
            values into a paged cache
``attend``  attention of each sequence's new tokens over its pages, one token or a chunk
"""

from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 128
MAX_LINEAR = 2.0 * 13056 * 16384 * 2048      # flops of the largest listed linear
MAX_ROPE = 13056 * 10 * 256                  # elements of the largest listed projection
MAX_ATTEND = 4.0 * 2048 * 8192 * 32 * 128    # flops of the largest listed attention, masks not counted
MAX_CACHE = 64 * 8192 * 8 * 128              # elements of the keys of the largest listed cache, padding counted


def listed() -> list[dict]:
    return [
        # One token through the fused q | k | v projection of the action expert.
        dict(name="linear_m1", kind="linear", m=1, n=2560, k=1024, bias=False),
        # One chunk of 50 action tokens through the expert's down projection: the long K of a small call.
        dict(name="linear_m50", kind="linear", m=50, n=1024, k=4096, bias=False),
        # An odd number of tokens and widths that end inside a block of 128 on both axes, with a bias.
        dict(name="linear_ragged_m777", kind="linear", m=777, n=1168, k=4304, bias=True),
        # Prefill of one sample through the backbone's fused gate | up matrix.
        dict(name="linear_m816", kind="linear", m=816, n=32768, k=2048, bias=False),
        # The largest: the backbone's down projection for a batch of 16 samples.
        dict(name="linear_m13056", kind="linear", m=13056, n=2048, k=16384, bias=False),
        # One decoded token: the smallest call, all latency.
        dict(name="rope_m1", kind="rope", t=1, heads=8, kv_heads=1, d=256, rot=256, interleaved=False, norm=True, gemma=False,
             page=16, dtype="bfloat16"),
        # Heads of 72, two thirds of them rotated in neighbouring pairs, grouped keys, half precision.
        dict(name="rope_ragged_m777", kind="rope", t=777, heads=12, kv_heads=3, d=72, rot=48, interleaved=True, norm=True,
             gemma=True, page=16, dtype="float16"),
        # Prefill of 16 samples.
        dict(name="rope_m13056", kind="rope", t=13056, heads=8, kv_heads=1, d=256, rot=256, interleaved=False, norm=True,
             gemma=False, page=16, dtype="bfloat16"),
        # The action chunk over its prefix and itself, every token sees every other: called in each layer of each Euler step.
        dict(name="attend_chunk_m50", kind="attend", batch=1, q=50, kv=866, heads=8, kv_heads=1, d=256, causal=False, window=0,
             page=16, dtype="bfloat16"),
        # A serving batch that decodes one token each over caches of different lengths.
        dict(name="attend_decode_b64", kind="attend", batch=64, q=1, kv=8192, heads=32, kv_heads=8, d=128, causal=True, window=0,
             page=64, dtype="bfloat16"),
        # Prefill of a batch of prefixes of different lengths, bidirectional.
        dict(name="attend_prefix_b16", kind="attend", batch=16, q=816, kv=816, heads=8, kv_heads=1, d=256, causal=False, window=0,
             page=16, dtype="bfloat16"),
        # A chunk of a long prompt behind what the cache holds of it: the most arithmetic.
        dict(name="attend_chunk_m2048", kind="attend", batch=1, q=2048, kv=8192, heads=32, kv_heads=8, d=128, causal=True, window=0,
             page=64, dtype="bfloat16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo: int, hi: int) -> int:
    """A multiple of 16, spread over the logarithm; two of three are multiples of 128 as models have them."""
    step = 128 if rng.random() < 0.67 else 16
    return max(step, round(_log_int(rng, lo, hi) / step) * step)


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "rope", "attend", "attend", "attend"])
    if kind == "linear":
        case = dict(kind=kind, m=_log_int(rng, 1, 13056), n=_width(rng, 256, 32768), k=_width(rng, 256, 16384), bias=rng.random() < 0.5)
        case["m"] = max(1, min(case["m"], int(MAX_LINEAR / (2.0 * case["n"] * case["k"]))))
        return case
    kv_heads = rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    page = rng.choice([1, 16, 16, 24, 64, 256])
    if kind == "rope":
        d = rng.choice([64, 72, 96, 128, 128, 256, 256])
        rot = d if rng.random() < 0.7 else {64: 32, 72: 48, 96: 64, 128: 64, 256: 128}[d]
        t = _log_int(rng, 1, 13056)
        t = max(1, min(t, MAX_ROPE // ((heads + 2 * kv_heads) * d)))
        return dict(kind=kind, t=t, heads=heads, kv_heads=kv_heads, d=d, rot=rot, interleaved=rng.random() < 0.3, norm=rng.random() < 0.8,
                    gemma=rng.random() < 0.4, page=page, dtype=dtype)
    d = rng.choice([64, 80, 128, 128, 256, 256])
    if rng.random() < 0.5:
        batch, q, kv = _log_int(rng, 1, 256), 1, _log_int(rng, 1, 32768)
    else:
        batch, q = _log_int(rng, 1, 16), _log_int(rng, 2, 2048)
        kv = q + (_log_int(rng, 1, 8192) if rng.random() < 0.67 else 0)
    kv = max(q, min(kv, MAX_CACHE // (batch * kv_heads * d), int(MAX_ATTEND / (4.0 * batch * q * heads * d))))
    q = max(1, min(q, int(MAX_ATTEND / (4.0 * batch * kv * heads * d))))
    return dict(kind=kind, batch=batch, q=q, kv=kv, heads=heads, kv_heads=kv_heads, d=d, causal=rng.random() < 0.7,
                window=_log_int(rng, 16, 4096) if rng.random() < 0.25 else 0, page=page, dtype=dtype)


# ---- building what a program holds ---------------------------------------------------------------------------

def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and cached keys (the new ones among them) of each sequence: the first has the case's, the others from a
    quarter of them upward."""
    rng = random.Random(case["batch"] * 1000003 + case["kv"])
    qs, kvs = [case["q"]], [case["kv"]]
    for _ in range(case["batch"] - 1):
        kv = rng.randint(max(1, case["kv"] // 4), case["kv"])
        kvs.append(kv)
        qs.append(min(kv, rng.randint(max(1, case["q"] // 4), case["q"])))
    return qs, kvs


class _Maker:
    def __init__(self, seed: int) -> None:
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(device=self.dev).manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.bfloat16, scale: float = 1.0):
        return (torch.randn(*shape, generator=self.gen, device=self.dev) * scale).to(dtype)

    def permutation(self, n: int):
        return torch.randperm(n, generator=self.gen, device=self.dev)


def _blocks(rows: int, cols: int) -> tuple[int, int]:
    return -(-rows // BLOCK), -(-cols // BLOCK)


def prepare(case: dict, seed: int) -> dict:
    make = _Maker(seed)
    state = dict(case)
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = make.normal(m, k)
        x[:, make.permutation(k)[: max(1, k // 100)]] *= 20.0     # the outlier channels of real activations
        bn, bk = _blocks(n, k)
        w = torch.zeros(bn * BLOCK, bk * BLOCK, device=make.dev)
        w[:n, :k] = make.normal(n, k, dtype=torch.float32, scale=0.02)
        tiles = w.view(bn, BLOCK, bk, BLOCK)
        scale = tiles.abs().amax(dim=(1, 3)).clamp_min(1e-12) / 448.0
        codes = (tiles / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(bn * BLOCK, bk * BLOCK)[:n, :k].contiguous()
        state |= dict(x=x, weight=codes, weight_scale=scale.contiguous(), bias_t=make.normal(n, scale=0.1) if case["bias"] else None)
        return state
    dtype = getattr(torch, case["dtype"])
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    if case["kind"] == "rope":
        t, rot = case["t"], case["rot"]
        limit = 2 * t + 64
        inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=make.dev) / rot)
        angle = torch.arange(limit, dtype=torch.float64, device=make.dev)[:, None] * inv
        pages = -(-t // page) + 2
        state |= dict(qkv=make.normal(t, (heads + 2 * kv_heads) * d, dtype=dtype),
                      cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous(),
                      positions=(torch.arange(t, device=make.dev) + int(seed) % 64),
                      q_weight=make.normal(d, dtype=dtype, scale=0.3) + (0.0 if case["gemma"] else 1.0) if case["norm"] else None,
                      k_weight=make.normal(d, dtype=dtype, scale=0.3) + (0.0 if case["gemma"] else 1.0) if case["norm"] else None,
                      k_pages=torch.zeros(pages, page, kv_heads, d, dtype=dtype, device=make.dev),
                      v_pages=torch.zeros(pages, page, kv_heads, d, dtype=dtype, device=make.dev),
                      # the tokens' pages in any order, inside a page one after another
                      slots=(make.permutation(pages)[:, None] * page + torch.arange(page, device=make.dev)).reshape(-1)[:t].contiguous())
        return state
    qs, kvs = _lengths(case)
    per = max(-(-kv // page) for kv in kvs)
    counts = torch.tensor([-(-kv // page) for kv in kvs], device=make.dev)
    pages = int(sum(-(-kv // page) for kv in kvs)) + 1
    order = make.permutation(pages).to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    index = first[:, None] + torch.arange(per, device=make.dev)[None, :]
    table = torch.where(torch.arange(per, device=make.dev)[None, :] < counts[:, None], order[index.clamp_max(pages - 1)],
                        torch.zeros((), dtype=torch.int32, device=make.dev))
    offsets = [0]
    for q in qs:
        offsets.append(offsets[-1] + q)
    state |= dict(query=make.normal(offsets[-1], heads, d, dtype=dtype, scale=2.0), k_pages=make.normal(pages, page, kv_heads, d, dtype=dtype),
                  v_pages=make.normal(pages, page, kv_heads, d, dtype=dtype), page_table=table.contiguous(),
                  q_offsets=torch.tensor(offsets, dtype=torch.int32, device=make.dev),
                  kv_lens=torch.tensor(kvs, dtype=torch.int32, device=make.dev), max_q=max(qs))
    return state


# ---- one pass ------------------------------------------------------------------------------------------------

def _plain_linear(s: dict):
    (m, k), n = s["x"].shape, s["weight"].shape[0]
    bn, bk = _blocks(n, k)
    x = torch.nn.functional.pad(s["x"].float(), (0, bk * BLOCK - k)).view(m, bk, BLOCK)
    # (a division by a number would be a product with its rounded reciprocal, which moves codes on a rounding border)
    scale = x.abs().amax(dim=2, keepdim=True).clamp_min(1e-12) / torch.full((), 448.0, device=x.device)
    x = ((x / scale).to(torch.float8_e4m3fn).float() * scale).view(m, bk * BLOCK)[:, :k]
    w = s["weight"].float() * s["weight_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    return (y + s["bias_t"].float() if s["bias_t"] is not None else y).to(torch.bfloat16)


def _plain_rotate(x, cos, sin, rot: int, interleaved: bool):
    """x [t, heads, d], cos and sin [t, 1, rot / 2]."""
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_rope(s: dict):
    t, heads, kv_heads, d, rot = s["t"], s["heads"], s["kv_heads"], s["d"], s["rot"]
    rows = s["qkv"].view(t, heads + 2 * kv_heads, d)
    q, k, v = rows[:, :heads].float(), rows[:, heads: heads + kv_heads].float(), rows[:, heads + kv_heads:]
    if s["norm"]:
        more = 1.0 if s["gemma"] else 0.0
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * (s["q_weight"].float() + more)
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * (s["k_weight"].float() + more)
    cos, sin = s["cos_sin"][s["positions"]][:, None, :].split(rot // 2, dim=-1)
    q, k = (_plain_rotate(x, cos, sin, rot, s["interleaved"]).to(rows.dtype) for x in (q, k))
    s["k_pages"].view(-1, kv_heads, d)[s["slots"]] = k
    s["v_pages"].view(-1, kv_heads, d)[s["slots"]] = v
    return [q, s["k_pages"], s["v_pages"]]


def _plain_attend(s: dict):
    heads, kv_heads, d, batch, q_max = s["heads"], s["kv_heads"], s["d"], s["batch"], s["max_q"]
    q, dev = s["query"], s["query"].device
    begin, lens = s["q_offsets"][:-1].long(), s["kv_lens"].long()
    counts = s["q_offsets"][1:].long() - begin
    at = torch.arange(q_max, device=dev)
    rows = (begin[:, None] + at).clamp_max(q.shape[0] - 1)                                    # [batch, q_max]
    q = q[rows].float().view(batch, q_max, kv_heads, -1, d).permute(0, 2, 3, 1, 4)             # [batch, kv_heads, group, q_max, d]
    group = q.shape[2]
    k, v = (p[s["page_table"].long()].flatten(1, 2).float().permute(0, 2, 1, 3).contiguous() for p in (s["k_pages"], s["v_pages"]))
    scores = q.reshape(batch, kv_heads, group * q_max, d) @ k.transpose(-1, -2).contiguous() * d ** -0.5
    j = torch.arange(k.shape[2], device=dev)
    position = (lens - counts)[:, None] + at                                                  # [batch, q_max]
    seen = (j < lens[:, None])[:, None, :].expand(batch, q_max, -1)
    if s["causal"]:
        seen = seen & (j <= position[..., None])
    if s["window"]:
        seen = seen & (j > position[..., None] - s["window"])
    scores = scores.view(batch, kv_heads, group, q_max, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p.view(batch, kv_heads, group * q_max, -1) @ v).view(batch, kv_heads, group, q_max, d) / total.clamp_min(1e-38)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * q_max, heads, d).to(s["query"].dtype)
    sequence = torch.searchsorted(s["q_offsets"].long(), torch.arange(s["query"].shape[0], device=dev), right=True) - 1
    return o[sequence * q_max + torch.arange(s["query"].shape[0], device=dev) - begin[sequence]]


def run(state: dict):
    s = state
    if own:
        from phyai_amd import ops

        if s["kind"] == "linear":
            return ops.fp8_block_linear(s["x"], s["weight"], s["weight_scale"], s["bias_t"])
        if s["kind"] == "rope":
            q, _ = ops.qk_norm_rope(s["qkv"], s["cos_sin"], s["positions"], s["heads"], s["kv_heads"], s["d"], q_weight=s["q_weight"],
                                    k_weight=s["k_weight"], eps=1e-6, gemma=s["gemma"], interleaved=s["interleaved"],
                                    k_pages=s["k_pages"], v_pages=s["v_pages"], slots=s["slots"])
            return [q, s["k_pages"], s["v_pages"]]
        return ops.paged_attention(s["query"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"],
                                   causal=s["causal"], window=s["window"] or None)
    return {"linear": _plain_linear, "rope": _plain_rope, "attend": _plain_attend}[s["kind"]](s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def _seen(case: dict, q: int, kv: int) -> int:
    """(row, key) pairs of one sequence and head that no mask takes away."""
    if not case["causal"] and not case["window"]:
        return q * kv
    total = 0
    for i in range(q):
        position = kv - q + i
        last = min(kv, position + 1) if case["causal"] else kv
        total += max(0, last - (max(0, position - case["window"] + 1) if case["window"] else 0))
    return total


def work(case: dict) -> dict:
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        bn, bk = _blocks(n, k)
        return {"bytes": 2.0 * m * k + n * k + 4.0 * bn * bk + 2.0 * m * n + (2.0 * n if case["bias"] else 0.0), "flops": 2.0 * m * n * k}
    if case["kind"] == "rope":
        elements = case["t"] * (case["heads"] + 2 * case["kv_heads"]) * case["d"]
        turned = case["t"] * (case["heads"] + case["kv_heads"]) * case["d"]
        return {"bytes": 4.0 * elements + case["t"] * (4.0 * case["rot"] + 16.0), "flops": 8.0 * turned}
    qs, kvs = _lengths(case)
    keys = 0
    for q, kv in zip(qs, kvs):     # a window keeps the oldest keys out of every row's sight
        keys += min(kv, q - 1 + case["window"]) if case["window"] else kv
    pairs = sum(_seen(case, q, kv) for q, kv in zip(qs, kvs))
    return {"bytes": 4.0 * sum(qs) * case["heads"] * case["d"] + 4.0 * keys * case["kv_heads"] * case["d"] + 4.0 * keys / case["page"],
            "flops": 4.0 * pairs * case["heads"] * case["d"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device=s["x"].device)
        w = s["weight"].float().double()
        for g in range(-(-k // BLOCK)):
            part = slice(g * BLOCK, min(k, (g + 1) * BLOCK))
            x = s["x"][:, part].double()
            scale = (x.abs().amax(1).clamp_min(1e-12) / torch.full((), 448.0, dtype=torch.float64, device=x.device)).float().double()  # a 32-bit number
            codes = (x / scale[:, None]).float().to(torch.float8_e4m3fn).double()
            columns = s["weight_scale"][:, g].double().repeat_interleave(BLOCK)[:n]
            y += (codes @ w[:, part].t()) * scale[:, None] * columns[None, :]
        return y if s["bias_t"] is None else y + s["bias_t"].double()
    if case["kind"] == "rope":
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
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        k_pages.view(-1, kv_heads, d)[s["slots"]] = parts[1]
        v_pages.view(-1, kv_heads, d)[s["slots"]] = rows[:, heads + kv_heads:]
        return [parts[0], k_pages, v_pages]
    qs, kvs = _lengths(case)
    out, begin = [], 0
    for b, (q, kv) in enumerate(zip(qs, kvs)):
        ids = s["page_table"][b, : -(-kv // case["page"])].long()
        k, v = (p[ids].reshape(-1, case["kv_heads"], case["d"])[:kv].double() for p in (s["k_pages"], s["v_pages"]))
        position = torch.arange(kv - q, kv, device=k.device)[:, None]
        j = torch.arange(kv, device=k.device)[None, :]
        hidden = torch.zeros(q, kv, dtype=torch.bool, device=k.device)
        if case["causal"]:
            hidden |= j > position
        if case["window"]:
            hidden |= j <= position - case["window"]
        o = torch.empty(q, case["heads"], case["d"], dtype=torch.float64, device=k.device)
        group = case["heads"] // case["kv_heads"]
        for h in range(case["heads"]):
            scores = (s["query"][begin: begin + q, h].double() @ k[:, h // group].t()) / math.sqrt(case["d"])
            o[:, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // group]
        out.append(o)
        begin += q
    return torch.cat(out)
