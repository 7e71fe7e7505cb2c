"""Attention of action chunks over a paged cache that holds their prefix.

The part of the reference's attention back end that the expert loop needs (a paged KV pool, its page
table, and the plan of a run over it): the prefix of every sequence goes into
pages once per layer (:meth:`PagedPrefixAttention.prefill`), then each denoise step writes the chunk's
keys and values behind it and attends over both.  Two kernels a call: ``ops.qk_norm_rope`` rotates the
fused projection's query and key heads and writes keys and values where they belong,
``ops.paged_attention`` reads them.  Page table, positions and lengths are made once, so a call is the
same launches every time and can be recorded into a graph.
"""

from __future__ import annotations

from typing import Sequence

import torch

from phyai_amd import ops


class PagedPrefixAttention:
    """``attend(fused_qkv, layer_index) -> [batch * chunk, heads * head_dim]`` for the expert's layers.

    ``prefix_len``: tokens of the prefix, one number or one per sequence.  The rows of ``fused_qkv`` are the sequences one
    after another, ``chunk`` tokens each, at positions ``prefix_len`` onwards; each sees its prefix and the whole chunk.
    ``norms``: per layer ``(q_weight, k_weight)`` of RMSNorms on the heads, if the model has them.  Keys are stored rotated.

    ``fp8``: the cache holds e4m3 codes with a power of two for each token and head (``ops.fp8_cache``), half the bytes.  ``softcap``: scores
    become ``softcap * tanh(score / softcap)``.  ``samples``: so many chunks start from one prefix (``prefix_len`` is one number, whole pages
    long): its keys and values are there once, :meth:`prefill` takes its tokens once, and a call reads them once for all chunks where that is
    the faster way.
    """

    def __init__(self, n_layers: int, chunk: int, prefix_len: int | Sequence[int], num_heads: int = 8, head_dim: int = 256,
                 num_kv_heads: int = 1, *, device, dtype: torch.dtype = torch.bfloat16, page_size: int = 16, rope_base: float = 10000.0,
                 norms: Sequence[tuple[torch.Tensor, torch.Tensor]] | None = None, eps: float = 1e-6, fp8: bool = False,
                 softcap: float | None = None, samples: int = 1) -> None:
        lens = [int(prefix_len)] if isinstance(prefix_len, int) else [int(n) for n in prefix_len]
        if samples < 1 or (samples > 1 and (len(lens) != 1 or lens[0] % page_size)):
            raise ValueError(f"PagedPrefixAttention: {samples} samples of one prefix need one prefix length that is a multiple of page_size="
                             f"{page_size}, got prefix_len={prefix_len}")
        if n_layers <= 0 or chunk <= 0 or page_size <= 0 or not lens or min(lens) < 0:
            raise ValueError(f"PagedPrefixAttention needs layers, a chunk, pages of some size and prefix lengths of at least 0, got "
                             f"n_layers={n_layers}, chunk={chunk}, page_size={page_size}, prefix_len={prefix_len}")
        if norms is not None and len(norms) != n_layers:
            raise ValueError(f"norms has {len(norms)} entries for {n_layers} layers")
        self.n_layers, self.chunk, self.prefix_lens, self.page_size = n_layers, chunk, tuple(lens), page_size
        self.heads, self.kv_heads, self.hd, self.norms, self.eps = num_heads, num_kv_heads, head_dim, norms, eps
        self.fp8, self.softcap, self.samples = fp8, softcap, samples
        # page table: each sequence's pages one after another, behind those of the prefix that samples share
        shared = lens[0] // page_size if samples > 1 else 0
        rows = lens * samples
        need = [-(-(n + chunk) // page_size) - shared for n in rows]
        first = [shared + sum(need[:b]) for b in range(len(need))]
        table = torch.full((len(rows), shared + max(need)), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :shared] = torch.arange(shared)
            table[b, shared: shared + n] = torch.arange(first[b], first[b] + n)
        self.page_table = table.to(device)
        self._shared = shared * page_size
        pages = shared + sum(need)
        if fp8:
            pools = [ops.fp8_cache(pages, page_size, num_kv_heads, head_dim, device=device) for _ in range(n_layers)]
            self.k_pages, self.v_pages, self.k_scales, self.v_scales = (list(x) for x in zip(*pools))
        else:
            pool = (pages, page_size, num_kv_heads, head_dim)
            self.k_pages = [torch.zeros(pool, dtype=dtype, device=device) for _ in range(n_layers)]
            self.v_pages = [torch.zeros(pool, dtype=dtype, device=device) for _ in range(n_layers)]
            self.k_scales = self.v_scales = [None] * n_layers
        self.cos_sin = ops.rope_table(max(lens) + chunk, head_dim, rope_base, device=device)
        # (slots count from a sequence's first page as if it lay in front of its own ones, which is so without samples)
        self._prefix = self._tokens([0] if samples > 1 else first, [0] * len(lens), lens, device)
        self._chunk = self._tokens([f - shared for f in first], rows, [chunk] * len(rows), device)

    def _tokens(self, first: list[int], start: list[int], count: list[int], device):
        """What a run over ``count[b]`` tokens of every sequence from ``start[b]`` on needs: positions, slots, offsets, lengths."""
        spans = [torch.arange(s, s + n, dtype=torch.int64) for s, n in zip(start, count)]
        slots = [p + f * self.page_size for p, f in zip(spans, first)]
        offsets = torch.tensor([sum(count[:b]) for b in range(len(count) + 1)], dtype=torch.int32)
        lens = torch.tensor([s + n for s, n in zip(start, count)], dtype=torch.int32)
        return tuple(t.to(device) for t in (torch.cat(spans), torch.cat(slots), offsets, lens))

    def _attend(self, fused: torch.Tensor, index: int, tokens) -> torch.Tensor:
        positions, slots, offsets, lens = tokens
        q_weight, k_weight = self.norms[index] if self.norms is not None else (None, None)
        k_pages, v_pages = self.k_pages[index], self.v_pages[index]
        scales = dict(k_scales=self.k_scales[index], v_scales=self.v_scales[index])
        q, _ = ops.qk_norm_rope(fused, self.cos_sin, positions, self.heads, self.kv_heads, self.hd, q_weight=q_weight, k_weight=k_weight,
                                eps=self.eps, k_pages=k_pages, v_pages=v_pages, slots=slots, **scales)
        several = tokens is self._chunk and self.samples > 1
        table = self.page_table if several or self.samples == 1 else self.page_table[:1]
        return ops.paged_attention(q, k_pages, v_pages, table, offsets, lens, causal=False, softcap=self.softcap,
                                   shared_prefix=self._shared if several else 0, **scales).view(-1, self.heads * self.hd)

    def prefill(self, fused: torch.Tensor, index: int) -> torch.Tensor:
        """The prefix tokens of all sequences (one after another) into layer ``index``'s pages; their attention over each
        other, which the prefix's own layers go on with."""
        return self._attend(fused, index, self._prefix)

    def __call__(self, fused: torch.Tensor, index: int) -> torch.Tensor:
        return self._attend(fused, index, self._chunk)


__all__ = ["PagedPrefixAttention"]
