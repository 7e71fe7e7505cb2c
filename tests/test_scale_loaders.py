"""Checkpoint scales of fused layers whose spec keeps them as columns: one per row, and one per leg."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from phyai_amd.linear import Fp8Spec, QKVParallelLinear


class ColumnScales(Fp8Spec):
    """Scales as ``[rows, 1]`` (one per output row) or ``[legs, 1]`` (one per fused matrix), as some checkpoints keep them."""

    per_leg = False

    def allocate(self, layer, request):
        super().allocate(layer, request)
        n = len(request.logical_widths) if self.per_leg else request.weight_shape[0]
        layer.weight_scale = nn.Parameter(torch.ones(n, 1), requires_grad=False)


class LegScales(ColumnScales):
    per_leg = True


class Model(nn.Module):
    def __init__(self, spec):
        super().__init__()
        self.qkv = QKVParallelLinear(64, 32, 4, 2, bias=False, params_dtype=torch.bfloat16, spec=spec, prefix="l.qkv_proj")


def load(tmp_path, spec, scale_of):
    from safetensors.torch import save_file

    from phyai_amd.weights import load_pretrained

    model = Model(spec)
    widths = dict(zip("qkv", (128, 64, 64)))
    held = {}
    for i, (leg, n) in enumerate(widths.items()):
        held[f"l.{leg}_proj.weight"] = torch.full((n, 64), float(i)).to(torch.float8_e4m3fn)
        held[f"l.{leg}_proj.weight_scale"] = scale_of(i, n)
    save_file(held, str(tmp_path / "model.safetensors"))
    report = load_pretrained(model, tmp_path)
    assert not report.missing and not report.unexpected
    return model.qkv.weight_scale, widths


@pytest.mark.parametrize("scalar", [False, True])
def test_a_scale_per_row_as_a_column(tmp_path, scalar):
    def scale_of(i, n):
        return torch.tensor(i + 1.0) if scalar else torch.arange(n, dtype=torch.float32)[:, None] + 1000 * i

    got, widths = load(tmp_path, ColumnScales(), scale_of)
    want = torch.cat([scale_of(i, n).expand(n, 1) for i, n in enumerate(widths.values())])
    assert torch.equal(got, want)


def test_a_scale_per_leg_as_a_column(tmp_path):
    got, _ = load(tmp_path, LegScales(), lambda i, n: torch.tensor([i + 0.5]))
    assert got.flatten().tolist() == [0.5, 1.5, 2.5]
