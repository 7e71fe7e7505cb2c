"""Forms of the operators around a cache in 8 bits that only large calls or forced choices reach, against plain forms in 64 bits: chunks a
thread of the residual's norm, groups of two heads, the ends of the powers' range."""

from __future__ import annotations

import pytest
import torch

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
