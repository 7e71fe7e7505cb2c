"""Block-scaled linears whose output lies in the buffer of their input."""

from __future__ import annotations

import pytest
import torch

import layer_oracle as oracle
from conftest import seeded

pytestmark = pytest.mark.gpu


def ops():
    from phyai_amd import ops as o

    return o


@pytest.mark.parametrize("m", [1, 7, 300])
def test_a_linear_beside_its_input_in_one_buffer(dev, m):
    """Output columns of the rows that hold the input: no overlap, whatever the kernel."""
    w, ws = (t.to(dev) for t in oracle.block_weight(256, 256, torch.Generator().manual_seed(1)))
    x = seeded((m, 256), 2)
    want = ops().fp8_block_linear(x.to(dev), w, ws)
    both = torch.cat([x, torch.zeros(m, 256, dtype=torch.bfloat16)], dim=1).to(dev)
    from phyai_amd import _lib

    lib = _lib.load()
    need = lib.phyai_layer_block_linear_workspace_bytes(m, 256, 256)
    work = torch.zeros(max(need, 1), dtype=torch.uint8, device=dev)
    rc = lib.phyai_layer_block_linear(both.data_ptr(), 512, w.data_ptr(), ws.data_ptr(), None, both.data_ptr() + 512, 512, m, 256, 256,
                                      work.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(both[:, 256:], want) and torch.equal(both[:, :256].cpu(), x)
    small = ops().fp8_block_linear(x[:5].to(dev), w, ws)
    rows = x[:5].to(dev)
    with pytest.raises(RuntimeError):
        ops().fp8_block_linear(rows, w, ws, out=rows)
    assert torch.equal(rows.cpu(), x[:5]) and small.shape == rows.shape
