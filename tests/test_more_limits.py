"""Host logic of the operators around a cache in 8 bits that decides about a launch: no GPU needed, and with one there is nothing to see
here (the buffers are the host's)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from phyai_amd import _lib

ELAUNCH = -4   # phyai_fp8.h: all checks are passed, and there is no device


def norm_call(lib, **over):
    raw = (ctypes.c_char * 65792)()
    p = (ctypes.addressof(raw) + 255) // 256 * 256
    at = dict(x=p, ldx=64, res=p + 4096, ldr=64, w=p + 61440, gemma=0, eps=1e-6, M=4, D=64, total=p + 8192, ldt=64, xq=p + 16384, xs=p + 32768, row=1, block=1)
    for name, value in over.items():
        at[name] = value if name not in ("total", "xq") else p + value
    return lib.phyai_layer_add_rmsnorm_quant(*at.values(), None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would be launched on the host's memory")
@pytest.mark.parametrize("value", ["0", "", "x", "-3", "9", "1", "4"])
def test_a_forced_number_of_chunks_is_one_that_there_is(monkeypatch, value):
    """Anything but 1 to 4 is no number of chunks a thread: zero of them was a division by zero."""
    monkeypatch.setenv("PHYAI_LAYER_ADD_NORM", value)
    assert norm_call(_lib.load()) == ELAUNCH


@pytest.mark.skipif(torch.cuda.is_available(), reason="would be launched on the host's memory")
@pytest.mark.parametrize("strides", [dict(ldx=72), dict(ldt=72), dict(ldr=72, ldx=80)])
def test_one_row_in_place_has_no_stride(strides):
    """A total in the place of x: strides that differ mean different rows, but for one row nothing."""
    lib = _lib.load()
    raw = (ctypes.c_char * 65792)()
    p = (ctypes.addressof(raw) + 255) // 256 * 256
    at = dict(ldx=64, ldr=64, ldt=64) | strides

    def call(M):
        return lib.phyai_layer_add_rmsnorm_quant(p, at["ldx"], p + 4096, at["ldr"], p + 61440, 0, 1e-6, M, 64, p, at["ldt"], p + 16384, p + 32768, 1, 1, None)

    assert call(1) == ELAUNCH
    if at["ldx"] != at["ldt"]:
        assert call(2) == -1 and b"total overlaps" in lib.phyai_layer_last_error()


@pytest.mark.parametrize("over,what", [(dict(total=16), b"total overlaps an input"), (dict(total=4096 + 128), b"total overlaps an input"),
                                       (dict(total=0, ldt=72), b"total overlaps an input"), (dict(xq=0), b"xq overlaps an input"),
                                       (dict(xq=4096), b"xq overlaps an input"), (dict(xq=8192), b"xq overlaps total")])
def test_overlaps_are_what_is_refused(over, what):
    lib = _lib.load()
    assert norm_call(lib, **over) == -1 and what in lib.phyai_layer_last_error(), lib.phyai_layer_last_error()
