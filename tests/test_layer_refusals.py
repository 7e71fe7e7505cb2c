"""Calls around attention that are refused on the host: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest

EINVAL, EWORKSPACE = -1, -3   # phyai_fp8.h


@pytest.mark.parametrize("scale,code", [(2.0 ** 127, EWORKSPACE), (2.35e38, EWORKSPACE), (2.37e38, EINVAL), (3.4e38, EINVAL)])
def test_attention_refuses_a_scale_that_overflows_in_base_two(scale, code):
    """Scores are taken to base 2: a scale times log2(e) beyond fp32 would turn a score of 0 into NaN.  (What is not refused for its
    scale is refused here for its missing workspace, before anything is launched.)"""
    from phyai_amd import _lib

    lib = _lib.load()
    raw = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(raw) + 255) // 256 * 256
    strides = (ctypes.c_int64 * 3)(16 * 64, 64, 64)
    assert lib.phyai_layer_paged_attention_workspace_bytes(1, 1, 1, 1, 64, 4096) > 0
    rc = lib.phyai_layer_paged_attention(p, 64, 64, p, p, strides, 256, 16, p, 256, 256, p, p, p, 1, 1, 1, 1, 64, scale, 1, 0, 0, None, 0, None)
    assert rc == code, lib.phyai_layer_last_error()
    if code == EINVAL:
        assert b"scale" in lib.phyai_layer_last_error()
