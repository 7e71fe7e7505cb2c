"""Calls around attention that are refused on the host: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

EINVAL, EWORKSPACE, ELAUNCH = -1, -3, -4   # phyai_fp8.h


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


@pytest.mark.parametrize("M,stride,at,N,refused", [
    (1, 512, 0, 128, True), (1, 512, 256, 128, False), (1, 512, -128, 128, False), (1, 512, -120, 128, True), (1, 512, 248, 128, True),
    (4, 512, 0, 128, True), (4, 512, 256, 128, False), (4, 512, 256, 256, False), (4, 512, 248, 128, True), (4, 512, 384, 128, False),
    (4, 512, -256, 256, False), (4, 512, -128, 128, False), (4, 512, -120, 128, True), (4, 512, 392, 128, True), (4, 512, 1536 + 256, 128, False),
    (4, 512, 512, 128, True), (4, 512, 2048, 128, False),
])
def test_few_rows_refuse_an_output_that_lies_in_their_input(M, stride, at, N, refused):
    """x: rows of 256 elements, `stride` apart; out: N elements from `at` on, in rows as far apart."""
    from phyai_amd import _lib

    if torch.cuda.is_available():
        pytest.skip("host memory: the calls that are not refused must not be launched")
    lib = _lib.load()
    raw = (ctypes.c_char * 65536)()
    p = (ctypes.addressof(raw) + 16384) // 256 * 256
    rc = lib.phyai_layer_block_linear(p, stride, p + 32768, p + 32768, None, p + 2 * at, stride, M, N, 256, None, 0, None)
    assert (rc == EINVAL and b"overlaps" in lib.phyai_layer_last_error()) if refused else rc == ELAUNCH, (rc, lib.phyai_layer_last_error())


def test_codes_refuse_an_output_that_lies_in_them():
    from phyai_amd import _lib

    lib = _lib.load()
    raw = (ctypes.c_char * 65536)()
    p = (ctypes.addressof(raw) + 16384) // 256 * 256
    for out in (p, p + 1024, p - 1024):
        assert lib.phyai_layer_block_gemm(p, p + 32768, 2, 1, p + 32768, p + 32768, None, out, 256, 8, 256, 256, None) == EINVAL
        assert b"overlaps" in lib.phyai_layer_last_error()
