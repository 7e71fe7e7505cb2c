"""Calls of the operators around a cache in 8 bits that are refused on the host, before anything is launched: no GPU needed."""

from __future__ import annotations

import ctypes

import pytest

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3   # phyai_fp8.h


@pytest.fixture(scope="module")
def lib():
    from phyai_amd import _lib

    return _lib.load()


def buffer(n=65536):
    raw = (ctypes.c_char * (n + 256))()
    return raw, (ctypes.addressof(raw) + 255) // 256 * 256


def three(*values):
    return (ctypes.c_int64 * 3)(*values)


def refuses(call, kinds):
    for code, cases in kinds.items():
        for over in cases:
            assert call(**over) == code, over


def test_add_rmsnorm_quant(lib):
    raw, p = buffer()
    good = dict(x=p, ldx=64, res=p + 4096, ldr=64, w=p, gemma=0, eps=1e-6, M=4, D=64, total=p + 8192, ldt=64, xq=p + 16384, xs=p + 32768, row=1, block=1)

    def call(**over):
        return lib.phyai_layer_add_rmsnorm_quant(*(good | over).values(), None)

    assert call(M=0, x=None, res=None, w=None, total=None, xq=None, xs=None) == 0
    refuses(call, {EINVAL: [dict(x=None), dict(res=None), dict(w=None), dict(total=None), dict(xq=None), dict(xs=None), dict(x=p + 8), dict(res=p + 8),
                            dict(w=p + 8), dict(total=p + 8), dict(xq=p + 4), dict(xs=p + 2), dict(ldx=56), dict(ldr=56), dict(ldt=56), dict(ldx=68),
                            dict(ldr=68), dict(ldt=68), dict(row=0), dict(row=-1), dict(block=-1), dict(M=-1), dict(D=0),
                            # a total that is an input in part, codes in an input or in the total
                            dict(total=p + 16), dict(total=p + 4096 + 128), dict(total=p, ldt=72), dict(xq=p), dict(xq=p + 4096), dict(xq=p + 8192)],
                   EUNSUPPORTED: [dict(D=60, ldx=64), dict(M=2 ** 31), dict(D=2 ** 29, ldx=2 ** 29, ldr=2 ** 29, ldt=2 ** 29)]})
    assert b"overlaps" in lib.phyai_layer_last_error() or lib.phyai_layer_last_error()


def test_calls_of_more_threads_than_a_launch_has(lib):
    raw, p = buffer()
    norm = [p, 64, p + 4096, 64, p, 0, 1e-6, 2 ** 26, 64, p + 8192, 64, p + 16384, p + 32768, 1, 1, None]
    assert lib.phyai_layer_add_rmsnorm_quant(*norm) == EUNSUPPORTED
    norm[7], norm[8] = 2 ** 22, 8192
    norm[1] = norm[3] = norm[10] = 8192
    assert lib.phyai_layer_add_rmsnorm_quant(*norm) == EUNSUPPORTED
    s, b = three(64, 64, 64), three(4, 1, 1)
    assert lib.phyai_layer_cache_read(p, p, s, s, p, p, b, b, p, 4, 4, p, p, 2 ** 26, 1, 512, 0, None) == EUNSUPPORTED


def test_a_workspace_is_that_of_the_window_that_a_call_takes(lib):
    need = lib.phyai_layer_paged_attention_more_workspace_bytes
    for window in (2 ** 31, 2 ** 40, 2 ** 63 - 1):
        for width in (400, 2 ** 30):
            assert need(4, 2, 1, 1, 64, 16, width, 0, window) == need(4, 2, 1, 1, 64, 16, width, 0, 2 ** 31 - 1) > 0


def test_head_rope_fp8(lib):
    raw, p = buffer()
    s, b = three(64, 64, 64), three(4, 1, 1)
    good = dict(qkv=p, ld=192, qw=None, kw=None, cs=p, rows=10, pos=p, q=p, kp=p, vp=p, ks=s, vs=s, ksc=p, vsc=p, kss=b, vss=b, slots=p, pages=4, page=4,
                T=4, H=1, KV=1, D=64, rot=64, eps=1e-6, gemma=0, inter=0, type=0)

    def call(**over):
        return lib.phyai_layer_head_rope_fp8(*(good | over).values(), None)

    assert call(T=0, qkv=None, pos=None, q=None) == 0
    refuses(call, {EINVAL: [dict(qkv=None), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(ksc=None), dict(vsc=None), dict(kss=None),
                            dict(vss=None), dict(slots=None), dict(page=0), dict(pages=-1), dict(kp=p + 8), dict(ks=three(64, 72, 64)),
                            dict(vs=three(-64, 64, 64)), dict(kss=three(4, -1, 1)), dict(vss=three(-4, 1, 1)), dict(type=2), dict(T=-1)],
                   EUNSUPPORTED: [dict(D=72, ld=216), dict(D=60, rot=56), dict(pages=2 ** 16, page=2 ** 15)]})


def test_cache_read(lib):
    raw, p = buffer()
    s, b = three(64, 64, 64), three(4, 1, 1)
    good = dict(kp=p, vp=p, ks=s, vs=s, ksc=p, vsc=p, kss=b, vss=b, slots=p, pages=4, page=4, k=p, v=p, T=4, KV=1, D=64, type=0)

    def call(**over):
        return lib.phyai_layer_cache_read(*(good | over).values(), None)

    assert call(T=0, kp=None, vp=None, slots=None, k=None, v=None) == 0
    refuses(call, {EINVAL: [dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(ksc=None), dict(vsc=None), dict(kss=None), dict(vss=None),
                            dict(slots=None), dict(k=None), dict(v=None), dict(kp=p + 8), dict(vp=p + 8), dict(k=p + 8), dict(v=p + 8), dict(slots=p + 4),
                            dict(ks=three(64, 8, 64)), dict(vs=three(64, 64, -16)), dict(kss=three(-1, 1, 1)), dict(page=0), dict(pages=-1), dict(T=-1),
                            dict(KV=0), dict(D=0), dict(type=2), dict(KV=65536)],
                   EUNSUPPORTED: [dict(D=72), dict(D=528), dict(T=2 ** 31), dict(pages=2 ** 16, page=2 ** 15), dict(T=2 ** 30, KV=2)]})


def test_paged_attention_more(lib):
    from phyai_amd._lib import AttentionOptions

    raw, p = buffer()
    strides = three(16 * 64, 64, 64)
    good = dict(q=p, qt=64, qh=64, k=p, v=p, s=strides, pages=8, page=16, table=p, ts=400, width=400, off=p, lens=p, out=p, T=4, B=2, H=1, KV=1, D=64,
                scale=0.125, causal=1, window=0, type=0)

    def call(options=True, more=None, **over):
        o = AttentionOptions(**(dict(k_scales=p, v_scales=p, scale_strides=three(16, 1, 1)) | (more or {})))
        return lib.phyai_layer_paged_attention_more(*(good | over).values(), ctypes.byref(o) if options else None, None, 0, None)

    need = lib.phyai_layer_paged_attention_more_workspace_bytes
    assert need(4, 2, 1, 1, 64, 16, 400, 0, 0) > 0
    assert need(4, 2, 1, 1, 64, 16, 400, 15, 0) == need(4, 2, 1, 1, 64, 16, 400, 0, 0) and need(40, 40, 1, 1, 64, 16, 400, 3200, 0) > 0
    assert need(4, 2, 1, 1, 64, 0, 400, 16, 0) == 0 == need(0, 2, 1, 1, 64, 16, 400, 16, 0)
    assert call() == EWORKSPACE                       # (nothing else to be refused)
    assert call(T=0, q=None, out=None) == 0
    # (2 scale log2(e) / softcap is 3.6e37 here, a number of fp32, and 3.6e38 below, none)
    assert call(more=dict(softcap=1e-38)) == EWORKSPACE
    nan = float("nan")
    refuses(lambda **over: call(**over), {EINVAL: [
        dict(options=False), dict(more=dict(k_scales=None)), dict(more=dict(v_scales=None)), dict(more=dict(scale_strides=three(16, -1, 1))),
        dict(more=dict(softcap=-1.0)), dict(more=dict(softcap=nan)), dict(more=dict(softcap=3e38)), dict(more=dict(softcap=1e-39)), dict(more=dict(shared_prefix=-1)),
        dict(more=dict(prefix_lens=p + 2)), dict(s=three(16 * 64, 72, 64)), dict(k=None), dict(k=p + 8), dict(scale=0.0), dict(H=3, KV=2)],
        EUNSUPPORTED: [dict(D=72), dict(D=272)]})


def test_a_window_of_options_reaches_the_structure():
    """The structure in Python lies like the one in C: 8-byte pointers and numbers, the cap last."""
    from phyai_amd._lib import AttentionOptions

    offsets = [getattr(AttentionOptions, n).offset for n, _ in AttentionOptions._fields_]
    assert offsets == [0, 8, 16, 40, 48, 56] and ctypes.sizeof(AttentionOptions) == 64
