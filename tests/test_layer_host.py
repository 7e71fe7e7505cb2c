"""The second C interface (include/phyai_layer.h), block-scaled layers and their checkpoints: what needs no GPU."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch
from torch import nn

from conftest import seeded

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "phyai_layer.h")
EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3


def declared():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(phyai_layer_[a-z0-9_]+)\s*\(", text)))


@pytest.fixture(scope="module")
def lib():
    from phyai_amd import _lib

    return _lib.load()


def test_every_declared_entry_point_is_exported_and_described(lib):
    from phyai_amd import _lib

    assert sorted(_lib.LAYER_SIGNATURES) == declared()
    assert all(hasattr(lib, name) for name in declared())
    version = int(re.search(r"#define PHYAI_LAYER_ABI_VERSION (\d+)", open(HEADER).read()).group(1))
    assert lib.phyai_layer_abi_version() == version == _lib.LAYER_ABI_VERSION


def buffer(n=4096):
    raw = (ctypes.c_char * (n + 256))()
    return raw, (ctypes.addressof(raw) + 255) // 256 * 256


# ---- refusals, all before anything is launched -----------------------------------------------------------------------

def test_block_linear_refuses_on_the_host(lib):
    raw, p = buffer()
    good = dict(x=p, ldx=256, w=p, ws=p, bias=None, out=p, ldo=64, M=300, N=64, K=256, work=None, size=0)

    def call(**kw):
        a = good | kw
        return lib.phyai_layer_block_linear(a["x"], a["ldx"], a["w"], a["ws"], a["bias"], a["out"], a["ldo"], a["M"], a["N"], a["K"], a["work"],
                                            a["size"], None)

    assert call(M=0, x=None, w=None, ws=None, out=None) == 0
    for kw in (dict(x=None), dict(w=None), dict(ws=None), dict(out=None), dict(x=p + 8), dict(w=p + 8), dict(out=p + 4), dict(bias=p + 1),
               dict(ldx=248), dict(ldx=260), dict(ldo=60), dict(ldo=66), dict(M=-1), dict(N=0), dict(K=0)):
        assert call(**kw) == EINVAL, kw
    for kw in (dict(N=56), dict(K=248), dict(K=250), dict(M=2 ** 31), dict(M=2 ** 23, K=512, ldx=512), dict(N=2 ** 31, ldo=2 ** 31), dict(M=1, N=2 ** 24, K=256, ldo=2 ** 24)):
        assert call(**kw) == EUNSUPPORTED, kw
    large = dict(M=2000, N=2560, K=1024, ldx=1024, ldo=2560)   # (few rows need none)
    need = lib.phyai_layer_block_linear_workspace_bytes(2000, 2560, 1024)
    assert need >= 2000 * 1024 + 2000 * 8 * 4
    for kw in (dict(), dict(work=p, size=need - 1), dict(work=p + 64, size=need)):
        assert call(**large, **kw) == EWORKSPACE, kw
    assert b"workspace" in lib.phyai_layer_last_error()
    assert lib.phyai_layer_block_linear_workspace_bytes(1, 1024, 4096) == 0 == lib.phyai_layer_block_linear_workspace_bytes(-1, 64, 64)


def test_block_quant_and_gemm_refuse_on_the_host(lib):
    raw, p = buffer()
    quant, gemm = lib.phyai_layer_block_quant, lib.phyai_layer_block_gemm
    assert quant(None, 64, 0, 64, None, None, 1, 1, None) == 0
    for a in ((None, 64, 4, 64, p, p, 1, 1), (p + 8, 64, 4, 64, p, p, 1, 1), (p, 64, 4, 64, None, p, 1, 1), (p, 64, 4, 64, p + 4, p, 1, 1),
              (p, 64, 4, 64, p, p + 2, 1, 1), (p, 64, 4, 64, p, p, 0, 1), (p, 64, 4, 64, p, p, 1, -1), (p, 56, 4, 64, p, p, 1, 1), (p, 64, -4, 64, p, p, 1, 1)):
        assert quant(*a, None) == EINVAL, a
    assert quant(p, 64, 4, 60, p, p, 1, 1, None) == EUNSUPPORTED
    assert quant(p, 1 << 20, 1 << 20, 1 << 20, p, p, 1, 1, None) == EUNSUPPORTED
    assert gemm(None, None, 1, 1, None, None, None, None, 64, 0, 64, 64, None) == 0
    for a in ((None, p, 1, 1), (p, None, 1, 1), (p + 8, p, 1, 1), (p, p + 2, 1, 1)):
        assert gemm(*a, p, p, None, p, 64, 4, 64, 64, None) == EINVAL, a
    for strides in ((-1, 1), (1, -1), (1 << 31, 0), (1 << 28, 0)):
        assert gemm(p, p, *strides, p, p, None, p, 64, 4, 64, 64, None) == EUNSUPPORTED, strides


def test_head_rope_refuses_on_the_host(lib):
    raw, p = buffer()
    s3 = (ctypes.c_int64 * 3)(64, 64, 64)
    good = dict(qkv=p, ld=192, qw=None, kw=None, cs=p, rows=10, pos=p, q=p, k=p, kp=None, vp=None, ks=None, vs=None, slots=None, pages=0, page=0,
                T=4, H=1, KV=1, D=64, rot=64, eps=1e-6, gemma=0, inter=0, type=0)

    def call(**over):
        a = good | over
        return lib.phyai_layer_head_rope(*a.values(), None)

    assert call(T=0, qkv=None, pos=None, q=None) == 0
    for over in (dict(qkv=None), dict(cs=None), dict(pos=None), dict(q=None), dict(rows=0), dict(ld=184), dict(ld=196), dict(qkv=p + 8), dict(pos=p + 4),
                 dict(q=p + 8), dict(k=p + 8), dict(qw=p), dict(kw=p), dict(qw=p + 8, kw=p), dict(T=-1), dict(H=0), dict(KV=0), dict(D=0), dict(rot=72),
                 dict(rot=-8), dict(type=2), dict(H=65536), dict(k=None), dict(k=None, kp=p, vp=p, ks=s3, vs=s3, slots=None, pages=4, page=4),
                 dict(k=None, kp=p, vp=p, ks=s3, vs=None, slots=p, pages=4, page=4), dict(k=None, kp=p, vp=p, ks=s3, vs=s3, slots=p, pages=4, page=0),
                 dict(k=None, kp=p + 8, vp=p, ks=s3, vs=s3, slots=p, pages=4, page=4),
                 dict(k=None, kp=p, vp=p, ks=(ctypes.c_int64 * 3)(64, 60, 64), vs=s3, slots=p, pages=4, page=4),
                 dict(k=None, kp=p, vp=p, ks=s3, vs=(ctypes.c_int64 * 3)(64, -64, 64), slots=p, pages=4, page=4)):
        assert call(**over) == EINVAL, over
    for over in (dict(D=60, rot=56), dict(rot=60), dict(D=520, ld=1560), dict(k=None, kp=p, vp=p, ks=s3, vs=s3, slots=p, pages=2 ** 16, page=2 ** 15)):
        assert call(**over) == EUNSUPPORTED, over


def test_paged_attention_refuses_on_the_host(lib):
    raw, p = buffer()
    strides = (ctypes.c_int64 * 3)(16 * 64, 64, 64)
    good = dict(q=p, qt=64, qh=64, k=p, v=p, s=strides, pages=8, page=16, table=p, ts=4, width=4, off=p, lens=p, out=p, T=4, B=2, H=1, KV=1, D=64,
                scale=0.125, causal=1, window=0, type=0, work=None, size=0)

    def call(**over):
        a = good | over
        return lib.phyai_layer_paged_attention(*a.values(), None)

    assert call(T=0, q=None, out=None) == 0 and call(B=0, q=None) == 0
    for over in (dict(q=None), dict(out=None), dict(off=None), dict(lens=None), dict(k=None), dict(v=None), dict(s=None), dict(table=None), dict(q=p + 8),
                 dict(out=p + 8), dict(k=p + 8), dict(table=p + 2), dict(off=p + 2), dict(lens=p + 1), dict(qt=60), dict(qh=-8),
                 dict(s=(ctypes.c_int64 * 3)(1024, 60, 64)), dict(H=3, KV=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                 dict(scale=float("inf")), dict(window=-1), dict(type=5), dict(ts=3), dict(T=-1), dict(B=-1), dict(H=0), dict(KV=0), dict(D=0), dict(page=0),
                 dict(pages=-1), dict(width=-1)):
        assert call(**over) == EINVAL, over
    for over in (dict(D=60), dict(D=264), dict(T=2 ** 30), dict(B=2 ** 30), dict(page=2 ** 20, width=2 ** 10, ts=2 ** 10), dict(KV=65536, H=65536),
                 dict(s=(ctypes.c_int64 * 3)(1024, 2 ** 28, 64))):
        assert call(**over) == EUNSUPPORTED, over
    # few rows over long sequences are split, and the parts want a workspace
    need = lib.phyai_layer_paged_attention_workspace_bytes(4, 2, 1, 1, 64, 2 ** 16)
    assert need > 0
    long = dict(page=256, width=256, ts=256)
    for over in (dict(), dict(work=p, size=need - 1), dict(work=p + 16, size=need)):
        assert call(**long, **over) == EWORKSPACE, over
    size = lib.phyai_layer_paged_attention_workspace_bytes
    assert size(0, 2, 1, 1, 64, 100) == 0 == size(4, 2, 3, 2, 64, 2 ** 16) and size(4096, 1, 8, 8, 128, 8192) == 0


# ---- layers, dispatch, checkpoints ---------------------------------------------------------------------------------

def block_spec():
    from phyai_amd.quant import Fp8Spec, Granularity

    return Fp8Spec(granularity=Granularity.BLOCK, block_shape=(128, 128))


def test_block_linears_go_to_their_own_kernel(monkeypatch):
    import phyai_amd.linear as L
    from phyai_amd.linear import KernelProbe
    from phyai_amd.quant import Fp8Spec, Granularity
    from phyai_amd.state import Mode, NoBackendError

    assert "hip_fp8_block" in [cls.name for cls, _ in L.list_registered_linear_kernels()]
    kernel = L.HipFp8BlockKernel()

    def probe(spec="fp8_block_128_128", N=256, K=256, sm=95, mode=Mode.EAGER, dtype=torch.bfloat16):
        return KernelProbe(spec_id=spec, M_bucket=4, N=N, K=K, in_dtype=dtype, out_dtype=torch.bfloat16, sm=sm, mode=mode)

    assert kernel.supports_capture() and kernel.can_handle(probe()) and kernel.can_handle(probe(mode=Mode.GRAPH_CAPTURING))
    for bad in (probe("fp8_per_channel"), probe("bf16"), probe("fp8_block_64_64"), probe(sm=0), probe(sm=80), probe(N=24), probe(K=24), probe(dtype=torch.float16)):
        assert not kernel.can_handle(bad)
    d = L.init(validate=False)
    monkeypatch.setattr(d, "_sm", 95)
    for M in (1, 50, 13056):
        assert d.select(spec_id="fp8_block_128_128", M=M, N=2560, K=1024, in_dtype=torch.bfloat16, out_dtype=torch.bfloat16).name == "hip_fp8_block"
    with pytest.raises(NoBackendError, match="fp8_block_64_64"):
        d.select(spec_id="fp8_block_64_64", M=4, N=256, K=256, in_dtype=torch.bfloat16, out_dtype=torch.bfloat16)
    layer = L.ReplicatedLinear(256, 128, bias=False, params_dtype=torch.bfloat16, spec=Fp8Spec(granularity=Granularity.BLOCK, block_shape=(128, 128)),
                               device="cpu")
    assert layer.weight_scale.shape == (1, 2) and not layer.supports_fused_epilogue(torch.zeros(1, 256, dtype=torch.bfloat16))
    wrong = nn.Module()
    wrong.spec = Fp8Spec()
    with pytest.raises(RuntimeError, match="fp8_per_channel"):
        kernel.apply(wrong, torch.zeros(1, 256, dtype=torch.bfloat16), None)
    wrong.spec = block_spec()
    with pytest.raises(RuntimeError, match="per token"):
        kernel.apply(wrong, L.ActivationView(torch.zeros(1, 256), torch.ones(1), Granularity.PER_TENSOR), None)
    L._reset_for_test()


class Block(nn.Module):
    def __init__(self, widths=(256, 256), heads=2, kv=1, hd=128):
        super().__init__()
        from phyai_amd.linear import MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear

        kw = dict(params_dtype=torch.bfloat16, device="cpu", bias=False)
        self.qkv_proj = QKVParallelLinear(256, hd, heads, kv, prefix="l.self_attn.qkv_proj", spec=block_spec(), **kw)
        self.gate_up_proj = MergedColumnParallelLinear(256, list(widths), prefix="l.mlp.gate_up_proj", spec=block_spec(), **kw)
        self.down_proj = RowParallelLinear(256, 256, prefix="l.mlp.down_proj", spec=block_spec(), **kw)


SHAPES = {"l.self_attn.q_proj": 256, "l.self_attn.k_proj": 128, "l.self_attn.v_proj": 128, "l.mlp.gate_proj": 256, "l.mlp.up_proj": 256, "l.mlp.down_proj": 256}


def checkpoint(scale_name, shapes=SHAPES):
    out = {}
    for i, (name, n) in enumerate(shapes.items()):
        out[f"{name}.weight"] = (seeded((n, 256), i).float() * 50).to(torch.float8_e4m3fn)
        out[f"{name}.{scale_name}"] = torch.rand(-(-n // 128), 2, generator=torch.Generator().manual_seed(i)) + 0.5
    return out


@pytest.mark.parametrize("scale_name", ["weight_scale", "weight_scale_inv"])
def test_loader_puts_block_scales_of_fused_layers_where_their_rows_are(tmp_path, scale_name):
    from safetensors.torch import save_file

    from phyai_amd.weights import load_pretrained

    held = checkpoint(scale_name)
    save_file(held, str(tmp_path / "model.safetensors"))
    model = Block()
    report = load_pretrained(model, tmp_path)
    assert not report.missing and not report.unexpected and len(report.loaded) == 12
    for layer, names in ((model.qkv_proj, ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj")),
                         (model.gate_up_proj, ("mlp.gate_proj", "mlp.up_proj")), (model.down_proj, ("mlp.down_proj",))):
        assert torch.equal(layer.weight_scale, torch.cat([held[f"l.{n}.{scale_name}"] for n in names]))
        assert torch.equal(layer.weight.view(torch.uint8), torch.cat([held[f"l.{n}.weight"] for n in names]).view(torch.uint8))


def test_loader_refuses_legs_that_are_not_whole_blocks(tmp_path):
    from safetensors.torch import save_file

    from phyai_amd.weights import load_pretrained

    save_file(checkpoint("weight_scale", SHAPES | {"l.mlp.gate_proj": 192, "l.mlp.up_proj": 320}), str(tmp_path / "model.safetensors"))
    with pytest.raises(ValueError, match="whole blocks"):
        load_pretrained(Block(widths=(192, 320)), tmp_path)
    held = checkpoint("weight_scale")
    held["l.mlp.up_proj.weight_scale"] = torch.ones(2, 3)
    save_file(held, str(tmp_path / "model.safetensors"))
    with pytest.raises(ValueError, match="scales"):
        load_pretrained(Block(), tmp_path)


def test_rope_table_far_out():
    from phyai_amd import ops

    table = ops.rope_table(100001, 64, device="cpu")
    angle = 100000 * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert table.shape == (100001, 64) and torch.equal(table[100000], torch.cat([angle.cos(), angle.sin()]).float())
    assert ops.rope_table(0, 64, device="cpu").shape == (0, 64)


def test_paged_prefix_attention_lays_sequences_out_in_pages():
    from phyai_amd.runtime import PagedPrefixAttention

    a = PagedPrefixAttention(2, 5, [7, 0, 12], 4, 32, 2, device="cpu", page_size=8)
    assert a.page_table.tolist() == [[0, 1, -1], [2, -1, -1], [3, 4, 5]] and a.k_pages[1].shape == (6, 8, 2, 32)
    positions, slots, offsets, lens = a._chunk
    assert positions.tolist() == [7, 8, 9, 10, 11, 0, 1, 2, 3, 4, 12, 13, 14, 15, 16] and offsets.tolist() == [0, 5, 10, 15] and lens.tolist() == [12, 5, 17]
    assert slots.tolist() == [7, 8, 9, 10, 11, 16, 17, 18, 19, 20, 36, 37, 38, 39, 40]
    positions, slots, offsets, lens = a._prefix
    assert positions.tolist() == list(range(7)) + list(range(12)) and slots.tolist() == list(range(7)) + list(range(24, 36))
    assert offsets.tolist() == [0, 7, 7, 19] and lens.tolist() == [7, 0, 12]
    for bad in (dict(prefix_len=-1), dict(chunk=0), dict(page_size=0), dict(prefix_len=[]), dict(norms=[])):
        kw = dict(n_layers=1, chunk=5, prefix_len=3, device="cpu") | bad
        with pytest.raises(ValueError):
            PagedPrefixAttention(**kw)
