"""Host side of attention under a sliding window: refusals (before anything is launched), workspace sizes, the oracle's rule."""
import ctypes

import pytest
import torch

import window_oracle as wo
from image_caption_amd import _lib, ops

PTR = 1 << 20           # never dereferenced: every call below is refused on the host


def desc(**kw):
    d = _lib.AttnWindowDesc()
    base = dict(q=PTR, k=PTR, v=PTR, o=PTR, dtype=_lib.BF16, B=2, H=4, Hkv=2, S=64, hd=64, q_start=0, nq=64, window=8, prefix_len=2)
    for x in "qkvo":
        base.update({f"{x}_bs": 64 * 64 * 4, f"{x}_hs": 64 * 64, f"{x}_ss": 64})
    base.update(kw)
    for name, val in base.items():
        setattr(d, name, val)
    return d



BAD = [
    (dict(q=None), "null"), (dict(o=None), "null"), (dict(dtype=7), "dtype"), (dict(H=5), "Hkv must divide H"), (dict(Hkv=0), "Hkv"),
    (dict(hd=80), "head dim"), (dict(hd=256), "head dim"), (dict(B=0), "B 0"), (dict(S=0, nq=0), "0 keys"), (dict(S=1 << 28), "keys"),
    (dict(nq=0), "queries"), (dict(q_start=1), "queries"), (dict(q_start=-1, nq=3), "queries"), (dict(window=-1), "window"),
    (dict(prefix_len=-2), "prefix"), (dict(k=PTR + 8), "aligned"), (dict(q_ss=65), "stride"), (dict(v_hs=-64), "stride"),
    (dict(k_ss=1 << 24), "too far apart"), (dict(B=1 << 20, H=1 << 13, Hkv=1 << 13), "queries of"),
    (dict(drop=_lib.Dropout(1.0, 1, 2)), "dropout probability"), (dict(S=200000, nq=64, drop=_lib.Dropout(0.1, 1, 2)), "dropout index space"),
]


@pytest.mark.parametrize("change,text", BAD)
def test_forward_refuses(change, text):
    lib = _lib.load()
    assert lib.capdec_attn_window_fwd(ctypes.byref(desc(**change)), None) == -1
    assert text in lib.capdec_last_error().decode(), lib.capdec_last_error()


@pytest.mark.parametrize("change,text", BAD)
def test_backward_refuses_the_same(change, text):
    lib = _lib.load()
    b = _lib.AttnWindowBwdDesc()
    b.fwd = desc(**change)
    assert lib.capdec_attn_window_bwd(ctypes.byref(b), None) == -1
    assert text in lib.capdec_last_error().decode()


def bwd_desc(fwd, **kw):
    b = _lib.AttnWindowBwdDesc()
    b.fwd = fwd
    b.fwd.lse = PTR
    base = dict(dout=PTR, dq=PTR, dk=PTR, dv=PTR, delta=PTR, dq_scale=1.0)
    base.update(kw)
    for name, val in base.items():
        setattr(b, name, val)
    return b


def test_backward_refuses_missing_operands_and_small_workspaces():
    lib = _lib.load()
    assert lib.capdec_attn_window_bwd(None, None) == -1
    for name in ("dout", "dq", "dk", "dv", "delta"):
        assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(desc(), **{name: None})), None) == -1
        assert b"null" in lib.capdec_last_error()
    b = bwd_desc(desc())
    b.fwd.lse = None
    assert lib.capdec_attn_window_bwd(ctypes.byref(b), None) == -1
    assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(desc(), dk_ss=3)), None) == -1
    assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(desc(), dv=PTR + 4)), None) == -1
    # a long sequence on one head: the prefix tile's rows are cut, which needs a workspace
    need = lib.capdec_attn_window_bwd_workspace(1, 1, 1, 8192, 8192, 64, 64, 4)
    assert need > 0
    f = desc(B=1, H=1, Hkv=1, S=8192, nq=8192, window=64, prefix_len=4)
    assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(f)), None) == -3
    f.workspace, f.workspace_bytes = PTR, need - 1
    assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(f)), None) == -3


def test_forward_refuses_a_small_workspace():
    lib = _lib.load()
    need = lib.capdec_attn_window_fwd_workspace(1, 8, 8, 65536, 1, 64, 0, 0)
    assert need > 0
    f = desc(B=1, H=8, Hkv=8, S=65536, q_start=65535, nq=1, window=0, prefix_len=0)
    f.workspace, f.workspace_bytes = PTR, need - 1
    assert lib.capdec_attn_window_fwd(ctypes.byref(f), None) == -3


def test_decode_refuses():
    lib = _lib.load()

    def call(q=PTR, kv=PTR, o=PTR, dtype=1, B=1, H=4, Hkv=2, hd=64, smax=32, n=8, window=0, prefix=0, ws=None, wsb=0):
        return lib.capdec_attn_window_decode(q, kv, o, dtype, B, H, Hkv, hd, smax, n, None, window, prefix, ws, wsb, None)

    for bad in (dict(n=0), dict(n=33), dict(smax=0), dict(q=None), dict(kv=None), dict(o=None), dict(H=5), dict(hd=48), dict(dtype=2), dict(window=-1)):
        assert call(**bad) == -1, bad


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.capdec_attn_window_fwd_workspace(0, 4, 2, 64, 64, 64, 0, 0) == 0
    assert lib.capdec_attn_window_fwd_workspace(256, 8, 8, 229, 32, 96, 16, 197) == 0       # enough workgroups without a cut
    full = lib.capdec_attn_window_decode_workspace(2, 8, 2, 128, 65536, 0, 0)
    assert full > 0
    for smax in (1, 100, 5000, 65536):                                                      # one workspace fits every shorter length
        assert lib.capdec_attn_window_decode_workspace(2, 8, 2, 128, smax, 0, 0) <= full
    for window in (1, 100, 70000):
        assert lib.capdec_attn_window_decode_workspace(2, 8, 2, 128, 65536, window, 4) <= full


def test_wrappers_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 4, 32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.attn_window_fwd(q, q, q, q, window=4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.attn_window_bwd(q, q, q, q, torch.zeros(1, 2, 4), q, q, q, q, torch.zeros(1, 2, 4), window=4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.attn_window_decode(q[:, :, 0], torch.zeros(1, 2, 2, 4, 32), q[:, :, 0], window=4)


@pytest.mark.parametrize("window,prefix,is_open", [(0, 0, False), (1, 0, False), (3, 2, False), (3, 2, True), (0, 5, True), (9, 20, True)])
def test_oracle_rule_spelled_out(window, prefix, is_open):
    lens = [9, 4, 0]
    got = wo.masks(3, 9, 6, 3, lens, window, prefix, is_open, "cpu")
    for b, n in enumerate(lens):
        assert torch.equal(got[b], wo.visible(9, range(3, 9), n, window, prefix, is_open))


def test_oracle_gradients_against_differences():
    """The oracle's formulas are the derivatives of its forward (64 bits, central differences)."""
    g = torch.Generator().manual_seed(5)
    q, k, v, d = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((1, 4, 5, 8), (1, 2, 7, 8), (1, 2, 7, 8), (1, 4, 5, 8)))
    see = wo.masks(1, 7, 5, 2, [6], 3, 2, True, "cpu")
    wo.HALF[torch.float64] = 0.0
    try:
        o, lse, _, _ = wo.forward(q, k, v, see)
        (dq, _), (dk, _), (dv, _) = wo.backward(q, k, v, o, lse, d, see, 1.0)
        for t, grad in ((q, dq), (k, dk), (v, dv)):
            for idx in torch.randint(0, t.numel(), (12,), generator=g).tolist():
                vals = []
                for sign in (1, -1):
                    keep = t.view(-1)[idx].item()
                    t.view(-1)[idx] += sign * 1e-5
                    vals.append((wo.forward(q, k, v, see)[0] * torch.where(see.any(-1)[:, None, :, None], d, 0.0)).sum().item())
                    t.view(-1)[idx] = keep
                assert abs((vals[0] - vals[1]) / 2e-5 - grad.reshape(-1)[idx].item()) < 1e-7
    finally:
        del wo.HALF[torch.float64]


def test_struct_layouts_match_c(tmp_path):
    import os
    import subprocess

    from helpers import ROOT
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "capdec.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n",'
                   'sizeof(capdec_attn_window_desc), offsetof(capdec_attn_window_desc, lens), offsetof(capdec_attn_window_desc, workspace_bytes),'
                   'sizeof(capdec_attn_window_bwd_desc), offsetof(capdec_attn_window_bwd_desc, dout), offsetof(capdec_attn_window_bwd_desc, delta));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    W, WB = _lib.AttnWindowDesc, _lib.AttnWindowBwdDesc
    assert got == [ctypes.sizeof(W), W.lens.offset, W.workspace_bytes.offset, ctypes.sizeof(WB), WB.dout.offset, WB.delta.offset]


@pytest.mark.parametrize("mode,window", [("prefix_window", 3), ("window", 3), ("prefix_window", 0), ("window", 0)])
def test_model_mask_is_the_oracles(mode, window):
    from image_caption_amd.decoder import TransformerDecoder
    from image_caption_amd.engine import EngineOptions
    from oracle import ref_cpu
    m = TransformerDecoder(64, 2, 6, 128, 0.0, 503, options=EngineOptions(mask_mode=mode, window=window))
    m.prefix_len = 4
    see = wo.masks(1, 12, 12, 0, [12], window, 4, mode == "prefix_window", "cpu")[0]
    assert torch.equal(m.create_caption_mask(12) == 0, see)
    if window:
        assert torch.equal(ref_cpu.caption_mask(12, f"{mode}:{window}", 4) == 0, see)


def test_engine_options_refused():
    from image_caption_amd.engine import DecoderEngine, EngineOptions, ModelGeometry
    geo = ModelGeometry(64, 2, 128, 503)
    for bad in (dict(mask_mode="windows"), dict(window=4), dict(mask_mode="prefix_window", window=-1), dict(kv_cache_bits=8)):
        with pytest.raises(ValueError):
            DecoderEngine(geo, EngineOptions(**bad))


def test_engine_refuses_head_dimensions_without_kernels():
    from image_caption_amd.engine import DecoderEngine, EngineOptions, ModelGeometry
    for opt in (dict(mask_mode="window", window=3), dict(mask_mode="prefix_window"), dict(kv_cache_bits=4)):
        with pytest.raises(ValueError, match="head dimension"):
            DecoderEngine(ModelGeometry(96, 2, 128, 503), EngineOptions(**opt))
        DecoderEngine(ModelGeometry(64, 2, 128, 503), EngineOptions(**opt))
