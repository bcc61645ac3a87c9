"""Host side of the 4-bit cache: sizes, refusals before anything is launched, the struct's layout."""
import ctypes
import os
import subprocess

import pytest
import torch

from helpers import ROOT
from image_caption_amd import _lib, ops

PTR = 1 << 20           # never dereferenced: every call below is refused on the host


def rows(**kw):
    r = _lib.Kv4Rows()
    base = dict(k=PTR, v=PTR, k_bs=64 * 64, k_hs=64 * 8, k_ss=64, v_bs=64 * 64, v_hs=64 * 8, v_ss=64, dtype=_lib.BF16, n=8)
    base.update(kw)
    for name, val in base.items():
        setattr(r, name, val)
    return r


def test_sizes():
    lib = _lib.load()
    assert lib.capdec_kv4_head_bytes(32, 128) == 32 * (2 * 64 + 2 * 16)          # 4 bits a value, 4 bytes a group of 32
    assert lib.capdec_kv4_head_bytes(33, 96) == 64 * (2 * 48 + 2 * 12)           # rows come in blocks of 32
    assert lib.capdec_kv4_head_bytes(0, 64) == 0 and lib.capdec_kv4_head_bytes(10, 48) == 0
    full = lib.capdec_attn_decode_kv4_workspace(2, 8, 2, 128, 65536, 0, 0)
    assert full > 0
    for smax in (1, 500, 5000, 65536):
        assert lib.capdec_attn_decode_kv4_workspace(2, 8, 2, 128, smax, 0, 0) <= full
    assert lib.capdec_attn_decode_kv4_workspace(256, 8, 8, 96, 229, 0, 0) == 0


def test_append_and_unpack_refuse():
    lib = _lib.load()

    def append(r=None, cache=PTR, B=2, Hkv=2, smax=64, hd=64, start=0, starts=None, counts=None, **kw):
        return lib.capdec_kv4_append(ctypes.byref(r or rows(**kw)), cache, B, Hkv, smax, hd, start, starts, counts, None)

    def unpack(r=None, cache=PTR, B=2, Hkv=2, smax=64, hd=64, start=0, starts=None, **kw):
        return lib.capdec_kv4_unpack(cache, ctypes.byref(r or rows(**kw)), B, Hkv, smax, hd, start, starts, None)

    common = [dict(cache=None), dict(cache=PTR + 4), dict(B=0), dict(Hkv=0), dict(smax=0), dict(smax=1 << 28), dict(hd=48), dict(n=0), dict(dtype=5),
              dict(start=-1), dict(start=57), dict(n=65)]
    for bad in common + [dict(k=None), dict(v=None), dict(k=PTR + 2), dict(k_ss=60), dict(v_hs=-64), dict(n=1 << 24, smax=1 << 25)]:
        assert append(**bad) == -1, bad
    for bad in common + [dict(k=None, v=None)]:
        assert unpack(**bad) == -1, bad
    assert lib.capdec_kv4_append(None, PTR, 2, 2, 64, 64, 0, None, None, None) == -1


def test_attention_refuses():
    lib = _lib.load()

    def call(q=PTR, cache=PTR, o=PTR, dtype=1, B=1, H=4, Hkv=2, hd=64, smax=64, n=8, window=0, prefix=0, ws=None, wsb=0):
        return lib.capdec_attn_decode_kv4(q, cache, o, dtype, B, H, Hkv, hd, smax, n, None, window, prefix, ws, wsb, None)

    for bad in (dict(n=0), dict(n=65), dict(smax=0), dict(q=None), dict(q=PTR + 4), dict(o=None), dict(cache=None), dict(H=5), dict(H=0), dict(hd=40),
                dict(dtype=2), dict(window=-1), dict(prefix=-1)):
        assert call(**bad) == -1, bad
    need = lib.capdec_attn_decode_kv4_workspace(1, 4, 2, 64, 65536, 0, 0)
    assert call(smax=65536, n=65536, ws=PTR, wsb=need - 1) == -3
    assert call(smax=65536, n=65536, ws=PTR + 4, wsb=need) == -1


def test_struct_layout_matches_c(tmp_path):
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "capdec.h"\nint main(void){printf("%zu %zu %zu %zu %zu\\n", sizeof(capdec_kv4_rows),'
                   'offsetof(capdec_kv4_rows, v_ss), offsetof(capdec_kv4_rows, n), sizeof(capdec_decode_kv), offsetof(capdec_decode_kv, prefix_len));return 0;}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.Kv4Rows), _lib.Kv4Rows.v_ss.offset, _lib.Kv4Rows.n.offset,
                   ctypes.sizeof(_lib.DecodeKv), _lib.DecodeKv.prefix_len.offset]


def test_wrappers_refuse_cpu_tensors():
    x = torch.zeros(1, 2, 4, 32)
    c = ops.kv4_cache(1, 2, 8, 32, "cpu")
    for call in (lambda: ops.kv4_append(x, x, c, smax=8), lambda: ops.kv4_unpack(c, x, x, smax=8),
                 lambda: ops.attn_decode_kv4(x[:, :, 0].contiguous(), c, x[:, :, 0].contiguous(), smax=8)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError):
        ops.kv4_cache(1, 2, 8, 48, "cpu")
