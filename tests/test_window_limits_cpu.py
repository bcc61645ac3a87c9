"""Host side of the window-attention and 4-bit-cache calls at the ends of what they allow."""
import pytest
import torch

from image_caption_amd import ops

BIG = [1 << 31, 1 << 32, (1 << 32) + 5, 1 << 63, -(1 << 31) - 1]       # 2^32 + 5 would arrive as 5, 2^32 as 0


@pytest.mark.parametrize("big", BIG)
def test_numbers_past_32_bits_are_refused(big):
    """Before anything else is looked at (the tensors are on the CPU, which is refused later, as a RuntimeError)."""
    q = torch.zeros(1, 2, 4, 32)
    c = ops.kv4_cache(1, 2, 8, 32, "cpu")
    one, lse = q[:, :, 0].contiguous(), torch.zeros(1, 2, 4)
    kv = torch.zeros(1, 2, 2, 4, 32)
    calls = [lambda **kw: ops.attn_window_fwd(q, q, q, q, **{"window": 4, **kw}),
             lambda **kw: ops.attn_window_bwd(q, q, q, q, lse, q, q, q, q, lse, **{"window": 4, **kw}),
             lambda **kw: ops.attn_window_decode(one, kv, one, **{"window": 4, **kw}),
             lambda **kw: ops.attn_decode_kv4(one, c, one, **{"smax": 8, **kw})]
    for call in calls:
        for name in ("window", "prefix_len"):
            with pytest.raises(ValueError, match="2\\^31"):
                call(**{name: big})
    for call in calls[:2]:
        with pytest.raises(ValueError, match="2\\^31"):
            call(q_start=big)
    for call in calls[2:]:
        with pytest.raises(ValueError, match="2\\^31"):
            call(length=big)
    for call in (lambda **kw: ops.kv4_append(q, q, c, **{"smax": 8, **kw}), lambda **kw: ops.kv4_unpack(c, q, q, **{"smax": 8, **kw})):
        for name in ("smax", "start"):
            with pytest.raises(ValueError, match="2\\^31"):
                call(**{name: big})
    with pytest.raises(ValueError, match="2\\^31"):
        calls[3](smax=big)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.kv4_cache(1, 2, big, 32, "cpu")
    for size in (lambda w, p: ops.attn_window_fwd_workspace(1, 8, 8, 65536, 1, 64, window=w, prefix_len=p),
                 lambda w, p: ops.attn_window_bwd_workspace(1, 8, 8, 65536, 1, 64, window=w, prefix_len=p),
                 lambda w, p: ops.attn_window_decode_workspace(1, 8, 8, 64, 65536, window=w, prefix_len=p),
                 lambda w, p: ops.attn_decode_kv4_workspace(1, 8, 8, 64, 65536, window=w, prefix_len=p)):
        for w, p in ((big, 0), (0, big)):
            with pytest.raises(ValueError, match="2\\^31"):
                size(w, p)


def test_largest_numbers_that_fit_mean_no_limit():
    top = (1 << 31) - 1
    assert ops.attn_window_decode_workspace(2, 8, 2, 128, 65536, window=top) == ops.attn_window_decode_workspace(2, 8, 2, 128, 65536, window=0)
    assert ops.attn_window_decode_workspace(2, 8, 2, 128, 65536, window=5, prefix_len=top) == ops.attn_window_decode_workspace(2, 8, 2, 128, 65536, window=0)


def test_engine_refuses_a_window_past_32_bits():
    from image_caption_amd.engine import DecoderEngine, EngineOptions, ModelGeometry
    geo = ModelGeometry(64, 2, 128, 503)
    DecoderEngine(geo, EngineOptions(mask_mode="window", window=(1 << 31) - 1))
    for w in (1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError, match="window"):
            DecoderEngine(geo, EngineOptions(mask_mode="window", window=w))


def decode_step(kv, **kw):
    """The return code of a decoding step over made-up addresses, all of which the host must refuse (a launch would give -2 here)."""
    import ctypes
    from image_caption_amd import _lib
    at = 1 << 20
    nb = kw.pop("n_blocks", 2)
    blocks = (_lib.BlockParams * nb)()
    for i in range(nb):
        for name, _ in _lib.BlockParams._fields_:
            setattr(blocks[i], name, at)
    for name, val in kw.pop("last", {}).items():
        setattr(blocks[nb - 1], name, val)
    d = _lib.DecodeDesc()
    base = dict(B=2, d_model=64, nhead=2, dim_ff=128, vocab=100, n_blocks=nb, smax=40, dtype=_lib.BF16, ln_eps=1e-5, head_w=at, emb=at, x_last=at, ids=at,
                done=at, out=at, max_len=8, t=0, s_new=20, workspace=at, workspace_bytes=1 << 40)
    base.update(kw)
    for name, val in base.items():
        setattr(d, name, val)
    d.blocks = blocks
    lib = _lib.load()
    return lib.capdec_decode_step_kv(ctypes.byref(d), kv, None), lib.capdec_last_error().decode()


@pytest.mark.parametrize("four,window", [(1, 0), (0, 5), (1, 5)])
def test_decode_step_refuses_before_it_advances_the_tokens(four, window):
    from image_caption_amd import _lib
    kv = _lib.DecodeKv(four, window, 3)
    for bad, text in ((dict(d_model=96), "head dim 48"), (dict(last=dict(kv_cache=(1 << 20) + 8)), "aligned"), (dict(last=dict(kv_cache=None)), "null"),
                      (dict(last=dict(linear2_w=None)), "null"), (dict(smax=1 << 28), "smax")):
        rc, why = decode_step(kv, **bad)
        assert rc == -1 and text in why, (bad, rc, why)
    rc, why = decode_step(None, last=dict(norm2_b=None))
    assert rc == -1 and "null" in why


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("name", ["k_ss", "v_ss"])
def test_key_strides_whose_products_wrap_are_refused(name, dtype):
    """64 or 128 rows of 2^58 elements and more are 0 in 64 bits; nothing of the addresses may reach a launch (-2 here)."""
    import ctypes
    from image_caption_amd import _lib
    from test_window_attention_cpu import bwd_desc, desc
    lib = _lib.load()
    code = (_lib.BF16, _lib.F32)[dtype]
    for stride in (1 << 25, 1 << 56, 1 << 57, 1 << 58, 1 << 60, (1 << 62) + 64):
        d = desc(dtype=code, **{name: stride})
        assert lib.capdec_attn_window_fwd(ctypes.byref(d), None) == -1 and b"too far apart" in lib.capdec_last_error(), stride
        assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(d)), None) == -1 and b"too far apart" in lib.capdec_last_error(), stride


def test_more_rows_than_32_bits_are_refused():
    """16 queries of 2^30 heads on one K/V head: queries * heads * heads is 2^64, which 64 bits hold as 0."""
    import ctypes
    from image_caption_amd import _lib
    from test_window_attention_cpu import bwd_desc, desc
    lib = _lib.load()
    d = desc(B=1, H=1 << 30, Hkv=1, nq=16, q_start=48)
    assert lib.capdec_attn_window_fwd(ctypes.byref(d), None) == -1 and b"queries of" in lib.capdec_last_error()
    assert lib.capdec_attn_window_bwd(ctypes.byref(bwd_desc(d)), None) == -1 and b"queries of" in lib.capdec_last_error()
