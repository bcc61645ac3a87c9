"""Attention under a sliding window (forward, backward, one token over a cache) against plain attention in 64 bits."""
import math

import pytest
import torch

import window_oracle as wo
from image_caption_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float32]


def make(B, H, Hkv, S, nq, hd, dtype, seed=0, packed=False):
    """q, k, v, dout; packed: views of one [S, B, (H + 2 Hkv) hd] projection, rows of a sequence B apart."""
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)

    scale = hd ** -0.5
    if packed:
        x = normal(S, B, H + 2 * Hkv, hd)
        x[:, :, :H] *= scale
        x = x.to(dtype)
        q, k, v = (t.permute(1, 2, 0, 3) for t in (x[:, :, :H], x[:, :, H:H + Hkv], x[:, :, H + Hkv:]))
        q = q[:, :, S - nq:]
    else:
        q, k, v = (normal(B, H, nq, hd) * scale).to(dtype), normal(B, Hkv, S, hd).to(dtype), normal(B, Hkv, S, hd).to(dtype)
    return q, k, v, normal(B, H, nq, hd).to(dtype)


def lens_of(spec, B, S):
    return [S] * B if spec is None else [min(S, spec[b % len(spec)]) for b in range(B)]


def run_fwd(q, k, v, lens, *, split=True, **kw):
    B, H, nq, hd = q.shape
    o = torch.full((B, H, nq, hd), float("nan"), dtype=q.dtype, device=DEV)
    lse = torch.full((B, H, nq), float("nan"), device=DEV)
    ws = None
    if split:
        ws = torch.full((ops.attn_window_fwd_workspace(B, H, k.shape[1], k.shape[2], nq, hd, window=kw["window"], prefix_len=kw["prefix_len"]) + 16,),
                        255, dtype=torch.uint8, device=DEV)
    ops.attn_window_fwd(q, k, v, o, lens=lens, lse=lse, workspace=ws, **kw)
    return o, lse


# B, H, Hkv, S, nq, hd, window, prefix, open, lens
CASES = [
    (1, 1, 1, 1, 1, 32, 0, 0, False, None),                        # one token
    (2, 2, 2, 5, 5, 64, 1, 0, False, (5, 0)),                      # each sees itself; an empty sequence
    (3, 8, 8, 229, 32, 96, 16, 197, True, None),                   # the captioning model's scored rows
    (2, 8, 8, 229, 229, 96, 16, 197, True, (229, 200)),            # all rows, a padded one (a length inside the text)
    (2, 4, 2, 130, 130, 128, 17, 3, False, (130, 1)),
    (1, 6, 2, 333, 333, 64, 64, 0, False, None),                   # three heads to a K/V head, an exact multiple of a tile as window
    (2, 4, 4, 257, 100, 32, 0, 0, False, (257, 180)),              # causal, last rows; sequences that end inside them
    (1, 8, 1, 600, 600, 64, 33, 130, False, None),                 # a prefix of more than one key tile
    (1, 16, 2, 700, 7, 128, 500, 9, True, None),                   # few rows of many heads
    (2, 2, 1, 300, 300, 96, 1000, 5000, True, (300, 64)),          # window and prefix past the end: everything visible, a length at a tile's end
    (1, 5, 1, 1500, 1500, 32, 100, 4, False, (1450,)),
    (1, 40, 1, 200, 2, 64, 50, 0, False, None),                    # more heads than a tile has rows
    (5, 2, 2, 64, 64, 32, 8, 2, True, (64, 33, 32, 31, 2)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(case, dtype):
    B, H, Hkv, S, nq, hd, window, prefix, is_open, spec = case
    print(case, dtype, flush=True)
    q, k, v, dout = make(B, H, Hkv, S, nq, hd, dtype, packed=nq == S)
    ns = lens_of(spec, B, S)
    lens = None if spec is None else torch.tensor(ns, dtype=torch.int32, device=DEV)
    kw = dict(window=window, prefix_len=prefix, prefix_open=is_open, q_start=S - nq)
    see = wo.masks(B, S, nq, S - nq, ns, window, prefix, is_open, DEV)
    want, want_lse, bound, bound_lse = wo.forward(q, k, v, see)
    for split in (True, False):
        o, lse = run_fwd(q, k, v, lens, split=split, **kw)
        wo.assert_within(o, want, bound, f"o split={split}")
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        wo.assert_within(lse.masked_fill(empty, 0.0), want_lse.masked_fill(empty, 0.0), bound_lse, "lse")
        assert not o[empty].any()
    dq = torch.full_like(q.contiguous(), float("nan"))
    dkv = torch.full((B, Hkv, 2, S, hd), float("nan"), dtype=dtype, device=DEV)
    delta = torch.empty(B, H, nq, device=DEV)
    grads = dq, dkv[:, :, 0], dkv[:, :, 1]
    ops.attn_window_bwd(q, k, v, o, lse, dout, *grads, delta, lens=lens, dq_scale=hd ** -0.5, **kw)
    oracle = wo.backward(q, k, v, o, lse, dout, see, hd ** -0.5)
    for got, (w, bd), what in zip(grads, oracle, ("dq", "dk", "dv")):
        wo.assert_within(got, w, bd, what)
    # the same bits again
    first = [t.clone() for t in grads]
    ops.attn_window_bwd(q, k, v, o, lse, dout, *grads, delta, lens=lens, dq_scale=hd ** -0.5, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [9, 90])
def test_rows_past_the_end_may_hold_anything(dtype, nq):
    """NaN and infinities behind each sequence: K, V, q, dout, and (no sequence is that long) the lse and o of such rows."""
    B, H, Hkv, S, hd = 3, 4, 2, 90, 64
    ns = [90, 61, 0]
    q, k, v, dout = make(B, H, Hkv, S, nq, hd, dtype)
    clean = [t.clone() for t in (q, k, v, dout)]
    for b, n in enumerate(ns):
        for t, off in ((q, S - nq), (k, 0), (v, 0), (dout, S - nq)):
            t[b, :, max(0, n - off):] = float("nan") if b == 1 else float("inf")
    lens = torch.tensor(ns, dtype=torch.int32, device=DEV)
    kw = dict(window=20, prefix_len=2, prefix_open=False, q_start=S - nq)
    res = []
    for qq, kk, vv, dd in ((q, k, v, dout), clean):
        o, lse = run_fwd(qq, kk, vv, lens, **kw)
        dq, dk, dv = torch.empty_like(qq), torch.empty_like(kk), torch.empty_like(vv)
        ops.attn_window_bwd(qq, kk, vv, o, lse, dd, dq, dk, dv, torch.empty(B, H, nq, device=DEV), lens=lens, **kw)
        res.append((o, lse, dq, dk, dv))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    for b, n in enumerate(ns):
        assert not res[0][3][b, :, n:].any() and not res[0][4][b, :, n:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S,q_start,nq,window,prefix,is_open,hd", [
    (300, 200, 60, 30, 5, False, 64),                              # a gap inside a tile, and keys behind the last query
    (300, 200, 60, 30, 150, True, 128),
    (300, 100, 1, 10, 0, False, 32),
    (200, 150, 30, 20, 70, False, 96),                             # the one-kernel backward (bf16)
    (700, 500, 150, 40, 270, False, 64),
])
def test_keys_that_no_query_sees_may_hold_anything(S, q_start, nq, window, prefix, is_open, hd, dtype):
    B, H, Hkv = 2, 4, 2
    q, k, v, dout = make(B, H, Hkv, S, nq, hd, dtype)
    seen = wo.masks(B, S, nq, q_start, [S] * B, window, prefix, is_open, DEV)[0].any(0)
    assert not seen.all()
    kw = dict(window=window, prefix_len=prefix, prefix_open=is_open, q_start=q_start)
    res = []
    for fill in (0.0, float("nan"), float("inf")):
        k[:, :, ~seen], v[:, :, ~seen] = fill, -fill
        for split in (True, False):
            o, lse = run_fwd(q, k, v, None, split=split, **kw)
            dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
            ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, torch.empty(B, H, nq, device=DEV), **kw)
            assert not dk[:, :, ~seen].any() and not dv[:, :, ~seen].any()
            res.append((o, lse, dq, dk, dv))
    for other in (2, 4):
        for a, b in zip(res[0] + res[1], res[other] + res[other + 1]):
            assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_past_rows_that_left_the_window(dtype):
    q, cache, o = torch.randn(2, 4, 64, device=DEV, dtype=dtype), torch.randn(2, 2, 2, 900, 64, device=DEV, dtype=dtype), torch.empty(2, 4, 64, device=DEV, dtype=dtype)
    lens = torch.tensor([700, 333], dtype=torch.int32, device=DEV)
    res = []
    for fill in (0.0, float("nan")):
        for b, n in enumerate((700, 333)):
            cache[b, :, :, 10:n - 45] = fill
            cache[b, :, :, n:] = fill
        ops.attn_window_decode(q, cache, o, window=45, prefix_len=10, lens=lens)
        res.append(o.clone())
    assert torch.isfinite(res[1]).all() and torch.equal(*res)


def test_lengths_out_of_range_are_taken_into_it():
    q, k, v, _ = make(2, 2, 2, 40, 40, 32, torch.bfloat16)
    kw = dict(window=7, prefix_len=1, prefix_open=False, q_start=0)
    wild = run_fwd(q, k, v, torch.tensor([-5, 10 ** 9], dtype=torch.int32, device=DEV), **kw)
    tame = run_fwd(q, k, v, torch.tensor([0, 40], dtype=torch.int32, device=DEV), **kw)
    assert torch.equal(wild[0], tame[0]) and torch.equal(wild[1], tame[1])


def test_large_scores():
    """Scores of several hundred, growing and falling along the keys: the running maximum moves and stays exact."""
    q, k, v, _ = make(1, 2, 2, 400, 400, 64, torch.bfloat16)
    k = (k * (torch.linspace(0, 60, 400, device=DEV).sin() * 40)[:, None]).to(torch.bfloat16)
    see = wo.masks(1, 400, 400, 0, [400], 0, 0, False, DEV)
    want, want_lse, bound, bound_lse = wo.forward(q, k, v, see)
    o, lse = run_fwd(q, k, v, None, window=0, prefix_len=0, prefix_open=False, q_start=0)
    wo.assert_within(o, want, bound, "o")
    wo.assert_within(lse, want_lse, bound_lse, "lse")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [20, 150])
def test_dropout(dtype, nq):
    B, H, Hkv, S, hd = 2, 4, 2, 150, 64
    q, k, v, dout = make(B, H, Hkv, S, nq, hd, dtype)
    drop = ops.dropout_keys(7, 3, 1, 0.25)
    keep = ops.attn_dropout_mask(drop, B, H, S, DEV)[:, :, S - nq:].double() / 0.75
    kw = dict(window=40, prefix_len=5, prefix_open=True, q_start=S - nq)
    see = wo.masks(B, S, nq, S - nq, [S] * B, 40, 5, True, DEV)
    want, _, bound, _ = wo.forward(q, k, v, see, keep)
    o, lse = run_fwd(q, k, v, None, drop=drop, **kw)
    wo.assert_within(o, want, bound, "o")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, torch.empty(B, H, nq, device=DEV), drop=drop, dq_scale=0.5, **kw)
    for got, (w, bd), what in zip((dq, dk, dv), wo.backward(q, k, v, o, lse, dout, see, 0.5, keep), ("dq", "dk", "dv")):
        wo.assert_within(got, w, bd, what)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefix_gradients_from_many_rows(dtype):
    """A short prefix under a long sequence: its keys' gradients come from every row, in chunks joined afterwards."""
    B, H, Hkv, S, hd = 1, 4, 2, 4100, 32
    q, k, v, dout = make(B, H, Hkv, S, S, hd, dtype)
    kw = dict(window=70, prefix_len=4, prefix_open=False, q_start=0)
    assert ops.attn_window_bwd_workspace(B, H, Hkv, S, S, hd, window=70, prefix_len=4) > 0
    see = wo.masks(B, S, S, 0, [S], 70, 4, False, DEV)
    o, lse = run_fwd(q, k, v, None, **kw)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, torch.empty(B, H, S, device=DEV), **kw)
    for got, (w, bd), what in zip((dq, dk, dv), wo.backward(q, k, v, o, lse, dout, see, 1.0), ("dq", "dk", "dv")):
        wo.assert_within(got, w, bd, what)


# many short sequences: dQ, dK and dV from one kernel
SHORT = [
    (20, 8, 8, 229, 229, 96, 16, 197, True),
    (16, 16, 8, 256, 256, 64, 0, 0, False),                        # two heads to a K/V head, every row block full
    (64, 6, 2, 131, 40, 32, 10, 2, False),                         # last rows only, three heads to a K/V head
    (130, 1, 1, 200, 1, 96, 0, 7, False),                          # one row
    (33, 20, 4, 160, 160, 64, 31, 150, True),                      # more rows than four keys' worth
    (128, 1, 1, 255, 255, 32, 1, 0, False),                        # each row sees itself
    (64, 6, 2, 131, 40, 64, 10, 2, False),
    (3, 1, 1, 256, 256, 64, 1, 0, False),
    (2, 3, 3, 1, 1, 96, 0, 0, False),                              # one token
    (300, 4, 1, 70, 70, 64, 20, 5, True),                          # 280 rows, more workgroups than CUs
]


@pytest.mark.parametrize("mode", ["plain", "ragged", "dropout"])
@pytest.mark.parametrize("case", SHORT)
def test_backward_of_many_short_sequences(case, mode):
    B, H, Hkv, S, nq, hd, window, prefix, is_open = case
    print(case, mode, flush=True)
    q, k, v, dout = make(B, H, Hkv, S, nq, hd, torch.bfloat16, seed=2, packed=nq == S)
    ns = [S] * B
    if mode == "ragged":
        ends = [0, 1, S, S - 1, 31, 32, 33, S - nq, S - nq + 1, 97, 128, 129]
        ns = [min(S, max(0, ends[b % len(ends)])) for b in range(B)]
    lens = torch.tensor(ns, dtype=torch.int32, device=DEV) if mode == "ragged" else None
    kw = dict(window=window, prefix_len=prefix, prefix_open=is_open, q_start=S - nq)
    keep = None
    if mode == "dropout":
        kw["drop"] = ops.dropout_keys(5, 1, 2, 0.3)
        keep = ops.attn_dropout_mask(kw["drop"], B, H, S, DEV)[:, :, S - nq:].double() / 0.7
    see = wo.masks(B, S, nq, S - nq, ns, window, prefix, is_open, DEV)
    o, lse = run_fwd(q, k, v, lens, **kw)
    oracle = wo.backward(q, k, v, o, lse, dout, see, hd ** -0.5, keep)
    for b, n in enumerate(ns):                                     # what lies behind the ends may be anything
        for t, off in ((q, S - nq), (k, 0), (v, 0), (dout, S - nq), (o, S - nq)):
            t[b, :, max(0, n - off):] = float("nan")
        lse[b, :, max(0, n - S + nq):] = float("nan")
    grads = torch.full((B, H, nq, hd), float("nan"), dtype=torch.bfloat16, device=DEV), *torch.full((2, B, S, Hkv, hd), float("nan"), dtype=torch.bfloat16, device=DEV).transpose(2, 3)
    delta = torch.empty(B, H, nq, device=DEV)
    ops.attn_window_bwd(q, k, v, o, lse, dout, *grads, delta, lens=lens, dq_scale=hd ** -0.5, **kw)
    for got, (w, bd), what in zip(grads, oracle, ("dq", "dk", "dv")):
        wo.assert_within(got, w, bd, what)
    first = [t.clone() for t in grads]
    ops.attn_window_bwd(q, k, v, o, lse, dout, *grads, delta, lens=lens, dq_scale=hd ** -0.5, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, grads))


def test_gradients_against_differences():
    """float32: directional derivatives of sum(o * dout) by central differences of the kernel's own forward, summed in 64 bits."""
    B, H, Hkv, S, hd = 2, 4, 2, 70, 32
    q, k, v, dout = make(B, H, Hkv, S, S, hd, torch.float32)
    kw = dict(window=12, prefix_len=3, prefix_open=True, q_start=0)
    o, lse = run_fwd(q, k, v, None, **kw)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, torch.empty(B, H, S, device=DEV), **kw)
    eps = 2.0 ** -7
    for n, (t, grad) in enumerate(((q, dq), (k, dk), (v, dv))):
        way = torch.randn(t.shape, generator=torch.Generator(device=DEV).manual_seed(90 + n), device=DEV)
        way = way / way.double().norm().float()
        val = []
        for sign in (1, -1):
            ops_in = [x + sign * eps * way if x is t else x for x in (q, k, v)]
            val.append((run_fwd(*ops_in, None, **kw)[0].double() * dout.double()).sum().item())
        slope, want = (val[0] - val[1]) / (2 * eps), (grad.double() * way.double()).sum().item()
        # third derivatives: about eps^2 times the gradient's size; rounding: 2^-24 |o||dout| sqrt(terms) / eps
        size = grad.double().norm().item()
        noise = 2.0 ** -24 * (o.double() * dout.double()).norm().item() * 8 / eps
        assert abs(slope - want) <= 4 * eps * eps * size + 4 * noise, (n, slope, want)


# ------------------------------------------------------------------ one token over a cache
def decode_case(B, H, Hkv, hd, smax, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn(B, H, hd, generator=g, device=DEV) * hd ** -0.5).to(dtype)
    return q, torch.randn(B, Hkv, 2, smax, hd, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hkv,hd,smax,length,window,prefix,spec", [
    (1, 1, 1, 32, 1, 1, 0, 0, None),
    (4, 8, 8, 96, 229, 229, 16, 197, None),
    (3, 8, 2, 128, 300, 257, 40, 4, (257, 0, 1)),
    (2, 12, 4, 64, 3000, 2999, 0, 0, (2999, 1500)),                # cut along the keys
    (1, 32, 8, 128, 5000, 4097, 1000, 70, None),
    (2, 80, 2, 32, 500, 500, 100, 3, (500, 99)),                   # forty heads to a K/V head
    (9, 2, 2, 96, 64, 64, 5, 0, (64, 63, 33, 32, 31, 6, 5, 4, 1)),
])
def test_decode(B, H, Hkv, hd, smax, length, window, prefix, spec, dtype):
    print(B, H, Hkv, hd, smax, length, dtype, flush=True)
    q, cache = decode_case(B, H, Hkv, hd, smax, dtype)
    ns = lens_of(spec, B, length)
    for b, n in enumerate(ns):
        cache[b, :, :, n:] = float("nan")                          # rows not yet written
    lens = None if spec is None else torch.tensor(ns, dtype=torch.int32, device=DEV)
    ws = torch.empty(ops.attn_window_decode_workspace(B, H, Hkv, hd, smax, window=window, prefix_len=prefix), dtype=torch.uint8, device=DEV)
    outs = []
    for w in (ws, None):
        o = torch.full_like(q, float("nan"))
        ops.attn_window_decode(q, cache, o, window=window, prefix_len=prefix, length=length, lens=lens, workspace=w)
        outs.append(o)
        for b, n in enumerate(ns):
            if n == 0:
                assert not o[b].any()
                continue
            see = wo.masks(1, n, 1, n - 1, [n], window, prefix, False, DEV)
            want, _, bound, _ = wo.forward(q[b:b + 1].unsqueeze(2), cache[b:b + 1, :, 0, :n], cache[b:b + 1, :, 1, :n], see)
            wo.assert_within(o[b], want[0, :, 0], bound[0, :, 0], f"sequence {b}")
    flat = torch.empty(B, H * hd, dtype=dtype, device=DEV)
    ops.attn_window_decode(q.view(B, H * hd), cache, flat, window=window, prefix_len=prefix, length=length, lens=lens, workspace=ws)
    assert torch.equal(flat.view_as(outs[0]), outs[0])


def test_decode_past_two_gigabytes_of_one_head():
    """Offsets of a head's last rows pass 2^31 bytes (f32, hd 128: 512 bytes a row)."""
    smax = (1 << 22) + 300
    cache = torch.zeros(1, 1, 2, smax, 128, device=DEV)
    cache[:, :, 0, -64:] = torch.randn(64, 128, device=DEV)
    cache[:, :, 1, -64:] = torch.randn(64, 128, device=DEV)
    q = torch.randn(1, 2, 128, device=DEV) * 128 ** -0.5
    o = torch.empty_like(q)
    ops.attn_window_decode(q, cache, o, window=50, prefix_len=0)
    see = wo.masks(1, 64, 1, 63, [64], 50, 0, False, DEV)
    want, _, bound, _ = wo.forward(q.unsqueeze(2), cache[:, :, 0, -64:], cache[:, :, 1, -64:], see)
    wo.assert_within(o, want[:, :, 0], bound[:, :, 0], "o")


# ------------------------------------------------------------------ streams, graphs, two calls at once
def test_graph_replays_follow_new_inputs_and_lengths():
    B, H, Hkv, hd, smax = 2, 8, 2, 64, 3000
    q, cache = decode_case(B, H, Hkv, hd, smax, torch.bfloat16)
    lens = torch.tensor([3000, 10], dtype=torch.int32, device=DEV)
    o, eager = torch.empty_like(q), torch.empty_like(q)
    ws, ws2 = (torch.empty(ops.attn_window_decode_workspace(B, H, Hkv, hd, smax, window=0), dtype=torch.uint8, device=DEV) for _ in range(2))
    fq, fk, fv, dout = make(1, 4, 2, 400, 400, 64, torch.bfloat16)
    fo, flse, delta = torch.empty_like(fq), torch.empty(1, 4, 400, device=DEV), torch.empty(1, 4, 400, device=DEV)
    grads = [torch.empty_like(t) for t in (fq, fk, fv)]
    bws = torch.empty(ops.attn_window_bwd_workspace(1, 4, 2, 400, 400, 64, window=30, prefix_len=4), dtype=torch.uint8, device=DEV)
    kw = dict(window=30, prefix_len=4)

    def work(out, w):
        ops.attn_window_decode(q, cache, out, window=0, lens=lens, workspace=w)
        ops.attn_window_fwd(fq, fk, fv, fo, lse=flse, **kw)
        ops.attn_window_bwd(fq, fk, fv, fo, flse, dout, *grads, delta, workspace=bws, **kw)

    work(o, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(o, ws)
    for step in range(4):
        g = torch.Generator(device=DEV).manual_seed(50 + step)
        q.copy_(torch.randn(q.shape, generator=g, device=DEV) * 0.1)
        fk.copy_(torch.randn(fk.shape, generator=g, device=DEV))
        lens.copy_(torch.tensor([700 * step + 1, 2999 - step], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (o, fo, *grads)]
        work(eager, ws2)
        torch.cuda.synchronize()
        for a, b in zip(got, (eager, fo, *grads)):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    cases = [decode_case(2, 8, 2, 128, 5000, torch.bfloat16, seed=s) for s in (1, 2)]
    wss = [torch.empty(ops.attn_window_decode_workspace(2, 8, 2, 128, 5000, window=0), dtype=torch.uint8, device=DEV) for _ in cases]
    alone = []
    for (q, cache), ws in zip(cases, wss):
        o = torch.empty_like(q)
        ops.attn_window_decode(q, cache, o, window=0, workspace=ws)
        alone.append(o)
    torch.cuda.synchronize()
    outs = [torch.empty_like(q) for q, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for (q, cache), ws, o, st in zip(cases, wss, outs, streams):
            with torch.cuda.stream(st):
                ops.attn_window_decode(q, cache, o, window=0, workspace=ws)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))


@pytest.mark.parametrize("B,H,S", [(4, 8, 229), (1, 4, 400)])       # one kernel for all three gradients, and two
def test_backward_in_a_graph_and_on_two_streams(B, H, S):
    hd, kw = 96, dict(window=20, prefix_len=100, prefix_open=True)
    size = ops.attn_window_bwd_workspace(B, H, H, S, S, hd, window=20, prefix_len=100)
    sets = []
    for seed in (1, 2):
        q, k, v, dout = make(B, H, H, S, S, hd, torch.bfloat16, seed=seed)
        o, lse = run_fwd(q, k, v, None, q_start=0, **kw)
        sets.append(dict(ins=(q, k, v, o, lse, dout), grads=[torch.empty_like(t) for t in (q, k, v)], delta=torch.empty(B, H, S, device=DEV),
                         ws=torch.empty(size, dtype=torch.uint8, device=DEV)))

    def work(c, grads):
        ops.attn_window_bwd(*c["ins"], *grads, c["delta"], workspace=c["ws"], **kw)

    alone = []
    for c in sets:
        grads = [torch.empty_like(t) for t in c["grads"]]
        work(c, grads)
        alone.append(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(sets[0], sets[0]["grads"])
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for t in (*sets[0]["grads"], *sets[1]["grads"]):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            work(sets[1], sets[1]["grads"])
        torch.cuda.synchronize()
        for c, want in zip(sets, alone):
            assert all(torch.equal(a, b) for a, b in zip(c["grads"], want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [100, 300])
def test_broadcast_inputs(S, dtype):
    """One row of keys for all positions, one sequence for the whole batch, one gradient for every head: stride 0 along any axis."""
    B, H, Hkv, hd = 3, 4, 2, 64
    q, k, v, dout = make(B, H, Hkv, S, S, hd, dtype)
    kw = dict(window=17, prefix_len=3, prefix_open=False)
    for qq, kk, vv, dd in ((q[:1].expand_as(q), k[:, :, :1].expand_as(k), v, dout[:, :1].expand_as(dout)),
                           (q[:, :, :1].expand_as(q), k[:1].expand_as(k), v[:, :1].expand_as(v), dout[:, :, :1].expand_as(dout)),
                           (q, k[:, :1].expand_as(k), v[:, :, :1].expand_as(v), dout[:1].expand_as(dout))):
        res = []
        for args in ((qq, kk, vv, dd), tuple(t.contiguous() for t in (qq, kk, vv, dd))):
            o, lse = run_fwd(*args[:3], None, q_start=0, **kw)
            grads = [torch.full((B, h, S, hd), float("nan"), dtype=dtype, device=DEV) for h in (H, Hkv, Hkv)]
            ops.attn_window_bwd(*args[:3], o, lse, args[3], *grads, torch.empty(B, H, S, device=DEV), **kw)
            res.append((o, lse, *grads))
        assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*res))


# ------------------------------------------------------------------ refusals of the wrappers
def test_wrapper_refusals(monkeypatch):
    q, k, v, _ = make(1, 4, 2, 20, 20, 32, torch.bfloat16)
    o = torch.empty_like(q)
    for bad in (dict(q=q[:, :, :, ::2]), dict(k=k.float()), dict(v=v[:, :, :10]), dict(o=o[:, :1].expand(1, 4, 20, 32)), dict(o=o.float()),
                dict(lse=torch.empty(1, 4, 19, device=DEV)), dict(lens=torch.tensor([20], device=DEV)), dict(q=q.half(), k=k.half(), v=v.half(), o=o.half())):
        args = dict(q=q, k=k, v=v, o=o, window=3)
        args.update(bad)
        with pytest.raises((ValueError, TypeError)):
            ops.attn_window_fwd(**args)
    with pytest.raises(RuntimeError, match="queries"):
        ops.attn_window_fwd(q, k, v, o, window=3, q_start=1)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.attn_window_fwd(q, torch.empty(k.numel() + 8, dtype=k.dtype, device=DEV)[4:4 + k.numel()].view(k.shape), v, o, window=3)
    with pytest.raises(ValueError):
        ops.attn_window_bwd(q, k, v, o, None, o, o, k, v, torch.empty(80, device=DEV), window=3)
    cache = torch.zeros(1, 2, 2, 20, 32, dtype=torch.bfloat16, device=DEV)
    for qq, cc in ((q[:, :, 0, :], cache[:, :, :, ::2]), (q[:, :, 0, :].contiguous(), cache.float()), (q[0:1, 0], cache[:, :1].expand(2, 1, 2, 20, 32))):
        with pytest.raises(ValueError):
            ops.attn_window_decode(qq, cc, torch.empty_like(qq), window=3)
    with pytest.raises(RuntimeError, match="length"):
        ops.attn_window_decode(q[:, :, 0].contiguous(), cache, torch.empty(1, 4, 32, dtype=q.dtype, device=DEV), window=3, length=21)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(RuntimeError, match="current device"):
        ops.attn_window_fwd(q, k, v, o, window=3)


def test_empty_batches_and_no_queries():
    q, k, v, _ = make(2, 2, 2, 6, 6, 32, torch.bfloat16)
    none = q[:, :, :0]
    ops.attn_window_fwd(none, k, v, none.clone(), window=2)
    dk, dv = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    ops.attn_window_bwd(none, k, v, none, torch.empty(2, 2, 0, device=DEV), none, none.clone(), dk, dv, torch.empty(0, device=DEV), window=2)
    assert not dk.any() and not dv.any()
    ops.attn_window_fwd(q[:0], k[:0], v[:0], q[:0].clone(), window=2)
