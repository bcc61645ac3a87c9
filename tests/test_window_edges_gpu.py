"""Window attention at the ends of what its description allows."""
import pytest
import torch

import window_oracle as wo
from image_caption_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_backward_of_few_queries_before_very_many_keys():
    """128 heads on one K/V head over 2^24 positions, two queries at the front: (keys behind the first query) * heads is 2^31."""
    H, S, nq, hd = 128, 1 << 24, 2, 32
    print(H, S, nq, hd, flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    q = (torch.randn(1, H, nq, hd, generator=g, device=DEV) * hd ** -0.5).bfloat16()
    dout = torch.randn(1, H, nq, hd, generator=g, device=DEV).bfloat16()
    k, v = (torch.zeros(1, 1, S, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    for t in (k, v):
        t[:, :, :nq] = torch.randn(1, 1, nq, hd, generator=g, device=DEV).bfloat16()
    kw = dict(window=8, prefix_len=0)
    o, lse, delta = torch.empty_like(q), torch.empty(1, H, nq, device=DEV), torch.empty(1, H, nq, device=DEV)
    ops.attn_window_fwd(q, k, v, o, lse=lse, **kw)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, delta, **kw)
    see = wo.masks(1, nq, nq, 0, [nq], 8, 0, False, DEV)
    oracle = wo.backward(q, k[:, :, :nq], v[:, :, :nq], o, lse, dout, see, 1.0)
    for got, (want, bound), what in zip((dq, dk[:, :, :nq], dv[:, :, :nq]), oracle, ("dq", "dk", "dv")):
        wo.assert_within(got, want, bound, what)
    assert not dk[:, :, nq:].any() and not dv[:, :, nq:].any()


def run(q, k, v, dout, bwd=True, lens=None, **kw):
    B, H, nq, hd = q.shape
    o, lse = torch.full_like(q, float("nan")), torch.full((B, H, nq), float("nan"), device=DEV)
    size = ops.attn_window_fwd_workspace(B, H, k.shape[1], k.shape[2], nq, hd, window=kw["window"], prefix_len=kw["prefix_len"])
    ops.attn_window_fwd(q, k, v, o, lse=lse, lens=lens, workspace=torch.empty(size, dtype=torch.uint8, device=DEV), **kw)
    if not bwd:
        return o, lse
    dq, dk, dv = torch.full_like(q, float("nan")), torch.full(k.shape, float("nan"), dtype=k.dtype, device=DEV), torch.full(v.shape, float("nan"), dtype=v.dtype, device=DEV)
    ops.attn_window_bwd(q, k, v, o, lse, dout, dq, dk, dv, torch.empty(B, H, nq, device=DEV), lens=lens, **kw)
    return o, lse, dq, dk, dv


# B, H, Hkv, S, nq, hd, window, prefix, open: the one-kernel backward; dQ of many rows and of few; a padded batch of each
COMMON = [
    (40, 8, 8, 229, 229, 96, 16, 197, True),
    (64, 8, 4, 256, 100, 64, 0, 0, False),
    (4, 16, 4, 900, 900, 128, 200, 4, False),
    (8, 16, 4, 1100, 1100, 64, 0, 0, False),
    (16, 8, 4, 700, 700, 32, 90, 130, False),
    (8, 12, 4, 600, 600, 96, 300, 0, False),
    (2, 8, 2, 500, 12, 128, 0, 0, False),
    (3, 4, 4, 400, 50, 64, 100, 3, False),
    (4, 8, 8, 229, 229, 128, 16, 197, True),
    (2, 4, 4, 9000, 100, 32, 0, 0, False),                           # long rows: dQ is a small mean over many keys
    (1, 4, 2, 10000, 64, 128, 0, 4, False),
    (1, 8, 2, 5000, 300, 64, 3000, 4, False),
]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("offset", [0.0, 0.6, 2.0, 8.0, 50.0])
@pytest.mark.parametrize("case", COMMON)
def test_bf16_gradients_where_keys_have_a_common_part(case, offset, ragged):
    """A common part of a sequence's keys changes no probability, so dQ (a row of dS sums to 0) and dK do not depend on it either.
    Against gradients in 64 bits with an output that was never rounded.  Of a gradient's size in the mean square: its own rounding and
    dS's 0.0017 each (a uniform error of at most half a step, 2^-8 at the lower end of a binade), so half a step, 2^-8 = 0.0039,
    has room for both.  On top of it, by the formula itself, comes what the rounding of the saved output does to delta: an error e_i = dO_i (bf16(o_i) - o_i)
    moves dQ_i by e_i sum_j P_ij K_j and dK_j by sum_i P_ij e_i Q_i.  It is formed here in 64 bits, with K's mean taken out: a
    long row's dQ is a mean over its keys that shrinks like 1 / sqrt(n), while sum_j P_ij K_j stays (9000 keys: 0.0042)."""
    B, H, Hkv, S, nq, hd, window, prefix, is_open = case
    print(case, offset, ragged, flush=True)
    g = torch.Generator(device=DEV).manual_seed(17)

    def normal(*s):
        return torch.randn(*s, generator=g, device=DEV)

    q, dout = (normal(B, H, nq, hd) * hd ** -0.5).bfloat16(), normal(B, H, nq, hd).bfloat16()
    k = (normal(B, Hkv, S, hd) + offset * normal(1, Hkv, 1, hd)).bfloat16()
    v = (normal(B, Hkv, S, hd) + 0.25 * normal(1, Hkv, 1, hd)).bfloat16()
    ns = [S - 61 * (b % 4) if ragged else S for b in range(B)]
    lens = torch.tensor(ns, dtype=torch.int32, device=DEV) if ragged else None
    _, _, dq, dk, dv = run(q, k, v, dout, lens=lens, window=window, prefix_len=prefix, prefix_open=is_open, q_start=S - nq)
    see = wo.masks(B, S, nq, S - nq, ns, window, prefix, is_open, DEV)
    off, size, saved = (torch.zeros(3, dtype=torch.float64, device=DEV) for _ in range(3))
    for b in range(0, B, 4):
        part = slice(b, min(B, b + 4))
        exact_o, exact_lse, _, _ = wo.forward(q[part], k[part], v[part], see[part])
        wants = wo.backward(q[part], k[part], v[part], exact_o, exact_lse, dout[part], see[part], 1.0)
        for i, (got, (want, _)) in enumerate(zip((dq[part], dk[part], dv[part]), wants)):
            off[i] += (got.double() - want).square().sum()
            size[i] += want.square().sum()
        G, seen, rows = H // Hkv, see[part].any(1)[:, None, :, None], see[part].any(-1)[:, None, :, None]
        kd = k[part].double().masked_fill(~seen, 0.0)
        centred = (kd - kd.sum(2, keepdim=True) / seen.sum(2, keepdim=True)).masked_fill(~seen, 0.0).repeat_interleave(G, 1)
        qd = q[part].double()
        p = torch.exp(qd @ kd.repeat_interleave(G, 1).transpose(-1, -2) - exact_lse.masked_fill(exact_lse == -float("inf"), 0.0)[..., None]) * see[part][:, None]
        e = (dout[part].double() * (exact_o.bfloat16().double() - exact_o)).sum(-1, keepdim=True).masked_fill(~rows, 0.0)
        saved[0] += (e * (p @ centred)).square().sum()
        saved[1] += ((p * e).transpose(-1, -2) @ qd).unflatten(1, (Hkv, G)).sum(2).square().sum()
    rel, limit = (off / size).sqrt().tolist(), (2.0 ** -8 + (saved / size).sqrt()).tolist()
    print("dq, dk, dv off by", rel, "of", limit, flush=True)
    assert all(x <= y for x, y in zip(rel, limit)), (rel, limit)


def test_keys_that_are_all_alike_get_no_dq():
    """Every key the same: no query can tell them apart, and dQ is what the roundings leave of 0, not a multiple of the key."""
    for B, S, hd in ((2, 200, 64), (1, 600, 128)):
        g = torch.Generator(device=DEV).manual_seed(3)
        q, dout, v = (torch.randn(B, 4, S, hd, generator=g, device=DEV).bfloat16() for _ in range(3))
        k = (100 * torch.randn(B, 4, 1, hd, generator=g, device=DEV)).bfloat16().expand(B, 4, S, hd)
        _, _, dq, _, _ = run(q * hd ** -0.5, k, v, dout, window=0, prefix_len=0)
        # rows that see 32 keys of their tile or more; the sum of 32-bit products left over, of values up to 100 * hd
        assert dq[:, :, 128:].abs().max().item() <= 2.0 ** -10


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [32, 96, 128])
@pytest.mark.parametrize("S,nq,window,prefix", [(150, 150, 40, 3), (150, 9, 0, 0), (260, 260, 100, 130)])
def test_key_rows_far_apart(S, nq, window, prefix, hd, dtype):
    """K and V rows almost 32 MiB apart, as a projection of thousands of sequences has them: the bits of the same rows packed."""
    B, H, Hkv = 1, 4, 2
    print(S, nq, window, prefix, hd, dtype, flush=True)
    size = torch.empty(0, dtype=dtype).element_size()
    row = (1 << 25) // size - 16 // size                                  # elements: 16 bytes below 32 MiB
    buf = torch.empty((S - 1) * row + 2 * Hkv * hd, dtype=dtype, device=DEV)
    far = buf.as_strided((B, 2, Hkv, S, hd), (0, Hkv * hd, hd, row, 1))
    g = torch.Generator(device=DEV).manual_seed(9)
    near = torch.randn(B, 2, Hkv, S, hd, generator=g, device=DEV).to(dtype)
    far.copy_(near)
    q = (torch.randn(B, H, nq, hd, generator=g, device=DEV) * hd ** -0.5).to(dtype)
    dout = torch.randn(B, H, nq, hd, generator=g, device=DEV).to(dtype)
    kw = dict(window=window, prefix_len=prefix, q_start=S - nq)
    for a, b in zip(run(q, far[:, 0], far[:, 1], dout, **kw), run(q, near[:, 0], near[:, 1], dout, **kw)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_key_rows_too_far_apart_are_refused():
    q = torch.zeros(1, 1, 2, 32, dtype=torch.bfloat16, device=DEV)
    buf = torch.empty((1 << 24) + 32, dtype=torch.bfloat16, device=DEV)
    k = buf.as_strided((1, 1, 2, 32), (0, 0, 1 << 24, 1))
    with pytest.raises(RuntimeError, match="too far apart"):
        ops.attn_window_fwd(q, k, k, torch.empty_like(q), window=0)


@pytest.mark.parametrize("bits", [0, 4])
def test_engine_refuses_a_batch_before_it_starts(bits):
    from helpers import TINY
    import helpers
    from test_parity_gpu import BF16, make_model
    sh = TINY
    model = make_model(sh, helpers.make_state_dict(sh, seed=5), BF16, mask_mode="prefix_window", window=3, kv_cache_bits=bits)
    B = (1 << 25) // (3 * sh.d * 2) + 1
    img, sos, cap = (torch.zeros(1, n, sh.d, device=DEV).expand(B, n, sh.d) for n in (sh.P, 1, sh.L))
    with pytest.raises(ValueError, match=f"at most {B - 1} sequences"):
        model.caption_loss((img, sos, cap), torch.zeros(1, sh.L, dtype=torch.int64, device=DEV).expand(B, sh.L))
    if bits:
        with pytest.raises(ValueError, match=f"at most {B - 1} sequences"):
            model.generate(img, sos, helpers.make_token_table(sh, seed=6).to(DEV), max_len=2)
    assert not model.engine._bufs                                         # nothing was allocated for it


def test_one_kernel_backward_needs_no_workspace():
    """Few short heads in bf16: the sizes' workspace is for f32 (partial sums); the one-kernel form neither needs nor touches it."""
    B, H, S, hd, kw = 1, 3, 256, 64, dict(window=9, prefix_len=5)
    assert ops.attn_window_bwd_workspace(B, H, H, S, S, hd, **kw) > 0
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v, dout = (torch.randn(B, H, S, hd, generator=g, device=DEV) for _ in range(4))
    for dtype in (torch.bfloat16, torch.float32):
        args = [t.to(dtype) for t in (q, k, v)]
        o, lse = run(*args, None, bwd=False, **kw)
        res = []
        for ws in (torch.empty(0, dtype=torch.uint8, device=DEV), None):
            grads = [torch.full_like(t, float("nan")) for t in args]
            call = lambda: ops.attn_window_bwd(*args, o, lse, dout.to(dtype), *grads, torch.empty(B, H, S, device=DEV), workspace=ws, **kw)
            if ws is not None and dtype == torch.float32:
                with pytest.raises(RuntimeError, match="workspace 0 bytes"):
                    call()
            else:
                call()
                res.append(grads)
        if dtype == torch.bfloat16:
            assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(*res))


@pytest.mark.parametrize("dropout", [0.0, 0.1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mode,window,nb", [("prefix_window", 4, 2), ("window", 3, 1)])
def test_model_gradients_repeat_bit_for_bit(mode, window, nb, dtype, dropout):
    """The window kernels have no atomics, so every gradient that passes through them has the same bits each time; only linear1.bias, whose
    column sums some of the framework's products form with atomics, and which feeds nothing else, may differ in its last ones."""
    import helpers
    from helpers import TINY
    from oracle import ref_cpu
    from image_caption_amd.engine import block_key
    from test_parity_gpu import make_model
    sds = [helpers.make_state_dict(TINY, seed=930 + i) for i in range(nb)]
    full = dict(sds[0])
    for i in range(1, nb):
        for key in ref_cpu.BLOCK_KEYS:
            full[block_key(i, key, nb)] = sds[i][key]
    img, sos, cap, labels = (t.to(DEV) for t in helpers.make_embeddings(TINY, seed=609))
    runs = []
    for _ in range(3):
        model = make_model(TINY, full, dtype, dropout=dropout, n_blocks=nb, mask_mode=mode, window=window, activation="gelu")
        model.train()
        loss, correct = model.caption_loss((img, sos, cap), labels)
        loss.backward()
        runs.append({"loss": loss.detach(), "correct": correct, **{key: p.grad for key, p in model.named_parameters()}})
    for other in runs[1:]:
        for key, t in runs[0].items():
            assert torch.isfinite(t).all(), key
            if key.endswith("linear1.bias"):
                # sums of the same numbers in another order: a few units of the column's absolute sum, which 2^-16 of the largest covers
                assert (t - other[key]).abs().max() <= 2.0 ** -16 * t.abs().max() + 1e-12, key
            else:
                assert torch.equal(t, other[key]), key


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,S,nq,hd,window,prefix", [
    (40, 8, 8, 100, 48, 64, 20, 3),                                  # 33..64 rows and a tile for every CU: the waves split the rows in bf16, the keys in f32
    (75, 8, 4, 900, 24, 32, 0, 0),                                   # the same with two heads to a K/V head, and few enough to cut along the keys
    (35, 8, 8, 229, 33, 96, 16, 197),
    (33, 8, 8, 300, 64, 128, 40, 0),
    (70, 4, 4, 130, 32, 64, 0, 0),
])
def test_rows_between_the_two_shapes_of_workgroup(B, H, Hkv, S, nq, hd, window, prefix, dtype):
    print(B, H, Hkv, S, nq, hd, window, prefix, dtype, flush=True)
    g = torch.Generator(device=DEV).manual_seed(23)
    q, dout = (torch.randn(B, H, nq, hd, generator=g, device=DEV) * hd ** -0.5).to(dtype), torch.randn(B, H, nq, hd, generator=g, device=DEV).to(dtype)
    k, v = (torch.randn(B, Hkv, S, hd, generator=g, device=DEV).to(dtype) for _ in range(2))
    ns = [S - 17 * (b % 5) for b in range(B)]
    lens = torch.tensor(ns, dtype=torch.int32, device=DEV)
    kw = dict(window=window, prefix_len=prefix, q_start=S - nq)
    see = wo.masks(B, S, nq, S - nq, ns, window, prefix, False, DEV)
    want, want_lse, bound, _ = wo.forward(q, k, v, see)
    o, lse, *grads = run(q, k, v, dout, lens=lens, **kw)
    wo.assert_within(o, want, bound, "o")
    whole = torch.full_like(q, float("nan"))
    ops.attn_window_fwd(q, k, v, whole, lens=lens, **kw)
    wo.assert_within(whole, want, bound, "o in one piece")
    for got, (w, bd), what in zip(grads, wo.backward(q, k, v, o, lse, dout, see, 1.0), ("dq", "dk", "dv")):
        wo.assert_within(got, w, bd, what)


# B, H, Hkv, S, nq, hd, window, prefix, open, lens: a sequence of one, window 1 alone, a first row that sees itself, prefixes that add a key or do not
ALONE = [
    (3, 8, 2, 1, 1, 32, 1, 1, True, None),
    (2, 2, 2, 1, 1, 64, 0, 0, False, None),
    (300, 1, 1, 1, 1, 96, 0, 4, True, None),
    (2, 8, 4, 200, 200, 64, 1, 0, False, None),
    (2, 8, 4, 300, 300, 128, 1, 0, False, (300, 131)),
    (40, 8, 8, 140, 50, 64, 1, 0, True, None),
    (2, 4, 2, 300, 300, 32, 20, 3, False, None),
    (2, 4, 4, 90, 90, 96, 5, 1, True, None),
    (2, 4, 4, 90, 90, 128, 1, 1, True, None),
    (3, 4, 4, 150, 150, 64, 30, 5, True, (150, 1, 2)),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", ALONE)
def test_a_query_that_sees_one_key_has_no_gradient_for_its_score(case, dtype):
    """Its probability is 1 whatever the score: its dQ and its share of dK are 0, not what two sums of the same numbers leave."""
    B, H, Hkv, S, nq, hd, window, prefix, is_open, spec = case
    print(case, dtype, flush=True)
    g = torch.Generator(device=DEV).manual_seed(29)
    q, dout = (torch.randn(B, H, nq, hd, generator=g, device=DEV) * hd ** -0.5).to(dtype), torch.randn(B, H, nq, hd, generator=g, device=DEV).to(dtype)
    k, v = (torch.randn(B, Hkv, S, hd, generator=g, device=DEV).to(dtype) for _ in range(2))
    ns = [S] * B if spec is None else list(spec)
    lens = None if spec is None else torch.tensor(ns, dtype=torch.int32, device=DEV)
    kw = dict(window=window, prefix_len=prefix, prefix_open=is_open, q_start=S - nq)
    see = wo.masks(B, S, nq, S - nq, ns, window, prefix, is_open, DEV)
    alone = see.sum(-1) == 1                                              # [B, nq]
    assert alone.any()
    o, lse, dq, dk, dv = run(q, k, v, dout, lens=lens, **kw)
    assert not dq[alone[:, None].expand(B, H, nq)].any()
    others = (see & ~alone[:, :, None]).any(1)                            # [B, S]: keys that some other query sees
    assert not dk[~others[:, None].expand(B, Hkv, S)].any()
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()
    for got, (want, bound), what in zip((dq, dk, dv), wo.backward(q, k, v, o, lse, dout, see, 1.0), ("dq", "dk", "dv")):
        wo.assert_within(got, want, bound, what)


@pytest.mark.parametrize("B,H,Hkv,S,nq,hd", [(64, 8, 8, 300, 40, 64), (65, 16, 8, 200, 20, 32), (63, 8, 8, 700, 64, 128), (32, 16, 8, 1500, 30, 96)])
def test_rows_between_the_shapes_with_two_workgroups_for_a_cu(B, H, Hkv, S, nq, hd):
    """33..64 rows in bf16 on either side of 512 K/V heads."""
    print(B, H, Hkv, S, nq, hd, flush=True)
    g = torch.Generator(device=DEV).manual_seed(31)
    q, dout = ((torch.randn(B, H, nq, hd, generator=g, device=DEV) * x).bfloat16() for x in (hd ** -0.5, 1.0))
    k, v = (torch.randn(B, Hkv, S, hd, generator=g, device=DEV).bfloat16() for _ in range(2))
    kw = dict(window=0, prefix_len=0, q_start=S - nq)
    o, lse, *grads = run(q, k, v, dout, **kw)
    for b in range(0, B, 16):
        part = slice(b, min(B, b + 16))
        see = wo.masks(part.stop - part.start, S, nq, S - nq, [S] * (part.stop - part.start), 0, 0, False, DEV)
        want, _, bound, _ = wo.forward(q[part], k[part], v[part], see)
        wo.assert_within(o[part], want, bound, "o")
        for got, (w, bd), what in zip(grads, wo.backward(q[part], k[part], v[part], o[part], lse[part], dout[part], see, 1.0), ("dq", "dk", "dv")):
            wo.assert_within(got[part], w, bd, what)
