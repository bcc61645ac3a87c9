"""The 4-bit cache (append, read back) against the format's own steps in torch, and attention over it against plain
attention in 64 bits on the values the cache stands for."""
import math

import pytest
import torch

import window_oracle as wo
from image_caption_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float32]


def quantise(x):
    """(level, scale, offset) by the format's 32-bit steps, the divisions by a tensor on the CPU (IEEE)."""
    g = x.float().cpu().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    off, scale = lo.bfloat16().float(), ((hi - lo) * torch.tensor(1.0 / 15.0)).bfloat16().float()
    inv = torch.where(scale == 0, torch.zeros_like(scale), torch.ones_like(scale) / torch.where(scale == 0, torch.ones_like(scale), scale))
    level = torch.round((g - off) * inv).clamp(0, 15)
    return level.to(DEV), scale.to(DEV), off.to(DEV)


def values(x):
    level, scale, off = quantise(x)
    return (off + scale * level).flatten(-2)


def rows(B, Hkv, n, hd, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    shift = torch.randn(1, Hkv, 1, hd, generator=g, device=DEV)
    k, v = (torch.randn(B, Hkv, n, hd, generator=g, device=DEV) * 2 ** torch.randint(-3, 4, (1, 1, n, 1), generator=g, device=DEV) + shift for _ in range(2))
    return k.to(dtype), v.to(dtype)


def back(cache, smax, hd, Hkv, n=None, **kw):
    B = cache.shape[0]
    k, v = (torch.full((B, Hkv, smax if n is None else n, hd), float("nan"), device=DEV) for _ in range(2))
    ops.kv4_unpack(cache, k, v, smax=smax, **kw)
    return k, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("B,Hkv,n,smax,start", [(1, 1, 1, 1, 0), (2, 3, 33, 40, 5), (3, 2, 64, 128, 64), (1, 2, 200, 229, 29)])
def test_append_and_read_back(B, Hkv, n, smax, start, hd, dtype):
    print(B, Hkv, n, smax, start, hd, dtype, flush=True)
    k, v = rows(B, Hkv, n, hd, dtype)
    k[0, 0, 0, :32] = 1.5                                            # a group of one value: scale 0
    cache = ops.kv4_cache(B, Hkv, smax, hd, DEV)
    ops.kv4_append(k, v, cache, smax=smax, start=start)
    bk, bv = back(cache, smax, hd, Hkv)
    assert torch.equal(bk[:, :, start:start + n], values(k)) and torch.equal(bv[:, :, start:start + n], values(v))
    assert (bk[0, 0, start, :32] == 1.5).all()
    for t in (bk, bv):                                               # the other rows still stand for what a new cache holds
        t[:, :, start:start + n] = 0
        assert not t.any()
    lk = torch.full((B, Hkv, n, hd), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.kv4_unpack(cache, lk, None, smax=smax, start=start)
    assert torch.equal(lk, values(k).bfloat16())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_one_by_one_give_the_same_cache(dtype):
    """Appending piece by piece, in any cut and each sequence at its own place, leaves the bytes of one large append."""
    B, Hkv, hd, smax = 3, 2, 96, 100
    k, v = rows(B, Hkv, smax, hd, dtype)
    whole = ops.kv4_append(k, v, ops.kv4_cache(B, Hkv, smax, hd, DEV), smax=smax)
    cache = ops.kv4_cache(B, Hkv, smax, hd, DEV)
    at = [0] * B
    for step in ([1, 2, 31], [1, 40, 1], [30, 1, 17], [33, 5, 51], [35, 52, 0]):
        n = max(step)
        pk, pv = torch.full((B, Hkv, n, hd), float("nan"), dtype=dtype, device=DEV), torch.full((B, Hkv, n, hd), float("nan"), dtype=dtype, device=DEV)
        for b in range(B):
            pk[b, :, :step[b]], pv[b, :, :step[b]] = k[b, :, at[b]:at[b] + step[b]], v[b, :, at[b]:at[b] + step[b]]
        starts = torch.tensor(at, dtype=torch.int32, device=DEV)
        ops.kv4_append(pk, pv, cache, smax=smax, starts=starts, counts=torch.tensor(step, dtype=torch.int32, device=DEV))
        at = [a + s for a, s in zip(at, step)]
    assert at == [100] * B
    assert torch.equal(cache, whole)


def test_views_of_a_projection_and_outside_rows():
    """k and v as views of a packed [n * B, 3 d] projection; rows that would fall outside the cache are dropped, counts are taken into 0..n."""
    B, Hkv, hd, n, smax = 3, 4, 64, 10, 24
    qkv = torch.randn(n, B, 3, Hkv, hd, device=DEV).to(torch.bfloat16)
    k, v = qkv[:, :, 1].permute(1, 2, 0, 3), qkv[:, :, 2].permute(1, 2, 0, 3)
    cache = ops.kv4_cache(B, Hkv, smax, hd, DEV)
    ops.kv4_append(k, v, cache, smax=smax, starts=torch.tensor([-3, 20, 5], dtype=torch.int32, device=DEV),
                   counts=torch.tensor([10, 99, -1], dtype=torch.int32, device=DEV))
    bk, bv = back(cache, smax, hd, Hkv)
    want_k, want_v = torch.zeros_like(bk), torch.zeros_like(bv)
    for want, src in ((want_k, k), (want_v, v)):
        want[0, :, :7] = values(src[0, :, 3:])
        want[1, :, 20:] = values(src[1, :, :4])
    assert torch.equal(bk, want_k) and torch.equal(bv, want_v)
    part, _ = back(cache, smax, hd, Hkv, n=6, starts=torch.tensor([-2, 22, 0], dtype=torch.int32, device=DEV))
    assert torch.isnan(part[0, :, :2]).all() and torch.equal(part[0, :, 2:], want_k[0, :, :4])
    assert torch.equal(part[1, :, :2], want_k[1, :, 22:]) and torch.isnan(part[1, :, 2:]).all()


def oracle(q, k, v, see):
    """o and its bound; k, v: (level, scale, offset) of [Hkv, n, ...], q [H, hd] of one sequence."""
    h = wo.HALF[q.dtype]
    Hkv, n = k[0].shape[:2]
    G = q.shape[0] // Hkv
    (kl, ksc, kof), (vl, vsc, vof) = ((t.double().repeat_interleave(G, 0) for t in x) for x in (k, v))
    kd, vd = (kof + ksc * kl).flatten(-2), (vof + vsc * vl).flatten(-2)
    qd = q.double()
    s = (kd @ qd[..., None]).squeeze(-1).masked_fill(~see, -math.inf)                     # [H, n]
    p = torch.softmax(s, -1)
    o = (p[..., None] * vd).sum(1)
    # a score is a 32-bit sum of terms up to 2 * 16 scale |q| (levels as 1 + n/16 times 16 q, the surplus subtracted) and offset |q|
    qa = qd.abs().unflatten(-1, (-1, 32)).sum(-1)                                        # [H, groups]
    size = (((48 * ksc + kof.abs()).squeeze(-1) * qa[:, None]).sum(-1)).masked_fill(~see, 0.0).amax(-1)
    ds = (q.shape[1] + 16) * wo.U * size
    rel = 2 * ds + (n + 32) * wo.U + 4 * wo.U * s.masked_fill(~see, 0.0).abs().amax(-1)
    spread = (p[..., None] * (vsc * vl).flatten(-2)).sum(1)                               # what the rounded operand carries
    terms = (p[..., None] * (48 * vsc + vof.abs()).expand_as(vl).flatten(-2)).sum(1)       # what 32-bit sums carry
    tol = h if q.dtype == torch.bfloat16 else 2.0 ** -23                                  # f32: three parts, 24 bits
    mass = (p[..., None] * vd.abs()).sum(1)
    err = spread * tol + terms * (n + 64) * wo.U + (mass + spread) * rel[:, None]
    return o, err + h * (o.abs() + err) + 1e-30


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hkv,hd,smax,length,window,prefix,spec", [
    (1, 1, 1, 32, 1, 1, 0, 0, None),
    (4, 8, 8, 96, 229, 229, 0, 0, None),
    (2, 8, 8, 96, 229, 201, 16, 197, None),
    (3, 8, 2, 128, 300, 257, 0, 0, (257, 0, 1)),
    (2, 6, 2, 64, 300, 300, 40, 4, (300, 77)),
    (1, 16, 2, 64, 3000, 2999, 0, 0, None),                          # eight heads to a K/V head
    (2, 40, 2, 32, 700, 700, 100, 35, (700, 99)),                    # twenty: two groups of heads
    (1, 12, 1, 96, 5000, 4000, 0, 0, None),
    (2, 2, 1, 128, 9000, 9000, 0, 0, (9000, 4500)),                  # cut along the keys
    (9, 2, 2, 128, 64, 64, 5, 0, (64, 63, 33, 32, 31, 6, 5, 4, 1)),
])
def test_attention(B, H, Hkv, hd, smax, length, window, prefix, spec, dtype):
    print(B, H, Hkv, hd, smax, length, dtype, flush=True)
    k, v = rows(B, Hkv, smax, hd, dtype)
    q = (torch.randn(B, H, hd, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV) * hd ** -0.5).to(dtype)
    ns = [length] * B if spec is None else [spec[b % len(spec)] for b in range(B)]
    counts = torch.tensor(ns, dtype=torch.int32, device=DEV)
    cache = torch.full_like(ops.kv4_cache(B, Hkv, smax, hd, DEV), 255)     # rows never written: scales and offsets are NaN
    ops.kv4_append(k, v, cache, smax=smax, counts=counts)
    lens = None if spec is None else counts
    ws = torch.full((ops.attn_decode_kv4_workspace(B, H, Hkv, hd, smax, window=window, prefix_len=prefix),), 255, dtype=torch.uint8, device=DEV)
    qk, qv = quantise(k), quantise(v)
    for w in (ws, None):
        o = torch.full_like(q, float("nan"))
        ops.attn_decode_kv4(q, cache, o, smax=smax, window=window, prefix_len=prefix, length=length, lens=lens, workspace=w)
        for b, n in enumerate(ns):
            if n == 0:
                assert not o[b].any()
                continue
            see = wo.masks(1, n, 1, n - 1, [n], window, prefix, False, DEV)[0, 0]
            want, bound = oracle(q[b], tuple(t[b, :, :n] for t in qk), tuple(t[b, :, :n] for t in qv), see)
            wo.assert_within(o[b], want, bound, f"sequence {b} of {n}, workspace {w is not None}")
        again = torch.empty_like(q)
        ops.attn_decode_kv4(q, cache, again, smax=smax, window=window, prefix_len=prefix, length=length, lens=lens, workspace=w)
        assert torch.equal(o, again)


def test_append_and_attend_in_a_graph():
    """A decoding step as a program captures it: append the new row at each sequence's end, attend; lengths advance on the device."""
    B, H, Hkv, hd, smax = 3, 8, 4, 64, 3000
    k, v = rows(B, Hkv, smax, hd, torch.bfloat16)
    caches = [ops.kv4_cache(B, Hkv, smax, hd, DEV) for _ in range(2)]
    first = [2000, 31, 5]
    for c in caches:
        ops.kv4_append(k, v, c, smax=smax, counts=torch.tensor(first, dtype=torch.int32, device=DEV))
    new_k, new_v = (torch.zeros(B, Hkv, 1, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(B, H, hd, dtype=torch.bfloat16, device=DEV)
    wss = [torch.empty(ops.attn_decode_kv4_workspace(B, H, Hkv, hd, smax), dtype=torch.uint8, device=DEV) for _ in range(2)]
    ends = [torch.tensor(first, dtype=torch.int32, device=DEV) for _ in range(2)]
    outs = [torch.empty_like(q) for _ in range(2)]

    def step(i):
        ops.kv4_append(new_k, new_v, caches[i], smax=smax, starts=ends[i])
        ends[i].add_(1)
        ops.attn_decode_kv4(q, caches[i], outs[i], smax=smax, lens=ends[i], workspace=wss[i])

    step(0)                                     # warm up, then take the state back
    ends[0].copy_(torch.tensor(first, dtype=torch.int32))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    for t in range(5):
        g = torch.Generator(device=DEV).manual_seed(t)
        for x in (new_k, new_v, q):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV) * 0.3)
        graph.replay()
        torch.cuda.synchronize()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(caches[0], caches[1]) and torch.equal(ends[0], ends[1])


def test_offsets_past_four_gigabytes():
    """The last sequence's piece lies past 4 GiB of the cache, and a head's own rows past 2^27."""
    smax, hd, B = 1 << 24, 128, 3                                       # 2.7 GB a piece
    cache = torch.zeros(B, 1, ops.kv4_cache(1, 1, 32, hd, DEV).shape[2] * (smax // 32), dtype=torch.uint8, device=DEV)
    k, v = rows(B, 1, 64, hd, torch.bfloat16)
    ops.kv4_append(k, v, cache, smax=smax, start=smax - 64)
    bk, bv = back(cache, smax, hd, 1, n=64, start=smax - 64)
    assert torch.equal(bk, values(k)) and torch.equal(bv, values(v))
    q = torch.randn(B, 2, hd, device=DEV).to(torch.bfloat16) * hd ** -0.5
    o = torch.empty_like(q)
    ops.attn_decode_kv4(q, cache, o, smax=smax, window=50)
    for b in range(B):
        see = wo.masks(1, 64, 1, 63, [64], 50, 0, False, DEV)[0, 0]
        want, bound = oracle(q[b], tuple(t[b] for t in quantise(k)), tuple(t[b] for t in quantise(v)), see)
        wo.assert_within(o[b], want, bound, "o")


def test_wrapper_refusals(monkeypatch):
    cache = ops.kv4_cache(2, 2, 40, 64, DEV)
    k, v = rows(2, 2, 8, 64, torch.bfloat16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ops.kv4_append(k, v.float(), cache, smax=40), lambda: ops.kv4_append(k, v, cache, smax=100),
                 lambda: ops.kv4_append(k[:, :, :, :32], v, cache, smax=40), lambda: ops.kv4_append(k[:1], v[:1], cache, smax=40),
                 lambda: ops.kv4_append(k, v, cache, smax=40, starts=torch.zeros(2, dtype=torch.int64, device=DEV)),
                 lambda: ops.kv4_append(k, v, cache, smax=40, counts=torch.zeros(3, dtype=torch.int32, device=DEV)),
                 lambda: ops.kv4_unpack(cache, k[:, :1].expand(2, 2, 8, 64), None, smax=40), lambda: ops.kv4_unpack(cache, None, None, smax=40),
                 lambda: ops.attn_decode_kv4(q, cache, q.float(), smax=40), lambda: ops.attn_decode_kv4(q[:, :, ::2], cache, q, smax=40)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="outside a cache"):
        ops.kv4_append(k, v, cache, smax=40, start=33)
    with pytest.raises(RuntimeError, match="length"):
        ops.attn_decode_kv4(q, cache, torch.empty_like(q), smax=40, length=41)
    ops.kv4_append(k[:, :, :0], v[:, :, :0], cache, smax=40)              # nothing to append
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(RuntimeError, match="current device"):
        ops.kv4_append(k, v, cache, smax=40)
