"""Cases of the window-attention and 4-bit-cache operators, with their plain forms.

``own`` False: ``run`` computes each operator with elementary torch operations in 32 bits.  ``own`` True: ``run`` makes the
calls a user makes (image_caption_amd.ops).  ``exact`` is the definition in 64 bits, written apart from the plain form.

Operators (``op`` of a case):
  fwd     attention under a sliding window with first keys that stay visible: output and log-sum-exp
  bwd     its gradients with respect to q, k and v
  token   one query per sequence (its last position) over a K/V cache, under the same visibility
  append  quantise new K/V rows into a cache of 4 bits per value; returned as the values the rows now stand for
  token4  one query per sequence over such a cache

Visibility of key j to the query at position i of a sequence of length n (i, j < n):
  j <= i and (j < prefix or window == 0 or i - j < window), and with ``open`` also every j < prefix.
A query that sees nothing gives 0 (log-sum-exp -inf).  Query head h reads K/V head h // (H / Hkv); q carries hd^-0.5.

4 bits: per row and group of 32 channels, in 32-bit steps: offset = bf16(min), scale = bf16((max - min) * f32(1/15)),
level = clamp(rint((x - offset) * (1 / scale)), 0, 15) (0 where scale is 0); value = offset + scale * level.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_GROUP = 32


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # the one-block captioning model's step: 32 scored rows of 229 at batch 256, the image rows open to every query
        dict(name="fwd_caption", op="fwd", dtype="bf16", B=256, H=8, Hkv=8, S=229, nq=32, hd=96, window=16, prefix=197, open=True, ragged=False),
        # a long prompt on shared K/V heads with four first tokens kept
        dict(name="fwd_prompt", op="fwd", dtype="bf16", B=2, H=32, Hkv=8, S=8192, nq=8192, hd=128, window=1024, prefix=4, open=False, ragged=False),
        # the 32-bit mode on a padded batch of odd length, three query heads to a K/V head
        dict(name="fwd_ragged_f32", op="fwd", dtype="f32", B=5, H=6, Hkv=2, S=517, nq=517, hd=32, window=100, prefix=3, open=False, ragged=True),
        # a block of a stack: every row of the captioning sequence carries gradients
        dict(name="bwd_caption_stack", op="bwd", dtype="bf16", B=128, H=8, Hkv=8, S=229, nq=229, hd=96, window=16, prefix=197, open=True, ragged=False),
        # training on long documents: the first tokens' keys collect gradients from every query
        dict(name="bwd_long", op="bwd", dtype="bf16", B=1, H=16, Hkv=4, S=8192, nq=8192, hd=128, window=1024, prefix=4, open=False, ragged=False),
        # the 32-bit mode, padded batch
        dict(name="bwd_ragged_f32", op="bwd", dtype="f32", B=3, H=4, Hkv=2, S=333, nq=333, hd=64, window=50, prefix=0, open=False, ragged=True),
        # captioning one image at a time in a batch of 8: launch latency
        dict(name="token_caption", op="token", dtype="bf16", B=8, H=8, Hkv=8, S=229, hd=96, window=16, prefix=197, ragged=False),
        # serving long contexts of different lengths
        dict(name="token_long", op="token", dtype="bf16", B=32, H=32, Hkv=8, S=32768, hd=128, window=8192, prefix=64, ragged=True),
        # filling the cache with the image prefix at batch 256
        dict(name="append_prompt", op="append", dtype="bf16", B=256, Hkv=8, n=198, S=229, hd=96, ragged=False),
        # one new row per sequence, each at its own place
        dict(name="append_token_f32", op="append", dtype="f32", B=64, Hkv=8, n=1, S=1000, hd=128, ragged=True),
        # captioning at batch 256, whole cache visible
        dict(name="token4_caption", op="token4", dtype="bf16", B=256, H=8, Hkv=8, S=229, hd=96, window=0, prefix=0, ragged=False),
        # few sequences with long histories
        dict(name="token4_long", op="token4", dtype="bf16", B=4, H=32, Hkv=8, S=131072, hd=128, window=0, prefix=0, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same ranges; no costlier than the largest listed one."""
    while True:
        op = rng.choice(["fwd", "fwd", "bwd", "bwd", "token", "append", "token4"])
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), B=_log(rng, 1, 256), Hkv=rng.choice([1, 2, 4, 8]),
                 hd=rng.choice([32, 64, 96, 128]), ragged=rng.random() < 0.5)
        if op == "append":
            c["n"] = _log(rng, 1, 4096)
            c["S"] = c["n"] + rng.randrange(0, 600)
        else:
            c["H"] = c["Hkv"] * rng.choice([1, 1, 2, 3, 4, 8])
            c["S"] = _log(rng, 1, 12000 if op in ("fwd", "bwd") else 100000)
            c["window"] = rng.choice([0, _log(rng, 1, max(2, c["S"])), _log(rng, 1, max(2, c["S"]))])
            c["prefix"] = min(c["S"], rng.choice([0, rng.randrange(1, 9), rng.randrange(1, 300)]))
            if op in ("fwd", "bwd"):
                c["open"] = rng.random() < 0.3
                c["nq"] = c["S"] if rng.random() < 0.7 else rng.randrange(1, min(c["S"], 200) + 1)
        w = work(c)
        slow = 8 if c["dtype"] == "f32" else 1
        state = 4 * c["B"] * c["S"] * c["hd"] * (2 * c["Hkv"] + c.get("H", 0))       # bytes in 32 bits
        if w["flops"] * slow <= (5e11 if op in ("fwd", "bwd") else 5e12) and w["bytes"] <= 4e9 and state <= 6e9:
            return c


def _lens(c):
    """Lengths of the sequences: a property of the case, not of the seed."""
    if not c["ragged"]:
        return [c["S"]] * c["B"]
    r = random.Random(c["B"] * 1000003 + c["S"])
    out = [max(1, int(round(c["S"] * (0.25 + 0.75 * r.random())))) for _ in range(c["B"])]
    out[0] = c["S"]
    return out


def _starts(c):
    """Where each sequence's new rows go."""
    if not c["ragged"]:
        return [0] * c["B"]
    r = random.Random(c["B"] * 1000003 + c["S"])
    return [r.randint(0, c["S"] - c["n"]) for _ in range(c["B"])]


def _count_visible(n, positions, window, prefix, is_open):
    """Visible (query, key) pairs for the queries at `positions` (a range) of a sequence of length n."""
    i = np.arange(positions.start, min(positions.stop, n), dtype=np.int64)
    lo = np.zeros_like(i) if window == 0 else np.maximum(0, i - window + 1)
    seen = i + 1 - lo + np.minimum(prefix, lo)
    if is_open:
        seen += np.maximum(0, min(prefix, n) - (i + 1))
    return int(seen.sum())


def work(c):
    e, B, hd, Hkv = _BYTES[c["dtype"]], c["B"], c["hd"], c["Hkv"]
    row4 = hd // 2 + 4 * (hd // _GROUP)                          # bytes of a 4-bit row with its scales and offsets
    if c["op"] == "append":
        rows = B * Hkv * c["n"]
        return {"bytes": 2 * rows * (hd * e + row4), "flops": 2 * rows * hd * 6}
    H, S, lens = c["H"], c["S"], _lens(c)
    if c["op"] in ("token", "token4"):
        pairs = sum(_count_visible(n, range(n - 1, n), c["window"], c["prefix"], False) for n in lens)
        kv = 2 * Hkv * pairs * (hd * e if c["op"] == "token" else row4)
        return {"bytes": kv + 2 * B * H * hd * e, "flops": 4 * H * pairs * hd}
    positions = range(S - c["nq"], S)
    counts = {n: _count_visible(n, positions, c["window"], c["prefix"], c["open"]) for n in set(lens)}
    pairs = sum(counts[n] for n in lens)

    def rows_seen(n):
        if n <= positions.start:
            return 0
        lo = 0 if c["window"] == 0 else max(0, positions.start - c["window"] + 1)
        return n - lo + min(c["prefix"], lo)

    q, lse = B * H * c["nq"] * hd * e, B * H * c["nq"] * 4
    kv, whole = 2 * Hkv * sum(map(rows_seen, lens)) * hd * e, 2 * B * Hkv * S * hd * e
    if c["op"] == "fwd":
        return {"bytes": 2 * q + kv + lse, "flops": 4 * H * pairs * hd}
    return {"bytes": 4 * q + kv + whole + lse, "flops": 10 * H * pairs * hd}


# ---------------------------------------------------------------------------- inputs
def _inputs(c, seed):
    """Rows as a model's projections give them: unit variance, channels with their own offsets, first keys that attract."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, B, Hkv, hd = _DTYPES[c["dtype"]], c["B"], c["Hkv"], c["hd"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    rows = c["n"] if c["op"] == "append" else c["S"]
    shift_k, shift_v = normal(1, Hkv, 1, hd) * 0.5, normal(1, Hkv, 1, hd) * 0.25
    toward = normal(1, Hkv, 1, hd)
    # the layout of a cache [B, Hkv, 2, S, hd]: k and v are views of one tensor
    kv = torch.empty(B, Hkv, 2, rows, hd, dtype=dt, device="cuda")
    for b in range(0, B, max(1, (1 << 27) // max(1, Hkv * rows * hd))):
        part = kv[b:b + max(1, (1 << 27) // max(1, Hkv * rows * hd))]
        part[:, :, 0] = normal(*part[:, :, 0].shape) + shift_k
        part[:, :, 1] = normal(*part[:, :, 1].shape) + shift_v
    x = {"kv": kv, "k": kv[:, :, 0], "v": kv[:, :, 1]}
    if c["op"] == "append":
        return x
    H = c["H"]
    first = min(c["prefix"], 4, rows)
    if first:
        kv[:, :, 0, :first] += (0.5 * toward).to(dt)
    nq = c["nq"] if c["op"] in ("fwd", "bwd") else 1
    q = normal(B, Hkv, H // Hkv, nq, hd) + 0.5 * toward.unsqueeze(2)
    x["q"] = (q * hd ** -0.5).reshape(B, H, nq, hd).to(dt)
    if c["op"] == "bwd":
        x["dout"] = normal(B, H, nq, hd).to(dt)
    return x


def prepare(c, seed):
    """What a program holds before the call: inputs, output buffers, lengths, the filled cache, the forward's output."""
    st = _inputs(c, seed)
    st["c"] = c
    dev, dt, B, Hkv, S, hd = "cuda", _DTYPES[c["dtype"]], c["B"], c["Hkv"], c["S"], c["hd"]
    op = c["op"]
    if op == "append":
        st["starts"] = torch.tensor(_starts(c), dtype=torch.int32, device=dev)
        if own:
            from image_caption_amd import ops
            st["cache"] = ops.kv4_cache(B, Hkv, S, hd, dev)
            st["k_out"] = torch.empty(B, Hkv, c["n"], hd, dtype=torch.float32, device=dev)
            st["v_out"] = torch.empty_like(st["k_out"])
        return st
    lens = _lens(c)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev) if c["ragged"] else None
    st["lens64"] = torch.tensor(lens, dtype=torch.int64, device=dev)
    if op == "token4":
        if own:
            from image_caption_amd import ops
            st["cache"] = ops.kv4_cache(B, Hkv, S, hd, dev)
            ops.kv4_append(st["k"], st["v"], st["cache"], smax=S)
        else:
            st["k4"], st["v4"] = _quantise(st["k"]), _quantise(st["v"])
        for name in ("kv", "k", "v"):
            del st[name]
    if op == "bwd":
        st["o"], st["lse"] = _plain_fwd(c, st["q"], st["k"], st["v"], st["lens64"])
    if own:
        from image_caption_amd import ops
        if op == "bwd":
            st["dq"] = torch.empty_like(st["q"])
            st["dkv"] = torch.empty_like(st["kv"])
            st["delta"] = torch.empty(B, c["H"], c["nq"], dtype=torch.float32, device=dev)
            st["ws"] = torch.empty(ops.attn_window_bwd_workspace(B, c["H"], Hkv, S, c["nq"], hd, window=c["window"], prefix_len=c["prefix"]),
                                   dtype=torch.uint8, device=dev)
        else:
            st["o"] = torch.empty_like(st["q"])
        if op == "fwd":
            st["lse"] = torch.empty(B, c["H"], c["nq"], dtype=torch.float32, device=dev)
            st["ws"] = torch.empty(ops.attn_window_fwd_workspace(B, c["H"], Hkv, S, c["nq"], hd, window=c["window"], prefix_len=c["prefix"]),
                                   dtype=torch.uint8, device=dev)
        if op in ("token", "token4"):
            size = ops.attn_window_decode_workspace if op == "token" else ops.attn_decode_kv4_workspace
            st["ws"] = torch.empty(size(B, c["H"], Hkv, hd, S, window=c["window"], prefix_len=c["prefix"]), dtype=torch.uint8, device=dev)
    return st


# ---------------------------------------------------------------------------- a pass
def run(st):
    c = st["c"]
    return (_own if own else _plain)(c, st)


def _own(c, st):
    from image_caption_amd import ops
    op = c["op"]
    if op == "append":
        ops.kv4_append(st["k"], st["v"], st["cache"], smax=c["S"], starts=st["starts"])
        ops.kv4_unpack(st["cache"], st["k_out"], st["v_out"], smax=c["S"], starts=st["starts"])
        return st["k_out"], st["v_out"]
    mask = dict(window=c["window"], prefix_len=c["prefix"])
    if op == "token":
        q, o = st["q"].squeeze(2), st["o"].squeeze(2)
        ops.attn_window_decode(q, st["kv"], o, length=c["S"], lens=st["lens"], workspace=st["ws"], **mask)
        return st["o"]
    if op == "token4":
        q, o = st["q"].squeeze(2), st["o"].squeeze(2)
        ops.attn_decode_kv4(q, st["cache"], o, smax=c["S"], length=c["S"], lens=st["lens"], workspace=st["ws"], **mask)
        return st["o"]
    mask.update(prefix_open=c["open"], q_start=c["S"] - c["nq"], lens=st["lens"])
    if op == "fwd":
        ops.attn_window_fwd(st["q"], st["k"], st["v"], st["o"], lse=st["lse"], workspace=st["ws"], **mask)
        return st["o"], st["lse"]
    ops.attn_window_bwd(st["q"], st["k"], st["v"], st["o"], st["lse"], st["dout"], st["dq"], st["dkv"][:, :, 0], st["dkv"][:, :, 1],
                        st["delta"], dq_scale=c["hd"] ** -0.5, workspace=st["ws"], **mask)
    return st["dq"], st["dkv"][:, :, 0], st["dkv"][:, :, 1]


# ---------------------------------------------------------------------------- the plain forms
def _quantise(x):
    """(level, scale, offset) of rows [..., hd]."""
    g = x.float().unflatten(-1, (-1, _GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    off = lo.bfloat16().float()
    scale = ((hi - lo) * (1.0 / 15.0)).bfloat16().float()
    inv = torch.where(scale == 0, torch.zeros_like(scale), torch.reciprocal(scale))
    level = torch.clamp(torch.round((g - off) * inv), 0, 15).to(torch.uint8)
    return level, scale, off


def _values(quantised):
    level, scale, off = quantised
    return (off + scale * level.float()).flatten(-2)


def _blocks(c, elements=1 << 28):
    """Ranges of query positions whose scores fit in one block, with the keys any of them can see."""
    S, nq = c["S"], c["nq"]
    step = max(1, min(nq, 1024, elements // max(1, c["B"] * c["H"] * S)))
    for r0 in range(0, nq, step):
        r1 = min(nq, r0 + step)
        i0, i1 = S - nq + r0, S - nq + r1 - 1
        lo = 0 if c["window"] == 0 else max(0, i0 - c["window"] + 1)
        seen = max(min(c["prefix"], lo), 0)
        hi = max(i1 + 1, min(c["prefix"], S) if c["open"] else 0)
        keys = torch.cat([torch.arange(0, seen, device="cuda"), torch.arange(lo, hi, device="cuda")])
        yield r0, r1, torch.arange(i0, i1 + 1, device="cuda"), keys


def _mask(i, j, lens, window, prefix, is_open):
    """[B, 1, 1, queries, keys]"""
    i, j, n = i.view(1, -1, 1), j.view(1, 1, -1), lens.view(-1, 1, 1)
    near = (j < prefix) | (i - j < window) if window else torch.ones_like(i - j, dtype=torch.bool)
    see = (j <= i) & near
    if is_open:
        see = see | (j < prefix)
    return (see & (i < n) & (j < n)).unsqueeze(1).unsqueeze(1)


def _softmax(s, see):
    """Probabilities over the visible keys and the log-sum-exp; zeros where nothing is visible."""
    s = torch.where(see, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    return p / torch.where(z == 0, torch.ones_like(z), z), (m + torch.log(z)).squeeze(-1)


def _plain_fwd(c, q, k, v, lens):
    B, H, nq, hd = q.shape
    G = H // c["Hkv"]
    qf, kf, vf = q.float().view(B, c["Hkv"], G, nq, hd), k.float().unsqueeze(2), v.float().unsqueeze(2)
    o = torch.empty(B, c["Hkv"], G, nq, hd, dtype=torch.float32, device="cuda")
    lse = torch.empty(B, c["Hkv"], G, nq, dtype=torch.float32, device="cuda")
    for r0, r1, i, keys in _blocks(c):
        see = _mask(i, keys, lens, c["window"], c["prefix"], c["open"])
        s = torch.matmul(qf[:, :, :, r0:r1], kf[:, :, :, keys].transpose(-1, -2))
        p, lse[:, :, :, r0:r1] = _softmax(s, see)
        o[:, :, :, r0:r1] = torch.matmul(p, vf[:, :, :, keys])
    return o.view(B, H, nq, hd).to(q.dtype), lse.view(B, H, nq)


def _plain_bwd(c, st):
    q, k, v, dout, lens = st["q"], st["k"], st["v"], st["dout"], st["lens64"]
    B, H, nq, hd = q.shape
    Hkv, G = c["Hkv"], H // c["Hkv"]
    qf, df = q.float().view(B, Hkv, G, nq, hd), dout.float().view(B, Hkv, G, nq, hd)
    kf, vf = k.float().unsqueeze(2), v.float().unsqueeze(2)
    dq = torch.empty_like(qf)
    dk = torch.zeros(B, Hkv, c["S"], hd, dtype=torch.float32, device="cuda")
    dv = torch.zeros_like(dk)
    for r0, r1, i, keys in _blocks(c):
        see = _mask(i, keys, lens, c["window"], c["prefix"], c["open"])
        kb, vb, qb, db = kf[:, :, :, keys], vf[:, :, :, keys], qf[:, :, :, r0:r1], df[:, :, :, r0:r1]
        p, _ = _softmax(torch.matmul(qb, kb.transpose(-1, -2)), see)
        dp = torch.matmul(db, vb.transpose(-1, -2))
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dq[:, :, :, r0:r1] = torch.matmul(ds, kb) * hd ** -0.5
        dk[:, :, keys] += torch.matmul(ds.transpose(-1, -2), qb).sum(2)
        dv[:, :, keys] += torch.matmul(p.transpose(-1, -2), db).sum(2)
    return dq.view(B, H, nq, hd).to(q.dtype), dk.to(q.dtype), dv.to(q.dtype)


def _plain_token(c, q, k, v, lens):
    """k, v in 32 bits [B, Hkv, S, hd]."""
    B, H, _, hd = q.shape
    j = torch.arange(c["S"], device="cuda").view(1, -1)
    i = lens.view(-1, 1) - 1
    see = j <= i
    if c["window"]:
        see = see & ((j < c["prefix"]) | (i - j < c["window"]))
    s = torch.matmul(q.float().view(B, c["Hkv"], H // c["Hkv"], hd), k.transpose(-1, -2))
    p, _ = _softmax(s, see.view(B, 1, 1, -1))
    return torch.matmul(p, v).view(B, H, 1, hd).to(q.dtype)


def _plain(c, st):
    op = c["op"]
    if op == "append":
        return _values(_quantise(st["k"])), _values(_quantise(st["v"]))
    if op == "token":
        return _plain_token(c, st["q"], st["k"].float(), st["v"].float(), st["lens64"])
    if op == "token4":
        return _plain_token(c, st["q"], _values(st["k4"]), _values(st["v4"]), st["lens64"])
    if op == "fwd":
        return _plain_fwd(c, st["q"], st["k"], st["v"], st["lens64"])
    return _plain_bwd(c, st)


# ---------------------------------------------------------------------------- the definition in 64 bits
def _exact_4bit(x):
    """What a row stands for: the levels by the format's 32-bit steps, the value itself in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for t in range(0, x.shape[-1], _GROUP):
        g = x[..., t:t + _GROUP].float()
        lowest = torch.min(g, -1, keepdim=True).values
        span = torch.max(g, -1, keepdim=True).values - lowest
        offset, scale = lowest.to(torch.bfloat16).float(), (span * torch.tensor(1.0 / 15.0, device="cuda")).to(torch.bfloat16).float()
        one = torch.ones_like(scale)
        steps = torch.where(scale > 0, (g - offset) * (one / torch.where(scale > 0, scale, one)), torch.zeros_like(g))
        out[..., t:t + _GROUP] = offset.double() + scale.double() * torch.round(steps).clamp(0, 15).double()
    return out


def exact(c, seed):
    x = _inputs(c, seed)
    op, B, Hkv, S, hd = c["op"], c["B"], c["Hkv"], c["S"], c["hd"]
    if op == "append":
        return _exact_4bit(x["k"]), _exact_4bit(x["v"])
    H, lens = c["H"], _lens(c)
    G = H // Hkv
    if op in ("token", "token4"):
        out = torch.zeros(B, H, 1, hd, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            first = min(c["prefix"], n)
            lo = 0 if c["window"] == 0 else max(0, n - c["window"])
            rows = list(range(0, min(first, lo))) + list(range(lo, n))
            rows = torch.tensor(rows, device="cuda")
            for h in range(Hkv):
                k, v = x["k"][b, h][rows], x["v"][b, h][rows]
                k, v = (_exact_4bit(k), _exact_4bit(v)) if op == "token4" else (k.double(), v.double())
                s = x["q"][b, h * G:(h + 1) * G, 0].double() @ k.t()
                out[b, h * G:(h + 1) * G, 0] = torch.softmax(s, -1) @ v
        return out
    nq = c["nq"]
    pairs = B * H * nq * S
    if pairs > 3e10:                                          # a dense 64-bit score matrix per head: about 20 s here
        return None
    i = torch.arange(S - nq, S, device="cuda")[:, None]
    j = torch.arange(S, device="cuda")[None, :]
    hidden = j > i
    if c["window"]:
        hidden = hidden | ((j >= c["prefix"]) & (j <= i - c["window"]))
    if c["open"]:
        hidden = hidden & (j >= c["prefix"])
    o = torch.zeros(B, H, nq, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, nq), -math.inf, dtype=torch.float64, device="cuda")
    dk = torch.zeros(B, Hkv, S, hd, dtype=torch.float64, device="cuda")
    dv, dq = torch.zeros_like(dk), torch.zeros_like(o)
    for b, n in enumerate(lens):
        live = max(0, n - (S - nq))                           # queries before the sequence's end
        if live == 0:
            continue
        for h in range(H):
            q, k, v = x["q"][b, h, :live].double(), x["k"][b, h // G, :n].double(), x["v"][b, h // G, :n].double()
            s = (q @ k.t()).masked_fill_(hidden[:live, :n], -math.inf)
            norm = torch.logsumexp(s, -1, keepdim=True)
            empty = norm == -math.inf
            p = torch.exp(s - norm.masked_fill(empty, 0.0))
            if op == "fwd":
                o[b, h, :live], lse[b, h, :live] = p @ v, norm[:, 0]
                continue
            d = x["dout"][b, h, :live].double()
            ds = p * (d @ v.t() - (d * (p @ v)).sum(-1, keepdim=True))
            dq[b, h, :live] = ds @ k * hd ** -0.5
            dk[b, h // G, :n] += ds.t() @ q
            dv[b, h // G, :n] += p.t() @ d
    return (o, lse) if op == "fwd" else (dq, dk, dv)
