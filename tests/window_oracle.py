"""Plain 64-bit attention under a sliding window, with the elementwise error bounds of a kernel that rounds its
probabilities (and, in the backward, their gradients) once to the inputs' type and keeps everything else in 32 bits."""
import math

import torch

# half a step, relative to the value
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
U = 2.0 ** -24


def visible(S, positions, n, window, prefix, is_open):
    """[queries, S] bool for a sequence of n rows."""
    out = torch.zeros(len(positions), S, dtype=torch.bool)
    for r, i in enumerate(positions):
        for j in range(S):
            if i >= n or j >= n:
                continue
            out[r, j] = (j <= i and (j < prefix or window == 0 or i - j < window)) or (is_open and j < prefix)
    return out


def masks(B, S, nq, q_start, lens, window, prefix, is_open, device):
    """[B, nq, S]; the rule is applied with index arithmetic (`visible` is the same thing spelled out)."""
    i = torch.arange(q_start, q_start + nq, device=device)[:, None]
    j = torch.arange(S, device=device)[None, :]
    see = (j <= i) & ((j < prefix) | torch.tensor(window == 0, device=device) | (i - j < window))
    if is_open:
        see = see | (j < prefix)
    n = torch.tensor(lens, device=device)[:, None, None]
    return see[None] & (i[None] < n) & (j[None] < n)


def forward(q, k, v, see, keep=None):
    """(o, lse, bound of o, bound of lse).  keep: dropout factors [B, H, nq, S] or None."""
    B, H, nq, hd = q.shape
    G = H // k.shape[1]
    n = torch.where(see.any(-1).unsqueeze(1), 1.0, 0.0)                    # rows that see something
    dead_k = ~see.any(1)[:, None, :, None]                                 # rows of K / V nobody sees may hold anything
    qd = torch.where((n > 0).unsqueeze(-1), q.double(), torch.zeros((), dtype=torch.float64, device=q.device))
    kd = k.double().masked_fill(dead_k, 0.0).repeat_interleave(G, 1)
    vd = v.double().masked_fill(dead_k, 0.0).repeat_interleave(G, 1)
    s = (qd @ kd.transpose(-1, -2)).masked_fill(~see[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(see[:, None], torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None]), torch.zeros((), dtype=torch.float64, device=q.device))
    pk = p if keep is None else p * keep
    o = pk @ vd
    size = (qd.abs() @ kd.abs().transpose(-1, -2)).masked_fill(~see[:, None], 0.0).amax(-1)      # of a score's terms
    h = HALF[q.dtype]
    mass = pk @ vd.abs()
    nvis = see.sum(-1)[:, None].double()
    # a score is a 32-bit sum of hd exact (bf16) or rounded (f32) products; its error moves every probability, relatively, by
    # as much; exp2 and its argument add a few units, the sums over the keys nvis units
    ds = (hd + 2) * U * size
    rel = 2 * ds + (nvis + 24 + 2 * size) * U
    tol_p = h if q.dtype == torch.bfloat16 else 0.0                       # probabilities rounded to be an operand
    bound = mass * (tol_p + rel[..., None]) + h * (o.abs() + mass * tol_p) + 1e-30
    return o, lse, bound, ds + (nvis + 24 + lse.masked_fill(lse == -math.inf, 0.0).abs()) * U + 2 * U * size


def backward(q, k, v, o, lse, dout, see, dq_scale, keep=None):
    """Gradients from the given o and lse, and their bounds: ((dq, bound), (dk, bound), (dv, bound))."""
    B, H, nq, hd = q.shape
    Hkv = k.shape[1]
    G = H // Hkv
    live = see.any(-1)[:, None, :, None]
    dead_k = ~see.any(1)[:, None, :, None]
    z = torch.zeros((), dtype=torch.float64, device=q.device)
    qd, dd, od = (torch.where(live, t.double(), z) for t in (q, dout, o))
    kd, vd = (t.double().masked_fill(dead_k, 0.0).repeat_interleave(G, 1) for t in (k, v))
    s = qd @ kd.transpose(-1, -2)
    p = torch.where(see[:, None], torch.exp(s - lse.double().masked_fill(lse == -math.inf, 0.0)[..., None]), z)
    dp = dd @ vd.transpose(-1, -2)
    f = 1.0 if keep is None else keep
    delta = (dd * od).sum(-1, keepdim=True)
    ds = p * (f * dp - delta)
    pk = p * f

    def group(x):
        return x.unflatten(1, (Hkv, G)).sum(2)

    dq, dk, dv = dq_scale * (ds @ kd), group(ds.transpose(-1, -2) @ qd), group(pk.transpose(-1, -2) @ dd)
    h = HALF[q.dtype]
    tol = h if q.dtype == torch.bfloat16 else 0.0
    size = torch.where(see[:, None], qd.abs() @ kd.abs().transpose(-1, -2), z)
    rel = ((2 * hd + 32) + 4 * size) * U + (hd + 2) * U * size                # of a recomputed probability
    err_p = p * (tol + rel)
    mag = f * (dd.abs() @ vd.abs().transpose(-1, -2)) + (dd * od).abs().sum(-1, keepdim=True)
    err_ds = ds.abs() * tol + p * mag * ((hd + 8) * U + rel) * (1 + tol)
    nsum = max(nq * G, k.shape[2]) * U                                       # a 32-bit sum over rows or keys
    bq = dq_scale * (err_ds @ kd.abs() + nsum * (ds.abs() @ kd.abs()))
    bk = group(err_ds.transpose(-1, -2) @ qd.abs() + nsum * (ds.abs().transpose(-1, -2) @ qd.abs()))
    bv = group((f * err_p).transpose(-1, -2) @ dd.abs() + nsum * (pk.transpose(-1, -2) @ dd.abs()))
    return tuple((g, b + h * (g.abs() + b) + 1e-30) for g, b in ((dq, bq), (dk, bk), (dv, bv)))


def assert_within(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    worst = (off / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} times the bound (largest error {off.max().item():.3g})"
