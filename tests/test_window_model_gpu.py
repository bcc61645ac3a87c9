"""The captioning model under window masks and with a 4-bit K/V cache: training against the oracle's autograd, greedy
decoding against full recomputation, and the 4-bit cache against the same loop with quantised rows in torch."""
import pytest
import torch

import helpers
from helpers import TINY
from oracle import ref_cpu
from image_caption_amd import ops
from image_caption_amd.decoder import CaptionTrainer
from image_caption_amd.engine import KernelTimer, block_key
from test_kv4_gpu import values
from test_parity_gpu import BF16, DEV, F32, check_grads, make_model

pytestmark = pytest.mark.gpu


def stacked(nb, seed, head_gain=1.0):
    sds = [helpers.make_state_dict(TINY, seed=seed + i, head_gain=head_gain) for i in range(nb)]
    full = dict(sds[0])
    for i in range(1, nb):
        for k in ref_cpu.BLOCK_KEYS:
            full[block_key(i, k, nb)] = sds[i][k]
    return sds, full


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mode,window,nb,scored", [("prefix_window", 3, 1, True), ("prefix_window", 5, 2, True), ("window", 4, 2, True), ("window", 1, 1, False)])
def test_training_vs_oracle(dtype, mode, window, nb, scored):
    sh = TINY
    sds, full = stacked(nb, 900)
    img, sos, cap, labels = helpers.make_embeddings(sh, seed=606)
    model = make_model(sh, full, dtype, n_blocks=nb, mask_mode=mode, window=window, activation="gelu", scored_rows_only=scored)
    model.train()
    loss, correct = model.caption_loss((img.to(DEV), sos.to(DEV), cap.to(DEV)), labels.to(DEV))
    loss.backward()
    leaf = [{k: sds[i][k].clone().requires_grad_(True) for k in ref_cpu.BLOCK_KEYS} for i in range(nb)]
    head = {k: sds[0][k].clone().requires_grad_(True) for k in ref_cpu.PARAM_KEYS[12:]}
    x = ref_cpu.concat_prefix(img, sos, cap)
    lg = ref_cpu.decoder_forward(x, leaf, head, sh.nhead, mask_mode=f"{mode}:{window}", prefix_len=sh.P, activation="gelu")
    lo, co, _ = ref_cpu.caption_loss(lg, labels, sh.L)
    lo.backward()
    assert abs(loss.item() - lo.item()) <= (1e-5 if dtype == F32 else 1e-2) * lo.item()
    if dtype == F32:
        assert int(correct.item()) == co
    grads = {k: head[k].grad for k in head}
    for i in range(nb):
        for k in ref_cpu.BLOCK_KEYS:
            grads[block_key(i, k, nb)] = leaf[i][k].grad
    check_grads(model, grads, dtype, activation="gelu", gated_bar=0.998)
    # the reference's forward, whose backward returns an input gradient
    model.prefix_len = sh.P
    xin = x.to(DEV).requires_grad_(True)
    out = model(xin)
    assert (out.cpu() - lg).abs().max().item() <= (1e-4 if dtype == F32 else 0.05) * lg.abs().max().item()
    if dtype == F32:
        xc = x.clone().requires_grad_(True)
        up = torch.randn(lg.shape, generator=torch.Generator().manual_seed(1))
        ref_cpu.decoder_forward(xc, leaf, head, sh.nhead, mask_mode=f"{mode}:{window}", prefix_len=sh.P, activation="gelu").backward(up)
        out.backward(up.to(DEV))
        assert (xin.grad.cpu() - xc.grad).abs().max().item() <= 1e-4 * xc.grad.abs().max().item()


def test_a_window_that_hides_nothing_is_prefix_causal():
    """window >= S (and no window) give the prefix-causal model, dropout masks included: the same hash indexes the same probabilities."""
    sh = TINY
    sds, full = stacked(2, 910)
    img, sos, cap, labels = (t.to(DEV) for t in helpers.make_embeddings(sh, seed=607))
    grads = []
    for opt in (dict(mask_mode="prefix_causal"), dict(mask_mode="prefix_window", window=1000), dict(mask_mode="prefix_window")):
        model = make_model(sh, full, F32, dropout=0.2, n_blocks=2, **opt)
        model.train()
        loss, _ = model.caption_loss((img, sos, cap), labels)
        loss.backward()
        grads.append({k: p.grad for k, p in model.named_parameters()})
    for other in grads[1:]:
        for k, g in grads[0].items():
            assert (g - other[k]).abs().max().item() <= 1e-4 * g.abs().max().item() + 1e-9, k


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_trainer_step_runs_and_repeats(dtype):
    """Two trainers from the same start take the same steps, bit for bit (no atomics in the window kernels), ragged last batch included."""
    sh = TINY
    _, full = stacked(2, 920)
    runs = []
    for _ in range(2):
        model = make_model(sh, full, dtype, dropout=0.1, n_blocks=2, mask_mode="prefix_window", window=4, activation="gelu")
        tr = CaptionTrainer(model, lr=1e-3, weight_decay=0.0)
        model.train()
        img, sos, cap, labels = (t.to(DEV) for t in helpers.make_embeddings(sh, seed=608))
        for n in (3, 2, 3):
            loss, _, rows = tr.step((img[:n].contiguous(), sos[:n].contiguous(), cap[:n].contiguous()), labels[:n].contiguous())
        assert torch.isfinite(loss).all()
        runs.append(tr.store.w.clone())
    same = runs[0] == runs[1]
    for key, shape, off in tr.store.layout:                    # (the framework sums linear1.bias with atomics in some epilogues)
        if not key.endswith("linear1.bias"):
            assert same[off:off + torch.Size(shape).numel()].all() or (runs[0] - runs[1])[off:off + torch.Size(shape).numel()].abs().max() < 1e-5, key


@pytest.mark.parametrize("mode,window,nb", [("prefix_window", 3, 2), ("window", 4, 1)])
def test_greedy_under_a_window_matches_full_recomputation(mode, window, nb):
    sh = TINY
    sds, full = stacked(nb, 940, head_gain=4.0)
    img, sos, _, _ = helpers.make_embeddings(sh, seed=1515)
    emb = helpers.make_token_table(sh, seed=1616)
    pos = 0.3 * torch.randn(sh.S, sh.d, generator=torch.Generator().manual_seed(6))
    model = make_model(sh, full, F32, n_blocks=nb, mask_mode=mode, window=window, activation="gelu")
    V = sh.vocab
    args = (img.to(DEV), sos.to(DEV), emb.to(DEV))
    ids, mg = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    blocks = [{k: sds[i][k] for k in ref_cpu.BLOCK_KEYS} for i in range(nb)]
    head = {k: sds[0][k] for k in ref_cpu.PARAM_KEYS[12:]}
    with torch.no_grad():
        want, margins = ref_cpu.greedy_decode(img, sos, emb, blocks, head, sh.nhead, sh.L, V - 3, V - 2, V - 1, mask_mode=f"{mode}:{window}",
                                              activation="gelu", pos=pos, return_margins=True)
    safe = (margins > 1e-3).cumprod(dim=1).bool()
    assert safe.float().mean().item() > 0.5
    assert torch.equal(ids.cpu()[safe], want[safe])
    model.engine.timer = KernelTimer()                         # launch by launch: the same kernels
    ids2, mg2 = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    assert torch.equal(ids, ids2) and torch.equal(mg, mg2)


def greedy_quantised(sh, blocks, head, img, sos, emb, pos, mode, window, max_len):
    """The loop of DecoderEngine.generate in torch (32 bits, CPU): the prompt attends to its own rows, the cache keeps quantised ones."""
    B, P, d = img.shape
    H, hd, V = sh.nhead, d // sh.nhead, sh.vocab
    x = torch.cat([img, sos, emb[V - 3].expand(B, 1, d)], 1).transpose(0, 1) + pos[:P + 2, None]
    mask = ref_cpu.caption_mask(P + 2, mode if not window else f"{mode}:{window}", P)
    caches = []

    def heads(t):
        return t.reshape(t.shape[0], B, H, hd).permute(1, 2, 0, 3)

    def block(x, p, attend):
        h = ref_cpu.layer_norm(x, p["norm1.weight"], p["norm1.bias"])
        q, k, v = (heads(t) for t in (h @ p["self_attn.in_proj_weight"].t() + p["self_attn.in_proj_bias"]).split(d, -1))
        o = attend(q * hd ** -0.5, k, v).permute(2, 0, 1, 3).reshape(x.shape)
        x = x + o @ p["self_attn.out_proj.weight"].t() + p["self_attn.out_proj.bias"]
        h = ref_cpu.layer_norm(x, p["norm2.weight"], p["norm2.bias"])
        return x + torch.nn.functional.gelu(h @ p["linear1.weight"].t() + p["linear1.bias"]) @ p["linear2.weight"].t() + p["linear2.bias"]

    def prompt(q, k, v):
        caches.append([values(k).cpu(), values(v).cpu()])
        return torch.softmax(q @ k.transpose(-1, -2) + mask, -1) @ v

    for p in blocks:
        x = block(x, p, prompt)
    out, margins, done = torch.full((B, max_len), V - 1), torch.zeros(B, max_len), torch.zeros(B, dtype=torch.bool)
    for t in range(max_len):
        top = (x[-1] @ head["output_projection.weight"].t() + head["output_projection.bias"]).topk(2, -1)
        margins[:, t] = top.values[:, 0] - top.values[:, 1]
        tok = torch.where(done, torch.full_like(top.indices[:, 0], V - 1), top.indices[:, 0])
        out[:, t] = tok
        done |= tok == V - 2
        s = P + 2 + t
        if t + 1 == max_len:
            break
        x = (emb[tok] + pos[s])[None]
        seen = torch.arange(s + 1)
        hide = (seen >= P) & (s - seen >= window) if window else torch.zeros(s + 1, dtype=torch.bool)
        for i, p in enumerate(blocks):
            def step(q, k, v, i=i):
                caches[i] = [torch.cat([c, values(n).cpu()], 2) for c, n in zip(caches[i], (k, v))]
                return torch.softmax((q @ caches[i][0].transpose(-1, -2)).masked_fill(hide, float("-inf")), -1) @ caches[i][1]
            x = block(x, p, step)
    return out, margins


@pytest.mark.parametrize("mode,window,nb", [("reference", 0, 1), ("prefix_causal", 0, 2), ("prefix_window", 3, 2)])
def test_greedy_over_a_4_bit_cache(mode, window, nb):
    sh = TINY
    sds, full = stacked(nb, 950, head_gain=4.0)
    img, sos, _, _ = helpers.make_embeddings(sh, seed=1717)
    emb = helpers.make_token_table(sh, seed=1818)
    pos = 0.3 * torch.randn(sh.S, sh.d, generator=torch.Generator().manual_seed(8))
    blocks = [{k: sds[i][k] for k in ref_cpu.BLOCK_KEYS} for i in range(nb)]
    head = {k: sds[0][k] for k in ref_cpu.PARAM_KEYS[12:]}
    with torch.no_grad():
        want, margins = greedy_quantised(sh, blocks, head, img, sos, emb, pos, mode, window, sh.L)
    model = make_model(sh, full, F32, n_blocks=nb, mask_mode=mode, window=window, activation="gelu", kv_cache_bits=4)
    args = (img.to(DEV), sos.to(DEV), emb.to(DEV))
    ids, mg = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    # the two compute the rows before quantising with different 32-bit sums: a level at a rounding border may differ by one,
    # which moves a logit by far less than this margin
    safe = (margins > 0.05).cumprod(dim=1).bool()
    assert safe.float().mean().item() > 0.4
    assert torch.equal(ids.cpu()[safe], want[safe])
    model.engine.timer = KernelTimer()
    ids2, mg2 = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    assert torch.equal(ids, ids2) and torch.equal(mg, mg2)
    # bf16: the composed step and the launches one by one agree, twice in a row over the same (now used) cache
    model = make_model(sh, full, BF16, n_blocks=nb, mask_mode=mode, window=window, activation="gelu", kv_cache_bits=4)
    a = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    b = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    model.engine.timer = KernelTimer()
    c = model.generate(*args, max_len=sh.L, pos=pos.to(DEV), return_margins=True)
    for other in (b, c):
        assert torch.equal(a[0], other[0]) and torch.equal(a[1], other[1])


def test_append_then_attend_then_window_over_one_cache():
    """The operators as a serving loop runs them: a windowed prompt, its rows into the cache, tokens appended and attended to."""
    B, H, Hkv, hd, P, T, window, keep = 2, 4, 2, 64, 90, 6, 40, 3
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(B, n, P + T, hd, generator=g, device=DEV).to(BF16) for n in (H, Hkv, Hkv))
    q = q * hd ** -0.5
    smax = P + T
    cache = ops.kv4_cache(B, Hkv, smax, hd, DEV)
    plain = torch.zeros(B, Hkv, 2, smax, hd, dtype=BF16, device=DEV)
    o = torch.empty_like(q)
    ops.attn_window_fwd(q[:, :, :P], k[:, :, :P], v[:, :, :P], o[:, :, :P], window=window, prefix_len=keep)
    ops.kv4_append(k[:, :, :P], v[:, :, :P], cache, smax=smax)
    o4 = o.clone()
    # the exact cache holds what the 4-bit one stands for, so the two single-token paths must agree to their rounding
    for t in range(T):
        s = P + t
        ops.kv4_append(k[:, :, s:s + 1], v[:, :, s:s + 1], cache, smax=smax, start=s)
        kk, vv = (torch.empty(B, Hkv, smax, hd, device=DEV) for _ in range(2))
        ops.kv4_unpack(cache, kk, vv, smax=smax)
        plain32 = torch.stack([kk, vv], 2).contiguous()
        a = torch.empty(B, H, hd, device=DEV)
        ops.attn_window_decode(q[:, :, s].float().contiguous(), plain32, a, window=window, prefix_len=keep, length=s + 1)
        b = torch.empty(B, H, hd, device=DEV)
        ops.attn_decode_kv4(q[:, :, s].float().contiguous(), cache, b, smax=smax, window=window, prefix_len=keep, length=s + 1)
        assert (a - b).abs().max().item() <= 1e-5 * a.abs().max().item() + 1e-5
    del plain, o4


def test_decode_step_with_a_cache_description_refuses():
    import ctypes as C

    from image_caption_amd import _lib
    lib = _lib.load()
    kv = _lib.DecodeKv(1, 4, 2)
    dd = _lib.DecodeDesc()
    assert lib.capdec_decode_step_kv(C.byref(dd), kv, None) == -1
    base, with_kv = lib.capdec_decode_step_workspace(4, 64, 128, 100, _lib.F32), lib.capdec_decode_step_kv_workspace(4, 64, 2, 128, 100, _lib.F32, 16, kv)
    assert with_kv >= base + 2 * 4 * 64 * 4
    assert lib.capdec_decode_step_kv_workspace(4, 64, 3, 128, 100, _lib.F32, 16, kv) == 0
