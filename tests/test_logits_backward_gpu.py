"""Backward of the reference's forward (all-rows logits) with an input gradient, and through a stack of blocks."""
import pytest
import torch

import helpers
from helpers import TINY
from oracle import ref_cpu
from image_caption_amd.engine import block_key
from test_parity_gpu import DEV, F32, check_grads, make_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nb", [1, 2, 3])
def test_input_and_parameter_gradients(nb):
    sh = TINY
    sds = [helpers.make_state_dict(sh, seed=970 + i) for i in range(nb)]
    full = dict(sds[0])
    for i in range(1, nb):
        for k in ref_cpu.BLOCK_KEYS:
            full[block_key(i, k, nb)] = sds[i][k]
    img, sos, cap, _ = helpers.make_embeddings(sh, seed=61)
    x = ref_cpu.concat_prefix(img, sos, cap)
    model = make_model(sh, full, F32, n_blocks=nb, mask_mode="prefix_causal", activation="gelu")
    model.prefix_len = sh.P
    model.train()
    xin = x.to(DEV).requires_grad_(True)
    out = model(xin)
    up = torch.randn(out.shape, generator=torch.Generator().manual_seed(2))
    out.backward(up.to(DEV))
    leaf = [{k: sds[i][k].clone().requires_grad_(True) for k in ref_cpu.BLOCK_KEYS} for i in range(nb)]
    head = {k: sds[0][k].clone().requires_grad_(True) for k in ref_cpu.PARAM_KEYS[12:]}
    xc = x.clone().requires_grad_(True)
    ref_cpu.decoder_forward(xc, leaf, head, sh.nhead, mask_mode="prefix_causal", prefix_len=sh.P, activation="gelu").backward(up)
    assert (xin.grad.cpu() - xc.grad).abs().max().item() <= 1e-4 * xc.grad.abs().max().item()
    grads = {k: head[k].grad for k in head}
    for i in range(nb):
        for k in ref_cpu.BLOCK_KEYS:
            grads[block_key(i, k, nb)] = leaf[i][k].grad
    check_grads(model, grads, F32, activation="gelu")
