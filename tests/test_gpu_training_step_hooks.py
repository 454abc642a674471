"""A model whose loss comes straight from its hidden states and an unembedding that does
something when it is called: its logits are formed, as by the model that forms them always.

Bars: float32 as the model's other tests have them (loss 1e-5 relative, gradients 1e-4
relative L2)."""

import pytest
import torch
from torch.nn.utils import prune

from conftest import announce
from model_helpers import _wkv7_mod, loss_and_grads, tokens
from test_gpu_training_step import DEV, build, compare

pytestmark = pytest.mark.gpu


def test_pruned_unembedding():
    """Its weight is made anew by a hook before each call: two steps, the second from weights
    that the first one changed."""
    announce("pruned unembedding, loss in pieces")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 32, 97))
    got = []
    for loss in ("logits", "pieces"):
        model = build(wkv7_dtype=torch.float32, loss=loss)
        prune.l1_unstructured(model.unembed, "weight", amount=0.4)
        steps = []
        for _ in range(2):
            steps.append(loss_and_grads(model, wk.KernelPretrain, inputs, targets))
            with torch.no_grad():
                for p in model.parameters():
                    if p.grad is not None:
                        p.sub_(0.1 * p.grad)
        got.append(steps)
    assert "unembed.weight_orig" in got[1][0][1]
    for a, b in zip(*got):
        compare(a, b, 1e-5, 1e-4)


def test_hooks_run():
    announce("hooks on the unembedding, loss in pieces")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 32, 97))
    want = loss_and_grads(build(wkv7_dtype=torch.float32), wk.KernelPretrain, inputs, targets)
    for register in ("register_forward_pre_hook", "register_forward_hook", "register_full_backward_hook",
                     "register_full_backward_pre_hook"):
        model, ran = build(wkv7_dtype=torch.float32, loss="pieces"), []
        handle = getattr(model.unembed, register)(lambda *a: ran.append(1))
        compare(want, loss_and_grads(model, wk.KernelPretrain, inputs, targets), 1e-5, 1e-4)
        assert ran
        handle.remove()
        ran.clear()
        compare(want, loss_and_grads(model, wk.KernelPretrain, inputs, targets), 1e-5, 1e-4)
        assert not ran
