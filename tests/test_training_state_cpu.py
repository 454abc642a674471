"""The model's dropout state on the CPU: who has one, and what a recomputed forward does."""

import functools

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from model_helpers import TorchKernel, _model_mod, tokens


def build(dropout=0.25):
    m = _model_mod()
    return m.AutoRegressiveModel(97, 2, 128, 2, neighbor_ops="torch", wkv7_dtype=torch.float32,
                                 dropout=dropout).init_random(0.2, torch.Generator().manual_seed(1))


def grads(model, loss):
    model.zero_grad(set_to_none=True)
    loss.backward()
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_whole_forward_is_not_computed_again(reentrant):
    """It would take the next step's masks: refused, where a model that does not drop
    is recomputed as it was."""
    inputs, targets = tokens(2, 32, 97)
    anchor = torch.ones((), requires_grad=True)             # a reentrant checkpoint wants one

    def loss_of(model, one):
        return model(inputs, targets, TorchKernel) * one
    model = build().seed_dropout(3)
    loss = checkpoint(loss_of, model, anchor, use_reentrant=reentrant)
    assert model.dropout_rng.tolist() == [3, 1]
    with pytest.raises(RuntimeError, match="masks"):
        loss.backward()
    assert model.dropout_rng.tolist() == [3, 1]
    plain = build(0.0)
    want = grads(plain, plain(inputs, targets, TorchKernel))
    got = grads(plain, checkpoint(loss_of, plain, anchor, use_reentrant=reentrant))
    assert want.keys() == got.keys() and all(torch.equal(want[n], got[n]) for n in want)


@pytest.mark.parametrize("reentrant", [False, True])
def test_cells_computed_again_take_their_own_masks(reentrant):
    inputs, targets = tokens(2, 32, 97)
    model = build().seed_dropout(3, 7)
    want = grads(model, model(inputs, targets, TorchKernel))
    for cell in model.cells.cells:
        cell.forward = functools.partial(checkpoint, cell.forward, use_reentrant=reentrant)
    model.seed_dropout(3, 7)
    got = grads(model, model(inputs, targets, TorchKernel))
    assert model.dropout_rng.tolist() == [3, 8]
    assert want.keys() == got.keys() and all(torch.equal(want[n], got[n]) for n in want)


def test_a_model_that_does_not_drop_has_no_buffer():
    """Wrappers broadcast a model's buffers before each forward: one that does not drop has
    none, as before there was dropout."""
    model = build(0.0)
    assert not list(model.buffers()) and model.dropout_rng is None
    assert model.seed_dropout(5, 2) is model and not list(model.buffers())
    inputs, targets = tokens(2, 32, 97)
    assert torch.isfinite(model.train()(inputs, targets, TorchKernel))
    assert [n for n, _ in build().named_buffers()] == ["dropout_rng"]
    # one that begins to drop later begins where it was told
    model.dropout = 0.25
    for cell in model.cells.cells:
        cell.dropout = 0.25
    assert torch.equal(model(inputs, targets, TorchKernel), build().seed_dropout(5, 2)(inputs, targets, TorchKernel))
    assert model.dropout_rng.tolist() == [5, 3]
