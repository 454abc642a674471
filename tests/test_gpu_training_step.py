"""A training step that keeps neither its logits nor its dropout masks: the model with
``loss="pieces"`` and ``dropout``, on the kernels, against the same model with its
logits and with the masks in plain torch, in eager steps and in a captured one.

Bars: float32 as the model's other tests have them (loss 1e-5 relative, gradients
1e-4 relative L2). Under bf16 autocast the logits of the other path are rounded to
bf16: by up to 2^-8 of their size, here below 4, so a probability by 2^-6 of itself and
the loss by 2^-6; a gradient by 2^-6 and by three more roundings of 2^-8 on its way."""

import pytest
import torch

from conftest import announce, load_pkg, rel_l2
from model_helpers import TorchKernel, _model_mod, _wkv7_mod, loss_and_grads, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(seed=0, vocab=97, std=0.2, **kw):
    m = _model_mod()
    torch.manual_seed(seed)
    model = m.AutoRegressiveModel(vocab, 2, 128, 2, 64, **kw)
    return model.init_random(std, torch.Generator().manual_seed(seed)).to(DEV)


def compare(a, b, loss_tol, grad_tol):
    (l0, g0), (l1, g1) = a, b
    assert abs(l1 - l0) <= loss_tol * abs(l0), (l0, l1)
    assert g0.keys() == g1.keys()
    errs = {n: rel_l2(g1[n].float().cpu().numpy(), g0[n].float().cpu().numpy()) for n in g0}
    worst = max(errs, key=errs.get)
    assert errs[worst] <= grad_tol, (worst, errs[worst])


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("vocab", [97, 1000])
def test_pieces_against_logits(vocab, autocast):
    announce("model loss in pieces", vocab, autocast)
    wk = _wkv7_mod()
    dtype = torch.bfloat16 if autocast else torch.float32
    inputs, targets = (t.to(DEV) for t in tokens(2, 64, vocab))
    got = []
    for loss in ("logits", "pieces"):
        model = build(vocab=vocab, wkv7_dtype=dtype, loss=loss)
        with torch.autocast(DEV, dtype=torch.bfloat16, enabled=autocast):
            got.append(loss_and_grads(model, wk.KernelPretrain, inputs, targets))
    compare(*got, *((2.0 ** -6, 2.0 ** -6 + 3 * 2.0 ** -8) if autocast else (1e-5, 1e-4)))


def test_ignored_targets():
    announce("model loss in pieces, ignored targets")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(3, 32, 97))
    model = build(wkv7_dtype=torch.float32, loss="pieces")
    full = load_pkg().lm_loss
    targets[:, :20] = full.IGNORE_INDEX
    targets[2] = full.IGNORE_INDEX                          # a sequence of which nothing is learned
    l0, g0 = loss_and_grads(model, wk.KernelPretrain, inputs, targets)
    # the mean over the others: they alone, of the model's own logits
    other = build(wkv7_dtype=torch.float32)
    hidden = {}
    other.layer_norm_for_unembed.register_forward_hook(lambda m, i, o: hidden.update(x=o))
    other(inputs, targets.clamp(min=0), wk.KernelPretrain)
    z = other.unembed(hidden["x"].reshape(-1, 128)).double()
    keep = targets.reshape(-1) >= 0
    want = torch.nn.functional.cross_entropy(z[keep], targets.reshape(-1)[keep])
    assert abs(l0 - float(want.detach())) <= 1e-5 * float(want.detach())
    targets[:] = full.IGNORE_INDEX
    l1, g1 = loss_and_grads(model, wk.KernelPretrain, inputs, targets)
    assert l1 == 0.0 and all(not g.any() for g in g1.values())


def test_dropout_against_plain_torch():
    """The same masks, drawn by the kernel and in plain torch."""
    announce("model dropout")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 64, 97))
    got = []
    for ops in ("torch", "hip"):
        model = build(wkv7_dtype=torch.float32, neighbor_ops=ops, dropout=0.2).seed_dropout(99, 5)
        got.append(loss_and_grads(model, wk.KernelPretrain, inputs, targets))
        assert model.dropout_rng.tolist() == [99, 6]
    compare(*got, 1e-5, 1e-4)
    model = build(wkv7_dtype=torch.float32)
    l2, _ = loss_and_grads(model, wk.KernelPretrain, inputs, targets)
    assert l2 != got[1][0]
    dropped = build(wkv7_dtype=torch.float32, dropout=0.2).eval()
    l3, _ = loss_and_grads(dropped, wk.KernelPretrain, inputs, targets)
    assert l3 == l2


def test_train_steps():
    """Steps of the model's own training path, twice alike."""
    announce("train steps with dropout and the loss in pieces")
    m = _model_mod()
    inputs, targets = (t.to(DEV) for t in tokens(4, 64, 500))
    ends = []
    for _ in range(2):
        model = build(vocab=500, std=0.05, dropout=0.1, loss="pieces").seed_dropout(3)
        opt = m.make_optimizer(model)
        losses = [float(m.train_step(model, opt, inputs, targets, check_faults=True)) for _ in range(3)]
        assert model.dropout_rng.tolist() == [3, 3]
        ends.append((losses, [p.detach().clone() for p in model.parameters()]))
    assert ends[0][0] == ends[1][0] and len(set(ends[0][0])) == 3
    assert all(torch.isfinite(p).all() and torch.equal(p, q) for p, q in zip(ends[0][1], ends[1][1]))


def test_captured_step():
    """Forward and backward in a graph: each replay counts the step up and draws
    other masks, as the eager step does from the same state."""
    announce("captured step with dropout and the loss in pieces")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 64, 300))
    model = build(vocab=300, dropout=0.2, loss="pieces").seed_dropout(8)
    params = list(model.parameters())

    def step():
        with torch.autocast(DEV, dtype=torch.bfloat16, cache_enabled=False):
            loss = model(inputs, targets, wk.KernelPretrain)
        return (loss.detach(), *torch.autograd.grad(loss, params, allow_unused=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = set()
    for i in range(4):
        model.seed_dropout(8, 20 + i)
        graph.replay()
        torch.cuda.synchronize()
        assert model.dropout_rng.tolist() == [8, 21 + i]
        got = [None if o is None else o.clone() for o in out]
        model.seed_dropout(8, 20 + i)
        want = step()
        for a, b in zip(got, want):
            assert (a is None and b is None) or torch.equal(a, b)
        seen.add(float(got[0]))
    assert len(seen) == 4


def test_quantized_model_forms_its_logits():
    announce("4-bit model with the loss in pieces")
    pkg = load_pkg()
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 32, 160))
    got = []
    for loss in ("logits", "pieces"):
        model = build(vocab=160, loss=loss).eval()
        pkg.w4.quantize_model(model, group_size=64)
        with torch.no_grad(), torch.autocast(DEV, dtype=torch.bfloat16):
            got.append(model(inputs, targets, wk.KernelPretrain))
    assert torch.equal(*got)


def test_unembedding_with_a_bias_forms_its_logits():
    announce("unembedding with a bias, with the loss in pieces")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 32, 160))
    got = []
    for loss in ("logits", "pieces"):
        model = build(vocab=160, loss=loss)
        plain = model.unembed
        model.unembed = torch.nn.Linear(plain.in_features, 160, device=DEV)
        with torch.no_grad():
            model.unembed.weight.copy_(plain.weight)
            model.unembed.bias.copy_(torch.linspace(-2, 2, 160))
            with torch.autocast(DEV, dtype=torch.bfloat16):
                got.append(model(inputs, targets, wk.KernelPretrain))
    assert torch.equal(*got)
