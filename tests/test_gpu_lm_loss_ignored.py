"""The loss of logits with rows that are not learned (include/rwkv_lm_loss_ignore.h),
and a model with ``loss="pieces"`` whose logits are formed all the same (4-bit weights, an
unembedding with a bias), against float64 formulas.

Bars: a row's loss within 1e-5 of the larger of its log-sum-exp and its target's logit
(fp32 sums of up to 65536 terms and an exponential within 2^-20 of its value); a logit's
gradient within 2^-16 of its probability's share (the rounded log-sum-exp and argument, each
below 2^5, are 2^-19 off, the exponential 2^-20) and half a step of its type; the
model's float32 as its other tests have it (loss 1e-5 relative, gradients 1e-4 relative
L2)."""

import pytest
import torch

from conftest import announce, load_pkg
from model_helpers import _wkv7_mod, loss_and_grads, tokens
from test_gpu_training_step import build, compare

pytestmark = pytest.mark.gpu
pkg = load_pkg()
ll = pkg.lm_loss
DEV = "cuda"
BOTH = [torch.bfloat16, torch.float32]


def check(z, t, g, num_tokens, ignore):
    a = z.detach().requires_grad_()
    loss = ll.cross_entropy_l2wrap_rows(a, t, num_tokens, ignore)
    dz, = torch.autograd.grad(loss, a, g)
    dead = (t == ignore)[:, None]
    z64 = torch.where(dead, 0.0, z.double())
    at = torch.where(dead, 0, t.long()[:, None])
    lse, zt = torch.logsumexp(z64, 1, keepdim=True), z64.gather(1, at)
    want = torch.where(dead, 0.0, lse - zt)[:, 0]
    assert ((loss.double() - want).abs() <= 1e-5 * (lse.abs() + zt.abs())[:, 0]).all()
    assert (loss[dead[:, 0]] == 0).all()
    s = 1e-4 / num_tokens if num_tokens else 0.0
    gd = torch.where(dead, 0.0, g.double()[:, None])
    m, top = z64.max(1, keepdim=True)
    share = gd * torch.exp(z64 - lse)
    d = share.scatter_add(1, at, -gd).scatter_add(1, top, torch.where(dead, 0.0, s * m))
    miss = (dz.double() - d).abs()
    assert (miss <= share.abs() * 2.0 ** -16 + d.abs() * (torch.finfo(z.dtype).eps / 2 + 2.0 ** -22) + 1e-44).all()
    assert not dz[dead[:, 0]].any()
    return loss, dz


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (7, 97), (33, 512), (40, 1003), (300, 4099), (9, 65536), (600, 65529)])
def test_ignored_rows(rows, vocab, dtype):
    announce("loss of logits, ignored rows", rows, vocab, dtype)
    gen = torch.Generator(device=DEV).manual_seed(rows)
    z = (3.0 * torch.randn(rows, vocab, generator=gen, device=DEV)).to(dtype)
    full = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    g = torch.rand(rows, generator=gen, device=DEV) + 0.1
    r = torch.arange(rows, device=DEV)
    for dead in (r % 3 == 1, r > 0, r < 0, r >= 0):
        t = full.masked_fill(dead, -100)
        y = z.clone()
        for k, bad in enumerate((float("nan"), float("inf"), -float("inf"))):
            y[dead & (r % 3 == k)] = bad                   # whatever the logits there are
        check(y, t, g, rows, -100)
        check(y, t, g, 0, -100)
    for word in (0, vocab - 1):                             # a word of the vocabulary
        check(z, torch.where(r % 2 == 0, word, full), g, rows, word)


@pytest.mark.parametrize("dtype", BOTH)
def test_without_an_ignored_target_nothing_changes(dtype):
    announce("loss of logits, nothing ignored", dtype)
    for rows, vocab in ((5, 300), (64, 1000), (128, 65536)):
        gen = torch.Generator(device=DEV).manual_seed(vocab)
        z = torch.randn(rows, vocab, generator=gen, device=DEV).to(dtype)
        t = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
        t[0] = -100
        g = torch.rand(rows, generator=gen, device=DEV)
        got = []
        for ignore in (None, -7):
            a = z.detach().requires_grad_()
            loss = ll.cross_entropy_l2wrap_rows(a, t, rows, ignore)
            got.append((loss.detach(), torch.autograd.grad(loss, a, g)[0]))
        assert got[0][0][0].isnan() and torch.equal(got[0][0][1:], got[1][0][1:]) and got[1][0][0].isnan()
        assert torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32])
def test_the_mean(dtype):
    announce("loss of logits, the mean", dtype)
    gen = torch.Generator(device=DEV).manual_seed(1)
    z = torch.randn(90, 120 if dtype == torch.int8 else 200, generator=gen, device=DEV)
    t = torch.randint(0, z.shape[1], (90,), generator=gen, device=DEV)
    t[::2] = 156 if dtype == torch.uint8 else -100           # 156 in eight bits without a sign is not -100
    a = z.detach().requires_grad_()
    mean = ll.cross_entropy_l2wrap(a, t.to(dtype), -100)
    mean.backward()
    rows = ll.cross_entropy_l2wrap_rows(z, t, 90, -100)
    kept = int((t != -100).sum())
    assert torch.equal(mean.detach(), rows.sum() / kept)
    check(z, t, torch.full((90,), 1.0 / kept, device=DEV), 90, -100)
    none = ll.cross_entropy_l2wrap(z.requires_grad_(), torch.full_like(t, -100), -100)
    none.backward()
    assert float(none.detach()) == 0.0 and not z.grad.any()


def test_in_a_graph():
    """A replay ignores the rows that its targets say."""
    announce("loss of logits, ignored rows, graph")
    gen = torch.Generator(device=DEV).manual_seed(2)
    z = torch.randn(200, 1000, generator=gen, device=DEV)
    full = torch.randint(0, 1000, (200,), generator=gen, device=DEV)
    t, a = full.clone(), z.detach().clone().requires_grad_()

    def step():
        loss = ll.cross_entropy_l2wrap(a, t, -100)
        return loss.detach(), torch.autograd.grad(loss, a)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in (1, 2, 5, 200):
        t.copy_(full.masked_fill(torch.arange(200, device=DEV) % k != 0, -100))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def some_ignored(t):
    t = t.clone()
    t[:, :11] = ll.IGNORE_INDEX
    t[1] = ll.IGNORE_INDEX
    return t


def test_unembedding_with_a_bias():
    """The rows of the prompts leave nothing in the loss or in any gradient."""
    announce("unembedding with a bias, ignored targets")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(3, 32, 160))
    targets = some_ignored(targets)
    models = []
    for loss in ("pieces", "logits"):
        model = build(vocab=160, wkv7_dtype=torch.float32, loss=loss)
        plain = model.unembed
        model.unembed = torch.nn.Linear(plain.in_features, 160, device=DEV)
        with torch.no_grad():
            model.unembed.weight.copy_(plain.weight)
            model.unembed.bias.copy_(torch.linspace(-2, 2, 160))
        models.append(model)
    got = loss_and_grads(models[0], wk.KernelPretrain, inputs, targets)
    # the other's logits, by the formula
    hidden = {}
    models[1].layer_norm_for_unembed.register_forward_hook(lambda m, i, o: hidden.update(x=o))
    models[1](inputs, targets.clamp(min=0), wk.KernelPretrain)
    z = models[1].unembed(hidden["x"].reshape(-1, 128)).double()
    t = targets.reshape(-1)
    keep = t != ll.IGNORE_INDEX
    want = torch.nn.functional.cross_entropy(z[keep], t[keep])
    m, top = z.detach().max(1, keepdim=True)
    wrap = (m * keep[:, None] * (1e-4 / t.numel()) * z.gather(1, top)).sum()     # all rows count as tokens
    models[1].zero_grad(set_to_none=True)
    (want + wrap).backward()
    grads = {n: p.grad for n, p in models[1].named_parameters() if p.grad is not None}
    compare((float(want.detach()), grads), got, 1e-5, 1e-4)
    none, g = loss_and_grads(models[0], wk.KernelPretrain, inputs, torch.full_like(targets, ll.IGNORE_INDEX))
    assert none == 0.0 and all(not v.any() for v in g.values())


def test_quantized_unembedding():
    announce("4-bit model, ignored targets")
    wk = _wkv7_mod()
    inputs, targets = (t.to(DEV) for t in tokens(2, 32, 160))
    ignored = some_ignored(targets)
    model = build(vocab=160, loss="pieces").eval()
    pkg.w4.quantize_model(model, group_size=64)
    seen = {}
    model.unembed.register_forward_hook(lambda m, i, o: seen.update(z=o))
    with torch.no_grad(), torch.autocast(DEV, dtype=torch.bfloat16):
        got = model(inputs, ignored, wk.KernelPretrain)
    z, t = seen["z"].reshape(-1, 160).double(), ignored.reshape(-1)
    want = torch.nn.functional.cross_entropy(z, t, ignore_index=ll.IGNORE_INDEX)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
