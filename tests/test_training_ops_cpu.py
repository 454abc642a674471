"""The C ABI of the loss from hidden states and of the dropout without a GPU (what
the headers declare is exported, bad calls are refused on the host), the dropout's
generator against published numbers, and the model's dropout on the CPU."""

import os

import pytest
import torch

from conftest import REPO, load_pkg
from model_helpers import TorchKernel, _model_mod, tokens
from test_abi_cpu import declared_functions

FAKE = 1 << 24        # a pointer that is never followed


@pytest.fixture(scope="module")
def native():
    n = load_pkg()._native
    n.lib()
    return n


@pytest.mark.parametrize("header,exports", [("rwkv_linear_loss.h", "LINEAR_LOSS_EXPORTS"),
                                            ("rwkv_dropout.h", "DROPOUT_EXPORTS")])
def test_exports(native, header, exports):
    declared = declared_functions(os.path.join(REPO, "include", header), "rwkv_")
    assert set(declared) == set(getattr(native, exports))
    for name in declared:
        assert hasattr(native.lib(), name) and name in native._SIGNATURES


def test_linear_loss_workspaces(native):
    lib = native.lib()
    both = (lib.rwkv_linear_loss_forward_workspace_bytes, lib.rwkv_linear_loss_backward_workspace_bytes)
    for size in both:
        assert size(0, 8, 8, 0) == 0 and size(1, 1, 1, 1) > 0
        for bad in ((-1, 8, 8, 0), (1, 0, 8, 0), (1, 8, 0, 0), (1, 8, 8, 2), ((1 << 22) + 1, 8, 8, 0),
                    (8, (1 << 22) + 1, 8, 0), (8, 8, (1 << 16) + 1, 0)):
            assert size(*bad) == -1, bad
    forward, backward = both
    # no logits: a small part of [rows, vocab] for the forward, at most half a GiB of their gradient
    assert forward(8192, 65536, 768, 1) < 8192 * 65536 * 2 // 20
    assert backward(8192, 65536, 768, 1) < (512 << 20) + (8192 * 768 * 4) * 16 + (64 << 20)
    assert backward(1 << 16, 65536, 768, 1) < (512 << 20) + (1 << 16) * 768 * 4 * 16 + (256 << 20)
    for rows, vocab, c in ((1, 1, 1), (300, 1000, 100), (8192, 65536, 768), (1 << 22, 1 << 22, 64), (5, 70001, 1 << 16)):
        for dtype in (0, 1):
            assert forward(rows, vocab, c, dtype) > 0 and backward(rows, vocab, c, dtype) > 0


def test_linear_loss_refusals(native):
    lib = native.lib()
    x, w, t, lo, ls, mx, am, ws, g, dx, dw = (FAKE * i for i in range(1, 12))
    rows, vocab, c = 40, 300, 64
    need_f = lib.rwkv_linear_loss_forward_workspace_bytes(rows, vocab, c, 0)
    need_b = lib.rwkv_linear_loss_backward_workspace_bytes(rows, vocab, c, 0)
    assert max(need_f, need_b) < FAKE

    def forward(x=x, w=w, t=t, rows=rows, vocab=vocab, c=c, dtype=0, loss=lo, lse=ls, mx=mx, am=am, ws=ws, n=need_f):
        return lib.rwkv_linear_loss_forward(x, w, t, rows, vocab, c, dtype, -100, loss, lse, mx, am, ws, n, None)

    def backward(x=x, w=w, t=t, rows=rows, vocab=vocab, c=c, dtype=0, lse=ls, mx=mx, am=am, g=g, scale=0.1, dx=dx, dw=dw,
                 ws=ws, n=need_b):
        return lib.rwkv_linear_loss_backward(x, w, t, lse, mx, am, g, scale, rows, vocab, c, dtype, -100, dx, dw, ws, n, None)
    for call in (forward, backward):
        assert call(dtype=2) == 5
        for bad in (dict(rows=-1), dict(vocab=0), dict(c=0), dict(rows=(1 << 22) + 1), dict(vocab=(1 << 22) + 1),
                    dict(c=(1 << 16) + 1), dict(n=0)):
            assert call(**bad) == 2, bad
        for name in ("x", "w", "t", "lse", "mx", "am", "ws"):
            assert call(**{name: None}) == 1, name
        for bad in (dict(x=x + 4), dict(w=w + 8), dict(t=t + 4), dict(lse=ls + 2), dict(mx=mx + 1), dict(am=am + 2),
                    dict(ws=ws + 8)):
            assert call(**bad) == 6, bad
        assert call(ws=x) == 7 and call(ws=w) == 7 and call(ws=t) == 7
    # elements alone are aligned where rows are no whole pieces
    odd = dict(c=63, n=1 << 23)
    assert forward(x=x + 2, **odd) == 6 and forward(x=x + 2, dtype=1, am=am + 1, **odd) == 6
    assert forward(rows=0, x=None) == 0 and forward(n=need_f - 1) == 2 and backward(n=need_b - 1) == 2
    assert forward(loss=None) == 1 and forward(loss=lo + 2) == 6
    assert forward(loss=ls) == 7 and forward(lse=x) == 7 and forward(am=ws + need_f - 4) == 7
    assert backward(g=None) == 1 and backward(g=g + 2) == 6 and backward(dx=dx + 8) == 6 and backward(dw=dw + 4) == 6
    assert backward(dx=dw) == 7 and backward(dx=x) == 7 and backward(dw=w) == 7 and backward(dw=g) == 7
    assert backward(ws=dx) == 7 and backward(dx=None, dw=None) == 0 and backward(rows=0, x=None, dw=None) == 0
    for scale in (float("nan"), float("inf"), float("-inf")):
        assert backward(scale=scale) == 2


def test_dropout_refusals(native):
    lib = native.lib()
    x, r, rng, out = (FAKE * i for i in range(1, 5))

    def call(x=x, r=r, rng=rng, site=0, p=0.5, n=1000, dtype=0, odtype=0, out=out):
        return lib.rwkv_dropout(x, r, rng, site, p, n, dtype, odtype, out, None)
    assert call(dtype=2) == 5 and call(odtype=-1) == 5
    for bad in (dict(n=-1), dict(n=(1 << 40) + 1), dict(site=-1), dict(site=1 << 32), dict(p=-0.1), dict(p=1.0001),
                dict(p=float("nan"))):
        assert call(**bad) == 2, bad
    assert call(x=None) == 1 and call(rng=None) == 1 and call(out=None) == 1
    assert call(x=x + 2) == 6 and call(x=x + 1, dtype=1) == 6 and call(r=r + 2) == 6 and call(out=out + 2) == 6
    assert call(rng=rng + 4) == 6
    assert call(out=x) == 7 and call(out=r + 3996) == 7 and call(out=rng + 8) == 7
    assert call(n=0, x=None, out=None) == 0


def test_python_refuses():
    pkg = load_pkg()
    ll, dr = pkg.lm_loss, pkg.dropout
    h, w, t = torch.zeros(3, 64), torch.zeros(8, 64), torch.zeros(3, dtype=torch.int64)
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError):
        ll.linear_cross_entropy_l2wrap_rows(h, w, t, 3)
    with pytest.raises(ValueError):
        dr.dropout(h, 0.1, rng)
    with pytest.raises(ValueError):
        dr.dropout_add(h, h, 0.1, rng)
    m = _model_mod()
    for bad in (dict(dropout=-0.1), dict(dropout=1.5), dict(loss="none"), dict(loss="pieces", neighbor_ops="torch")):
        with pytest.raises(ValueError):
            m.AutoRegressiveModel(97, 1, 64, 1, **bad)


def test_generator_known_answers():
    """The known answers that come with the generator's publication (Random123)."""
    philox = load_pkg().dropout._philox
    ones = 0xFFFFFFFF
    for counter, seed, want in (
            ((0, 0, 0, 0), 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, -1, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), 0x299F31D0A4093822,
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = philox(*(torch.tensor([c]) for c in counter), torch.tensor(seed))
        assert tuple(int(g) for g in got) == want


def test_keep_mask():
    dr = load_pkg().dropout
    rng = torch.tensor([1234567890123, 7])
    a = dr.keep_mask((50, 41), 0.3, rng, 2)
    # by the flat index: a longer tensor begins alike
    assert a.shape == (50, 41) and torch.equal(dr.keep_mask((4001,), 0.3, rng, 2)[:2050], a.reshape(-1))
    for other in (dr.keep_mask((50, 41), 0.3, rng, 3), dr.keep_mask((50, 41), 0.3, rng + torch.tensor([0, 1]), 2),
                  dr.keep_mask((50, 41), 0.3, rng + torch.tensor([1 << 32, 0]), 2)):
        assert not torch.equal(a, other)
    # the step counts modulo 2^32, negative numbers as their bits
    assert torch.equal(a, dr.keep_mask((50, 41), 0.3, rng - torch.tensor([0, 1 << 32]), 2))
    assert dr.keep_mask((100,), 0.0, rng).all() and not dr.keep_mask((100,), 1.0, rng).any()
    assert dr.keep_mask((0,), 0.5, rng).shape == (0,)
    # more is dropped, nothing comes back
    assert not (dr.keep_mask((50, 41), 0.6, rng, 2) & ~a).any()
    # n kept of 2^16: five standard deviations of the binomial
    for p in (0.1, 0.5, 0.9):
        n, k = 1 << 16, dr.keep_probability(p)
        kept = int(dr.keep_mask((n,), p, rng, 5).sum())
        assert abs(kept - n * k) < 5 * (n * k * (1 - k)) ** 0.5


def test_model_drops_in_training_alone():
    m = _model_mod()
    gen = torch.Generator().manual_seed(1)
    model = m.AutoRegressiveModel(97, 2, 128, 2, neighbor_ops="torch", wkv7_dtype=torch.float32,
                                  dropout=0.25).init_random(0.2, gen)
    plain = m.AutoRegressiveModel(97, 2, 128, 2, neighbor_ops="torch", wkv7_dtype=torch.float32)
    assert "dropout_rng" not in model.state_dict()
    plain.load_state_dict(model.state_dict())
    inputs, targets = tokens(2, 32, 97)
    model.seed_dropout(5, 10)
    first = model(inputs, targets, TorchKernel)
    assert model.dropout_rng.tolist() == [5, 11]
    second = model(inputs, targets, TorchKernel)
    assert float(first.detach()) != float(second.detach())
    assert torch.equal(model.seed_dropout(5, 10)(inputs, targets, TorchKernel), first)
    # both forwards' masks are their own: the first one's backward is not disturbed by the second
    (first + second).backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)
    model.eval()
    assert float(model(inputs, targets, TorchKernel)) == float(plain(inputs, targets, TorchKernel))
    assert model.dropout_rng.tolist() == [5, 11]
    plain.train()
    assert float(plain(inputs, targets, TorchKernel)) == float(model(inputs, targets, TorchKernel))


def test_keep_mask_refuses():
    d = load_pkg().dropout
    rng = torch.tensor([1, 2])
    for bad in (lambda: d.keep_mask((3,), 1.5, rng), lambda: d.keep_mask((3,), float("nan"), rng),
                lambda: d.keep_mask((3,), 0.5, rng, -1), lambda: d.keep_mask((3,), 0.5, rng, 1 << 32),
                lambda: d.keep_mask((3,), 0.5, torch.tensor([1, 2, 3])), lambda: d.keep_mask((3,), 0.5, rng.int())):
        with pytest.raises(ValueError):
            bad()


def test_workspaces_of_the_largest_sizes_are_planned_at_once(native):
    """Planned anew for each call: a size of many tiles takes the host no longer."""
    import time
    size = native.lib().rwkv_linear_loss_backward_workspace_bytes
    for rows, vocab, c in ((1 << 22, 1 << 22, 2048), (1 << 22, 1, 2048), (1, 1 << 22, 2048), (1 << 22, 256, 2048), (1 << 17, 1 << 17, 1 << 16)):
        for dtype in (0, 1):
            start = time.perf_counter()
            assert size(rows, vocab, c, dtype) > 0
            assert time.perf_counter() - start < 0.05
