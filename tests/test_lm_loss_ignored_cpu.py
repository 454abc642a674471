"""The C ABI of the loss of logits with ignored rows (include/rwkv_lm_loss_ignore.h)
without a GPU: what the header declares is exported, bad calls are refused on the host as
rwkv_lm_loss.h's are."""

import os

import pytest

from conftest import REPO, load_pkg
from test_abi_cpu import declared_functions

FAKE = 1 << 24        # a pointer that is never followed


@pytest.fixture(scope="module")
def native():
    n = load_pkg()._native
    n.lib()
    return n


def test_exports(native):
    declared = declared_functions(os.path.join(REPO, "include", "rwkv_lm_loss_ignore.h"), "rwkv_")
    assert set(declared) == set(native.LOSS_IGNORE_EXPORTS)
    for name in declared:
        assert hasattr(native.lib(), name) and name in native._SIGNATURES


def test_refusals(native):
    x, t, loss, lse, mx, am, g, dx = (FAKE * i for i in range(1, 9))
    lib = native.lib()

    def forward(x=x, t=t, rows=4, vocab=64, dtype=1, ignore=-100, loss=loss, lse=lse, mx=mx, am=am):
        return lib.rwkv_cross_entropy_l2wrap_ignore_forward(x, t, rows, vocab, dtype, ignore, loss, lse, mx, am, None)

    def backward(x=x, t=t, rows=4, vocab=64, dtype=1, ignore=-100, lse=lse, mx=mx, am=am, g=g, scale=1e-4, dx=dx):
        return lib.rwkv_cross_entropy_l2wrap_ignore_backward(x, t, lse, mx, am, g, scale, rows, vocab, dtype, ignore, dx, None)
    for call in (forward, backward):
        assert call(dtype=4) == 5
        for bad in (dict(vocab=0), dict(rows=-1), dict(rows=1 << 31), dict(rows=(1 << 31) - 1, vocab=(1 << 31) - 1)):
            assert call(**bad) == 2, bad
        for name in ("x", "t", "lse", "mx", "am"):
            assert call(**{name: None}) == 1, name
        for bad in (dict(x=x + 8), dict(t=t + 4), dict(lse=lse + 2), dict(mx=mx + 1), dict(am=am + 3)):
            assert call(**bad) == 6, bad
        assert call(rows=0, x=None, t=None) == 0
    assert forward(loss=None) == 1 and forward(loss=lse) == 7 and forward(am=x) == 7 and forward(loss=loss + 2) == 6
    assert backward(dx=None) == 1 and backward(g=None) == 1 and backward(dx=x) == 7 and backward(dx=g) == 7
    assert backward(dx=dx + 8) == 6 and backward(vocab=63, dx=dx + 1) == 6
    for scale in (float("nan"), float("inf")):
        assert backward(scale=scale) == 2
