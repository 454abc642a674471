"""The C ABI of the 4-bit products and of the token scores without a GPU: what
the headers declare is exported, and bad calls are refused on the host."""

import os

import pytest
import torch

from conftest import REPO, load_pkg
from test_abi_cpu import declared_functions

FAKE = 1 << 20        # a pointer that is never followed


@pytest.fixture(scope="module")
def native():
    n = load_pkg()._native
    n.lib()
    return n


@pytest.mark.parametrize("header,exports", [("rwkv_w4.h", "W4_EXPORTS"), ("rwkv_decode_w4.h", "DECODE_W4_EXPORTS"),
                                            ("rwkv_token_scores.h", "SCORES_EXPORTS")])
def test_exports(native, header, exports):
    declared = declared_functions(os.path.join(REPO, "include", header), "rwkv_")
    assert set(declared) == set(getattr(native, exports))
    for name in declared:
        assert hasattr(native.lib(), name) and name in native._SIGNATURES


def test_w4_sizes(native):
    lib = native.lib()
    assert lib.rwkv_w4_packed_bytes(1, 1) == 1024 and lib.rwkv_w4_packed_bytes(17, 129) == 4096
    assert lib.rwkv_w4_packed_bytes(768, 768) == 768 * 768 // 2
    assert lib.rwkv_w4_scales_bytes(768, 768, 64) == 768 * 12 * 2
    assert lib.rwkv_w4_scales_bytes(17, 129, 32) == 32 * 8 * 2
    assert lib.rwkv_w4_packed_bytes(1 << 26, 512 * 128 - 128) == (1 << 22) * 511 * 1024
    for bad in ((0, 1), (1, 0), (-1, 5), ((1 << 26) + 1, 8), (8, (1 << 26) + 1), (1 << 26, 512 * 128)):
        assert lib.rwkv_w4_packed_bytes(*bad) == -1 and lib.rwkv_w4_scales_bytes(*bad, 64) == -1
    assert lib.rwkv_w4_scales_bytes(8, 8, 16) == -1


def test_w4_refusals(native):
    lib = native.lib()
    w, p, s, x, y = (FAKE * i for i in (1, 10, 20, 30, 40))

    def quantize(weight=w, out=32, d_in=256, group=64, dtype=0, packed=p, scales=s):
        return lib.rwkv_w4_quantize(weight, out, d_in, group, dtype, packed, scales, None)

    def restore(packed=p, scales=s, out=32, d_in=256, group=64, dtype=0, weight=w):
        return lib.rwkv_w4_dequantize(packed, scales, out, d_in, group, dtype, weight, None)

    def linear(x=x, packed=p, scales=s, rows=4, out=32, d_in=256, group=64, dtype=0, y=y, ws=None, nbytes=0):
        return lib.rwkv_w4_linear(x, packed, scales, rows, out, d_in, group, dtype, y, ws, nbytes, None)
    for call in (quantize, restore, linear):
        assert call(dtype=2) == 5
        for bad in (dict(out=0), dict(d_in=-1), dict(group=48), dict(out=(1 << 26) + 1)):
            assert call(**bad) == 2, bad
        assert call(packed=None) == 1 and call(scales=None) == 1
        assert call(packed=p + 8) == 6 and call(scales=s + 2) == 6
    for call in (quantize, restore):
        assert call(weight=None) == 1 and call(weight=w + 2) == 6
        assert call(weight=p) == 7 and call(weight=s) == 7
    assert quantize(packed=s) == 7
    assert linear(rows=-1) == 2 and linear(rows=(1 << 20) + 1) == 2
    assert linear(x=None) == 1 and linear(y=None) == 1
    assert linear(x=x + 2) == 6 and linear(y=y + 1) == 6 and linear(y=y + 1, dtype=1) == 6
    for other in (x, p, s):
        assert linear(y=other) == 7
    assert linear(y=x + 4 * 256 * 4 - 4) == 7
    assert linear(rows=0, x=None, y=None) == 0
    # a call whose inputs are shared needs its workspace
    size = lib.rwkv_w4_linear_workspace_bytes
    assert size(16, 768, 1 << 14, 1) == 0 and size(0, 8, 8, 0) == 0
    assert size(-1, 8, 8, 0) == size(1, 0, 8, 0) == size(1, 8, 8, 2) == size((1 << 20) + 1, 8, 8, 0) == -1
    needed = size(100, 32, 1 << 14, 1)
    big = dict(rows=100, d_in=1 << 14, dtype=1, x=FAKE * 50, y=FAKE * 60, packed=FAKE * 70, scales=FAKE * 80)
    assert needed > 0
    assert linear(**big) == 2 and linear(**big, ws=FAKE * 90, nbytes=needed - 1) == 2
    assert linear(**big, nbytes=needed) == 1 and linear(**big, ws=FAKE * 90 + 8, nbytes=needed) == 6
    assert linear(**big, ws=FAKE * 50, nbytes=needed) == 7 and linear(**big, ws=FAKE * 60, nbytes=needed) == 7


def test_decode_w4_refusals():
    import ctypes
    if torch.cuda.is_available():
        pytest.skip("an accepted call would launch on addresses that are not memory")
    from test_decode_step_cpu import GIB, HIP, NULL, SHAPE, ALIGNMENT, OVERLAP, _params
    native = load_pkg()._native
    lib = native.lib()
    rows, heads, C = 3, 3, 192
    need = lib.rwkv_decode_workspace_bytes(rows, heads)

    def weights(group=64, **over):
        q = native.DecodeW4Weights()
        q.group = group
        for i, (name, kind) in enumerate(q._fields_[:-1]):
            setattr(q, name, native.W4Matrix((2000 + 2 * i) * GIB, (2001 + 2 * i) * GIB))
        for name, at in over.items():
            setattr(q, name, native.W4Matrix(*at))
        return q

    def cell(q, p=None, **over):
        p = p or _params(native, True)
        for name in ("receptance", "key", "value", "output", "channel_key", "channel_value"):
            setattr(p, name, None)                                  # not looked at
        a = dict(x=GIB, ws=9 * GIB, nbytes=need)
        a.update(over)
        return lib.rwkv_decode_cell_w4(
            ctypes.addressof(p), ctypes.addressof(q) if q else None, a["x"], 2 * GIB, 3 * GIB, 4 * GIB, 5 * GIB,
            6 * GIB, 7 * GIB, 8 * GIB, rows, heads, 4, 1, 1, a["ws"], a["nbytes"], None)
    assert cell(weights()) == HIP and cell(None) == NULL            # nothing to refuse but the missing GPU
    for group in (0, 16, 48, 256):
        assert cell(weights(group)) == SHAPE
    assert cell(weights(key=(None, GIB * 99))) == NULL and cell(weights(output=(GIB * 99, None))) == NULL
    assert cell(weights(value=(GIB * 99 + 8, GIB * 98))) == ALIGNMENT
    last = weights().channel_value
    size, scales = lib.rwkv_w4_packed_bytes(C, 4 * C), lib.rwkv_w4_scales_bytes(C, 4 * C, 64)
    assert cell(weights(), x=last.packed + size - 16) == OVERLAP and cell(weights(), x=last.packed + size) == HIP
    assert cell(weights(), ws=last.scales + scales - 16) == OVERLAP and cell(weights(), ws=last.scales + scales) == HIP
    assert cell(weights(), nbytes=need - 1) == SHAPE

    def head(q=(4 * GIB, 5 * GIB), group=32, vocab=50, logits=6 * GIB, ws=7 * GIB):
        m = native.W4Matrix(*q) if q else None
        return lib.rwkv_decode_head_w4(GIB, 2 * GIB, 3 * GIB, 1e-5, ctypes.addressof(m) if m else None, group, rows,
                                       heads, vocab, logits, ws, need, None)
    assert head() == HIP and head(None) == NULL and head((None, GIB)) == NULL and head((GIB * 4, None)) == NULL
    assert head(group=8) == SHAPE and head(vocab=0) == SHAPE and head(vocab=(1 << 26) + 1) == SHAPE
    assert head((4 * GIB + 4, 5 * GIB)) == ALIGNMENT
    assert head(logits=4 * GIB) == OVERLAP and head(logits=5 * GIB) == OVERLAP and head(ws=5 * GIB) == OVERLAP


def test_token_scores_refusals(native):
    lib = native.lib()
    x, t, lp, en, mx, ls, tl, ti, tg = (FAKE * i for i in (1, 100, 101, 102, 103, 104, 105, 106, 107))

    def forward(logits=x, tokens=t, rows=4, vocab=1000, top=5, dtype=0, log_prob=lp, entropy=en,
                row_max=mx, log_sum=ls, top_lp=tl, ids=ti):
        return lib.rwkv_token_scores_forward(logits, tokens, rows, vocab, top, dtype, log_prob, entropy,
                                             row_max, log_sum, top_lp, ids, None)

    def backward(logits=x, tokens=t, row_max=mx, log_sum=ls, entropy=en, ids=ti, g=lp, h=tl, tg=tg,
                 rows=4, vocab=1000, top=5, dtype=0, grad=FAKE * 200):
        return lib.rwkv_token_scores_backward(logits, tokens, row_max, log_sum, entropy, ids, g, h, tg,
                                              rows, vocab, top, dtype, grad, None)
    for call in (forward, backward):
        assert call(dtype=3) == 5
        for bad in (dict(rows=-1), dict(vocab=0), dict(top=-1), dict(top=65), dict(vocab=4), dict(vocab=1 << 31),
                    dict(rows=1 << 31)):
            assert call(**bad) == 2, bad
        for name in ("logits", "tokens", "entropy", "ids"):
            assert call(**{name: None}) == 1, name
        assert call(logits=x + 2) == 6 and call(logits=x + 1, dtype=1) == 6 and call(tokens=t + 4) == 6
        assert call(rows=0, logits=None) == 0
    assert forward(log_prob=None) == 1 and forward(top_lp=None) == 1
    assert forward(log_prob=lp + 2) == 6 and forward(ids=ti + 4) == 6
    assert forward(entropy=lp) == 7 and forward(row_max=x) == 7 and forward(ids=t) == 7
    assert forward(log_sum=ls + 1) == 6
    assert backward(grad=None) == 1 and backward(row_max=None) == 1 and backward(log_sum=None) == 1
    assert backward(grad=x) == 7 and backward(grad=FAKE * 100 - 8) == 7 and backward(g=FAKE * 200) == 7
    assert backward(g=lp + 2) == 6 and backward(tg=tg + 1) == 6


def test_python_refuses_host_tensors():
    pkg = load_pkg()
    with pytest.raises(ValueError):
        pkg.w4.quantize(torch.zeros(16, 64))
    with pytest.raises(ValueError):
        pkg.token_scores.token_scores(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))
    # a weight can be described without a GPU, and is checked
    packed = torch.zeros(1, 1, 4, 16, 16, dtype=torch.uint8)
    scales = torch.zeros(1, 1, 16, 2, dtype=torch.bfloat16)
    w = pkg.w4.W4Weight(packed, scales, 3, 5, 64)
    with pytest.raises(ValueError):
        pkg.w4.linear(torch.zeros(2, 5), w)
    for bad in ((packed, scales, 3, 5, 32), (packed, scales, 17, 5, 64), (packed, scales, 3, 129, 64),
                (packed, scales.float(), 3, 5, 64), (packed, scales, 0, 5, 64), (packed, scales, 3, 5, 16)):
        with pytest.raises(ValueError):
            pkg.w4.W4Weight(*bad)
