"""Models with 4-bit weights: the fused decode step against their modules, and
what scores a text with them."""

import pytest
import torch

from conftest import announce, load_pkg
from model_helpers import tiny_model
from test_gpu_decode_step import DEV, _err, _infer, _model, _state, _wide_model

pytestmark = pytest.mark.gpu


def _quantized(heads=2, vocab=97, group=64, cells=2):
    return load_pkg().w4.quantize_model(_model(heads, vocab, cells), group)


@pytest.mark.parametrize("rows,slots,heads,vocab,group,state_dtype", [
    (1, 1, 1, 1, 32, torch.bfloat16), (3, 5, 2, 97, 64, torch.bfloat16), (16, 16, 2, 16, 128, torch.float32),
    (17, 20, 3, 33, 32, torch.bfloat16), (33, 33, 3, 97, 128, torch.float32), (64, 70, 2, 130, 64, torch.bfloat16),
])
def test_a_fused_step_matches_the_modules(monkeypatch, rows, slots, heads, vocab, group, state_dtype):
    # both round at the same places and differ in the order of sums: 1e-2, as with fp32 weights
    announce("4-bit decode step", rows, slots, heads, vocab, group, str(state_dtype))
    decode = load_pkg().decode
    model = _quantized(heads, vocab, group)
    ids = torch.randperm(slots, generator=torch.Generator().manual_seed(rows))[:rows].to(DEV)
    toks = torch.randint(0, vocab, (rows, 1), generator=torch.Generator().manual_seed(3)).to(DEV)
    a, b = _state(model, slots, state_dtype, 7), _state(model, slots, state_dtype, 7)
    taken = []
    real = decode.step
    monkeypatch.setattr(decode, "step", lambda *x: taken.append(real(*x)) or taken[-1])
    got = _infer(model, toks, ids, a)
    monkeypatch.setattr(decode, "step", lambda *x: None)
    want = _infer(model, toks, ids, b)
    torch.cuda.synchronize()
    assert taken[0] is not None and got.dtype == want.dtype and got.shape == want.shape
    assert _err(got, want) < 1e-2
    for x, y in zip(a.state + a.shift_time + a.shift_channel, b.state + b.shift_time + b.shift_channel):
        assert x.dtype == y.dtype and _err(x, y) < 1e-2


@pytest.mark.parametrize("rows,slots,heads,vocab,group,state_dtype", [
    (17, 17, 12, 200, 64, torch.bfloat16), (64, 64, 12, 97, 32, torch.bfloat16), (40, 41, 33, 130, 128, torch.bfloat16),
    (64, 64, 32, 50, 64, torch.float32)])
def test_a_step_of_wide_cells_matches_the_modules(monkeypatch, rows, slots, heads, vocab, group, state_dtype):
    # wide enough that the products of more than 16 rows take w4.hip's tiles, with either finish
    test_a_fused_step_matches_the_modules(monkeypatch, rows, slots, heads, vocab, group, state_dtype)


def test_it_is_the_model_whose_weights_they_stand_for():
    # the same weights as fp32 parameters, which the products round to bf16: 2^-9 of
    # each, as much again as the activations' own rounding
    announce("4-bit model against its restored weights")
    w4 = load_pkg().w4
    model, plain = _quantized(3, 61, 32), _model(3, 61)
    with torch.no_grad():
        for (_, q), (_, p) in zip(model.named_modules(), plain.named_modules()):
            if isinstance(q, w4.W4Linear):
                p.weight.copy_(w4.dequantize(q.weight))
    ids, toks = torch.arange(5, device=DEV), torch.arange(5, device=DEV).reshape(5, 1)
    got = _infer(model, toks, ids, _state(model, 5, torch.float32, 1))
    want = _infer(plain, toks, ids, _state(plain, 5, torch.float32, 1))
    assert _err(got, want) < 2e-2


def test_what_stays_with_the_modules():
    announce("4-bit decode steps that stay with the modules")
    pkg = load_pkg()
    model = _quantized()
    st = _state(model, 4, torch.bfloat16, 1)
    ids, toks = torch.arange(3, device=DEV), torch.zeros(3, 1, dtype=torch.long, device=DEV)

    def taken():
        with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
            return pkg.decode.step(model, toks, ids, st, None, "last") is not None
    assert taken()
    mixer = model.cells.cells[1].channel_mixer
    old, seen = mixer.key, []
    hook = old.register_forward_hook(lambda *x: seen.append(1))
    assert not taken()
    _infer(model, toks, ids, st)
    assert seen == [1]
    hook.remove()
    mixer.key = torch.nn.Linear(128, 512, bias=False, device=DEV)                # one matrix of another kind
    assert not taken()
    mixer.key = pkg.w4.W4Linear(pkg.w4.quantize(torch.randn(512, 128, device=DEV), 32))   # or group size
    assert not taken()
    mixer.key = pkg.w4.W4Linear(pkg.w4.quantize(torch.randn(256, 128, device=DEV), 64))   # or shape
    assert not taken()
    mixer.key = old
    assert taken()
    model.unembed = torch.nn.Linear(128, 97, bias=False, device=DEV)             # the head is its own
    assert taken()


def test_a_captured_step_replays():
    announce("4-bit decode step in a graph")
    model = _quantized()
    ids, toks = torch.arange(3, device=DEV), torch.arange(3, device=DEV).reshape(3, 1)
    calls = [torch.tensor(t, device=DEV).reshape(3, 1) for t in ([5, 6, 7], [1, 1, 1], [96, 0, 50])]

    def logits(t):
        return _infer(model, t, ids, _state(model, 4, torch.bfloat16, 1)).clone()
    want = [logits(t) for t in calls]
    st = _state(model, 4, torch.bfloat16, 1)
    first = [t.clone() for t in st.state]
    shifts = [t.clone() for t in st.shift_time + st.shift_channel]
    held_t, held_c = list(st.shift_time), list(st.shift_channel)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _infer(model, toks, ids, st)
    for t, w in zip(calls * 2, want * 2):
        toks.copy_(t)
        for x, y in zip(st.state, first):
            x.copy_(y)
        for x, y in zip(held_t + held_c, shifts):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


@pytest.mark.parametrize("bits", [32, 4])
def test_scoring_a_text(bits):
    announce("scoring a text", bits)
    pkg = load_pkg()
    model = _quantized() if bits == 4 else _model()
    ids = torch.tensor([2, 0], device=DEV)
    text = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(5)).to(DEV)
    a, b = _state(model, 3, torch.bfloat16, 4), _state(model, 3, torch.bfloat16, 4)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.score(text, ids, a, top=4)
        logits = model.infer(text, ids, b, unembed_mode="full")
    assert got.log_prob.shape == got.entropy.shape == (2, 8) and got.top_ids.shape == (2, 8, 4)
    want = torch.log_softmax(logits.double(), -1)
    # log p of up to 8 in fp32: 2^-21
    at = want[:, :-1].gather(2, text[:, 1:, None])[..., 0]
    assert (got.log_prob.double() - at).abs().max() < 1e-5
    assert torch.equal(got.top_ids, torch.sort(logits[:, :-1].float(), dim=2, descending=True, stable=True).indices[..., :4])
    assert torch.equal(a.state[0], b.state[0])
    with torch.autocast("cuda", dtype=torch.bfloat16):
        one = model.score(text[:, :1], ids, a)
    assert one.log_prob.shape == (2, 0) and one.top_ids.shape == (2, 0, 0)
    # a served step and its answer
    with torch.autocast("cuda", dtype=torch.bfloat16):
        step = model.infer(text[:, -1:], ids, a)
    s = pkg.token_scores.token_scores(step[:, 0], step[:, 0].argmax(1), 3)
    assert torch.equal(s.log_prob, s.top_log_probs[:, 0]) and (s.entropy > 0).all()


def _slots(st):
    return [t.clone() for t in st.state + st.shift_time + st.shift_channel + [st.elapsed_t]]


@pytest.mark.parametrize("top", [-1, 65, 98])
def test_a_refused_score_leaves_the_slots(top):
    announce("refused score", top)
    model = _model()
    st = _state(model, 3, torch.bfloat16, 4)
    before = _slots(st)
    text, ids = torch.zeros(2, 5, dtype=torch.long, device=DEV), torch.tensor([2, 0], device=DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(ValueError):
        model.score(text, ids, st, top=top)
    assert all(torch.equal(x, y) for x, y in zip(_slots(st), before))


def test_scores_under_fp16_autocast():
    """Logits that the scores do not read are not refused once the slots are advanced."""
    announce("score, fp16 autocast")
    model = tiny_model(seed=1, cells=2, heads=2, vocab=97, std=0.2, wkv7_dtype=torch.bfloat16,
                       neighbor_ops="torch").to(DEV)
    text = torch.randint(0, 97, (2, 5), generator=torch.Generator().manual_seed(6)).to(DEV)
    ids = torch.tensor([2, 0], device=DEV)
    a, b = _state(model, 3, torch.bfloat16, 4), _state(model, 3, torch.bfloat16, 4)
    with torch.autocast("cuda", dtype=torch.float16):
        logits = model.infer(text, ids, b, unembed_mode="full")
        got = model.score(text, ids, a, top=3)
    assert logits.dtype == torch.float16
    at = torch.log_softmax(logits.double(), -1)[:, :-1].gather(2, text[:, 1:, None])[..., 0]
    assert (got.log_prob.double() - at).abs().max() < 1e-5           # log p of up to 8 in fp32, as above
    assert all(torch.equal(x, y) for x, y in zip(_slots(a), _slots(b)))


@pytest.mark.parametrize("rows,heads,group,state_dtype", [
    # (row tiles, column tiles) of the launch that receptance, key and value share: from
    # C = 2752 on two column tiles, from 5504 four, beyond 32 rows two; up to 16
    # sequences the channel mixer's key has two from C = 2048 on and four from 4096
    (1, 32, 64, torch.bfloat16), (8, 43, 32, torch.bfloat16), (16, 64, 128, torch.float32), (1, 85, 64, torch.bfloat16),
    (16, 86, 32, torch.bfloat16), (8, 87, 128, torch.bfloat16), (1, 128, 64, torch.bfloat16),
    (17, 43, 128, torch.bfloat16), (32, 64, 32, torch.float32), (17, 86, 64, torch.bfloat16), (32, 87, 32, torch.bfloat16),
    (33, 43, 64, torch.bfloat16), (40, 64, 128, torch.bfloat16), (64, 87, 32, torch.bfloat16),
    # the other products on w4.hip's two column tiles of up to 32 rows, and its tiles of 64 rows
    (17, 128, 32, torch.bfloat16), (64, 128, 128, torch.bfloat16)])
def test_a_step_with_several_column_tiles_matches_the_modules(monkeypatch, rows, heads, group, state_dtype):
    announce("4-bit decode step, column tiles", rows, heads, group, str(state_dtype))
    tiles = 3 * heads * 64 // 16, 4 * heads * 64 // 16
    assert tiles[0] >= 512 or rows <= 16 and tiles[1] >= 512      # what a launch has to have for two of them
    pkg = load_pkg()
    model = pkg.w4.quantize_model(_wide_model(heads), group)
    ids, toks = torch.arange(rows, device=DEV), torch.arange(rows, device=DEV).reshape(rows, 1) % 33
    a, b = _state(model, rows, state_dtype, 7), _state(model, rows, state_dtype, 7)
    taken = []
    real = pkg.decode.step
    monkeypatch.setattr(pkg.decode, "step", lambda *x: taken.append(real(*x)) or taken[-1])
    got = _infer(model, toks, ids, a)
    monkeypatch.setattr(pkg.decode, "step", lambda *x: None)
    want = _infer(model, toks, ids, b)
    assert taken[0] is not None and _err(got, want) < 1e-2
    for x, y in zip(a.state + a.shift_time + a.shift_channel, b.state + b.shift_time + b.shift_channel):
        assert _err(x, y) < 1e-2
