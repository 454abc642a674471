"""The loss straight from hidden states and unembedding, and its gradients, against
float64 formulas on the GPU: every tile's edge, ignored rows and rows without a loss,
ties, extreme sizes of numbers, streams and graphs.

Errors are bounded element by element. With u = 2^-24 and A = sum_k |x_k| |w_k|:

* a logit is a sum of exact products (bf16) in fp32, at most c additions; the matrix
  cores may cut off where fp32 arithmetic rounds, so each counts 2u. fp32 operands
  are two fp16 numbers: 2^-22 of an element is lost (its two roundings, 2^-11 each),
  or 2^-38 of the operand's largest magnitude, and lo lo, 2^-22 of a product; three
  products are added;
* the exponentials' sum adds positive terms: 32 words a lane, three joins and then
  a 16th of the tiles of 64 to 256, and 16 joins; an exponential is within 2^-20 of its
  value (its argument, below 16 where it counts, is rounded twice);
* D is rounded to fp16 (2^-11; 2^-25 of 2^13 below its range), for the hidden
  gradient of bf16 operands to bf16 after that (2^-8, but at the target and the
  argmax), or held to 2^-22 (fp32); a gradient adds vocab or rows terms;
* the result is rounded to its type: 2^-8 (bf16), u (fp32).
"""

import math

import pytest
import torch

from conftest import announce, load_pkg

pytestmark = pytest.mark.gpu
ll = load_pkg().lm_loss
U = 2.0 ** -24
BOTH = [torch.bfloat16, torch.float32]
DEV = "cuda"


def make(rows, vocab, c, dtype, seed=0, spread=2.5, lift=6.0):
    """Logits of standard deviation ``spread``, the target's lifted by up to ``lift``."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn(vocab, c, generator=g, device=DEV) * (spread / math.sqrt(c))
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    toward = w[t] / w[t].norm(dim=1, keepdim=True).clamp(min=1e-3)
    x = torch.randn(rows, c, generator=g, device=DEV) + toward * (lift / spread) * torch.rand(rows, 1, generator=g, device=DEV)
    return x.to(dtype), w.to(dtype), t


def logit_error(x, w):
    """Bound of |z - exact z| over a row's words: [rows, 1]."""
    c = x.shape[1]
    a = x.double().abs() @ w.double().abs().t()
    if x.dtype == torch.bfloat16:
        e = a * (c * 2 * U)
    else:
        floor = 2.0 ** -38 * (x.double().abs().max() * w.double().abs().sum(1)[None, :]
                              + w.double().abs().max() * x.double().abs().sum(1)[:, None])
        e = a * (3 * 2.0 ** -22 + 3 * c * 2 * U) + 2 * floor
    return e.amax(1, keepdim=True)


def check(x, w, t, g, num_tokens, ignore=-100):
    rows, c = x.shape
    vocab = w.shape[0]
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ll.linear_cross_entropy_l2wrap_rows(xr, wr, t, num_tokens, ignore)
    dx, dw = torch.autograd.grad(loss, (xr, wr), g)
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == x.dtype
    with torch.no_grad():
        assert torch.equal(ll.linear_cross_entropy_l2wrap_rows(x, w, t, num_tokens, ignore), loss) or loss.isnan().any()

    x64, w64 = x.double(), w.double()
    dead = t == ignore
    inside = (t >= 0) & (t < vocab) & ~dead
    x64 = torch.where(dead[:, None], torch.zeros_like(x64), x64)
    z = x64 @ w64.t()
    m, top = z.max(dim=1, keepdim=True).values, (z == z.max(dim=1, keepdim=True).values).int().argmax(dim=1, keepdim=True)
    lse = torch.logsumexp(z, dim=1, keepdim=True)
    at = torch.where(inside, t, 0)[:, None]
    want = torch.where(dead, 0.0, torch.where(inside, (lse - z.gather(1, at))[:, 0], math.nan))
    ez = logit_error(torch.where(dead[:, None], torch.zeros_like(x), x), w)
    adds = 32 + 3 + -(-vocab // 1024) + 17
    e_lse = ez + adds * 2 * U + 2.0 ** -20 + 2 * U * lse.abs()
    bound = (ez + e_lse)[:, 0] + 2 * U * (lse.abs() + z.abs().amax(1, keepdim=True))[:, 0]
    assert torch.equal(loss.isnan(), want.isnan())
    fine = ~want.isnan()
    err = (loss.double() - want).abs()
    assert (err[fine] <= bound[fine]).all(), float((err / bound)[fine].max())
    assert (loss[fine] >= 0).all() and (loss[dead] == 0).all()

    s = 1e-4 / num_tokens if num_tokens > 0 else 0.0
    gd = torch.where(dead, 0.0, g.double())[:, None]
    p = torch.exp(z - lse)
    wrap = torch.where(dead[:, None], 0.0, s * m)
    d = gd * p
    d.scatter_add_(1, at, torch.where(inside[:, None], -gd, 0.0))
    d.scatter_add_(1, top, wrap)
    reference = max(float(torch.where(dead[:, None], 0.0, g.double()[:, None]).abs().max()), float(wrap.abs().max())) or 1.0
    # of D before it is rounded: p's error, and that of what is added to it
    de = gd.abs() * p * (ez + e_lse + 2.0 ** -19) + 4 * U * (gd.abs() * p + d.abs())
    de.scatter_add_(1, at, torch.where(inside[:, None], gd.abs() * 4 * U, 0.0))
    de.scatter_add_(1, top, wrap.abs() * 8 * U + s * ez)
    bf = x.dtype == torch.bfloat16
    held = d.abs() * (2.0 ** -11 if bf else 2.0 ** -22) + reference * 2.0 ** -38
    again = d.abs() * 2.0 ** -8 if bf else torch.zeros_like(d)
    if bf:
        again.scatter_(1, at, torch.where(inside[:, None], 0.0, again.gather(1, at)))
        again.scatter_(1, top, 0.0)
    out = 2.0 ** -8 if bf else 2 * U
    # the other operand's own two fp16 numbers, or x's one; the sums
    of_x, of_w = (2.0 ** -38, 0.0) if bf else (2.0 ** -22, 2.0 ** -22)
    for got, dm, om, err_d, terms, of in ((dx, d, w64, de + held + again, vocab, of_w), (dw, d.t(), x64, (de + held).t(), rows, of_x)):
        exact = dm @ om
        size = dm.abs() @ om.abs()
        lost = of * size + (2.0 ** -38 * om.abs().max() * dm.abs().sum(1, keepdim=True))
        limit = err_d @ om.abs() + lost + size * ((3 * terms + 64) * 2 * U + 2.0 ** -22) + exact.abs() * out + 1e-44
        miss = (got.double() - exact).abs()
        assert (miss <= limit).all(), (float((miss / limit).max()), terms)
    return loss, dx, dw


SIZES = [(1, 1, 1), (1, 2, 64), (2, 255, 8), (3, 256, 64), (5, 257, 65), (255, 300, 128), (256, 511, 192),
         (257, 512, 100), (64, 4097, 320), (300, 1000, 384), (513, 700, 256), (1000, 2049, 33), (128, 8192, 768),
         (31, 513, 1000), (96, 256, 256), (700, 300, 512),
         # rows shared among workgroups, tiles of every size, the vocabulary's end inside each
         (5000, 300, 64), (3000, 1000, 128), (1100, 70, 192), (9000, 256, 100), (129, 129, 64), (64, 16449, 64),
         (200, 16500, 128), (30, 8001, 320), (1023, 2300, 65), (256, 32769, 64)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,c", SIZES)
def test_sizes(rows, vocab, c, dtype):
    announce("linear loss", rows, vocab, c, dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=rows + vocab)
    t[::7] = -100
    if rows > 1:
        t[1] = vocab - 1
    g = torch.randn(rows, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    check(x, w, t, torch.full((rows,), 1.0 / rows, device=DEV), rows)
    check(x, w, t, g, 3)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,c", [(600, 65536, 64), (2000, 20011, 192), (260, 65529, 256)])
def test_larger(rows, vocab, c, dtype):
    announce("linear loss, larger", rows, vocab, c, dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=5)
    check(x, w, t, torch.full((rows,), 1.0 / rows, device=DEV), rows)


def test_several_pieces():
    """More than half a GiB of D: pieces of the vocabulary, the last one smaller."""
    rows, vocab, c = 9000, 40001, 64
    announce("linear loss, pieces", rows, vocab, c)
    x, w, t = make(rows, vocab, c, torch.bfloat16, seed=8)
    g = torch.full((rows,), 1.0 / rows, device=DEV)
    loss, dx, dw = check(x, w, t, g, rows)
    # a row's loss depends on the others by the tiles alone, in which its logits (the same
    # numbers) are added up: two sums of one row, each within the module's bound of a sum
    few = ll.linear_cross_entropy_l2wrap_rows(x[:50], w, t[:50], rows)
    adds = 32 + 3 + -(-vocab // 1024) + 17
    assert (few - loss[:50]).abs().max() <= 2 * (adds * 2 * U + 2.0 ** -20 + 2 * U * 20)
    assert torch.equal(ll.linear_cross_entropy_l2wrap_rows(x[:8000], w, t[:8000], rows), loss[:8000])


def test_the_operator_of_logits_agrees():
    """cross_entropy_l2wrap of fp32 logits, and the mean."""
    announce("linear loss against the operator of logits")
    x, w, t = make(77, 1003, 128, torch.float32, seed=4)
    a, b = (v.detach().requires_grad_() for v in (x, w))
    c, d = (v.detach().requires_grad_() for v in (x, w))
    one = ll.linear_cross_entropy_l2wrap(a, b, t)
    two = ll.cross_entropy_l2wrap((c.double() @ d.double().t()).float(), t)
    one.backward(), two.backward()
    one, two = one.detach(), two.detach()
    assert abs(float(one) - float(two)) <= 1e-5 * float(two)
    for p, q in ((a, c), (b, d)):
        assert float((p.grad - q.grad).norm() / q.grad.norm()) <= 1e-5
    t[:60] = -100
    part = ll.linear_cross_entropy_l2wrap(x, w, t)
    rows = ll.linear_cross_entropy_l2wrap_rows(x, w, t, 77)
    assert abs(float(part) - float(rows[60:].mean())) <= 1e-6 * float(part)


@pytest.mark.parametrize("dtype", BOTH)
def test_ignored_and_invalid_rows(dtype):
    announce("linear loss, ignored rows", dtype)
    rows, vocab, c = 40, 500, 64
    x, w, t = make(rows, vocab, c, dtype, seed=11)
    g = torch.rand(rows, device=DEV) + 0.1
    t[3], t[4], t[5], t[6] = -1, vocab, vocab + 11, -101          # no such word: NaN losses, no target term
    t[10:20] = -100
    x[10], x[11] = math.nan, math.inf                             # what is ignored may hold anything
    x[12] = 1e30 if dtype == torch.float32 else 3e38
    check(x, w, t, g, rows)
    t[7] = 9
    check(x, w, torch.where(t == -100, 9, t), g, rows, ignore=9)  # a word of the vocabulary
    # all of them
    t[:] = -100
    loss, dx, dw = check(x, w, t, g, rows)
    assert not loss.any() and not dx.any() and not dw.any()
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    mean = ll.linear_cross_entropy_l2wrap(a, b, t)
    mean.backward()
    assert float(mean.detach()) == 0.0 and not a.grad.any() and not b.grad.any()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,c", [(1023, 64), (1024, 64), (1025, 100), (4000, 192)])
def test_many_rows_of_which_some_are_ignored(rows, c, dtype):
    """From 1024 rows on, those that are learned are brought together first."""
    announce("linear loss, many rows, some ignored", rows, c, dtype)
    vocab = 700
    x, w, t = make(rows, vocab, c, dtype, seed=12)
    full = t.clone()
    g = torch.rand(rows, device=DEV) + 0.1
    r = torch.arange(rows, device=DEV)
    for dead in (r % 3 != 1, r < rows - 1, r > 0, r < 0, (r // 70) % 2 == 0, r % 64 == 63, r >= 512, r >= 0):
        t = full.masked_fill(dead, -100)
        t[2] = -7 if rows == 1025 and not dead[2] else t[2]
        y = torch.where(dead[:, None], torch.full_like(x, math.nan), x)
        loss, dx, dw = check(y, w, t, g, rows)
        assert not dx[dead].any()
    assert not dw.any()


@pytest.mark.parametrize("dtype", BOTH)
def test_nan_and_infinite_numbers(dtype):
    """A row's own NaN or infinity costs that row's loss and hidden gradient, and every
    word's weight gradient. A word's costs the rows whose logit is NaN or plus infinity;
    minus infinity is a probability of 0, which three products of fp32 halves do not
    keep (inf - inf)."""
    announce("linear loss, NaN and infinities", dtype)
    rows, vocab, c = 30, 600, 64
    x, w, t = make(rows, vocab, c, dtype, seed=13)
    clean = ll.linear_cross_entropy_l2wrap_rows(x, w, t, rows)
    for bad in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[5, 3] = bad
        a, b = y.requires_grad_(), w.detach().requires_grad_()
        loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, rows)
        others = torch.arange(rows, device=DEV) != 5
        if dtype == torch.bfloat16:
            assert torch.equal(loss[others], clean[others])
        else:
            assert (loss[others] - clean[others]).abs().max() < 1e-5
        assert loss[5].isnan()
        dx, dw = torch.autograd.grad(loss, (a, b), torch.ones(rows, device=DEV))
        assert dx[others].isfinite().all() and dx[5].isnan().all() and dw.isnan().all(dim=1).any()
        v = w.clone()
        v[77, 0] = bad
        z = x.double() @ v.double().t()
        lost = z.isnan().any(1) | (z == math.inf).any(1) | (torch.full((rows,), dtype == torch.float32, device=DEV))
        got = ll.linear_cross_entropy_l2wrap_rows(x, v, torch.where(t == 77, 78, t), rows)
        assert torch.equal(got.isnan(), lost)
        want = torch.logsumexp(z, 1) - z[torch.arange(rows, device=DEV), torch.where(t == 77, 78, t)]
        assert (got[~lost].double() - want[~lost]).abs().max() < 1e-4 if (~lost).any() else True


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("scale_x,scale_w", [(1e-18, 1e18), (1e15, 1e-15), (1e-30, 1.0), (0.0, 1.0), (1.0, 0.0), (30.0, 1.0)])
def test_scales(scale_x, scale_w, dtype):
    """Operands of any size, logits of none, and rows that are all but certain."""
    announce("linear loss, scales", scale_x, scale_w, dtype)
    x, w, t = make(50, 400, 64, torch.float32, seed=17)
    check((x * scale_x).to(dtype), (w * scale_w).to(dtype), t, torch.rand(50, device=DEV), 50)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 0.0])
def test_row_gradients_of_any_size(size, dtype):
    announce("linear loss, row gradients", size, dtype)
    x, w, t = make(60, 300, 128, dtype, seed=19)
    g = torch.randn(60, device=DEV) * size
    check(x, w, t, g, 0)                                 # l2wrap off
    check(x, w, t, g, 60)
    g[::2] *= 1e-5                                       # rows of very different weight
    check(x, w, t, g, 0)


@pytest.mark.parametrize("dtype", BOTH)
def test_first_of_equal_maxima(dtype):
    """Equal words, in one tile and in several: l2wrap's term goes to the first."""
    announce("linear loss, ties", dtype)
    rows, vocab, c = 20, 1500, 64
    x, w, t = make(rows, vocab, c, dtype, seed=23)
    for places in ((5, 6), (100, 200, 255), (255, 256), (300, 900, 1499), (0, 1499)):
        v = w.clone()
        v[list(places)] = (x.float().mean(0) * 0).to(dtype) + (3.0 * x[0].float() / x[0].float().norm()).to(dtype)
        _, kept = ll._linear_forward(x[:1].contiguous(), v, t[:1], -100)
        assert int(kept[2].view(torch.int32)) == places[0], places
        a, b = x[:1].detach().requires_grad_(), v.detach().requires_grad_()
        loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t[:1], 1)
        _, dw = torch.autograd.grad(loss, (a, b), torch.zeros(1, device=DEV))
        touched = dw.abs().sum(1).nonzero()[:, 0].tolist()
        assert touched == [places[0]]                    # nothing but l2wrap's term is left
    # a vocabulary of zeros: every word ties
    loss, _, _ = check(x, torch.zeros_like(w), t, torch.ones(rows, device=DEV), rows)
    assert (loss - math.log(vocab)).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", BOTH)
def test_one_gradient_alone(dtype):
    announce("linear loss, one gradient", dtype)
    x, w, t = make(300, 700, 192, dtype, seed=29)
    g = torch.rand(300, device=DEV)
    _, dx, dw = check(x, w, t, g, 300)
    a = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(a, w, t, 300), a, g)[0], dx)
    b = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(x, b, t, 300), b, g)[0], dw)


@pytest.mark.parametrize("dtype", BOTH)
def test_gradient_against_differences(dtype):
    """Central differences of the loss in float64, along a direction."""
    announce("linear loss, differences", dtype)
    x, w, t = make(20, 300, 64, dtype, seed=31)
    g = torch.rand(20, device=DEV, dtype=torch.float64)
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(a, b, t, 0), (a, b), g.float())
    gen = torch.Generator(device=DEV).manual_seed(1)
    vx, vw = (torch.randn(v.shape, generator=gen, device=DEV, dtype=torch.float64) for v in (x, w))

    def f(h):
        z = (x.double() + h * vx) @ (w.double() + h * vw).t()
        return float((g * (torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0])).sum())
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    size = float((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum())
    assert abs(got - want) <= (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5) * size


def test_layouts_streams_and_determinism():
    announce("linear loss, layouts and streams")
    x, w, t = make(333, 1111, 256, torch.bfloat16, seed=37)
    g = torch.rand(333, device=DEV)
    loss, dx, dw = check(x, w, t, g, 333)
    wide = torch.zeros(333, 300, dtype=x.dtype, device=DEV)
    wide[:, 3:259] = x
    flat = torch.empty(w.numel() + 1, dtype=w.dtype, device=DEV)      # off a 16-byte boundary
    flat[1:] = w.reshape(-1)
    for a, b in ((wide[:, 3:259], w.t().contiguous().t()), (x, flat[1:].view_as(w))):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        got = ll.linear_cross_entropy_l2wrap_rows(a, b, t.int(), 333)
        assert torch.equal(got, loss)
        for p, q in zip(torch.autograd.grad(got, (a, b), g), (dx, dw)):
            assert torch.equal(p, q)
    # two at a time, on streams of their own
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    results = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                l = ll.linear_cross_entropy_l2wrap_rows(a, b, t, 333)
                r.append((l, *torch.autograd.grad(l, (a, b), g)))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for r in results:
        for got in r:
            assert all(torch.equal(p, q) for p, q in zip(got, (loss, dx, dw)))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,c", [(100, 900, 64), (600, 8000, 256)])
def test_in_a_graph(rows, vocab, c, dtype):
    """Forward and backward captured, replayed on new inputs with eager work between."""
    announce("linear loss, graph", rows, vocab, c, dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=41)
    g = torch.rand(rows, device=DEV)
    a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()

    def step():
        loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, rows)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b), g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x2, w2, t2 = make(rows, vocab, c, dtype, seed=100 + seed)
        with torch.no_grad():
            a.copy_(x2), b.copy_(w2), t.copy_(t2), g.copy_(torch.rand(rows, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def test_no_rows():
    announce("linear loss, no rows")
    for dtype in BOTH:
        for c in (64, 33):
            a = torch.zeros(0, c, dtype=dtype, device=DEV, requires_grad=True)
            b = torch.ones(65, c, dtype=dtype, device=DEV, requires_grad=True)
            loss = ll.linear_cross_entropy_l2wrap_rows(a, b, torch.zeros(0, dtype=torch.int64, device=DEV), 0)
            da, db = torch.autograd.grad(loss, (a, b), torch.zeros(0, device=DEV))
            assert loss.shape == (0,) and da.shape == (0, c) and not db.any()


def test_memory_stays_small():
    """No [rows, vocab] array is made: 4096 x 65536 logits in bf16 are half a GiB, and
    the forward takes a small part of that."""
    announce("linear loss, memory")
    x, w, t = make(4096, 65536, 64, torch.bfloat16, seed=43)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ll.linear_cross_entropy_l2wrap_rows(x, w, t, 4096)
    assert torch.cuda.max_memory_allocated() - before < 4096 * 65536 * 2 // 16


def test_refusals():
    announce("linear loss, refusals")
    x, w, t = make(4, 30, 64, torch.float32)
    f = ll.linear_cross_entropy_l2wrap_rows
    for bad, exc in [(lambda: f(x, w.cpu(), t, 4), ValueError), (lambda: f(x, w, t.cpu(), 4), ValueError),
                     (lambda: f(x, w[:, :32], t, 4), ValueError), (lambda: f(x, w, t[:2], 4), ValueError),
                     (lambda: f(x[0], w, t, 4), ValueError), (lambda: f(x, w[:0], t, 4), ValueError),
                     (lambda: f(x[:, :0], w[:, :0], t, 4), ValueError), (lambda: f(x, w.bfloat16(), t, 4), TypeError),
                     (lambda: f(x.half(), w.half(), t, 4), TypeError), (lambda: f(x, w, t.float(), 4), TypeError),
                     (lambda: f(x, w, t > 3, 4), TypeError)]:
        with pytest.raises(exc):
            bad()
    with pytest.raises(ValueError):
        wide = torch.zeros(1, (1 << 16) + 1, device=DEV)
        f(wide, wide, t[:1], 1)
    a = x.requires_grad_()
    grad, = torch.autograd.grad(f(a, w, t, 4).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        dual = fw.make_dual(x.detach(), torch.ones_like(x))
        for args in ((dual, w), (x.detach(), fw.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError):
                f(*args, t, 4)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32])
def test_targets_of_narrow_types(dtype):
    """The mean counts rows by the targets' own values: 156 in eight bits without a sign
    is not -100."""
    announce("linear loss, narrow targets", dtype)
    x, w, t = make(40, 120 if dtype == torch.int8 else 200, 64, torch.float32, seed=51)
    if dtype == torch.uint8:
        t[::2] = 156
    else:
        t[::3] = -100
    assert torch.equal(ll.linear_cross_entropy_l2wrap(x, w, t.to(dtype)), ll.linear_cross_entropy_l2wrap(x, w, t))
    rows = ll.linear_cross_entropy_l2wrap_rows(x, w, t.to(dtype), 40)
    assert torch.equal(ll.linear_cross_entropy_l2wrap(x, w, t.to(dtype)), rows.sum() / (t != -100).sum())


@pytest.mark.parametrize("vocab", [1, 40, 700])
def test_logits_of_minus_infinity(vocab):
    """Words of bf16 whose logit is minus infinity: probability 0; where there is no other
    word no loss, and a NaN among them is not lost."""
    announce("linear loss, minus infinity", vocab)
    x, w, t = make(9, vocab, 64, torch.bfloat16, seed=53)
    x[:, 0] = 1.0
    inf = w.clone()
    inf[:, 0] = -math.inf
    assert ll.linear_cross_entropy_l2wrap_rows(x, inf, t, 9).isnan().all()
    last = torch.full_like(t, vocab - 1)
    one = inf.clone()
    one[vocab - 1] = w[vocab - 1]
    loss = ll.linear_cross_entropy_l2wrap_rows(x, one, last, 9)
    assert (loss.abs() <= 2.0 ** -20 + 64 * U * (x.double() @ w[vocab - 1].double()).abs().max()).all()
    if vocab > 1:
        assert (ll.linear_cross_entropy_l2wrap_rows(x, one, last - 1, 9) == math.inf).all()
        one[0, 3] = math.nan                      # a NaN in a tile of minus infinities
        assert ll.linear_cross_entropy_l2wrap_rows(x, one, last, 9).isnan().all()


@pytest.mark.parametrize("dtype,rows,vocab,c", [(torch.float32, 129, 65536, 2048), (torch.float32, 1025, 65529, 257),
                                                (torch.bfloat16, 4097, 65536, 256), (torch.bfloat16, 2500, 20011, 1400)])
def test_much_work_of_which_some_is_ignored(dtype, rows, vocab, c):
    """Where there is enough to do, the rows that are learned are brought together first."""
    announce("linear loss, much work, some ignored", dtype, rows, vocab, c)
    x, w, t = make(rows, vocab, c, dtype, seed=61)
    full = t.clone()
    g = torch.rand(rows, device=DEV) + 0.1
    r = torch.arange(rows, device=DEV)
    for dead in (r % 3 != 1, r < rows - 1, r % 8 == 0, (r // 70) % 2 == 0):
        t = full.masked_fill(dead, -100)
        y = torch.where(dead[:, None], torch.full_like(x, math.nan), x)
        loss, dx, dw = check(y, w, t, g, rows)
        assert not dx[dead].any()
        del loss, dx, dw
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    none = ll.linear_cross_entropy_l2wrap_rows(a, b, torch.full_like(t, -100), rows)
    assert not none.any() and not any(v.any() for v in torch.autograd.grad(none, (a, b), g))


@pytest.mark.parametrize("dtype", BOTH)
def test_in_a_graph_with_much_work(dtype):
    """The rows are counted on the device: a replay takes other rows than the capture."""
    rows, vocab, c = 1100, 65536, 1024 if dtype == torch.bfloat16 else 256
    announce("linear loss, graph, much work", dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=67)
    g = torch.rand(rows, device=DEV)
    a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()

    def step():
        loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, rows)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b), g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    full = t.clone()
    for k in (1, 2, 5, 1100):
        t.copy_(full.masked_fill(torch.arange(rows, device=DEV) % k != 0, -100))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,c", [(40, 500, 2048), (65, 130, 4000), (1, 3, 5000), (300, 513, 1472), (7, 70, 2999)])
def test_few_tiles_of_many_channels(rows, vocab, c, dtype):
    announce("linear loss, many channels", rows, vocab, c, dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=71)
    t[1::5] = -100
    check(x, w, t, torch.rand(rows, device=DEV) + 0.1, rows)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,c", [(3, 1 << 20, 5), (64, 13000, 333), (20, 33000, 130)])
def test_many_words_of_few_channels(rows, vocab, c, dtype):
    """D is far below its floor for most words: 2^-38 of the largest factor."""
    announce("linear loss, many words", rows, vocab, c, dtype)
    x, w, t = make(rows, vocab, c, dtype, seed=rows + c)
    t[1::7] = -100
    check(x, w, t, torch.rand(rows, device=DEV) + 0.1, rows)
