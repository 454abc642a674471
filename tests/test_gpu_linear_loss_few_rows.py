"""The loss from hidden states and its gradients in fp32 where there are few rows and many
words: the unembedding is not packed first but made three bf16 numbers an element on its
way to the products. Against float64 formulas on the GPU.

Three bf16 numbers, cut off and not rounded, hold an fp32 number whole: the second is
below 2^-7 of it, the third below 2^-15. Six of nine products are formed; those left out
are below 2 2^-22 + 2^-30 of a product, below 2^-20 with room. With u = 2^-24, six sums of n
products are 6 n additions of at most 2u of what is added up (the matrix cores may cut
off). An exponential is within 2^-20 of its value, a result rounded by u; the
exponentials' sum adds 32 words a lane, and joins.
"""

import math

import pytest
import torch

from conftest import announce, load_pkg
from test_gpu_linear_loss import make

pytestmark = pytest.mark.gpu
pkg = load_pkg()
ll = pkg.lm_loss
U = 2.0 ** -24
LEFT_OUT = 2.0 ** -20
DEV = "cuda"


def run(x, w, t, g, num_tokens, ignore=-100):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, num_tokens, ignore)
    return (loss.detach(), *torch.autograd.grad(loss, (a, b), g))


def check(x, w, t, g, num_tokens):
    (rows, c), vocab = x.shape, w.shape[0]
    loss, dx, dw = run(x, w, t, g, num_tokens)
    dead = (t == -100)[:, None]
    x64, w64 = torch.where(dead, 0.0, x.double()), w.double()
    z, size = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    m, top = z.max(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = torch.where(dead, 0, t[:, None])
    ez = (size * (LEFT_OUT + 6 * c * 2 * U)).amax(1, keepdim=True)
    e_lse = ez + (32 + 5 + -(-vocab // 1024) + 17) * 2 * U + 2.0 ** -20 + 2 * U * lse.abs()
    want = torch.where(dead, 0.0, lse - z.gather(1, at))
    miss = (loss[:, None].double() - want).abs()
    assert (miss <= ez + e_lse + 2 * U * (lse.abs() + z.abs().amax(1, keepdim=True))).all()
    gd, s = torch.where(dead, 0.0, g.double()[:, None]), 1e-4 / num_tokens if num_tokens else 0.0
    p, wrap = torch.exp(z - lse), torch.where(dead, 0.0, s * m)
    d = (gd * p).scatter_add(1, at, -gd).scatter_add(1, top, wrap)
    reference = max(float(gd.abs().max()), float(wrap.abs().max())) or 1.0
    de = gd.abs() * p * (ez + e_lse + 2.0 ** -19) + 4 * U * (gd.abs() * p + d.abs()) + reference * 2.0 ** -120
    de = de.scatter_add(1, at, gd.abs() * 4 * U).scatter_add(1, top, wrap.abs() * 8 * U + s * ez)
    for got, dm, e, om, terms in ((dx, d, de, w64, vocab), (dw, d.t(), de.t(), x64, rows)):
        exact, size = dm @ om, dm.abs() @ om.abs()
        # D's factor and its inverse, the shares' sums and the result's rounding: 300 additions
        bound = e @ om.abs() + size * (LEFT_OUT + (6 * terms + 300) * 2 * U) + exact.abs() * 4 * U + 1e-44
        miss = (got.double() - exact).abs()
        assert (miss <= bound).all(), float((miss / bound).max())
    return loss, dx, dw


# tiles of 256 words and of 64 and the vocabulary's end in each; channels that end within
# 32, within a tile of 128 or 256; one tile of 64 rows and two
@pytest.mark.parametrize("rows,vocab,c", [
    (1, 65536, 64), (1, 1 << 22, 8), (2, 65529, 72), (16, 20011, 256), (17, 4099, 1032), (63, 16500, 384), (64, 8000, 1000),
    (64, 30001, 144), (65, 40001, 128), (100, 2051, 2056), (127, 65530, 96), (128, 70, 65528), (128, 33000, 264), (3, 128, 32776)])
def test_sizes(rows, vocab, c):
    announce("linear loss, few rows", rows, vocab, c)
    x, w, t = make(rows, vocab, c, torch.float32, seed=rows + c)
    t[1::7] = -100
    t[0] = vocab - 1
    g = torch.rand(rows, device=DEV) + 0.1
    loss, dx, dw = check(x, w, t, g, rows)
    a = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(a, w, t, rows), a, g)[0], dx)
    b = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(x, b, t, rows), b, g)[0], dw)
    with torch.no_grad():
        assert torch.equal(ll.linear_cross_entropy_l2wrap_rows(x, w, t, rows), loss)


def test_either_side_of_the_rules():
    """Rows and words on both sides of where the form changes, and channels that it does
    not take: the same answers but for the sums' orders."""
    announce("linear loss, few rows, the rules' sides")
    for rows, vocab, c in ((128, 16384, 256), (129, 16384, 256), (128, 16383, 256), (128, 16400, 257), (128, 16400, 260)):
        x, w, t = make(rows, vocab, c, torch.float32, seed=3)
        check(x, w, t, torch.ones(rows, device=DEV) / rows, rows)


@pytest.mark.parametrize("scale_x,scale_w", [(1e-18, 1e18), (1e15, 1e-15), (1e-25, 1.0), (0.0, 1.0), (1.0, 0.0), (30.0, 1.0)])
def test_scales(scale_x, scale_w):
    announce("linear loss, few rows, scales", scale_x, scale_w)
    x, w, t = make(20, 20000, 256, torch.float32, seed=17)
    check(x * scale_x, w * scale_w, t, torch.rand(20, device=DEV), 20)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 0.0])
def test_row_gradients_of_any_size(size):
    announce("linear loss, few rows, row gradients", size)
    x, w, t = make(30, 20000, 256, torch.float32, seed=19)
    g = torch.randn(30, device=DEV) * size
    check(x, w, t, g, 0)
    check(x, w, t, g, 30)


def test_ignored_and_invalid_rows():
    announce("linear loss, few rows, ignored rows")
    x, w, t = make(40, 20000, 256, torch.float32, seed=11)
    g = torch.rand(40, device=DEV) + 0.1
    t[10:20] = -100
    clean = check(x, w, t, g, 40)
    x[10], x[11], x[12] = math.nan, math.inf, 1e38
    for p, q in zip(run(x, w, t, g, 40), clean):
        assert torch.equal(p, q)
    t[3], t[4], t[5] = -1, 20000, 20100                  # no such word, but within a tile
    loss, dx, dw = run(x, w, t, g, 40)
    assert loss.isnan().nonzero()[:, 0].tolist() == [3, 4, 5] and dx.isfinite().all() and dw.isfinite().all()
    t[:] = -100
    assert not any(v.any() for v in run(x, w, t, g, 40))


def test_first_of_equal_maxima():
    announce("linear loss, few rows, ties")
    x, w, t = make(5, 17000, 256, torch.float32, seed=23)
    for places in ((5, 6), (63, 64), (100, 200, 255), (255, 256), (300, 900, 16999), (0, 16999)):
        v = w.clone()
        v[list(places)] = 3.0 * x[0] / x[0].norm()
        _, kept = ll._linear_forward(x[:1].contiguous(), v, t[:1], -100)
        assert int(kept[2].view(torch.int32)) == places[0], places
    loss, _, _ = run(x, torch.zeros_like(w), t, torch.ones(5, device=DEV), 5)
    assert (loss - math.log(17000)).abs().max() < 1e-5


def test_nan_and_infinite_numbers():
    """Of a row: its own loss and hidden gradient. Of a word: every row's (inf - inf)."""
    announce("linear loss, few rows, NaN and infinities")
    x, w, t = make(30, 20000, 256, torch.float32, seed=13)
    ones = torch.ones(30, device=DEV)
    clean = run(x, w, t, ones, 30)
    others = torch.arange(30, device=DEV) != 5
    for bad in (math.nan, math.inf, -math.inf):
        y = x.clone()
        y[5, 3] = bad
        loss, dx, _ = run(y, w, t, ones, 30)
        assert loss[5].isnan() and dx[5].isnan().all()
        assert torch.equal(loss[others], clean[0][others]) and torch.equal(dx[others], clean[1][others])
        v = w.clone()
        v[77, 250] = bad
        assert ll.linear_cross_entropy_l2wrap_rows(x, v, t, 30).isnan().all()


def test_in_a_graph():
    announce("linear loss, few rows, graph")
    rows, vocab, c = 70, 9000, 512
    x, w, t = make(rows, vocab, c, torch.float32, seed=41)
    g = torch.rand(rows, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, w, t, g, rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, w, t, g, rows)
    for seed in range(4):
        x2, w2, t2 = make(rows, vocab, c, torch.float32, seed=100 + seed)
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, run(x, w, t, g, rows)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,c", [(70, 300, 12), (1100, 300, 20), (300, 900, 132), (20, 40000, 108)])
def test_rows_that_begin_anywhere(rows, vocab, c, dtype):
    """The C entry points take operands and gradients at any element where c is no
    multiple of 8: one element off a 16-byte boundary, against the same call at one."""
    announce("linear loss, any alignment", rows, vocab, c, dtype)
    native, stream = pkg._native, torch.cuda.current_stream().cuda_stream
    x, w, t = make(rows, vocab, c, dtype, seed=47)
    g = torch.rand(rows, device=DEV)
    code = pkg.neighbors._code(dtype)
    results = []
    for off in (0, 1):
        def placed(v):
            flat = torch.full((v.numel() + 9,), 7.0, dtype=dtype, device=DEV)
            flat[off:off + v.numel()] = v.reshape(-1)
            return flat
        fx, fw, fdx, fdw = placed(x), placed(w), placed(torch.zeros_like(x)), placed(torch.zeros_like(w))
        px, pw, pdx, pdw = (v[off:].data_ptr() for v in (fx, fw, fdx, fdw))
        row = torch.empty(4, rows, device=DEV)
        n = max(native.lib().rwkv_linear_loss_forward_workspace_bytes(rows, vocab, c, code),
                native.lib().rwkv_linear_loss_backward_workspace_bytes(rows, vocab, c, code))
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        native.call("rwkv_linear_loss_forward", px, pw, t.data_ptr(), rows, vocab, c, code, -100, row[0].data_ptr(), row[1].data_ptr(),
                    row[2].data_ptr(), row[3].data_ptr(), ws.data_ptr(), n, stream)
        native.call("rwkv_linear_loss_backward", px, pw, t.data_ptr(), row[1].data_ptr(), row[2].data_ptr(), row[3].data_ptr(),
                    g.data_ptr(), 1e-4 / rows, rows, vocab, c, code, -100, pdx, pdw, ws.data_ptr(), n, stream)
        torch.cuda.synchronize()
        for flat, v in ((fdx, x), (fdw, w)):
            assert (flat[:off] == 7).all() and (flat[off + v.numel():] == 7).all()
        results.append((row[0].clone(), fdx[off:off + x.numel()].clone(), fdw[off:off + w.numel()].clone()))
    for p, q in zip(*results):
        assert torch.equal(p, q)


@pytest.mark.parametrize("rows,vocab,c", [(40, 100000, 333), (64, 5000, 1001), (128, 16500, 514), (1, 66, 65535), (100, 9000, 1260)])
def test_rows_of_no_whole_eights(rows, vocab, c):
    announce("linear loss, few rows of no whole eights", rows, vocab, c)
    x, w, t = make(rows, vocab, c, torch.float32, seed=rows + c)
    t[1::7] = -100
    check(x, w, t, torch.rand(rows, device=DEV) + 0.1, rows)


@pytest.mark.parametrize("rows,vocab,c", [(40, 75601, 333), (64, 25200, 1001), (1, 1 << 22, 7), (128, 50001, 514), (100, 20011, 1260), (9, 12288, 2051)])
def test_copied_rows(rows, vocab, c):
    """Rows that begin anywhere, of words enough to be copied to rows that do not."""
    announce("linear loss, few rows, copied", rows, vocab, c)
    x, w, t = make(rows, vocab, c, torch.float32, seed=rows + c)
    t[1::7] = -100
    check(x, w, t, torch.rand(rows, device=DEV) + 0.1, rows)


@pytest.mark.parametrize("rows,vocab,c", [(17, 12288, 1032), (64, 13000, 1000), (100, 16384, 2056), (3, 12300, 4104), (128, 12289, 344)])
def test_many_channels(rows, vocab, c):
    announce("linear loss, few rows, many channels", rows, vocab, c)
    x, w, t = make(rows, vocab, c, torch.float32, seed=rows + c)
    t[1::7] = -100
    check(x, w, t, torch.rand(rows, device=DEV) + 0.1, rows)


@pytest.mark.parametrize("c", [512, 1900])
def test_in_a_graph_of_many_words(c):
    announce("linear loss, few rows, graph, many words", c)
    rows, vocab = 70, 14000
    x, w, t = make(rows, vocab, c, torch.float32, seed=43)
    g = torch.rand(rows, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, w, t, g, rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, w, t, g, rows)
    for seed in range(4):
        x2, w2, t2 = make(rows, vocab, c, torch.float32, seed=200 + seed)
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, run(x, w, t, g, rows)):
            assert torch.equal(p, q)
