"""The loss from hidden states in each of its forms, at sizes at which the form is the one
that runs: rows brought together (rows vocab c from 2^36 on, fp32 2^34), few rows of fp32
whose unembedding is copied first (vocab c from 6 2^22 on, c no multiple of 8), operands
beyond 2^32 bytes held in several planes, means of many rows in a graph.

Bounds of an element are test_gpu_linear_loss.py's, whose docstring derives them."""

import pytest
import torch

from conftest import announce, load_pkg
from test_gpu_linear_loss import BOTH, DEV, check, make

pytestmark = pytest.mark.gpu
pkg = load_pkg()
ll = pkg.lm_loss


@pytest.mark.parametrize("dtype,rows,vocab,c", [(torch.bfloat16, 1100, 65536, 1024), (torch.float32, 300, 65536, 1024)])
def test_rows_brought_together(dtype, rows, vocab, c):
    announce("linear loss, rows brought together", dtype, rows, vocab, c)
    x, w, t = make(rows, vocab, c, dtype, seed=12)
    full = t.clone()
    g = torch.rand(rows, device=DEV) + 0.1
    r = torch.arange(rows, device=DEV)
    for dead in (r < 0, r < rows - 1, r > 0, r % 64 == 63, r >= rows // 2, r < 130, r >= 0):
        t = full.masked_fill(dead, -100)
        y = torch.where(dead[:, None], torch.full_like(x, float("nan")), x)
        loss, dx, dw = check(y, w, t, g, rows)
        assert not dx[dead].any()
        a = y.detach().requires_grad_()                  # each gradient alone
        assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(a, w, t, rows), a, g)[0], dx)
        b = w.detach().requires_grad_()
        assert torch.equal(torch.autograd.grad(ll.linear_cross_entropy_l2wrap_rows(y, b, t, rows), b, g)[0], dw)
        del loss, dx, a, b
    assert not dw.any()


@pytest.mark.parametrize("c", [108, 109])
def test_copied_rows_that_begin_anywhere(c):
    """The C entry points with an unembedding and gradients one element off a 16-byte
    boundary, against the same call at one."""
    rows, vocab = 20, 240000
    announce("linear loss, copied rows, any alignment", rows, vocab, c)
    native, stream = pkg._native, torch.cuda.current_stream().cuda_stream
    x, w, t = make(rows, vocab, c, torch.float32, seed=47)
    t[4] = -100
    g = torch.rand(rows, device=DEV)
    loss, dx, dw = check(x, w, t, g, rows)
    lib = native.lib()
    n = max(lib.rwkv_linear_loss_forward_workspace_bytes(rows, vocab, c, 0),
            lib.rwkv_linear_loss_backward_workspace_bytes(rows, vocab, c, 0))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    for off in (0, 1, 2, 3):
        def placed(v):
            flat = torch.full((v.numel() + 9,), 7.0, device=DEV)
            flat[off:off + v.numel()] = v.reshape(-1)
            return flat
        fx, fw, fdx, fdw = placed(x), placed(w), placed(torch.zeros_like(x)), placed(torch.zeros_like(w))
        px, pw, pdx, pdw = (v[off:].data_ptr() for v in (fx, fw, fdx, fdw))
        row = torch.empty(4, rows, device=DEV)
        native.call("rwkv_linear_loss_forward", px, pw, t.data_ptr(), rows, vocab, c, 0, -100, *(v.data_ptr() for v in row),
                    ws.data_ptr(), n, stream)
        native.call("rwkv_linear_loss_backward", px, pw, t.data_ptr(), *(v.data_ptr() for v in row[1:]), g.data_ptr(),
                    1e-4 / rows, rows, vocab, c, 0, -100, pdx, pdw, ws.data_ptr(), n, stream)
        torch.cuda.synchronize()
        for flat, v in ((fdx, x), (fdw, w)):
            assert (flat[:off] == 7).all() and (flat[off + v.numel():] == 7).all()
        assert torch.equal(row[0], loss)
        assert torch.equal(fdx[off:off + x.numel()].view_as(x), dx) and torch.equal(fdw[off:off + w.numel()].view_as(w), dw)


@pytest.mark.parametrize("dtype", BOTH)
def test_no_rows_at_any_element(dtype):
    announce("linear loss, no rows, any alignment", dtype)
    native, stream = pkg._native, torch.cuda.current_stream().cuda_stream
    vocab, c = 33, 65
    for off in (0, 1, 3):
        flat = torch.full((vocab * c + 9,), 7.0, dtype=dtype, device=DEV)
        native.call("rwkv_linear_loss_backward", None, None, None, None, None, None, None, 0.0, 0, vocab, c,
                    pkg.neighbors._code(dtype), -100, None, flat[off:].data_ptr(), None, 0, stream)
        torch.cuda.synchronize()
        assert not flat[off:off + vocab * c].any()
        assert (flat[:off] == 7).all() and (flat[off + vocab * c:] == 7).all()


def pieces(n, size):
    return [(i, min(i + size, n)) for i in range(0, n, size)]


@pytest.mark.parametrize("rows,vocab,c", [(40, 300_000, 4096), (150, 290_000, 4095)])
def test_planes_beyond_32_bits(rows, vocab, c):
    """fp32 operands beyond 2^32 bytes, read where they are and packed, to bars that an array
    behind the first does not pass unread: without it an element has 11 bits, which moves a
    logit (of 4096 products of standard deviation 2^-5) by 5e-4 and a gradient by 2^-12 of
    itself. With all arrays a logit's some 768 additions, of numbers of 4 at most and 2^-24
    of them each, are within 2e-4; a gradient's, 400 of 2^-24 of itself, within 2^-15, and the
    probabilities' part of a word that is no target by the logit's error."""
    announce("linear loss, large fp32", rows, vocab, c)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, c, generator=gen, device=DEV)
    w = torch.randn(vocab, c, generator=gen, device=DEV) * (2.0 / c ** 0.5)
    t = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    t[-1], t[rows // 2] = vocab - 1, -100
    g = torch.full((rows,), 1.0 / rows, device=DEV)
    a, b = x.requires_grad_(), w.requires_grad_()
    loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, 0)
    dx, dw = torch.autograd.grad(loss, (a, b), g)
    with torch.no_grad():
        live, loss = t != -100, loss.detach()
        z = torch.cat([x.double() @ w[i:j].double().t() for i, j in pieces(vocab, 1 << 15)], dim=1)
        at = t.clamp(min=0)[:, None]
        lse = torch.logsumexp(z, 1, keepdim=True)
        want = torch.where(live, (lse - z.gather(1, at))[:, 0], 0.0)
        assert (loss.double() - want).abs().max() < 2.5e-4
        d = torch.exp(z - lse).scatter_add(1, at, torch.full_like(lse, -1.0)) * torch.where(live, g, 0.0).double()[:, None]
        exact = sum(d[:, i:j] @ w[i:j].double() for i, j in pieces(vocab, 1 << 15))
        assert ((dx.double() - exact).norm(dim=1) <= 2.0 ** -14 * exact.norm(dim=1)).all()
        assert not dx[rows // 2].any()
        words = torch.randint(0, vocab, (200,), generator=gen, device=DEV)
        for take, bar in ((t[live], 2.0 ** -14), (words[~torch.isin(words, t)], 2.0 ** -14 + 2.5e-4)):
            exact = d[:, take].t() @ x.double()
            assert ((dw[take].double() - exact).norm(dim=1) <= bar * exact.norm(dim=1)).all()


@pytest.mark.parametrize("rows", [8192, 300_000, 1_200_000])
def test_the_mean_of_many_rows_in_a_graph(rows):
    """Sums over many rows beside the kernels: each replay as the eager call."""
    announce("linear loss, the mean in a graph", rows)
    x, w, t = make(rows, 40, 64, torch.bfloat16, seed=3)
    full = t.clone()
    a, b = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()

    def step():
        loss = ll.linear_cross_entropy_l2wrap(a, b, t)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in (1, 2, 3, 5, 7, rows):
        t.copy_(full.masked_fill(torch.arange(rows, device=DEV) % k != 0, -100))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for p, q in zip(got, step()):
            assert torch.equal(p, q)
