"""Dropout on the GPU against the generator in plain torch: every element's fate,
values rounded once, sizes and alignments at which vectors end, gradients, streams
and graphs. The results are compared bit for bit: fp32 products and sums of two
numbers, rounded once, have one value, but that a product and the addition behind it
may be one operation (within 2^-24 of the larger of the two)."""

import math

import pytest
import torch

from conftest import announce, load_pkg

pytestmark = pytest.mark.gpu
dr = load_pkg().dropout
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def rng_of(seed=123456789012345, step=3):
    return torch.tensor([seed, step], device=DEV)


def scale_of(p):
    kept = dr.keep_probability(p)
    return 1.0 / kept if kept else 0.0


def expected(x, p, rng, site):
    keep = dr.keep_mask(x.shape, p, rng, site)
    return torch.where(keep, x.float() * torch.tensor(scale_of(p), dtype=F32, device=DEV), 0.0), keep


def normal(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.937, 1.0])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 2047, 2048, 2049, 100003])
def test_values_and_gradient(n, p, dtype):
    announce("dropout", n, p, dtype)
    rng, site = rng_of(), n % 5
    x, g = normal(n, dtype, 1).requires_grad_(), normal(n, dtype, 2)
    y = dr.dropout(x, p, rng, site)
    want, keep = expected(x.detach(), p, rng, site)
    assert y.dtype == dtype and torch.equal(y, want.to(dtype))
    dx, = torch.autograd.grad(y, x, g)
    assert dx.dtype == dtype and torch.equal(dx, expected(g, p, rng, site)[0].to(dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rdtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1,), (3, 5), (2, 9, 64), (127, 768), (33, 100)])
def test_add(shape, rdtype, dtype):
    announce("dropout_add", shape, rdtype, dtype)
    rng = rng_of(-5, 1 << 40)
    for p in (0.1, 0.5):
        r, x = normal(shape, rdtype, 3).requires_grad_(), normal(shape, dtype, 4).requires_grad_()
        y = dr.dropout_add(r, x, p, rng, 4294967295)
        want, keep = expected(x.detach(), p, rng, 4294967295)
        total = r.detach().double() + want.double()
        # the product's rounding or none, the sum's, and the type's
        bound = (want.double().abs() + total.abs()) * 2.0 ** -24 + total.abs() * (2.0 ** -8 if rdtype == BF else 2.0 ** -24)
        assert y.dtype == rdtype and ((y.double() - total).abs() <= bound).all()
        assert torch.equal(y[~keep], r.detach()[~keep])
        g = normal(shape, rdtype, 5)
        dres, dx = torch.autograd.grad(y, (r, x), g)
        assert torch.equal(dres, g) and torch.equal(dx, expected(g, p, rng, 4294967295)[0].to(dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("offset", [1, 2, 5])
def test_any_alignment_and_stride(offset, dtype):
    announce("dropout alignment", offset, dtype)
    rng, base = rng_of(), normal(5000, dtype, 6)
    x = base[offset:offset + 4001]
    assert torch.equal(dr.dropout(x, 0.3, rng), dr.dropout(x.clone(), 0.3, rng))
    square = normal((60, 70), dtype, 7)
    assert torch.equal(dr.dropout(square.t(), 0.3, rng), dr.dropout(square.t().contiguous(), 0.3, rng))
    r = base[offset + 1:offset + 4002]
    assert torch.equal(dr.dropout_add(r, x, 0.3, rng), dr.dropout_add(r.clone(), x.clone(), 0.3, rng))
    # a gradient of another layout, and a broadcast input
    a = square.t().requires_grad_()
    g = normal((60, 70), dtype, 8).t()
    assert torch.equal(torch.autograd.grad(dr.dropout(a, 0.3, rng), a, g)[0], expected(g, 0.3, rng, 0)[0].to(dtype))
    row = normal(64, dtype, 9).requires_grad_()
    y = dr.dropout(row.expand(50, 64), 0.5, rng)
    y.float().sum().backward()
    keep = dr.keep_mask((50, 64), 0.5, rng)
    # sums of at most 50 twos
    assert torch.equal(row.grad.float(), 2.0 * keep.float().sum(0))


def test_what_is_dropped_is_zero():
    announce("dropout of NaN and infinities")
    rng = rng_of()
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.full((1000,), bad, device=DEV)
        keep = dr.keep_mask((1000,), 0.5, rng)
        y = dr.dropout(x, 0.5, rng)
        assert (y[~keep] == 0).all() and not y[keep].isfinite().any()
        r = normal(1000, F32, 1)
        assert torch.equal(dr.dropout_add(r, x, 0.5, rng)[~keep], r[~keep])
        a = normal(1000, F32, 2).requires_grad_()
        dx, = torch.autograd.grad(dr.dropout(a, 0.5, rng), a, x)
        assert (dx[~keep] == 0).all()
    # p = 1 leaves nothing, whatever it is
    assert not dr.dropout(torch.full((77,), math.nan, device=DEV), 1.0, rng).any()
    assert dr.dropout(torch.zeros(0, 5, device=DEV), 0.5, rng).shape == (0, 5)


def test_counters_beyond_32_bits():
    """Element 2^35 + 8 k draws at counter 2^32 + k."""
    n = (1 << 35) + 4096
    if torch.cuda.mem_get_info()[0] < 5 * n:
        pytest.skip("needs 160 GiB of free memory")
    announce("dropout of 2^35 elements")
    x = torch.ones(n, dtype=BF, device=DEV)
    y = dr.dropout(x, 0.5, rng_of(), 9)
    q = torch.arange(512, device=DEV)
    one = torch.ones_like(q)
    words = torch.stack(dr._philox(q, one, 9 * one, 3 * one, torch.tensor(123456789012345, device=DEV)), dim=1)
    keep = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1) < 32768
    assert torch.equal(y[1 << 35:] != 0, keep)
    assert torch.equal(y[:4096] != 0, dr.keep_mask((4096,), 0.5, rng_of(), 9))


def test_second_derivative_and_changed_rng():
    announce("dropout, second derivative")
    rng = rng_of()
    x = normal(300, F32, 1).requires_grad_()
    y = dr.dropout(x * x, 0.4, rng)
    gx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    ggx, = torch.autograd.grad(gx.sum(), x)
    keep = dr.keep_mask((300,), 0.4, rng)
    assert torch.allclose(ggx, torch.where(keep, 2 * scale_of(0.4), 0.0), rtol=1e-6)
    y = dr.dropout(x, 0.4, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda z: dr.dropout(z, 0.4, rng), (x.detach(),), (torch.ones(300, device=DEV),))


def test_streams_and_graph():
    """Two streams at a time; and a captured step that counts itself, replayed: another
    mask each time, the backward's the forward's own."""
    announce("dropout, streams and graph")
    x, r, g = normal((200, 128), BF, 1), normal((200, 128), F32, 2), normal((200, 128), F32, 3)
    rng = rng_of(77, 0)
    a, b = x.clone().requires_grad_(), r.clone().requires_grad_()

    def step():
        mine = rng.clone()
        rng[1] += 1
        y = dr.dropout_add(b, a, 0.25, mine, 6)
        return (y.detach(), *torch.autograd.grad(y, (b, a), g))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    out = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            out.append(dr.dropout_add(r, x, 0.25, rng, i))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i, y in enumerate(out):
        assert torch.equal(y, dr.dropout_add(r, x, 0.25, rng, i))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    seen = []
    for replay in range(4):
        rng[1] = 10 + replay
        graph.replay()
        torch.cuda.synchronize()
        assert int(rng[1]) == 11 + replay
        rng[1] = 10 + replay
        for p, q in zip(captured, step()):
            assert torch.equal(p, q)
        seen.append(captured[0].clone())
    assert not any(torch.equal(seen[i], seen[j]) for i in range(4) for j in range(i))


def test_refusals():
    announce("dropout refusals")
    x, rng = normal((4, 5), F32), rng_of()
    for bad, exc in [(lambda: dr.dropout(x.cpu(), 0.1, rng.cpu()), ValueError), (lambda: dr.dropout(x, 0.1, rng.cpu()), ValueError),
                     (lambda: dr.dropout(x, 0.1, rng.int()), ValueError), (lambda: dr.dropout(x, 0.1, rng[:1]), ValueError),
                     (lambda: dr.dropout(x, -0.1, rng), ValueError), (lambda: dr.dropout(x, 1.1, rng), ValueError),
                     (lambda: dr.dropout(x, math.nan, rng), ValueError), (lambda: dr.dropout(x, 0.1, rng, -1), ValueError),
                     (lambda: dr.dropout(x, 0.1, rng, 1 << 32), ValueError), (lambda: dr.dropout(x.half(), 0.1, rng), TypeError),
                     (lambda: dr.dropout_add(x, x[:2], 0.1, rng), ValueError), (lambda: dr.dropout_add(x[0], x, 0.1, rng), ValueError),
                     (lambda: dr.dropout_add(x.double(), x, 0.1, rng), TypeError),
                     (lambda: dr.dropout_add(x, x.cpu(), 0.1, rng), ValueError)]:
        with pytest.raises(exc):
            bad()
