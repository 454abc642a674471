"""Token scores and their gradient on the GPU against float64 formulas, with
masks that leave a row little or nothing, ties, ragged and long vocabularies."""

import math

import pytest
import torch

from conftest import announce, load_pkg

pytestmark = pytest.mark.gpu
pkg = load_pkg()
ts = pkg.token_scores
LOWEST = {torch.float32: torch.finfo(torch.float32).min, torch.bfloat16: torch.finfo(torch.bfloat16).min}
BOTH = [torch.float32, torch.bfloat16]


def make(rows, vocab, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * scale).to(dtype)
    return x, torch.randint(0, vocab, (rows,), generator=g)


def reference(x, tokens, top):
    """In float64, by the definition; rows without a distribution NaN and -1."""
    d = x.double()
    m = d.max(1, keepdim=True).values
    log_p = d - m - torch.log(torch.exp(d - m).sum(1, keepdim=True))
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)
    valid = torch.isfinite(m.squeeze(1)) & ~d.isnan().any(1)
    log_p[~valid], entropy[~valid] = math.nan, math.nan
    ids = torch.sort(d, dim=1, descending=True, stable=True).indices[:, :top]
    top_lp = log_p.gather(1, ids)
    ids[~valid] = -1
    inside = (tokens >= 0) & (tokens < x.shape[1])
    lp = log_p.gather(1, tokens.clamp(0, x.shape[1] - 1).unsqueeze(1)).squeeze(1)
    lp[~inside] = math.nan
    return lp, entropy, top_lp, ids, log_p, p


def sum_error(vocab):
    """Relative error of a sum of positive fp32 terms: a thread adds at most
    vocab / 64 of them and the threads' sums take 32 additions, 2^-24 each; a
    term's exponential is within 2^-21 (its argument, rounded twice, is below
    2^3 where it counts)."""
    return (vocab / 64 + 32) * 2.0 ** -24 + 2.0 ** -21


def check(x, tokens, top):
    out = ts.token_scores(x.cuda(), tokens.cuda(), top)
    lp, entropy, top_lp, ids, _, _ = reference(x, tokens, top)
    assert torch.equal(out.top_ids.cpu(), ids)
    e = sum_error(x.shape[1])
    for got, want, rel in ((out.log_prob, lp, 2.0 ** -22), (out.top_log_probs, top_lp, 2.0 ** -22),
                           (out.entropy, entropy, 4 * e)):
        assert got.dtype == torch.float32
        got = got.cpu().double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        fine = want.isfinite()
        # log p is x - m - log s: two roundings of its size and the sum's error; the
        # terms of the entropy, log s and the mean of d, are together at most twice log vocab
        bound = rel * want[fine].abs() + (2 + 2 * math.log(x.shape[1])) * 2.0 ** -22 + 4 * e
        err = (got[fine] - want[fine]).abs()
        assert (err <= bound).all(), float((err / bound).max())
    return out


VOCABS = (1, 2, 3, 63, 64, 65, 127, 256, 300, 511, 1000, 2048, 4097, 8192, 9001, 16384, 20000, 32768, 50001, 65529,
          65536, 65544, 100003, 131072, 200000)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", VOCABS)
def test_forward(vocab, dtype):
    for rows, top in ((1, min(vocab, 5)), (5, min(vocab, 64)), (3, 0), (2, 1)):
        announce("token scores", rows, vocab, top, dtype)
        check(*make(rows, vocab, dtype, seed=vocab + top), top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,top", [(64, 1000, 20), (300, 4096, 3), (700, 256, 64), (1100, 97, 10),
                                            (2100, 33, 2), (40, 65536, 20), (300, 20011, 7), (40, 65536, 32),
                                            (40, 65536, 33), (600, 65536, 64), (300, 300, 33), (64, 2000, 33),
                                            (500, 640, 64), (90, 1024, 64), (64, 4096, 48), (700, 8000, 40)])
def test_forward_many_rows(rows, vocab, top, dtype):
    announce("token scores rows", rows, vocab, top, dtype)
    check(*make(rows, vocab, dtype, seed=7), top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [100, 1025, 5000, 65536, 70001, 150000])
def test_masks_and_ties(vocab, dtype):
    announce("token scores masks", vocab, dtype)
    x, tokens = make(16, vocab, dtype, seed=3)
    x[0] = -math.inf                                     # nothing is left
    x[1, 1:] = -math.inf                                 # one token
    tokens[1] = 0
    x[2, 7:] = -math.inf                                 # a few, and the given token masked
    tokens[2] = vocab - 1
    x[3] = 1.25                                          # all alike
    x[4] = LOWEST[dtype]                                 # a mask by the lowest value, everywhere
    x[5, 3:] = LOWEST[dtype]
    x[6, vocab // 2] = math.nan
    x[7, vocab - 1] = math.inf
    x[8] = torch.arange(vocab, dtype=torch.float32).to(dtype) / 64     # rising, in bf16 with long ties
    x[9] = -torch.arange(vocab, dtype=torch.float32).to(dtype) / 64
    x[10] = torch.round(x[10].float()).to(dtype)         # thousands of ties at every level
    x[11, :vocab // 2] += 60.0                           # all of the mass in one half
    x[12] *= 40.0                                        # nearly a one-hot row
    x[13] = -0.0
    x[13, ::2] = 0.0                                     # zeros of both signs are equal
    tokens[14], tokens[15] = -1, vocab
    for top in (0, 1, 20, 32, 33, 64):
        check(x, tokens, top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [4096, 65536, 140000])
@pytest.mark.parametrize("stride", [64, 512, 1024, 8192])
def test_alternatives_that_lie_unevenly(vocab, stride, dtype):
    """The largest logits at one distance from each other, in one run, and all
    rising: selection may not rely on their being spread out."""
    announce("token scores uneven", vocab, stride, dtype)
    x, tokens = make(3, vocab, dtype, seed=5, scale=0.5)
    x[0, ::stride] += 16.0
    x[1, vocab // 3: vocab // 3 + stride] += 16.0
    x[2] = torch.sort(x[2].float()).values.to(dtype)
    check(x, tokens, 64)


def gradient(x, tokens, top, g, h, t):
    """Of sum g log_prob + h entropy + t top_log_probs, by the formula in float64."""
    lp, entropy, _, ids, log_p, p = reference(x, tokens, top)
    V = x.shape[1]
    own = torch.zeros_like(p)
    inside = (tokens >= 0) & (tokens < V)
    own.scatter_add_(1, tokens.clamp(0, V - 1).unsqueeze(1), (g * inside).unsqueeze(1))
    if top:
        own.scatter_add_(1, ids.clamp(min=0), t)
    inner = (g + t.sum(1)).unsqueeze(1) + h.unsqueeze(1) * (log_p + entropy.unsqueeze(1))
    grad = own - torch.where(p > 0, p * inner, torch.zeros_like(p))
    grad[entropy.isnan()] = math.nan
    size = torch.where(p > 0, p * ((g.abs() + t.abs().sum(1)).unsqueeze(1) + h.abs().unsqueeze(1)
                                   * (log_p.abs() + entropy.abs().unsqueeze(1))), torch.zeros_like(p))
    return grad, own, size


def run_gradient(x, tokens, top, g, h, t):
    xg = x.cuda().requires_grad_()
    out = ts.token_scores(xg, tokens.cuda(), top)
    pairs = [(o, w) for o, w in ((out.log_prob, g), (out.entropy, h), (out.top_log_probs, t)) if w is not None]
    return torch.autograd.grad([o for o, _ in pairs], xg, [w.float().cuda() for _, w in pairs])[0]


def weights(rows, top, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, generator=gen, dtype=torch.float64).float().double(),
            torch.randn(rows, generator=gen, dtype=torch.float64).float().double(),
            torch.randn(rows, top, generator=gen, dtype=torch.float64).float().double())


def check_gradient(x, tokens, top, seed=11):
    g, h, t = weights(x.shape[0], top, seed)
    got = run_gradient(x, tokens, top, g, h, t)
    assert got.dtype == x.dtype and got.shape == x.shape
    got = got.cpu().double()
    want, own, size = gradient(x, tokens, top, g, h, t)
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    # p has the error of log p (log s's, the difference's own 2^-22 |log p| and the
    # exponential's), the sums of the weights a rounding each, then one for the type
    e = 4 * sum_error(x.shape[1]) + (2 * math.log(x.shape[1]) + 40) * 2.0 ** -22
    bound = (2 * e * size + (top + 4) * 2.0 ** -23 * (size + own.abs())
             + (2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -23) * want.abs() + 1e-37)
    err = (got - want).abs()
    assert (err[fine] <= bound[fine]).all(), float((err[fine] / bound[fine]).max())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 63, 20), (4, 64, 64), (33, 1000, 0), (9, 4097, 5),
                                            (300, 300, 10), (600, 97, 1), (7, 65536, 32), (3, 65529, 64), (2, 131072, 20),
                                            (2, 100003, 3)])
def test_gradient(rows, vocab, top, dtype):
    announce("token scores gradient", rows, vocab, top, dtype)
    check_gradient(*make(rows, vocab, dtype, seed=rows), top)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [100, 5000, 65536])
def test_gradient_of_masked_rows(vocab, dtype):
    announce("token scores gradient masks", vocab, dtype)
    x, tokens = make(10, vocab, dtype, seed=4)
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    tokens[1] = 0
    x[2, 7:] = -math.inf
    tokens[2] = vocab - 1                                # the given token is masked
    x[3] = 0.5
    x[4] = LOWEST[dtype]
    x[5, 3:] = LOWEST[dtype]
    x[6, 1] = math.nan
    x[7, 2] = math.inf
    tokens[8], tokens[9] = -1, vocab + 5
    # of what is masked only the token's and the alternatives' own terms are left
    for top in (0, 20):
        check_gradient(x, tokens, top)


@pytest.mark.parametrize("which", ["g", "h", "t", "gh"])
def test_gradient_of_some_outputs(which):
    announce("token scores gradient of", which)
    x, tokens = make(6, 700, torch.float32, seed=8)
    g, h, t = weights(6, 9, 12)
    zero = [torch.zeros_like(w) for w in (g, h, t)]
    full = [w if n in which else z for n, w, z in zip("ght", (g, h, t), zero)]
    some = [w if n in which else None for n, w in zip("ght", (g, h, t))]
    want = run_gradient(x, tokens, 9, *full)
    assert torch.equal(run_gradient(x, tokens, 9, *some), want)


def test_gradient_against_differences():
    """(L(x + e v) - L(x - e v)) / 2e along random v. The outputs are within 2e-6
    of their values here (vocabulary 50, |log p| below 8), 2e-6 / e for each unit of
    weight; the third derivative along |v| <= 1 is below 8 (6 for log sum exp's
    third cumulant, the entropy's with log p's factor) a unit of weight."""
    announce("token scores differences")
    rows, vocab, top, e = 4, 50, 6, 2.0 ** -6
    gen = torch.Generator().manual_seed(2)
    # logits 0.1 apart: a step of 2^-6 changes no order
    x = torch.stack([torch.randperm(vocab, generator=gen) for _ in range(rows)]).float() * 0.1
    tokens = torch.randint(0, vocab, (rows,), generator=gen)
    g, h, t = weights(rows, top, 13)
    grad = run_gradient(x, tokens, top, g, h, t).cpu().double()

    def loss(z):
        o = ts.token_scores(z.cuda(), tokens.cuda(), top)
        return float((o.log_prob.cpu().double() * g).sum() + (o.entropy.cpu().double() * h).sum()
                     + (o.top_log_probs.cpu().double() * t).sum())
    mass = float(g.abs().sum() + 8 * h.abs().sum() + t.abs().sum())
    for _ in range(8):
        v = torch.rand(rows, vocab, generator=gen) * 2 - 1
        up, down = x + e * v, x - e * v
        step = (up.double() - down.double()) / (2 * e)
        diff = (loss(up) - loss(down)) / (2 * e)
        assert abs(diff - float((grad * step).sum())) <= mass * (2e-6 / e + 8 * e * e / 6)


def test_shapes_streams_and_graphs():
    announce("token scores shapes")
    x, tokens = make(6, 1000, torch.bfloat16, seed=9)
    out = check(x, tokens, 4)
    x, tokens = x.cuda(), tokens.cuda()
    cube = ts.token_scores(x.view(2, 3, 1000), tokens.view(2, 3).to(torch.int32), 4)
    assert cube.log_prob.shape == (2, 3) and cube.top_ids.shape == (2, 3, 4)
    for a, b in zip(out, cube):
        assert torch.equal(a, b.reshape(a.shape))
    assert torch.equal(ts.token_scores(x.view(2, 3, 1000)[:, 1], tokens.view(2, 3)[:, 1]).log_prob, cube.log_prob[:, 1])
    one = ts.token_scores(x[0], tokens[0], 2)
    assert one.log_prob.shape == () and one.top_ids.shape == (2,) and torch.equal(one.entropy, out.entropy[0])
    none = ts.token_scores(x[:0], tokens[:0], 3)
    assert none.log_prob.shape == (0,) and none.top_ids.shape == (0, 3)
    flat = torch.randn(1 + 3 * 1000, device="cuda")
    odd = flat[1:].view(3, 1000)                              # rows that begin anywhere
    for a, b in zip(ts.token_scores(odd, tokens[:3], 5), ts.token_scores(odd.clone(), tokens[:3], 5)):
        assert torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        there = ts.token_scores(x, tokens, 4)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(there, out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,vocab", [(2, 65536), (40, 1000), (1, 150000)])
def test_replays(rows, vocab):
    announce("token scores graph", rows, vocab)
    xs = [make(rows, vocab, torch.bfloat16, seed=20 + i) for i in range(3)]
    want = [ts.token_scores(x.cuda(), t.cuda(), 10) for x, t in xs]
    x, tokens = xs[0][0].cuda(), xs[0][1].cuda()
    ts.token_scores(x, tokens, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ts.token_scores(x, tokens, 10)
    for (a, t), w in zip(xs + xs, want + want):
        x.copy_(a)
        tokens.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        for got, b in zip(out, w):
            assert torch.equal(got, b)


def test_more_rows_than_a_launch_holds():
    announce("token scores, 2^21 + 5 rows")
    rows, vocab = (1 << 21) + 5, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, vocab, generator=g, device="cuda").requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    out = ts.token_scores(x, tokens, 2)
    w = torch.randn(rows, generator=g, device="cuda")
    grad, = torch.autograd.grad((out.log_prob, out.entropy, out.top_log_probs), x,
                                (w, 2 * w, torch.stack([w, -w], 1)))
    for part in (slice(0, 9), slice((1 << 21) - 4, None)):       # around the cut, alone
        y = x.detach()[part].requires_grad_()
        few = ts.token_scores(y, tokens[part], 2)
        for a, b in zip(out, few):
            assert torch.equal(a[part], b)
        alone, = torch.autograd.grad((few.log_prob, few.entropy, few.top_log_probs), y,
                                     (w[part], 2 * w[part], torch.stack([w[part], -w[part]], 1)))
        assert torch.equal(grad[part], alone)
    want = torch.log_softmax(x.detach().double(), 1).gather(1, tokens[:, None])[:, 0]
    assert (out.log_prob.double() - want).abs().max() < 1e-5


def test_there_is_no_second_derivative():
    announce("token scores, second derivative")
    x, tokens = make(3, 40, torch.float32)
    x = x.cuda().requires_grad_()
    grad, = torch.autograd.grad(ts.token_scores(x, tokens.cuda()).log_prob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_refusals():
    announce("token scores refusals")
    x, tokens = make(4, 30, torch.float32)
    x, tokens = x.cuda(), tokens.cuda()
    for bad, exc in [(lambda: ts.token_scores(x.cpu(), tokens.cpu()), ValueError),
                     (lambda: ts.token_scores(x, tokens.cpu()), ValueError),
                     (lambda: ts.token_scores(x, tokens[:2]), ValueError),
                     (lambda: ts.token_scores(x, tokens.float()), TypeError),
                     (lambda: ts.token_scores(x.half(), tokens), TypeError),
                     (lambda: ts.token_scores(x, tokens, -1), ValueError),
                     (lambda: ts.token_scores(x, tokens, 31), ValueError),
                     (lambda: ts.token_scores(x.repeat(1, 4), tokens, 65), ValueError),
                     (lambda: ts.token_scores(x[:, :0], tokens), ValueError)]:
        with pytest.raises(exc):
            bad()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [1, 100, 700, 5000, 30000, 65536, 140000])
def test_signs_of_certain_rows(vocab, dtype):
    """A token that has all of the probability, or all but a rounding: no log
    probability above zero, no entropy below it."""
    announce("token scores of certain rows", vocab, dtype)
    x, tokens = make(64, vocab, dtype, seed=21)
    top = torch.linspace(0, 90, 64).to(dtype)
    x[:, vocab // 2] += top
    x[:32, :vocab // 2] = -math.inf
    x[:32, vocab // 2 + 1:] = -math.inf
    tokens[:] = vocab // 2
    for k in (0, 1, min(vocab, 33)):
        out = check(x, tokens, k)
        assert (out.log_prob <= 0).all() and (out.top_log_probs <= 0).all() and (out.entropy >= 0).all()


def test_forward_mode_is_refused():
    """Outputs without a tangent would be read as constants."""
    announce("token scores, forward mode")
    fw = torch.autograd.forward_ad
    x, tokens = make(3, 40, torch.float32)
    x, tokens = x.cuda(), tokens.cuda()
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                ts.token_scores(dual, tokens, 2)
        with pytest.raises(NotImplementedError):
            ts.token_scores(dual[0], tokens[0])
        with pytest.raises(NotImplementedError):
            ts.token_scores(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), tokens)
        want = ts.token_scores(x, tokens, 2)                  # no tangent: nothing is lost
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda z: ts.token_scores(z, tokens).log_prob, (x,), (torch.ones_like(x),))
    for a, b in zip(ts.token_scores(x, tokens, 2), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("rows,vocab,top", [(513, 65536, 20), (520, 33000, 32), (513, 70001, 5), (300, 70001, 0)])
def test_many_long_rows(rows, vocab, top, dtype):
    """Rows of several chunks of 32768 (bf16, more than 512 rows, up to 32
    alternatives) or other sizes, masked in one chunk, in all but one and in all."""
    announce("token scores, many long rows", rows, vocab, top, dtype)
    x, tokens = make(rows, vocab, dtype, seed=23)
    chunk, left = 32768, max(top // 2, 1)
    last = (vocab - 1) // chunk * chunk
    x[0, :chunk - left] = -math.inf                      # the first chunk has fewer than `top`
    x[1, :chunk] = -math.inf                             # or none
    x[2, last + left:] = -math.inf                       # so has the last
    x[3, last:] = -math.inf
    x[4, left:] = -math.inf                              # the row has, in its first chunk
    x[5, :vocab - left] = -math.inf                      # in its last
    x[6, 1:vocab - 1] = -math.inf                        # one at each end
    x[7] = -math.inf
    x[8, :chunk] = LOWEST[dtype]                         # far below what follows
    x[9, last:] += 300.0                                 # all of the mass is in the last chunk
    x[10, :chunk] += 300.0                               # in the first
    x[11] = 0.75
    x[12, chunk - 1], x[12, chunk] = 50.0, 50.0          # equal ones on both sides
    x[13, vocab - 1] = math.nan
    x[14, 0] = math.inf
    x[rows - 1] = torch.sort(x[rows - 1].float()).values.to(dtype)
    tokens[2], tokens[4], tokens[5] = vocab - 1, 0, vocab - 1
    check(x, tokens, top)
