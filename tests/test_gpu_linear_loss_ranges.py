"""The loss from hidden states at the ends of its ranges: rows of very different weight,
operands and row gradients near the ends of their types, logits far from zero. Against
float64 formulas on the GPU.

Errors are bounded element by element as in test_gpu_linear_loss.py, whose docstring
derives them, but for what is held to a fixed step: with f_r the larger of a row's |g_r|
and |l2wrap term|, and F the largest of them,

* D is held over 2^e m, e the row's own exponent (2^e <= f_r) and 1 <= m < 2, at 2^13: half
  of fp16's last step, 2^-25, is 2^-37 f_r or less;
* what the weight gradient multiplies with D is x 2^(e - E), 2^E <= F, at 2^13 for x's
  largest: half a step is 2^(E - e) 2^-38 max|x|, and 2^(E - e) <= 2 F / f_r;
* a result below its type's normal numbers is rounded by half its last step (bf16 2^-134).
"""

import math

import pytest
import torch

from conftest import announce, load_pkg
from test_gpu_linear_loss import BOTH, DEV, U, logit_error, make

pytestmark = pytest.mark.gpu
ll = load_pkg().lm_loss


def run(x, w, t, g, num_tokens):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, num_tokens)
    return (loss.detach(), *torch.autograd.grad(loss, (a, b), g))


def check_gradients(x, w, t, g, num_tokens):
    """Each row of the hidden gradient within bounds of that row's own size."""
    (rows, c), vocab = x.shape, w.shape[0]
    loss, dx, dw = run(x, w, t, g, num_tokens)
    dead = (t == -100)[:, None]
    x64, w64 = torch.where(dead, 0.0, x.double()), w.double()
    z = x64 @ w64.t()
    m, top = z.max(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = torch.where(dead, 0, t[:, None])
    ez = logit_error(torch.where(dead, torch.zeros_like(x), x), w)
    e_lse = ez + (32 + 3 + -(-vocab // 1024) + 17) * 2 * U + 2.0 ** -20 + 2 * U * lse.abs()
    gd, s = torch.where(dead, 0.0, g.double()[:, None]), 1e-4 / num_tokens if num_tokens else 0.0
    wrap = torch.where(dead, 0.0, s * m)
    share = gd * torch.exp(z - lse)
    d = share.scatter_add(1, at, -gd).scatter_add(1, top, wrap)
    factor = torch.maximum(gd.abs(), wrap.abs())
    largest = factor.max()
    de = share.abs() * (ez + e_lse + 2.0 ** -19) + 4 * U * (share.abs() + d.abs())
    de = de.scatter_add(1, at, gd.abs() * 4 * U).scatter_add(1, top, wrap.abs() * 8 * U + s * ez)
    bf = x.dtype == torch.bfloat16
    held = d.abs() * (2.0 ** -11 if bf else 2.0 ** -22) + factor * 2.0 ** -37
    again = d.abs() * (2.0 ** -8 if bf else 0.0)
    again = again.scatter(1, at, 0.0).scatter(1, top, 0.0)
    out, of = (2.0 ** -8, 0.0) if bf else (2 * U, 2.0 ** -22)
    last = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2 + 1e-44
    size = d.abs() @ w64.abs()
    exact = d @ w64
    limit = (de + held + again) @ w64.abs() + of * size + 2.0 ** -38 * w64.abs().max() * d.abs().sum(1, keepdim=True)
    limit += size * ((3 * vocab + 64) * 2 * U + 2.0 ** -22) + exact.abs() * out + last
    miss = (dx.double() - exact).abs()
    assert (miss <= limit).all(), float((miss / limit).max())
    exact, size = d.t() @ x64, d.abs().t() @ x64.abs()
    step = (d.abs() / torch.where(factor > 0, factor, 1.0)).sum(0)[:, None] * (largest * 2.0 ** -37 * x64.abs().max())
    limit = (de + held).t() @ x64.abs() + of * size + step + size * ((3 * rows + 64) * 2 * U + 2.0 ** -22)
    limit += exact.abs() * out + last
    miss = (dw.double() - exact).abs()
    assert (miss <= limit).all(), float((miss / limit).max())
    return loss, dx, dw


# tiles of every size, sums and none, rows brought together, few rows of fp32, copied operands
@pytest.mark.parametrize("dtype,rows,vocab,c", [
    (torch.bfloat16, 40, 600, 64), (torch.float32, 40, 600, 64), (torch.bfloat16, 96, 256, 100), (torch.float32, 96, 256, 100),
    (torch.float32, 256, 256, 256), (torch.bfloat16, 700, 3000, 192), (torch.float32, 700, 3000, 192),
    (torch.bfloat16, 1100, 65536, 1024), (torch.float32, 300, 65536, 1024), (torch.float32, 50, 70000, 64)])
def test_rows_of_any_weight(dtype, rows, vocab, c):
    announce("linear loss, rows of any weight", dtype, rows, vocab, c)
    x, w, t = make(rows, vocab, c, dtype, seed=rows, spread=1.0, lift=0.0)
    t[3::9] = -100
    gen = torch.Generator(device=DEV).manual_seed(4)
    weight = (1.0 + torch.rand(rows, generator=gen, device=DEV)) * torch.where(torch.arange(rows, device=DEV) % 2 == 0, 1.0, -1.0)
    weight *= 2.0 ** -(1.5 * (torch.randperm(rows, generator=gen, device=DEV) % 41))
    check_gradients(x, w, t, weight, 0)
    check_gradients(x, w, t, weight, rows)               # l2wrap's term is the larger one for most rows
    weight[::5] = 0.0
    check_gradients(x, w, t, weight * 1e-8, 0)


@pytest.mark.parametrize("dtype", BOTH)
def test_an_infinite_row_gradient(dtype):
    """It is that row's alone, but for the weight gradient."""
    announce("linear loss, an infinite row gradient", dtype)
    x, w, t = make(30, 300, 64, dtype, seed=3)
    g = torch.rand(30, device=DEV) + 0.1
    g[7] = 0.0
    clean = run(x, w, t, g, 30)
    others = torch.arange(30, device=DEV) != 7
    for bad in (math.inf, -math.inf, math.nan):
        g[7] = bad
        loss, dx, dw = run(x, w, t, g, 30)
        assert torch.equal(loss, clean[0]) and torch.equal(dx[others], clean[1][others])
        assert not dx[7].isfinite().any() and not dw[t[7]].isfinite().any()


@pytest.mark.parametrize("dtype,scale_x,scale_w,size", [
    (torch.float32, 120, -120, -10), (torch.float32, -120, 120, -10), (torch.float32, 110, -110, 6), (torch.float32, -124, 110, 10),
    (torch.bfloat16, 120, -120, -10), (torch.bfloat16, -100, 100, -10), (torch.bfloat16, -124, 105, 10)])
def test_operands_near_the_ends_of_their_type(dtype, scale_x, scale_w, size):
    """With row gradients that bring the result back: 1024 rows of 2^-10 whose gradient
    adds up at one word to the size of the operand."""
    announce("linear loss, operands near the ends", dtype, scale_x, scale_w, size)
    x, w, t = make(1024, 50, 64, torch.float32, seed=5)
    t[:] = 7
    x, w = (x.abs() * 2.0 ** scale_x).to(dtype), (w * 2.0 ** scale_w).to(dtype)
    g = torch.full((1024,), 2.0 ** size, device=DEV)
    loss, dx, dw = check_gradients(x, w, t, g, 0)
    assert loss.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [100, 9000, 70000])
def test_logits_far_from_zero(vocab, dtype):
    """Logits of 2^17 and an eighth's multiple up to 8, which both types and fp32 sums hold whole:
    losses and probabilities are those of the multiples alone. The exponentials' sum is
    within ``adds`` roundings and an exponential's 2^-20."""
    announce("linear loss, logits far from zero", vocab, dtype)
    rows = 20
    gen = torch.Generator(device=DEV).manual_seed(vocab)
    x, w = torch.zeros(rows, 64, device=DEV), torch.zeros(vocab, 64, device=DEV)
    x[:, 0], x[:, 1], w[:, 0] = 2.0 ** 8, 1.0, 2.0 ** 9
    w[:, 1] = torch.randint(-64, 65, (vocab,), generator=gen, device=DEV) / 8.0
    t = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    g = torch.rand(rows, generator=gen, device=DEV) + 0.5
    loss, _, dw = run(x.to(dtype), w.to(dtype), t, g, 0)
    z = w[:, 1].double()
    lse = torch.logsumexp(z, 0)
    adds = (32 + 5 + -(-vocab // 1024) + 17) * 2 * U + 2.0 ** -20
    want = lse - z[t]
    assert ((loss.double() - want).abs() <= adds + 4 * U * want).all()
    d = g.double()[:, None] * torch.exp(z - lse)[None, :]
    held = d * (adds + 2.0 ** -19 + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22)) + 2.0 ** -37 * g.double()[:, None]
    d[torch.arange(rows), t] -= g.double()
    held[torch.arange(rows), t] += (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -21) * g.double()
    for channel, of in ((0, 2.0 ** 8), (1, 1.0)):
        exact, size = of * d.sum(0), of * d.abs().sum(0)
        limit = of * held.sum(0) + size * (3 * rows + 64) * 2 * U + exact.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else 2 * U)
        miss = (dw[:, channel].double() - exact).abs()
        assert (miss <= limit).all(), float((miss / limit).max())


@pytest.mark.parametrize("dtype", BOTH)
def test_two_sure_words(dtype):
    """Equal words far from zero share the probability; a word 15 below another has
    exp(-15) of it, which the loss holds to a few steps of the sum, 2^-24 each."""
    announce("linear loss, two sure words", dtype)
    x, w = torch.zeros(1, 64, device=DEV), torch.full((300, 64), 0.0, device=DEV)
    x[:, 0] = 2.0 ** 8
    w[3, 0] = w[70, 0] = 2.0 ** 9
    t, one = torch.tensor([70], device=DEV), torch.ones(1, device=DEV)
    loss, _, dw = run(x.to(dtype), w.to(dtype), t, one, 0)
    assert abs(float(loss) - math.log(2)) <= 2.0 ** -22
    # 2^-20 of an exponential, and the results' rounding: 0.5 itself is held whole
    near = 2.0 ** -8 + 2.0 ** -19 if dtype == torch.bfloat16 else 2.0 ** -18
    assert abs(float(dw[3, 0]) / 128 - 1) <= near and abs(float(dw[70, 0]) / -128 - 1) <= near
    x[:, 0], w[:, 0] = 1.0, -40.0
    w[3, 0], w[70, 0] = 15.0, 30.0
    loss, _, _ = run(x.to(dtype), w.to(dtype), t, one, 0)
    assert abs(float(loss) - math.log1p(math.exp(-15.0))) <= 2.0 ** -22
