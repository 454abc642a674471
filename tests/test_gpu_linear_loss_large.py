"""The loss from hidden states where operands pass 2^31 elements or 2^32 bytes, against
fp32 arithmetic in pieces: the loss of every row, the hidden gradient, and rows of
the weight gradient from all over the vocabulary."""

import pytest
import torch

from conftest import announce, load_pkg

pytestmark = pytest.mark.gpu
ll = load_pkg().lm_loss
DEV = "cuda"


def pieces(n, size):
    return [(i, min(i + size, n)) for i in range(0, n, size)]


@pytest.mark.parametrize("rows,vocab,c,dtype", [
    (40, 600_000, 4096, torch.bfloat16),       # w: 2.46e9 elements
    (40, 300_000, 4096, torch.float32),        # w: 4.9e9 bytes, read where it is
    (150, 290_000, 4095, torch.float32),       # and packed
    (1_100_000, 300, 2048, torch.bfloat16),    # x: 2.25e9 elements
    (70_000, 60_000, 64, torch.bfloat16)])     # 4.2e9 logits, in pieces
def test_offsets_beyond_32_bits(rows, vocab, c, dtype):
    announce("linear loss, large", rows, vocab, c, dtype)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, c, generator=gen, device=DEV, dtype=dtype)
    w = torch.randn(vocab, c, generator=gen, device=DEV, dtype=dtype) * (2.0 / c ** 0.5)
    t = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    t[-1] = vocab - 1
    t[rows // 2] = -100
    g = torch.full((rows,), 1.0 / rows, device=DEV)
    a, b = x.requires_grad_(), w.requires_grad_()
    loss = ll.linear_cross_entropy_l2wrap_rows(a, b, t, 0)
    dx, dw = torch.autograd.grad(loss, (a, b), g)
    loss, live = loss.detach(), t != -100
    with torch.no_grad():
        take = torch.unique(torch.cat([torch.randint(0, rows, (60,), generator=gen, device=DEV),
                                       torch.tensor([0, rows - 1, rows // 2], device=DEV)])) if rows > 1000 else torch.arange(rows, device=DEV)
        xs, ts = x[take].float(), t[take]
        z = torch.cat([xs @ w[i:j].float().t() for i, j in pieces(vocab, 1 << 16)], dim=1)
        lse = torch.logsumexp(z.double(), 1)
        want = torch.where(live[take], lse - z.double().gather(1, ts.clamp(min=0)[:, None])[:, 0], 0.0)
        # a logit is below 12 here and its fp32 sums within 2^-13 of it on either side
        assert (loss[take].double() - want).abs().max() < 5e-3
        d = torch.exp(z - lse[:, None].float())
        d[torch.arange(len(take), device=DEV), ts.clamp(min=0)] -= 1.0
        d *= torch.where(live[take], g[take], 0.0)[:, None]
        exact = sum(d[:, i:j] @ w[i:j].float() for i, j in pieces(vocab, 1 << 16))
        # result and, for bf16, D are rounded to bf16: 2^-8 each
        scale = exact.norm(dim=1, keepdim=True)
        assert ((dx[take].float() - exact).norm(dim=1, keepdim=True) <= 2.0 ** -6 * scale + 1e-12).all()
        assert not dx[rows // 2].any()
        words = torch.unique(torch.cat([torch.randint(0, vocab, (50,), generator=gen, device=DEV), t[-1:], t[:1],
                                        torch.tensor([0], device=DEV)]))
        exact = torch.zeros(len(words), c, device=DEV, dtype=torch.float64)
        for i, j in pieces(rows, 1 << 14):
            zz = x[i:j].float() @ w[words].float().t()
            # the rows' log-sum-exp by way of their losses, which were checked on a sample
            at = torch.where(live[i:j], t[i:j], 0)
            zt = (x[i:j].float() * w[at].float()).sum(1)
            p = torch.exp(zz - (loss[i:j] + zt)[:, None])
            p -= (words[None, :] == t[i:j, None]).float()
            p *= torch.where(live[i:j], g[i:j], 0.0)[:, None]
            exact += p.double().t() @ x[i:j].double()
        got = dw[words].double()
        assert ((got - exact).norm(dim=1) <= 2.0 ** -6 * exact.norm(dim=1) + 1e-12).all()
