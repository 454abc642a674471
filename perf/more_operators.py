"""Performance cases of a training step that keeps neither its logits nor its
dropout masks: the cross entropy of a language model straight from the last
hidden states and the unembedding, with l2wrap, and dropout from a
counter-based generator.

* ``loss``     the loss of every row, from hidden states [rows, c] and the
               unembedding [vocab, c]: a validation pass;
* ``train``    the same, and the gradients of the hidden states and of the
               unembedding;
* ``drop``     dropout of an activation, and the gradient of its input;
* ``add``      dropout of a mixer's output added to the residual stream, and the
               gradients of both.

With ``own`` false, ``run`` computes them with elementary torch operations in
float32. ``exact`` restates them in float64.

The mask. Element i (of the contiguous tensor) is kept where the 16-bit number
u_i is below T = round((1 - p) 65536), and then multiplied by 65536 / T. u_8q+2k
and u_8q+2k+1 are the low and the high half of word k of Philox4x32-10 (Salmon,
Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) at
the counter (q mod 2^32, q / 2^32, site, step mod 2^32) and the key (seed mod
2^32, seed / 2^32). ``rng`` is [seed, step] on the GPU.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORED = -100
L2WRAP = 1e-4


# ----------------------------------------------------------------------- cases
def listed():
    return [
        # a byte-level model on a short text: the smallest step
        {"name": "train_bytes", "kind": "train", "dtype": "bf16", "rows": 96, "c": 256, "vocab": 256,
         "weighted": False},
        # the 0.1B model on one short sequence
        {"name": "train_short", "kind": "train", "dtype": "bf16", "rows": 512, "c": 768, "vocab": 65536,
         "weighted": False},
        # its training step, 16 sequences of 512 tokens
        {"name": "train_step", "kind": "train", "dtype": "bf16", "rows": 8192, "c": 768, "vocab": 65536,
         "weighted": False},
        # a wide model
        {"name": "train_wide", "kind": "train", "dtype": "bf16", "rows": 2048, "c": 4096, "vocab": 65536,
         "weighted": False},
        # rows weighted by an advantage or a sequence's length, ragged batch and vocabulary
        {"name": "train_weighted", "kind": "train", "dtype": "bf16", "rows": 1777, "c": 2560, "vocab": 65529,
         "weighted": True},
        # a model trained in float32
        {"name": "train_f32", "kind": "train", "dtype": "f32", "rows": 1024, "c": 1024, "vocab": 32000,
         "weighted": False},
        # validation of one short text, and of a long one
        {"name": "loss_short", "kind": "loss", "dtype": "bf16", "rows": 64, "c": 768, "vocab": 65536,
         "weighted": False},
        {"name": "loss_text", "kind": "loss", "dtype": "bf16", "rows": 4096, "c": 2048, "vocab": 65536,
         "weighted": False},
        # fine-tuning a small batch
        {"name": "drop_small", "kind": "drop", "dtype": "bf16", "rows": 127, "c": 768, "p": 0.1},
        # an embedding's dropout in float32
        {"name": "drop_f32", "kind": "drop", "dtype": "f32", "rows": 8192, "c": 1024, "p": 0.5},
        # a cell of the 0.1B model's training step: bf16 mixer output, float32 residual stream
        {"name": "add_step", "kind": "add", "dtype": "bf16", "residual": "f32", "rows": 8192, "c": 768, "p": 0.1},
        # of a wide model, all in bf16
        {"name": "add_wide", "kind": "add", "dtype": "bf16", "residual": "bf16", "rows": 16384, "c": 4096,
         "p": 0.05},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("loss", "train", "train", "drop", "add"))
    case = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f32"))}
    if kind in ("drop", "add"):
        case["c"] = _log_int(rng, 64, 4096)
        case["rows"] = _log_int(rng, 1, min(16384, (1 << 25) // case["c"]))
        case["p"] = rng.choice((0.05, 0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)))
        if kind == "add":
            case["residual"] = "f32" if case["dtype"] == "f32" else rng.choice(("f32", "bf16"))
        return case
    # a model's width is a multiple of its head size mostly
    case["c"] = 64 * _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 33, 4096)
    case["vocab"] = _log_int(rng, 64, 1 << 17)
    most = (1 << 38) if case["dtype"] == "bf16" else (1 << 36)
    case["rows"] = _log_int(rng, 1, max(1, min(8192, (1 << 29) // case["vocab"],
                                               most // (case["vocab"] * case["c"]))))
    case["weighted"] = rng.random() < 0.3
    return case


# ---------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def prepare(case, seed):
    gen = _gen(seed)
    dt = DTYPES[case["dtype"]]
    rows, c = case["rows"], case["c"]
    if case["kind"] in ("drop", "add"):
        state = {"case": case, "x": _normal(gen, rows, c).to(dt), "rng": torch.tensor([seed * 2654435761 + 11, 40 + seed % 1000], device=DEV),
                 "site": seed % 24}
        if case["kind"] == "add":
            state["residual"] = (3.0 * _normal(gen, rows, c)).to(DTYPES[case["residual"]])
        state["grad"] = _normal(gen, rows, c).to(state["residual"].dtype if case["kind"] == "add" else dt)
        return state
    vocab = case["vocab"]
    # logits of standard deviation 2.5; the target's is lifted by up to 12, as in text that
    # the model mostly foresees
    weight = _normal(gen, vocab, c).mul_(2.5 / math.sqrt(c))
    targets = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    cos = (torch.rand(rows, 1, generator=gen, device=DEV) * (12.0 / (2.5 * math.sqrt(c)))).clamp(max=0.9)
    toward = weight[targets]
    toward = toward / toward.norm(dim=1, keepdim=True)
    noise = _normal(gen, rows, c)
    hidden = cos * math.sqrt(c) * toward + torch.sqrt(1 - cos * cos) * noise
    # the prompts' tokens and the padding are not learned: runs of rows, an eighth of all
    targets = targets.masked_fill((torch.arange(rows, device=DEV) // 16) % 8 == 3, IGNORED)
    kept = max(1, sum(1 for r in range(rows) if (r // 16) % 8 != 3))
    row_grad = torch.full((rows,), 1.0 / kept, device=DEV)
    if case["weighted"]:
        row_grad *= _normal(gen, rows)
    return {"case": case, "hidden": hidden.to(dt), "weight": weight.to(dt), "targets": targets,
            "row_grad": row_grad}


# ------------------------------------------------------------------ plain form
def _plain_loss(state):
    x, w, t = state["hidden"].float(), state["weight"].float(), state["targets"]
    z = x @ w.t()
    m = z.amax(dim=1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(dim=1, keepdim=True))
    kept = t != IGNORED
    at = torch.where(kept, t, 0).unsqueeze(1)
    loss = torch.where(kept, (lse - z.gather(1, at)).squeeze(1), 0.0)
    return loss, x, w, z, m, lse, kept, at


def _plain_train(state):
    loss, x, w, z, m, lse, kept, at = _plain_loss(state)
    rows, vocab = z.shape
    g = (state["row_grad"] * kept).unsqueeze(1)
    ids = torch.arange(vocab, device=DEV)
    top = torch.where(z == m, ids, vocab).amin(dim=1, keepdim=True)      # the first of equals
    d = g * torch.exp(z - lse)
    d.scatter_add_(1, at, -g)
    d.scatter_add_(1, top, (L2WRAP / rows) * m * kept.unsqueeze(1))
    dt = state["hidden"].dtype
    return {"loss": loss, "hidden_grad": (d @ w).to(dt), "weight_grad": (d.t() @ x).to(dt)}


LOW32 = 0xFFFFFFFF


def _plain_words(rng, site, groups):
    """Philox4x32-10 at the counters (0 .. groups - 1, site, step): four int64 tensors below 2^32."""
    q = torch.arange(groups, device=DEV)
    c0, c1 = q & LOW32, q >> 32
    c2, c3 = torch.full_like(q, site), (rng[1] & LOW32).expand_as(q)
    k0, k1 = rng[0] & LOW32, (rng[0] >> 32) & LOW32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57                  # mod 2^64: the high half is masked off its sign
        c0, c1, c2, c3 = (((b >> 32) & LOW32) ^ c1 ^ k0, b & LOW32, ((a >> 32) & LOW32) ^ c3 ^ k1, a & LOW32)
        k0, k1 = (k0 + 0x9E3779B9) & LOW32, (k1 + 0xBB67AE85) & LOW32
    return c0, c1, c2, c3


def _threshold(p):
    return int(round((1.0 - p) * 65536))


def _plain_mask(state):
    n = state["x"].numel()
    words = torch.stack(_plain_words(state["rng"], state["site"], -(-n // 8)), dim=1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:n]
    return (halves < _threshold(state["case"]["p"])).view_as(state["x"])


def _plain_drop(state):
    keep, scale = _plain_mask(state), 65536.0 / _threshold(state["case"]["p"])
    y = torch.where(keep, state["x"].float() * scale, 0.0)
    dx = torch.where(keep, state["grad"].float() * scale, 0.0).to(state["x"].dtype)
    if state["case"]["kind"] == "drop":
        return {"out": y.to(state["x"].dtype), "x_grad": dx}
    r = state["residual"]
    return {"out": (r.float() + y).to(r.dtype), "x_grad": dx, "residual_grad": state["grad"]}


def _run_plain(state):
    kind = state["case"]["kind"]
    if kind == "loss":
        return {"loss": _plain_loss(state)[0]}
    return _plain_train(state) if kind == "train" else _plain_drop(state)


# ------------------------------------------------------------------- framework
def _run_own(state):
    pkg = importlib.import_module("rwkv-rs_amd")
    case = state["case"]
    if case["kind"] in ("loss", "train"):
        hidden, weight = state["hidden"], state["weight"]
        if case["kind"] == "train":
            hidden, weight = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = pkg.lm_loss.linear_cross_entropy_l2wrap_rows(hidden, weight, state["targets"], case["rows"])
        if case["kind"] == "loss":
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (hidden, weight), state["row_grad"])
        return {"loss": loss.detach(), "hidden_grad": dx, "weight_grad": dw}
    x = state["x"].detach().requires_grad_()
    if case["kind"] == "drop":
        y = pkg.dropout.dropout(x, case["p"], state["rng"], state["site"])
        dx, = torch.autograd.grad(y, x, state["grad"])
        return {"out": y.detach(), "x_grad": dx}
    r = state["residual"].detach().requires_grad_()
    y = pkg.dropout.dropout_add(r, x, case["p"], state["rng"], state["site"])
    dr, dx = torch.autograd.grad(y, (r, x), state["grad"])
    return {"out": y.detach(), "x_grad": dx, "residual_grad": dr}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    n = case["rows"] * case["c"]
    if case["kind"] == "drop":
        return {"bytes": 4 * size * n, "flops": 2 * n}
    if case["kind"] == "add":
        res = 2 if case["residual"] == "bf16" else 4
        return {"bytes": (2 * size + 3 * res) * n, "flops": 3 * n}
    operands = size * (n + case["vocab"] * case["c"])
    products = 2 * n * case["vocab"]
    if case["kind"] == "loss":
        return {"bytes": operands + 12 * case["rows"], "flops": products}
    return {"bytes": 2 * operands + 16 * case["rows"], "flops": 3 * products}


# --------------------------------------------------------------------- 64 bits
def _philox_reference(rng, site, groups):
    """The generator once more, on 16-bit limbs: no product leaves 63 bits."""
    seed, step = (int(v) for v in rng.tolist())
    c = [torch.arange(groups, dtype=torch.int64, device=DEV) % (1 << 32),
         torch.arange(groups, dtype=torch.int64, device=DEV) // (1 << 32),
         torch.full((groups,), site, dtype=torch.int64, device=DEV),
         torch.full((groups,), step % (1 << 32), dtype=torch.int64, device=DEV)]
    key = [seed % (1 << 32), (seed >> 32) % (1 << 32)]

    def mul(v, m):
        low, high = v * (m & 0xFFFF), v * (m >> 16)
        mid = high + low // 65536
        return mid // 65536, (mid % 65536) * 65536 + low % 65536
    for i in range(10):
        (ah, al), (bh, bl) = mul(c[0], 0xD2511F53), mul(c[2], 0xCD9E8D57)
        c = [bh ^ c[1] ^ ((key[0] + i * 0x9E3779B9) % (1 << 32)), bl,
             ah ^ c[3] ^ ((key[1] + i * 0xBB67AE85) % (1 << 32)), al]
    return c


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("drop", "add"):
        x = state["x"].double()
        words = _philox_reference(state["rng"], state["site"], (x.numel() + 7) // 8)
        u = torch.stack([h for w in words for h in (w % 65536, w // 65536)], dim=1).flatten()[:x.numel()]
        t = _threshold(case["p"])
        factor = torch.where(u.view(x.shape) < t, 65536 / t, 0.0).double()
        out = {"out": x * factor, "x_grad": state["grad"].double() * factor}
        if case["kind"] == "add":
            out = {"out": out["out"] + state["residual"].double(), "x_grad": out["x_grad"],
                   "residual_grad": state["grad"].double()}
        return out
    x, w = state["hidden"].double().requires_grad_(), state["weight"].double().requires_grad_()
    t = state["targets"]
    kept = (t != IGNORED).double()
    with torch.set_grad_enabled(case["kind"] == "train"):
        z = torch.mm(x, w.t())
        loss = kept * (torch.logsumexp(z, dim=1) - z[torch.arange(len(t), device=DEV), t.clamp(min=0)])
    out = {"loss": loss.detach()}
    if case["kind"] == "train":
        # l2wrap adds its term to the logits' gradient, whatever that is multiplied with
        top = z.detach().max(dim=1)
        wrap = (top.values * kept * (L2WRAP / case["rows"])).detach()
        total = (loss * state["row_grad"].double()).sum() + (
            wrap * z.gather(1, top.indices.unsqueeze(1)).squeeze(1)).sum()
        out["hidden_grad"], out["weight_grad"] = torch.autograd.grad(total, (x, w))
    return out
