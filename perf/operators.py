"""Performance cases of the operators a served or fine-tuned model needs beside
its recurrence: products of a few rows with 4-bit weights, the quantisation of
those weights, and the scores of given tokens (log probability, entropy, top
alternatives) with their gradient.

* ``linear``    rows of activations times a 4-bit weight matrix: one token of a
                few sequences, or a prompt's tokens;
* ``quantize``  a weight matrix to 4 bits, and back to the values it stands for;
* ``scores``    log probability of a given token, entropy and top alternatives
                of every row of logits;
* ``train``     the same, and the gradient of the logits.

With ``own`` false, ``run`` computes them with elementary torch operations in
float32. ``exact`` restates them in float64.

The 4-bit format. A weight is a sign and one of the magnitudes 0, 0.5, 1, 1.5,
2, 3, 4, 6 (a 4-bit float: two exponent bits, one mantissa bit), times the
bfloat16 scale of its group of 32, 64 or 128 inputs. The matrix is stored in
blocks of 16 outputs and 128 inputs, padded with zero weights:
``packed[n, k, g, r, 4 * j + b]`` (uint8) holds the weights of output 16 n + r
at the inputs 128 k + 32 j + 8 g + 2 b (low half) and the next (high half);
``scales[n, k, r, q]`` belongs to output 16 n + r and the inputs from
128 k + group * q on.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ----------------------------------------------------------------------- cases
def listed():
    return [
        # a served step's answers: eight sequences, the five best alternatives
        {"name": "scores_served", "kind": "scores", "dtype": "bf16", "rows": 8, "vocab": 65536, "top": 5},
        # scoring a long text against a model: every token of it
        {"name": "scores_text", "kind": "scores", "dtype": "bf16", "rows": 4096, "vocab": 65536, "top": 20},
        # a byte-level model, many short rows
        {"name": "scores_bytes", "kind": "scores", "dtype": "bf16", "rows": 8192, "vocab": 256, "top": 3},
        # policy gradient with an entropy term
        {"name": "train_policy", "kind": "train", "dtype": "bf16", "rows": 2048, "vocab": 65536, "top": 0},
        # distillation on the top alternatives, float32 logits of a ragged vocabulary
        {"name": "train_distill", "kind": "train", "dtype": "f32", "rows": 256, "vocab": 65529, "top": 32},
        # a projection of the 0.1B model, one sequence
        {"name": "linear_projection", "kind": "linear", "dtype": "bf16", "rows": 1, "in": 768, "out": 768,
         "group": 64},
        # its unembedding, eight sequences
        {"name": "linear_unembed", "kind": "linear", "dtype": "bf16", "rows": 8, "in": 768, "out": 65536,
         "group": 64},
        # the channel mixer's key of a wide model, one sequence
        {"name": "linear_wide", "kind": "linear", "dtype": "bf16", "rows": 1, "in": 4096, "out": 16384,
         "group": 128},
        # a batch that is no multiple of a tile, float32 activations
        {"name": "linear_batch_f32", "kind": "linear", "dtype": "f32", "rows": 17, "in": 2560, "out": 10240,
         "group": 32},
        # a prompt
        {"name": "linear_prompt", "kind": "linear", "dtype": "bf16", "rows": 512, "in": 2048, "out": 8192,
         "group": 64},
        # quantising the unembedding
        {"name": "quantize_unembed", "kind": "quantize", "dtype": "f32", "in": 768, "out": 65536, "group": 64},
        # a small matrix of odd sizes
        {"name": "quantize_odd", "kind": "quantize", "dtype": "bf16", "in": 1000, "out": 777, "group": 128},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("scores", "train", "linear", "linear", "quantize"))
    case = {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "f32"))}
    if kind in ("scores", "train"):
        vocab = _log_int(rng, 64, 1 << 18)
        most = 1 << (28 if kind == "scores" and case["dtype"] == "bf16" else 26)
        rows = _log_int(rng, 1, max(1, min(8192, most // vocab)))
        return {**case, "rows": rows, "vocab": vocab, "top": rng.choice((0, 1, rng.randint(2, 20), rng.randint(2, 64)))}
    group = rng.choice((32, 64, 128))
    d_in = _log_int(rng, 64, 16384)
    if rng.random() < 0.7:
        d_in = 64 * max(1, d_in // 64)
    d_out = _log_int(rng, 64, min(65536, (1 << 26) // d_in))
    case |= {"in": d_in, "out": d_out, "group": group}
    if kind == "linear":
        case["rows"] = _log_int(rng, 1, max(1, min(512, (1 << 33) // (d_in * d_out))))
    return case


# ---------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _scales_and_codes(weight, group):
    """The format's scales [out, groups] (bfloat16) and codes [out, inputs padded to 128] (uint8)."""
    d_out, d_in = weight.shape
    pad = -d_in % 128
    w = torch.nn.functional.pad(weight.float(), (0, pad)).reshape(d_out, -1, group)
    scale = (w.abs().amax(dim=2) * (1.0 / 6.0)).to(torch.bfloat16)
    s, a = scale.float().unsqueeze(2), w.abs()
    # the midpoints between magnitudes; a tie goes to the even mantissa
    code = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s)
            + (a > 2.5 * s) + (a >= 3.5 * s) + (a > 5.0 * s))
    code = torch.where((w < 0) & (code > 0), code + 8, code)
    return scale, code.reshape(d_out, d_in + pad)


def _pack(scale, code, group):
    d_out, d_in = code.shape
    rows = -d_out % 16
    code = torch.nn.functional.pad(code, (0, 0, 0, rows)).reshape(-1, 16, d_in // 128, 4, 4, 4, 2)
    code = code.permute(0, 2, 4, 1, 3, 5, 6)              # n, k, g, r, j, b, half
    packed = (code[..., 0] | (code[..., 1] << 4)).reshape(code.shape[0], d_in // 128, 4, 16, 16)
    scale = torch.nn.functional.pad(scale, (0, 0, 0, rows)).reshape(-1, 16, d_in // 128, 128 // group)
    return packed.contiguous(), scale.transpose(1, 2).contiguous()


def _values(packed, scales, d_out, d_in, group):
    """The weights [out, in] a packed matrix stands for, in float32."""
    n, k = packed.shape[:2]
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=DEV)
    b = packed.reshape(n, k, 4, 16, 4, 4)
    code = torch.stack((b & 15, b >> 4), dim=-1).permute(0, 3, 1, 4, 2, 5, 6)   # n, r, k, j, g, b, half
    v = table[code.reshape(-1).int()].reshape(16 * n, k * 128 // group, group)
    s = scales.transpose(1, 2).reshape(16 * n, k * 128 // group, 1).float()
    return (v * s).reshape(16 * n, 128 * k)[:d_out, :d_in]


def prepare(case, seed):
    gen = _gen(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "quantize":
        return {"case": case, "weight": (0.02 * _normal(gen, case["out"], case["in"])).to(dt)}
    if case["kind"] == "linear":
        d_in, d_out, group = case["in"], case["out"], case["group"]
        packed, scales = _pack(*_scales_and_codes(0.02 * _normal(gen, d_out, d_in), group), group)
        x = _normal(gen, case["rows"], d_in)
        x[:, ::97] *= 8.0                                 # a few channels stand out
        return {"case": case, "packed": packed, "scales": scales, "x": x.to(dt)}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    logits = _normal(gen, rows, vocab).mul_(2.5)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    # text: the given token is mostly a likely one
    lift = 12.0 * torch.rand(rows, 1, generator=gen, device=DEV)
    logits.scatter_add_(1, tokens.unsqueeze(1), lift)
    # every eighth row is under a grammar that leaves about thirty tokens
    some = logits[5::8]
    if some.numel():
        keep = torch.rand(some.shape, generator=gen, device=DEV) < 30.0 / vocab
        keep.scatter_(1, tokens[5::8].unsqueeze(1), True)
        some.masked_fill_(~keep, -math.inf)
    state = {"case": case, "logits": logits.to(dt), "tokens": tokens}
    if case["kind"] == "train":
        state["g_log_prob"] = _normal(gen, rows) / rows            # an advantage
        state["g_entropy"] = -0.01 * torch.rand(rows, generator=gen, device=DEV) / rows
        state["g_top"] = -torch.softmax(_normal(gen, rows, top), dim=1) / rows
    return state


# ------------------------------------------------------------------ plain form
def _plain_scores(logits, tokens, top):
    x = logits.float()
    m = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(dim=1, keepdim=True)
    lse = m + torch.log(total)
    p = e / total
    entropy = torch.log(total).squeeze(1) - torch.where(p > 0, p * (x - m), 0.0).sum(dim=1)
    log_prob = (x.gather(1, tokens.unsqueeze(1)) - lse).squeeze(1)
    # one number orders the alternatives: the logit as an ordered integer, then the lower index
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    order += 0x7FFFFFFF - torch.arange(x.shape[1], device=DEV)
    ids = 0x7FFFFFFF - (torch.topk(order, top, dim=1).values & 0xFFFFFFFF)
    return {"log_prob": log_prob, "entropy": entropy, "top_log_probs": x.gather(1, ids) - lse,
            "top_ids": ids}, x, lse, p


def _plain_train(state):
    case, logits, tokens = state["case"], state["logits"], state["tokens"]
    out, x, lse, p = _plain_scores(logits, tokens, case["top"])
    g, h, t = state["g_log_prob"], state["g_entropy"], state["g_top"]
    inner = (g + t.sum(dim=1)).unsqueeze(1) + h.unsqueeze(1) * (x - lse + out["entropy"].unsqueeze(1))
    grad = torch.where(p > 0, -p * inner, 0.0)
    grad.scatter_add_(1, tokens.unsqueeze(1), g.unsqueeze(1))
    grad.scatter_add_(1, out["top_ids"], t)
    return {**out, "logits_grad": grad.to(logits.dtype)}


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "quantize":
        scale, code = _scales_and_codes(state["weight"], case["group"])
        table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=DEV)
        v = table[code.int()].reshape(case["out"], -1, case["group"]) * scale.float().unsqueeze(2)
        return v.reshape(case["out"], -1)[:, :case["in"]].contiguous()
    if case["kind"] == "linear":
        w = _values(state["packed"], state["scales"], case["out"], case["in"], case["group"])
        return (state["x"].float() @ w.t()).to(state["x"].dtype)
    if case["kind"] == "scores":
        return _plain_scores(state["logits"], state["tokens"], case["top"])[0]
    return _plain_train(state)


# ------------------------------------------------------------------- framework
def _run_own(state):
    pkg = importlib.import_module("rwkv-rs_amd")
    case = state["case"]
    if case["kind"] == "quantize":
        return pkg.w4.dequantize(pkg.w4.quantize(state["weight"], case["group"]))
    if case["kind"] == "linear":
        w = pkg.w4.W4Weight(state["packed"], state["scales"], case["out"], case["in"], case["group"])
        return pkg.w4.linear(state["x"], w)
    logits = state["logits"]
    if case["kind"] == "train":
        logits = logits.detach().requires_grad_()
    s = pkg.token_scores.token_scores(logits, state["tokens"], case["top"])
    out = {"log_prob": s.log_prob, "entropy": s.entropy, "top_log_probs": s.top_log_probs,
           "top_ids": s.top_ids}
    if case["kind"] == "train":
        out["logits_grad"], = torch.autograd.grad(
            (s.log_prob, s.entropy, s.top_log_probs), logits,
            (state["g_log_prob"], state["g_entropy"], state["g_top"]))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] in ("scores", "train"):
        n = case["rows"] * case["vocab"]
        per_row = case["rows"] * (8 + 8 + 12 * case["top"])
        if case["kind"] == "scores":
            return {"bytes": size * n + per_row, "flops": 6 * n}
        return {"bytes": 2 * size * n + per_row + case["rows"] * (8 + 4 * case["top"]), "flops": 12 * n}
    n = case["in"] * case["out"]
    stored = n // 2 + 2 * (-(-case["in"] // case["group"])) * case["out"]
    if case["kind"] == "quantize":
        return {"bytes": size * n + 4 * n, "flops": 8 * n}
    return {"bytes": stored + size * case["rows"] * (case["in"] + case["out"]), "flops": 2 * case["rows"] * n}


# --------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantize":
        w = state["weight"].double()
        d_out, d_in, group = case["out"], case["in"], case["group"]
        whole = torch.zeros(d_out, -(-d_in // group) * group, dtype=torch.float64, device=DEV)
        whole[:, :d_in] = w
        whole = whole.view(d_out, -1, group)
        s = (whole.abs().max(dim=2, keepdim=True).values / 6).float().to(torch.bfloat16).double()
        q = whole.abs() / torch.where(s > 0, s, 1.0)
        # spacing 0.5 below 2, 1 below 4, 2 above; round() takes ties to even multiples of the spacing
        step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0))
        q = (torch.round(q / step) * step).clamp(max=6.0)
        return (torch.sign(whole) * q * s).view(d_out, -1)[:, :d_in].contiguous()
    if case["kind"] == "linear":
        n, k = state["packed"].shape[:2]
        code = state["packed"].view(n, k, 4, 16, 4, 4)
        w = torch.empty(n, 16, k, 4, 4, 4, 2, dtype=torch.float64, device=DEV)
        for half in (0, 1):
            c = (code >> (4 * half)) & 15
            e, frac = (c >> 1) & 3, (c & 1).double()
            mag = torch.where(e == 0, 0.5 * frac, (1 + 0.5 * frac) * torch.exp2(e.double() - 1))
            w[..., half] = torch.where(c > 7, -mag, mag).permute(0, 3, 1, 4, 2, 5)
        s = state["scales"].double().permute(0, 2, 1, 3).reshape(16 * n, -1)
        w = w.view(16 * n, 128 * k) * s.repeat_interleave(case["group"], dim=1)
        return state["x"].double() @ w[:case["out"], :case["in"]].t().contiguous()
    x = state["logits"].double()
    log_p = torch.log_softmax(x, dim=1)
    p = torch.exp(log_p)
    entropy = -torch.nan_to_num(p * log_p, nan=0.0).sum(dim=1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    at = state["tokens"].unsqueeze(1)
    out = {"log_prob": log_p.gather(1, at).squeeze(1), "entropy": entropy,
           "top_log_probs": log_p.gather(1, ids), "top_ids": None}
    if case["kind"] == "train":
        weights = torch.zeros_like(p).scatter_(1, at, state["g_log_prob"].double().unsqueeze(1))
        weights.scatter_add_(1, ids, state["g_top"].double())
        slope = torch.nan_to_num(p * (log_p + entropy.unsqueeze(1)), nan=0.0)
        out["logits_grad"] = (weights - p * weights.sum(dim=1, keepdim=True)
                              - state["g_entropy"].double().unsqueeze(1) * slope)
    return out
