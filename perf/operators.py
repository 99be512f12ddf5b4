"""What is measured of the clear half of the model: the operators of `perseus_b200.clear` that stand on either side of the
encrypted decode. A client runs its prompts in the clear to obtain the K and V rows that the encrypted caches hold
(`linear`, `prompt_attention`), scores hidden states against a vocabulary (`vocab_loss`), and fits the head and the MLP
to the polynomials that the encrypted step evaluates (`vocab_loss_grad`, `linear_grad`).

`own` false: the plain forms below, elementary torch operations in 32 bits. `own` true: the framework's operators.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GELU_BOUND = 3.0  # the bound of the MLP's polynomial GELU in this repository's model
IGNORE = -100


# ------------------------------------------------------------------------------------------------ polynomials
def _interpolant(f, degree=7):
    """Power-basis coefficients of the Chebyshev interpolant of f on [-1, 1]."""
    k = np.arange(degree + 1)
    u = np.cos((2 * k + 1) * np.pi / (2 * (degree + 1)))
    return [float(c) for c in np.polynomial.polynomial.polyfit(u, f(u), degree)]


def _gelu_coeffs():
    erf = np.vectorize(math.erf)
    return _interpolant(lambda u: 0.5 * GELU_BOUND * u * (1.0 + erf(GELU_BOUND * u / math.sqrt(2.0))))


def _weight_coeffs(tokens):
    """The polynomial that stands in for softmax over `tokens` cached tokens: exp(s) / tokens on [-1, 1]."""
    return _interpolant(lambda u: np.exp(u) / tokens)


def _horner(coeffs, u):
    r = torch.full_like(u, coeffs[-1])
    for c in reversed(coeffs[:-1]):
        r = r * u + c
    return r


def _act(z, act, c):
    """act(z) in z's type: the identity, z Phi(z), or the polynomial c in z / bound."""
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    if act == "poly":
        return _horner(c, z / GELU_BOUND)
    return z


def _act_slope(z, act, c):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "poly":
        return _horner([i * c[i] / GELU_BOUND for i in range(1, len(c))], z / GELU_BOUND)
    return torch.ones_like(z)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token's MLP up projection, the call that a client repeats per token: latency
        {"name": "linear, one token", "op": "linear", "type": "bf16", "m": 1, "k": 768, "n": 3072, "act": "gelu",
         "bias": True, "residual": "", "out": ""},
        # the same projection for a batch of packed prompts under the polynomial GELU: a prefill's largest product
        {"name": "linear, packed prompts", "op": "linear", "type": "bf16", "m": 8192, "k": 768, "n": 3072, "act": "poly",
         "bias": True, "residual": "", "out": ""},
        # a pruned width with nothing on a boundary, the residual stream kept in 32 bits
        {"name": "linear, ragged", "op": "linear", "type": "f16", "m": 1237, "k": 765, "n": 1001, "act": "",
         "bias": True, "residual": "f32", "out": "f32"},
        # fitting the MLP to the polynomial activation: the up projection's backward pass over a batch
        {"name": "linear_grad, packed prompts", "op": "linear_grad", "type": "bf16", "m": 8192, "k": 768, "n": 3072,
         "act": "poly", "bias": True},
        # a small batch through the padded width, no activation
        {"name": "linear_grad, small batch", "op": "linear_grad", "type": "f16", "m": 509, "k": 1024, "n": 768, "act": "",
         "bias": True},
        # one new token of four sequences against 256 earlier ones: the check of an encrypted step in the clear
        {"name": "attention, single tokens", "op": "attention", "type": "bf16", "heads": 12, "kv_heads": 12, "dim": 64,
         "seqs": 4, "longest": 1, "past": 255, "spread": False, "weights": "softmax"},
        # a batch of prompts of many lengths under the encrypted step's polynomial weights
        {"name": "attention, packed prompts", "op": "attention", "type": "bf16", "heads": 12, "kv_heads": 12, "dim": 64,
         "seqs": 24, "longest": 1024, "past": 0, "spread": True, "weights": "poly"},
        # one long document, grouped heads
        {"name": "attention, long prompt", "op": "attention", "type": "bf16", "heads": 12, "kv_heads": 4, "dim": 64,
         "seqs": 1, "longest": 8192, "past": 0, "spread": False, "weights": "softmax"},
        # wide heads, few groups, odd lengths with some tokens cached already
        {"name": "attention, wide heads", "op": "attention", "type": "f16", "heads": 16, "kv_heads": 2, "dim": 128,
         "seqs": 5, "longest": 2047, "past": 333, "spread": True, "weights": "softmax"},
        # scoring a few answers
        {"name": "vocab, score", "op": "vocab_loss", "type": "bf16", "rows": 16, "vocab": 50000, "dim": 768},
        # a training step's loss and gradient over a batch
        {"name": "vocab, training step", "op": "vocab_step", "type": "bf16", "rows": 4096, "vocab": 50000, "dim": 768},
        # an odd batch and an odd vocabulary at the padded width
        {"name": "vocab, odd step", "op": "vocab_step", "type": "f16", "rows": 517, "vocab": 32003, "dim": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "attention", "attention", "vocab_loss", "vocab_step"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op in ("linear", "linear_grad"):
        while True:
            c = {"op": op, "type": kind, "m": _log(rng, 1, 16384), "k": _log(rng, 48, 4096), "n": _log(rng, 48, 4096)}
            if rng.random() < 0.6:  # widths of models, the rest falls as it falls
                c["k"], c["n"] = max(64, c["k"] // 64 * 64), max(64, c["n"] // 64 * 64)
            if 3072 not in (c["m"], c["k"], c["n"]) and c["m"] * c["k"] * c["n"] <= 8192 * 768 * 3072:
                break
        c |= {"act": rng.choice(["", "gelu", "poly"]), "bias": rng.random() < 0.7}
        if op == "linear":
            c |= {"residual": rng.choice(["", "same", "f32"]), "out": rng.choice(["", "", "f32"])}
        return c
    if op == "attention":
        heads, kv = rng.choice([(12, 12), (12, 4), (12, 1), (16, 2), (9, 3), (6, 6)])
        c = {"op": op, "type": kind, "heads": heads, "kv_heads": kv, "dim": rng.choice([64, 64, 128, 32, 40, 80]),
             "seqs": _log(rng, 1, 32), "longest": _log(rng, 1, 8192), "past": rng.choice([0, 0, _log(rng, 1, 4096)]),
             "spread": rng.random() < 0.6, "weights": rng.choice(["softmax", "softmax", "poly"])}
        while c["seqs"] * c["longest"] > 8192 or c["seqs"] * c["longest"] * (c["longest"] + c["past"]) * c["dim"] * heads > \
                8192 * 8192 * 64 * 12:
            c["seqs"], c["longest"] = max(1, c["seqs"] // 2), max(1, c["longest"] - c["longest"] // 8)
            c["past"] = c["past"] * 3 // 4
        return c
    while True:
        c = {"op": op, "type": kind, "rows": _log(rng, 1, 8192), "vocab": _log(rng, 1000, 50000),
             "dim": max(64, _log(rng, 64, 2048) // 8 * 8)}
        if 3072 not in c.values() and c["rows"] * c["vocab"] * c["dim"] <= 4096 * 50000 * 768:
            return c


def _lengths(case):
    """New and all tokens of each sequence: all alike, or spread between one token and the longest."""
    n, longest, past = case["seqs"], case["longest"], case["past"]
    if case["spread"]:
        q = [max(1, longest - (longest * ((i * 7) % n)) // n - (i * 13) % 5) for i in range(n)]
        return q, [x + (past * ((i * 5) % n)) // n for i, x in enumerate(q)]
    return [longest] * n, [longest + past] * n


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    s = {"case": case}
    if case["op"] in ("linear", "linear_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)  # normalised activations
        s["w"] = normal(k, n, std=0.55 / math.sqrt(k))  # N(0, 0.02) at this repository's width
        s["bias"] = normal(n, std=0.02) if case["bias"] else None
        s["coeffs"] = _gelu_coeffs() if case["act"] == "poly" else None
        if case["op"] == "linear":
            s["residual"] = normal(m, n, dtype=torch.float32 if case["residual"] == "f32" else t) if case["residual"] else None
        else:
            s["dy"] = normal(m, n, std=0.1)
    elif case["op"] == "attention":
        q_lens, k_lens = _lengths(case)
        std = 1.0 if case["weights"] == "softmax" else 0.5  # the polynomial stands in for exp on scores within [-1, 1]
        s["q"] = normal(sum(q_lens), case["heads"], case["dim"], std=std)
        s["k"] = normal(sum(k_lens), case["kv_heads"], case["dim"], std=std)
        s["v"] = normal(sum(k_lens), case["kv_heads"], case["dim"])
        s["q_lens"], s["k_lens"] = q_lens, k_lens
        s["coeffs"] = _weight_coeffs(max(k_lens)) if case["weights"] == "poly" else None
    else:
        r, v, d = case["rows"], case["vocab"], case["dim"]
        s["h"] = normal(r, d)
        s["w"] = normal(v, d, std=2.0 / math.sqrt(d))
        t0 = torch.randint(0, v, (r,), generator=g, device="cuda")
        keep = torch.rand(r, generator=g, device="cuda") >= 0.05  # positions that are not scored
        keep[0] = True
        s["targets"] = torch.where(keep, t0, torch.full_like(t0, IGNORE))
        s["weight"] = keep.float() / keep.sum()  # the mean over the scored positions
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"], s["coeffs"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[c["out"] or c["type"]])


def _plain_linear_grad(s):
    c, t = s["case"], s["x"].dtype
    x, w, dz = s["x"].float(), s["w"].float(), s["dy"].float()
    if c["act"]:
        z = x @ w
        if s["bias"] is not None:
            z = z + s["bias"].float()
        dz = dz * _act_slope(z, c["act"], s["coeffs"])
    db = dz.sum(0).to(t) if s["bias"] is not None else None
    return (dz @ w.t()).to(t), (x.t() @ dz).to(t), db


def _padded(lens, device):
    """Row of each padded position and whether it is one: [sequences][longest]."""
    lens = torch.tensor(lens, device=device)
    first = torch.cumsum(lens, 0) - lens
    at = torch.arange(int(lens.max()), device=device)
    there = at[None] < lens[:, None]
    return torch.where(there, first[:, None] + at[None], torch.zeros_like(first)[:, None]), there


def _plain_attention(s):
    c = s["case"]
    dev, group = s["q"].device, c["heads"] // c["kv_heads"]
    qi, q_there = _padded(s["q_lens"], dev)
    ki, k_there = _padded(s["k_lens"], dev)
    past = torch.tensor([k - q for q, k in zip(s["q_lens"], s["k_lens"])], device=dev)
    q = s["q"][qi].float().transpose(1, 2)  # [sequence][head][token][dim]
    k = s["k"][ki].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"][ki].float().transpose(1, 2).repeat_interleave(group, 1)
    i, j = torch.arange(qi.shape[1], device=dev), torch.arange(ki.shape[1], device=dev)
    visible = (j[None, None] <= i[None, :, None] + past[:, None, None]) & k_there[:, None]
    p = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(c["dim"])
    if c["weights"] == "poly":
        p = _horner(s["coeffs"], p).masked_fill_(~visible[:, None], 0.0)
        o = torch.matmul(p, v)
    else:
        p = p.masked_fill_(~visible[:, None], -math.inf)
        p = p.sub_(p.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.transpose(1, 2)[q_there].to(s["q"].dtype)


def _plain_vocab_loss(s):
    logits = s["h"].float() @ s["w"].float().t()
    top = logits.amax(1)
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(1))
    scored = s["targets"] != IGNORE
    at = torch.where(scored, s["targets"], 0)
    loss = torch.where(scored, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    return logits, lse, loss


def _plain_vocab_step(s):
    t = s["h"].dtype
    logits, lse, loss = _plain_vocab_loss(s)
    scored = s["targets"] != IGNORE
    at = torch.where(scored, s["targets"], 0)
    d = torch.exp(logits - lse[:, None])
    d.scatter_add_(1, at[:, None], torch.full_like(lse, -1.0)[:, None])
    d *= torch.where(scored, s["weight"], 0.0)[:, None]
    return loss, lse, (d @ s["w"].float()).to(t), (d.t() @ s["h"].float()).to(t)


# ------------------------------------------------------------------------------------------------ a pass
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "linear":
            return _plain_linear(s)
        if op == "linear_grad":
            return _plain_linear_grad(s)
        if op == "attention":
            return _plain_attention(s)
        if op == "vocab_loss":
            return _plain_vocab_loss(s)[2:0:-1]
        return _plain_vocab_step(s)
    from perseus_b200 import clear

    if op in ("linear", "linear_grad"):
        act = clear.Poly(s["coeffs"], GELU_BOUND) if c["act"] == "poly" else c["act"] or None
    if op == "linear":
        return clear.linear(s["x"], s["w"], bias=s["bias"], act=act, residual=s["residual"],
                            out_dtype=TYPES[c["out"] or c["type"]])
    if op == "linear_grad":
        return clear.linear_grad(s["dy"], s["x"], s["w"], bias=s["bias"], act=act)
    if op == "attention":
        return clear.prompt_attention(s["q"], s["k"], s["v"], s["q_lens"], s["k_lens"], weights=s["coeffs"])
    loss, lse = clear.vocab_loss(s["h"], s["w"], s["targets"], ignore=IGNORE)
    if op == "vocab_loss":
        return loss, lse
    return (loss, lse) + clear.vocab_loss_grad(s["h"], s["w"], s["targets"], lse, s["weight"], ignore=IGNORE)


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    size = 2
    if case["op"] in ("linear", "linear_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        if case["op"] == "linear":
            res = {"": 0, "same": 2, "f32": 4}[case["residual"]]
            out = 4 if case["out"] == "f32" else 2
            return {"bytes": size * (m * k + k * n + n * case["bias"]) + m * n * (res + out), "flops": 2 * m * n * k}
        # an activation's slope needs the product z again, which is no input
        return {"bytes": size * (m * n + 2 * m * k + 2 * k * n + 2 * n * case["bias"]),
                "flops": (6 if case["act"] else 4) * m * n * k}
    if case["op"] == "attention":
        q_lens, k_lens = _lengths(case)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(q_lens, k_lens))
        d = case["dim"]
        return {"bytes": size * d * (2 * sum(q_lens) * case["heads"] + 2 * sum(k_lens) * case["kv_heads"]),
                "flops": 4 * pairs * d * case["heads"]}
    r, v, d = case["rows"], case["vocab"], case["dim"]
    if case["op"] == "vocab_loss":
        return {"bytes": size * (r * d + v * d) + 16 * r, "flops": 2 * r * v * d}
    return {"bytes": size * 2 * (r * d + v * d) + 20 * r, "flops": 6 * r * v * d}


# ------------------------------------------------------------------------------------------------ 64 bits
def _f64(x):
    return x.to(torch.float64)


def _exact_poly(coeffs, u):
    return sum(c * u**i for i, c in enumerate(coeffs))


def _exact_linear(s, grad):
    c = s["case"]
    x, w = _f64(s["x"]), _f64(s["w"])
    z = torch.einsum("mk,kn->mn", x, w)
    if s["bias"] is not None:
        z += _f64(s["bias"])[None, :]
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if not grad:
        y = {"": lambda: z, "gelu": lambda: z * phi, "poly": lambda: _exact_poly(_gelu_coeffs(), z / GELU_BOUND)}[c["act"]]()
        return y if s["residual"] is None else y + _f64(s["residual"])
    slope = {"": lambda: 1.0, "gelu": lambda: phi + z * torch.exp(-z**2 / 2) / math.sqrt(2 * math.pi),
             "poly": lambda: _exact_poly([i * a / GELU_BOUND for i, a in enumerate(_gelu_coeffs())][1:], z / GELU_BOUND)}[c["act"]]()
    dz = _f64(s["dy"]) * slope
    return (torch.einsum("mn,kn->mk", dz, w), torch.einsum("mk,mn->kn", x, dz),
            dz.sum(0) if s["bias"] is not None else None)


def _exact_attention(s):
    c = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    group = c["heads"] // c["kv_heads"]
    for nq, nk in zip(s["q_lens"], s["k_lens"]):
        gone = torch.arange(nk, device="cuda")[None, :] > torch.arange(nq, device="cuda")[:, None] + (nk - nq)
        for h in range(c["heads"]):
            q, k, v = (_f64(s["q"][q0:q0 + nq, h]), _f64(s["k"][k0:k0 + nk, h // group]), _f64(s["v"][k0:k0 + nk, h // group]))
            sc = (q @ k.T) * c["dim"] ** -0.5
            if c["weights"] == "poly":
                p = _exact_poly(_weight_coeffs(max(s["k_lens"])), sc)
                p[gone] = 0
            else:
                sc[gone] = -math.inf
                p = torch.softmax(sc, 1)
            out[q0:q0 + nq, h] = p @ v
        q0, k0 = q0 + nq, k0 + nk
    return out


def _exact_vocab(s, grad):
    r = s["h"].shape[0]
    h, w = _f64(s["h"]), _f64(s["w"])
    lse, loss = torch.empty(r, dtype=torch.float64, device="cuda"), torch.zeros(r, dtype=torch.float64, device="cuda")
    dh, dw = torch.empty_like(h), torch.zeros_like(w)
    for a in range(0, r, 1024):
        rows = slice(a, min(r, a + 1024))
        lg = h[rows] @ w.T
        lse[rows] = torch.logsumexp(lg, 1)
        t = s["targets"][rows]
        here = (t != IGNORE).nonzero()[:, 0]
        loss[rows][here] = lse[rows][here] - lg[here, t[here]]
        if grad:
            d = torch.softmax(lg, 1)
            d[here, t[here]] -= 1
            d *= (_f64(s["weight"][rows]) * (t != IGNORE))[:, None]
            dh[rows] = d @ w
            dw += d.T @ h[rows]
    return (loss, lse, dh, dw) if grad else (loss, lse)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "linear_grad"):
        return _exact_linear(s, case["op"] == "linear_grad")
    if case["op"] == "attention":
        return _exact_attention(s)
    return _exact_vocab(s, case["op"] == "vocab_step")
