"""Plain 64-bit forms of the clear half's operators (perseus_b200.clear), and the errors that their arithmetic may make:
one rounding of the result to its type, 32-bit sums (K 2^-23 of the sum of the terms' sizes bounds any order of
summation), and where a product's operand is an intermediate value, its one rounding to 16 bits."""
import math

import torch

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}  # half a unit in the last place
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, torch.float32: 2.0**-149}  # the smallest value
S = 2.0**-23


def act(z, kind):
    if kind == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if kind is not None:
        return sum(c * (z / kind.bound) ** i for i, c in enumerate(kind.coeffs))
    return z


def slope(z, kind):
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind is not None:
        return sum(i * c / kind.bound * (z / kind.bound) ** (i - 1) for i, c in enumerate(kind.coeffs) if i)
    return torch.ones_like(z)


def _poly_size(z, kind):
    """The sum of the terms' sizes of a polynomial: what its 32-bit evaluation errs by, in units of 16 S."""
    return sum(abs(c) * (z.abs() / kind.bound) ** i for i, c in enumerate(kind.coeffs)) if not isinstance(kind, str) else 1 + z.abs()


def linear(x, w, bias, kind, residual, out_dtype):
    """(result, bound on the error per element)"""
    x, w = x.double(), w.double()
    b = 0.0 if bias is None else bias.double()
    z = x @ w + b
    dz = (x.shape[-1] + 4) * S * (x.abs() @ w.abs() + (0.0 if bias is None else bias.double().abs()))
    y = act(z, kind)
    err = dz * (slope(z, kind).abs() + 1.0) if kind is not None else dz
    if kind is not None:
        err = err + 16 * S * _poly_size(z, kind)
    if residual is not None:
        y = y + residual.double()
        err = err + 2 * S * y.abs()
    return y, err + U[out_dtype] * y.abs() + TINY[out_dtype]


def linear_grad(dy, x, w, bias, kind, db_dtype):
    t = x.dtype
    x, w, dy = x.double(), w.double(), dy.double()
    z = x @ w + (0.0 if bias is None else bias.double())
    k = x.shape[1]
    ez = (k + 4) * S * (x.abs() @ w.abs() + (0.0 if bias is None else bias.double().abs()))
    dz = dy * slope(z, kind)
    if kind is None:
        e = torch.zeros_like(dz)
        r = e
    else:  # |act''| <= 1.2 for GELU; a polynomial's from its coefficients
        second = 1.2 if isinstance(kind, str) else sum(
            i * (i - 1) * abs(c) / kind.bound**2 * (z.abs() / kind.bound) ** (i - 2) for i, c in enumerate(kind.coeffs) if i > 1)
        size = 2.0 if isinstance(kind, str) else sum(
            i * abs(c) / kind.bound * (z.abs() / kind.bound) ** (i - 1) for i, c in enumerate(kind.coeffs) if i)
        e = dy.abs() * (second * ez * 1.01 + 16 * S * size)
        r = e + U[t] * dz.abs() + TINY[t]  # as an operand of the products: rounded to 16 bits
    m, n = dy.shape
    a = dz.abs()
    out = []
    dx, ex = dz @ w.t(), r @ w.abs().t() + (n + 4) * S * (a @ w.abs().t())
    dw, ew = x.t() @ dz, x.abs().t() @ r + (m + 4) * S * (x.abs().t() @ a)
    db, eb = dz.sum(0), e.sum(0) + (m + 4) * S * a.sum(0)
    for y, err, ty in ((dx, ex, t), (dw, ew, t), (db, eb, db_dtype)):
        out.append((y, err + U[ty] * y.abs() + TINY[ty]))
    return out


def attention(q, k, v, q_lens, k_lens, scale, causal, weights):
    t, group = q.dtype, q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        for h in range(q.shape[1]):
            a, b = q[q0:q0 + nq, h].double(), k[k0:k0 + nk, h // group].double()
            c = v[k0:k0 + nk, h // group].double()
            s = a @ b.t() * scale
            es = (q.shape[2] + 4) * S * (a.abs() @ b.abs().t()) * abs(scale) + 2 * S * s.abs()
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = torch.arange(nk, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (nk - nq)
            if weights is None:
                p = torch.where(seen, s, -math.inf)
                top = p.amax(1, keepdim=True) if nk else torch.zeros(nq, 1, dtype=torch.float64, device=q.device)
                p = torch.where(seen, torch.exp(p - top.clamp_min(-1e300)), 0.0)
                l = p.sum(1, keepdim=True)
                p = torch.where(l > 0, p / l.clamp_min(1e-300), 0.0)
                # the exponent's error, once for the weight and once for the sum; 2^-20 of the exponential itself; a
                # weight below the type's smallest is lost
                ep = p * (2 * es.amax(1, keepdim=True) + 2.0**-19 + nk * S + U[t]) + TINY[t] if nk else p
                ep = torch.where(seen, ep, 0.0)
            else:
                p = torch.where(seen, sum(co * s**i for i, co in enumerate(weights)), 0.0)
                size = sum(abs(co) * s.abs() ** i for i, co in enumerate(weights))
                ds = sum(i * abs(co) * s.abs() ** (i - 1) for i, co in enumerate(weights) if i)
                ep = torch.where(seen, ds * es + 16 * S * size + U[t] * p.abs() + TINY[t] * max(map(abs, weights)), 0.0)
            o = p @ c
            out[q0:q0 + nq, h] = o
            err[q0:q0 + nq, h] = ep @ c.abs() + (nk + 4) * S * (p.abs() @ c.abs()) + U[t] * o.abs() + TINY[t]
        q0, k0 = q0 + nq, k0 + nk
    return out, err


def vocab(h, w, targets, weight, ignore):
    """((loss, bound), (lse, bound), (dh, bound), (dw, bound))"""
    t = h.dtype
    h, w = h.double(), w.double()
    lg = h @ w.t()
    el = (h.shape[1] + 4) * S * (h.abs() @ w.abs().t())
    lse = torch.logsumexp(lg, 1)
    at = targets.clamp_min(0)
    scored = targets != ignore
    loss = torch.where(scored, lse - lg.gather(1, at[:, None])[:, 0], 0.0)
    # the logits' error, the sum's and the logarithm's
    e_lse = el.amax(1) + 2.0**-18 + 4 * S * lse.abs() + 4 * S * lg.abs().amax(1)
    out = [(loss, torch.where(scored, e_lse + el.amax(1) + 4 * S * loss.abs(), 0.0)), (lse, e_lse)]
    p = torch.exp(lg - lse[:, None])
    g = torch.where(scored, weight.double(), 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    d = (p - hot) * g
    # p's relative error, then the rounding to 16 bits (the values are scaled to the type's range: the smallest counts
    # against the largest weight)
    ed = p * g.abs() * (el + e_lse[:, None] + 2.0**-18) + U[t] * d.abs() + TINY[t] * g.abs().amax() * 2.0**-4
    for y, err, n in ((d @ w, ed @ w.abs(), w.shape[0]), (d.t() @ h, ed.t() @ h.abs(), h.shape[0])):
        size = (d.abs() @ w.abs()) if y.shape == h.shape and y is not None and n == w.shape[0] else (d.abs().t() @ h.abs())
        out.append((y, err + (n + 4) * S * size + U[t] * y.abs() + TINY[t]))
    return out


def close(got, want):
    """got (any type) within want's bound everywhere"""
    y, err = want
    assert got.shape == y.shape, (got.shape, y.shape)
    g = got.double()
    bad = ~((g - y).abs() <= err)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {i}: {g[i].item()} against {y[i].item()} "
                             f"+- {err[i].item():.3g}")
