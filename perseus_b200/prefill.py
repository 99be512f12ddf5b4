"""A client's pass of its prompts through the layers in the clear: the K and V rows that the encrypted decoder's caches
start from (model.Decoder.load), and the loss and gradients of hidden states against an output head.

The layer is model.py's (model.plain_layer's formulas for every token of a prompt at once): LayerNorm, Q/K/V projections,
causal attention, output projection and residual, LayerNorm, MLP and residual, with either the polynomials that the
encrypted step evaluates (`poly=True`: what the encrypted caches must hold for the decode to continue the same model) or
softmax, GELU and the exact LayerNorm (the model that the polynomials approximate). Projections, activations and
attention run on the operators of clear.py in 16 bits with a 32-bit residual stream.
"""
from dataclasses import dataclass

import torch

from . import attention as A
from . import block as B
from . import clear
from . import model as M


@dataclass
class Layer:
    """One layer's weights on the device: the LayerNorms' affine parts folded into the projections that follow them
    (block.fold_norm), Q, K and V side by side."""

    wqkv: torch.Tensor
    bqkv: torch.Tensor
    wo: torch.Tensor
    bo: torch.Tensor
    w_up: torch.Tensor
    b_up: torch.Tensor
    w_down: torch.Tensor
    b_down: torch.Tensor


def load(weights, device="cuda", dtype=torch.bfloat16):
    """model.LayerWeights (numpy) as Layers: matrices in `dtype`, biases in float32."""
    def mat(x):
        return torch.as_tensor(x, dtype=torch.float32).to(device=device, dtype=dtype).contiguous()

    def vec(x):
        return torch.as_tensor(x, dtype=torch.float32, device=device)

    out = []
    for w in weights:
        a = B.fold_norm(w.attn, w.gamma1, w.beta1)
        qkv = [torch.as_tensor(x) for x in (a.wq, a.wk, a.wv)]
        out.append(Layer(mat(torch.cat(qkv, 1)), vec(torch.cat([torch.as_tensor(x) for x in (a.bq, a.bk, a.bv)])),
                         mat(a.wo), vec(a.bo), mat(w.gamma2[:, None] * w.w_up), vec(w.beta2 @ w.w_up + w.b_up),
                         mat(w.w_down), vec(w.b_down)))
    return out


def _norm(x, cfg, poly):
    """LayerNorm without its affine part, in x's 32 bits: block.NormCfg.plain for every row."""
    c = x - x.mean(-1, keepdim=True)
    u = (c * c).mean(-1, keepdim=True) + cfg.eps
    if not poly:
        return c * torch.rsqrt(u)
    z = (2 * u - cfg.lo - cfg.hi) / (cfg.hi - cfg.lo)
    r = torch.zeros_like(z)
    for co in reversed(cfg.coeffs()):
        r = r * z + co
    return c * r


def prefill(x, lens, layers, cfg, poly=True):
    """x: the prompts' embeddings packed along the tokens [sum lens, d] (float32, on the device), lens their lengths (each
    at most cfg.tokens), layers from load, cfg a model.ModelCfg. Returns (Ks, Vs, y): per layer a list with one float32
    [len, d] tensor per prompt, as Decoder.load takes them (as numpy, one sequence's or a list of them), and the last
    layer's output [sum lens, d]."""
    if len(lens) == 0 or sum(lens) != x.shape[0] or max(lens) > cfg.tokens:
        raise ValueError(f"prefill: {len(lens)} prompts of {sum(lens)} tokens (at most {cfg.tokens} each), x has {x.shape[0]}")
    d, heads, dh = cfg.heads * cfg.head_dim, cfg.heads, cfg.head_dim
    if x.shape[1] != d:
        raise ValueError(f"prefill: rows of {x.shape[1]}, the model's are {d}")
    act = clear.Poly(M.gelu_poly(cfg.gelu_bound), cfg.gelu_bound) if poly else "gelu"
    weights = A.softmax_poly(cfg.tokens) if poly else None
    x = x.float()
    Ks, Vs = [], []
    for w in layers:
        n = _norm(x, cfg.norm, poly).to(w.wqkv.dtype)
        qkv = clear.linear(n, w.wqkv, bias=w.bqkv)
        q, k, v = qkv.view(-1, 3, heads, dh).unbind(1)
        Ks.append([t.float().reshape(-1, d) for t in k.split(list(lens))])
        Vs.append([t.float().reshape(-1, d) for t in v.split(list(lens))])
        att = clear.prompt_attention(q, k, v, lens, weights=weights)
        x = clear.linear(att.view(-1, d), w.wo, bias=w.bo, residual=x, out_dtype=torch.float32)
        n = _norm(x, cfg.norm, poly).to(w.w_up.dtype)
        u = clear.linear(n, w.w_up, bias=w.b_up, act=act)
        x = clear.linear(u, w.w_down, bias=w.b_down, residual=x, out_dtype=torch.float32)
    return Ks, Vs, x


@dataclass
class Tail:
    """What fit_step trains: the last layer's MLP (w_up, b_up, w_down, b_down of a Layer) and the output head
    [vocab, d]."""

    layer: Layer
    head: torch.Tensor


def fit_step(r, targets, tail, cfg, ignore=-100, poly=True):
    """One step's loss and gradients of the tail on residual streams r [rows, d] (float32: a layer's input to its second
    LayerNorm, of prefilled prompts or decrypted): y = r + MLP(LayerNorm(r)), the mean cross entropy of y against the head
    over the targets that are not `ignore`. Returns (loss, {"head", "w_up", "b_up", "w_down", "b_down"}): a scalar tensor
    and the gradients, nothing updated. Gradients are of the weights' types, or float32 for float16 layers: a mean over
    many rows leaves float16's normal range, so those are formed of a multiple of the loss and divided after."""
    w = tail.layer
    act = clear.Poly(M.gelu_poly(cfg.gelu_bound), cfg.gelu_bound) if poly else "gelu"
    n = _norm(r, cfg.norm, poly).to(w.w_up.dtype)
    u = clear.linear(n, w.w_up, bias=w.b_up, act=act)
    y = clear.linear(u, w.w_down, bias=w.b_down, residual=r)
    loss, lse = clear.vocab_loss(y, tail.head, targets, ignore)
    scored = (targets != ignore).float()
    count = scored.sum().clamp_min(1.0)
    weight = scored / count
    # float16 ends at 65504 and loses bits below 2^-14: 64 leaves room for gradients of 1000, and for rows by the thousands
    scale = count.clamp_max(64.0) if y.dtype is torch.float16 else None
    dy, dhead = clear.vocab_loss_grad(y, tail.head, targets, lse, weight if scale is None else weight * scale, ignore)
    du, dw_down, db_down = clear.linear_grad(dy, u, w.w_down, bias=w.b_down)
    _, dw_up, db_up = clear.linear_grad(du, n, w.w_up, bias=w.b_up, act=act, needs=(False, True, True))
    grads = {"head": dhead, "w_up": dw_up, "b_up": db_up, "w_down": dw_down, "b_down": db_down}
    if scale is not None:
        grads = {n: g.float() / scale for n, g in grads.items()}
    return (loss * weight).sum(), grads
