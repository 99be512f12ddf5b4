"""The clear half of the model: what a client computes on its own side of the encrypted decode, as CUDA operators.

The encrypted decoder (perseus_b200.model.Decoder.load) starts from the K and V rows of the client's prompt and ends at a
hidden state. Before it, the prompt's pass through the layers in the clear: `linear` (projections and MLP, with bias,
activation and residual) and `prompt_attention` (whole prompts packed along the tokens, with softmax or with the
polynomial weights that the encrypted step evaluates). After it, the score of hidden states against a vocabulary,
`vocab_loss`. `vocab_loss_grad` and `linear_grad` give the gradients that fit the head and the MLP to the polynomials.
perseus_b200.prefill runs them together.

Operands are CUDA tensors of torch.bfloat16 or torch.float16 (one type per call), sums are 32-bit, results are rounded
once. Three intermediate values are rounded to 16 bits as well, as operands of a second product: prompt_attention's weights
before they meet v, linear_grad's dy act'(z) under an activation (scaled to float16's range), vocab_loss_grad's slopes; what
is computed from the first two then errs about 1.4 times as much as by its own rounding. Every call runs on the current stream, without a host copy or sync. Results are plain tensors: nothing is recorded
for autograd.
"""
import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib as L

_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NO_COEF = (C.c_float * 8)()


@dataclass(frozen=True)
class Poly:
    """The activation sum_i coeffs[i] (z / bound)^i, at most 8 coefficients: model.gelu_poly(bound) gives the encrypted
    MLP's."""

    coeffs: tuple
    bound: float = 1.0

    def __post_init__(self):
        object.__setattr__(self, "coeffs", tuple(float(c) for c in self.coeffs))
        if not 1 <= len(self.coeffs) <= 8 or not all(map(math.isfinite, self.coeffs)):
            raise ValueError(f"Poly: 1 to 8 finite coefficients, got {self.coeffs}")
        if not (self.bound > 0 and math.isfinite(self.bound)):
            raise ValueError(f"Poly: bound {self.bound}")
        object.__setattr__(self, "_c", (C.c_float * 8)(*self.coeffs))


def _act(act):
    if act is None:
        return 0, 1.0, _NO_COEF
    if isinstance(act, Poly):
        return 2, act.bound, act._c
    if act == "gelu":
        return 1, 1.0, _NO_COEF
    raise ValueError(f"act {act!r}: None, 'gelu' or a Poly")


def _is(name, t, like, dims):
    """t: a CUDA tensor with `dims` dimensions, 16-bit, or of like's type and device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor, got {t.device if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.dim() != dims:
        raise ValueError(f"{name}: {dims} dimensions, got shape {tuple(t.shape)}")
    if like is None:
        if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
            raise ValueError(f"{name}: bfloat16 or float16, got {t.dtype}")
    elif t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name}: {like.dtype} on {like.device}, got {t.dtype} on {t.device}")


def _aside(name, t, like, shape):
    """An optional operand of like's type or float32."""
    if t.shape != shape or not t.is_cuda or t.get_device() != like.get_device() or \
            (t.dtype is not like.dtype and t.dtype is not torch.float32):
        raise ValueError(f"{name}: {tuple(shape)} of {like.dtype} or float32 on {like.device}, got {tuple(t.shape)} of "
                         f"{t.dtype} on {t.device}")


def _rows(t):
    """(t, the pitch of its rows) with adjacent columns and rows that do not overlap (a copy where it is not so)."""
    r, c = t.shape
    sr, sc = t.stride()
    if sc != 1 and c != 1 or sr < c and r != 1:
        return t.contiguous(), c
    return t, sr if r > 1 else c


def _weight(w):
    """(w, its rows' pitch, whether its memory is the transposed matrix)."""
    k, n = w.shape
    sk, sn = w.stride()
    if sn == 1 and sk >= n:
        return w, sk, 0
    if sk == 1 and sn >= k:
        return w, sn, 1
    return w.contiguous(), n, 0


_MOST = 2**31 - 1025


def _sizes(op, *sizes):
    """The entries count in 32 bits; ctypes would cut what is beyond."""
    if max(sizes) > _MOST:
        raise ValueError(f"{op}: sizes of at most {_MOST}, got {sizes}")


def _flat(name, t):
    """[..., c] as rows, also where there are none."""
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        raise ValueError(f"{name}: a CUDA tensor [..., columns]")
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _launch(op, args, like):
    dev = like.get_device()
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _launch(op, args, like)
    entry = _ENTRY.get(op)
    if entry is None:
        lib = L.lib()
        entry = _ENTRY[op] = getattr(lib, f"pcb_clear_{op}_ws"), getattr(lib, f"pcb_clear_{op}")
    need = entry[0](args)
    if need < 0:
        L.check(int(need), f"pcb_clear_{op}")
    ws = like.new_empty(need, dtype=torch.uint8) if need else None  # lives until the launches are queued
    rc = entry[1](args, None if ws is None else ws.data_ptr(), need, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        L.check(rc, f"pcb_clear_{op}")


_ENTRY = {}


def linear(x, w, bias=None, act=None, residual=None, out_dtype=None):
    """act(x w + bias) + residual for x [..., k], w [k, n] (a transposed view of an [n, k] matrix is read as it lies).
    act: None, "gelu" (z Phi(z)) or a Poly. bias [n] and residual [..., n] are of x's type or float32; the result is of
    `out_dtype`: x's type (default) or float32."""
    x2 = _flat("x", x)
    flat = x2 is x
    _is("x", x2, None, 2)
    _is("w", w, x2, 2)
    m, k = x2.shape
    kw, n = w.shape
    if kw != k or k < 1:
        raise ValueError(f"linear: x {tuple(x.shape)} against w {tuple(w.shape)}")
    _sizes("linear", m, k, n)
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype is not x.dtype and out_dtype is not torch.float32:
        raise ValueError(f"linear: out_dtype {out_dtype}: {x.dtype} or float32")
    kind, bound, coef = _act(act)
    t = _TYPE[x.dtype]
    bias_ptr = res_ptr = None
    bias_type, res_type, res_pitch = t, t, n
    if bias is not None:
        _aside("bias", bias, x2, (n,))
        bias = bias.contiguous()
        bias_ptr, bias_type = bias.data_ptr(), _TYPE[bias.dtype]
    if residual is not None:
        _aside("residual", residual, x2, (m, n) if flat else x.shape[:-1] + (n,))
        residual, res_pitch = _rows(_flat("residual", residual))
        res_ptr, res_type = residual.data_ptr(), _TYPE[residual.dtype]
    x2, x_pitch = _rows(x2)
    w, w_pitch, w_cols = _weight(w)
    y = x2.new_empty((m, n)) if out_dtype is x.dtype else x2.new_empty((m, n), dtype=out_dtype)
    if m and n:
        _launch("linear", L.ClearLinear(x2.data_ptr(), w.data_ptr(), bias_ptr, res_ptr, y.data_ptr(), x_pitch, w_pitch,
                                        res_pitch, n, m, k, n, t, w_cols, bias_type, res_type, _TYPE[out_dtype], kind,
                                        bound, coef), x2)
    return y if flat else y.reshape(x.shape[:-1] + (n,))


def linear_grad(dy, x, w, bias=None, act=None, needs=(True, True, True)):
    """The gradients (dx, dw, db) of linear(x, w, bias, act) for the gradient dy [..., n] of its result (a residual's
    gradient is dy itself). The product x w + bias is formed again where there is an activation, so the forward call keeps
    nothing. dx is of x's shape, dw of w's (laid out as w is), both of x's type; db [n] is of bias's type, None without a
    bias. needs: which of the three are wanted, the others are None."""
    x2 = _flat("x", x)
    _is("x", x2, None, 2)
    _is("w", w, x, 2)
    m, k = x2.shape
    n = w.shape[1]
    if w.shape[0] != k or k < 1 or n < 1:
        raise ValueError(f"linear_grad: x {tuple(x.shape)} against w {tuple(w.shape)}")
    _sizes("linear_grad", m, k, n)
    if not isinstance(dy, torch.Tensor) or dy.shape != x.shape[:-1] + (n,):
        raise ValueError(f"linear_grad: dy of shape {tuple(x.shape[:-1]) + (n,)}")
    dy2 = _flat("dy", dy)
    _is("dy", dy2, x, 2)
    kind, bound, coef = _act(act)
    if bias is not None:
        _aside("bias", bias, x, (n,))
        bias = bias.contiguous()
    x2, x_pitch = _rows(x2)
    dy2, dy_pitch = _rows(dy2)
    w, w_pitch, w_cols = _weight(w)
    t = _TYPE[x.dtype]
    dx = x2.new_empty((m, k)) if needs[0] else None
    dw = None
    if needs[1]:
        dw = x2.new_empty((n, k)).t() if w_cols else x2.new_empty((k, n))
    db = bias.new_empty(n) if needs[2] and bias is not None else None
    if dx is not None or dw is not None or db is not None:
        _launch("linear_grad", L.ClearLinearGrad(
            dy2.data_ptr(), x2.data_ptr(), w.data_ptr(), None if bias is None else bias.data_ptr(),
            None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
            None if db is None else db.data_ptr(), dy_pitch, x_pitch, w_pitch, k, k if w_cols else n, m, k, n, t, w_cols,
            t if bias is None else _TYPE[bias.dtype], t if db is None else _TYPE[db.dtype], kind, bound, coef), x2)
    if dx is not None and x.dim() != 2:
        dx = dx.reshape(x.shape)
    return dx, dw, db


def prompt_attention(q, k, v, q_lens, k_lens=None, scale=None, causal=True, weights=None):
    """Attention of sequences packed along the tokens: q [sum q_lens, heads, dim], k and v [sum k_lens, kv_heads, dim],
    heads a multiple of kv_heads (query head h reads K/V head h // (heads / kv_heads)), dim <= 128. q_lens, k_lens: the
    sequences' lengths on the host; k_lens defaults to q_lens, a longer one means that the queries are the sequence's last
    tokens (a single token against a cache has q_lens 1). Causal: query i sees key j iff j <= i + k_len - q_len; a query
    that sees nothing gets zeros. scale defaults to 1 / sqrt(dim). weights: None for softmax, or the coefficients c_0..c_7
    of the polynomial that stands in for it (attention.softmax_poly): sum_j p(s_j) v_j, not normalised, as the encrypted
    step computes it."""
    _is("q", q, None, 3)
    _is("k", k, q, 3)
    _is("v", v, q, 3)
    q_rows, heads, dim = q.shape
    k_rows, kv_heads = k.shape[:2]
    if k.shape[2] != dim or v.shape != k.shape:
        raise ValueError(f"prompt_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if not 1 <= dim <= 128 or kv_heads < 1 or heads % kv_heads or not 1 <= heads // kv_heads <= 128:
        raise ValueError(f"prompt_attention: {heads} heads over {kv_heads}, dim {dim} (a multiple, at most 128 to one; 1..128)")
    k_lens = q_lens if k_lens is None else k_lens
    nseq = len(q_lens)
    if len(k_lens) != nseq:
        raise ValueError(f"prompt_attention: {nseq} q_lens, {len(k_lens)} k_lens")
    if nseq and (max(max(q_lens), max(k_lens)) > _MOST or min(min(q_lens), min(k_lens)) < -_MOST):
        raise ValueError(f"prompt_attention: lengths of at most {_MOST}")
    coef = () if weights is None else tuple(weights)
    if weights is not None and not 1 <= len(coef) <= 8:
        raise ValueError(f"prompt_attention: 1 to 8 coefficients, got {len(coef)}")
    out = q.new_empty((q_rows, heads, dim))
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    if dim != 1 and (sq[2] != 1 or sk[2] != 1 or sv[2] != 1):
        q, k, v = (t if t.stride(2) == 1 else t.contiguous() for t in (q, k, v))
        sq, sk, sv = q.stride(), k.stride(), v.stride()
    lens = C.c_int32 * nseq
    ql = lens(*q_lens)
    kl = ql if k_lens is q_lens else lens(*k_lens)
    _launch("attention", L.ClearAttention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), C.addressof(ql), C.addressof(kl), sq[0], sq[1], sk[0],
        sk[1], sv[0], sv[1], heads * dim, dim, q_rows, k_rows, nseq, heads, kv_heads, dim, _TYPE[q.dtype], int(causal),
        len(coef), 1.0 / math.sqrt(dim) if scale is None else scale, (C.c_float * 8)(*coef) if coef else _NO_COEF), q)
    return out


def _vocab_args(who, h, w, targets, lse, loss, ignore):
    _is("h", h, None, 2)
    _is("w", w, h, 2)
    rows, dim = h.shape
    if w.shape[1] != dim or dim < 1 or w.shape[0] < 1:
        raise ValueError(f"{who}: h {tuple(h.shape)} against w {tuple(w.shape)}")
    _sizes(who, rows, w.shape[0], dim)
    if targets.shape != (rows,) or targets.dtype != torch.int64 or targets.device != h.device:
        raise ValueError(f"{who}: targets of shape ({rows},) in int64 on {h.device}, got {tuple(targets.shape)} of "
                         f"{targets.dtype} on {targets.device}")
    h, h_pitch = _rows(h)
    w, w_pitch = _rows(w)
    targets = targets.contiguous()
    args = L.ClearVocab(h.data_ptr(), w.data_ptr(), targets.data_ptr(), None if loss is None else loss.data_ptr(),
                        lse.data_ptr(), h_pitch, w_pitch, ignore, rows, w.shape[0], dim, _TYPE[h.dtype])
    return args, (h, w, targets)  # the tensors that args points into


def vocab_loss(h, w, targets, ignore=-100):
    """Softmax cross entropy of hidden states h [rows, dim] against the vocabulary w [vocab, dim]: (loss, lse), both
    [rows] in float32, lse = log sum_v exp(<h, w_v>), loss = lse - <h, w_target>, 0 where the target is `ignore` (any
    other target outside the vocabulary gives NaN). The logits are never stored whole."""
    _is("h", h, None, 2)
    rows = h.shape[0]
    _sizes("vocab_loss", rows)
    loss = h.new_empty(rows, dtype=torch.float32)
    lse = h.new_empty(rows, dtype=torch.float32)
    args, keep = _vocab_args("vocab_loss", h, w, targets, lse, loss, ignore)
    if rows:
        _launch("vocab_loss", args, h)
    return loss, lse


def vocab_loss_grad(h, w, targets, lse, weight, ignore=-100, needs=(True, True)):
    """The gradients (dh, dw), of h's and w's shape and type, of sum_r weight[r] loss[r] (weight [rows] float32: 1 /
    count for the mean); lse from vocab_loss on the same h and w. The logits are formed again, a piece of the vocabulary
    at a time. An ignored row's dh is 0 whatever the row holds; its h has to be finite for dw. needs: which of the two are
    wanted, the other is None."""
    args, keep = _vocab_args("vocab_loss_grad", h, w, targets, lse, None, ignore)
    rows, dim = h.shape
    for name, t in (("lse", lse), ("weight", weight)):
        if t.shape != (rows,) or t.dtype != torch.float32 or t.device != h.device:
            raise ValueError(f"vocab_loss_grad: {name} of shape ({rows},) in float32 on {h.device}")
    lse, weight = lse.contiguous(), weight.contiguous()
    args.lse = lse.data_ptr()
    dh = h.new_empty((rows, dim)) if needs[0] else None
    dw = h.new_empty((w.shape[0], dim)) if needs[1] else None
    if dh is not None or dw is not None:
        _launch("vocab_grad", L.ClearVocabGrad(args, weight.data_ptr(), None if dh is None else dh.data_ptr(),
                                               None if dw is None else dw.data_ptr(), dim, dim), h)
    return dh, dw
