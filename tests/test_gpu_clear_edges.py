"""The clear half's operators (perseus_b200.clear) where values, sizes or masks are at their ends, against the 64-bit forms
of tests/_clear_ref.py."""
import math

import numpy as np
import pytest
import torch

from perseus_b200 import _lib as L
from perseus_b200 import attention as A
from perseus_b200 import clear
from perseus_b200 import model as M
from perseus_b200 import prefill as PF
from tests import _clear_ref as R

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
GELU_POLY = clear.Poly(tuple(M.gelu_poly(3.0)), 3.0)


def rnd(seed, *shape, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
@pytest.mark.parametrize("dim", [64, 40, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_masked_large_values_stay_out(weights, dim, dtype):
    """The type's largest finite values in V where they are masked: a later token's, the neighbouring sequence's."""
    big = torch.finfo(dtype).max
    lens, scale = [77, 50, 90], dim**-0.5
    q, k, v = rnd(1, 217, 4, dim, std=0.5, dtype=dtype), rnd(2, 217, 4, dim, std=0.5, dtype=dtype), rnd(3, 217, 4, dim, dtype=dtype)
    want = R.attention(q, k, v, lens, lens, scale, True, weights)
    v[77:127] = big
    got = clear.prompt_attention(q, k, v, lens, weights=weights)
    for s in (slice(0, 77), slice(127, 217)):
        R.close(got[s], (want[0][s], want[1][s]))
    for bad in (6, 71, 150):
        v = rnd(3, 217, 4, dim, dtype=dtype)
        want = R.attention(q, k, v, [217], [217], scale, True, weights)
        v[bad:bad + 2] = -big
        got = clear.prompt_attention(q, k, v, [217], weights=weights)
        R.close(got[:bad], (want[0][:bad], want[1][:bad]))


@pytest.mark.parametrize("past", [0, 4000])
def test_attention_weights_that_vanish(past):
    """Visible keys whose weight is below 2^-150 of the largest: nothing of their values, up to the type's largest."""
    n = 9 + past
    q, k, v = torch.zeros(1, 1, 64, dtype=BF, device="cuda"), torch.zeros(n, 1, 64, dtype=BF, device="cuda"), rnd(3, n, 1, 64)
    q[0, 0, 0] = 8.0
    k[1:, 0, 0] = -3000.0
    v[1:] = 3.0e38
    got = clear.prompt_attention(q, k, v, [1], [n], causal=False)
    assert torch.equal(got, v[:1])


@pytest.mark.parametrize("n", [5, 200, 5000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_scores_of_minus_infinity(n, dim):
    """A key whose score is -inf weighs nothing; where every visible score is -inf there is no softmax (NaN), however the
    keys are split over blocks; a query that sees no key has zeros."""
    q, k, v = rnd(1, 3, 2, dim), rnd(2, n, 2, dim), rnd(3, n, 2, dim)
    want = R.attention(q[:, :, 1:], k[1:, :, 1:], v[1:, :, 1:], [3], [n - 1], dim**-0.5, False, None)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[0, :, 0] = -math.inf
    got = clear.prompt_attention(q, k, v, [3], [n], causal=False)
    R.close(got[..., 1:], want)
    k[..., 0] = -math.inf
    assert torch.isnan(clear.prompt_attention(q, k, v, [3], [n], causal=False)).all()
    q = rnd(4, n + 2, 2, dim)
    q[..., 0] = 1.0
    got = clear.prompt_attention(q, k, v, [n + 2], [n])
    assert not got[:2].any() and torch.isnan(got[2:]).all()


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_blind_rows_beside_values_that_are_not_finite(weights, dim, bad):
    """Queries that see no key are zero whatever the keys that others see, and the next sequence's, hold."""
    q_lens, k_lens = [100, 50], [60, 50]
    q, k, v = rnd(1, 150, 4, dim, std=0.5), rnd(2, 110, 2, dim, std=0.5), rnd(3, 110, 2, dim)
    want = R.attention(q, k, v, q_lens, k_lens, dim**-0.5, True, weights)
    v[60:] = bad  # the second sequence's
    got = clear.prompt_attention(q, k, v, q_lens, k_lens, weights=weights)
    assert not got[:40].any()
    R.close(got[:100], (want[0][:100], want[1][:100]))
    v[59] = bad  # a key that the last query alone sees
    got = clear.prompt_attention(q, k, v, q_lens, k_lens, weights=weights)
    assert not got[:40].any()
    R.close(got[:99], (want[0][:99], want[1][:99]))
    k[58:] = bad
    got = clear.prompt_attention(q, k, v, q_lens, k_lens, weights=weights)
    assert not got[:40].any()
    R.close(got[:98], (want[0][:98], want[1][:98]))


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
@pytest.mark.parametrize("dim,dtype", [(64, BF), (64, HF), (128, BF), (40, HF)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_one_value_that_is_not_finite(weights, dim, dtype, bad):
    """It reaches its own dim of the queries that see it and nothing else; a query or key that is not finite, its rows whole."""
    n, at, d, scale = 700, 301, 5, dim**-0.5
    q, k, v = rnd(1, n, 4, dim, std=0.5, dtype=dtype), rnd(2, n, 2, dim, std=0.5, dtype=dtype), rnd(3, n, 2, dim, dtype=dtype)
    want = R.attention(q, k, v, [n], [n], scale, True, weights)
    v[at, 1, d] = bad
    got = clear.prompt_attention(q, k, v, [n], weights=weights)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at:, 2:, d] = True
    assert not torch.isfinite(got[hit]).any()
    R.close(got[~hit], (want[0][~hit], want[1][~hit]))
    v[at, 1, d] = 0.0
    q[at, 1, d] = bad
    k[at + 50, 1, d] = math.nan
    want = R.attention(q, torch.where(torch.isnan(k), 0.0, k), v, [n], [n], scale, True, weights)
    got = clear.prompt_attention(q, k, v, [n], weights=weights)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[at, 1] = hit[at + 50:, 2:] = True
    assert not torch.isfinite(got[hit]).any()
    R.close(got[~hit], (want[0][~hit], want[1][~hit]))


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
def test_attention_time_with_values_that_are_not_finite(weights):
    """Rows that see such a value are not computed again key by key, which would take some thousand times the call's time."""
    n = 4096
    q, k, v = rnd(1, n, 12, 64, std=0.5), rnd(2, n, 4, 64, std=0.5), rnd(3, n, 4, 64)

    def ms():
        best = math.inf
        for _ in range(3):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record()
            clear.prompt_attention(q, k, v, [n], weights=weights)
            e[1].record()
            torch.cuda.synchronize()
            best = min(best, e[0].elapsed_time(e[1]))
        return best
    clean = ms()
    v[1] = math.nan
    assert ms() < 100 * clean
    k[1] = math.nan
    assert ms() < 100 * clean


# ------------------------------------------------------------------------------------------------ vocabulary
def vocab_case(rows, vocab, dim, dtype, std=2.0, seed=0):
    h, w = rnd(seed + 1, rows, dim, dtype=dtype), rnd(seed + 2, vocab, dim, std=std * dim**-0.5, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[1::4] = -100
    weight = torch.rand(rows, generator=g, device="cuda") / rows
    return h, w, t, weight


@pytest.mark.parametrize("low", ["lowest", "-inf"])
@pytest.mark.parametrize("rows,vocab", [(20, 700), (300, 5000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_vocab_masked_entries(low, rows, vocab, dtype):
    """Entries that a constant channel masks with the type's lowest value or -inf, whole column blocks of them: the loss and
    the gradients are those of the vocabulary without them."""
    h, w, t, weight = vocab_case(rows, vocab, 64, dtype)
    out = torch.zeros(vocab, dtype=torch.bool, device="cuda")
    out[:300] = out[320:333] = out[384:448] = out[-50:] = True
    out[:512:64] = True
    keep = (~out).nonzero()[:, 0]
    t = torch.where(t == -100, t, keep[t % len(keep)])
    h[:, 0], w[:, 0] = 1.0, 0.0
    within = torch.where(t == -100, t, torch.searchsorted(keep, t.clamp_min(0)))
    want = R.vocab(h, w[keep], within, weight, -100)
    w[out, 0] = torch.finfo(dtype).min if low == "lowest" else -math.inf
    loss, lse = clear.vocab_loss(h, w, t)
    R.close(loss, want[0])
    R.close(lse, want[1])
    dh, dw = clear.vocab_loss_grad(h, w, t, lse, weight)
    assert not dw[out].any()
    R.close(dw[keep], want[3])
    if low == "lowest":  # (a slope of zero times -inf is no number in dh's own product)
        R.close(dh, want[2])


def test_vocab_all_entries_alike_at_the_ends():
    """Rows whose logits are all the type's lowest, or all its largest, value."""
    ends = torch.tensor([torch.finfo(BF).min, torch.finfo(BF).max], device="cuda").to(BF)
    h, w = torch.zeros(2, 64, dtype=BF, device="cuda"), torch.zeros(500, 64, dtype=BF, device="cuda")
    h[:, 0], w[:, 0] = ends, 1.0
    loss, lse = clear.vocab_loss(h, w, torch.tensor([3, 499], device="cuda"))
    # log 500 is below a unit in the last place of 3.4e38
    assert torch.equal(lse, ends.float()) and not loss.any()


def test_vocab_ignored_rows_that_are_not_finite():
    """dl is 0 on ignored rows, whatever their hidden states and lse hold: dh there is 0 and the other rows' stays."""
    h, w, t, weight = vocab_case(200, 900, 64, BF)
    want = R.vocab(h, w, t, weight, -100)
    h[1], h[5, 3], h[9, 0] = math.nan, math.inf, -math.inf
    assert (t[[1, 5, 9]] == -100).all()
    loss, lse = clear.vocab_loss(h, w, t)
    assert not loss[[1, 5, 9]].any() and not torch.isfinite(lse[[1, 5, 9]]).any()
    dh, _ = clear.vocab_loss_grad(h, w, t, lse, weight, needs=(True, False))
    assert not dh[1::4].any()
    R.close(dh, want[2])


# ------------------------------------------------------------------------------------------------ linear
@pytest.mark.parametrize("m,k,n,splits", [(200, 136, 328, False), (9, 8192, 768, True)])
@pytest.mark.parametrize("out", [BF, F32], ids=str)
def test_linear_gelu_of_infinity(m, k, n, splits, out):
    """z Phi(z) of +inf is +inf, of NaN and (0 times inf) of -inf NaN; with the sums of k in parts and whole."""
    x, w = rnd(1, m, k), rnd(2, k, n, std=k**-0.5)
    w[5] = w[5].abs() + 0.01
    x[1, 5], x[3, 5], x[4, 6] = math.inf, -math.inf, math.nan
    need = L.lib().pcb_clear_linear_ws(L.ClearLinear(x.data_ptr(), w.data_ptr(), None, None, x.data_ptr(), k, n, 0, n, m, k, n, 0,
                                                     0, 0, 0, 0, 1, 1.0))
    assert (need > 0) == splits
    y = clear.linear(x, w, act="gelu", out_dtype=out)
    assert (y[1] == math.inf).all() and torch.isnan(y[3:5]).all()
    rows = [i for i in range(m) if i not in (1, 3, 4)]
    R.close(y[rows], R.linear(x[rows], w, None, "gelu", None, out))


def grad_bounds(dy, x, w, bias, kind):
    """R.linear_grad's bounds where dz, as an operand in float16, errs by its rounding and by no more than 2^-32 of the
    largest dy times the largest slope that any z within the polynomial's bound (GELU: any z) has."""
    most = 1.13 if kind == "gelu" else sum(i * abs(c) / kind.bound for i, c in enumerate(kind.coeffs))
    want = R.linear_grad(dy, x, w, bias, kind, F32)
    less = R.TINY[HF] - 2.0**-32 * float(dy.double().abs().max()) * most
    wd, xd = w.double().abs(), x.double().abs()
    return [(want[0][0], want[0][1] - less * wd.sum(1)), (want[1][0], want[1][1] - less * xd.sum(0)[:, None]), want[2]]


@pytest.mark.parametrize("act", ["gelu", GELU_POLY], ids=["gelu", "poly"])
@pytest.mark.parametrize("size", [1e-6, 1e-4])
@pytest.mark.parametrize("m,k,n", [(3000, 96, 264), (70, 1024, 1000)])
def test_linear_grad_small_dy_in_float16(act, size, m, k, n):
    """Gradients of a mean over many rows: dz stays far below float16's normal range while sums over the rows do not."""
    x, w = rnd(1, m, k, dtype=HF), rnd(2, k, n, std=0.5 * k**-0.5, dtype=HF)
    b, dy = rnd(3, n, std=0.2, dtype=F32), rnd(4, m, n, std=size, dtype=HF)
    for got, want in zip(clear.linear_grad(dy, x, w, bias=b, act=act), grad_bounds(dy, x, w, b, act)):
        R.close(got, want)


def test_linear_grad_large_dy_in_float16():
    """dz beyond float16's range between operands and results that are within it."""
    m, n = 300, 136
    x, w = rnd(1, m, 64, std=0.01, dtype=HF), rnd(2, 64, n, std=0.02, dtype=HF)
    x[:, 0], w[0] = 1.0, 1.4  # z about 1.4, where GELU's slope is 1.129
    dy = torch.where(torch.arange(m, device="cuda")[:, None] % 2 == 0, 60000.0, -60000.0).to(HF).repeat(1, n)
    b = torch.zeros(n, device="cuda")
    assert (R.slope(x.double() @ w.double(), "gelu") * 60000 > 65520).all()
    _, dw, db = clear.linear_grad(dy, x, w, bias=b, act="gelu", needs=(False, True, True))
    want = grad_bounds(dy, x, w, b, "gelu")
    assert want[1][0].abs().max() < 65504
    R.close(dw, want[1])
    R.close(db, want[2])


def test_linear_grad_more_rows_than_a_launch_has_blocks():
    """Column sums of more than 65535 x 256 rows, of whole numbers whose sums are exact in 32 bits."""
    m = 65535 * 256 + 258
    x, w, row = rnd(1, m, 8, dtype=HF), rnd(2, 8, 3, dtype=HF), torch.arange(m, device="cuda")
    dy = torch.stack([row % 4 == 0, row >= m - 1000, row % 2 == 0], 1).to(HF)
    dy[:, 2] = 1 - 2 * dy[:, 2]
    b = torch.zeros(3, device="cuda")
    for needs in ((False, False, True), (True, False, True)):
        dx, _, db = clear.linear_grad(dy, x, w, bias=b, needs=needs)
        assert torch.equal(db, dy.double().sum(0).float())
    for part in (slice(0, 1000), slice(m - 1000, m)):
        want = dy[part].double() @ w.double().t()
        R.close(dx[part], (want, (2.0**-11 + 8 * R.S) * (dy[part].double().abs() @ w.double().abs().t())))


def inside(t, pitch):
    """(a matrix of t's shape within rows of `pitch`, whether everything around it is untouched)"""
    whole = torch.full((t.shape[0] + 1, pitch), 77.0, dtype=t.dtype, device="cuda")
    at = whole[:t.shape[0], :t.shape[1]]

    def untouched():
        return bool((whole[:, t.shape[1]:] == 77.0).all() and (whole[-1] == 77.0).all())
    return at, untouched


@pytest.mark.parametrize("m,k,n,pitch", [(200, 72, 129, 136), (1, 64, 1, 8), (300, 1100, 271, 272), (9, 8192, 765, 768), (600, 64, 8, 16)])
@pytest.mark.parametrize("out", [BF, F32], ids=str)
def test_linear_into_columns_of_a_wider_matrix(m, k, n, pitch, out):
    """The C entry's results in aligned rows that go on after them: nothing past a row's last column is written."""
    x, w = rnd(1, m, k), rnd(2, k, n, std=k**-0.5)
    want = R.linear(x, w, None, None, None, out)
    y, untouched = inside(want[0].to(out), pitch)
    clear._launch("linear", L.ClearLinear(x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), k, n, 0, pitch, m, k, n, 0, 0, 0, 0,
                                          0 if out == BF else 2, 0, 1.0), x)
    R.close(y, want)
    assert untouched()


@pytest.mark.parametrize("act", [None, "gelu"], ids=["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(70, 33, 45), (600, 129, 257)])
def test_gradients_into_columns_of_wider_matrices(act, m, k, n):
    x, w, dy = rnd(1, m, k), rnd(2, k, n, std=k**-0.5), rnd(3, m, n)
    want = R.linear_grad(dy, x, w, None, act, F32)
    up = lambda c: c // 8 * 8 + 8  # noqa: E731
    (dx, dx_ok), (dw, dw_ok) = inside(x, up(k)), inside(w, up(n))
    clear._launch("linear_grad", L.ClearLinearGrad(dy.data_ptr(), x.data_ptr(), w.data_ptr(), None, dx.data_ptr(), dw.data_ptr(), None,
                                                   n, k, n, up(k), up(n), m, k, n, 0, 0, 0, 0, 0 if act is None else 1, 1.0), x)
    R.close(dx, want[0])
    R.close(dw, want[1])
    assert dx_ok() and dw_ok()
    h, v, t, weight = vocab_case(m, 1003, k, BF)
    loss, lse = clear.vocab_loss(h, v, t)
    want = R.vocab(h, v, t, weight, -100)
    (dh, dh_ok), (dv, dv_ok) = inside(h, up(k)), inside(v, up(k))
    args = L.ClearVocab(h.data_ptr(), v.data_ptr(), t.data_ptr(), None, lse.data_ptr(), k, k, -100, m, 1003, k, 0)
    clear._launch("vocab_grad", L.ClearVocabGrad(args, weight.data_ptr(), dh.data_ptr(), dv.data_ptr(), up(k), up(k)), h)
    R.close(dh, want[2])
    R.close(dv, want[3])
    assert dh_ok() and dv_ok()


def test_linear_empty_shapes_of_more_dimensions():
    x, w = rnd(1, 2, 3, 32), rnd(2, 32, 48)
    y = clear.linear(x, w[:, :0], residual=rnd(3, 2, 3, 0), bias=rnd(4, 0))
    assert y.shape == (2, 3, 0)
    assert clear.linear(x[:, :0], w, residual=rnd(3, 2, 0, 48)).shape == (2, 0, 48)
    for call in (lambda: clear.linear(x[..., :0], w[:0]), lambda: clear.linear_grad(rnd(1, 2, 3, 48), x[..., :0], w[:0]),
                 lambda: clear.linear_grad(rnd(1, 2, 3, 0), x, w[:, :0])):
        with pytest.raises(ValueError):
            call()


def test_sizes_beyond_31_bits_are_refused():
    """No size reaches the entries cut to 32 bits."""
    one = torch.ones(1, 1, dtype=BF, device="cuda")
    many, few = one.expand(2**32 + 5, 1), rnd(1, 5, 1)
    t, v = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, device="cuda")
    q = rnd(2, 10, 1, 64)
    for call in (lambda: clear.linear(many, one), lambda: clear.linear(one, many.t()), lambda: clear.linear(many.t(), many),
                 lambda: clear.linear_grad(many, many, one), lambda: clear.linear_grad(many.t(), one, many.t()),
                 lambda: clear.linear_grad(one, many.t(), many), lambda: clear.vocab_loss(one, many, t),
                 lambda: clear.vocab_loss(many, few, t.expand(2**32 + 5)),
                 lambda: clear.vocab_loss_grad(one, many, t, v, v),
                 lambda: clear.prompt_attention(q, q, q, [2**32 + 10]), lambda: clear.prompt_attention(q, q, q, [10], [10 - 2**32])):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------------ fitting in float16
@pytest.mark.parametrize("poly", [True, False], ids=["poly", "exact"])
def test_fit_step_in_float16(poly):
    """The gradients of a mean over many rows in float16 layers against 64-bit autograd: within a few units of 2^-11 of
    each gradient's size."""
    cfg = M.ModelCfg(layers=1, d=128, width=128, heads=2, head_dim=64, mlp=512, tokens=64)
    layer = PF.load([M.random_layer(np.random.default_rng(1), 128, 512)], dtype=HF)[0]
    tail = PF.Tail(layer, rnd(1, 500, 128, std=0.02, dtype=HF))
    rows = 4096
    r = rnd(2, rows, 128, dtype=F32)
    t = torch.randint(0, 500, (rows,), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    t[::9] = -100
    loss, grads = PF.fit_step(r, t, tail, cfg, poly=poly)
    p = {n: getattr(layer, n).double().requires_grad_() for n in ("w_up", "b_up", "w_down", "b_down")}
    p["head"] = tail.head.double().requires_grad_()
    act = clear.Poly(M.gelu_poly(cfg.gelu_bound), cfg.gelu_bound) if poly else "gelu"
    n = PF._norm(r.double(), cfg.norm, poly)
    y = R.act(n @ p["w_up"] + p["b_up"], act) @ p["w_down"] + p["b_down"] + r.double()
    want = torch.nn.functional.cross_entropy(y @ p["head"].t(), t, ignore_index=-100)
    want.backward()
    assert abs(float(loss) - want.item()) < 16 * 2.0**-11 * want.item()
    for name, g in grads.items():
        assert g.dtype == F32
        d = p[name].grad
        assert (g.double() - d).norm() <= 16 * 2.0**-11 * d.norm(), name
