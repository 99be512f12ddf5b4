"""The clear half's operators (perseus_b200.clear) against plain 64-bit forms, per element within the bounds of
tests/_clear_ref.py; gradients also against differences of the 64-bit losses; the path of perseus_b200.prefill against
model.plain_layer."""
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


@pytest.fixture(autouse=True)
def no_timeouts():
    yield
    torch.cuda.synchronize()
    assert L.lib().pcb_device_timeouts() == 0


# ------------------------------------------------------------------------------------------------ linear
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (1, 768, 2304), (2, 1, 1), (7, 17, 5), (64, 128, 192), (127, 129, 255),
                                   (128, 64, 256), (129, 200, 257), (300, 765, 1001), (517, 72, 1000), (1000, 2050, 88),
                                   (9, 4096, 768), (2049, 768, 768)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_shapes(m, k, n, dtype):
    x, w, b = rnd(1, m, k, dtype=dtype), rnd(2, k, n, std=k**-0.5, dtype=dtype), rnd(3, n, dtype=dtype)
    R.close(clear.linear(x, w, bias=b), R.linear(x, w, b, None, None, dtype))


@pytest.mark.parametrize("act", [None, "gelu", GELU_POLY, clear.Poly((0.25, -1.0, 0.5))], ids=["none", "gelu", "poly7", "poly2"])
@pytest.mark.parametrize("bias", [None, BF, F32], ids=str)
@pytest.mark.parametrize("residual", [None, BF, F32], ids=str)
@pytest.mark.parametrize("out", [BF, F32], ids=str)
def test_linear_epilogues(act, bias, residual, out):
    m, k, n = 200, 136, 328
    x, w = rnd(1, m, k), rnd(2, k, n, std=0.5 * k**-0.5)
    b = None if bias is None else rnd(3, n, std=0.2, dtype=bias)
    r = None if residual is None else rnd(4, m, n, dtype=residual)
    y = clear.linear(x, w, bias=b, act=act, residual=r, out_dtype=out)
    assert y.dtype == out
    R.close(y, R.linear(x, w, b, act, r, out))


@pytest.mark.parametrize("act,residual", [(None, None), (None, BF), ("gelu", None), (GELU_POLY, F32)],
                         ids=["none", "residual", "gelu", "poly"])
def test_linear_operand_beyond_l2(act, residual):
    """An A above 64 MB: its tiles go in bands of 2048 rows, the last one lower."""
    m, k, n = 4900, 6600, 1000
    x, w = rnd(1, m, k), rnd(2, k, n, std=0.5 * k**-0.5)
    r = None if residual is None else rnd(3, m, n, dtype=residual)
    R.close(clear.linear(x, w, act=act, residual=r), R.linear(x, w, None, act, r, BF))


@pytest.mark.parametrize("act", [None, GELU_POLY], ids=["none", "poly"])
def test_linear_grad_operands_beyond_l2(act):
    m, k, n = 6600, 4900, 1000
    x, w, dy = rnd(1, m, k), rnd(2, k, n, std=0.5 * k**-0.5), rnd(3, m, n)
    dx, dw, _ = clear.linear_grad(dy, x, w, act=act, needs=(True, True, False))
    want = R.linear_grad(dy, x, w, None, act, BF)
    R.close(dx, want[0])
    R.close(dw, want[1])


def test_linear_strides_and_order():
    """Rows of a wider tensor, a transposed weight, an odd first element, a broadcast row, a 4-d batch."""
    big = rnd(1, 150, 400)
    w = rnd(2, 96, 130, std=0.1)
    wt = rnd(3, 130, 96, std=0.1).t()
    for x in (big[:, 8:104], big[:, 3:99], big[1:140:3, 16:112], big[:1, :96].expand(50, 96), big.t()[:140, 5:101]):
        for ww in (w, wt, rnd(4, 200, 131, std=0.1)[7:103, 1:], rnd(5, 131, 203, std=0.1)[1:, 11:107].t()):
            R.close(clear.linear(x, ww), R.linear(x, ww, None, None, None, BF))
    x4 = rnd(6, 3, 2, 5, 96)
    r4 = rnd(7, 3, 5, 2, 130).transpose(1, 2)
    y = clear.linear(x4, w, residual=r4)
    R.close(y.reshape(30, 130), R.linear(x4.reshape(30, 96), w, None, None, r4.reshape(30, 130), BF))
    res = rnd(8, 150, 301)[:, 1:131]
    R.close(clear.linear(big[:, :96], w, residual=res), R.linear(big[:, :96], w, None, None, res, BF))


def test_linear_empty():
    w = rnd(1, 32, 48)
    assert clear.linear(rnd(2, 0, 32), w).shape == (0, 48)
    assert clear.linear(rnd(2, 5, 32), w[:, :0]).shape == (5, 0)
    dx, dw, db = clear.linear_grad(rnd(2, 0, 48), rnd(3, 0, 32), w, bias=rnd(4, 48), act="gelu")
    assert dx.shape == (0, 32) and not dw.any() and not db.any()


def test_linear_nonfinite_stays_in_its_row():
    x, w = rnd(1, 140, 72), rnd(2, 72, 80)
    x[3, 5] = math.inf
    x[131, 70] = math.nan
    y = clear.linear(x, w)
    rows = [i for i in range(140) if i not in (3, 131)]
    assert torch.isfinite(y[rows]).all() and not torch.isfinite(y[3]).any() and torch.isnan(y[131]).all()
    R.close(y[rows], R.linear(x[rows], w, None, None, None, BF))


def test_linear_on_another_stream():
    x, w = rnd(1, 600, 768), rnd(2, 768, 768, std=0.04)
    want = clear.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [clear.linear(x, w) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


def test_linear_in_a_graph():
    x, w, b = rnd(1, 33, 768), rnd(2, 768, 1024, std=0.04), rnd(3, 1024)
    clear.linear(x, w, bias=b, act="gelu")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = clear.linear(x, w, bias=b, act="gelu")
    for seed in (5, 6):
        x.copy_(rnd(seed, 33, 768))
        g.replay()
        torch.cuda.synchronize()
        R.close(y, R.linear(x, w, b, "gelu", None, BF))


@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (3, 40, 7), (129, 130, 131), (500, 96, 264), (700, 765, 300), (2100, 128, 520)])
@pytest.mark.parametrize("act", [None, "gelu", GELU_POLY], ids=["none", "gelu", "poly"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_grad(m, k, n, act, dtype):
    x, w = rnd(1, m, k, dtype=dtype), rnd(2, k, n, std=0.5 * k**-0.5, dtype=dtype)
    b, dy = rnd(3, n, std=0.2, dtype=F32), rnd(4, m, n, dtype=dtype)
    for got, want in zip(clear.linear_grad(dy, x, w, bias=b, act=act), R.linear_grad(dy, x, w, b, act, F32)):
        R.close(got, want)


def test_linear_grad_orders_and_needs():
    x, dy = rnd(1, 90, 301)[:, 1:201], rnd(2, 90, 155)[:, 2:152]
    for w in (rnd(3, 200, 150, std=0.05), rnd(3, 150, 200, std=0.05).t()):
        want = R.linear_grad(dy, x, w, None, "gelu", BF)
        dx, dw, db = clear.linear_grad(dy, x, w, act="gelu")
        assert db is None and dw.stride() == w.stride()
        R.close(dx, want[0])
        R.close(dw, want[1])
    assert clear.linear_grad(dy, x, w, act="gelu", needs=(False, True, False))[0] is None
    R.close(clear.linear_grad(dy, x, w, bias=torch.zeros(150, device="cuda"), act="gelu", needs=(False, False, True))[2],
            R.linear_grad(dy, x, w, None, "gelu", F32)[2])


def test_linear_grad_against_differences():
    """The directional derivative of <y, g> by central differences of the 64-bit form."""
    x, w, b, g = rnd(1, 40, 24), rnd(2, 24, 56, std=0.1), rnd(3, 56, std=0.1, dtype=F32), rnd(4, 40, 56)
    grads = clear.linear_grad(g, x, w, bias=b, act="gelu")
    for i, (t, gr) in enumerate(zip((x, w, b), grads)):
        d = rnd(10 + i, *t.shape, dtype=torch.float64)
        at = [x.double(), w.double(), b.double()]

        def f(e):
            u = list(at)
            u[i] = u[i] + e * d
            return (R.act(u[0] @ u[1] + u[2], "gelu") * g.double()).sum()
        slope = (f(1e-5) - f(-1e-5)) / 2e-5  # its own error is below 1e-7 of the terms
        bound = R.linear_grad(g, x, w, b, "gelu", F32)[i][1]
        assert abs(slope - (gr.double() * d).sum()) <= (bound * d.abs()).sum() + 1e-6 * (gr.double() * d).abs().sum()


def test_linear_is_the_same_every_time():
    x, w, dy = rnd(1, 1000, 256), rnd(2, 256, 384, std=0.06), rnd(3, 1000, 384)
    one = clear.linear_grad(dy, x, w, bias=rnd(4, 384), act="gelu")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(one, clear.linear_grad(dy, x, w, bias=rnd(4, 384), act="gelu")))


def test_linear_far_offsets():
    """Inputs and results past 2^31 elements."""
    m, n = 1_500_000, 200
    x = torch.zeros(m, 1536, dtype=BF, device="cuda")
    x[-n:] = rnd(1, n, 1536)
    w = rnd(2, 1536, 8, std=0.03)
    y = clear.linear(x, w)
    assert not y[:-n].any()
    R.close(y[-n:], R.linear(x[-n:], w, None, None, None, BF))
    dx, dw, _ = clear.linear_grad(y, x, w)
    want = R.linear_grad(y[-n:], x[-n:], w, None, None, BF)
    R.close(dx[-n:], want[0])
    R.close(dw, want[1])
    del x, y, dx
    x = torch.zeros(m, 64, dtype=BF, device="cuda")
    x[-n:] = rnd(3, n, 64)
    w, b = rnd(4, 64, 1536, std=0.1), rnd(5, 1536, dtype=F32)
    y = clear.linear(x, w, bias=b, act="gelu")
    R.close(y[-n:], R.linear(x[-n:], w, b, "gelu", None, BF))
    R.close(y[:n], R.linear(x[:n], w, b, "gelu", None, BF))


def test_linear_grad_long_sums():
    """Sums over many rows, some thousands of 64-row blocks, split and not."""
    x, dy, w = rnd(1, 300_001, 72), rnd(2, 300_001, 136), rnd(3, 72, 136, std=0.1)
    for act in (None, GELU_POLY):
        for got, want in zip(clear.linear_grad(dy, x, w, bias=rnd(4, 136, dtype=F32), act=act),
                             R.linear_grad(dy, x, w, rnd(4, 136, dtype=F32), act, F32)):
            R.close(got, want)


# ------------------------------------------------------------------------------------------------ attention
def attend(q_lens, k_lens, heads, kv, dim, dtype=BF, weights=None, causal=True, std=1.0, scale=None, seed=0):
    q = rnd(seed + 1, sum(q_lens), heads, dim, std=std, dtype=dtype)
    k, v = rnd(seed + 2, sum(k_lens), kv, dim, std=std, dtype=dtype), rnd(seed + 3, sum(k_lens), kv, dim, dtype=dtype)
    got = clear.prompt_attention(q, k, v, q_lens, k_lens, scale=scale, causal=causal, weights=weights)
    R.close(got, R.attention(q, k, v, q_lens, k_lens, dim**-0.5 if scale is None else scale, causal, weights))


@pytest.mark.parametrize("length", [1, 2, 31, 64, 127, 128, 129, 255, 256, 257, 400, 1025])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_lengths(length, dim):
    attend([length], [length], 4, 4, dim)


@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (12, 4), (12, 1), (9, 3), (16, 2), (5, 1), (128, 1)])
@pytest.mark.parametrize("dim,dtype", [(64, BF), (128, HF), (40, HF), (80, BF), (8, BF), (33, BF), (1, HF)])
def test_attention_heads(heads, kv, dim, dtype):
    attend([3, 130, 61], [3, 130, 61], heads, kv, dim, dtype)


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256)), (0.5, 0.25)], ids=["softmax", "poly7", "poly1"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_packed(weights, causal, dtype):
    """Ragged batches, earlier tokens, no queries, no keys, more queries than keys (the first see nothing)."""
    q_lens, k_lens = [1, 200, 0, 17, 130, 64, 5, 1], [1, 200, 40, 300, 130, 50, 0, 513]
    attend(q_lens, k_lens, 6, 2, 64, dtype, weights, causal, std=1.0 if weights is None else 0.5)


@pytest.mark.parametrize("past", [0, 1, 126, 127, 128, 2500, 20000])
@pytest.mark.parametrize("heads,kv", [(12, 12), (16, 2)])
def test_attention_single_tokens(past, heads, kv):
    attend([1, 1], [1 + past, 1 + past // 2], heads, kv, 64)
    attend([1, 2], [1 + past, 2 + past], heads, kv, 128, HF, tuple(A.softmax_poly(1 + past)), std=0.4)


def test_attention_many_short():
    n = 700
    lens = [i % 5 for i in range(n)]
    attend(lens, lens, 2, 2, 64)


def test_attention_empty():
    q = rnd(1, 4, 2, 64)
    none = rnd(2, 0, 2, 64)
    assert clear.prompt_attention(none, none, none, []).shape == (0, 2, 64)
    assert clear.prompt_attention(none, q, q, [0], [4]).shape == (0, 2, 64)
    assert not clear.prompt_attention(q, none, none, [4], [0]).any()


def test_attention_strides():
    """q, k, v as views of one projection, odd strides, transposed heads."""
    lens = [70, 133]
    qkv = rnd(1, 203, 3, 12, 64)
    q, k, v = qkv.unbind(1)
    R.close(clear.prompt_attention(q, k, v, lens), R.attention(q, k, v, lens, lens, 0.125, True, None))
    odd = rnd(2, 203 * 12 * 67).view(203, 12, 67)
    q, k, v = odd[..., :64], odd[..., 1:65], odd[..., 3:67]
    R.close(clear.prompt_attention(q, k, v, lens), R.attention(q, k, v, lens, lens, 0.125, True, None))
    t = rnd(3, 12, 203, 64).transpose(0, 1)
    R.close(clear.prompt_attention(t, t, t, lens), R.attention(t, t, t, lens, lens, 0.125, True, None))
    e = rnd(4, 203, 1, 64).expand(203, 4, 64)  # one head's keys shared by every head through a stride of zero
    q = rnd(5, 203, 4, 64)
    R.close(clear.prompt_attention(q, e, e, lens), R.attention(q, e, e, lens, lens, 0.125, True, None))


def test_attention_large_scores():
    """Scores far apart and far from zero: the running maximum moves, weights vanish."""
    attend([300], [300], 4, 2, 64, std=6.0)
    attend([300], [300], 4, 2, 64, std=1.0, scale=-0.7)
    attend([300], [300], 4, 2, 64, scale=0.0)
    n = 520
    q, v = rnd(1, n, 2, 64), rnd(2, n, 2, 64)
    k = (q[:1].float() * torch.linspace(-3, 3, n, device="cuda")[:, None, None]).to(BF)  # rising maxima
    R.close(clear.prompt_attention(q, k, v, [n]), R.attention(q, k, v, [n], [n], 0.125, True, None))


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
def test_attention_neighbours_stay_out(weights):
    """A sequence whose values and keys are not finite does not reach the sequences packed before and after it."""
    lens = [77, 50, 90]
    q, k, v = rnd(1, 217, 4, 64, std=0.5), rnd(2, 217, 4, 64, std=0.5), rnd(3, 217, 4, 64)
    want = R.attention(q, k, v, lens, lens, 0.125, True, weights)
    k[77:127], v[77:127] = math.nan, math.inf
    got = clear.prompt_attention(q, k, v, lens, weights=weights)
    for s in (slice(0, 77), slice(127, 217)):
        R.close(got[s], (want[0][s], want[1][s]))


@pytest.mark.parametrize("weights", [None, tuple(A.softmax_poly(256))], ids=["softmax", "poly"])
@pytest.mark.parametrize("bad", [0, 100, 127, 128, 199])
def test_attention_masked_keys_stay_out(weights, bad):
    """A later token's key and value that are not finite do not reach the queries that do not see it."""
    q, k, v = rnd(1, 200, 4, 64, std=0.5), rnd(2, 200, 2, 64, std=0.5), rnd(3, 200, 2, 64)
    want = R.attention(q, k, v, [200], [200], 0.125, True, weights)
    k[bad], v[bad] = math.nan, math.nan
    got = clear.prompt_attention(q, k, v, [200], weights=weights)
    R.close(got[:bad], (want[0][:bad], want[1][:bad]))
    assert torch.isnan(got[bad:]).all()
    v[bad] = math.inf
    k[bad] = 0
    got = clear.prompt_attention(q, k, v, [200], weights=weights)
    R.close(got[:bad], (want[0][:bad], want[1][:bad]))
    assert not torch.isfinite(got[bad]).any()


def test_attention_split_keys_not_finite():
    """Few queries against many keys, which are split over blocks: a key that only the last query sees."""
    n = 5000
    q, k, v = rnd(1, 2, 4, 64, std=0.5), rnd(2, n, 2, 64, std=0.5), rnd(3, n, 2, 64)
    want = R.attention(q, k, v, [2], [n], 0.125, True, None)
    v[n - 1] = math.inf
    got = clear.prompt_attention(q, k, v, [2], [n])
    R.close(got[:1], (want[0][:1], want[1][:1]))
    assert not torch.isfinite(got[1]).any()
    k[n - 1] = math.nan
    got = clear.prompt_attention(q, k, v, [2], [n])
    R.close(got[:1], (want[0][:1], want[1][:1]))
    assert torch.isnan(got[1]).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_is_the_same_every_time(dim):
    lens = [1300, 7, 900, 2100]
    q, k, v = rnd(1, sum(lens), 6, dim), rnd(2, sum(lens), 2, dim), rnd(3, sum(lens), 2, dim)
    one = clear.prompt_attention(q, k, v, lens)
    R.close(one, R.attention(q, k, v, lens, lens, dim**-0.5, True, None))
    for _ in range(20):
        assert torch.equal(clear.prompt_attention(q, k, v, lens), one)


def test_attention_far_offsets():
    """Rows past 2^31 elements of k and v."""
    rows = 140000
    kv = torch.zeros(rows, 129, 128, dtype=BF, device="cuda")  # 2.3e9 elements
    n = 300
    kv[-n:, 128] = rnd(1, n, 128)
    q = rnd(2, n, 1, 128)
    k = kv[:, 128:]
    got = clear.prompt_attention(q, k, k, [0, n], [rows - n, n])
    R.close(got, R.attention(q, k[-n:], k[-n:], [n], [n], 128**-0.5, True, None))


def test_attention_on_another_stream_and_in_a_graph():
    lens = [64, 200]
    q, k, v = (rnd(i, 264, 4, 64) for i in (1, 2, 3))
    want = clear.prompt_attention(q, k, v, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = clear.prompt_attention(q, k, v, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = clear.prompt_attention(q, k, v, lens)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ vocabulary
def vocab_case(rows, vocab, dim, dtype, std=2.0, seed=0):
    h, w = rnd(seed + 1, rows, dim, dtype=dtype), rnd(seed + 2, vocab, dim, std=std * dim**-0.5, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[1::4] = -100
    weight = torch.rand(rows, generator=g, device="cuda") / rows
    return h, w, t, weight


@pytest.mark.parametrize("rows,vocab,dim", [(1, 1000, 64), (1, 1, 8), (5, 33, 17), (127, 257, 72), (128, 4096, 128),
                                            (130, 12345, 200), (300, 50000, 96), (1500, 1003, 765), (64, 5000, 2048)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_vocab(rows, vocab, dim, dtype):
    h, w, t, weight = vocab_case(rows, vocab, dim, dtype)
    want = R.vocab(h, w, t, weight, -100)
    loss, lse = clear.vocab_loss(h, w, t)
    R.close(loss, want[0])
    R.close(lse, want[1])
    dh, dw = clear.vocab_loss_grad(h, w, t, lse, weight)
    R.close(dh, want[2])
    R.close(dw, want[3])


def test_vocab_slopes_beyond_l2():
    h, w, targets, weight = vocab_case(1100, 40000, 320, BF)
    loss, lse = clear.vocab_loss(h, w, targets)
    dh, dw = clear.vocab_loss_grad(h, w, targets, lse, weight)
    for got, want in zip((loss, lse, dh, dw), R.vocab(h, w, targets, weight, -100)):
        R.close(got, want)


def test_vocab_strides_and_needs():
    h, w, t, weight = vocab_case(90, 700, 64, BF)
    hs, ws = rnd(5, 90, 131)[:, 1:65], rnd(6, 700, 200, std=0.2)[:, 8:72]
    hs.copy_(h)
    ws.copy_(w)
    want = R.vocab(h, w, t, weight, -100)
    loss, lse = clear.vocab_loss(hs, ws, t)
    R.close(loss, want[0])
    dh, none = clear.vocab_loss_grad(hs, ws, t, lse, weight, needs=(True, False))
    assert none is None
    R.close(dh, want[2])
    none, dw = clear.vocab_loss_grad(hs, ws, t, lse, weight, needs=(False, True))
    assert none is None
    R.close(dw, want[3])


def test_vocab_ignored_and_odd_targets():
    h, w, t, weight = vocab_case(40, 300, 64, BF)
    t[:] = 7
    loss, lse = clear.vocab_loss(h, w, t, ignore=7)
    dh, dw = clear.vocab_loss_grad(h, w, t, lse, weight, ignore=7)
    assert not loss.any() and not dh.any() and not dw.any()
    t[:] = torch.arange(40, device="cuda")
    t[3], t[4] = 300, -5
    loss, lse = clear.vocab_loss(h, w, t)
    assert torch.isnan(loss[[3, 4]]).all() and torch.isfinite(loss).sum() == 38 and torch.isfinite(lse).all()
    t[:] = torch.where(torch.arange(40, device="cuda") % 2 == 0, 0, 299)  # the first and the last entry
    want = R.vocab(h, w, t, weight, -100)
    loss, lse = clear.vocab_loss(h, w, t)
    R.close(loss, want[0])
    for got, wa in zip(clear.vocab_loss_grad(h, w, t, lse, weight), want[2:]):
        R.close(got, wa)
    empty = clear.vocab_loss(h[:0], w, t[:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0,)
    dh, dw = clear.vocab_loss_grad(h[:0], w, t[:0], empty[1], weight[:0])
    assert dh.shape == (0, 64) and dw.shape == (300, 64) and not dw.any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_vocab_large_logits_and_weights(dtype):
    """Logits of hundreds; weights across six orders of magnitude, negative ones, zeros, all zeros."""
    h, w, t, weight = vocab_case(200, 3000, 64, dtype, std=60.0)
    weight = weight * 10.0 ** torch.linspace(-6, 0, 200, device="cuda") * torch.where(torch.arange(200, device="cuda") % 3 == 0, -1, 1)
    weight[5] = 0
    want = R.vocab(h, w, t, weight, -100)
    loss, lse = clear.vocab_loss(h, w, t)
    R.close(loss, want[0])
    R.close(lse, want[1])
    for got, wa in zip(clear.vocab_loss_grad(h, w, t, lse, weight), want[2:]):
        R.close(got, wa)
    dh, dw = clear.vocab_loss_grad(h, w, t, lse, torch.zeros_like(weight))
    assert not dh.any() and not dw.any()
    for f in (1e-30, 1e30):  # scales with the weight until the result's type ends
        if f < 1 or dtype == BF:
            dh, dw = clear.vocab_loss_grad(h, w, t, lse, weight * f)
            assert torch.isfinite(dh).all() and torch.isfinite(dw).all()


def test_vocab_gradient_against_differences():
    h, w, t, weight = vocab_case(30, 90, 24, BF)
    _, lse = clear.vocab_loss(h, w, t)
    grads = clear.vocab_loss_grad(h, w, t, lse, weight)
    bounds = R.vocab(h, w, t, weight, -100)[2:]

    def f(a, b):
        lg = a @ b.t()
        l = torch.logsumexp(lg, 1) - lg.gather(1, t.clamp_min(0)[:, None])[:, 0]
        return (torch.where(t != -100, l, 0.0) * weight.double()).sum()
    for i, (g, (_, bound)) in enumerate(zip(grads, bounds)):
        d = rnd(20 + i, *g.shape, dtype=torch.float64)
        at = [h.double(), w.double()]
        up, dn = list(at), list(at)
        up[i], dn[i] = up[i] + 1e-5 * d, dn[i] - 1e-5 * d
        slope = (f(*up) - f(*dn)) / 2e-5
        assert abs(slope - (g.double() * d).sum()) <= (bound * d.abs()).sum() + 1e-6 * (g.double() * d).abs().sum()


def test_vocab_nonfinite_row():
    h, w, t, weight = vocab_case(60, 500, 64, BF)
    want = R.vocab(h, w, t, weight, -100)
    h[8, 3] = math.nan
    loss, lse = clear.vocab_loss(h, w, t)
    rows = [i for i in range(60) if i != 8]
    assert torch.isnan(lse[8])
    R.close(loss[rows], tuple(x[rows] for x in want[0]))
    dh, _ = clear.vocab_loss_grad(h, w, t, lse, weight)
    R.close(dh[rows], tuple(x[rows] for x in want[2]))


def test_vocab_far_offsets():
    """A vocabulary past 2^31 elements: zeros but for its last entries."""
    vocab, dim, n = 2_900_000, 768, 64
    w = torch.zeros(vocab, dim, dtype=BF, device="cuda")
    w[-n:] = rnd(1, n, dim, std=0.1)
    h = rnd(2, 5, dim)
    t = torch.tensor([vocab - 1, 0, vocab - n, -100, vocab - 2], device="cuda")
    loss, lse = clear.vocab_loss(h, w, t)
    lg = h.double() @ w[-n:].double().t()
    want = torch.log(vocab - n + torch.exp(lg).sum(1))
    hit = torch.zeros(5, dtype=torch.float64, device="cuda")
    hit[0], hit[2], hit[4] = lg[0, -1], lg[2, 0], lg[4, -2]
    # a sum of 2.9e6 ones in blocks of 128 and their joining, and the logits' error
    err = (dim + 4) * R.S * (h.double().abs() @ w[-n:].double().abs().t()).amax(1) + 2.0**-16
    R.close(lse, (want, err))
    R.close(loss, (torch.where(t == -100, 0.0, want - hit), 2 * err))
    weight = torch.full((5,), 0.25, device="cuda")
    dh, dw = clear.vocab_loss_grad(h, w, t, lse, weight)
    p = torch.exp(lg - want[:, None])
    hot = torch.zeros(5, n, dtype=torch.float64, device="cuda")
    hot[0, -1] = hot[2, 0] = hot[4, -2] = 1.0
    d = (p - hot) * torch.where(t == -100, 0.0, 0.25).double()[:, None]
    ed = 2 * err[:, None] * p * 0.25 + R.U[BF] * d.abs() + 2.0**-133
    R.close(dh, (d @ w[-n:].double(), ed @ w[-n:].double().abs() + (n + 4) * R.S * (d.abs() @ w[-n:].double().abs()) + R.U[BF] * (d @ w[-n:].double()).abs() + 2.0**-133))
    R.close(dw[-n:], (d.t() @ h.double(), ed.t() @ h.double().abs() + 9 * R.S * (d.abs().t() @ h.double().abs()) + R.U[BF] * (d.t() @ h.double()).abs() + 2.0**-133))


def test_vocab_is_the_same_every_time():
    h, w, t, weight = vocab_case(513, 9001, 256, BF)
    loss, lse = clear.vocab_loss(h, w, t)
    one = clear.vocab_loss_grad(h, w, t, lse, weight)
    for _ in range(3):
        assert torch.equal(clear.vocab_loss(h, w, t)[0], loss)
        assert all(torch.equal(a, b) for a, b in zip(one, clear.vocab_loss_grad(h, w, t, lse, weight)))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x, w = rnd(1, 8, 32), rnd(2, 32, 16)
    q, k = rnd(3, 10, 4, 64), rnd(4, 10, 2, 64)
    t, lse = torch.zeros(8, dtype=torch.int64, device="cuda"), torch.zeros(8, device="cuda")
    vw = rnd(5, 20, 32)
    for call in (lambda: clear.linear(x, w.half()), lambda: clear.linear(x.float(), w.float()), lambda: clear.linear(x.cpu(), w),
                 lambda: clear.linear(x, w[:30]), lambda: clear.linear(x, w, bias=rnd(1, 15)),
                 lambda: clear.linear(x, w, bias=rnd(1, 16, dtype=HF)), lambda: clear.linear(x, w, residual=rnd(1, 8, 15)),
                 lambda: clear.linear(x, w, act="relu"), lambda: clear.linear(x, w, out_dtype=HF),
                 lambda: clear.linear(x[:, :0], w[:0]), lambda: clear.linear_grad(rnd(1, 8, 15), x, w),
                 lambda: clear.linear_grad(rnd(1, 8, 16, dtype=HF), x, w), lambda: clear.Poly(()), lambda: clear.Poly([1.0] * 9),
                 lambda: clear.Poly([1.0], 0.0), lambda: clear.Poly([math.nan]),
                 lambda: clear.prompt_attention(q, rnd(4, 10, 3, 64), rnd(4, 10, 3, 64), [10]),
                 lambda: clear.prompt_attention(q, k, rnd(4, 10, 2, 32), [10]), lambda: clear.prompt_attention(q, k, k, [4, 6], [10]),
                 lambda: clear.prompt_attention(rnd(1, 10, 2, 129), rnd(1, 10, 2, 129), rnd(1, 10, 2, 129), [10]),
                 lambda: clear.prompt_attention(q, k, k, [10], weights=[0.1] * 9),
                 lambda: clear.vocab_loss(x, rnd(5, 20, 31), t), lambda: clear.vocab_loss(x, vw, t[:7]),
                 lambda: clear.vocab_loss(x, vw, t.int()), lambda: clear.vocab_loss_grad(x, vw, t, lse.half(), lse),
                 lambda: clear.vocab_loss_grad(x, vw, t, lse, lse[:7])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: clear.prompt_attention(q, k, k, [11]), lambda: clear.prompt_attention(q, k, k, [12, -2]),
                 lambda: clear.prompt_attention(q, k, k, [10], scale=math.inf),
                 lambda: clear.prompt_attention(q, k, k, [10], weights=[math.nan])):
        with pytest.raises(L.PcbError):
            call()


# ------------------------------------------------------------------------------------------------ the path
def test_prefill_gives_the_caches_of_plain_layer():
    """The polynomial model: K, V of every layer and the output against model.plain_layer token by token (64 bits)."""
    cfg = M.ModelCfg(layers=2, d=128, width=128, heads=2, head_dim=64, mlp=512, tokens=32)
    rng = np.random.default_rng(3)
    weights = [M.random_layer(rng, 128, 512) for _ in range(2)]
    coeffs = A.softmax_poly(cfg.tokens)
    lens = [5, 32, 1]
    xs = [rng.normal(0, 1, (n, 128)) for n in lens]
    Ks, Vs, y = PF.prefill(torch.as_tensor(np.concatenate(xs), dtype=torch.float32, device="cuda"), lens,
                           PF.load(weights, dtype=HF), cfg)
    at = 0
    for b, x in enumerate(xs):
        caches = [[np.zeros((0, 128)), np.zeros((0, 128))] for _ in weights]
        for tok in x:
            out = M.plain_decode(tok, weights, caches, cfg, coeffs)
            # 16-bit operands of 11 bits through two layers of sums of terms of size one: a few units of 2^-11 each
            assert np.abs(y[at].double().cpu().numpy() - out).max() < 16 * 2.0**-11
            at += 1
        for l, (K, V) in enumerate(caches):
            assert np.abs(Ks[l][b].double().cpu().numpy() - K).max() < 16 * 2.0**-11
            assert np.abs(Vs[l][b].double().cpu().numpy() - V).max() < 16 * 2.0**-11


def test_prefill_exact_functions_and_refusals():
    cfg = M.ModelCfg(layers=1, d=128, width=128, heads=2, head_dim=64, mlp=512, tokens=64)
    layers = PF.load([M.random_layer(np.random.default_rng(1), 128, 512)], dtype=HF)
    x = rnd(1, 60, 128, dtype=F32)
    Ks, Vs, y = PF.prefill(x, [60], layers, cfg, poly=False)
    w = layers[0]

    def norm(t):
        return torch.nn.functional.layer_norm(t, (128,), eps=cfg.norm.eps)
    q, k, v = (norm(x.double()) @ w.wqkv.double() + w.bqkv.double()).view(60, 3, 2, 64).unbind(1)
    att = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1) for t in (q, k, v)), is_causal=True)
    r = att.transpose(0, 1).reshape(60, 128) @ w.wo.double() + w.bo.double() + x.double()
    want = R.act(norm(r) @ w.w_up.double() + w.b_up.double(), "gelu") @ w.w_down.double() + w.b_down.double() + r
    assert (y.double() - want).abs().max() < 16 * 2.0**-11
    assert (Ks[0][0].double() - k.reshape(60, 128)).abs().max() < 16 * 2.0**-11
    with pytest.raises(ValueError):
        PF.prefill(x, [59], layers, cfg)
    with pytest.raises(ValueError):
        PF.prefill(rnd(1, 65, 128, dtype=F32), [65], layers, cfg)


def test_fit_step_lowers_the_loss():
    """A step against the gradients lowers the mean loss by about the gradients' squared norm times the step."""
    cfg = M.ModelCfg(layers=1, d=128, width=128, heads=2, head_dim=64, mlp=512, tokens=64)
    layer = PF.load([M.random_layer(np.random.default_rng(1), 128, 512)])[0]
    tail = PF.Tail(layer, rnd(1, 500, 128, std=0.1))
    r = rnd(2, 256, 128, dtype=F32)
    t = torch.randint(0, 500, (256,), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    t[::9] = -100
    loss, grads = PF.fit_step(r, t, tail, cfg)
    sq = sum(float(g.double().square().sum()) for g in grads.values())
    step = 0.05 / sq  # a fall of about 0.05
    for name, g in grads.items():
        owner = tail if name == "head" else layer
        old = getattr(owner, name)
        setattr(owner, name, (old.float() - step * g.float()).to(old.dtype))
    after, _ = PF.fit_step(r, t, tail, cfg)
    assert 0.02 < float(loss - after) < 0.08, (float(loss), float(after))
