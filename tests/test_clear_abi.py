"""The clear half's C entries without a GPU: refusals on the host before any launch (the pointers are fakes that no
kernel sees), and the workspace sizes."""
import ctypes as C

import pytest

from perseus_b200 import _lib as L


def linear(**over):
    a = dict(x=0x1000, w=0x2000, bias=None, residual=None, y=0x3000, x_pitch=64, w_pitch=32, residual_pitch=0, y_pitch=32, m=4,
             k=64, n=32, type=0, w_cols=0, bias_type=0, residual_type=0, y_type=0, act=0, bound=1.0)
    a.update(over)
    return L.ClearLinear(*[a[f[0]] for f in L.ClearLinear._fields_[:-1]])


def grad(**over):
    a = dict(dy=0x1000, x=0x2000, w=0x3000, bias=None, dx=0x4000, dw=0x5000, db=None, dy_pitch=32, x_pitch=64, w_pitch=32,
             dx_pitch=64, dw_pitch=32, m=4, k=64, n=32, type=0, w_cols=0, bias_type=0, db_type=0, act=0, bound=1.0)
    a.update(over)
    return L.ClearLinearGrad(*[a[f[0]] for f in L.ClearLinearGrad._fields_[:-1]])


LENS = (C.c_int32 * 2)(3, 5)


def attention(**over):
    a = dict(q=0x1000, k=0x2000, v=0x3000, out=0x4000, q_lens=C.addressof(LENS), k_lens=C.addressof(LENS), q_pitch=256, q_head=64,
             k_pitch=128, k_head=64, v_pitch=128, v_head=64, out_pitch=256, out_head=64, q_rows=8, k_rows=8, nseq=2, heads=4,
             kv_heads=2, dim=64, type=0, causal=1, ncoef=0, scale=0.125)
    a.update(over)
    return L.ClearAttention(*[a[f[0]] for f in L.ClearAttention._fields_[:-1]])


def vocab(**over):
    a = dict(h=0x1000, w=0x2000, targets=0x3000, loss=0x4000, lse=0x5000, h_pitch=64, w_pitch=64, ignore=-100, rows=4, vocab=100,
             dim=64, type=0)
    a.update(over)
    return L.ClearVocab(*[a[f[0]] for f in L.ClearVocab._fields_])


BAD = [("linear", linear, dict(x=None)), ("linear", linear, dict(y=None)), ("linear", linear, dict(k=0)),
       ("linear", linear, dict(m=-1)), ("linear", linear, dict(type=2)), ("linear", linear, dict(act=3)),
       ("linear", linear, dict(act=2, bound=0.0)), ("linear", linear, dict(x_pitch=63)), ("linear", linear, dict(w_pitch=31)),
       ("linear", linear, dict(w_cols=1)), ("linear", linear, dict(y_type=1)), ("linear", linear, dict(bias=0x10, bias_type=1)),
       ("linear_grad", grad, dict(dy=None)), ("linear_grad", grad, dict(n=0)), ("linear_grad", grad, dict(type=2)),
       ("linear_grad", grad, dict(dw_pitch=31)), ("linear_grad", grad, dict(db=0x10, db_type=1)),
       ("attention", attention, dict(q=None)), ("attention", attention, dict(heads=3)), ("attention", attention, dict(dim=129)),
       ("attention", attention, dict(q_rows=9)), ("attention", attention, dict(k_rows=7)), ("attention", attention, dict(ncoef=9)),
       ("attention", attention, dict(q_lens=None)), ("attention", attention, dict(scale=float("nan"))),
       ("attention", attention, dict(q_pitch=-1)), ("attention", attention, dict(type=2)),
       ("vocab_loss", vocab, dict(w=None)), ("vocab_loss", vocab, dict(loss=None)), ("vocab_loss", vocab, dict(vocab=0)),
       ("vocab_loss", vocab, dict(h_pitch=63)), ("vocab_loss", vocab, dict(type=2))]


@pytest.mark.parametrize("op,make,over", BAD, ids=[f"{o}-{next(iter(v))}" for o, _, v in BAD])
def test_refused(op, make, over):
    a = make(**over)
    lib = L.lib()
    assert getattr(lib, f"pcb_clear_{op}_ws")(a) == -1
    assert op.split("_")[0] in lib.pcb_last_error().decode()
    assert getattr(lib, f"pcb_clear_{op}")(a, None, 0, None) == -1


def test_null_and_workspace():
    lib = L.lib()
    for op in ("linear", "linear_grad", "attention", "vocab_loss", "vocab_grad"):
        assert getattr(lib, f"pcb_clear_{op}_ws")(None) == -1
        assert getattr(lib, f"pcb_clear_{op}")(None, None, 0, None) == -1
    g = L.ClearVocabGrad(vocab(), 0x6000, 0x7000, 0x8000, 64, 64)
    need = lib.pcb_clear_vocab_grad_ws(g)
    assert need > 0
    assert lib.pcb_clear_vocab_grad(g, None, 0, None) == -1 and "workspace" in lib.pcb_last_error().decode()
    assert lib.pcb_clear_vocab_grad(g, 0x1001, need, None) == -1
    assert lib.pcb_clear_vocab_grad(g, 0x1000, need - 1, None) == -1
    g.weight = None
    assert lib.pcb_clear_vocab_grad_ws(g) == -1


def test_nothing_to_do():
    """Empty operands return without a launch."""
    lib = L.lib()
    before = lib.pcb_launch_count()
    assert lib.pcb_clear_linear(linear(m=0), None, 0, None) == 0 and lib.pcb_clear_linear(linear(n=0), None, 0, None) == 0
    assert lib.pcb_clear_attention(attention(nseq=0, q_rows=0, k_rows=0), None, 0, None) == 0
    assert lib.pcb_clear_vocab_loss(vocab(rows=0), None, 0, None) == 0
    assert lib.pcb_launch_count() == before
