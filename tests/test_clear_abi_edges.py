"""Refusals of the clear half's C entries at the ends of their ranges, on the host (the pointers are fakes that no kernel
sees)."""
import pytest

from perseus_b200 import _lib as L
from tests.test_clear_abi import attention, grad, linear, vocab

MOST = 2**31 - 1025  # indexes of tiles that reach past the last row or column stay within 32 bits


def refused(op, a, word):
    lib = L.lib()
    assert getattr(lib, f"pcb_clear_{op}_ws")(a) == -1
    assert word in lib.pcb_last_error().decode()
    assert getattr(lib, f"pcb_clear_{op}")(a, None, 0, None) == -1


@pytest.mark.parametrize("op,make,over", [
    ("linear", linear, dict(m=MOST + 1)), ("linear", linear, dict(k=MOST + 1, x_pitch=MOST + 1)),
    ("linear", linear, dict(n=MOST + 1, w_pitch=MOST + 1, y_pitch=MOST + 1)), ("linear_grad", grad, dict(m=MOST + 1)),
    ("linear_grad", grad, dict(k=MOST + 1, x_pitch=MOST + 1, dx_pitch=MOST + 1)),
    ("linear_grad", grad, dict(n=MOST + 1, w_pitch=MOST + 1, dy_pitch=MOST + 1, dw_pitch=MOST + 1)),
    ("attention", attention, dict(q_rows=MOST + 1)), ("attention", attention, dict(k_rows=MOST + 1)),
    ("vocab_loss", vocab, dict(rows=MOST + 1)), ("vocab_loss", vocab, dict(vocab=MOST + 1)),
    ("vocab_loss", vocab, dict(dim=MOST + 1, h_pitch=MOST + 1, w_pitch=MOST + 1))],
    ids=lambda x: next(iter(x)) if isinstance(x, dict) else x if isinstance(x, str) else "")
def test_sizes(op, make, over):
    refused(op, make(**over), str(MOST + 1) if op != "attention" else str(MOST))


@pytest.mark.parametrize("op,make,over", [
    ("linear", linear, dict(x=0x1001)), ("linear", linear, dict(w=0x1001)), ("linear", linear, dict(y=0x1001)),
    ("linear", linear, dict(y=0x1002, y_type=2)), ("linear", linear, dict(bias=0x1001)),
    ("linear", linear, dict(bias=0x1002, bias_type=2)), ("linear", linear, dict(residual=0x1001, residual_pitch=32)),
    ("linear", linear, dict(residual=0x1002, residual_type=2, residual_pitch=32)),
    ("linear_grad", grad, dict(dy=0x1001)), ("linear_grad", grad, dict(x=0x1001)), ("linear_grad", grad, dict(w=0x1001)),
    ("linear_grad", grad, dict(dx=0x1001)), ("linear_grad", grad, dict(dw=0x1001)), ("linear_grad", grad, dict(bias=0x1001)),
    ("linear_grad", grad, dict(bias=0x1002, bias_type=2)), ("linear_grad", grad, dict(db=0x1001)),
    ("linear_grad", grad, dict(db=0x1002, db_type=2)),
    ("attention", attention, dict(q=0x1001)), ("attention", attention, dict(k=0x1001)),
    ("attention", attention, dict(v=0x1001)), ("attention", attention, dict(out=0x1001)),
    ("vocab_loss", vocab, dict(h=0x1001)), ("vocab_loss", vocab, dict(w=0x1001)), ("vocab_loss", vocab, dict(targets=0x1004)),
    ("vocab_loss", vocab, dict(loss=0x1002)), ("vocab_loss", vocab, dict(lse=0x1002))],
    ids=lambda x: "-".join(f"{n}" for n in x) if isinstance(x, dict) else x if isinstance(x, str) else "")
def test_pointers_off_their_elements(op, make, over):
    """A device pointer that no load of its type can take is refused before any launch."""
    refused(op, make(**over), "off its elements")


def test_vocab_gradient_pointers_off_their_elements():
    refused("vocab_grad", L.ClearVocabGrad(vocab(), 0x6002, 0x7000, 0x8000, 64, 64), "off its elements")
    refused("vocab_grad", L.ClearVocabGrad(vocab(), 0x6000, 0x7001, 0x8000, 64, 64), "off its elements")
    refused("vocab_grad", L.ClearVocabGrad(vocab(), 0x6000, 0x7000, 0x8001, 64, 64), "off its elements")
    refused("vocab_grad", L.ClearVocabGrad(vocab(targets=0x1004), 0x6000, 0x7000, 0x8000, 64, 64), "off its elements")
