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
