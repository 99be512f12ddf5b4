"""The clear half's operators (perseus_b200.clear) where values, sizes or masks are at their ends, against the 64-bit forms
of tests/_clear_ref.py."""
import math

import pytest
import torch

from perseus_b200 import attention as A
from perseus_b200 import clear
from tests import _clear_ref as R

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


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
