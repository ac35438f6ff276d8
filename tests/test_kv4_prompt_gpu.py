"""Prompts over the 4-bit KV cache where the kernel for prompts takes the call (which every test looks up), against 64 bits (needs a B200).

Its operands are fp16: probabilities, values and keys are rounded, by e = 2^-11 relative at most each; what is far below the largest visible
magnitude is held to 2^-25 of it, as probabilities are (2^-24, times 2^6): 2^-22 max|v|.  The roundings of p and v add up to 2 e sum p|v| at most.
A score moves by d = scale * sum q k e with independent roundings: by more than 7 e scale |q k| (2-norm of the products) with a probability
below 2 exp(-49/2) (Hoeffding) each, and the context by 2 d sum p|v| at most.  The result is rounded once, by 2^-8 of the value:
    |got - want| <= 2^-8 |want| + (2 e + 2 * 7 e |q k|) sum p|v| + 2^-22 max|v|.
Over a whole result the roundings are independent, with a standard deviation of at most e each, so its 2-norm is held to
    ||got - want|| <= 2^-8 ||want|| + 2 e || (2 + |q k|) sqrt(sum p^2 v^2) || + 2^-22 ||max|v|||
(twice the expectation of what does not come from the last rounding)."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4
from test_kv4_gpu import randn

pytestmark = pytest.mark.gpu

FP16 = 2.0 ** -11


def attend_prompt(c, q, pos, **kw):
    took, got = R.kernels(lambda: c.attend(q, pos, **kw))
    assert took == {"prompt"}
    return got


def assert_near(got, q, k, v, pos, slots, heads, scale, window=0, sinks=0, e=FP16, rows=None):
    """``rows [n, T]``: which of them count (all by default)."""
    args = (q, k, v, pos, slots, heads, scale, window, sinks)
    want, top, (pv, qk) = R.attend(*args)
    dev = R.spread(*args)
    if rows is not None:
        got, want, top, pv, qk, dev = (t[rows] for t in (got, want, top, pv, qk, dev))
    off = got.double() - want
    far = off.abs() - (2.0 ** -8 * want.abs() + (2 * e + 14 * e * qk) * pv + 2.0 ** -22 * top)
    assert bool((far <= 0).all()), float(far.max())
    assert float(off.norm()) <= 2.0 ** -8 * float(want.norm()) + 2 * e * float(((2 + qk) * dev).norm()) + 2.0 ** -22 * float(top.norm())


def size(D):
    """Tokens, query heads, KV heads of a call that fills the GPU well enough for this kernel."""
    return (320, 32, 8) if D == 128 else (400, 32, 8)


# ----------------------------------------------------------------------------- small scores
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_gain,k_gain,scale", [(0.0, 0.0, None), (0.0, 1e-3, None), (1e-20, 1e-20, None), (1e-12, 0.0, None), (1.0, 1.0, 1e-39), (1e-28, 1e-10, 1e37),
                                                 (1e-30, 1e-30, 1e-30), (0.0, 1e30, -1.0)])
def test_small_queries_and_keys(D, q_gain, k_gain, scale):
    """Scores of nothing, or of next to nothing, behind a causal border: the mean of what a row sees, and no product of small factors that
    makes a masked score no number."""
    T, heads, n_kv = size(D)
    slots = T + 50
    c = KVCache4(1, n_kv, slots, D)
    c.append(randn(1, 1, slots, n_kv * D, gain=k_gain), randn(2, 1, slots, n_kv * D), torch.arange(slots, device="cuda"))
    q = randn(3, 1, T, heads * D, gain=q_gain)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    scale = D ** -0.5 if scale is None else scale
    got = attend_prompt(c, q, pos, scale=scale)
    assert_near(got, q, *R.cache_values(c.tiles, D), pos, slots, heads, scale)


@pytest.mark.parametrize("D", [64, 128])
def test_a_fresh_cache(D):
    T, heads, n_kv = size(D)
    pos = torch.arange(T, device="cuda")[None]
    c = KVCache4(1, n_kv, T, D)
    assert not bool(attend_prompt(c, torch.zeros(1, T, heads * D, dtype=torch.bfloat16, device="cuda"), pos).any())
