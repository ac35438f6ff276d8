"""Prompts over the 4-bit KV cache where the kernel for prompts takes the call (which every test looks up), against 64 bits (needs a B200).

Its operands are fp16: probabilities, values and keys are rounded, by e = 2^-11 relative at most each; what is far below the largest visible
magnitude is held to 2^-25 of it, as probabilities are (2^-24, times 2^6): 2^-22 max|v|.  The roundings of p and v add up to 2 e sum p|v| at most.
A score moves by d = scale * sum q k e with independent roundings: by more than 7 e scale |q k| (2-norm of the products) with a probability
below 2 exp(-49/2) (Hoeffding) each, and the context by 2 d sum p|v| at most.

Codes are expanded by a multiply-add whose constant -(2^11 + z) s is rounded twice, by 2^-13 of a step s each: a value is off by 2^-12 s, and 15 s is
at most 2 max|v| of its group (and its own rounding to bf16, 2^-8): 2^-14 max|v|.  In a key it is the same for half the channels of a group:
scale 2^-12 s sum|q| over 32 channels, at most 2^-12 s sqrt(32) scale |q| for each group; s is a third of the standard deviation of 64 normal
values (range 4.8), so for up to two groups together at most 2^-12 sqrt(2) sqrt(32) / 3 scale |q k| < 2 e scale |q k|: 9 in place of the 7 above.

The result is rounded once, by 2^-8 of the value:
    |got - want| <= 2^-8 |want| + (2 e + 2 * 9 e |q k|) sum p|v| + (2^-14 + 2^-22) max|v|.
Over a whole result the roundings are independent, with a standard deviation of at most e each, so its 2-norm is held to
    ||got - want|| <= 2^-8 ||want|| + 2 e || (2 + |q k|) sqrt(sum p^2 v^2) || + 2^-14 || max|v| sqrt(sum p^2) || + 2^-22 ||max|v|||
(twice the expectation of what does not come from the last rounding)."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4
from test_kv4_gpu import copy_slots, filled, randn

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
    dev, even = R.spread(*args)
    if rows is not None:
        got, want, top, pv, qk, dev, even = (t[rows] for t in (got, want, top, pv, qk, dev, even))
    off = got.double() - want
    far = off.abs() - (2.0 ** -8 * want.abs() + (2 * e + 18 * e * qk) * pv + (2.0 ** -14 + 2.0 ** -22) * top)
    assert bool((far <= 0).all()), float(far.max())
    assert float(off.norm()) <= (2.0 ** -8 * float(want.norm()) + 2 * e * float(((2 + qk) * dev).norm()) + 2.0 ** -14 * float((top * even).norm())
                                 + 2.0 ** -22 * float(top.norm()))


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


@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_zeros(D):
    T, heads, n_kv = size(D)
    c, k, v = filled(1, n_kv, T, D, gain=1e-3)
    q = randn(3, 1, T, heads * D)
    q[:, 5:140] = 0.0
    q[:, 300] = 0.0
    pos = torch.arange(T, device="cuda")[None]
    assert_near(attend_prompt(c, q, pos), q, k, v, pos, T, heads, D ** -0.5)


# ----------------------------------------------------------------------------- masks, sizes
CASES = [  # n, T, heads, n_kv, D, slots, positions of the last token per sequence, window, sinks, gain
    (1, 320, 32, 8, 128, 600, [599], 0, 0, 1.0),               # five key tiles
    (1, 400, 32, 8, 64, 700, [690], 0, 0, 1.0),
    (4, 100, 32, 8, 128, 128, [99, 127, 100, 120], 0, 0, 1.0),  # one
    (4, 100, 32, 8, 64, 128, [99, 127, 100, 120], 0, 0, 1.0),
    (3, 130, 32, 8, 128, 500, [129, 499, 300], 0, 0, 1.0),     # sequences
    (3, 150, 32, 4, 64, 500, [149, 499, 255], 0, 0, 1.0),
    (2, 600, 7, 1, 128, 900, [899, 620], 0, 0, 1.0),           # heads that do not divide 128 rows
    (2, 700, 9, 3, 64, 900, [899, 700], 0, 0, 1.0),
    (2, 150, 40, 1, 128, 600, [599, 149], 0, 0, 1.0),
    (1, 1000, 8, 8, 128, 1000, [999], 0, 0, 1.0),              # no sharing
    (1, 1200, 8, 8, 64, 1300, [1250], 0, 0, 1.0),
    (1, 80, 128, 1, 128, 300, [299], 0, 0, 1.0),               # a token a CTA
    (4, 64, 32, 8, 128, 4096, [4095, 63, 2000, 4000], 0, 0, 1.0),     # many key tiles
    (1, 400, 32, 8, 128, 3000, [2999], 0, 0, 12.0),            # scores far apart: the maximum moves
    (1, 400, 32, 8, 64, 1500, [1499], 0, 0, 12.0),
    (1, 700, 16, 2, 128, 1500, [1400], 300, 5, 1.0),           # windows; a gap behind the first slots
    (2, 400, 32, 8, 128, 2000, [1900, 1000], 100, 3, 1.0),
    (1, 900, 16, 4, 64, 1500, [1400], 200, 130, 1.0),          # first slots of more than a key tile
    (1, 400, 32, 8, 64, 600, [599], 1, 0, 1.0),                # a window of one, without and with first slots
    (1, 400, 32, 8, 64, 600, [599], 1, 1, 1.0),
    (1, 320, 32, 8, 128, 600, [599], 64, 530, 1.0),            # first slots that reach into the window; more than there are
    (1, 320, 32, 8, 128, 600, [599], 64, 5000, 1.0),
    (1, 320, 32, 8, 128, 600, [599], 1 << 30, 0, 1.0),
]


@pytest.mark.parametrize("n,T,heads,n_kv,D,slots,last,window,sinks,gain", CASES)
def test_attention_matches_fp64(n, T, heads, n_kv, D, slots, last, window, sinks, gain):
    c, k, v = filled(n, n_kv, slots, D, seed=slots)
    q = randn(T + 1, n, T, heads * D, gain=gain)
    pos = torch.stack([torch.arange(p - T + 1, p + 1) for p in last]).cuda()
    assert int(pos.min()) >= 0
    got = attend_prompt(c, q, pos, window=window, sinks=sinks)
    assert_near(got, q, k, v, pos, slots, heads, D ** -0.5, window, sinks)
    assert torch.equal(got, c.attend(q, pos, window=window, sinks=sinks)) and c.device_status() == 0
