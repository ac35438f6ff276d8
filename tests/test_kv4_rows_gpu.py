"""Attention of few rows over the 4-bit KV cache where the tokens of a call see slots of very different magnitude, against 64 bits (needs a B200).

Weights times value scales are 16-bit floats, e = 2^-11 relative at most each and 2^-31 of the largest value scale of the group that a row sees; scores, sums and
results are fp32 and the tensor cores' sums; one rounding to bf16 at the end:
    |got - want| <= 2^-8 |want| + 2 e sum p|v| + 2^-18 max|v|,    ||got - want|| <= 2^-8 ||want|| + 2 e ||sqrt(sum p^2 v^2)|| + 2^-18 ||max|v|||.
The last term: a tensor core's sum may lose 2^-23 of itself with every product that is added; a warp adds at most 20 in these tests, to sums of codes and
of zeros that grow to 3 max|v| together: 20 / 2 * 3 * 2^-23 max|v|.  The 2-norm is that of each row."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4
from test_kv4_gpu import randn

pytestmark = pytest.mark.gpu

E = 2.0 ** -11


def assert_near(got, q, k, v, pos, slots, heads, scale, window=0, sinks=0):
    args = (q, k, v, pos, slots, heads, scale, window, sinks)
    want, top, (pv, _) = R.attend(*args)
    off = got.double() - want
    far = off.abs() - (2.0 ** -8 * want.abs() + 2 * E * pv + 2.0 ** -18 * top)
    assert bool((far <= 0).all()), float(far.max())
    if not bool((pos < 0).all()):
        # row by row, so that one of large values does not cover the others
        norm = lambda t: t.view(-1, t.shape[-1]).norm(dim=1)
        assert bool((norm(off) <= 2.0 ** -8 * norm(want) + 2 * E * norm(R.spread(*args)[0]) + 2.0 ** -18 * norm(top)).all())


# ----------------------------------------------------------------------------- magnitudes far apart
@pytest.mark.parametrize("T,heads,n_kv,D,slots", [(5, 8, 2, 128, 200), (5, 4, 2, 64, 200), (7, 4, 1, 64, 200), (40, 4, 2, 64, 200), (11, 4, 2, 128, 300), (6, 2, 1, 192, 200),
                                                  (20, 4, 2, 256, 200), (3, 8, 1, 128, 40000), (5, 4, 1, 64, 40000), (5, 2, 1, 256, 40000), (2, 8, 8, 128, 9000)])
@pytest.mark.parametrize("size_of", [1e8, 1e13, 1e35])
def test_a_huge_value_does_not_reach_rows_that_do_not_see_it(T, heads, n_kv, D, slots, size_of):
    """Tokens one after the other, the middle one's value far above all others in one group: the tokens before it, and those whose window has left
    it behind, are what they are without it, though they share a tile of columns and of slots."""
    c = KVCache4(2, n_kv, slots, D)
    at = slots - 60
    pos = torch.stack([at - T // 2 + torch.arange(T), at - 1 - torch.arange(T)]).cuda()
    k, v = randn(1, 2, slots, n_kv * D), randn(2, 2, slots, n_kv * D)
    v[:, at, D - 60] = size_of                                                        # KV head 0, last group
    v[1, at - 33, D * (n_kv - 1) + 5] = -size_of                                      # the other end of the other sequence's window
    c.append(k, v, torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 2, T, heads * D)
    for window, sinks in ((0, 0), (3, 0), (32, 0), (32, 4)):
        got = c.attend(q, pos, window=window, sinks=sinks)
        assert_near(got, q, kd, vd, pos, slots, heads, D ** -0.5, window, sinks)
    far = pos.clone()
    far[0] = -1                                                                       # padding, and tokens that begin far apart
    far[1, 0] = 3
    assert_near(c.attend(q, far, window=40), q, kd, vd, far, slots, heads, D ** -0.5, 40)


@pytest.mark.parametrize("T,heads,D", [(1, 4, 128), (6, 4, 128), (9, 2, 64), (4, 2, 256)])
def test_magnitudes_that_fall_and_rise_by_many_powers_of_two(T, heads, D):
    """Values of 2^-60 to 2^60 from slot to slot: every row against the largest that it sees itself."""
    slots = 900
    c = KVCache4(1, 1, slots, D)
    rise = torch.exp2(60 * torch.sin(torch.arange(slots, device="cuda").float() / 60))[None, :, None]
    c.append(randn(1, 1, slots, D), (randn(2, 1, slots, D).float() * rise).bfloat16(), torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 1, T, heads * D)
    for end in (40, 95, 288, 480, 899):
        for window in (0, 1, 9):
            pos = (end - 7 * T + 7 * torch.arange(1, T + 1, device="cuda"))[None]
            assert_near(c.attend(q, pos, window=window), q, kd, vd, pos, slots, heads, D ** -0.5, window)
