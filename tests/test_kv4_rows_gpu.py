"""Attention of few rows over the 4-bit KV cache where its work goes by a list of tiles in equal ranges (which needs scratch, and every test
asks for it), and where the tokens of a call see slots of very different magnitude; against 64 bits (needs a B200).

Weights times value scales are 16-bit floats, e = 2^-11 relative at most each and 2^-31 of the largest value scale of the group that a row sees; scores, sums and
results are fp32 and the tensor cores' sums; one rounding to bf16 at the end:
    |got - want| <= 2^-8 |want| + 2 e sum p|v| + 2^-16 max|v|,    ||got - want|| <= 2^-8 ||want|| + 2 e ||sqrt(sum p^2 v^2)|| + 2^-16 ||max|v|||.
The last term: a tensor core cuts each of the 16 products of a step at a quarter of the last place of its running sum, 2^-21 of it in all at most; a warp
takes at most 20 steps in these tests, to sums of codes and of zeros that grow to 3 max|v| together: 20 / 2 * 3 * 2^-21 max|v| < 2^-16 max|v|.  The
2-norm is that of each row."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4, _lib
from test_kv4_gpu import filled, randn

pytestmark = pytest.mark.gpu

E = 2.0 ** -11


def assert_near(got, q, k, v, pos, slots, heads, scale, window=0, sinks=0):
    args = (q, k, v, pos, slots, heads, scale, window, sinks)
    want, top, (pv, _) = R.attend(*args)
    off = got.double() - want
    far = off.abs() - (2.0 ** -8 * want.abs() + 2 * E * pv + 2.0 ** -16 * top)
    assert bool((far <= 0).all()), float(far.max())
    if not bool((pos < 0).all()):
        # row by row, so that one of large values does not cover the others
        norm = lambda t: t.view(-1, t.shape[-1]).norm(dim=1)
        assert bool((norm(off) <= 2.0 ** -8 * norm(want) + 2 * E * norm(R.spread(*args)[0]) + 2.0 ** -16 * norm(top)).all())


def needs_scratch(c, q, window=0, sinks=0):
    n, T, width = q.shape
    assert R.form(c, n, T, width // c.head_dim, window, sinks) == _lib.KV4_LIST
    return _lib.load().cobalt_kv4_attend_scratch_bytes(n, T, width // c.head_dim, c.n_kv_heads, c.head_dim, c.slots, window, sinks)


# ----------------------------------------------------------------------------- the list of tiles
LISTS = [  # n, T, heads, n_kv, D, slots, positions of the last token per sequence, window, sinks: one, two, three and four groups of eight columns
    (4, 1, 16, 4, 128, 30000, [29999, 31, 12345, 20000], 0, 0),
    (3, 3, 10, 2, 128, 30000, [29999, 2, 17000], 0, 0),
    (2, 1, 12, 1, 128, 30000, [29999, 64], 25000, 3),
    (1, 9, 4, 1, 128, 60000, [59990], 0, 0),                   # three tiles of columns
    (5, 3, 4, 1, 64, 40000, [39999, 5000, 2, 30, 31999], 0, 0),
    (3, 5, 4, 1, 64, 40000, [39999, 4, 20001], 0, 0),
    (2, 5, 8, 2, 64, 40000, [39000, 39999], 35000, 40),
    (1, 17, 4, 1, 64, 60000, [59999], 0, 0),
    (2, 8, 4, 1, 64, 40000, [39999, 100], 0, 0),
    (1, 40, 2, 1, 64, 60000, [59999], 0, 0),
    (1, 3, 4, 1, 192, 60000, [59999], 0, 0),
    (2, 5, 2, 1, 256, 30000, [29998, 7], 0, 0),
]


@pytest.mark.parametrize("n,T,heads,n_kv,D,slots,last,window,sinks", LISTS)
def test_lists_match_fp64(n, T, heads, n_kv, D, slots, last, window, sinks):
    c, k, v = filled(n, n_kv, slots, D, seed=slots)
    q = randn(T + 1, n, T, heads * D)
    pos = torch.stack([torch.arange(p - T + 1, p + 1) for p in last]).cuda()
    assert needs_scratch(c, q, window, sinks) > 0
    got = c.attend(q, pos, window=window, sinks=sinks)
    assert_near(got, q, k, v, pos, slots, heads, D ** -0.5, window, sinks)
    assert torch.equal(got, c.attend(q, pos, window=window, sinks=sinks)) and c.device_status() == 0
    pos[0, 0] = -1                                                                     # padding, and a token behind the cache
    pos[-1, -1] = slots + 5
    assert_near(c.attend(q, pos, window=window, sinks=sinks), q, k, v, pos, slots, heads, D ** -0.5, window, sinks)


def test_two_streams_at_once_with_scratch():
    """Calls that need scratch, at once on two streams and from a captured graph: results are those of one stream."""
    c, _, _ = filled(2, 2, 40000, 64)
    q = [randn(i, 1, 3, 8 * 64) for i in range(2)]
    pos = [torch.tensor([[39997, 39998, 39999]], device="cuda") - 7777 * i for i in range(2)]
    assert needs_scratch(c, q[0]) > 0
    want = [c.attend(q[i], pos[i], seq=i) for i in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = [c.attend(q[i], pos[i], seq=i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(q[i], pos[i], seq=i))
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i]) and all(torch.equal(a, b) for a, b in zip(inside, want))


def test_graphs_with_scratch_follow_positions():
    """Two graphs of one cache, replayed in turn with other queries and positions, eager calls between them."""
    c, k, v = filled(2, 1, 30000, 128)
    q, pos = randn(1, 2, 3, 8 * 128), torch.tensor([[10, 11, 12], [100, 101, 102]], device="cuda")
    assert needs_scratch(c, q) > 0
    c.attend(q, pos)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(q, pos))
        graphs.append(g)
    for step in range(6):
        pos += torch.tensor([[4900], [977 * step]], device="cuda")
        q.copy_(randn(10 + step, *q.shape))
        graphs[step % 2].replay()
        assert torch.equal(outs[step % 2], c.attend(q, pos))
    assert_near(outs[1], q, k, v, pos, 30000, 8, 128 ** -0.5)


def test_scratch_is_checked():
    """Too small, none, or off its boundary: an error code, nothing launched."""
    c, _, _ = filled(1, 1, 40000, 64)
    q = randn(1, 1, 1, 4 * 64)
    pos = torch.tensor([[39999]], device="cuda")
    lib, need = _lib.load(), needs_scratch(c, q)
    assert need > 0
    scratch, out = torch.empty(need + 256, dtype=torch.uint8, device="cuda"), torch.full_like(q, 5.0)
    for at, size in ((None, need), (scratch.data_ptr(), need - 1), (scratch.data_ptr() + 16, need)):
        rc = lib.cobalt_kv4_attend(q.data_ptr(), 256, c.tiles.data_ptr(), 0, pos.data_ptr(), 0, out.data_ptr(), 1, 1, 4, 1, 64, 40000, 0, 0, 0.125, at, size,
                                   torch.cuda.current_stream().cuda_stream)
        assert rc == -2 and bool((out == 5.0).all())


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
