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
(twice the expectation of what does not come from the last rounding).  Where groups of the slots that 128 rows see lie more than 2^20 apart, the
operands are bf16: e = 2^-8."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4, _lib
from test_kv4_gpu import copy_slots, filled, randn

pytestmark = pytest.mark.gpu

FP16, BF16 = 2.0 ** -11, 2.0 ** -8


def attend_prompt(c, q, pos, **kw):
    assert R.form(c, *q.shape[:2], q.shape[2] // c.head_dim, kw.get("window", 0), kw.get("sinks", 0)) == _lib.KV4_PROMPT
    return c.attend(q, pos, **kw)


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


# ----------------------------------------------------------------------------- large scores
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_gain,k_gain,scale", [(1e3, 1e3, None), (3e4, 1e4, None), (1e8, 1e6, None), (1e18, 1e18, -0.1), (1.0, 1.0, 1e30)])
def test_large_scores(D, q_gain, k_gain, scale):
    """Scores so far apart that one slot has all the weight: its value, where no other score comes near it (nearer than operands' roundings tell apart:
    2 * 9 e |q k| and 2^-8 of the scores, which is more than fp32 takes), and finite everywhere."""
    (T, heads, n_kv), slots = size(D), 450
    c = KVCache4(1, n_kv, slots, D)
    c.append(randn(1, 1, slots, n_kv * D, gain=k_gain), randn(2, 1, slots, n_kv * D), torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 1, T, heads * D, gain=q_gain)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    scale = D ** -0.5 if scale is None else scale
    got = attend_prompt(c, q, pos, scale=scale)
    assert bool(torch.isfinite(got.float()).all())
    see, clear = R.visible(pos, slots, 0, 0)[0], 0
    for h in range(heads):
        s = (q.view(T, heads, D)[:, h].double() @ kd[0, h // 4, :slots].T * scale).masked_fill(~see, float("-inf"))
        (first, second), j = s.topk(2, 1)[0].T, s.argmax(1)
        qk = (q.view(T, heads, D)[:, h].double().square() @ kd[0, h // 4, :slots].square().T).sqrt().amax(1) * abs(scale)
        sure = first - second > 2 * 9 * FP16 * qk + 2.0 ** -8 * s.masked_fill(~see, 0.0).abs().amax(1) + 30
        want = vd[0, h // 4, :slots][j]
        off = (got.view(T, heads, D)[:, h].double() - want).abs()
        tol = 2.0 ** -8 * want.abs() + 2 * FP16 * want.abs() + 2.0 ** -14 * vd.abs().amax()
        assert bool((off <= tol)[sure].all())
        clear += int(sure.sum())
    assert clear > T * heads // 2


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


@pytest.mark.parametrize("D", [64, 128])
def test_positions_in_any_order(D):
    """Tokens of a prompt need not follow one another: padding among them, repeated and shuffled positions, some behind the cache."""
    (T, heads, n_kv), slots = size(D), 500
    c, k, v = filled(2, n_kv, slots, D)
    q = randn(8, 2, T, heads * D)
    pos = torch.randint(-60, slots, (2, T), generator=torch.Generator().manual_seed(D)).cuda()
    pos[1, :128] = -1                                                                  # whole CTAs without a slot
    pos[0, 7], pos[0, 8], pos[0, 9] = slots + 30, 1 << 40, -(1 << 63)
    for window, sinks in ((0, 0), (90, 0), (90, 7)):
        out = torch.full((3, T, heads * D), 5.0, dtype=torch.bfloat16, device="cuda")
        got = attend_prompt(c, q, pos, window=window, sinks=sinks, out=out[:2])
        assert_near(got, q, k, v, pos, slots, heads, D ** -0.5, window, sinks)
        assert not bool(got[pos < 0].any()) and bool((out[2] == 5.0).all())
        assert window == 0 or sinks or not bool(got[0, 8].any())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.5])
def test_scales_of_any_sign(D, scale):
    (T, heads, n_kv), slots = size(D), 500
    c, k, v = filled(1, n_kv, slots, D)
    q = randn(1, 1, T, heads * D)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    assert_near(attend_prompt(c, q, pos, window=200, sinks=2, scale=scale), q, k, v, pos, slots, heads, scale, 200, 2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("k_gain,v_gain,q_gain", [(1e-6, 1e-5, 1.0), (1e4, 1e6, 1e-4), (1e-20, 1e30, 1e20), (1e33, 1e33, 1e-33)])
def test_ranges_of_keys_values_and_queries(D, k_gain, v_gain, q_gain):
    """bf16 inputs of any size whose scores are ordinary; value scales that differ from slot to slot by up to 2^16."""
    (T, heads, n_kv), slots = size(D), 450
    c = KVCache4(1, n_kv, slots, D)
    apart = torch.exp2(torch.randint(-8, 9, (1, slots, 1), generator=torch.Generator().manual_seed(1)).float()).cuda()
    c.append(randn(1, 1, slots, n_kv * D, gain=k_gain), (randn(2, 1, slots, n_kv * D).float() * v_gain * apart).bfloat16(), torch.arange(slots, device="cuda"))
    q = randn(3, 1, T, heads * D, gain=q_gain)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    assert_near(attend_prompt(c, q, pos), q, *R.cache_values(c.tiles, D), pos, slots, heads, D ** -0.5)


# ----------------------------------------------------------------------------- what is hidden, what is no number
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("byte", [0xFF, 0x7F, 0x00])
def test_what_is_hidden_is_not_seen(D, byte):
    """Slots that no token sees hold other bytes (which read as NaN, as huge values, as zeros): the same bits."""
    (T, heads, n_kv), slots = size(D), 700
    c, _, _ = filled(2, n_kv, slots, D)
    pos = torch.stack([torch.arange(p - T + 1, p + 1) for p in (520, 660)]).cuda()
    q = randn(3, 2, T, heads * D)
    want = attend_prompt(c, q, pos, window=90, sinks=3)
    other = KVCache4(2, n_kv, slots, D)
    other.tiles.fill_(byte)
    see = R.visible(pos, slots, 90, 3).any(1)
    for b in range(2):
        copy_slots(c.tiles[b:b + 1], other.tiles[b:b + 1], see[b].nonzero().flatten().tolist(), D)
    assert torch.equal(attend_prompt(other, q, pos, window=90, sinks=3), want)


@pytest.mark.parametrize("D", [64, 128])
def test_groups_that_are_not_finite_reach_who_sees_them(D):
    """A value group that is no number: NaN in its channels for the rows that see its slot; a key: the whole row; a query: its own row.  The slot
    lies inside the rows and key tiles of one CTA, before and behind whole ones."""
    (T, heads, n_kv), slots, bad, rep = size(D), 450, 230, 4
    g = D // 64 - 1                                                                   # the last group of KV head 1
    k, v = randn(1, 1, slots, n_kv * D), randn(2, 1, slots, n_kv * D)
    kbad, vbad = k.clone(), v.clone()
    kbad[0, bad, D + 1], vbad[0, bad, D + 64 * g + 5] = float("nan"), float("inf")
    q = randn(3, 1, T, heads * D)
    pos = (10 + torch.arange(T, device="cuda"))[None]
    for keys, values in ((k, vbad), (kbad, v)):
        c = KVCache4(1, n_kv, slots, D)
        c.append(keys, values, torch.arange(slots, device="cuda"))
        kd, vd = R.cache_values(c.tiles, D)
        for window, sinks in ((0, 0), (9, 0), (9, 300)):
            got = attend_prompt(c, q, pos, window=window, sinks=sinks)
            nan = torch.isnan(got.float()).view(T, heads, D)
            see = R.visible(pos, slots, window, sinks)[0, :, bad]
            want = torch.zeros(T, heads, D, dtype=torch.bool, device="cuda")
            if values is vbad:
                want[:, rep:2 * rep, 64 * g:64 * g + 64] = see[:, None, None]
            else:
                want[:, rep:2 * rep] = see[:, None, None]
            assert torch.equal(nan, want)
            assert_near(got, q, kd, vd, pos, slots, heads, D ** -0.5, window, sinks, rows=~see[None])
    c = KVCache4(1, n_kv, slots, D)
    c.append(k, v, torch.arange(slots, device="cuda"))
    q[0, 37, 5], q[0, 300, 3 * D] = float("inf"), float("nan")
    nan = torch.isnan(attend_prompt(c, q, pos).float()).view(T, heads, D)
    assert bool(nan[37, 0].all()) and bool(nan[300, 3].all()) and int(nan.sum()) == 2 * D


# ----------------------------------------------------------------------------- memory
@pytest.mark.parametrize("D", [64, 128])
def test_the_result_may_take_the_place_of_the_queries(D):
    (T, heads, n_kv), slots = size(D), 450
    c, _, _ = filled(1, n_kv, slots, D)
    q = randn(1, 1, T, heads * D)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    want = attend_prompt(c, q, pos)
    assert attend_prompt(c, q, pos, out=q) is q and torch.equal(q, want)
    fused = randn(2, 1, T, heads * D + 24)                                             # rows with a stride of their own
    assert torch.equal(attend_prompt(c, fused[..., 8:-16], pos), c.attend(fused[..., 8:-16].contiguous(), pos))


@pytest.mark.parametrize("D", [64, 128])
def test_captured_and_replayed_with_other_positions(D):
    (T, heads, n_kv), slots = size(D), 900
    c, other = KVCache4(2, n_kv, slots, D), KVCache4(2, n_kv, slots, D)
    fill = randn(1, 2, slots, n_kv * D), randn(2, 2, slots, n_kv * D)
    for x in (c, other):
        x.append(*fill, torch.arange(slots, device="cuda"))
    inv = 1.0 / (1e4 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    q, k, v = randn(3, 2, T, heads * D), randn(4, 2, T, n_kv * D), randn(5, 2, T, n_kv * D)
    pos = torch.stack([torch.arange(T), 200 + torch.arange(T)]).cuda()

    def once(cache):
        return cache.attend(cache.append(k, v, pos, q=q, inv_freq=inv), pos, window=200, sinks=4)

    assert R.form(c, 2, T, heads, 200, 4) == _lib.KV4_PROMPT
    once(c)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once(c))
        graphs.append(g)
    once(other)
    for step in range(4):
        pos += 60
        q.copy_(randn(10 + step, *q.shape)); k.copy_(randn(20 + step, *k.shape)); v.copy_(randn(30 + step, *v.shape))
        graphs[step % 2].replay()
        got = outs[step % 2].clone()
        assert torch.equal(got, once(other)) and torch.equal(c.tiles, other.tiles)


@pytest.mark.parametrize("T,D,slots", [(256, 128, 30_000_000), (384, 64, 60_000_000)])
def test_slots_beyond_4_gb_of_one_head(T, D, slots):
    """The last slots of a head whose tiles take more than 2^32 bytes, against the same slots at the beginning of a small cache."""
    heads, used = 64, 500
    far, near = KVCache4(1, 1, slots, D), KVCache4(1, 1, used, D)
    assert far.nbytes() > 1 << 32
    q, k, v = randn(1, 1, T, heads * D), randn(2, 1, used, D), randn(3, 1, used, D)
    at = torch.arange(used, device="cuda")[None]
    first = (slots - used) // 128 * 128
    near.append(k, v, at)
    far.append(k, v, at + first)
    pos = (used - T + torch.arange(T, device="cuda"))[None]
    want = attend_prompt(near, q, pos, window=90)
    assert_near(want, q, *R.cache_values(near.tiles, D), pos, used, heads, D ** -0.5, 90)
    assert torch.equal(attend_prompt(far, q, pos + first, window=90), want)


def test_prompts_of_a_decoder():
    """The prompt of a decoder with a 4-bit cache goes through this kernel, and every layer's attention is that of 64 bits."""
    from cobalt_b200 import SparseQuantConfig
    from cobalt_b200.decoder import CobaltDecoder, build_random_decoder
    from oracle import model_oracle as MO
    cfg = MO.llama_config(hidden=512, layers=2, heads=32, kv_heads=8, head_dim=128, inter=1024, vocab=1008)
    dec = build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), 400, torch.device("cuda"), batch=2, kv_bits=4)
    checked = []

    class Checked(CobaltDecoder):
        def _attend4(self, q, positions, layer, seq, n):
            got = super()._attend4(q, positions, layer, seq, n)
            c, T = self.kv4[layer], q.shape[0] // n
            k, v = R.cache_values(c.tiles[seq:seq + n], c.head_dim)
            assert_near(got.view(n, T, -1), q.view(n, T, -1), k, v, positions.expand(n, T), c.slots, self.nh, self.scale)
            checked.append(layer)
            return got

    chk = Checked(cfg, dec.lin, dec.P, 400, dec.dev, batch=2, kv_bits=4)
    ids = torch.randint(0, 1000, (2, 330), generator=torch.Generator().manual_seed(1))
    assert R.form(dec.kv4[0], 2, 330, 32) == _lib.KV4_PROMPT                          # both prompts together
    assert torch.equal(chk.prefill(ids), dec.prefill(ids)) and checked == [0, 1]


# ----------------------------------------------------------------------------- magnitudes far apart
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["key", "value", "value in the last group", "both"])
@pytest.mark.parametrize("size_of", [1e8, 1e13, 1e30])
def test_a_huge_slot_does_not_reach_rows_that_do_not_see_it(D, what, size_of):
    """A finite key or value far above all others, in the slot of a token in the middle of a CTA's rows: the rows before it, and (window) those
    that have left it behind, are what they are without it, to within the operands' rounding."""
    (T, heads, n_kv), slots = size(D), 450
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    at = int(pos[0, T // 2 + 9])
    k, v = randn(1, 1, slots, n_kv * D), randn(2, 1, slots, n_kv * D)
    channels = torch.arange(n_kv, device="cuda") * D + (D - 1 if "last" in what else 3)
    if what in ("key", "both"):
        k[0, at, channels] = size_of
    if what != "key":
        v[0, at, channels] = -size_of
    c = KVCache4(1, n_kv, slots, D)
    c.append(k, v, torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 1, T, heads * D)
    for window, sinks in ((0, 0), (20, 0), (20, 2)):
        got = attend_prompt(c, q, pos, window=window, sinks=sinks)
        see = R.visible(pos, slots, window, sinks)[0, :, at]
        assert bool(torch.isfinite(got.float()).all())
        assert_near(got, q, kd, vd, pos, slots, heads, D ** -0.5, window, sinks, e=BF16, rows=~see[None])
        if what in ("value", "value in the last group"):
            assert_near(got, q, kd, vd, pos, slots, heads, D ** -0.5, window, sinks, e=BF16, rows=see[None])


@pytest.mark.parametrize("D", [64, 128])
def test_magnitudes_that_fall_and_rise_by_many_powers_of_two(D):
    """Keys and values of 2^-60 to 2^60 from slot to slot, queries to match: every row against what it sees itself."""
    (T, heads, n_kv), slots = size(D), 450
    at = torch.arange(slots, device="cuda")
    c = KVCache4(1, n_kv, slots, D)
    rise = torch.exp2(60 * torch.sin(at.float() / 40))[None, :, None]
    c.append(randn(1, 1, slots, n_kv * D, gain=2.0 ** -8), (randn(2, 1, slots, n_kv * D).float() * rise).bfloat16(), at)
    q = randn(3, 1, T, heads * D)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    for window, sinks in ((0, 0), (9, 0), (1, 0)):
        got = attend_prompt(c, q, pos, window=window, sinks=sinks)
        assert_near(got, q, *R.cache_values(c.tiles, D), pos, slots, heads, D ** -0.5, window, sinks, e=BF16)


@pytest.mark.parametrize("D", [64, 128])
def test_a_constant_group_near_the_end_of_fp32(D):
    """256 s is such a group's value, 271 s would be beyond fp32; the rows before it do not see it, those behind have it in its channels only."""
    (T, heads, n_kv), slots = size(D), 450
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    at = int(pos[0, T // 2 + 9])
    k, v = randn(1, 1, slots, n_kv * D), randn(2, 1, slots, n_kv * D)
    v[0, at, :64] = -3.3e38
    c = KVCache4(1, n_kv, slots, D)
    c.append(k, v, torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 1, T, heads * D)
    got = attend_prompt(c, q, pos)
    see = R.visible(pos, slots, 0, 0)[0, :, at]
    assert bool(torch.isfinite(got.float()).all())
    for rows in (see, ~see):
        assert_near(got, q, kd, vd, pos, slots, heads, D ** -0.5, e=BF16, rows=rows[None])
