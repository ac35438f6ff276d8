"""4-bit KV cache on the GPU: writing, reading back and attention against plain torch in 64 bits (needs a B200).

Writing and reading are compared bit for bit with fp32 operations on the CPU.  Attention: the result is one rounding to bf16 (2^-8 of the
value) of sums whose weights may be rounded to 16-bit floats on the way (2^-11 each, so at most 2^-11 of the largest visible value), with
everything else in fp32 (below that again): |got - want| <= 2^-8 |want| + 2^-10 max|v|.

Prompts (64 rows per KV head and more, heads of 64 and 128) have fp16 operands: probabilities, values and keys are rounded, 2^-11 relative at
most each.  The first two add up to 2 * 2^-11 sum p|v|.  A score moves by d = scale * sum q k e with |e| <= 2^-11 independent roundings: by
more than 7 * 2^-11 * scale * |q k| (2-norm of the products) with a probability below 2 exp(-49/2) (Hoeffding) each, and the context by
2 d sum p|v| at most.  Values far below the largest visible one are held to 2^-25 of it, as probabilities are (2^-24, times 2^6): 2^-22 max|v|.
So |got - want| <= 2^-8 |want| + (2 * 2^-11 + 2 d) sum p|v| + 2^-22 max|v|."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import KVCache4, _lib

pytestmark = pytest.mark.gpu


def randn(seed, *shape, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * gain).bfloat16()


def filled(n_seq, n_kv, slots, D, seed=0, gain=1.0):
    """A cache whose every slot was written, and its fp64 keys and values."""
    c = KVCache4(n_seq, n_kv, slots, D)
    c.append(randn(seed, n_seq, slots, n_kv * D, gain=gain), randn(seed + 1, n_seq, slots, n_kv * D), torch.arange(slots, device="cuda"))
    return (c, *R.cache_values(c.tiles, D))


def assert_near(got, ref, cache, heads):
    want, top, (pv, qk) = ref
    off = (got.double() - want).abs()
    rep = heads // cache.n_kv_heads
    if cache.head_dim in (64, 128) and rep <= 128 and rep * got.shape[1] >= 64:
        # (such calls go to either kernel, whichever is expected to be faster)
        tol = 2.0 ** -8 * want.abs() + torch.maximum((2 * 2.0 ** -11 + 2 * 7 * 2.0 ** -11 * qk) * pv + 2.0 ** -22 * top, 2.0 ** -10 * top)
    else:
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -10 * top
    far = off - tol
    assert bool((far <= 0).all()), (float(far.max()), float(tol.max()))


# ----------------------------------------------------------------------------- writing
def expected_tiles(k, v, positions, slots, n_kv, D):
    """{(seq, head, slot): parts} comparison: returns codes, scale, zero of keys and values [n, T, n_kv, ...] on the CPU."""
    n, T = k.shape[:2]
    return R.quantise(k.view(n, T, n_kv, D).cpu()), R.quantise(v.view(n, T, n_kv, D).cpu())


def stored_parts(c, positions):
    """The same, read from the cache's bytes."""
    n, T = positions.shape
    out = []
    for codes, s, z in R.tile_parts(c.tiles.cpu(), c.head_dim):
        flat = [x.reshape(c.n_seq, c.n_kv_heads, -1, x.shape[-1]) for x in (codes, s, z)]
        out.append([torch.stack([x[b][:, positions[b]].transpose(0, 1) for b in range(n)]) for x in flat])
    return out


def same(a, b):
    return torch.equal(a, b) if not a.is_floating_point() else torch.equal(torch.nan_to_num(a.double(), 7e9), torch.nan_to_num(b.double(), 7e9))


@pytest.mark.parametrize("n,T,n_kv,D,slots,start", [(1, 1, 1, 64, 1, 0), (1, 1, 8, 128, 2048, 1000), (3, 5, 2, 128, 40, 30), (2, 70, 3, 192, 100, 7),
                                                    (1, 33, 1, 256, 64, 31), (16, 1, 4, 64, 33, 32), (1, 300, 16, 128, 301, 1)])
def test_written_codes_are_those_of_the_format(n, T, n_kv, D, slots, start):
    k, v = randn(T, n, T, n_kv * D), randn(T + 1, n, T, n_kv * D, gain=30.0)
    pos = (start + torch.arange(T, device="cuda")).expand(n, T).contiguous()
    c = KVCache4(n, n_kv, slots, D)
    c.tiles.fill_(0xA5)
    before = c.tiles.clone()
    assert c.append(k, v, pos) is None
    kept = pos.cpu().clamp(max=slots - 1)
    for want, got in zip(expected_tiles(k, v, pos, slots, n_kv, D), stored_parts(c, kept)):
        for w, g in zip(want, got):
            inside = (pos < slots).cpu()
            assert same(w.to(g.dtype)[inside], g[inside])
    rest = torch.ones(c.tiles.shape[2] * 32, dtype=torch.bool)                       # every other slot as it was
    rest[start:start + T] = False
    for a, b in zip(R.tile_parts(before.cpu(), D), R.tile_parts(c.tiles.cpu(), D)):
        for x, y in zip(a, b):
            assert same(x.reshape(n, n_kv, -1, x.shape[-1])[:, :, rest], y.reshape(n, n_kv, -1, y.shape[-1])[:, :, rest])


def test_awkward_groups():
    """Constant, zero, tiny, huge and one-step groups, and groups with values that are not finite."""
    rows = [torch.full((64,), 3.140625), torch.zeros(64), torch.full((64,), -1e-39), torch.randn(64) * 1e-38, torch.randn(64) * 1e37,
            torch.linspace(-3e38, 3e38, 64), torch.tensor([1.0] * 63 + [1.0078125]), torch.tensor([0.0] * 63 + [1e-40]), torch.tensor([-0.0] * 32 + [0.0] * 32),
            torch.tensor([float("nan")] + [1.0] * 63), torch.tensor([1.0] * 63 + [float("inf")]), torch.tensor([float("-inf")] * 64),
            torch.tensor([float("nan")] * 64), torch.tensor([float("inf"), float("-inf")] * 32)]
    x = torch.stack(rows).bfloat16().cuda().unsqueeze(0)
    T = x.shape[1]
    c = KVCache4(1, 1, T, 64)
    pos = torch.arange(T, device="cuda").unsqueeze(0)
    c.append(x, x, pos)
    for want, got in zip(expected_tiles(x, x, pos, T, 1, 64), stored_parts(c, pos.cpu())):
        for w, g in zip(want, got):
            assert same(w.to(g.dtype), g)
    k, v = c.read(pos)
    assert same(k, v) and torch.equal(k[0, 0, 0].float().cpu(), rows[0]) and not bool(k[0, 1].any())
    assert bool(torch.isnan(k[0, [5, 9, 10, 11, 12, 13]].float()).all()) and bool(torch.isfinite(k[0, :5].float()).all())


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_and_norm(D, norm):
    """Rotated as the bf16 cache rotates; a value may differ by a rounding where cosine, sine or the mean do in their last bit: one bf16
    step (2^-7 of the larger of the pair), for a few of them."""
    n, T, heads, n_kv = 2, 9, 6, 3
    q, k, v = randn(1, n, T, heads * D), randn(2, n, T, n_kv * D), randn(3, n, T, n_kv * D)
    w = randn(4, 2, D, gain=0.1)
    pos = torch.stack([torch.arange(T) * 37, 4000 + torch.arange(T)]).cuda()
    inv = 1.0 / (1e4 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    c = KVCache4(n, n_kv, 5000, D)
    before = q.clone()
    got = c.append(k, v, pos, q=q, inv_freq=inv, q_norm=w[0].contiguous() if norm else None, k_norm=w[1].contiguous() if norm else None, eps=1e-6)
    assert torch.equal(q, before)
    qc, kc = q.view(n, T, heads, D).cpu(), k.view(n, T, n_kv, D).cpu()
    if norm:
        qc, kc = R.head_norm(qc, w[0].cpu(), 1e-6), R.head_norm(kc, w[1].cpu(), 1e-6)
    want = R.rotate(qc, pos.cpu(), inv.cpu()).reshape(n, T, -1)
    step = 2.0 ** -7 * torch.cat([qc, qc.roll(D // 2, -1)], -1).view(n, T, heads, 2, D).abs().amax(3).reshape(n, T, -1).float() * (2.0 if norm else 1.0)
    off = (got.cpu().float() - want.float()).abs()
    assert bool((off <= step).all()) and float((off > 0).float().mean()) < 0.02
    # in place: the same; and the stored keys are the quantised rotated keys
    alias = q.clone()
    c2 = KVCache4(n, n_kv, 5000, D)
    assert c2.append(k, v, pos, q=alias, inv_freq=inv, q_norm=w[0].contiguous() if norm else None, k_norm=w[1].contiguous() if norm else None, eps=1e-6,
                     q_out=alias) is alias
    assert torch.equal(alias, got) and torch.equal(c.tiles, c2.tiles)
    kq = c.append(k, v, pos, q=k.clone(), inv_freq=inv, q_norm=w[1].contiguous() if norm else None, k_norm=w[1].contiguous() if norm else None, eps=1e-6)
    kr, vr = c.read(pos)
    assert same(kr.cpu(), R.values(*R.quantise(kq.view(n, T, n_kv, D).cpu())).float().bfloat16())
    assert same(vr.cpu(), R.values(*R.quantise(v.view(n, T, n_kv, D).cpu())).float().bfloat16())


def test_keys_match_the_bf16_cache():
    """The rotated keys are those that ``cobalt_rope_kv`` writes, bit for bit (no norm: no sum whose order could differ)."""
    T, heads, n_kv, D = 40, 8, 2, 128
    q, k, v = randn(1, T, heads * D), randn(2, T, n_kv * D), randn(3, T, n_kv * D)
    pos = torch.arange(500, 500 + T, device="cuda")
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    kc, vc = torch.zeros(n_kv, 600, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(n_kv, 600, D, dtype=torch.bfloat16, device="cuda")
    qr = q.clone()
    rc = _lib.load().cobalt_rope_kv(qr.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), inv.data_ptr(), kc.data_ptr(), vc.data_ptr(), T, heads, n_kv, D,
                                    600, None, None, 1e-6, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    c = KVCache4(1, n_kv, 600, D)
    assert torch.equal(c.append(k, v, pos, q=q, inv_freq=inv), qr)
    got = stored_parts(c, pos.cpu()[None])
    for want, g in zip((R.quantise(kc[:, 500:540].transpose(0, 1).cpu()), R.quantise(vc[:, 500:540].transpose(0, 1).cpu())), got):
        for w, x in zip(want, g):
            assert same(w.to(x.dtype), x[0])


def test_positions_outside_are_not_stored_and_read_as_zeros():
    c, k, v = filled(2, 2, 50, 64)
    before = c.tiles.clone()
    pos = torch.tensor([[-1, 50, 1 << 40], [-(1 << 62), 63, 51]], device="cuda")
    c.append(randn(5, 2, 3, 128), randn(6, 2, 3, 128), pos)
    assert torch.equal(c.tiles, before)
    a, b = c.read(pos)
    assert not bool(a.any()) and not bool(b.any())


def test_strided_rows_and_one_shared_row_of_positions():
    """q, k and v as slices of one fused projection; positions [T] for every sequence; sequences from the middle of a cache."""
    n, T, heads, n_kv, D = 2, 6, 4, 2, 64
    fused = randn(9, n, T, (heads + 2 * n_kv) * D + 6)
    q, k, v = fused[..., :heads * D], fused[..., heads * D:(heads + n_kv) * D], fused[..., (heads + n_kv) * D + 2:(heads + 2 * n_kv) * D + 2]
    pos = torch.arange(3, 3 + T, device="cuda")
    a, b = KVCache4(4, n_kv, 40, D), KVCache4(4, n_kv, 40, D)
    inv = torch.ones(D // 2, device="cuda")
    qa = a.append(k, v, pos, q=q, inv_freq=inv, seq=1)
    qb = b.append(k.contiguous(), v.contiguous(), pos.expand(n, T).contiguous(), q=q.contiguous(), inv_freq=inv, seq=1)
    assert torch.equal(a.tiles, b.tiles) and torch.equal(qa, qb) and not bool(a.tiles[[0, 3]].any())
    assert torch.equal(a.attend(fused[..., :heads * D], pos, seq=1), b.attend(q.contiguous(), pos.expand(n, T).contiguous(), seq=1))
    odd = torch.empty(n * T * heads * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(n, T, heads * D)
    odd.copy_(q)
    assert torch.equal(a.attend(odd, pos, seq=1), a.attend(q, pos, seq=1))            # a row off its 4-byte boundary is copied
    r = a.read(pos, seq=1, n=2)
    assert r[0].shape == (n, T, n_kv, D) and all(torch.equal(x, y) for x, y in zip(r, a.read(pos.expand(n, T), seq=1)))


# ----------------------------------------------------------------------------- attention
CASES = [  # n, T, heads, n_kv, D, slots, positions of the last token per sequence, window, sinks, gain
    (1, 1, 1, 1, 64, 1, [0], 0, 0, 1.0),                       # one slot
    (1, 1, 8, 2, 128, 40, [31], 0, 0, 1.0),                    # a tile to its last slot, one more, one less
    (1, 1, 8, 2, 128, 40, [32], 0, 0, 1.0),
    (1, 1, 8, 2, 128, 40, [30], 0, 0, 1.0),
    (1, 1, 32, 8, 128, 2048, [1000], 0, 0, 1.0),
    (3, 1, 7, 1, 128, 1500, [0, 1499, 700], 0, 0, 1.0),        # lengths apart, seven heads to one
    (4, 1, 16, 16, 64, 700, [5, 699, 64, 300], 0, 0, 1.0),     # no sharing
    (2, 1, 24, 2, 128, 900, [899, 10], 0, 0, 1.0),             # twelve heads to one
    (2, 1, 40, 1, 64, 333, [332, 200], 0, 0, 1.0),
    (2, 1, 12, 4, 192, 515, [514, 31], 0, 0, 1.0),
    (2, 1, 8, 1, 256, 1000, [999, 513], 0, 0, 1.0),
    (2, 3, 8, 2, 256, 300, [299, 100], 33, 2, 1.0),
    (1, 1, 8, 2, 128, 4000, [3999], 100, 0, 1.0),              # a window that begins and ends inside tiles
    (2, 1, 8, 2, 128, 4000, [3999, 50], 100, 4, 1.0),          # first slots; a window longer than the sequence
    (1, 1, 4, 4, 64, 4000, [3990], 1, 0, 1.0),                 # a window of one
    (1, 1, 4, 4, 64, 4000, [3990], 1, 1, 1.0),
    (1, 1, 4, 2, 128, 600, [599], 64, 1000, 1.0),              # more first slots than the cache has
    (1, 1, 4, 2, 128, 600, [599], 64, 530, 1.0),               # first slots that reach into the window
    (1, 1, 4, 2, 128, 600, [599], 1 << 30, 0, 1.0),
    (2, 5, 16, 4, 64, 900, [899, 4], 0, 0, 1.0),               # several new tokens
    (2, 17, 8, 2, 128, 300, [299, 16], 20, 3, 1.0),
    (1, 3, 3, 3, 192, 77, [76], 0, 0, 1.0),
    (1, 1, 8, 2, 128, 3000, [2999], 0, 0, 12.0),               # scores far apart
    (1, 2, 8, 2, 64, 3000, [2999], 500, 4, 12.0),
    (1, 150, 8, 2, 128, 700, [699], 0, 0, 1.0),                # prompts
    (1, 129, 1, 1, 64, 129, [128], 0, 0, 1.0),
    (3, 100, 6, 2, 128, 350, [99, 349, 200], 0, 0, 1.0),
    (2, 77, 16, 1, 64, 500, [499, 300], 60, 5, 1.0),
    (1, 300, 5, 1, 128, 300, [299], 100, 0, 4.0),
    (1, 64, 4, 2, 256, 200, [199], 0, 0, 1.0),
    (1, 200, 4, 4, 192, 200, [199], 50, 1, 1.0),
    (1, 40, 130, 1, 64, 60, [59], 0, 0, 1.0),                  # more heads to one than a tile has rows
    (1, 64, 1, 1, 128, 64, [63], 0, 0, 1.0),                   # the smallest prompt
    (2, 257, 8, 8, 64, 1000, [999, 256], 0, 0, 1.0),
    (1, 500, 12, 4, 128, 1500, [1400], 300, 5, 1.0),           # a window that leaves a gap behind the first slots
    (2, 130, 7, 1, 128, 600, [599, 400], 128, 130, 1.0),       # heads that do not divide 128 rows
    (1, 90, 128, 1, 64, 100, [99], 0, 0, 1.0),                 # a row per head: one token a CTA
    (1, 400, 4, 4, 128, 3000, [2999], 0, 0, 12.0),
    (3, 1, 8, 2, 64, 40000, [39999, 5, 20001], 0, 0, 1.0),     # few and long heads: their tiles in equal ranges
    (2, 1, 4, 1, 128, 30000, [29999, 28000], 27001, 40, 4.0),
    (5, 2, 12, 1, 64, 24000, [23999, 1, 12000, 31, 32], 0, 0, 1.0),
    (3, 1, 3, 1, 192, 20000, [19999, 19000, 100], 0, 0, 1.0),
    (2, 1, 2, 1, 256, 20000, [17777, 19999], 0, 0, 1.0),
    (4, 3, 5, 1, 128, 21000, [20999, 20000, 2, 640], 20500, 3, 1.0),
    (100, 1, 16, 16, 64, 100, list(range(100)), 0, 0, 1.0),    # heads enough for several CTAs per SM
    (300, 1, 2, 1, 64, 260, [(7 * i) % 260 for i in range(300)], 0, 0, 1.0),   # more sequences than a list takes
]


@pytest.mark.parametrize("n,T,heads,n_kv,D,slots,last,window,sinks,gain", CASES)
def test_attention_matches_fp64(n, T, heads, n_kv, D, slots, last, window, sinks, gain):
    c, k, v = filled(n, n_kv, slots, D, seed=slots)
    q = randn(T + 1, n, T, heads * D, gain=gain)
    pos = torch.stack([torch.arange(p - T + 1, p + 1) for p in last]).cuda()
    assert int(pos.min()) >= 0
    got = c.attend(q, pos, window=window, sinks=sinks)
    assert_near(got, R.attend(q, k, v, pos, slots, heads, D ** -0.5, window, sinks), c, heads)
    assert torch.equal(got, c.attend(q, pos, window=window, sinks=sinks)) and c.device_status() == 0


# at most eight heads, long enough for the widest clusters: even and ragged lengths, sequences that leave most CTAs of a cluster without
# a key, a window with first slots, every width, several columns a tile
@pytest.mark.parametrize("n,T,heads,n_kv,D,slots,last,window,sinks,gain", [
    (1, 1, 32, 8, 128, 9000, [8999], 0, 0, 1.0),
    (4, 1, 8, 1, 256, 9001, [9000, 0, 31, 4500], 0, 0, 1.0),
    (2, 3, 14, 2, 64, 6000, [5999, 2], 0, 0, 4.0),
    (2, 1, 3, 3, 192, 6017, [6016, 100], 0, 0, 1.0),
    (1, 2, 8, 4, 128, 12000, [11999], 9000, 5, 1.0),
    (8, 1, 8, 1, 128, 16000, [15999, 1, 64, 8000, 15000, 0, 12345, 33], 0, 0, 1.0),
])
def test_few_long_heads_match_fp64(n, T, heads, n_kv, D, slots, last, window, sinks, gain):
    test_attention_matches_fp64(n, T, heads, n_kv, D, slots, last, window, sinks, gain)


@pytest.mark.parametrize("T", [1, 4, 80])
def test_what_is_hidden_is_not_seen(T):
    """Slots behind a token, before its window, or left by an earlier sequence (here: bytes that read as NaN and infinities) do not reach it."""
    n, heads, n_kv, D, slots = 2, 8, 2, 128, 400
    c, k, v = filled(n, n_kv, slots, D)
    last = [233, 330]
    pos = torch.stack([torch.arange(p - T + 1, p + 1) for p in last]).cuda()
    q = randn(3, n, T, heads * D)
    want = c.attend(q, pos, window=90, sinks=3)
    parts = c.tiles.view(n, n_kv, -1, 36 * D)
    poison = KVCache4(n, n_kv, slots, D)
    poison.tiles.fill_(0xFF)                                                         # scales and zeros are NaN
    spoilt = poison.tiles
    see = R.visible(pos, c.tiles.shape[2] * 32, 90, 3).any(1)                         # [n, slots of all tiles]
    for b in range(n):                                                               # write the visible slots into the spoilt cache
        at = see[b].nonzero().flatten()
        seen = KVCache4.wrap(spoilt[b:b + 1], D, slots)
        src = KVCache4.wrap(parts[b:b + 1], D, slots)
        kk, vv = src.read(at)
        # reading back and writing again may round codes differently: copy the bytes of whole slots instead
        copy_slots(src.tiles, seen.tiles, at.tolist(), D)
    got = poison.attend(q, pos, window=90, sinks=3)
    assert torch.equal(got, want)


def copy_slots(src, dst, slots, D):
    """The bytes of single slots, from the format's description."""
    G = D // 64
    s, d = src.view(src.shape[0], src.shape[1], -1, 36 * D), dst.view(dst.shape[0], dst.shape[1], -1, 36 * D)
    for j in slots:
        t, i = divmod(j, 32)
        at = []
        for g in range(G):
            at += list(range(g * 1024 + i * 32, g * 1024 + i * 32 + 32))
            p = i // 2
            for ch in range(8):
                a = 16 * D + g * 1024 + p * 64 + (ch ^ ((p & 2) << 1)) * 8 + (i % 2) * 4
                at += list(range(a, a + 4))
            a = 32 * D + (i * G + g) * 4
            at += list(range(a, a + 4))
            a = 34 * D + (i * G + g) * 2
            at += [a, a + 1]
            a = 35 * D + (g * 32 + i) * 2
            at += [a, a + 1]
        idx = torch.tensor(at, device=src.device)
        d[:, :, t, idx] = s[:, :, t, idx]


@pytest.mark.parametrize("T,D", [(1, 128), (3, 64), (90, 128), (40, 256)])
def test_padding_rows_are_zero_and_others_unmoved(T, D):
    """Tokens at negative positions see nothing; positions behind the cache see what there is, or nothing outside their window."""
    n, heads, n_kv, slots = 3, 4, 2, 100
    c, k, v = filled(n, n_kv, slots, D)
    q = randn(8, n, T, heads * D)
    pos = torch.full((n, T), -1, device="cuda")
    pos[1] = torch.arange(T, device="cuda") % slots
    pos[2, -1] = 120
    got = c.attend(q, pos)
    assert not bool(got[0].any()) and not bool(got[2, :-1].any())
    assert_near(got, R.attend(q, k, v, pos, slots, heads, D ** -0.5), c, heads)
    pos[2] = 1 << 40
    got = c.attend(q, pos, window=50)
    assert not bool(got[2].any())
    assert_near(got, R.attend(q, k, v, pos, slots, heads, D ** -0.5, 50), c, heads)
    got = c.attend(q, pos, window=50, sinks=7)
    assert_near(got, R.attend(q, k, v, pos, slots, heads, D ** -0.5, 50, 7), c, heads)
    out = torch.full((n + 1, T, heads * D), 5.0, dtype=torch.bfloat16, device="cuda")
    c.attend(q, pos, out=out[:n])
    assert bool((out[n] == 5.0).all())                                               # rows behind the last sequence


@pytest.mark.parametrize("T", [1, 70])
def test_groups_that_are_not_finite(T):
    """A NaN key makes the rows that see it NaN; a NaN value the channels of its group; an infinite query its own rows."""
    heads, n_kv, D, slots = 4, 2, 128, 200
    c = KVCache4(1, n_kv, slots, D)
    k, v = randn(1, 1, slots, n_kv * D), randn(2, 1, slots, n_kv * D)
    v[0, 60, 70] = float("inf")                                                      # head 0, channels 64..127
    v[0, 199, 0] = float("nan")                                                      # behind every token below
    c.append(k, v, torch.arange(slots, device="cuda"))
    q = randn(3, 1, T, heads * D)
    pos = torch.full((1, T), 150, device="cuda")
    got = c.attend(q, pos).view(T, heads, D)
    nan = torch.isnan(got.float())
    assert bool(nan[:, :2, 64:].all()) and not bool(nan[:, :2, :64].any()) and not bool(nan[:, 2:].any())
    k[0, 60, 130] = float("nan")                                                     # head 1
    c.append(k, randn(2, 1, slots, n_kv * D), torch.arange(slots, device="cuda"))
    pos[0, 0] = 30                                                                   # this row does not see slot 60
    nan = torch.isnan(c.attend(q, pos).view(T, heads, D).float())
    assert not bool(nan[:, :2].any()) and not bool(nan[0].any()) and bool(nan[1:, 2:].all())
    c.append(randn(1, 1, slots, n_kv * D), randn(2, 1, slots, n_kv * D), torch.arange(slots, device="cuda"))
    q[0, T - 1, 5] = float("inf")
    nan = torch.isnan(c.attend(q, pos).view(T, heads, D).float())
    assert bool(nan[T - 1, 0].all()) and int(nan.sum()) == D


@pytest.mark.parametrize("T,D", [(70, 128), (70, 64), (5, 128), (20, 256)])
def test_a_value_group_that_is_no_number_reaches_who_sees_it(T, D):
    """Tokens one after the other; the value of slot 40 is not finite in one group: rows behind it have NaN there, rows before it and those whose
    window has left it behind do not, though they share a tile of rows and of slots."""
    heads, n_kv, slots = 4, 2, 200
    c = KVCache4(1, n_kv, slots, D)
    v = randn(2, 1, slots, n_kv * D)
    v[0, 40, D + 3] = float("inf")                                                   # head 1, first group
    c.append(randn(1, 1, slots, n_kv * D), v, torch.arange(slots, device="cuda"))
    q = randn(3, 1, T, heads * D)
    pos = (40 - T // 2 + torch.arange(T, device="cuda"))[None]
    for window, sinks in ((0, 0), (9, 0), (9, 45)):
        nan = torch.isnan(c.attend(q, pos, window=window, sinks=sinks).view(T, heads, D).float())
        see = R.visible(pos, slots, window, sinks)[0, :, 40]
        assert not bool(nan[:, :2].any()) and not bool(nan[:, 2:, 64:].any())
        assert torch.equal(nan[:, 2:, :64], see[:, None, None].expand(T, 2, 64))


@pytest.mark.parametrize("T", [1, 2, 70])
@pytest.mark.parametrize("k_gain,v_gain,q_gain", [(1e-6, 1e-5, 1.0), (1e4, 1e6, 1e-4), (1e-20, 1e30, 1e20), (1.0, 1e-30, 1.0), (1e15, 1.0, 1e-15), (1e33, 1e33, 1e-33)])
def test_ranges_of_keys_values_and_queries(T, k_gain, v_gain, q_gain):
    """bf16 inputs of any size whose scores are ordinary; scales that differ from slot to slot by many powers of two."""
    heads, n_kv, D, slots = 4, 2, 128, 300
    c = KVCache4(1, n_kv, slots, D)
    spread = torch.exp2(torch.randint(-12, 13, (1, slots, 1), generator=torch.Generator().manual_seed(1)).float()).cuda()
    k = randn(1, 1, slots, n_kv * D, gain=k_gain)
    v = (randn(2, 1, slots, n_kv * D).float() * v_gain * spread).bfloat16()
    c.append(k, v, torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = randn(3, 1, T, heads * D, gain=q_gain)
    pos = torch.full((1, T), slots - 1, device="cuda")
    assert_near(c.attend(q, pos), R.attend(q, kd, vd, pos, slots, heads, D ** -0.5), c, heads)


def test_long_flat_rows():
    """20000 slots of nearly equal weight beside a first slot that outweighs each of them by e^9: small weights add up, and are not lost."""
    heads, n_kv, D, slots = 4, 1, 64, 20000
    c = KVCache4(1, n_kv, slots, D)
    k = randn(1, 1, slots, D, gain=0.01)
    k[0, 0] = 1.0
    v = randn(2, 1, slots, D, gain=0.1) + 1.0
    v[0, 0] = -1.0
    c.append(k, v, torch.arange(slots, device="cuda"))
    kd, vd = R.cache_values(c.tiles, D)
    q = torch.full((1, 1, heads * D), 9.0 / 8, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((1, 1), slots - 1, device="cuda")
    assert_near(c.attend(q, pos), R.attend(q, kd, vd, pos, slots, heads, D ** -0.5), c, heads)


def test_scale_and_equal_heads():
    """``scale`` counts; query heads that are equal give equal results whatever group of columns they fall in; sequences do not mix."""
    n, heads, n_kv, D, slots = 2, 20, 2, 128, 700
    c, k, v = filled(n, n_kv, slots, D)
    q = randn(1, n, 1, n_kv * D).view(n, 1, n_kv, 1, D).expand(n, 1, n_kv, heads // n_kv, D).reshape(n, 1, heads * D)
    pos = torch.tensor([[699], [350]], device="cuda")
    got = c.attend(q, pos, scale=0.3)
    assert_near(got, R.attend(q, k, v, pos, slots, heads, 0.3), c, heads)
    g = got.view(n, n_kv, heads // n_kv, D)
    assert torch.equal(g, g[:, :, :1].expand_as(g))
    alone = torch.cat([c.attend(q[b:b + 1], pos[b:b + 1], scale=0.3, seq=b) for b in range(n)])
    assert_near(alone, R.attend(q, k, v, pos, slots, heads, 0.3), c, heads)


@pytest.mark.parametrize("T", [1, 6, 300])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
def test_scales_of_any_sign(T, scale):
    """A negative scale turns the scores round, none at all makes every visible slot equal."""
    heads, n_kv, D, slots = 8, 2, 128, 500
    c, k, v = filled(1, n_kv, slots, D)
    q = randn(1, 1, T, heads * D)
    pos = (slots - T + torch.arange(T, device="cuda"))[None]
    assert_near(c.attend(q, pos, window=200, sinks=2, scale=scale), R.attend(q, k, v, pos, slots, heads, scale, 200, 2), c, heads)


@pytest.mark.parametrize("n,T,heads,n_kv,D,slots", [(1, 1, 8, 2, 128, 2000), (2, 1, 8, 1, 64, 30000), (1, 400, 8, 2, 128, 400), (40, 3, 16, 16, 64, 90)])
def test_the_result_may_take_the_place_of_the_queries(n, T, heads, n_kv, D, slots):
    c, _, _ = filled(n, n_kv, slots, D)
    q = randn(1, n, T, heads * D)
    pos = (slots - T + torch.arange(T, device="cuda")).expand(n, T)
    want = c.attend(q, pos)
    assert c.attend(q, pos, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("T", [1, 100])
def test_captured_and_replayed_with_other_positions(T):
    """Append and attend in one graph; positions, keys and queries change between replays; a second graph of the same cache is alive and an
    eager call runs between them."""
    n, heads, n_kv, D, slots = 2, 8, 2, 128, 900
    c, other = KVCache4(n, n_kv, slots, D), KVCache4(n, n_kv, slots, D)
    fill = randn(1, n, slots, n_kv * D), randn(2, n, slots, n_kv * D)
    for x in (c, other):
        x.append(*fill, torch.arange(slots, device="cuda"))
    inv = 1.0 / (1e4 ** (torch.arange(0, D, 2, dtype=torch.float32, device="cuda") / D))
    q, k, v = randn(3, n, T, heads * D), randn(4, n, T, n_kv * D), randn(5, n, T, n_kv * D)
    pos = torch.stack([torch.arange(T), 300 + torch.arange(T)]).cuda()

    def once(cache):
        return cache.attend(cache.append(k, v, pos, q=q, inv_freq=inv), pos, window=200, sinks=4)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once(c)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(once(c))
        graphs.append(g)
    once(other)
    for step in range(4):
        pos += 111
        q.copy_(randn(10 + step, n, T, heads * D)); k.copy_(randn(20 + step, n, T, n_kv * D)); v.copy_(randn(30 + step, n, T, n_kv * D))
        graphs[step % 2].replay()
        got = outs[step % 2].clone()
        assert torch.equal(got, once(other)) and torch.equal(c.tiles, other.tiles)


def test_two_streams_at_once():
    """Calls on two streams share nothing: results are those of one stream."""
    c, _, _ = filled(2, 4, 3000, 128)
    q = [randn(i, 1, 1, 16 * 128) for i in range(2)]
    pos = torch.tensor([[2999]], device="cuda")
    want = [c.attend(q[i], pos, seq=i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.attend(q[i], pos, seq=i))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_offsets_beyond_32_bits():
    """Two sequences that lie 5 GB apart in one buffer."""
    n_kv, D, slots, apart = 2, 64, 100, 5 << 30
    buf = torch.empty(apart + (1 << 20), dtype=torch.uint8, device="cuda")
    tiles = buf.as_strided((2, n_kv, 4, 36 * D), (apart, 4 * 36 * D, 36 * D, 1))
    c, plain = KVCache4.wrap(tiles, D, slots), KVCache4(2, n_kv, slots, D)
    q, k, v = randn(1, 2, slots, 4 * D), randn(2, 2, slots, n_kv * D), randn(3, 2, slots, n_kv * D)
    pos = torch.arange(slots, device="cuda")
    for x in (c, plain):
        x.append(k, v, pos)
    last = torch.full((2, 1), slots - 1, device="cuda")
    assert torch.equal(c.attend(q, pos), plain.attend(q, pos)) and torch.equal(c.attend(q[:, -1:], last), plain.attend(q[:, -1:], last))
    assert all(torch.equal(a, b) for a, b in zip(c.read(pos), plain.read(pos)))


@pytest.mark.parametrize("T,D,slots", [(1, 128, 30_000_000), (70, 128, 30_000_000), (70, 64, 60_000_000), (1, 256, 15_000_000)])
def test_slots_beyond_4_gb_of_one_head(T, D, slots):
    """The last slots of a head whose tiles take more than 2^32 bytes, against the same slots at the beginning of a small cache."""
    heads, used = 8, 192
    far, near = KVCache4(1, 1, slots, D), KVCache4(1, 1, used, D)
    assert far.nbytes() > 1 << 32
    q, k, v = randn(1, 1, T, heads * D), randn(2, 1, used, D), randn(3, 1, used, D)
    at = torch.arange(used, device="cuda")[None]
    first = (slots - used) // 32 * 32
    near.append(k, v, at)
    far.append(k, v, at + first)
    assert all(torch.equal(a, b) for a, b in zip(near.read(at), far.read(at + first)))
    kd, vd = R.cache_values(near.tiles, D)
    pos = (used - T + torch.arange(T, device="cuda"))[None]
    ref = R.attend(q, kd, vd, pos, used, heads, D ** -0.5, 90)
    assert_near(near.attend(q, pos, window=90), ref, near, heads)
    assert_near(far.attend(q, pos + first, window=90), ref, far, heads)


def test_refusals_of_gpu_tensors():
    c = KVCache4(2, 2, 40, 64)
    x, pos = torch.zeros(2, 3, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 3, dtype=torch.long, device="cuda")
    for bad in (lambda: c.append(x.half(), x, pos), lambda: c.append(x, x, pos.int()), lambda: c.attend(x.float(), pos), lambda: c.read(pos.int()),
                lambda: c.attend(x, pos.cpu())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: c.append(x, x[:, :2], pos), lambda: c.append(x, x, pos[:, :2]), lambda: c.append(x, x, pos, seq=1), lambda: c.append(x[..., :64], x, pos),
                lambda: c.append(x, x, pos, q_norm=x[0, 0, :64]), lambda: c.append(x, x, pos, inv_freq=torch.ones(64, device="cuda")),
                lambda: c.append(x, x, pos, k_norm=torch.ones(64, device="cuda")), lambda: c.append(x, x, pos, q=x, q_out=x[:, :, ::2]),
                lambda: c.attend(x[..., :64], pos), lambda: c.attend(x, pos, window=-1), lambda: c.attend(x, pos, sinks=-1), lambda: c.attend(x, pos, seq=-1),
                lambda: c.attend(x, pos, out=x[:1]), lambda: c.attend(x, pos, out=x.transpose(0, 1)), lambda: c.read(pos[None])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        c.attend(x.clone().requires_grad_(), pos)
    with torch.no_grad():
        c.attend(x.clone().requires_grad_(), pos)
    none = torch.zeros(0, 3, 128, dtype=torch.bfloat16, device="cuda")
    assert c.attend(none, pos[:0]).shape == none.shape and c.append(none, none, pos[:0]) is None
    assert c.read(pos[:, :0])[0].shape == (2, 0, 2, 64)
