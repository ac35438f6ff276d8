"""4-bit KV cache, what needs no GPU: refusals of the C ABI and of ``KVCache4``, and the format's reference against itself."""
import pytest
import torch

import kv4_reference as R


@pytest.fixture(scope="module")
def lib():
    from cobalt_b200 import build, _lib
    build.build()
    return _lib.load()


def test_tile_bytes(lib):
    assert [lib.cobalt_kv4_tile_bytes(d) for d in (64, 128, 192, 256)] == [36 * d for d in (64, 128, 192, 256)]
    assert [lib.cobalt_kv4_tile_bytes(d) for d in (0, -64, 32, 96, 320)] == [0] * 5


def _append(lib, **kw):
    a = dict(k=4096, ld_k=128, v=4096, ld_v=128, q=None, ld_q=0, qo=None, ld_qo=0, pos=4096, ps=1, tiles=4096, ts=1 << 20, n=1, T=1, nh=0, nkv=1, D=128,
             slots=64, f=None, qn=None, kn=None, eps=1e-6) | kw
    return lib.cobalt_kv4_append(*a.values(), None)


def _read(lib, **kw):
    a = dict(tiles=4096, ts=1 << 20, pos=4096, ps=1, k=4096, v=4096, n=1, T=1, nkv=1, D=128, slots=64) | kw
    return lib.cobalt_kv4_read(*a.values(), None)


def _attend(lib, **kw):
    a = dict(q=4096, ld_q=128, tiles=4096, ts=1 << 20, pos=4096, ps=1, out=4096, n=1, T=1, nh=1, nkv=1, D=128, slots=64, w=0, s=0, scale=1.0, scratch=None,
             sb=0) | kw
    return lib.cobalt_kv4_attend(*a.values(), None)


BAD = [dict(tiles=None), dict(tiles=4104), dict(pos=None), dict(pos=4100), dict(ps=-1), dict(ts=-16), dict(ts=8), dict(n=2, ts=2 * 4608 - 16), dict(n=0),
       dict(T=0), dict(nkv=0), dict(slots=0), dict(D=96), dict(D=320), dict(D=0)]


@pytest.mark.parametrize("kw", BAD)
def test_bad_caches_are_refused_before_any_launch(lib, kw):
    for call in (_append, _read, _attend):
        assert call(lib, **kw) == -1, call


@pytest.mark.parametrize("kw", [dict(n=1 << 16, T=1 << 15, ts=1 << 30), dict(nkv=1 << 17, ld_k=1 << 24, ld_v=1 << 24), dict(slots=1 << 30)])
def test_sizes_beyond_the_kernels_counts_are_refused(lib, kw):
    assert _append(lib, **kw) == -6
    kw = {k: v for k, v in kw.items() if k in ("n", "T", "ts", "nkv", "slots")}
    assert _read(lib, **kw) == -6 and _attend(lib, **kw) == -6


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k=4104), dict(ld_k=132), dict(ld_v=126), dict(q=4096, nh=0, qo=4096),
                                dict(q=4096, nh=1, ld_q=128, qo=None, ld_qo=128), dict(q=4096, nh=1, ld_q=64, qo=4096, ld_qo=128), dict(q=4096, nh=1, ld_q=128, qo=4104, ld_qo=128), dict(qn=4096),
                                dict(f=4097), dict(kn=4098)])
def test_append_refuses(lib, kw):
    assert _append(lib, **kw) == -1


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=4104), dict(ld_q=132), dict(ld_q=64), dict(out=None), dict(out=4104), dict(nh=0), dict(nh=3, nkv=2, ld_q=512),
                                dict(w=-1), dict(s=-1)])
def test_attend_refuses(lib, kw):
    assert _attend(lib, **kw) == -1


def test_read_refuses(lib):
    assert _read(lib, k=None) == -1 and _read(lib, v=4104) == -1


def test_class_refuses():
    from cobalt_b200 import KVCache4
    for bad in (dict(n_seq=0), dict(n_kv_heads=0), dict(slots=0), dict(head_dim=96), dict(head_dim=512)):
        with pytest.raises(ValueError):
            KVCache4(**dict(dict(n_seq=1, n_kv_heads=1, slots=8, head_dim=64, device="cpu"), **bad))
    c = KVCache4(2, 3, 40, 128, device="cpu")
    assert c.tiles.shape == (2, 3, 2, 36 * 128) and c.slots == 40 and c.nbytes() == c.tiles.numel()
    x, pos = torch.zeros(1, 1, 384, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.long)
    for call in (lambda: c.append(x, x, pos), lambda: c.attend(x, pos), lambda: c.read(pos)):
        with pytest.raises(RuntimeError):                                             # no CPU path
            call()
    t = c.tiles
    for tiles, dim, slots in ((t.float(), 128, None), (t, 64, None), (t[0], 128, None), (t.transpose(0, 1), 128, None), (t[:, :, :1], 128, None), (t, 128, 32),
                              (t, 128, 65), (t[:0], 128, None)):
        with pytest.raises(ValueError):
            KVCache4.wrap(tiles, dim, slots)
    w = KVCache4.wrap(t, 128)
    assert w.slots == 64 and w.tiles.data_ptr() == t.data_ptr()
    assert KVCache4.wrap(torch.zeros(4, 3, 2, 36 * 128, dtype=torch.uint8)[::2], 128, 40).n_seq == 2


def test_reference_quantiser_keeps_to_its_bound():
    """|x - x'| <= s (1/2 + 15 2^-8 + |z| 2^-11 + 2^-16): half a code, the scale's rounding over 15 codes, the zero's, and the fp32 quotient."""
    g = torch.Generator().manual_seed(0)
    for gain, mean in ((1.0, 0.0), (1e-3, 1.0), (1e30, 0.0), (3.0, -100.0)):
        x = (torch.randn(200, 128, generator=g) * gain + mean).bfloat16()
        c, s, z = R.quantise(x)
        sd, zd = (t.double()[..., None].expand(-1, -1, 64).reshape(200, 128) for t in (s, z))
        assert bool(((x.double() - R.values(c, s, z)).abs() <= sd * (0.5 + 15 * 2.0 ** -8 + zd.abs() * 2.0 ** -11 + 2.0 ** -16)).all())
    const = torch.full((1, 64), -3.140625).bfloat16()
    assert torch.equal(R.values(*R.quantise(const)), const.double())
