"""Status words and forms of attention calls of the 4-bit KV cache, what needs no GPU."""
import pytest
import torch

from cobalt_b200 import KVCache4, _lib


@pytest.fixture(scope="module")
def lib():
    from cobalt_b200 import build
    build.build()
    return _lib.load()


def test_a_word_off_its_boundary_is_refused(lib):
    args = (4096, 128, 4096, 1 << 20, 4096, 1, 4096, 1, 1, 1, 1, 128, 64, 0, 0, 1.0, None, 0)
    assert lib.cobalt_kv4_attend_watched(*args, 4098, None) == -1
    assert lib.cobalt_kv4_attend_watched(*args[:7], 0, *args[8:], 4096, None) == -1 and lib.cobalt_kv4_attend_watched(*args[:6], 4104, *args[7:], None, None) == -1


def test_every_cache_has_a_word_of_its_own_or_the_one_it_is_given():
    word = torch.zeros(1, dtype=torch.int32)
    a, b, c, d = (KVCache4(1, 1, 40, 64, device="cpu", status=s) for s in (None, None, word, word))
    a._status.fill_(4)
    assert a.device_status() == 4 and a.device_status() == 0 and b.device_status() == 0
    word.fill_(3)
    assert c.device_status() == 3 and d.device_status() == 0
    e = KVCache4.wrap(a.tiles, 64, 40, status=word)
    word.fill_(2)
    assert e.device_status() == 2
    for bad in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ValueError):
            KVCache4(1, 1, 40, 64, device="cpu", status=bad)
        with pytest.raises(ValueError):
            KVCache4.wrap(a.tiles, 64, 40, status=bad)


def test_form_refuses(lib):
    good = (1, 1, 8, 2, 128, 64, 0, 0)
    for i, bad in ((0, 0), (1, 0), (2, 7), (3, 0), (4, 96), (5, 0), (6, -1), (7, -1)):
        assert lib.cobalt_kv4_attend_form(*good[:i], bad, *good[i + 1:]) == -1
    if not torch.cuda.is_available():
        assert lib.cobalt_kv4_attend_form(*good) < 0 and lib.cobalt_kv4_attend_scratch_bytes(*good) == 0      # no device to plan for
