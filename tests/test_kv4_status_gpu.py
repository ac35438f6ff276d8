"""Status words of the 4-bit KV cache on the GPU: a failure is told to those whom it concerns, and to nobody else (needs a B200)."""
import pytest
import torch

from cobalt_b200 import KVCache4, SparseQuantConfig, _lib
from cobalt_b200.decoder import CobaltDecoder, build_random_decoder
from oracle import model_oracle as MO
from test_kv4_gpu import filled, randn

pytestmark = pytest.mark.gpu


def test_decoders_do_not_hear_of_each_other():
    cfg = MO.llama_config(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, inter=1024, vocab=1008)
    a = build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), 64, torch.device("cuda"), kv_bits=4)
    b = CobaltDecoder(cfg, a.lin, a.P, 64, a.dev, kv_bits=4)
    assert len({c._word for d in (a, b) for c in d.kv4}) == 2                          # one for all layers of a decoder
    ids = torch.randint(0, 1000, (20,), generator=torch.Generator().manual_seed(1))
    want = a.generate(ids, 4)[1]
    a.kv4[1]._status.fill_(4)                                                         # as a wait of the last layer would leave it
    assert b.device_status() == 0 and torch.equal(b.generate(ids, 4)[1], want)
    assert a.device_status() == 4
    with pytest.raises(_lib.CobaltError):
        a.generate(ids, 4)
    assert a.device_status() == 0 and torch.equal(a.generate(ids, 4)[1], want)


def test_healthy_calls_leave_words_alone():
    """All three kernels, with a word of the cache's own and with the device's: nothing is written, and what is there stays for who asks."""
    word = torch.zeros(3, dtype=torch.int32, device="cuda")
    for n_kv, D, slots, T, heads in ((2, 128, 500, 1, 8), (1, 64, 40000, 3, 4), (8, 128, 400, 320, 32)):
        c, _, _ = filled(1, n_kv, slots, D)
        watched = KVCache4.wrap(c.tiles, D, slots, status=word[1:2])
        device = KVCache4.wrap(c.tiles, D, slots)
        q, pos = randn(1, 1, T, heads * D), (slots - T + torch.arange(T, device="cuda"))[None]
        for value in (0, 7):
            word.fill_(value)
            got = [x.attend(q, pos) for x in (c, watched, device)]
            assert all(torch.equal(got[0], g) for g in got[1:]) and word.tolist() == [value] * 3
        assert watched.device_status() == 7 and word.tolist() == [7, 0, 7] and c.device_status() == 0 and device.device_status() == 0


def test_arguments_that_require_a_gradient_are_refused():
    """Norm weights as parameters of a module, frequencies and results too, not q, k and v alone; under no_grad() they are taken."""
    c = KVCache4(1, 1, 40, 64)
    x, pos = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 1, dtype=torch.long, device="cuda")
    w, f = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16, device="cuda")), torch.ones(32, device="cuda", requires_grad=True)
    out = torch.zeros_like(x, requires_grad=True)
    calls = (lambda: c.append(x, x, pos, k_norm=w), lambda: c.append(x, x, pos, q=x, q_norm=w), lambda: c.append(x, x, pos, inv_freq=f),
             lambda: c.append(x, x, pos, q=x, q_out=out), lambda: c.attend(x, pos, out=out))
    for call in calls:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
