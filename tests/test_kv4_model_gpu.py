"""``CobaltDecoder`` with keys and values in 4 bits: the append and the attention as the layers use them (needs a B200).

Every attention call of a decoder is compared with attention in fp64 from the same queries and the bytes of the same caches, within the
bound of ``test_kv4_gpu.py``; the keys and values with what the format makes of the projections' outputs.  Logits of two runs are not
compared across attentions: a hidden value that rounds differently can move a code of the next layer by a whole step."""
import pytest
import torch

import kv4_reference as R
from cobalt_b200 import SparseQuantConfig
from cobalt_b200.decoder import CobaltDecoder, build_random_decoder
from oracle import model_oracle as MO
from test_kv4_gpu import assert_near

pytestmark = pytest.mark.gpu


def config(family, head_dim=64, window=16):
    if family == "gemma":
        return MO.gemma3_config(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=head_dim, inter=1024, vocab=1008, sliding_window=window, pattern=2,
                                query_pre_attn_scalar=96, rope_scaling={"rope_type": "linear", "factor": 8.0})
    return MO.llama_config(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=head_dim, inter=1024, vocab=1008)


class Checked(CobaltDecoder):
    """Checks every eager call; counts them."""
    calls = 0

    def _append4(self, q, k, v, positions, layer, seq, n):
        T = q.shape[0] // n
        super()._append4(q, k, v, positions, layer, seq, n)
        if not torch.cuda.is_current_stream_capturing():
            pos = positions.expand(n, T) if positions.shape[0] == T else positions.view(n, T)
            want = R.values(*R.quantise(v.view(n, T, self.nkv, -1).cpu())).float().bfloat16()          # as it is read back
            assert torch.equal(self.kv4[layer].read(pos.contiguous(), seq=seq)[1].cpu(), want)

    def _attend4(self, q, positions, layer, seq, n):
        got = super()._attend4(q, positions, layer, seq, n)
        if not torch.cuda.is_current_stream_capturing():
            cfg, c, T = self.cfg, self.kv4[layer], q.shape[0] // n
            window = int(cfg.get("sliding_window") or 0) if self.types[layer] == "sliding_attention" else 0
            k, v = R.cache_values(c.tiles[seq:seq + n], c.head_dim)
            pos = positions.expand(n, T) if positions.shape[0] == T else positions.view(n, T)
            ref = R.attend(q.view(n, T, -1), k, v, pos, c.slots, self.nh, self.scale, window, self.sinks if window else 0)
            assert_near(got.view(n, T, -1), ref, c, self.nh)
            self.calls += 1
        return got


@pytest.mark.parametrize("family,head_dim,batch,T,sinks", [("llama", 64, 1, 40, 0), ("gemma", 64, 3, 40, 0), ("gemma", 64, 2, 37, 3), ("llama", 128, 2, 21, 0),
                                                           ("gemma", 256, 1, 50, 2), ("llama", 192, 1, 9, 0)])
def test_every_layer_of_a_decoder(family, head_dim, batch, T, sinks):
    cfg = config(family, head_dim)
    dec = build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), T + 30, torch.device("cuda"), batch=batch, head_bits=4, kv_bits=4, attention_sinks=sinks)
    chk = Checked(cfg, dec.lin, dec.P, T + 30, dec.dev, batch=batch, head=dec.head, kv_bits=4, attention_sinks=sinks)
    assert dec.k_cache is None and len(dec.kv4) == 2
    ids = torch.randint(0, 1000, (batch, T) if batch > 1 else (T,), generator=torch.Generator().manual_seed(T))
    teacher = torch.randint(0, 1000, (12, batch) if batch > 1 else (12,), generator=torch.Generator().manual_seed(T + 1))
    _, want = chk.generate(ids, 12, teacher=teacher, use_graph=False)
    assert chk.calls == 2 * ((1 if T > 16 else batch) + 11)                          # layers x (prompts together + steps)
    _, got = dec.generate(ids, 12, teacher=teacher)                                  # the captured step: the same bits
    assert torch.equal(got, want) and dec.device_status() == 0
    assert all(torch.equal(a.read(torch.arange(T + 11, device="cuda"))[i], b.read(torch.arange(T + 11, device="cuda"))[i])
               for a, b in zip(dec.kv4, chk.kv4) for i in range(2))


def test_first_slots_count():
    """With a window, the first slots change what later tokens see; without one they change nothing."""
    cfg = config("gemma")
    ids = torch.randint(0, 1000, (60,), generator=torch.Generator().manual_seed(1))
    q = SparseQuantConfig(4, 0.5, 0.5)
    a, b = (build_random_decoder(cfg, q, 64, torch.device("cuda"), kv_bits=4, attention_sinks=n).prefill(ids) for n in (0, 4))
    assert torch.equal(a[:16], b[:16]) and not torch.equal(a[20:], b[20:])
    cfg = config("llama")
    a, b = (build_random_decoder(cfg, q, 64, torch.device("cuda"), kv_bits=4, attention_sinks=n).prefill(ids) for n in (0, 4))
    assert torch.equal(a, b)


def test_captured_step_lives_beside_eager_calls_and_other_decoders():
    """Two decoders with captured steps over caches of their own; prompts and eager steps of one between replays of the other."""
    cfg = config("llama")
    q = SparseQuantConfig(4, 0.5, 0.5)
    ids = torch.randint(0, 1000, (2, 33), generator=torch.Generator().manual_seed(1))
    a = build_random_decoder(cfg, q, 64, torch.device("cuda"), batch=2, kv_bits=4)
    b = CobaltDecoder(cfg, a.lin, a.P, 64, a.dev, batch=2, kv_bits=4)
    want = a.generate(ids, 10)[1]
    b.generate(ids.flip(0), 6)
    assert torch.equal(a.generate(ids, 10)[1], want)
    b.prefill(ids)
    assert torch.equal(a.generate(ids, 10)[1], want) and torch.equal(b.generate(ids, 10, use_graph=False)[1], want)


def test_refusals():
    cfg = config("llama")
    dec = build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), 16, torch.device("cuda"))
    for bad in (dict(kv_bits=8), dict(attention_sinks=2), dict(kv_bits=4, attention_sinks=-1)):
        with pytest.raises(ValueError):
            CobaltDecoder(cfg, dec.lin, dec.P, 16, dec.dev, **bad)
