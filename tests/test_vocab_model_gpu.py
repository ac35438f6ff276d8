"""Embedding and head loss where the framework uses them, and together (needs a B200)."""
import pytest
import torch
import torch.nn.functional as F

import cobalt_b200 as cb
from cobalt_b200 import SparseQuantConfig
from cobalt_b200.decoder import build_random_decoder
from oracle import model_oracle as MO

pytestmark = pytest.mark.gpu


def decoder(family, batch=1, head_bits=0, kv_bits=16, max_ctx=96):
    cfg = MO.gemma3_config(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, inter=1024, vocab=1008, sliding_window=16, pattern=2, query_pre_attn_scalar=96,
                           rope_scaling={"rope_type": "linear", "factor": 8.0}) if family == "gemma" else \
        MO.llama_config(hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, inter=1024, vocab=1008)
    return build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), max_ctx, torch.device("cuda"), batch=batch, head_bits=head_bits, kv_bits=kv_bits)


@pytest.mark.parametrize("family", ["llama", "gemma"])
def test_the_decoders_embedding_keeps_its_bits(family):
    dec = decoder(family)
    table = dec.P["model.embed_tokens.weight"]
    ids = torch.randint(0, 1008, (77,), generator=torch.Generator().manual_seed(1)).cuda()
    want = table.index_select(0, ids)
    if family == "gemma":
        want = want * torch.tensor(512.0 ** 0.5, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(dec._embed(ids), want) and torch.equal(dec._embed(ids.int()), want)
    assert not bool(dec._embed(torch.tensor([-1, 1008], device="cuda")).any())


@pytest.mark.parametrize("family,batch,T,head_bits,kv_bits", [("llama", 1, 40, 0, 16), ("llama", 1, 2, 0, 16), ("llama", 3, 33, 4, 16), ("gemma", 1, 9, 0, 16),
                                                              ("gemma", 4, 50, 0, 16), ("gemma", 2, 12, 4, 16), ("gemma", 2, 21, 0, 4)])
def test_score_against_the_logits_of_prefill(family, batch, T, head_bits, kv_bits):
    """Hidden states are the same, so the loss differs from that of bf16 logits by their rounding alone: 2^-8 of a logit, twice."""
    dec = decoder(family, batch, head_bits, kv_bits)
    ids = torch.randint(0, 1008, (batch, T) if batch > 1 else (T,), generator=torch.Generator().manual_seed(T)).cuda()
    logits = dec.prefill(ids).view(batch, T, -1)[:, :-1].double()
    targets = ids.view(batch, T)[:, 1:]
    want = F.cross_entropy(logits.transpose(1, 2), targets, reduction="none")
    got = dec.score(ids)
    assert got.shape == (want.shape if batch > 1 else want.shape[1:]) and got.dtype is torch.float32 and not got.requires_grad
    # (a 4-bit cache adds its sums in the same order both times: the calls are the same)
    slack = 2.0 ** -7 * logits.abs().amax(-1) + 2.0 ** -12
    assert bool(((got.view(batch, -1).double() - want).abs() <= slack).all())
    near = got.double().mean().item()
    assert abs(dec.score(ids, "mean").item() - near) < 1e-5 * near and abs(dec.score(ids, "sum").item() - near * got.numel()) < 1e-5 * near * got.numel()
    assert dec.device_status() == 0
    if batch > 1:                                                      # padded at the end: what is there does not change
        ids[0, T // 2:] = -1
        padded = dec.score(ids)
        assert torch.equal(padded[1:], got[1:]) and not bool(padded[0, max(T // 2 - 1, 0):].any())
        assert torch.allclose(padded[0, :max(T // 2 - 1, 0)], got[0, :max(T // 2 - 1, 0)], atol=1e-3)


def test_score_of_one_token_and_refusals():
    dec = decoder("llama")
    assert dec.score(torch.tensor([3])).shape == (0,) and float(dec.score(torch.tensor([3]), "mean")) == 0
    for bad in (torch.zeros(0, dtype=torch.int64), torch.zeros(1, 1, 1, dtype=torch.int64), torch.zeros(97, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int64)):
        with pytest.raises(ValueError):
            dec.score(bad)


@pytest.mark.parametrize("family", ["llama", "gemma"])
def test_the_dense_head_can_be_tuned(family):
    """The gradient of score() with respect to the head is that of the loss over the last hidden states."""
    dec = decoder(family, batch=2)
    ids = torch.randint(0, 1008, (2, 30), generator=torch.Generator().manual_seed(5)).cuda()
    name = "model.embed_tokens.weight" if family == "gemma" else "lm_head.weight"
    head = dec.P[name].requires_grad_()
    loss = dec.score(ids, "mean")
    loss.backward()
    with torch.no_grad():
        x = dec._prefill(ids, True)
    leaf = head.detach().double().requires_grad_()
    ref = F.cross_entropy((x[:, :-1].double() @ leaf.T).flatten(0, 1), ids[:, 1:].flatten())
    ref.backward()
    assert abs(float(loss.detach()) - float(ref)) < 1e-5 * float(ref)
    # d and the result are rounded to bf16: each 2^-8 at most
    assert float((head.grad.double() - leaf.grad).norm() / leaf.grad.norm()) < 2.0 ** -7
    dec.generate(ids, 3)                                               # and the model still decodes


@pytest.mark.parametrize("n,V,H", [(50, 300, 64), (700, 5003, 256)])
def test_a_tied_table_through_both_ends(n, V, H):
    """Embedding, something in between, head loss: the gradient of the one table is the sum of both ends', as fp64 autograd has it."""
    g = torch.Generator(device="cuda").manual_seed(n)
    table = (torch.randn(V, H, generator=g, device="cuda") * 0.05).bfloat16()
    ids = torch.randint(0, V, (n,), generator=g, device="cuda")
    ids[::9] = -1
    targets = torch.roll(ids, -1)

    def step(t, embed, loss):
        h = embed(t)
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
        value = loss(h, t)
        return value, torch.autograd.grad(value, t)[0]

    leaf = table.clone().requires_grad_()
    got, d = step(leaf, lambda t: cb.embed(ids, t, 8.0), lambda h, t: cb.head_loss(h, t, targets))
    exact = table.double().requires_grad_()
    ok = ids >= 0
    want, e = step(exact, lambda t: torch.where(ok[:, None], t[ids.clamp_min(0)] * 8.0, 0.0),
                   lambda h, t: F.cross_entropy((h @ t.T)[targets >= 0], targets[targets >= 0]))
    # some sixteen roundings to bf16 on the way, forward and back (2^-8 each at most); everything else is exact to fp32
    assert abs(float(got.detach()) - float(want)) < 0.01 * float(want)
    assert float((d.double() - e).norm() / e.norm()) < 16 * 2.0 ** -8
