"""Embedding and head loss: calls that must not pass without a word (needs a B200)."""
import pytest
import torch

import cobalt_b200 as cb
from cobalt_b200 import SparseQuantConfig
from cobalt_b200.decoder import build_random_decoder
from oracle import model_oracle as MO

pytestmark = pytest.mark.gpu


def test_a_result_written_in_place_moves_its_version():
    """What saved the buffer that ``out`` names must notice that it was overwritten, as after every torch operation with ``out=``."""
    table = torch.randn(9, 16, device="cuda")
    ids = torch.tensor([1, 8, 3], device="cuda")
    buffers, w = torch.randn(2, 3, 16, device="cuda"), torch.randn(16, 4, device="cuda").requires_grad_()
    y = buffers[0] @ w
    kept = buffers._version
    cb.embed(ids[:0], table, out=buffers[0, :0])                       # nothing is written
    assert buffers._version == kept
    cb.embed(ids, table, out=buffers[0])
    assert buffers._version == kept + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        out = torch.empty(3, 16, device="cuda")
        assert torch.equal(cb.embed(ids, table, out=out), table[ids])


def test_a_result_must_not_lie_in_what_is_read():
    """Blocks would read rows that others have overwritten: refused before a launch."""
    table = torch.randn(40, 16, device="cuda")
    kept = table.clone()
    ids = torch.arange(10, device="cuda")
    for out in (table[:10], table[30:], table[5:15]):
        with pytest.raises(ValueError, match="overlap"):
            cb.embed(ids, table, out=out)
    with pytest.raises(ValueError, match="overlap"):                   # rows of the table on either side of it
        cb.embed(ids[:1], table[::2, :8], out=table[1, :8].view(1, 8))
    flat = torch.zeros(90, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        cb.embed(flat[70:80], table, out=flat[:80].view(torch.float32).view(10, 16))
    torch.cuda.synchronize()
    assert torch.equal(table, kept) and not bool(flat.any())
    both = torch.empty(50, 16, device="cuda")                          # behind one another is as good as apart
    both[:40] = kept
    assert torch.equal(cb.embed(ids, both[:40], out=both[40:]), kept[:10]) and torch.equal(both[:40], kept)
    got = cb.embed(flat[80:], table, out=flat[:80].view(torch.float32).view(10, 16))
    assert torch.equal(got, kept[:1].expand(10, 16))


def test_derivatives_that_there_are_none_of_are_refused():
    """A tangent would be lost without a word, which reads as a derivative of zero; so would the second derivative of the embedding."""
    import torch.autograd.forward_ad as fwAD
    table, ids = torch.randn(9, 16, device="cuda"), torch.tensor([1, 8, 3], device="cuda")
    x, w = torch.randn(3, 16, device="cuda").bfloat16(), torch.randn(9, 16, device="cuda").bfloat16()
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: cb.embed(ids, dual(table)), lambda: cb.embed(ids, dual(table.clone().requires_grad_())), lambda: cb.embed_grad(dual(table[:3]), ids, 9),
                     lambda: cb.head_loss(dual(x), w, ids), lambda: cb.head_loss(x, dual(w), ids), lambda: cb.head_loss_and_grad(x, dual(w), ids),
                     lambda: cb.head_loss_and_grad(x, w, ids, grad=dual(torch.ones((), device="cuda")))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="forward-mode"):
            cb.embed(ids, table, out=dual(table[:3].clone()))
        assert torch.equal(cb.embed(ids, table), table[ids])
    grad = table[:3].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second"):
        cb.embed_grad(grad, ids, 9)
    with torch.no_grad():
        assert torch.equal(cb.embed_grad(grad, ids, 9)[ids], grad)


def test_a_captured_step_of_a_tied_table_beside_older_graphs():
    """Refused while a graph of the table made on another stream lives, whatever was made since; then captured, and replayed on new tokens."""
    V, H, n = 300, 64, 40
    table = torch.randn(V, H, device="cuda").bfloat16().requires_grad_()
    ids = torch.randint(0, V, (n,), device="cuda")

    def step():
        loss = cb.head_loss(cb.embed(ids, table, 2.0), table, ids.roll(-1))
        return loss, *torch.autograd.grad(loss, table)

    step()
    kept = cb.embed(ids, table)
    cb.head_loss(kept.detach(), table, ids)                            # dropped at once
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="still alive"):
            step()
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = step()
    for seed in (1, 2):
        ids.copy_(torch.randint(0, V, (n,), generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        want = step()
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


@pytest.mark.parametrize("width", [8, 33, 4096])
def test_ids_beyond_a_table_are_told(width):
    """-1 is padding; an id of the table's length or more comes from another vocabulary.  Both read zeros, the latter leaves its code."""
    table = torch.randn(9, width, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ids = torch.tensor([3, -1, 8, -(2 ** 63)], device="cuda")
    y = cb.embed(ids, table, 2.0, status=status)
    assert int(status) == 0 and torch.equal(y[::2], table[[3, 8]] * 2) and not bool(y[1::2].any())
    for bad in (9, 2 ** 40):
        ids[1] = bad
        assert torch.equal(cb.embed(ids, table.requires_grad_(), 2.0, status=status), y) and int(status) == 8
        status.fill_(5)                                                # the first code stays
        cb.embed(ids, table.detach(), status=status)
        assert int(status) == 5
        status.zero_()
    for wrong in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="status"):
            cb.embed(ids, table.detach(), status=wrong)


def test_a_decoder_tells_ids_of_another_vocabulary():
    """Refused at once in host memory; on the device they count as padding, and are told by device_status() and generate()."""
    cfg = MO.llama_config(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=64, inter=512, vocab=512)
    dec = build_random_decoder(cfg, SparseQuantConfig(4, 0.5, 0.5), 64, torch.device("cuda"))
    ids = torch.arange(20)
    want, _ = dec.generate(ids.cuda(), 4)
    ids[3] = 512
    for call in (dec.prefill, dec.score, lambda i: dec.generate(i, 4)):
        with pytest.raises(ValueError, match="512"):
            call(ids)
    with pytest.raises(ValueError, match="999"):
        dec.generate(torch.arange(20), 4, teacher=torch.tensor([1, 999, 2, 3]))
    assert dec.device_status() == 0
    for call in (dec.prefill, dec.score):
        call(ids.cuda())
        assert dec.device_status() == 8 and dec.device_status() == 0
    with pytest.raises(ValueError, match="outside the vocabulary"):
        dec.generate(ids.cuda(), 4)
    with pytest.raises(ValueError, match="outside the vocabulary"):    # in the captured step
        dec.generate(torch.arange(20), 4, teacher=torch.tensor([1, 999, 2, 3], device="cuda"))
    ids[3] = -1
    dec.score(ids.cuda())
    assert torch.equal(dec.generate(torch.arange(20).cuda(), 4)[0], want) and dec.device_status() == 0


@pytest.mark.parametrize("n", [20, 300])
def test_a_healthy_call_leaves_a_status_word_alone(n):
    x, w = torch.randn(n, 64, device="cuda").bfloat16(), torch.randn(500, 64, device="cuda").bfloat16()
    status = torch.full((1,), 3, dtype=torch.int32, device="cuda")
    loss, dx, dw = cb.head_loss_and_grad(x, w, torch.arange(n, device="cuda"), status=status)
    assert int(status) == 3 and bool(loss.isfinite()) and not bool(dx.isnan().any()) and not bool(dw.isnan().any()) and cb.head_loss_status() == 0


@pytest.mark.parametrize("n", [1, 20, 64, 65, 128])
def test_what_does_not_count_reaches_nothing_of_few_tokens(n):
    """Rows without a target may hold anything; if none has one, everything is zero; an infinite gradient stays in its token's row of dx."""
    V, H = 900, 136
    g = torch.Generator(device="cuda").manual_seed(n)
    x, w = torch.randn(n, H, generator=g, device="cuda").bfloat16(), (torch.randn(V, H, generator=g, device="cuda") * H ** -0.5).bfloat16()
    t = torch.randint(0, V, (n,), generator=g, device="cuda")
    out = torch.arange(n, device="cuda") % 3 == 1
    t[out] = -1
    anything = x.clone()
    anything[out] = float("nan")
    for reduction in ("mean", "sum", "none"):
        want, got = cb.head_loss_and_grad(x, w, t, reduction), cb.head_loss_and_grad(anything, w, t, reduction)
        assert all(torch.equal(a, b) for a, b in zip(want, got)) and not bool(got[1][out].any()) and bool(got[2].isfinite().all())
        loss, dx, dw = cb.head_loss_and_grad(torch.full_like(x, float("nan")), w, torch.full_like(t, V), reduction)
        assert not bool(loss.any()) and not bool(dx.any()) and not bool(dw.any())
    f = torch.ones(n, device="cuda")
    f[0] = float("inf")
    _, dx, _ = cb.head_loss_and_grad(x, w, t, "none", f)
    ones = cb.head_loss_and_grad(x, w, t, "none", torch.ones(n, device="cuda"))[1]
    assert not bool(dx[0].isfinite().any()) and torch.equal(dx[1:], ones[1:])


@pytest.mark.parametrize("n,V,H", [(40, 3, 65535 * 128 + 1), (20, 2, 65535 * 1024 + 8)])
def test_the_gradient_of_very_wide_rows(n, V, H):
    """More blocks of columns than a grid has in its second dimension, of values one by one and of 16 bytes.  Sums of small whole numbers are exact."""
    ids = torch.arange(n, device="cuda") % V
    ids[::7] = 0
    grad = (torch.arange(H, device="cuda") % 13 - 6).bfloat16()[None] * (torch.arange(n, device="cuda") % 3 - 1).bfloat16()[:, None]
    got = cb.embed_grad(grad, ids, V)
    for v in range(V):
        assert torch.equal(got[v], grad[ids == v].float().sum(0).bfloat16())
