"""Captured backward passes and older graphs of the same leaf, and what an operator leaves behind in it (no GPU needed: the kernels are stood in for, streams
and captures are what a test says).

torch waits for the stream on which a leaf's node was made when a backward pass reaches the leaf, and the node lives as long as any graph holds it.  In a
capture on another stream that wait ends the capture or the process, so the backward pass is to be refused before."""
import gc

import pytest
import torch

from cobalt_b200 import vocab


class Place:
    stream, capturing = 0, False


@pytest.fixture
def place(monkeypatch):
    """The operators on CPU tensors: right values do not matter, their graphs do."""
    now = Place()
    monkeypatch.setattr(vocab, "_raw_stream", lambda index: now.stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now.capturing)
    monkeypatch.setattr(vocab, "_gpu", lambda name, t: t.get_device())
    monkeypatch.setattr(vocab, "_embed", lambda ids, table, scale, *out: table.detach()[ids] * scale)
    monkeypatch.setattr(vocab, "embed_grad", lambda grad, ids, n_rows, scale: torch.ones(n_rows, grad.shape[-1], dtype=grad.dtype))
    monkeypatch.setattr(vocab, "_head_loss", lambda x, weight, *rest: (x.detach().float().sum(), torch.zeros(len(x), 2)))
    monkeypatch.setattr(vocab, "_head_loss_grad", lambda x, weight, *rest: (torch.ones_like(x), torch.ones_like(weight)))
    return now


IDS = torch.tensor([1, 2, 0])


def leaf(dtype=torch.bfloat16):
    return torch.randn(5, 8).to(dtype).requires_grad_()


def loss(w, x=None):
    return vocab.head_loss(torch.ones(3, 8).bfloat16() if x is None else x, w, IDS)


def refused(value, *inputs):
    with pytest.raises(RuntimeError, match="still alive"):
        torch.autograd.grad(value, inputs)


def test_a_graph_of_another_stream_is_remembered_behind_later_ones(place):
    w = leaf()
    kept = loss(w)
    loss(w)                                                            # dropped at once: an evaluation, a warm-up
    place.stream, place.capturing = 7, True
    refused(loss(w), w)
    place.capturing = False
    later = loss(w)                                                    # alive, made on the stream of the capture
    place.capturing = True
    refused(loss(w), w)
    del kept
    refused(loss(w), w)                                                # (the leaf's node is kept alive by the later graph)
    del later
    torch.autograd.grad(loss(w), w)


def test_a_table_at_both_ends_of_a_captured_step(place):
    table = leaf()
    kept = vocab.embed(IDS, table)
    place.stream, place.capturing = 7, True
    refused(loss(table, vocab.embed(IDS, table)), table)
    value = loss(table, vocab.embed(IDS, table))
    del kept
    refused(value, table)
    del value
    torch.autograd.grad(loss(table, vocab.embed(IDS, table)), table)


def test_a_leaf_behind_a_cast(place):
    """A master copy in fp32, cast for the operator."""
    w = leaf(torch.float32)
    kept = loss(w.bfloat16())
    place.stream, place.capturing = 7, True
    refused(loss(w.bfloat16()), w)
    del kept
    torch.autograd.grad(loss(w.bfloat16()), w)


def test_the_same_stream_and_eager_passes_go_through(place):
    w = leaf()
    kept = loss(w)
    place.stream = 7
    torch.autograd.grad(loss(w), w)                                    # eager: torch waits
    del kept
    kept = loss(w)
    place.capturing = True
    torch.autograd.grad(loss(w), w)
    assert kept.requires_grad


def test_nothing_is_left_behind_in_a_leaf(place):
    """Tensors with weak references cannot be swapped, which Module.to() and load_state_dict() do where torch is told so."""
    w = torch.nn.Parameter(leaf().detach())
    loss(w)
    vocab.embed(IDS, w)
    gc.collect()
    torch.utils.swap_tensors(w, torch.nn.Parameter(leaf().detach()))
    torch.autograd.grad(loss(w), w)
