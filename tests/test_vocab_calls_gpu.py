"""Embedding and head loss: calls that must not pass without a word (needs a B200)."""
import pytest
import torch

import cobalt_b200 as cb

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
