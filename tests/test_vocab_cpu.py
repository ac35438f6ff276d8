"""Embedding lookup and head loss: what is refused, in Python and at the C entries (no GPU needed)."""
import pytest
import torch

import cobalt_b200 as cb
from cobalt_b200 import _lib, vocab

A = 4096                                                               # an address that is never read: every call below ends before a launch


def test_tensors_off_the_gpu_are_refused():
    ids, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    for call in (lambda: cb.embed(ids, table), lambda: cb.embed_grad(torch.zeros(3, 8), ids, 5),
                 lambda: cb.head_loss(torch.zeros(3, 8).bfloat16(), torch.zeros(5, 8).bfloat16(), ids)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_rows_are_taken_where_they_lie_or_copied():
    m = torch.arange(7 * 24, dtype=torch.float32).view(7, 24).bfloat16()
    assert vocab._matrix("x", m, 24, 8)[0].data_ptr() == m.data_ptr()
    for odd in (m[:, 1:17], m.t()[:, :7].t()[:, :16].flip(1), m[:, ::2][:, :8], m[:1, :16].expand(3, 16), m.as_strided((5, 16), (12, 1))):
        width = odd.shape[1]
        got, apart = vocab._matrix("x", odd, width, 8)
        assert torch.equal(got, odd) and got.stride(1) == 1 and got.data_ptr() % 16 == 0 and apart % 8 == 0 and apart >= width
    part = m[:, 8:24]                                                  # a slice on 16-byte boundaries stays where it is
    got, apart = vocab._matrix("x", part, 16, 8)
    assert got.data_ptr() == part.data_ptr() and apart == 24
    with pytest.raises(ValueError):
        vocab._matrix("x", m, 23)


def test_embedding_arguments_at_the_c_entry():
    L = _lib.load()
    good = dict(ids=A, n=4, table=A, ld=64, type=2, n_rows=10, width=64, scale=1.0, out=A, ld_out=64)
    bad = [dict(ids=None), dict(table=None), dict(out=None), dict(n=0), dict(n=-1), dict(type=3), dict(n_rows=0), dict(width=0), dict(ld=63), dict(ld_out=63),
           dict(ids=A + 4), dict(table=A + 1), dict(out=A + 1), dict(type=0, table=A + 2)]
    for change in bad:
        assert L.cobalt_embed(*{**good, **change}.values(), None) == -1, change
    wide = dict(width=(1 << 28) + 1, ld=1 << 29)
    assert L.cobalt_embed(*{**good, **wide, 'ld_out': 1 << 29}.values(), None) == -6
    good = dict(ids=A, n=4, grad=A, ld=64, type=2, n_rows=10, width=64, scale=1.0, out=A, scratch=A, bytes=1 << 30)
    bad = [(dict(ids=None), -1), (dict(grad=None), -1), (dict(out=None), -1), (dict(out=A + 8), -1), (dict(n=0), -1), (dict(type=-1), -1), (dict(n_rows=0), -1),
           (dict(ld=60), -1), (dict(grad=A + 1), -1), (dict(scratch=None), -2), (dict(scratch=A + 16), -2), (dict(bytes=100), -2), (dict(n=(1 << 24) + 1), -6),
           (dict(n_rows=1 << 31), -6), (wide, -6)]
    for change, rc in bad:
        assert L.cobalt_embed_grad(*{**good, **change}.values(), None) == rc, change
    assert L.cobalt_embed_grad_scratch_bytes(0, 64) == 0 and L.cobalt_embed_grad_scratch_bytes((1 << 24) + 1, 64) == 0
    assert 0 < L.cobalt_embed_grad_scratch_bytes(5, 64) < L.cobalt_embed_grad_scratch_bytes(5000, 64)


def test_head_arguments_at_the_c_entry():
    L = _lib.load()
    good = dict(x=A, ldx=64, w=A, ldw=64, targets=A, n=4, hidden=64, vocab=100, loss=A, stats=A, total=A, mean=1, scratch=A, bytes=1 << 30, status=A)
    bad = [(dict(x=None), -1), (dict(w=None), -1), (dict(targets=None), -1), (dict(loss=None), -1), (dict(x=A + 8), -1), (dict(w=A + 8), -1), (dict(ldx=60), -1),
           (dict(ldx=68), -1), (dict(ldw=56), -1), (dict(n=0), -1), (dict(hidden=0), -1), (dict(hidden=60), -1), (dict(vocab=0), -1), (dict(targets=A + 4), -1),
           (dict(loss=A + 2), -1), (dict(stats=A + 4), -1), (dict(total=A + 2), -1), (dict(status=A + 2), -1), (dict(n=(1 << 20) + 1), -6),
           (dict(hidden=(1 << 16) + 8, ldx=1 << 17, ldw=1 << 17), -6), (dict(vocab=1 << 31), -6), (dict(scratch=None), -2), (dict(scratch=A + 128), -2)]
    for change, rc in bad:
        assert L.cobalt_head_loss(*{**good, **change}.values(), None) == rc, change
    good = dict(x=A, ldx=64, w=A, ldw=64, targets=A, stats=A, grad=A, step=0, mean=1, n=4, hidden=64, vocab=100, dx=A, ld_dx=64, dw=A, ld_dw=64, scratch=A,
                bytes=1 << 30, status=None)
    bad = [(dict(x=None), -1), (dict(w=None), -1), (dict(targets=None), -1), (dict(stats=None), -1), (dict(grad=None), -1), (dict(dx=None, dw=None), -1),
           (dict(step=2), -1), (dict(step=-1), -1), (dict(dx=A + 8), -1), (dict(dw=A + 8), -1), (dict(ld_dx=56), -1), (dict(ld_dw=68), -1), (dict(hidden=4), -1),
           (dict(grad=A + 2), -1), (dict(status=A + 1), -1), (dict(vocab=1 << 31), -6), (dict(scratch=None), -2), (dict(scratch=A + 128), -2)]
    for change, rc in bad:
        assert L.cobalt_head_loss_grad(*{**good, **change}.values(), None) == rc, change
    assert L.cobalt_head_loss_scratch_bytes(4, 60, 100) == 0 and L.cobalt_head_loss_scratch_bytes(0, 64, 100) == 0
    assert L.cobalt_vocab_status(None, None) == -1
