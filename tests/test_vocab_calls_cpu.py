"""Embedding and head loss: checks of arguments that need no GPU."""
from types import SimpleNamespace

import pytest
import torch

from cobalt_b200 import _lib, vocab
from cobalt_b200.decoder import CobaltDecoder


def test_which_tensors_share_memory():
    """The bytes from the first value to the last, whatever the strides."""
    m = torch.arange(600, dtype=torch.float32).view(30, 20)
    assert vocab._overlap(m, m) and vocab._overlap(m[3], m) and vocab._overlap(m[:10], m[9:]) and vocab._overlap(m[:, 3], m[29, 3:4])
    assert vocab._overlap(m[::2], m[1]) and vocab._overlap(m.t(), m[7:9]) and vocab._overlap(m.view(torch.int64)[3], m[3, 4:])
    assert vocab._overlap(m[:1, :1].expand(50, 60), m[0, :3]) and not vocab._overlap(m[:1, :1].expand(50, 60), m[0, 1:])
    assert not vocab._overlap(m[:10], m[10:]) and not vocab._overlap(m[5, :10], m[5, 10:]) and not vocab._overlap(m, m.clone()) and not vocab._overlap(m[:0], m)
    assert not vocab._overlap(m[:, 3], m[29, 4:])


def test_watched_lookup_at_the_c_entry():
    at = 4096                                                          # an address that is never read: every call ends before a launch
    good = dict(ids=at, n=4, table=at, ld=64, type=2, n_rows=10, width=64, scale=1.0, out=at, ld_out=64, status=at)
    for change in (dict(status=at + 2), dict(ids=None), dict(out=None), dict(n=0), dict(ld=63), dict(table=at + 1)):
        assert _lib.load().cobalt_embed_watched(*{**good, **change}.values(), None) == -1, change


def test_ids_beyond_the_vocabulary_in_a_decoder():
    """Host memory is looked at, the device's is not (its lookup tells); what was told is told once."""
    dec = SimpleNamespace(P={"model.embed_tokens.weight": torch.zeros(10, 4)}, id_status=torch.zeros(1, dtype=torch.int32), lin={}, prompt_status=torch.zeros(1, dtype=torch.int32),
                          att_fused=None, qkv=[], gate_up=[], o_f=[], down=[], head_f=None, reducer=None)
    CobaltDecoder._check_host_ids(dec, torch.tensor([[0, 9, -1]]))
    CobaltDecoder._check_host_ids(dec, torch.zeros(0, dtype=torch.int64))
    with pytest.raises(ValueError, match="token id 10 is outside the vocabulary of 10"):
        CobaltDecoder._check_host_ids(dec, torch.tensor([3, 10, 4], dtype=torch.int32))
    CobaltDecoder._check_looked_up(dec)
    for _ in range(2):
        assert CobaltDecoder.device_status(dec) == 0
        dec.id_status.fill_(8)
        assert CobaltDecoder.device_status(dec) == 8
    dec.id_status.fill_(8)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        CobaltDecoder._check_looked_up(dec)
    assert CobaltDecoder.device_status(dec) == 0


def test_a_decoder_tells_a_loss_that_gave_up_once():
    """The kernels write the word only while it is 0: it is cleared when it was told, so that the next one is told too.  (Set by hand: no wait is made to run out.)"""
    word = torch.zeros(1, dtype=torch.int32)
    dec = SimpleNamespace(score_status=word, lin={}, prompt_status=torch.zeros(1, dtype=torch.int32), att_fused=None, qkv=[], gate_up=[], o_f=[], down=[], head_f=None, reducer=None)
    for code in (2, 4):
        assert CobaltDecoder.device_status(dec) == 0
        word.fill_(code)
        assert CobaltDecoder.device_status(dec) == code and int(word) == 0
