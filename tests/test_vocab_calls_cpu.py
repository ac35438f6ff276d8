"""Embedding and head loss: checks of arguments that need no GPU."""
import torch

from cobalt_b200 import vocab


def test_which_tensors_share_memory():
    """The bytes from the first value to the last, whatever the strides."""
    m = torch.arange(600, dtype=torch.float32).view(30, 20)
    assert vocab._overlap(m, m) and vocab._overlap(m[3], m) and vocab._overlap(m[:10], m[9:]) and vocab._overlap(m[:, 3], m[29, 3:4])
    assert vocab._overlap(m[::2], m[1]) and vocab._overlap(m.t(), m[7:9]) and vocab._overlap(m.view(torch.int64)[3], m[3, 4:])
    assert vocab._overlap(m[:1, :1].expand(50, 60), m[0, :3]) and not vocab._overlap(m[:1, :1].expand(50, 60), m[0, 1:])
    assert not vocab._overlap(m[:10], m[10:]) and not vocab._overlap(m[5, :10], m[5, 10:]) and not vocab._overlap(m, m.clone()) and not vocab._overlap(m[:0], m)
    assert not vocab._overlap(m[:, 3], m[29, 4:])
