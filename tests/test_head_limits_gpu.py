"""Head loss at the ends of what its entries take: hidden columns, tokens, vocabulary (needs a B200).  Bounds as in test_head_loss_gpu.py."""
import pytest
import torch

import cobalt_b200 as cb
from test_head_loss_gpu import Exact, inputs, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,V,H", [(3, 300, 65536), (70, 200, 65528), (200, 300, 65536), (1 << 20, 3, 8), (5, 1 << 22, 8), (130, (1 << 22) + 1, 8)])
def test_largest_sizes(n, V, H):
    x, w, t = inputs(n, V, H, 1, 0.2, 2.0)
    e = Exact(x, w, t, torch.ones(n, device="cuda"))
    loss, dx, dw = cb.head_loss_and_grad(x, w, t, "none")
    near(loss, e.loss, e.tol)
    near(dx, e.dx, e.dx_tol)
    near(dw, e.dw, e.dw_tol)
    assert cb.head_loss_status() == 0


def test_one_more_is_refused():
    for n, V, H in ((2, 3, 65544), ((1 << 20) + 1, 3, 8)):
        x, w = torch.zeros(n, H, dtype=torch.bfloat16, device="cuda"), torch.zeros(V, H, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(cb._lib.CobaltError):
            cb.head_loss(x, w, torch.zeros(n, dtype=torch.int64, device="cuda"))
