"""4-bit KV cache: what asks for a gradient is refused, whichever argument it is (no GPU needed)."""
import pytest
import torch

from cobalt_b200 import KVCache4


def test_weights_and_results_that_require_a_gradient_are_refused():
    c = KVCache4(1, 1, 40, 64, device="cpu")
    weight = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16))
    freq = torch.ones(32, requires_grad=True)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    asks = ((lambda: c._weight("k_norm", weight, torch.bfloat16, 64)), (lambda: c._weight("inv_freq", freq, torch.float32, 32)),
            (lambda: c._result("out", torch.zeros_like(q, requires_grad=True), q)))
    for ask in asks:
        with pytest.raises(RuntimeError, match="requires a gradient"):
            ask()
        with torch.no_grad():
            ask()
    c._weight("k_norm", weight.detach(), torch.bfloat16, 64)
