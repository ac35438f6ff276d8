"""Head loss: how many bits its gradients keep (needs a B200).  The bounds are those of the formulas in 64 bits; a rounding to bf16 is off by half a step at
most, 2^-8 of the value."""
import pytest
import torch

import cobalt_b200 as cb

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("n,V,H", [(1, 1000, 8), (1, 4099, 64), (2, 700, 16), (5, 3001, 8), (32, 2000, 8), (33, 513, 16), (63, 260, 8), (64, 300, 8)])
def test_gradients_of_few_tokens_round_their_results_alone(n, V, H):
    """Up to 64 tokens the gradient of the logits goes into both products as two bf16 values: 2^-8 of it, and 2^-8 of the rest, so 2^-16.  A logit is off by
    (2^-15.9 + 2^-24) of the sum of its magnitudes S (the tensor core's cuts, see test_head_loss_gpu.py), a loss or a normaliser by twice that and a few
    fp32 roundings, a probability by both of them.  The products cut 17 / 16 * 2^-25 of the magnitudes for each of their columns, twice as many as there
    are tokens or rows; what is left is the result's own rounding.  (Rounded once, d alone would be off by as much as the result.)"""
    g = gen(n + V + H)
    x = torch.randn(n, H, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, H, generator=g, device="cuda") * H ** -0.5).bfloat16()
    t = torch.randint(0, V, (n,), generator=g, device="cuda")
    f = torch.rand(n, generator=g, device="cuda") + 0.5
    xd, wd = x.double(), w.double()
    l = xd @ wd.T
    lse = torch.logsumexp(l, 1, keepdim=True)
    off = (2.0 ** -15.9 + 2.0 ** -24) * (xd.abs() @ wd.abs().T).amax(1, keepdim=True)
    tol = 2 * off + 2.0 ** -21 + 2.0 ** -22 * (l.abs().amax(1, keepdim=True) * 2 + lse.abs() + 1)
    p = torch.exp(l - lse)
    d = p.clone()
    d[torch.arange(n), t] -= 1.0
    size = d.abs() * f.double()[:, None]
    err = (d.abs() * 2.0 ** -16 * 1.01 + p * (2 * tol + 2.0 ** -20) + 2.0 ** -22) * f.double()[:, None]
    d = d * f.double()[:, None]
    cut = 17 / 16 * 2.0 ** -25
    _, dx, dw = cb.head_loss_and_grad(x, w, t, "none", f)
    for got, want, slack in ((dx, d @ wd, err @ wd.abs() + 2 * V * cut * (size @ wd.abs())), (dw, d.T @ xd, err.T @ xd.abs() + 2 * n * cut * (size.T @ xd.abs()))):
        worst = ((got.double() - want).abs() - 1.01 * slack - want.abs() * 2.0 ** -8 - 1e-38).max()
        assert float(worst) <= 0, float(worst)


def long_sum(size, columns):
    """Bound of a sum of ``columns`` products of magnitudes ``size`` in all, cut in the tensor core over 4096 columns at a time (17 / 16 * 2^-25 of
    the magnitudes for each column) and added up in fp32"""
    return size * (4096 * 17 / 16 * 2.0 ** -25 + columns / 4096 * 2.0 ** -24)


def test_the_heads_gradient_over_very_many_tokens():
    """2^19 tokens, the first half pulling one way and the second the other: what is left is small against what was added up.  The rows of the head are zero, so
    probabilities are 1/2 and d = +-1/2, without an error."""
    n, H = 1 << 19, 64
    x = torch.randn(n, H, generator=gen(1), device="cuda").abs().bfloat16()
    w = torch.zeros(2, H, dtype=torch.bfloat16, device="cuda")
    t = (torch.arange(n, device="cuda") >= n // 2).long()
    _, _, dw = cb.head_loss_and_grad(x, w, t, "sum", need_x=False)
    half = 0.5 * x.double()
    want = half[n // 2:].sum(0) - half[:n // 2].sum(0)
    want = torch.stack([want, -want])
    worst = ((dw.double() - want).abs() - long_sum(half.sum(0), n) - want.abs() * 2.0 ** -8).max()
    assert float(worst) <= 0, float(worst)


@pytest.mark.parametrize("n,V,H", [(3, 1 << 18, 19200), (256, 1 << 19, 10240)])
def test_the_hidden_gradient_over_a_large_vocabulary(n, V, H):
    """x = 0: every probability is 1 / V, a power of two, so dx is the mean of the rows less the target's, which is made to be that mean as far as bf16 has it.  The rounding
    of 1 / V - 1 costs at most 1 / V."""
    x = torch.zeros(n, H, dtype=torch.bfloat16, device="cuda")
    w = torch.randn(V, H, generator=gen(2), device="cuda", dtype=torch.bfloat16).abs_()
    mean = sum(w[i:i + 4096].double().sum(0) for i in range(0, V, 4096)) / V
    w[V - 1] = mean.bfloat16()
    mean = sum(w[i:i + 4096].double().sum(0) for i in range(0, V, 4096)) / V
    t = torch.full((n,), V - 1, device="cuda")
    _, dx, _ = cb.head_loss_and_grad(x, w, t, "sum")
    want = mean - w[V - 1].double()
    slack = long_sum(mean + w[V - 1].double(), V) + w[V - 1].double() / V + want.abs() * 2.0 ** -8
    worst = ((dx.double() - want).abs() - slack).max()
    assert float(worst) <= 0, float(worst)


def against_differences(n, which):
    """(difference of the losses of two ends, the gradient's product with what is between them, bound).  Every value of one operand moves by one step of its
    grid the way the gradient points, so that nothing cancels; the grid is one of multiples that bf16 holds, middle and ends alike."""
    V, H = 500, 256
    g = gen(100 + n)
    x = (torch.randn(n, H, generator=g, device="cuda") * 64).round().clamp(-200, 200) / 64
    w = (torch.randn(V, H, generator=g, device="cuda") * 64).round().clamp(-200, 200) / 1024
    t = torch.randint(0, V, (n,), generator=g, device="cuda")
    step = 1 / 64 if which == 0 else 1 / 1024
    x, w = x.bfloat16(), w.bfloat16()
    _, dx, dw = cb.head_loss_and_grad(x, w, t, "sum")
    move = torch.sign((dx, dw)[which].double()) * step
    ends = []
    for s in (-1, 1):
        moved = ((x, w)[which].double() + s * move)
        assert torch.equal(moved.bfloat16().double(), moved)
        ends.append(cb.head_loss(*((moved.bfloat16(), w) if which == 0 else (x, moved.bfloat16())), t, "none").double().sum())
    xd, wd = x.double(), w.double()
    l = xd @ wd.T
    dl = move @ wd.T if which == 0 else xd @ move.T
    reach = dl.amax(1) - dl.amin(1)
    # what a central difference leaves out: a third cumulant of dl, at most sqrt(3) / 18 of its reach cubed, over 6, on either side, and a half more for what it
    # changes along the way (reaches are far below 1)
    left_out = (2 / 6 * 3 ** 0.5 / 18 * 1.5 * reach ** 3).sum()
    # a loss: logits (see test_head_loss_gpu.py), exponentials, and the roundings of fp32
    off = (2.0 ** -15.9 + 2.0 ** -24) * ((xd.abs() + move.abs() if which == 0 else xd.abs()) @ (wd.abs() if which == 0 else wd.abs() + move.abs()).T).amax(1)
    noise = 2 * (2 * off + 2.0 ** -21 + 2.0 ** -22 * (2 * l.abs().amax(1) + 10)).sum()
    # the gradient: d and the result rounded to bf16, 2^-8 each, and what the logits' error does to d (p times twice that, and at most 2 off of a sum over p)
    p = torch.softmax(l, 1)
    d = p.clone()
    d[torch.arange(n), t] -= 1.0
    err = d.abs() * 2.0 ** -8 + p * (4 * off[:, None] + 2.0 ** -19)
    grad = (dx, dw)[which].double()
    slack = (err @ wd.abs() if which == 0 else err.T @ xd.abs()) + grad.abs() * 2.0 ** -8
    want = 2 * (grad * move).sum()
    return float(ends[1] - ends[0]), float(want), float(left_out + noise + 2 * (slack * move.abs()).sum()), float(reach.max())


@pytest.mark.parametrize("n", [48, 100, 300])
@pytest.mark.parametrize("which", [0, 1])
def test_gradients_against_differences_along_themselves(n, which):
    """A gradient that was zero, negated or off by half would not pass."""
    got, want, bound, reach = against_differences(n, which)
    assert abs(got - want) <= bound, (got, want, bound)
    assert want > 0 and bound < 0.2 * want and reach < 1, (want, bound, reach)
