"""Embedding lookup and its gradient against fp64 (needs a B200).

Bounds.  Lookup: the fp32 product is rounded once (2^-24), the result once more (eps / 2 of its type, half its smallest step near zero).
Gradient: m rows are added in fp32 one after another and in partial sums (at most m + 40 additions of at most 2^-24 of the sum of
magnitudes each), scaled (2^-24) and rounded once."""
import math

import pytest
import torch

import cobalt_b200 as cb

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def some_ids(n, V, seed, kind="some"):
    g = gen(seed)
    if kind == "one":                                                  # all the same
        return torch.full((n,), V // 2, device="cuda")
    if kind == "none":
        return torch.full((n,), -1, device="cuda")
    ids = torch.randint(-1, V + 1, (n,), generator=g, device="cuda")
    if kind == "few":                                                  # most of them a few tokens
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.8, ids % 3, ids)
    if n > 2:
        ids[-1], ids[0] = 2 ** 40, -2 ** 63                            # far outside
    return ids


def lookup(ids, table, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    return torch.where(ok[..., None], table.double()[torch.where(ok, ids, 0)] * scale, 0.0)


def rounding(t, dtype):
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2 + 2.0 ** -24) + info.smallest_normal * info.eps / 2


def check_grad(got, grad, ids, V, scale):
    ok = (ids >= 0) & (ids < V)
    flat, rows = ids[ok], grad[ok].double() * scale
    want = torch.zeros(V, grad.shape[-1], dtype=torch.float64, device="cuda").index_add_(0, flat, rows)
    size = torch.zeros_like(want).index_add_(0, flat, rows.abs())
    m = torch.zeros(V, 1, dtype=torch.float64, device="cuda").index_add_(0, flat, torch.ones(len(flat), 1, dtype=torch.float64, device="cuda"))
    assert got.shape == want.shape and got.dtype is grad.dtype
    worst = ((got.double() - want).abs() - rounding(want, grad.dtype) - (m + 40) * 2.0 ** -24 * size * (1 + torch.finfo(grad.dtype).eps)).max()
    assert float(worst) <= 0, float(worst)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,H,scale", [(1, 1, 1, 1.0), (1, 32000, 4096, 1.0), (3, 7, 8, 73.5), (65, 1000, 1001, -0.37), (777, 300, 64, 1.0), (2000, 5000, 5376, 73.5)])
def test_lookup(n, V, H, scale, dtype):
    table = torch.randn(V, H, generator=gen(n + H), device="cuda").to(dtype)
    ids = some_ids(n, V, n)
    got = cb.embed(ids, table, scale)
    want = lookup(ids, table, torch.tensor(scale).double().item() if scale == 1.0 else float(torch.tensor(scale, dtype=torch.float32)))
    assert got.shape == (n, H) and got.dtype is dtype
    assert bool(((got.double() - want).abs() <= rounding(want, dtype)).all())
    if scale == 1.0:
        assert torch.equal(got, want.to(dtype))


def test_lookup_of_every_bit_pattern():
    """Scale 1 copies bits (NaN, infinities, negative zero, subnormals); another scale is torch's fp32 product."""
    for dtype in (torch.bfloat16, torch.float16):
        table = torch.arange(65536, device="cuda").to(torch.int16).view(dtype).view(64, 1024)
        ids = torch.arange(64, device="cuda")
        assert torch.equal(cb.embed(ids, table).view(torch.int16), table.view(torch.int16))
        got, want = cb.embed(ids, table, 1.7), (table.float() * 1.7).to(dtype)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(got.isnan(), want.isnan())


def test_lookup_strides_shapes_and_results():
    big = torch.randn(50, 200, generator=gen(1), device="cuda").bfloat16()
    ids = some_ids(24, 50, 2).view(2, 3, 4)
    for table in (big[:, 8:136], big[:, 3:100], big[::2, :64], big.t()[:64].t(), big[:1, :64].expand(50, 64), big[:, ::2]):
        want = cb.embed(ids, table.contiguous(), 2.0)
        assert want.shape == (2, 3, 4, table.shape[1]) and torch.equal(cb.embed(ids, table, 2.0), want)
        assert torch.equal(cb.embed(ids.transpose(0, 2), table, 2.0), want.transpose(0, 2))
        out = torch.full_like(want, 9.0)
        assert cb.embed(ids, table, 2.0, out=out) is out and torch.equal(out, want)
    odd = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 3, 4, 64)          # a result on a 2-byte boundary
    assert torch.equal(cb.embed(ids, big[:, :64], out=odd), cb.embed(ids, big[:, :64]))
    assert cb.embed(ids[:0], big).shape == (0, 3, 4, 200)
    assert cb.embed(torch.tensor(7, device="cuda"), big).shape == (200,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,H,kind", [(1, 1, 1, "some"), (1, 5, 8, "some"), (5, 2, 16, "none"), (31, 9, 64, "one"), (32, 40, 72, "few"), (33, 40, 65, "few"),
                                        (64, 3, 1001, "one"), (100, 30000, 128, "some"), (2048, 100, 40, "few"), (2049, 100, 40, "few"), (4096, 7, 24, "one"), (6143, 500, 24, "few"), (6144, 9, 40, "some"), (6145, 500, 24, "few"),
                                        (7000, 5000, 264, "few"), (20001, 333, 33, "few"),
                                        (32769, 40000, 16, "some"), (600001, 5000, 8, "few"),
                                        (8388611, 100000, 2, "some")])
def test_gradient(n, V, H, kind, dtype):
    ids = some_ids(n, V, n + 1, kind)
    grad = torch.randn(n, H, generator=gen(H), device="cuda").to(dtype)
    got = cb.embed_grad(grad, ids, V, 1.5)
    check_grad(got, grad, ids, V, 1.5)
    assert torch.equal(got, cb.embed_grad(grad, ids, V, 1.5))          # the same bits


def test_gradient_of_many_tokens_of_one_row():
    """Runs that cross very many tiles, at both ends of the sorted tokens, and rows that nobody looks up."""
    n, V, H = 70000, 1000, 128
    ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    ids[::7], ids[5::31] = V - 1, -1
    ids[100:200] = torch.arange(100, device="cuda") + 50
    grad = torch.randn(n, H, generator=gen(3), device="cuda").bfloat16()
    got = cb.embed_grad(grad, ids, V)
    check_grad(got, grad, ids, V, 1.0)
    assert not bool(got[200:V - 1].any())


def test_rows_without_a_place_are_not_read():
    ids = torch.tensor([3, -1, 9, 3, 1 << 33], device="cuda")
    grad = torch.ones(5, 16, device="cuda").bfloat16()
    grad[1], grad[2], grad[4] = math.nan, math.inf, math.nan           # 9 is outside a table of 9 rows
    got = cb.embed_grad(grad, ids, 9)
    want = torch.zeros(9, 16, device="cuda").bfloat16()
    want[3] = 2.0
    assert torch.equal(got, want)
    grad[0, 5] = math.nan                                              # one that counts reaches its row and column alone
    got = cb.embed_grad(grad, ids, 9)
    assert bool(got[3, 5].isnan()) and int(got.isnan().sum()) == 1


def test_gradient_strides():
    ids = some_ids(40, 30, 5).view(5, 8)
    base = torch.randn(5, 16, 200, generator=gen(6), device="cuda").bfloat16()
    for grad in (base[:, ::2, 8:72], base[:, :8, 1:66], base[:1, :8, :64].expand(5, 8, 64), base[:, :1, :64].expand(5, 8, 64), base[:, :8, ::2], base[0, 0, 0].expand(5, 8, 64)):
        assert torch.equal(cb.embed_grad(grad, ids, 30), cb.embed_grad(grad.contiguous(), ids, 30))
    assert not bool(cb.embed_grad(base[:0, :8], ids[:0], 4).any())


def test_autograd_and_differences():
    """The loss sum(y * c) is linear in the table: what autograd says is the difference of two losses, to the roundings of the two lookups."""
    V, H = 40, 64
    ids = some_ids(60, V, 8, "few")
    table = torch.randn(V, H, generator=gen(9), device="cuda").requires_grad_()
    c = torch.randn(60, H, generator=gen(10), device="cuda")
    y = cb.embed(ids, table, 3.0)
    (y * c).sum().backward()
    check_grad(table.grad, c, ids, V, 3.0)
    step = torch.randn(V, H, generator=gen(11), device="cuda")
    with torch.no_grad():
        moved = table + step
        far = ((cb.embed(ids, moved, 3.0).double() - y.double()) * c.double()).sum()
        along = (table.grad.double() * (moved.double() - table.double())).sum()
        noise = 2.0 ** -23 * ((lookup(ids, moved, 3.0).abs() + lookup(ids, table.detach(), 3.0).abs()) * c.abs()).sum() + \
            100 * 2.0 ** -24 * (cb.embed_grad(c.abs(), ids, V, 3.0).double() * step.double().abs()).sum()
    assert abs(float(far - along)) <= float(noise)
    with torch.no_grad():
        assert not cb.embed(ids, table).requires_grad


def test_offsets_beyond_32_bits():
    V, H = 600000, 4096                                                # 2.4 G values
    table = torch.zeros(V, H, dtype=torch.bfloat16, device="cuda")
    table[-3:] = torch.randn(3, H, generator=gen(12), device="cuda").bfloat16()
    ids = torch.tensor([V - 1, V - 3, 0, V - 1, V], device="cuda")
    y = cb.embed(ids, table)
    assert torch.equal(y[:2], table[[V - 1, V - 3]]) and torch.equal(y[3], y[0]) and not bool(y[4].any())
    d = cb.embed_grad(y, ids, V)
    assert torch.equal(d[V - 1].float(), (2 * y[0].float()).bfloat16().float()) and torch.equal(d[V - 3], y[1]) and not bool(d[1:V - 3].any()) and not bool(d[V - 2].any())


def test_streams_and_graphs():
    """Two streams at once, and a captured lookup with its gradient that follows new ids when replayed."""
    V, H, n = 500, 256, 3000
    table = torch.randn(V, H, generator=gen(13), device="cuda").bfloat16().requires_grad_()
    ids, grad = some_ids(n, V, 14, "few"), torch.randn(n, H, generator=gen(15), device="cuda").bfloat16()
    side = [torch.cuda.Stream() for _ in range(2)]
    want = cb.embed_grad(grad, ids, V)
    torch.cuda.synchronize()
    got = []
    for s in side * 3:
        with torch.cuda.stream(s):
            got.append(cb.embed_grad(grad, ids, V))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    kept = cb.embed(some_ids(n, V, 1), table)                          # an eager graph of the same leaf: its gradient is captured without one
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        y = cb.embed(ids, table, 2.0)
        with pytest.raises(RuntimeError, match="still alive"):
            torch.autograd.grad(y, table, grad)
    del y
    plain = torch.cuda.CUDAGraph()
    with torch.cuda.graph(plain):
        d0 = cb.embed_grad(grad, ids, V, 2.0)
    kept.sum().backward()
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cb.embed(ids, table, 2.0)
        (d,) = torch.autograd.grad(y, table, grad)
    for seed in (20, 21):
        ids.copy_(some_ids(n, V, seed, "few"))
        graph.replay(), plain.replay()
        assert torch.equal(d0, d) and torch.equal(y, cb.embed(ids, table.detach(), 2.0)) and torch.equal(d, cb.embed_grad(grad, ids, V, 2.0))


def test_refusals():
    ids, table = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(5, 8, device="cuda")
    with pytest.raises(TypeError):
        cb.embed(ids.int(), table)
    with pytest.raises(TypeError):
        cb.embed(ids, table.double())
    with pytest.raises(ValueError):
        cb.embed(ids.cpu(), table)
    with pytest.raises(ValueError):
        cb.embed(ids, table[0])
    with pytest.raises(ValueError):
        cb.embed(ids, table, out=torch.zeros(3, 8, device="cuda").t().contiguous().t())
    with pytest.raises(ValueError):
        cb.embed(ids, table, out=torch.zeros(2, 8, device="cuda"))
    with pytest.raises(RuntimeError):
        cb.embed(ids, table.clone().requires_grad_(), out=torch.zeros(3, 8, device="cuda"))
    for bad in (lambda: cb.embed_grad(table, ids, 5), lambda: cb.embed_grad(table[:3], ids, 0), lambda: cb.embed_grad(table[:3], ids.cpu(), 5)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        cb.embed_grad(table[:3].int(), ids, 5)
    wide = table[:1, :1].expand(3, 2 ** 32 + 8)                        # (a width of 8 in 32 bits)
    with pytest.raises(ValueError):
        cb.embed(ids, wide)
    with pytest.raises(ValueError):
        cb.embed_grad(wide, ids, 5)


def test_a_table_that_was_used_can_be_copied_and_saved(tmp_path):
    import copy
    table = torch.nn.Parameter(torch.randn(5, 8, device="cuda"))
    y = cb.embed(torch.tensor([1, 2], device="cuda"), table)
    assert torch.equal(copy.deepcopy(table), table)
    torch.save(table, tmp_path / "t.pt")
    y.sum().backward()
    assert float(table.grad.sum()) == 16
