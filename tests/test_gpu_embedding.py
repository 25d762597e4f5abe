"""GPU tests of the embedding and its gradient, against the plain 64-bit form.

Bounds.  The lookup is one float32 product rounded once more: half a step of the type, and 2^-24 of the value before it.
The gradient adds an index's rows in float32: a chunk of at most 64 rows one after the other, a run's pieces dealt to 32
threads (at most ``pieces / 32`` each, here below 40), the 32 sums in order, one product: fewer than 140 roundings, so
``140 * 2^-24`` of the sum of magnitudes, and half a step."""
import pytest
import torch

from oracle import rows_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def half_step(value, dtype):
    info = torch.finfo(dtype)
    return value.abs().clamp_min(info.tiny) * info.eps / 2


def run(idx, table, dy, scale=1.0, pad=None):
    from flexgemm_b200.ops.embedding import sparse_embedding
    t = table.to(DEV).requires_grad_(True)
    out = sparse_embedding(idx.to(DEV), t, scale=scale, padding_idx=pad)
    (g,) = torch.autograd.grad(out, [t], dy.to(DEV))
    return out, g


def check(idx, table, dy, scale=1.0, pad=None):
    out, g = run(idx, table, dy, scale, pad)
    t = table.dtype
    want = orc.embedding(idx, table, scale)
    assert out.shape == want.shape and out.dtype == t
    assert ((out.cpu().double() - want).abs() <= half_step(want, t) + 2.0 ** -23 * want.abs()).all()
    if scale == 1.0:
        assert torch.equal(out.cpu(), table[idx.long()])
    want, size = orc.embedding_grad(idx, dy, table.shape[0], scale, pad)
    bound = half_step(want, t) + 140 * 2.0 ** -24 * size * (1 + torch.finfo(t).eps)
    assert ((g.cpu().double() - want).abs() <= bound).all()
    return out, g


def problem(n, V, C, dtype, seed=0, spread=None):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, V, (n,), generator=g)
    if spread is not None:   # a share of the positions all hold one index
        idx[torch.rand(n, generator=g) < spread] = V // 3
    return idx, torch.randn(V, C, generator=g).to(dtype), torch.randn(n, C, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V,C,spread", [(1, 1, 8, None), (1, 500, 16, None), (2, 3, 1, None), (33, 7, 3, None), (300, 1, 64, None), (1000, 5000, 12, None),
                                          (5000, 40, 20, 0.5), (20000, 3000, 64, 0.3), (3000, 600, 2056, None), (9000, 70000, 36, 0.9), (4097, 512, 100, 1.0),
                                          (63, 511, 256, None), (64, 513, 256, 0.7)])
def test_matches_plain_form(n, V, C, spread, dtype):
    idx, table, dy = problem(n, V, C, dtype, seed=n + C, spread=spread)
    check(idx.int(), table, dy)
    check(idx, table, dy, scale=C ** 0.5, pad=V // 3)


def test_shapes_and_float_scale():
    idx, table, dy = problem(60, 30, 16, torch.float16, seed=1)
    flat, g = check(idx, table, dy, scale=0.3)
    out, g2 = run(idx.view(3, 4, 5), table, dy.view(3, 4, 5, 16), scale=0.3)
    assert out.shape == (3, 4, 5, 16) and torch.equal(out.view(60, 16), flat) and torch.equal(g, g2)
    from flexgemm_b200.ops.embedding import sparse_embedding
    one = sparse_embedding(idx[0].to(DEV), table.to(DEV), scale=0.3)
    assert one.shape == (16,) and torch.equal(one, flat[0])


def test_long_runs():
    """Runs that end at, just before and just behind the ends of chunks, sorted and in reverse."""
    lengths = [7, 8, 9, 16, 15, 1, 63, 64, 65, 128, 1, 1, 300, 8, 8, 8]
    idx = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    _, table, dy = problem(idx.numel(), len(lengths) + 2, 64, torch.float32, seed=2)
    check(idx, table, dy)
    check(idx.flip(0), table, dy)
    check(idx, table, dy, pad=12)


def test_one_index_at_every_position():
    idx = torch.full((300000,), 5)
    _, table, dy = problem(300000, 9, 8, torch.float32, seed=3)
    # pieces of 8 to 64 rows: at most 300000 / 8 / 32 = 1172 of them a thread, so the chain is 1172 + 64 + 32 + 2 roundings
    out, g = run(idx, table, dy)
    want, size = orc.embedding_grad(idx, dy, 9, 1.0)
    assert ((g.cpu().double() - want).abs() <= 1270 * 2.0 ** -24 * size).all() and torch.equal(out.cpu(), table[idx])


def test_repeated_calls_are_equal():
    idx, table, dy = problem(50000, 300, 32, torch.float32, seed=4, spread=0.4)
    first = run(idx, table, dy)
    for _ in range(4):
        again = run(idx, table, dy)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_special_values_pass():
    table = torch.tensor([[float("nan"), float("inf"), -float("inf"), -0.0], [1.0, 2.0, 3.0, 4.0]], dtype=torch.float16)
    from flexgemm_b200.ops.embedding import sparse_embedding
    out = sparse_embedding(torch.tensor([0, 1, 0], device=DEV), table.to(DEV)).cpu()
    assert torch.equal(out.view(torch.int16), table[[0, 1, 0]].view(torch.int16))
    dy = torch.ones(3, 4, dtype=torch.float16)
    dy[0] = float("nan")
    _, g = run(torch.tensor([0, 1, 1]), table, dy)
    assert torch.isnan(g[0]).all() and torch.equal(g[1].cpu(), torch.full((4,), 2.0, dtype=torch.float16))
    _, g = run(torch.tensor([0, 1, 1]), table, dy, pad=0)
    assert not g[0].any()


def test_index_beyond_the_table_raises_later():
    from flexgemm_b200.kernels import cuda as K
    from flexgemm_b200.ops.embedding import sparse_embedding
    table = torch.randn(10, 8, device=DEV)
    for bad in (10, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40):
        idx = torch.tensor([1, bad, 3], device=DEV)
        if abs(bad) < 2 ** 31:
            idx = idx.int()
        out = sparse_embedding(idx, table)
        torch.cuda.synchronize()
        assert torch.equal(out[[0, 2]], table[[1, 3]]) and not out[1].any()
        with pytest.raises(RuntimeError, match="index"):
            K.check_status(DEV)
    sparse_embedding(torch.tensor([1], device=DEV), table)
    torch.cuda.synchronize()
    K.check_status(DEV)


def test_streams_and_capture():
    from flexgemm_b200.ops.embedding import sparse_embedding
    idx, table, dy = problem(5000, 300, 32, torch.bfloat16, seed=5, spread=0.2)
    want = run(idx, table, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(idx, table, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    i, t, d = idx.to(DEV), table.to(DEV).requires_grad_(True), dy.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_embedding(i, t, scale=2.0)
        (g,) = torch.autograd.grad(out, [t], d)
    for seed in (6, 7):
        new = problem(5000, 300, 32, torch.bfloat16, seed=seed, spread=0.5)[0]
        i.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        again = run(new, table, dy, scale=2.0)
        assert torch.equal(out, again[0]) and torch.equal(g, again[1])


def test_layouts():
    idx, table, dy = problem(200, 50, 24, torch.float16, seed=8)
    want = run(idx, table, dy)
    wide = torch.zeros(50, 31, dtype=torch.float16)
    wide[:, 3:27] = table
    from flexgemm_b200.ops.embedding import sparse_embedding
    leaf = wide.to(DEV).requires_grad_(True)
    out = sparse_embedding(torch.stack([idx, idx], 1).to(DEV)[:, 0], leaf[:, 3:27])
    (g,) = torch.autograd.grad(out, [leaf], dy.to(DEV))
    assert torch.equal(out, want[0]) and torch.equal(g[:, 3:27], want[1]) and not g[:, :3].any()
    t = table.to(DEV).requires_grad_(True)
    sparse_embedding(idx.to(DEV), t).sum().backward()
    assert torch.equal(t.grad, run(idx, table, torch.ones_like(dy))[1])


def test_gradient_against_differences():
    """The call is linear in the table: a difference of two calls is exact up to their roundings."""
    from flexgemm_b200.ops.embedding import sparse_embedding
    idx, table, dy = problem(500, 40, 16, torch.float32, seed=9)
    _, g = run(idx, table, dy, scale=3.0)
    v = torch.randn(table.shape, generator=torch.Generator().manual_seed(10))
    loss = [(sparse_embedding(idx.to(DEV), (table + s * v).to(DEV), scale=3.0).double() * dy.to(DEV).double()).sum().item() for s in (1, -1)]
    want = (g.double() * v.to(DEV).double()).sum().item()
    size = (3 * (table.abs() + v.abs())[idx].double() * dy.abs().double()).sum().item()
    assert abs((loss[0] - loss[1]) / 2 - want) <= 150 * 2.0 ** -24 * size


def test_no_indices():
    from flexgemm_b200.ops.embedding import sparse_embedding
    t = torch.randn(4, 8, device=DEV, requires_grad=True)
    out = sparse_embedding(torch.zeros(0, 3, dtype=torch.int32, device=DEV), t)
    out.sum().backward()
    assert out.shape == (0, 3, 8) and t.grad.shape == (4, 8) and not t.grad.any()
