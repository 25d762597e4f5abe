"""The embedding's gradient of few positions (up to 4096, in one launch), against the plain 64-bit form, and where it borders on
the way of many.

Bounds.  An index's rows are added in float32: at most 32 of a chunk one after the other, then at most 128 chunks, and one product:
fewer than 162 roundings of the sum of magnitudes, and half a step of the type.  (Of more positions: see test_gpu_embedding.)"""
import pytest
import torch

from oracle import rows_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def grad(idx, table, dy, scale=1.0, pad=None):
    from flexgemm_b200.ops.embedding import sparse_embedding
    t = table.to(DEV).requires_grad_(True)
    junk = torch.full(table.shape, float("nan"), dtype=table.dtype, device=DEV)   # what is not cleared shows
    out = sparse_embedding(idx.to(DEV), t, scale=scale, padding_idx=pad)
    del junk
    return torch.autograd.grad(out, [t], dy.to(DEV))[0]


def check(idx, table, dy, scale=1.0, pad=None):
    got = grad(idx, table, dy, scale, pad)
    want, size = orc.embedding_grad(idx, dy, table.shape[0], scale, pad)
    info = torch.finfo(table.dtype)
    bound = want.abs().clamp_min(info.tiny) * info.eps / 2 + 162 * 2.0 ** -24 * size * (1 + info.eps)
    assert got.shape == table.shape and got.dtype == table.dtype
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert torch.equal(got, grad(idx, table, dy, scale, pad))
    return got


def problem(n, V, C, dtype, seed, share=0.0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, V, (n,), generator=g)
    idx[torch.rand(n, generator=g) < share] = V - 1
    return idx, torch.randn(V, C, generator=g).to(dtype), torch.randn(n, C, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V,C,share", [(1, 1, 1, 0), (1, 3000, 24, 0), (7, 2, 8, 0), (31, 511, 6, 0.3), (32, 512, 33, 0), (513, 513, 20, 0.5), (1024, 9, 256, 0),
                                         (2048, 4096, 512, 0.9), (2049, 70, 40, 1.0), (4095, 262143, 4, 0.2), (4096, 262144, 4, 0.5), (4096, 5, 64, 0), (4096, 4096, 2048, 0.1),
                                         (4096, 1, 36, 0), (4097, 1, 36, 0), (300, 40, 1028, 0.4), (4000, 60000, 100, 0.05), (600, 300, 257, 0.1)])
def test_matches_plain_form(n, V, C, share, dtype):
    idx, table, dy = problem(n, V, C, dtype, seed=n + C, share=share)
    check(idx.int(), table, dy)
    check(idx, table, dy, scale=0.3, pad=V - 1)


@pytest.mark.parametrize("length", [1, 7, 8, 9, 31, 32, 33, 128, 1000])
def test_runs_of_one_length(length):
    """Runs that end at, before and behind the ends of chunks, in order and shuffled."""
    V = 4000 // length
    idx = torch.arange(V).repeat_interleave(length)
    _, table, dy = problem(idx.numel(), V, 36, torch.float32, seed=length)
    check(idx, table, dy)
    check(idx[torch.randperm(idx.numel(), generator=torch.Generator().manual_seed(1))], table, dy)


def test_order_of_addition():
    """Rows of an index are added in the order of their positions, whatever lies between them: 8 of them one after the other."""
    dy = torch.zeros(64, 4)
    idx = torch.arange(64)
    big = [1.0, 2.0 ** 24, 1.0, -2.0 ** 24, 1.0]
    idx[torch.tensor([3, 17, 20, 41, 63])] = 3
    dy[torch.tensor([3, 17, 20, 41, 63])] = torch.tensor(big).view(-1, 1)
    want = 0.0
    for v in big:
        want = (torch.tensor(want) + torch.tensor(v)).item()   # float32
    assert (grad(idx, torch.zeros(64, 4), dy)[3] == want).all()


def test_no_position_counts():
    idx, table, dy = problem(500, 40, 16, torch.float16, seed=2)
    dy[:] = float("nan")
    assert not grad(torch.full_like(idx, 7), table, dy, pad=7).any()


def test_non_finite_rows_stay_with_their_index():
    idx, table, dy = problem(3000, 50, 16, torch.float32, seed=3)
    clean = grad(idx, table, dy, pad=4)
    dy[idx == 4] = float("nan")
    dy[idx == 9] = float("inf")
    got = grad(idx, table, dy, pad=4)
    keep = torch.arange(50) != 9
    assert torch.equal(got[keep], clean[keep]) and torch.isinf(got[9]).all() and not got[4].any()


def test_index_beyond_the_table():
    from flexgemm_b200.kernels import cuda as K
    from flexgemm_b200.ops.embedding import sparse_embedding
    table = torch.randn(10, 8, device=DEV, requires_grad=True)
    for bad in (10, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40):
        idx = torch.tensor([1, bad, 3], device=DEV)
        out = sparse_embedding(idx, table)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="index"):
            K.check_status(DEV)
        (g,) = torch.autograd.grad(out, [table], torch.ones_like(out))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="index"):
            K.check_status(DEV)
        want = torch.zeros_like(g)
        want[[1, 3]] = 1.0
        assert torch.equal(g, want)


@pytest.mark.parametrize("V", [2 ** 22 + 1, 20_000_001, 2 ** 27 + 5])
def test_large_tables(V):
    """Rows to be cleared beyond what a CTA looks at at a time, keys of three and four digits."""
    from flexgemm_b200.ops.embedding import sparse_embedding
    idx = torch.cat([torch.randint(0, V, (3000,), generator=torch.Generator().manual_seed(4)), torch.tensor([0, V - 1, V // 2, 65535, 65536, V - 1])]).to(DEV)
    table = torch.ones(V, 1, dtype=torch.float16, device=DEV, requires_grad=True)
    junk = torch.full((V, 1), float("nan"), dtype=torch.float16, device=DEV)
    del junk
    out = sparse_embedding(idx, table)
    (g,) = torch.autograd.grad(out, [table], torch.ones_like(out))
    rows, counts = idx.unique(return_counts=True)
    assert torch.equal(g[rows, 0], counts.half())
    g[rows] = 0
    assert not g.any()


def test_stream_capture_and_two_graphs():
    from flexgemm_b200.ops.embedding import sparse_embedding
    idx, table, dy = problem(1500, 300, 32, torch.bfloat16, seed=5, share=0.2)
    i, t, d = idx.to(DEV), table.to(DEV).requires_grad_(True), dy.to(DEV)
    graphs = []
    for scale in (1.0, 2.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (g,) = torch.autograd.grad(sparse_embedding(i, t, scale=scale), [t], d)
        graphs.append((graph, g, scale))
    for seed in (6, 7):
        new = problem(1500, 300, 32, torch.bfloat16, seed=seed, share=0.5)[0]
        i.copy_(new)
        for graph, g, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, g, scale in graphs:
            assert torch.equal(g, grad(new, table, dy, scale=scale))


def test_launches():
    """A call with gradient of up to 4096 positions is two launches, the lookup and the gradient; the way of many is taken beyond."""
    from flexgemm_b200 import _cabi
    from flexgemm_b200.ops.embedding import sparse_embedding
    count = _cabi.lib().fgb_launch_count
    def launches(n, C):
        idx, table, dy = problem(n, 300, C, torch.float32, seed=8)
        t = table.to(DEV).requires_grad_(True)
        i, d = idx.to(DEV), dy.to(DEV)
        before = count()
        torch.autograd.grad(sparse_embedding(i, t), [t], d)
        return count() - before
    assert launches(1, 8) == 2 and launches(2520, 64) == 2 and launches(4096, 1024) == 2
    assert launches(4097, 8) > 2 and launches(100, 1028) > 2
