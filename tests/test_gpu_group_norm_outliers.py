"""Group norm of samples whose first rows are far from the others: an outlier, or zeros in front of channels with a large
mean, where sums of distances from the first row would lose the variance.

Bounds.  A thread adds runs of rows, the first of 8 and the others of at most 64, and takes distances d from the first row in the
first run, from the mean of the rows before in the others.  The sum of a run's squares and the square of its sum are off by at most
n and 2 n roundings of sum d^2 (n rows).  With one row at a distance D much larger than the others' spread, which is the
first: 3 * 8 roundings of 7 D^2 in the first run, and of D^2 (64 rows, D / 8 away) 3 * 64 in the second; the distances after that are
smaller.  All squared distances together are 7 / 8 D^2 at least: (168 + 192) * 8 / 7 = 412 roundings of the variance, 206 of
1 / sqrt(variance); with D not much larger fewer.  Runs, lanes and blocks are joined by their means, some 30 roundings more.  With the 160
roundings of the terms that the other tests allow that is 396 * 2^-24 of the terms' magnitudes, and half a step of the type."""
import pytest
import torch

from oracle import rows_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CHAIN = 396 * 2.0 ** -24


def problem(lengths, C, dtype, first, seed):
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    spread = torch.rand(C, generator=g) + 0.25
    far = first != "zeros"
    centre = torch.randn(C, generator=g) * (1.0 if far else 300.0)
    x = torch.randn(n, C, generator=g) * spread + centre
    starts = [sum(lengths[:b]) for b, k in enumerate(lengths) if k > 16]
    for s in starts:
        x[s] = centre + first * spread * torch.randn(C, generator=g).sign() if far else 0.0
    return x.to(dtype), torch.randn(n, C, generator=g).to(dtype), (1 + 0.3 * torch.randn(C, generator=g)).to(dtype), (0.3 * torch.randn(C, generator=g)).to(dtype)


def assert_near(got, want, size, what):
    info = torch.finfo(got.dtype)
    bound = want.abs().clamp_min(info.tiny) * info.eps / 2 + CHAIN * size * (1 + info.eps)
    off = (got.detach().cpu().double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, the worst {(off / bound).max().item():.3g} times its bound"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("first", [30.0, 300.0, "zeros"])
@pytest.mark.parametrize("lengths,C,groups", [
    ([40], 64, 8),                          # a warp's worth
    ([4096], 8, 2),                         # one launch, clusters
    ([2000, 900, 1500], 64, 8),
    ([130] * 300, 36, 9),                   # single CTAs
    ([3] * 600 + [50000] + [2] * 100, 8, 2),  # a long sample among short ones
    ([166000], 16, 4),                      # blocks of rows
    ([30000, 20000], 100, 100),             # a channel a group
])
def test_first_row_far_from_the_others(lengths, C, groups, first, dtype):
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x, dy, w, b = problem(lengths, C, dtype, first, seed=C + len(lengths))
    ends = torch.tensor([0] + lengths).cumsum(0)
    e = ends.tolist()
    ref = orc.group_norm(x, list(zip(e[:-1], e[1:])), groups, w, b, 1e-5, True, dy)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    out = sparse_group_norm(leaves[0], ends.to(DEV), groups, leaves[1], leaves[2], activation="silu")
    grads = torch.autograd.grad(out, leaves, dy.to(DEV))
    assert_near(out, ref["y"], ref["z_size"] + ref["y"].abs(), "out")
    for k, got in zip(("dx", "dw", "db"), grads):
        assert_near(got, ref[k], ref[k + "_size"], k)


@pytest.mark.parametrize("lengths", [[200], [9, 70000], [40000] * 3])
def test_equal_rows(lengths):
    """All rows alike: the mean is the row, exactly, and the output the bias."""
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    row = torch.tensor([0.1, -3.3e4, 1e-3, 77.7, 3e38, -1e-30, 0.0, 123456.7])
    x = row.expand(sum(lengths), 8).contiguous().to(DEV)
    bias = torch.arange(8.0, device=DEV) + 1
    out = sparse_group_norm(x, torch.tensor([0] + lengths, device=DEV).cumsum(0), 8, None, bias)
    assert torch.equal(out, bias.expand_as(out))
