"""Grouped products of float32 data where every output is one product, so that no addition hides what the bf16 planes of
the operands leave out.

Bounds.  A plane has bf16's eight significant bits and takes what the planes before it left, rounded to nearest, so with half a step of
2^-8 |x - h| <= 2^-8 |x|, |x - h - m| <= 2^-16 |x|, |x - h - m - l| <= 2^-24 |x|.  Accurate products leave out m l, l m, l l and what three planes
leave: (2 + 2) * 2^-24 + 2^-32 of a product, and a little.  The tensor cores cut what they add to an accumulator at 2^-23 of the sum at most: once
for the large product, and for the small ones before it at 2^-7 of that.  What is added afterwards is zero.  Together less than
2^-22 + 2^-23 + 2^-27.  Where TF32 is allowed m m is left out, and what two planes leave: 3 * 2^-16 and 2^-24 of terms of third order, with the same cut.
A bias gradient of one row is its planes added up: what they leave, 2^-24 or 2^-16, and the cuts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _defaults():
    from flexgemm_b200.kernels import config
    yield
    config.allow_tf32 = True


def values(g, *size):
    """Full significands over twenty binades."""
    return (torch.rand(*size, generator=g) + 1) * torch.randn(*size, generator=g).sign() * 2.0 ** torch.randint(-10, 10, size, generator=g)


CASES = [
    # lengths, ci, co; no group has more rows than ci * co
    ([5], 512, 200),                 # few rows
    ([3, 5, 0, 9], 4104, 24),        # few rows, cut
    ([2, 7], 40, 4200),              # the same for the input gradient
    ([127, 128, 129, 1], 100, 36),   # tiles of 128 rows
    ([900], 64, 72),
    ([4500, 300], 72, 2056),         # pairs of CTAs
    ([3001, 1700], 2056, 72),
    ([9001], 1040, 640),             # pairs, all passes
    ([17] * 2000, 96, 64),           # the plan of 2000 groups leaves one stage of three planes
]


@pytest.mark.parametrize("tf32", [False, True])
@pytest.mark.parametrize("lengths,ci,co", CASES)
def test_single_products(lengths, ci, co, tf32):
    from flexgemm_b200.kernels import config
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    config.allow_tf32 = tf32
    cut = 2.0 ** -23 + 2.0 ** -27
    product, single = (3 * 2.0 ** -16 + cut + 2.0 ** -23, 2.0 ** -16 + cut) if tf32 else (2.0 ** -22 + cut, 2.0 ** -24 + cut)
    g = torch.Generator().manual_seed(ci + co)
    n, G = sum(lengths), len(lengths)
    group = torch.repeat_interleave(torch.arange(G), torch.tensor(lengths))
    ends = torch.tensor([0] + lengths).cumsum(0)
    rows = torch.arange(n)
    r = rows - ends[group]
    # one entry of each row of x and of dy, at places that no other row of the group shares
    i, o = r % ci, (r // ci + r) % co
    vx, vy, w = values(g, n), values(g, n), values(g, G, co, ci)
    x, dy = torch.zeros(n, ci), torch.zeros(n, co)
    x[rows, i], dy[rows, o] = vx, vy
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w)]
    bias = torch.zeros(G, co, device=DEV, requires_grad=True)
    out = sparse_grouped_linear(leaves[0], ends.to(DEV), leaves[1], bias)
    dx, dw, db = (t.cpu().double() for t in torch.autograd.grad(out, leaves + [bias], dy.to(DEV)))
    vx, vy, wd = vx.double().unsqueeze(1), vy.double().unsqueeze(1), w.double()
    def near(got, want, bound, what):
        off = (got - want).abs()
        bad = ~(off <= bound * want.abs())
        assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, the worst off by 2^{(off / want.abs()).nan_to_num(0).max().log2().item():.2f}"
    near(out.detach().cpu().double(), vx * wd[group, :, i], product, "out")
    near(dx, vy * wd[group, o, :], product, "grad_feats")
    want = torch.zeros(G, co, ci, dtype=torch.float64)
    want[group, o, i] = (vx * vy).squeeze(1)
    near(dw, want, product, "grad_weight")
    if max(lengths) <= min(ci, co):   # a row for each entry of db
        want = torch.zeros(G, co, dtype=torch.float64)
        want[group, o] = vy.squeeze(1)
        near(db, want, single, "grad_bias")


def test_many_groups_of_float32():
    """Some 2000 groups of more than 16 rows: whole tiles of 128, and one stage in shared memory."""
    from flexgemm_b200.kernels import config
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    from oracle import rows_oracle as orc
    config.allow_tf32 = False
    lengths = [17, 31, 0, 20] * 500 + [130, 9]
    g = torch.Generator().manual_seed(1)
    n, G, ci, co = sum(lengths) + 3, len(lengths), 96, 64
    x, dy, w = torch.randn(n, ci, generator=g), torch.randn(n, co, generator=g), torch.randn(G, co, ci, generator=g)
    ends = torch.tensor([0] + lengths).cumsum(0)
    e = ends.tolist()
    ref = orc.grouped_linear(x, list(zip(e[:-1], e[1:])), w, None, dy)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w)]
    out = sparse_grouped_linear(leaves[0], ends.to(DEV), leaves[1])
    dx, dw = torch.autograd.grad(out, leaves, dy.to(DEV))
    # planes: 2^-25 of the terms' magnitudes; additions: four blocks of 64 k at most, of 24 cuts each, and three roundings between them
    for got, k in ((out, "y"), (dx, "dx"), (dw, "dw")):
        assert ((got.detach().cpu().double() - ref[k]).abs() <= (99 * 2.0 ** -23 + 2.0 ** -25) * ref[k + "_size"]).all(), k
