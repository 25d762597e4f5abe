"""GPU tests of the group norm on ragged rows, against the plain 64-bit form.

Bounds.  A result is off by at most half a step of its type (``eps / 2`` of the value, or of the smallest normal number
below that) plus what the float32 arithmetic before it makes of its terms: with at most some 60 roundings on the way from
an input to a term and some 100 on the longest chain of a sum (a thread's rows, the lanes, the blocks), ``160 * 2^-24`` of
the terms' magnitudes (``oracle.rows_oracle`` gives them).  The 16-bit types' exponential is exact to 2^-20 for the z that
occur here (|z| < 16), ``16 * 2^-24`` of a term, which is inside that."""
import pytest
import torch

from oracle import rows_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
CHAIN = 160 * 2.0 ** -24


def half_step(value, dtype):
    info = torch.finfo(dtype)
    return value.abs().clamp_min(info.tiny) * info.eps / 2


def assert_near(got, want, size, dtype, what):
    got = got.detach().cpu().double()
    bound = half_step(want, dtype) + CHAIN * size * (1 + torch.finfo(dtype).eps)
    over = ((got - want).abs() - bound)
    bad = ~(over <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, the worst over its bound by {over.max().item():.3g}"


def problem(lengths, C, dtype, spare=0, seed=0, param=None, mean=1.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths) + spare
    centre = torch.randn(C, generator=g) * mean
    x = (torch.randn(n, C, generator=g) * (torch.rand(C, generator=g) + 0.25) + centre).to(dtype)
    dy = torch.randn(n, C, generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(param or dtype)
    b = (0.3 * torch.randn(C, generator=g)).to(param or dtype)
    ends = torch.tensor([0] + lengths).cumsum(0)
    return x, dy, w, b, ends


def bounds_of(ends):
    e = ends.tolist()
    return list(zip(e[:-1], e[1:]))


def run(x, dy, w, b, offsets, groups, act, eps=1e-5):
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    leaves = [t.to(DEV).requires_grad_(True) if t is not None else None for t in (x, w, b)]
    out = sparse_group_norm(leaves[0], offsets, groups, leaves[1], leaves[2], eps=eps, activation=act)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], dy.to(DEV))
    return out, grads


def check(x, dy, w, b, ends, groups, act, offsets=None, eps=1e-5):
    ref = orc.group_norm(x, bounds_of(ends), groups, w, b, eps, act == "silu", dy)
    out, grads = run(x, dy, w, b, ends.to(torch.int32).to(DEV) if offsets is None else offsets, groups, act, eps)
    assert_near(out, ref["y"], ref["z_size"] + ref["y"].abs(), x.dtype, "out")
    assert_near(grads[0], ref["dx"], ref["dx_size"], x.dtype, "grad_feats")
    if w is not None:
        assert_near(grads[1], ref["dw"], ref["dw_size"], w.dtype, "grad_weight")
    if b is not None:
        assert_near(grads[-1], ref["db"], ref["db_size"], b.dtype, "grad_bias")
    return out, grads


CASES = [
    # lengths, C, groups, spare rows
    ([1], 8, 1, 0),
    ([2], 1, 1, 0),
    ([5, 0, 1, 0, 0, 7], 16, 4, 3),
    ([0, 0, 9], 3, 3, 0),
    ([100, 900, 33], 20, 5, 0),
    ([257], 64, 32, 1),
    ([700, 1, 1500], 96, 12, 100),
    ([64] * 50, 32, 8, 0),
    ([0, 40, 0], 2056, 8, 0),
    ([30, 30], 1028, 4, 2),
    ([6000], 36, 9, 0),
    ([3000, 5000], 512, 32, 0),
    # samples too long for one launch
    ([20000, 0, 3], 36, 9, 50),
    ([12000, 5000], 100, 5, 7),
    ([40000], 16, 16, 0),
    ([900], 2056, 8, 0),
    ([30000, 1], 33, 3, 1),
    ([70000], 6, 1, 0),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,C,groups,spare", CASES)
def test_matches_plain_form(lengths, C, groups, spare, dtype):
    x, dy, w, b, ends = problem(lengths, C, dtype, spare, seed=C + len(lengths))
    for act in (None, "silu"):
        out, grads = check(x, dy, w, b, ends, groups, act)
        assert not out[ends[-1]:].any() and not grads[0][ends[-1]:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("lengths,C,groups", [
    ([7] * 30 + [3000, 0, 2500] + [7] * 500 + [2800, 4000] + [1] * 20, 96, 12),
    ([9000, 1] + [3] * 700 + [5000], 8, 2),
    ([4100] * 9 + [0] * 3000 + [2], 33, 3),
    ([2] * 900 + [20000], 64, 8),
])
def test_long_samples_among_short_ones(lengths, C, groups, dtype):
    x, dy, w, b, ends = problem(lengths, C, dtype, spare=5, seed=C)
    out, grads = check(x, dy, w, b, ends, groups, "silu")
    again = run(x, dy, w, b, ends.to(DEV), groups, "silu")
    assert torch.equal(out, again[0]) and all(torch.equal(u, v) for u, v in zip(grads, again[1]))
    assert not out[ends[-1]:].any() and not grads[0][ends[-1]:].any()


@pytest.mark.parametrize("w_on,b_on", [(False, False), (True, False), (False, True)])
def test_without_parameters(w_on, b_on):
    x, dy, w, b, ends = problem([40, 300], 24, torch.float16, seed=3)
    check(x, dy, w if w_on else None, b if b_on else None, ends, 6, "silu")


def test_float32_parameters_and_wide_offsets():
    x, dy, w, b, ends = problem([40, 300, 0, 11], 64, torch.bfloat16, spare=9, seed=4, param=torch.float32)
    check(x, dy, w, b, ends, 8, "silu", offsets=ends.to(DEV))


def test_dense_samples():
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x, dy, w, b, ends = problem([60, 60, 60], 16, torch.float32, seed=5)
    y, _ = check(x, dy, w, b, ends, 4, "silu")
    for shape in ((3, 60, 16), (3, 5, 12, 16)):
        got = sparse_group_norm(x.to(DEV).view(shape), None, 4, w.to(DEV), b.to(DEV), activation="silu")
        assert got.shape == shape and torch.equal(got.view(180, 16), y)
    one = sparse_group_norm(x.to(DEV), None, 4, w.to(DEV), b.to(DEV), activation="silu")
    whole = sparse_group_norm(x.to(DEV), torch.tensor([0, 180], device=DEV), 4, w.to(DEV), b.to(DEV), activation="silu")
    assert torch.equal(one, whole)


def test_many_more_samples_than_rows():
    """Most samples empty, offsets that begin behind the first row."""
    g = torch.Generator().manual_seed(6)
    n, B = 700, 5000
    ends = torch.sort(torch.randint(13, n - 20, (B + 1,), generator=g))[0]
    x, dy, w, b, _ = problem([n], 48, torch.float32, seed=7)
    out, grads = check(x, dy, w, b, ends, 6, "silu")
    assert not out[:int(ends[0])].any() and not out[int(ends[-1]):].any()


def test_rows_of_no_sample_count_for_nothing():
    x, dy, w, b, ends = problem([50, 20], 32, torch.float16, spare=40, seed=8)
    clean, clean_grads = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    for junk in (float("nan"), float("inf"), torch.finfo(torch.float16).min):
        x[70:], dy[70:] = junk, junk
        out, grads = run(x, dy, w, b, ends.to(DEV), 4, "silu")
        assert torch.equal(out, clean) and all(torch.equal(p, q) for p, q in zip(grads, clean_grads))


def test_nan_stays_in_its_sample_and_group():
    x, dy, w, b, ends = problem([50, 20], 32, torch.float32, seed=9)
    clean, _ = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    x[60, 9] = float("nan")   # second sample, second group
    out, _ = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    hit = torch.zeros(70, 32, dtype=torch.bool)
    hit[50:, 8:16] = True
    assert torch.equal(torch.isnan(out).cpu(), hit) and torch.equal(out[~hit.to(DEV)], clean[~hit.to(DEV)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mean_far_from_zero(dtype):
    """A spread of one around a mean of hundreds: plain sums of squares would lose the variance."""
    x, dy, w, b, ends = problem([4000, 90], 16, dtype, seed=10, mean=300.0)
    check(x, dy, w, b, ends, 16, None)


def test_constant_rows():
    x = torch.full((33, 8), 2.5, dtype=torch.float16)
    out, grads = run(x, torch.ones_like(x), torch.ones(8, dtype=torch.float16), torch.full((8,), 0.5, dtype=torch.float16), torch.tensor([0, 33], device=DEV),
                     2, None)
    assert torch.equal(out.cpu(), torch.full_like(x, 0.5)) and not grads[0].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_statistics_of_one_value(dtype):
    """One row a sample, one channel a group: the output is act(bias), the gradient zero, not what rounding leaves of it."""
    x, dy, w, b, ends = problem([1] * 5, 16, dtype, seed=17)
    for act in (None, "silu"):
        out, grads = run(x, dy, w, b, ends.to(DEV), 16, act)
        assert not grads[0].any() and not grads[1].any() and torch.equal(out, out[:1].expand_as(out))


def test_repeated_calls_are_equal():
    x, dy, w, b, ends = problem([3000, 2000], 64, torch.bfloat16, seed=11)
    first = run(x, dy, w, b, ends.to(DEV), 8, "silu")
    for _ in range(3):
        again = run(x, dy, w, b, ends.to(DEV), 8, "silu")
        assert torch.equal(first[0], again[0]) and all(torch.equal(p, q) for p, q in zip(first[1], again[1]))


def test_gradient_against_differences():
    """Central differences of the float32 call along a direction v with step h.  The loss is a sum of n C products, formed in
    64 bits; each output is off by some 2^-21 of a size of about one, so the quotient by 2^-21 sqrt(n C) |dy| / h; the
    third derivative along v adds about h^2 |dy| sqrt(n C)."""
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x, dy, w, b, ends = problem([30, 51], 24, torch.float32, seed=12)
    off = ends.to(DEV)
    _, grads = run(x, dy, w, b, off, 6, "silu")
    h = 2.0 ** -7
    g = torch.Generator().manual_seed(13)
    base = [x, w, b]
    for k in range(3):
        v = torch.randn(base[k].shape, generator=g)
        loss = []
        for sign in (1, -1):
            args = [t.to(DEV) for t in base]
            args[k] = (base[k] + sign * h * v).to(DEV)
            y = sparse_group_norm(args[0], off, 6, args[1], args[2], activation="silu")
            loss.append((y.double() * dy.to(DEV).double()).sum().item())
        quotient = (loss[0] - loss[1]) / (2 * h)
        want = (grads[k].double() * v.to(DEV).double()).sum().item()
        n = (x.numel()) ** 0.5
        assert abs(quotient - want) <= 3 * n * (2.0 ** -21 / h + 4 * h * h), (k, quotient, want)


def test_strided_and_shifted_inputs():
    """Rows of a wider buffer, a buffer that does not begin at a multiple of 16 bytes, an expanded gradient."""
    x, dy, w, b, ends = problem([50, 31], 24, torch.float16, seed=14)
    want, want_grads = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    wide = torch.zeros(81, 40, dtype=torch.float16)
    wide[:, 5:29] = x
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    leaf = wide.to(DEV).requires_grad_(True)
    out = sparse_group_norm(leaf[:, 5:29], ends.to(DEV), 4, w.to(DEV), b.to(DEV), activation="silu")
    (g,) = torch.autograd.grad(out, [leaf], dy.to(DEV))
    assert torch.equal(out, want) and torch.equal(g[:, 5:29], want_grads[0]) and not g[:, :5].any() and not g[:, 29:].any()
    flat = torch.zeros(81 * 24 + 1, dtype=torch.float16)
    flat[1:] = x.reshape(-1)
    out = sparse_group_norm(flat.to(DEV)[1:].view(81, 24), ends.to(DEV), 4, w.to(DEV), b.to(DEV), activation="silu")
    assert torch.equal(out, want)
    leaf = x.to(DEV).requires_grad_(True)
    sparse_group_norm(leaf, ends.to(DEV), 4, w.to(DEV), b.to(DEV), activation="silu").sum().backward()
    again = run(x, torch.ones_like(dy), w, b, ends.to(DEV), 4, "silu")[1][0]
    assert torch.equal(leaf.grad, again)


def test_other_streams_and_capture():
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x, dy, w, b, ends = problem([500, 301], 32, torch.float16, seed=15)
    want, want_grads = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, grads = run(x, dy, w, b, ends.to(DEV), 4, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(p, q) for p, q in zip(grads, want_grads))
    # forward and backward in one graph, replayed on other data of the same buffers
    args = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    off, d = ends.to(DEV), dy.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_group_norm(args[0], off, 4, args[1], args[2], activation="silu")
        grads = torch.autograd.grad(out, args, d)
    for shift in (0, 300, 77):
        off.copy_(torch.tensor([0, shift, 801]))
        graph.replay()
        torch.cuda.synchronize()
        again = run(x, dy, w, b, torch.tensor([0, shift, 801], device=DEV), 4, "silu")
        assert torch.equal(out, again[0]) and all(torch.equal(p, q) for p, q in zip(grads, again[1]))


def test_bad_offsets_raise_later():
    from flexgemm_b200.kernels import cuda as K
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x = torch.randn(40, 8, device=DEV)
    for bad in ([0, 30, 20, 40], [-1, 40], [0, 41], [5, 2]):
        sparse_group_norm(x, torch.tensor(bad, device=DEV), 2)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="offsets"):
            sparse_group_norm(x, torch.tensor([0, 40], device=DEV), 2)
        sparse_group_norm(x, torch.tensor([0, 40], device=DEV), 2)
        torch.cuda.synchronize()
        K.check_status(DEV)


def test_sample_offsets():
    from flexgemm_b200.kernels import cuda as K
    from flexgemm_b200.ops.utils import sample_offsets
    g = torch.Generator().manual_seed(16)
    for lengths in ([7], [0, 3, 0, 0, 900, 1, 0], [0, 0], [300] * 9):
        b = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
        coords = torch.cat([b.view(-1, 1), torch.randint(0, 9, (b.numel(), 3), generator=g)], dim=1).int().to(DEV)
        got = sample_offsets(coords, len(lengths))
        assert got.dtype == torch.int32 and got.tolist() == [0] + torch.tensor(lengths).cumsum(0).tolist()
    bad = torch.tensor([[0, 1, 1, 1], [2, 1, 1, 1], [1, 1, 1, 1]], dtype=torch.int32, device=DEV)
    for c, batch in ((bad, 3), (bad[:2], 2)):
        sample_offsets(c, batch)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="offsets"):
            K.check_status(DEV)


def test_second_derivative_and_tangents_are_refused():
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x = torch.randn(40, 8, device=DEV, requires_grad=True)
    y = sparse_group_norm(x, None, 2)
    (g,) = torch.autograd.grad(y.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            sparse_group_norm(dual, None, 2)


def test_no_rows():
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    w = torch.ones(8, device=DEV, requires_grad=True)
    out = sparse_group_norm(x, torch.zeros(4, dtype=torch.int64, device=DEV), 2, w)
    out.sum().backward()
    assert out.shape == (0, 8) and x.grad.shape == (0, 8) and not w.grad.any()


@pytest.mark.parametrize("C, samples", [(512, 3), (2056, 40), (96, 2000)])
def test_parameters_without_rows(C, samples):
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x = torch.zeros(0, C, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w, b = (torch.ones(C, dtype=torch.bfloat16, device=DEV, requires_grad=True) for _ in range(2))
    out = sparse_group_norm(x, torch.zeros(samples + 1, dtype=torch.int32, device=DEV), 8, w, b, activation="silu")
    gw, gb = torch.autograd.grad(out, (w, b), torch.zeros_like(out))
    torch.cuda.synchronize()
    assert not gw.any() and not gb.any()


def test_input_changed_before_backward_is_refused():
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x = torch.randn(40, 8, device=DEV, requires_grad=True)
    off = torch.tensor([0, 40], device=DEV)
    y = sparse_group_norm(x, off, 2)
    off.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
