"""GPU tests of the products grouped by row ranges, against the plain 64-bit form.

Bounds.  A result is off by at most half a step of its type (``eps / 2`` of the value, or of the smallest normal number
below that) and by what its sum loses before: products of 16-bit numbers are exact in float32, and a sum over k is built in
steps of 16, each of which rounds or cuts at 2^-23 of at most the sum of the terms' magnitudes (``*_size``); pieces and the
bias add fewer than 160 roundings more.  float32 data counts its plane products as steps of their own (6, or 3 where TF32
is allowed).  With planes of 8 bits rounded to nearest (|x - h| <= 2^-9 |x|, and so on), accurate products leave out less
than 2^-24 of a product, the others less than 2^-16 (m m, h l and l h: 3 * 2^-18)."""
import pytest
import torch

from oracle import rows_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _defaults():
    from flexgemm_b200.kernels import config
    config.allow_tf32 = False
    yield
    config.allow_tf32 = True


def half_step(value, dtype):
    info = torch.finfo(dtype)
    return value.abs().clamp_min(info.tiny) * info.eps / 2


def assert_near(got, want, size, k, what, tf32=False):
    t = got.dtype
    planes, left_out = (1, 0.0) if t != torch.float32 else (3, 2.0 ** -16) if tf32 else (6, 2.0 ** -24)
    lost = ((planes * (k + 15) / 16 + 160) * 2.0 ** -23 + left_out) * size
    over = (got.detach().cpu().double() - want).abs() - (half_step(want, t) + lost * (1 + torch.finfo(t).eps))
    bad = ~(over <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, the worst over its bound by {over.max().item():.3g}"


def problem(lengths, ci, co, dtype, spare=0, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    n, G = sum(lengths) + spare, len(lengths)
    x, dy = torch.randn(n, ci, generator=g).to(dtype), torch.randn(n, co, generator=g).to(dtype)
    w = (torch.randn(G, co, ci, generator=g) / ci ** 0.5).to(dtype)
    b = torch.randn(G, co, generator=g).to(dtype) if bias else None
    return x, dy, w, b, torch.tensor([0] + lengths).cumsum(0)


def run(x, dy, w, b, offsets):
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    leaves = [t.to(DEV).requires_grad_(True) if t is not None else None for t in (x, w, b)]
    out = sparse_grouped_linear(leaves[0], offsets.to(DEV), leaves[1], leaves[2])
    return out, torch.autograd.grad(out, [t for t in leaves if t is not None], dy.to(DEV))


def check(x, dy, w, b, ends, tf32=False):
    e = ends.tolist()
    ref = orc.grouped_linear(x, list(zip(e[:-1], e[1:])), w, b, dy)
    out, grads = run(x, dy, w, b, ends)
    ci, co, longest = x.shape[1], dy.shape[1], max(hi - lo for lo, hi in zip(e[:-1], e[1:]))
    assert_near(out, ref["y"], ref["y_size"], ci, "out", tf32)
    assert_near(grads[0], ref["dx"], ref["dx_size"], co, "grad_feats", tf32)
    assert_near(grads[1], ref["dw"], ref["dw_size"], longest, "grad_weight", tf32)
    if b is not None:
        assert_near(grads[2], ref["db"], ref["db_size"], longest, "grad_bias", tf32)
    assert not out[e[-1]:].any() and not grads[0][e[-1]:].any() and not out[:e[0]].any() and not grads[0][:e[0]].any()
    return out, grads


CASES = [
    # lengths, ci, co, spare
    ([1], 8, 8, 0),
    ([3, 0, 1, 0, 0, 2], 16, 24, 5),
    ([1, 1, 1], 64, 1024, 0),
    ([5], 512, 200, 0),
    ([40, 3, 64, 65, 0, 63], 72, 136, 1),
    ([0, 0, 7, 0], 3, 5, 2),
    ([100, 200], 6, 10, 0),
    ([127, 128, 129, 1], 100, 36, 3),
    ([500], 64, 64, 0),
    ([1000, 1, 0, 333], 256, 320, 40),
    ([700, 900], 264, 520, 0),
    ([15, 16, 17, 31, 33] * 30, 48, 96, 0),
    ([5000, 17], 128, 128, 0),
    ([2, 4000, 1], 1032, 40, 0),
    ([64] * 70, 32, 16, 0),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,ci,co,spare", CASES)
def test_matches_plain_form(lengths, ci, co, spare, dtype):
    check(*problem(lengths, ci, co, dtype, spare, seed=ci + co, bias=ci != 64))


VARIANTS = [
    # pairs of CTAs: forward, input gradient, weight gradient (rows cleared in both CTAs), narrower last tiles
    ([4500, 300], 72, 2056, 0),
    ([3001, 1700], 2056, 72, 7),
    ([9001], 1040, 640, 0),
    ([2100, 0, 4200], 136, 2824, 1),
    # few rows, cut along 4104 or 4200 channels
    ([3, 5, 0, 9], 4104, 24, 0),
    ([2, 7], 40, 4200, 3),
    ([11], 8200, 136, 0),
    # tiles of half as many columns
    ([200, 130], 80, 520, 0),
    # searches past more than 32 groups, few rows and many
    ([1] * 40 + [0] * 100 + [3] * 40 + [200], 24, 40, 2),
    ([0] * 40 + [2000] + [0] * 33 + [1900, 0], 64, 96, 0),
    # all rows in one of many groups
    ([0] * 60 + [900] + [0] * 20, 64, 72, 0),
    # the plan of many groups
    ([2, 1, 0, 3] * 500, 16, 24, 5),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,ci,co,spare", VARIANTS)
def test_variants(lengths, ci, co, spare, dtype):
    check(*problem(lengths, ci, co, dtype, spare, seed=ci, bias=ci != 40))


@pytest.mark.parametrize("lengths,ci,co", [([300, 500], 64, 72), ([4, 9], 128, 256), ([90], 20, 12)])
def test_float32_with_tf32_allowed(lengths, ci, co):
    from flexgemm_b200.kernels import config
    config.allow_tf32 = True
    check(*problem(lengths, ci, co, torch.float32, seed=1), tf32=True)


def test_backward_takes_the_setting_of_its_time():
    from flexgemm_b200.kernels import config
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, dy, w, b, ends = problem([200, 100], 64, 64, torch.float32, seed=2)
    want, grads = run(x, dy, w, b, ends)
    leaf = x.to(DEV).requires_grad_(True)
    config.allow_tf32 = True
    out = sparse_grouped_linear(leaf, ends.to(DEV), w.to(DEV), b.to(DEV))
    config.allow_tf32 = False
    (g,) = torch.autograd.grad(out, [leaf], dy.to(DEV))
    assert torch.equal(g, grads[0]) and not torch.equal(out, want)


def test_offsets_that_begin_behind_the_first_row():
    x, dy, w, b, _ = problem([400, 200, 100], 32, 48, torch.float16, spare=30, seed=3)
    check(x, dy, w, b, torch.tensor([17, 300, 300, 650], dtype=torch.int32))


@pytest.mark.parametrize("lengths", [[50, 300, 77], [5, 3, 9]])
def test_rows_of_others_count_for_nothing(lengths):
    """Infinities and NaN in the rows of no group and in another group's rows: tiles and blocks of rows reach into both."""
    x, dy, w, b, ends = problem(lengths, 64, 64, torch.bfloat16, spare=100, seed=4)
    clean, clean_grads = run(x, dy, w, b, ends)
    for junk in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        x2, dy2 = x.clone(), dy.clone()
        x2[ends[-1]:], dy2[ends[-1]:] = junk, junk
        out, grads = run(x2, dy2, w, b, ends)
        assert torch.equal(out, clean) and all(torch.equal(p, q) for p, q in zip(grads, clean_grads))
    x2, dy2 = x.clone(), dy.clone()
    x2[ends[1]:ends[2]], dy2[ends[1]:ends[2]] = float("nan"), float("nan")
    out, grads = run(x2, dy2, w, b, ends)
    for rows in (slice(0, ends[1]), slice(ends[2], None)):
        assert torch.equal(out[rows], clean[rows]) and torch.equal(grads[0][rows], clean_grads[0][rows])
    for g in (0, 2):
        assert torch.equal(grads[1][g], clean_grads[1][g]) and torch.equal(grads[2][g], clean_grads[2][g])
    assert torch.isnan(out[ends[1]:ends[2]]).all() and torch.isnan(grads[1][1]).all() and torch.isnan(grads[2][1]).all()


def test_large_and_small_float32():
    """The planes cover float32's range: values near its ends, and a non-finite one stays in its row."""
    x, dy, w, b, ends = problem([70, 30], 32, 16, torch.float32, seed=5)
    scale = torch.tensor([3e37, 1.0, 1e-30]).repeat(34)[:100].unsqueeze(1)
    x2 = x * scale
    x2[0, 0] = torch.finfo(torch.float32).max
    w2 = w * 1e-2
    e = ends.tolist()
    ref = orc.grouped_linear(x2, list(zip(e[:-1], e[1:])), w2, None)
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    out = sparse_grouped_linear(x2.to(DEV), ends.to(DEV), w2.to(DEV))
    assert_near(out, ref["y"], ref["y_size"], 32, "out")
    x2[5, 3] = float("inf")
    bad = sparse_grouped_linear(x2.to(DEV), ends.to(DEV), w2.to(DEV))
    assert not torch.isfinite(bad[5]).any()
    keep = torch.arange(100) != 5
    assert torch.equal(bad[keep], out[keep])


def test_repeated_calls_are_equal():
    for lengths, ci, co in (([9000, 2000], 128, 256), ([4, 7], 512, 256)):
        x, dy, w, b, ends = problem(lengths, ci, co, torch.bfloat16, seed=6)
        first = run(x, dy, w, b, ends)
        for _ in range(3):
            again = run(x, dy, w, b, ends)
            assert torch.equal(first[0], again[0]) and all(torch.equal(p, q) for p, q in zip(first[1], again[1]))


def test_some_gradients_only():
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, dy, w, b, ends = problem([100, 60], 32, 40, torch.float16, seed=7)
    _, want = run(x, dy, w, b, ends)
    for mask in range(1, 8):
        leaves = [t.to(DEV).requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        out = sparse_grouped_linear(leaves[0], ends.to(DEV), leaves[1], leaves[2])
        got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dy.to(DEV))
        assert all(torch.equal(p, q) for p, q in zip(got, [q for i, q in enumerate(want) if mask >> i & 1]))


def test_gradients_against_differences():
    """The call is linear in each argument: central differences of the float32 call are exact up to its rounding, which is
    2^-20 of the terms' magnitudes here (k <= 90)."""
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, dy, w, b, ends = problem([50, 0, 90], 24, 40, torch.float32, seed=8)
    _, grads = run(x, dy, w, b, ends)
    g = torch.Generator().manual_seed(9)
    e = ends.tolist()
    for k in range(3):
        v = torch.randn((x, w, b)[k].shape, generator=g)
        loss, size = [], 0.0
        for sign in (1, -1):
            args = [x, w, b]
            args[k] = args[k] + sign * v
            y = sparse_grouped_linear(args[0].to(DEV), ends.to(DEV), args[1].to(DEV), args[2].to(DEV))
            loss.append((y.double().cpu() * dy.double()).sum().item())
            size += (orc.grouped_linear(args[0], list(zip(e[:-1], e[1:])), args[1], args[2])["y_size"] * dy.abs()).sum().item()
        want = (grads[k].double().cpu() * v.double()).sum().item()
        assert abs((loss[0] - loss[1]) / 2 - want) <= 2.0 ** -20 * size, k


def test_layouts():
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, dy, w, b, ends = problem([100, 60], 32, 40, torch.float16, seed=10)
    want, want_grads = run(x, dy, w, b, ends)
    wide = torch.zeros(160, 50, dtype=torch.float16)
    wide[:, 7:39] = x
    leaf, wt = wide.to(DEV).requires_grad_(True), w.transpose(1, 2).contiguous().to(DEV).requires_grad_(True)
    out = sparse_grouped_linear(leaf[:, 7:39], ends.int().to(DEV), wt.transpose(1, 2), b.to(DEV))
    g, gw = torch.autograd.grad(out, [leaf, wt], dy.to(DEV))
    assert torch.equal(out, want) and torch.equal(g[:, 7:39], want_grads[0]) and torch.equal(gw.transpose(1, 2), want_grads[1])
    flat = torch.zeros(160 * 32 + 1, dtype=torch.float16)
    flat[1:] = x.reshape(-1)
    assert torch.equal(sparse_grouped_linear(flat.to(DEV)[1:].view(160, 32), ends.to(DEV), w.to(DEV), b.to(DEV)), want)
    leaf = x.to(DEV).requires_grad_(True)
    sparse_grouped_linear(leaf, ends.to(DEV), w.to(DEV), b.to(DEV)).sum().backward()   # an expanded gradient
    assert torch.equal(leaf.grad, run(x, torch.ones_like(dy), w, b, ends)[1][0])


def test_streams_and_capture():
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, dy, w, b, ends = problem([500, 301, 99], 64, 96, torch.float16, spare=100, seed=11)
    want, want_grads = run(x, dy, w, b, ends)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, grads = run(x, dy, w, b, ends)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(torch.equal(p, q) for p, q in zip(grads, want_grads))
    args = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    off, d = ends.to(DEV), dy.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_grouped_linear(args[0], off, args[1], args[2])
        grads = torch.autograd.grad(out, args, d)
    for new in ([0, 900, 900, 900], [0, 1, 2, 3], [10, 500, 500, 1000], ends.tolist()):
        off.copy_(torch.tensor(new))
        graph.replay()
        torch.cuda.synchronize()
        again = run(x, dy, w, b, torch.tensor(new))
        assert torch.equal(out, again[0]) and all(torch.equal(p, q) for p, q in zip(grads, again[1]))


def test_bad_offsets_raise_later():
    from flexgemm_b200.kernels import cuda as K
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    for n in (40, 400):
        x, w = torch.randn(n, 8, device=DEV, dtype=torch.float16), torch.randn(3, 16, 8, device=DEV, dtype=torch.float16)
        for bad in ([0, 30, 20, 40], [-1, 2, 3, 40], [0, 0, 0, n + 1], [n, 0, n, 0]):
            sparse_grouped_linear(x, torch.tensor(bad, device=DEV), w)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="offsets"):
                sparse_grouped_linear(x, torch.tensor([0, 1, 2, 3], device=DEV), w)
        sparse_grouped_linear(x, torch.tensor([0, 1, 2, 3], device=DEV), w)
        torch.cuda.synchronize()
        K.check_status(DEV)


def test_second_derivative_and_tangents_are_refused():
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, w = torch.randn(40, 8, device=DEV, requires_grad=True), torch.randn(1, 8, 8, device=DEV)
    off = torch.tensor([0, 40], device=DEV)
    (g,) = torch.autograd.grad(sparse_grouped_linear(x, off, w).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            sparse_grouped_linear(dual, off, w)


def test_no_rows():
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, w = torch.zeros(0, 8, device=DEV, requires_grad=True), torch.randn(2, 16, 8, device=DEV, requires_grad=True)
    out = sparse_grouped_linear(x, torch.zeros(3, dtype=torch.int32, device=DEV), w)
    out.sum().backward()
    assert out.shape == (0, 16) and x.grad.shape == (0, 8) and not w.grad.any()
