"""The layers on ragged rows and the convolutions as one network: labels -> embedding -> [group norm + SiLU, conv] twice + skip
-> a matrix for each sample, forward, gradients, a captured step -- against the same network in plain 64-bit torch on the CPU.

Bound.  The convolutions' own bar is 1e-4 of the largest value for accurate fp32; the two of them in each direction, and the
other layers (some 2^-20 of their terms, which are up to a few hundred times their sums), make less than 1e-3 of the
largest value of each output."""
import pytest
import torch

from oracle import rows_oracle
from oracle import submconv_oracle as orc

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
C, LABELS, GROUPS, OUT = 32, 11, 8, 24


@pytest.fixture(autouse=True)
def _defaults():
    from flexgemm_b200.kernels import config
    from flexgemm_b200.ops import spconv
    spconv.set_algorithm(spconv.Algorithm.MASKED_IMPLICIT_GEMM_SPLITK)
    config.allow_tf32 = False
    yield
    config.allow_tf32 = True


def make(seed, batch=3, res=16):
    from flexgemm_b200 import workloads
    g = torch.Generator().manual_seed(seed)
    coords = torch.from_numpy(workloads.shell_coords(res, batch, [1.0, 0.7, 0.9][:batch]))
    n = coords.shape[0]

    def randn(*size, scale=1.0):
        return torch.randn(*size, generator=g) * scale
    params = {"table": randn(LABELS, C), "gamma0": 1 + randn(C, scale=0.2), "beta0": randn(C, scale=0.2), "w0": randn(C, 3, 3, 3, C, scale=(27 * C) ** -0.5),
              "b0": randn(C, scale=0.1), "gamma1": 1 + randn(C, scale=0.2), "beta1": randn(C, scale=0.2), "w1": randn(C, 3, 3, 3, C, scale=(27 * C) ** -0.5),
              "b1": randn(C, scale=0.1), "head": randn(batch, OUT, C, scale=C ** -0.5), "head_b": randn(batch, OUT)}
    return coords, torch.randint(0, LABELS, (n,), generator=g), params, randn(n, OUT), torch.Size((batch, C, res, res, res))


def ours(coords, labels, p, shape):
    from flexgemm_b200.ops import spconv, utils
    from flexgemm_b200.ops.embedding import sparse_embedding
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    offsets = utils.sample_offsets(coords, shape[0])
    h = sparse_embedding(labels, p["table"], scale=C ** 0.5)
    y, cache = h, ours.cache
    for k in "01":
        y = sparse_group_norm(y, offsets, GROUPS, p["gamma" + k], p["beta" + k], activation="silu")
        y, cache = spconv.sparse_submanifold_conv3d(y, coords, shape, p["w" + k], p["b" + k], neighbor_cache=cache)
    return sparse_grouped_linear(h + y, offsets, p["head"], p["head_b"]), cache


ours.cache = None


def plain(coords, labels, p, shape):
    nbr = orc.neighbor_map(coords.numpy(), shape)
    n, ends = coords.shape[0], [0] + [int((coords[:, 0] <= b).sum()) for b in range(shape[0])]
    idx = torch.from_numpy(nbr.astype("int64"))
    h = p["table"][labels] * C ** 0.5
    y = h
    for k in "01":
        parts = [torch.nn.functional.silu(torch.nn.functional.group_norm(y[lo:hi].T.unsqueeze(0), GROUPS, p["gamma" + k], p["beta" + k])[0].T)
                 for lo, hi in zip(ends[:-1], ends[1:])]
        padded = torch.cat([torch.cat(parts), torch.zeros(1, C, dtype=torch.float64)])
        rows = torch.where(idx == 0xFFFFFFFF, torch.full_like(idx, n), idx)
        y = padded[rows].reshape(n, -1) @ p["w" + k].reshape(C, -1).T + p["b" + k]
    return torch.cat([(h + y)[lo:hi] @ p["head"][b].T + p["head_b"][b] for b, (lo, hi) in enumerate(zip(ends[:-1], ends[1:]))])


def test_network_and_gradients():
    coords, labels, params, grad, shape = make(1)
    ref_p = {k: v.double().requires_grad_(True) for k, v in params.items()}
    ref = plain(coords, labels, ref_p, shape)
    ref_g = torch.autograd.grad(ref, list(ref_p.values()), grad.double())
    p = {k: v.to(DEV).requires_grad_(True) for k, v in params.items()}
    out, _ = ours(coords.to(DEV), labels.to(DEV), p, shape)
    got = torch.autograd.grad(out, list(p.values()), grad.to(DEV))
    for name, a, b in [("out", out, ref)] + list(zip(p, got, ref_g)):
        err, scale = (a.detach().cpu().double() - b.detach()).abs().max().item(), b.detach().abs().max().item()
        assert err <= 1e-3 * scale, (name, err, scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured_training_step(dtype):
    """A step captured on one set of labels and replayed on others gives what the eager calls give."""
    coords, labels, params, grad, shape = make(2)
    p = {k: v.to(DEV).to(dtype).requires_grad_(True) for k, v in params.items()}
    c, lab, g = coords.to(DEV), labels.to(DEV), grad.to(DEV).to(dtype)
    ours.cache = ours(c, lab, p, shape)[1]   # the output is let go: a capture may meet no living graph of its leaves
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, _ = ours(c, lab, p, shape)
            grads = torch.autograd.grad(out, list(p.values()), g)
        for seed in (3, 4):
            lab.copy_(torch.randint(0, LABELS, labels.shape, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in (out, *grads)]
            want, _ = ours(c, lab, p, shape)
            want = (want, *torch.autograd.grad(want, list(p.values()), g))
            for a, b in zip(kept, want):
                assert torch.equal(a, b)
    finally:
        ours.cache = None


def test_samples_do_not_see_one_another():
    """Two samples in one call give what each gives alone: norms, convolutions and matrices are the sample's own."""
    coords, labels, params, grad, shape = make(5)
    p = {k: v.to(DEV) for k, v in params.items()}
    whole, _ = ours(coords.to(DEV), labels.to(DEV), p, shape)
    for b in range(shape[0]):
        mine = coords[:, 0] == b
        c = coords[mine].clone()
        c[:, 0] = 0
        q = dict(p, head=p["head"][b:b + 1], head_b=p["head_b"][b:b + 1])
        alone, _ = ours(c.contiguous().to(DEV), labels[mine].to(DEV), q, torch.Size((1,) + tuple(shape[1:])))
        scale = whole.abs().max().item()
        assert (alone - whole[mine.to(DEV)]).abs().max().item() <= 1e-3 * scale


def test_negated_gradients():
    """A gradient that says only by a flag that it is negated."""
    from flexgemm_b200.ops.embedding import sparse_embedding
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x = torch.randn(70, 16, device=DEV, requires_grad=True)
    w = torch.randn(2, 16, 16, device=DEV, requires_grad=True)
    ends = torch.tensor([0, 30, 70], device=DEV)
    for out, leaf in ((sparse_embedding(torch.arange(70, device=DEV), x, 2.0), x), (sparse_group_norm(x, ends, 4), x), (sparse_grouped_linear(x, ends, w), w)):
        dy = torch.randn_like(out)
        want = torch.autograd.grad(out, leaf, -dy, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(out, leaf, torch._neg_view(dy))[0], want)


def test_two_streams_at_once():
    coords, labels, params, grad, shape = make(6)
    p = {k: v.to(DEV) for k, v in params.items()}
    c, lab = coords.to(DEV), labels.to(DEV)
    want, cache = ours(c, lab, p, shape)
    ours.cache = cache
    try:
        want, _ = ours(c, lab, p, shape)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(4):
                    outs.append(ours(c, lab, p, shape)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    finally:
        ours.cache = None
