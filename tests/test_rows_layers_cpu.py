"""CPU-side checks of the layers on ragged rows: their oracle against torch's autograd, and what the calls and the C entry
points refuse before anything is launched."""
import ctypes

import pytest
import torch

from flexgemm_b200 import _build, _cabi
from oracle import rows_oracle as orc


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _cabi.lib()


def test_oracle_group_norm_is_torchs():
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(31, 12, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(12, generator=g, dtype=torch.float64) for _ in range(2))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    parts = [torch.nn.functional.silu(torch.nn.functional.group_norm(leaves[0][lo:hi].T.unsqueeze(0), 3, leaves[1], leaves[2], 1e-3)[0].T)
             for lo, hi in ((0, 9), (9, 31))]
    y = torch.cat(parts)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = orc.group_norm(x, [(0, 9), (9, 9), (9, 31)], 3, w, b, 1e-3, True, dy)
    for got, want in ((ref["y"], y), (ref["dx"], grads[0]), (ref["dw"], grads[1]), (ref["db"], grads[2])):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)


def test_oracle_embedding_is_torchs():
    g = torch.Generator().manual_seed(2)
    idx = torch.randint(0, 7, (40,), generator=g)
    table = torch.randn(7, 5, generator=g, dtype=torch.float64).requires_grad_(True)
    dy = torch.randn(40, 5, generator=g, dtype=torch.float64)
    out = torch.nn.functional.embedding(idx, table, padding_idx=3) * 2.5
    (want,) = torch.autograd.grad(out, [table], dy)
    assert torch.equal(orc.embedding(idx, table.detach(), 2.5), out.detach())
    got, size = orc.embedding_grad(idx, dy, 7, 2.5, padding=3)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12) and (size >= got.abs() - 1e-12).all()


def test_layers_are_attributes_of_the_package(lib):
    """As they are documented, after an import of the package alone."""
    import os
    import subprocess
    import sys
    code = "import flexgemm_b200.ops as ops; ops.embedding.sparse_embedding, ops.group_norm.sparse_group_norm, ops.grouped_linear.sparse_grouped_linear, " \
           "ops.utils.sample_offsets, ops.grid_sample.grid_sample_3d"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_group_norm_refuses(lib):
    from flexgemm_b200.ops.group_norm import sparse_group_norm
    x, off = torch.randn(10, 8), torch.tensor([0, 4, 10])
    with pytest.raises(NotImplementedError):
        sparse_group_norm(x, off, 4)
    for bad in (0, 3, -2, 2.0, None):
        with pytest.raises(ValueError):
            sparse_group_norm(x, off, bad)
    with pytest.raises(ValueError):
        sparse_group_norm(x, off, 4, activation="gelu")
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError):
            sparse_group_norm(x, off, 4, eps=eps)
    for shape in ((8,), (2, 5, 8)):
        with pytest.raises(AssertionError):
            sparse_group_norm(torch.randn(shape), off, 4)
    with pytest.raises(TypeError):
        sparse_group_norm(x.double(), off, 4)
    with pytest.raises(TypeError):
        sparse_group_norm(x, off.float(), 4)
    for bad in (torch.tensor([0]), torch.zeros(2, 2, dtype=torch.int64)):
        with pytest.raises(AssertionError):
            sparse_group_norm(x, bad, 4)
    for bad in (torch.ones(7), torch.ones(1, 8)):
        with pytest.raises(AssertionError):
            sparse_group_norm(x, off, 4, bad)
        with pytest.raises(AssertionError):
            sparse_group_norm(x, off, 4, None, bad)
    with pytest.raises(TypeError):
        sparse_group_norm(x, off, 4, torch.ones(8).half())
    with pytest.raises(TypeError):
        sparse_group_norm(x.half(), off, 4, torch.ones(8).half(), torch.ones(8))


def test_embedding_refuses(lib):
    from flexgemm_b200.ops.embedding import sparse_embedding
    table, idx = torch.randn(10, 8), torch.tensor([1, 2])
    with pytest.raises(NotImplementedError):
        sparse_embedding(idx, table)
    with pytest.raises(AssertionError):
        sparse_embedding(idx, table[0])
    for bad in (idx.float(), idx.to(torch.int16), idx.bool()):
        with pytest.raises(TypeError):
            sparse_embedding(bad, table)
    with pytest.raises(TypeError):
        sparse_embedding(idx, table.double())
    for bad in (10, -1, -11):
        with pytest.raises(ValueError):
            sparse_embedding(idx, table, padding_idx=bad)
    for bad in (torch.randn(0, 8), torch.randn(3, 0)):
        with pytest.raises(ValueError):
            sparse_embedding(idx, bad)


def test_sample_offsets_refuses(lib):
    from flexgemm_b200.ops.utils import sample_offsets
    c = torch.zeros(5, 4, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        sample_offsets(c, 1)
    with pytest.raises(AssertionError):
        sample_offsets(c[:, :3], 1)
    for bad in (0, -1, 2 ** 24):
        with pytest.raises(ValueError):
            sample_offsets(c, bad)


def test_sample_offsets_of_other_types(lib):
    from flexgemm_b200.ops import utils
    for dtype in (torch.float32, torch.float16, torch.bool):
        with pytest.raises(TypeError):
            utils.sample_offsets(torch.zeros(5, 4, dtype=dtype), 1)
    b = [-2 ** 40, -2 ** 32, -1, 0, 1, 2, 3, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1]
    got = utils._int32_coords(torch.tensor(b).view(-1, 1).expand(-1, 4), 3)
    assert got.dtype == torch.int32 and got[:, 0].tolist() == [-1, -1, -1, 0, 1, 2, 3, 3, 3, 3, 3]
    for dtype in (torch.int16, torch.int8, torch.uint8):
        assert utils._int32_coords(torch.tensor([[0, 1, 2, 3]], dtype=dtype), 1).tolist() == [[0, 1, 2, 3]]


def offsets_on_host(lib, batch_indices, batch):
    """The entries, what is recorded, and whether all else was left alone."""
    import numpy as np
    coords = np.zeros((len(batch_indices), 4), np.int32)
    coords[:, 0] = batch_indices
    buffer = np.full(batch + 1 + 32, -7, np.int32)
    entries = buffer[16:-16]
    code = lib.fgb_sample_offsets_host(coords.ctypes.data, len(coords), batch, entries.ctypes.data)
    return entries.tolist(), code, bool((buffer[:16] == -7).all() and (buffer[-16:] == -7).all())


def test_sample_offsets_arithmetic(lib):
    """The kernel's rows replayed on the host.  Batch indices at the ends of int32, as padding often has them: they are
    recorded, and nothing is written but the entries (an index that is added to before it is cut would wrap, and write from
    2^31 entries in front of them on)."""
    low, high = -2 ** 31, 2 ** 31 - 1
    for lengths in ([7], [0, 3, 0, 0, 9, 1, 0], [0, 0], [3] * 9):
        rows = [b for b, k in enumerate(lengths) for _ in range(k)]
        want = [sum(lengths[:b]) for b in range(len(lengths) + 1)]
        assert offsets_on_host(lib, rows, len(lengths)) == (want, 0, True)
    values = [low, low + 1, -2, -1, 0, 1, 2, 3, 4, 2 ** 24, high - 1, high]
    for a in values:
        for b in values:
            for rows in ([a], [a, b], [0, a, b], [a, b, 1], [a, 0, b]):
                entries, code, alone = offsets_on_host(lib, rows, 3)
                good = rows == sorted(rows) and rows[0] >= 0 and rows[-1] < 3
                assert alone and code == (0 if good else _cabi.S_BAD_OFFSETS), rows
                assert all(0 <= e <= len(rows) for e in entries), rows
    assert offsets_on_host(lib, [0, 1, high, high], 2) == ([0, 1, 2], _cabi.S_BAD_OFFSETS, True)
    assert lib.fgb_sample_offsets_host(None, 1, 1, None) == -1 and lib.fgb_sample_offsets_host(None, 0, 0, None) == -2


class NormCall(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("x", "grad_out", "out", "offsets", "weight", "bias", "mean", "rstd", "grad_weight", "grad_bias")] + \
               [("n", ctypes.c_int64), ("samples", ctypes.c_int64)] + \
               [(k, ctypes.c_int32) for k in ("offsets_bits", "c", "groups", "dtype", "param_dtype", "act")] + \
               [("eps", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64), ("status", ctypes.c_void_p)]


def test_group_norm_workspace_without_rows(lib):
    """The gradients of weight and bias go through the workspace also where there is no row, and so no grad_out."""
    call = dict(mean=1 << 20, rstd=1 << 20, n=0, samples=3, offsets_bits=32, offsets=1 << 20, c=512, groups=8, dtype=_cabi.F16, param_dtype=_cabi.F16, eps=1e-5)
    size = lambda **kw: lib.fgb_group_norm_workspace_bytes(ctypes.byref(NormCall(**{**call, **kw})))
    need = size(grad_out=1 << 20)
    assert size() == 0 and need >= 512 * 8
    assert size(grad_weight=1 << 20) == size(grad_bias=1 << 20) == need
    assert lib.fgb_group_norm_backward(ctypes.byref(NormCall(**{**call, "grad_weight": 1 << 20})), None) == -1


def test_group_norm_entry_points_refuse(lib):
    """Pointers are numbers here: every call is refused before a launch."""
    good = dict(x=1 << 20, out=1 << 21, offsets=1 << 22, mean=1 << 23, rstd=1 << 23, n=100, samples=3, offsets_bits=32, c=64, groups=8,
                dtype=_cabi.F16, param_dtype=_cabi.F16, act=0, eps=1e-5, workspace=1 << 24, workspace_bytes=1 << 40)

    def rc(fn=lib.fgb_group_norm_forward, **kw):
        call = NormCall(**{**good, **kw})
        return fn(ctypes.byref(call), None)
    assert lib.fgb_group_norm_workspace_bytes(ctypes.byref(NormCall(**{**good, "n": 100000, "samples": 1}))) > 0
    assert lib.fgb_group_norm_workspace_bytes(ctypes.byref(NormCall(**good))) == 0   # one launch: nothing between its passes
    assert lib.fgb_group_norm_workspace_bytes(ctypes.byref(NormCall(**{**good, "grad_out": 1 << 25}))) > 0
    assert lib.fgb_group_norm_workspace_bytes(None) == -1 and lib.fgb_group_norm_forward(None, None) == -1
    for kw, code in ((dict(dtype=9), -3), (dict(param_dtype=_cabi.BF16), -3), (dict(act=7), -3), (dict(offsets_bits=16), -3), (dict(n=-1), -2),
                     (dict(n=1 << 31), -2), (dict(samples=0), -2), (dict(samples=1 << 24), -2), (dict(groups=7), -2), (dict(c=0), -2),
                     (dict(offsets_bits=0), -2), (dict(samples=(1 << 24) - 1, c=65536, groups=65536), -2), (dict(offsets=None), -1), (dict(x=None), -1), (dict(out=None), -1),
                     (dict(mean=None), -1), (dict(workspace=None, n=100000, samples=1), -1), (dict(x=(1 << 20) + 8), -4), (dict(workspace=(1 << 24) + 16), -4),
                     (dict(workspace_bytes=10, n=100000, samples=1), -5)):
        assert rc(**kw) == code, kw
    assert rc(lib.fgb_group_norm_backward) == -1   # no grad_out


class EmbeddingCall(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("indices", "table", "out", "grad_out", "grad_table")] + \
               [(k, ctypes.c_int64) for k in ("n", "rows", "padding_idx")] + [(k, ctypes.c_int32) for k in ("index_bits", "c", "dtype")] + \
               [("scale", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64), ("status", ctypes.c_void_p)]


def test_embedding_entry_points_refuse(lib):
    good = dict(indices=1 << 20, table=1 << 21, out=1 << 22, grad_out=1 << 22, grad_table=1 << 23, n=100, rows=30, padding_idx=-1, index_bits=32, c=64,
                dtype=_cabi.BF16, scale=1.0, workspace=1 << 24, workspace_bytes=1 << 40)

    def rc(fn, **kw):
        return fn(ctypes.byref(EmbeddingCall(**{**good, **kw})), None)
    assert lib.fgb_embedding_workspace_bytes(ctypes.byref(EmbeddingCall(**good))) > 0
    for fn in (lib.fgb_embedding_forward, lib.fgb_embedding_backward):
        assert fn(None, None) == -1
        for kw, code in ((dict(dtype=5), -3), (dict(index_bits=8), -3), (dict(n=1 << 30), -2), (dict(n=-1), -2), (dict(rows=0), -2), (dict(c=0), -2),
                         (dict(rows=2 ** 31 - 1), -2), (dict(indices=None), -1)):
            assert rc(fn, **kw) == code, kw
    assert rc(lib.fgb_embedding_forward, table=None) == -1 and rc(lib.fgb_embedding_forward, out=(1 << 22) + 2) == -4
    assert rc(lib.fgb_embedding_backward, grad_out=None) == -1 and rc(lib.fgb_embedding_backward, workspace_bytes=64) == -5
    assert rc(lib.fgb_embedding_backward, workspace=(1 << 24) + 8) == -4 and rc(lib.fgb_embedding_forward, n=0) == 0


def test_oracle_grouped_linear_is_torchs():
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(20, 6, generator=g, dtype=torch.float64), torch.randn(20, 4, generator=g, dtype=torch.float64)
    w, b = torch.randn(3, 4, 6, generator=g, dtype=torch.float64), torch.randn(3, 4, generator=g, dtype=torch.float64)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = torch.cat([torch.nn.functional.linear(leaves[0][lo:hi], leaves[1][i], leaves[2][i]) for i, (lo, hi) in enumerate(((0, 13), (13, 13), (13, 20)))])
    grads = torch.autograd.grad(y, leaves, dy)
    ref = orc.grouped_linear(x, [(0, 13), (13, 13), (13, 20)], w, b, dy)
    for got, want in ((ref["y"], y), (ref["dx"], grads[0]), (ref["dw"], grads[1]), (ref["db"], grads[2])):
        assert torch.allclose(got, want, rtol=1e-11, atol=1e-12)


def test_grouped_linear_refuses(lib):
    from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
    x, off, w, b = torch.randn(10, 8), torch.tensor([0, 4, 10]), torch.randn(2, 5, 8), torch.randn(2, 5)
    with pytest.raises(NotImplementedError):
        sparse_grouped_linear(x, off, w, b)
    for args in ((x[0], off, w), (x, off, w[0]), (x[:, :7], off, w), (x, off[:2], w), (x, off.view(1, 3), w), (x, off, w, b[:, :4]), (x, off, w, b[0])):
        with pytest.raises(AssertionError):
            sparse_grouped_linear(*args)
    for args in ((x.double(), off, w.double()), (x, off.float(), w), (x, off, w.half()), (x, off, w, b.half())):
        with pytest.raises(TypeError):
            sparse_grouped_linear(*args)
    most = lib.fgb_grouped_linear_max_groups()
    with pytest.raises(ValueError):
        sparse_grouped_linear(x, torch.zeros(most + 2, dtype=torch.int32), torch.zeros(most + 1, 1, 8))


class GroupedCall(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("x", "weight", "bias", "grad_out", "out", "grad_x", "grad_weight", "grad_bias", "offsets")] + \
               [("n", ctypes.c_int64), ("groups", ctypes.c_int64)] + [(k, ctypes.c_int32) for k in ("offsets_bits", "ci", "co", "dtype")] + \
               [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64), ("status", ctypes.c_void_p)]


def test_grouped_linear_entry_points_refuse(lib):
    good = dict(x=1 << 20, weight=1 << 21, out=1 << 22, grad_out=1 << 22, grad_x=1 << 23, grad_weight=1 << 23, offsets=1 << 24, n=1000, groups=3,
                offsets_bits=32, ci=64, co=72, dtype=_cabi.F16, workspace=1 << 25, workspace_bytes=1 << 40)

    def rc(fn, **kw):
        return fn(ctypes.byref(GroupedCall(**{**good, **kw})), None)
    for backward in (0, 1):
        for dtype in range(4):
            assert lib.fgb_grouped_linear_workspace_bytes(ctypes.byref(GroupedCall(**{**good, "dtype": dtype})), backward) > 0
        assert lib.fgb_grouped_linear_workspace_bytes(None, backward) == -1
    for fn in (lib.fgb_grouped_linear_forward, lib.fgb_grouped_linear_backward):
        assert fn(None, None) == -1
        for kw, code in ((dict(dtype=4), -3), (dict(offsets_bits=0), -3), (dict(n=-1), -2), (dict(n=1 << 31), -2), (dict(groups=0), -2), (dict(groups=1 << 20), -2),
                         (dict(ci=0), -2), (dict(co=1 << 17), -2), (dict(n=(1 << 31) - 300, ci=65536, co=65536, dtype=_cabi.F32_IEEE), -2), (dict(offsets=None), -1),
                         (dict(weight=None), -1), (dict(workspace=None), -1), (dict(x=(1 << 20) + 2), -4), (dict(weight=(1 << 21) + 8), -4),
                         (dict(workspace=(1 << 25) + 64), -4), (dict(workspace_bytes=100), -5)):
            assert rc(fn, **kw) == code, (fn.__name__, kw)
    assert rc(lib.fgb_grouped_linear_forward, out=None) == -1 and rc(lib.fgb_grouped_linear_forward, n=0) == 0
    assert rc(lib.fgb_grouped_linear_backward, grad_out=None) == -1 and rc(lib.fgb_grouped_linear_backward, grad_weight=None, grad_bias=1 << 23) == -1
