"""Plain 64-bit forms of the layers on ragged rows, sample by sample: what the
tests of these layers compare with.  Written from the formulas; nothing of the
library is used."""
import torch


def silu_grad(z):
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def group_norm(x, bounds, groups, weight, bias, eps, silu, dy=None):
    """``bounds``: the ranges of the samples as a list of (lo, hi).  Returns y, and with ``dy`` also dx, dw, db and the
    magnitudes that error bounds are made of: of z, of dx's terms, of the sums' terms."""
    x = x.double()
    n, C = x.shape
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.double()
    out = {k: torch.zeros(n, C, dtype=torch.float64) for k in ("y", "dx", "z_size", "dx_size")}
    out |= {k: torch.zeros(C, dtype=torch.float64) for k in ("dw", "db", "dw_size", "db_size")}
    for lo, hi in bounds:
        if hi <= lo:
            continue
        v = x[lo:hi].reshape(hi - lo, groups, C // groups)
        mean = v.mean(dim=(0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean(dim=(0, 2), keepdim=True)
        r = 1 / torch.sqrt(var + eps)
        h = ((v - mean) * r).reshape(hi - lo, C)
        z = h * w + b
        out["y"][lo:hi] = z * torch.sigmoid(z) if silu else z
        r_c = r.expand_as(v).reshape(hi - lo, C)
        # a rounding of x - mean, or of the mean itself, counts this much in z
        out["z_size"][lo:hi] = (v.abs() + mean.abs()).reshape(hi - lo, C) * r_c * w.abs() + b.abs() + h.abs() * w.abs()
        if dy is None:
            continue
        dz = dy[lo:hi].double() * (silu_grad(z) if silu else 1.0)
        out["dw"] += (dz * h).sum(0)
        out["db"] += dz.sum(0)
        size = dy[lo:hi].double().abs() * (1 + out["z_size"][lo:hi])
        out["dw_size"] += (size * (1 + h.abs() + (v.abs() + mean.abs()).reshape(hi - lo, C) * r_c)).sum(0)
        out["db_size"] += size.sum(0)
        q = (dz * w).reshape(hi - lo, groups, C // groups)
        hg = h.reshape(hi - lo, groups, C // groups)
        m1, m2 = q.mean(dim=(0, 2), keepdim=True), (q * hg).mean(dim=(0, 2), keepdim=True)
        out["dx"][lo:hi] = (r * (q - m1 - hg * m2)).reshape(hi - lo, C)
        sw = (size * w.abs()).reshape(hi - lo, groups, C // groups)
        off = 1 + hg.abs() + (v.abs() + mean.abs()) * r
        out["dx_size"][lo:hi] = (r * (sw + (sw.mean(dim=(0, 2), keepdim=True) + (sw * off).mean(dim=(0, 2), keepdim=True) * off))).reshape(hi - lo, C)
    return out


def embedding(indices, table, scale):
    return table.double()[indices.long()] * scale


def embedding_grad(indices, grad, rows, scale, padding=None):
    """The gradient of the table, and the sum of its terms' magnitudes."""
    idx = indices.reshape(-1).long()
    g = grad.reshape(idx.numel(), -1).double() * scale
    if padding is not None:
        g = g * (idx != padding).unsqueeze(1)
    zero = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    return zero.index_add(0, idx, g), zero.index_add(0, idx, g.abs())


def grouped_linear(x, bounds, weight, bias, dy=None):
    """y, and with ``dy`` dx, dw, db; ``*_size``: the sums of the terms' magnitudes."""
    x, w = x.double(), weight.double()
    n, co, ci = x.shape[0], w.shape[1], w.shape[2]
    out = {"y": torch.zeros(n, co, dtype=torch.float64), "dx": torch.zeros(n, ci, dtype=torch.float64), "dw": torch.zeros_like(w),
           "db": torch.zeros(w.shape[0], co, dtype=torch.float64)}
    out |= {k + "_size": torch.zeros_like(v) for k, v in out.items()}
    for i, (lo, hi) in enumerate(bounds):
        if hi <= lo:
            continue
        b = bias[i].double() if bias is not None else torch.zeros(co, dtype=torch.float64)
        out["y"][lo:hi] = x[lo:hi] @ w[i].T + b
        out["y_size"][lo:hi] = x[lo:hi].abs() @ w[i].abs().T + b.abs()
        if dy is None:
            continue
        g = dy[lo:hi].double()
        out["dx"][lo:hi], out["dx_size"][lo:hi] = g @ w[i], g.abs() @ w[i].abs()
        out["dw"][i], out["dw_size"][i] = g.T @ x[lo:hi], g.abs().T @ x[lo:hi].abs()
        out["db"][i], out["db_size"][i] = g.sum(0), g.abs().sum(0)
    return out
