"""The layers that stand between the convolutions of a network on sparse voxels, as cases that can be timed.

Features are ``[N, C]`` rows; ``offsets`` (``[B + 1]``, on the GPU) says where the rows of each of ``B`` samples or experts
begin, and rows behind ``offsets[B]`` belong to nobody.

* ``embed``   ``sparse_embedding``: voxel labels become feature rows, ``scale * table[label]``; the gradient of the table
              is the sum of the rows of each label.
* ``norm``    ``sparse_group_norm``: mean and variance of each sample's channel groups, an affine map for each channel and
              an activation, in front of a convolution.
* ``linear``  ``sparse_grouped_linear``: every sample or expert multiplies its rows by a matrix of its own.

``train`` runs the backward pass for all inputs that carry a gradient, otherwise the call is made under ``no_grad``.  The
sizes follow the library's benchmarks and tests: spherical shells at resolutions 32 to 1024 (2520 to some 10^6 voxels), 1
to 8 objects, 16 to 1024 channels; the numbers of experts, labels and short samples are generic.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _embed(name, **kw):
    return dict(dict(name=name, kind="embed", rows=2520, labels=256, c=64, dtype="fp16", wide=False, skew=1.0, scale=1.0, padding=False, train=True), **kw)


def _norm(name, **kw):
    return dict(dict(name=name, kind="norm", rows=2520, samples=1, c=64, groups=32, dtype="fp16", act="silu", skew=0.5, spare=0, train=True), **kw)


def _linear(name, **kw):
    return dict(dict(name=name, kind="linear", rows=2520, groups=4, ci=64, co=64, dtype="fp16", bias=True, skew=0.5, spare=0, train=True), **kw)


def listed():
    return [
        # labels of a small object at inference: the smallest call
        _embed("embed_small", train=False),
        # the labels of a large surface, a few of them nearly everywhere
        _embed("embed_surface_train", rows=166000, labels=4096, c=256, wide=True, scale=16.0),
        # two objects at the highest resolution, narrow features, a large codebook, voxels without a label
        _embed("embed_hires_train", rows=1320000, labels=50000, c=64, dtype="bf16", skew=0.3, padding=True),
        # a small object at inference
        _norm("norm_small", train=False),
        # the residual stack's shape: four objects, 512 channels
        _norm("norm_stack_train", rows=39872, samples=4, c=512, dtype="bf16"),
        # the headline benchmark's shape: one large surface
        _norm("norm_surface_train", rows=166000, c=256),
        # thousands of short samples, some of them empty; channel groups off the powers of two; the buffer has spare rows
        _norm("norm_short_train", rows=80000, samples=2048, c=96, groups=12, dtype="fp32", act="none", skew=1.0, spare=777),
        # a few rows for many experts, as when a model answers step by step
        _linear("linear_step", rows=24, groups=64, ci=512, co=1024, dtype="bf16", skew=1.0, train=False),
        # a matrix for each of four objects
        _linear("linear_stack_train", rows=39872, groups=4, ci=512, co=512, dtype="bf16"),
        # a large surface dealt to 27 experts unevenly
        _linear("linear_surface_train", rows=166000, groups=27, ci=256, co=256, bias=False, skew=1.0),
        # accurate fp32, odd sizes
        _linear("linear_odd_train", rows=10007, groups=13, ci=100, co=36, dtype="fp32", skew=1.5, spare=61),
        # the largest products
        _linear("linear_wide_train", rows=131072, groups=16, ci=1024, co=1024, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "linear"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    train = rng.random() < 0.7
    if kind == "embed":
        c = rng.choice([16, 24, 36, 64, 100, 128, 256, 512])
        rows = _log(rng, 1, 84_000_000 // c if c > 64 else 1_300_000)
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return dict(kind=kind, rows=rows, labels=_log(rng, 1, 60000), c=c, dtype=dtype, wide=rng.random() < 0.5, skew=rng.choice([0.0, 0.3, 1.0, 2.0]),
                    scale=rng.choice([1.0, 0.5, math.sqrt(c)]), padding=rng.random() < 0.3, train=train)
    if kind == "norm":
        c = rng.choice([16, 20, 32, 48, 64, 96, 100, 128, 256, 320, 512, 1024])
        groups = rng.choice([g for g in (1, 2, 4, 5, 8, 10, 16, 25, 32, c) if c % g == 0])
        rows = _log(rng, 1, 42_000_000 // (c * (2 if dtype == "fp32" else 1)))
        samples = min(_log(rng, 1, 3000), 2 * rows) if rng.random() < 0.4 else rng.randint(1, 8)
        return dict(kind=kind, rows=rows, samples=samples, c=c, groups=groups, dtype=dtype, act=rng.choice(["silu", "silu", "none"]),
                    skew=rng.choice([0.0, 0.5, 1.5]), spare=rng.choice([0, 0, rng.randint(1, 300)]), train=train)
    ci, co = (rng.choice([6, 16, 36, 64, 100, 128, 200, 256, 384, 512, 1024]) for _ in range(2))
    most = min(170_000, 130_000_000_000 // (ci * co) // (8 if dtype == "fp32" else 1))
    return dict(kind=kind, rows=_log(rng, 1, most), groups=_log(rng, 1, 64), ci=ci, co=co, dtype=dtype, bias=rng.random() < 0.6,
                skew=rng.choice([0.0, 0.5, 1.5]), spare=rng.choice([0, 0, rng.randint(1, 300)]), train=train)


def _lengths(rows, parts, skew, seed):
    """Rows of each part: they add up to `rows`; the larger `skew`, the less even."""
    r = np.random.RandomState(seed % (1 << 31))
    share = np.exp(skew * r.standard_normal(parts))
    if skew >= 1.0 and parts > 4:
        share[r.randint(0, parts, max(1, parts // 8))] = 0.0  # some get nothing
    if share.sum() == 0.0:
        share[:] = 1.0
    return r.multinomial(rows, share / share.sum())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def randn(*size, scale=1.0, dtype=t):
        return (torch.randn(*size, generator=g, device="cuda") * scale).to(dtype)

    s = {"case": case}
    if case["kind"] == "embed":
        rows, labels, c = case["rows"], case["labels"], case["c"]
        # label k with a probability that falls like (k + 1)^-skew, the numbering shuffled; neighbours mostly share a label
        weight = torch.arange(1, labels + 1, dtype=torch.float64) ** -case["skew"]
        perm = torch.randperm(labels, generator=torch.Generator().manual_seed(seed + 1)).cuda()
        ends = (weight.cumsum(0) / weight.sum()).cuda()
        runs = torch.searchsorted(ends, torch.rand(rows // 4 + 1, generator=g, device="cuda", dtype=torch.float64)).clamp(max=labels - 1)
        place = torch.arange(rows, device="cuda") // 4
        apart = torch.rand(rows, generator=g, device="cuda") < 0.5
        other = torch.searchsorted(ends, torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)).clamp(max=labels - 1)
        s["indices"] = perm[torch.where(apart, other, runs[place])].to(torch.int64 if case["wide"] else torch.int32)
        s["table"] = randn(labels, c).requires_grad_(case["train"])
        s["padding"] = labels // 2 if case["padding"] else None
        if case["train"]:
            s["grad"] = randn(rows, c)
        return s
    rows, spare = case["rows"], case["spare"]
    parts = case["samples"] if case["kind"] == "norm" else case["groups"]
    lengths = _lengths(rows, parts, case["skew"], seed)
    s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
    if case["kind"] == "norm":
        c = case["c"]
        # features as a convolution leaves them: every channel with a mean and a spread of its own
        mean = torch.randn(c, generator=g, device="cuda")
        spread = torch.rand(c, generator=g, device="cuda") * 1.5 + 0.25
        s["feats"] = (torch.randn(rows + spare, c, generator=g, device="cuda") * spread + mean).to(t).requires_grad_(case["train"])
        s["weight"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(t).requires_grad_(case["train"])
        s["bias"] = randn(c, scale=0.2).requires_grad_(case["train"])
        if case["train"]:
            s["grad"] = randn(rows + spare, c)
        return s
    ci, co = case["ci"], case["co"]
    s["longest"] = int(lengths.max())
    s["feats"] = randn(rows + spare, ci).requires_grad_(case["train"])
    s["weight"] = randn(parts, co, ci, scale=1 / math.sqrt(ci)).requires_grad_(case["train"])
    s["bias"] = randn(parts, co).requires_grad_(case["train"]) if case["bias"] else None
    if case["train"]:
        s["grad"] = randn(rows + spare, co)
    return s


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    case = s["case"]
    if case["kind"] == "embed":
        from flexgemm_b200.ops.embedding import sparse_embedding

        def forward():
            return sparse_embedding(s["indices"], s["table"], scale=case["scale"], padding_idx=s["padding"])
        inputs = [s["table"]]
    elif case["kind"] == "norm":
        from flexgemm_b200.ops.group_norm import sparse_group_norm

        def forward():
            return sparse_group_norm(s["feats"], s["offsets"], case["groups"], s["weight"], s["bias"], eps=1e-5,
                                     activation=None if case["act"] == "none" else case["act"])
        inputs = [s["feats"], s["weight"], s["bias"]]
    else:
        from flexgemm_b200.kernels import config
        from flexgemm_b200.ops.grouped_linear import sparse_grouped_linear
        config.allow_tf32 = False  # fp32 products are accurate ones

        def forward():
            return sparse_grouped_linear(s["feats"], s["offsets"], s["weight"], s["bias"])
        inputs = [s["feats"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else [])
    if not case["train"]:
        with torch.no_grad():
            return {"out": forward()}
    out = forward()
    return {"out": out, "grads": list(torch.autograd.grad(out, inputs, s["grad"]))}


# ------------------------------------------------------------------ the plain forms
@torch.no_grad()
def _plain(s):
    return {"embed": _plain_embed, "norm": _plain_norm, "linear": _plain_linear}[s["case"]["kind"]](s, s["case"])


def _plain_embed(s, case):
    idx, table = s["indices"].long(), s["table"]
    out = (table.float()[idx] * case["scale"]).to(table.dtype)
    if not case["train"]:
        return {"out": out}
    rows = s["grad"].double() * case["scale"]  # a label may have 10^5 rows: their sum is taken in 64 bits
    if s["padding"] is not None:
        rows = rows * (idx != s["padding"]).unsqueeze(1)
    grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, idx, rows)
    return {"out": out, "grads": [grad.to(table.dtype)]}


def _owners(offsets, n):
    """The part that each row belongs to, and whether it belongs to one."""
    part = torch.searchsorted(offsets[1:].contiguous(), torch.arange(n, device=offsets.device, dtype=offsets.dtype), right=True)
    inside = part < offsets.numel() - 1
    return part.clamp(max=offsets.numel() - 2), inside


def _plain_norm(s, case):
    x, off, G = s["feats"].float(), s["offsets"].long(), case["groups"]
    n, c = x.shape
    part, inside = _owners(s["offsets"], n)
    count = ((off[1:] - off[:-1]) * (c // G)).clamp(min=1).unsqueeze(1)

    def mean_of(v):  # [n, G] -> the mean of each sample's entries [B, G]; a running sum in 64 bits, and its differences
        run = torch.cat([v.new_zeros(G, 1, dtype=torch.float64), v.double().t().contiguous().cumsum(1)], dim=1)
        return ((run[:, off[1:]] - run[:, off[:-1]]).t() / count).float()

    xg = x.view(n, G, c // G)
    d = xg - mean_of(xg.sum(2))[part].unsqueeze(2)
    rstd = 1 / torch.sqrt(mean_of((d * d).sum(2)) + 1e-5)
    rstd = rstd[part].unsqueeze(2)
    xhat = (d * rstd).view(n, c)
    w, b = s["weight"].float(), s["bias"].float()
    z = xhat * w + b
    sig = 1 / (1 + torch.exp(-z))
    y = z * sig if case["act"] == "silu" else z
    keep = inside.unsqueeze(1)
    out = torch.where(keep, y, torch.zeros_like(y)).to(s["feats"].dtype)
    if not case["train"]:
        return {"out": out}
    dz = s["grad"].float()
    if case["act"] == "silu":
        dz = dz * (sig * (1 + z * (1 - sig)))
    dz = torch.where(keep, dz, torch.zeros_like(dz))
    gw, gb = (dz * xhat).sum(0, dtype=torch.float64), dz.sum(0, dtype=torch.float64)
    dh = (dz * w).view(n, G, c // G)
    hg = xhat.view(n, G, c // G)
    m1, m2 = mean_of(dh.sum(2))[part].unsqueeze(2), mean_of((dh * hg).sum(2))[part].unsqueeze(2)
    gx = (rstd * (dh - m1 - hg * m2)).view(n, c)
    gx = torch.where(keep, gx, torch.zeros_like(gx))
    t = s["feats"].dtype
    return {"out": out, "grads": [gx.to(t), gw.to(t), gb.to(t)]}


def _plain_linear(s, case):
    x, w, off = s["feats"], s["weight"].float(), s["offsets"].long()
    n, t = x.shape[0], x.dtype
    G, co, ci = w.shape
    part, inside = _owners(s["offsets"], n)
    longest = max(s["longest"], 1)
    slot = part * longest + torch.arange(n, device=x.device) - off[part]  # a row's place among its part's, all padded to the longest
    slot = torch.where(inside, slot, torch.full_like(slot, G * longest))

    def spread(v):
        p = torch.zeros(G * longest + 1, v.shape[1], device=v.device)
        p[slot] = v.float()
        return p[:-1].view(G, longest, v.shape[1])

    def collect(p):
        p = p.reshape(G * longest, -1)
        return torch.where(inside.unsqueeze(1), p[slot.clamp(max=G * longest - 1)], p.new_zeros(())).to(t)

    xp = spread(x)
    out = xp @ w.transpose(1, 2)
    if s["bias"] is not None:
        out = out + s["bias"].float().unsqueeze(1)
    out = collect(out)
    if not case["train"]:
        return {"out": out}
    gp = spread(s["grad"])
    grads = [collect(gp @ w), (gp.transpose(1, 2) @ xp).to(t)]
    if s["bias"] is not None:
        grads.append(gp.sum(1, dtype=torch.float64).to(t))
    return {"out": out, "grads": grads}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    rows, train = case["rows"], case["train"]
    if case["kind"] == "embed":
        c = case["c"]
        used = min(case["labels"], rows)
        once = rows * (8 if case["wide"] else 4)
        fwd = once + used * c * e + rows * c * e
        bwd = once + rows * c * e + case["labels"] * c * e
        return {"bytes": fwd + (bwd if train else 0), "flops": rows * c * (2 if train else 1)}
    if case["kind"] == "norm":
        x = rows * case["c"] * e
        return {"bytes": 2 * x + (3 * x if train else 0), "flops": rows * case["c"] * (30 if train else 12)}
    ci, co = case["ci"], case["co"]
    w = min(case["groups"], rows) * ci * co * e
    fwd = rows * (ci + co) * e + w
    bwd = rows * (co + ci) * e + rows * ci * e + w + case["groups"] * ci * co * e  # grad_out and feats read, both gradients written, the weight read
    return {"bytes": fwd + (bwd if train else 0), "flops": 2 * rows * ci * co * (3 if train else 1)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "embed":
            idx, table = s["indices"].long(), s["table"].double()
            out = torch.index_select(table, 0, idx).mul_(case["scale"])
            if not case["train"]:
                return {"out": out}
            # rows in the order of their labels, summed by differences of the running sum
            keep = torch.ones(idx.numel(), dtype=torch.bool, device="cuda") if s["padding"] is None else idx != s["padding"]
            idx, rows = idx[keep], s["grad"][keep].double()
            order = torch.argsort(idx, stable=True)
            total = torch.cat([rows.new_zeros(1, case["c"]), rows[order].cumsum(0)])
            ends = torch.bincount(idx, minlength=case["labels"]).cumsum(0)
            starts = torch.cat([ends.new_zeros(1), ends[:-1]])
            return {"out": out, "grads": [(total[ends] - total[starts]) * case["scale"]]}
        bounds = s["offsets"].tolist()
        x = s["feats"].double()
        out = torch.zeros(x.shape[0], case["c"] if case["kind"] == "norm" else case["co"], dtype=torch.float64, device="cuda")
        w = s["weight"].double()
        b = s["bias"].double() if s["bias"] is not None else None
        dy = s["grad"].double() if case["train"] else None
        gx = torch.zeros_like(x)
        gw = torch.zeros_like(w)
        gb = torch.zeros_like(b) if b is not None else None
        for i, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
            if hi == lo:
                continue
            if case["kind"] == "linear":
                out[lo:hi] = x[lo:hi] @ w[i].T + (b[i] if b is not None else 0.0)
                if case["train"]:
                    gx[lo:hi] = dy[lo:hi] @ w[i]
                    gw[i] = dy[lo:hi].T @ x[lo:hi]
                    if b is not None:
                        gb[i] = dy[lo:hi].sum(0)
                continue
            c, G = case["c"], case["groups"]
            v = x[lo:hi].reshape(hi - lo, G, c // G)
            var, mean = torch.var_mean(v, dim=(0, 2), unbiased=False, keepdim=True)
            r = (var + 1e-5) ** -0.5
            h = ((v - mean) * r).reshape(hi - lo, c)
            z = h * w + b
            p = torch.sigmoid(z)
            out[lo:hi] = z * p if case["act"] == "silu" else z
            if case["train"]:
                dz = dy[lo:hi] * (p + z * p * (1 - p)) if case["act"] == "silu" else dy[lo:hi]
                gw += (dz * h).sum(0)
                gb += dz.sum(0)
                q = (dz * w).reshape(hi - lo, G, c // G)
                hv = h.reshape(hi - lo, G, c // G)
                gx[lo:hi] = (r * (q - q.mean(dim=(0, 2), keepdim=True) - hv * (q * hv).mean(dim=(0, 2), keepdim=True))).reshape(hi - lo, c)
        if not case["train"]:
            return {"out": out}
        return {"out": out, "grads": [gx, gw] + ([gb] if gb is not None else [])}
