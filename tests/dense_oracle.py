"""Plain statements in 64 bits, on the CPU, of the operators between sparse rows and dense matrices, and the error that each
kernel's arithmetic may make: sums of n terms in binary32 are off by at most n * 2^-24 times the sum of the terms' sizes, a
result's rounding to its type by half a step of it."""
import numpy as np
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half of the smallest step of the type, for results that are subnormal in it"""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]


def rows_of(ids, offsets, n_rows=None):
    """the elements of every row: a list of (row, first, last + 1)"""
    if offsets is None:
        n = ids.shape[0] if n_rows is None else n_rows
        k = ids.numel() // n if n else 0
        return [(r, r * k, r * k + k) for r in range(n)]
    o = offsets.tolist()
    return [(r, o[r], o[r + 1]) for r in range(len(o) - 1)]


def _parts(ids, weights, offsets, n_table):
    flat = ids.reshape(-1).cpu().long()
    w = torch.ones(flat.numel(), dtype=torch.float64) if weights is None else weights.reshape(-1).cpu().double()
    rows = rows_of(ids, offsets)
    row = torch.full((flat.numel(),), -1, dtype=torch.long)
    for r, lo, hi in rows:
        row[lo:hi] = r
    inside = (flat >= 0) & (flat < n_table) & (row >= 0)
    return flat, w, row, inside, len(rows)


def lookup(ids, table, weights=None, offsets=None, scale=1.0):
    """(result, sum of the sizes of its terms, number of terms), float64"""
    flat, w, row, inside, n = _parts(ids, weights, offsets, table.shape[0])
    t = table.cpu().double()
    out, size, terms = torch.zeros(n, t.shape[1]).double(), torch.zeros(n, t.shape[1]).double(), torch.zeros(n, 1).double()
    e = inside.nonzero()[:, 0]
    part = w[e, None] * t[flat[e]] * scale
    out.index_add_(0, row[e], part)
    size.index_add_(0, row[e], part.abs())
    terms.index_add_(0, row[e], torch.ones(e.numel(), 1).double())
    return out, size, terms


def lookup_grad_table(ids, grad, n_table, weights=None, offsets=None, scale=1.0):
    flat, w, row, inside, _ = _parts(ids, weights, offsets, n_table)
    g = grad.cpu().double()
    out, size, terms = torch.zeros(n_table, g.shape[1]).double(), torch.zeros(n_table, g.shape[1]).double(), torch.zeros(n_table, 1).double()
    e = inside.nonzero()[:, 0]
    part = w[e, None] * g[row[e]] * scale
    out.index_add_(0, flat[e], part)
    size.index_add_(0, flat[e], part.abs())
    terms.index_add_(0, flat[e], torch.ones(e.numel(), 1).double())
    return out, size, terms


def lookup_grad_weights(ids, grad, table, offsets=None, scale=1.0):
    flat, _, row, inside, _ = _parts(ids, None, offsets, table.shape[0])
    g, t = grad.cpu().double(), table.cpu().double()
    out, size = torch.zeros(flat.numel()).double(), torch.zeros(flat.numel()).double()
    e = inside.nonzero()[:, 0]
    part = g[row[e]] * t[flat[e]] * scale
    out[e], size[e] = part.sum(1), part.abs().sum(1)
    return out.view(ids.shape), size.view(ids.shape)


def assert_sum(got, want, size, terms, what=""):
    """a sum of `terms` products in binary32, scaled, rounded to got's type: each product and addition rounds once, and so
    does the scale"""
    tol = size * (terms + 3) * U32 + want.abs() * half_step(got.dtype) * (1 + 2.0 ** -7) + tiny(got.dtype)
    off = (got.cpu().double() - want).abs()
    assert got.shape == want.shape, what
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off - tol).max()):.3g} over its bound"


def sigmoid(x):
    return 1 / (1 + np.exp(-x))


def shares(s, score):
    """u of one row (float64), 0 where a score is not live"""
    live = s > -np.inf
    u = np.zeros_like(s)
    if live.any():
        if score == "softmax":
            m = s[live].max()
            with np.errstate(invalid="ignore"):
                u[live] = np.exp(np.where(s[live] == m, 0.0, s[live] - m))
            u /= u.sum()
        else:
            with np.errstate(over="ignore"):
                u[live] = sigmoid(s[live])
    return u


def logits(s, score):
    return s if score == "softmax" else np.minimum(s, 0) - np.log1p(np.exp(-np.abs(s)))


def softmax_over(x):
    with np.errstate(invalid="ignore"):
        e = np.exp(np.where(x == x.max(), 0.0, x - x.max()))
    return e / e.sum()


def winners(scores, k, score="softmax", bias=None, groups=1, top_groups=None, group_top=1, renormalise=False, scale=1.0):
    x = scores.cpu().double().numpy()
    n, e = x.shape
    top_groups = groups if top_groups is None else top_groups
    ids, weights = np.full((n, k), -1, np.int32), np.zeros((n, k))
    b = None if bias is None else bias.cpu().double().numpy()
    for r in range(n):
        s = x[r]
        u = shares(s, score)
        key = s.copy() if b is None and not (groups > 1 and group_top > 1) else (u if b is None else u + b)
        key[~(s > -np.inf)] = -np.inf
        key[np.isnan(key)] = -np.inf
        if groups > 1:
            parts = key.reshape(groups, -1)
            total = []
            for q in parts:
                best = np.sort(q[q > -np.inf])[::-1][:group_top]
                total.append(best.sum() if best.size else -np.inf)
            kept = np.argsort(-np.array(total), kind="stable")[:top_groups]
            mask = np.isin(np.arange(groups), kept)
            key = np.where(np.repeat(mask, e // groups), key, -np.inf)
        order = np.argsort(-key, kind="stable")[:k]
        order = np.sort(order[key[order] > -np.inf])
        ids[r, : order.size] = order
        if order.size:
            weights[r, : order.size] = scale * (softmax_over(logits(s[order], score)) if renormalise else u[order])
    return ids, weights


def winners_grad(scores, ids, grad_weights, score="softmax", renormalise=False, scale=1.0):
    """(gradient, a bound on the sizes of what is added up for each value)"""
    x, ids, g_all = scores.cpu().double().numpy(), ids.cpu().numpy(), grad_weights.cpu().double().numpy()
    out, size = np.zeros_like(x), np.zeros_like(x)
    for r in range(x.shape[0]):
        on = ids[r][ids[r] >= 0]
        g = g_all[r][ids[r] >= 0]
        if not on.size:
            continue
        s = x[r]
        if renormalise:
            p = softmax_over(logits(s[on], score))
            slope = 1.0 if score == "softmax" else sigmoid(-s[on])
            out[r, on] = scale * p * (g - (g * p).sum()) * slope
            size[r, on] = scale * p * (np.abs(g) + (np.abs(g) * p).sum()) * slope
        elif score == "sigmoid":
            out[r, on] = scale * g * sigmoid(s[on]) * sigmoid(-s[on])
            size[r, on] = np.abs(out[r, on])
        else:
            u = shares(s, score)
            dot, d_abs = (g * u[on]).sum(), (np.abs(g) * u[on]).sum()
            out[r], size[r] = -scale * u * dot, scale * u * d_abs
            out[r, on] += scale * u[on] * g
            size[r, on] += scale * u[on] * np.abs(g)
    return out, size
