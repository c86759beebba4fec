"""The paged append, paged attention and sampling in 64 bits, one sequence or row at a time, from their definitions."""
import math

import numpy as np
import torch


def paged_rows(pool, table_row, n):
    """Positions 0 .. n-1 of a sequence from a [pages][heads][rows][d] pool: [heads][n][d] in 64 bits."""
    page = pool.shape[2]
    at = torch.arange(n, device=pool.device)
    return pool[table_row[at // page].long(), :, at % page].permute(1, 0, 2).double()


def attention(q, k, v, position, scale, window=0):
    """q [n][heads][d] at positions position .. over k, v [kv_heads][c][d]: out, lse, and what bounds the error: the
    same average of |v| and of e^(s - m) (the reciprocal of the largest probability)."""
    n, heads, d = q.shape
    kv, c, _ = k.shape
    s = torch.einsum("ngd,gcd->gnc", q.double(), k.repeat_interleave(heads // kv, 0)) * scale
    key, at = torch.arange(c, device=q.device), position + torch.arange(n, device=q.device)[:, None]
    hidden = (key > at) | (key <= at - window if window else torch.zeros_like(key, dtype=torch.bool))
    s = s.masked_fill(hidden, -math.inf)
    m = s.amax(-1, keepdim=True) if c else torch.full((heads, n, 1), -math.inf, dtype=torch.float64, device=q.device)
    e = torch.where(hidden, 0.0, (s - m.clamp(min=-1e300)).exp())
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total.clamp(min=1e-300), 0.0)
    vv = v.repeat_interleave(heads // kv, 0)
    vv = torch.where(vv.isfinite(), vv, 0.0) if c else vv
    out, size = p @ vv, p @ vv.abs()
    lse = torch.where(total > 0, m + total.log(), -math.inf)[..., 0]
    flat = (~hidden).double().expand(heads, n, c) @ vv.abs() / total.clamp(min=1.0)
    return out.transpose(0, 1), lse.T, size.transpose(0, 1), flat.transpose(0, 1)


def normed_rotated(x, gamma, position, eps, base):
    """x [n][heads][d] at positions position .., RMSNorm with gamma (or none) and rotation, in 64 bits."""
    x = x.double()
    n, _, d = x.shape
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
    angle = (position + torch.arange(n, device=x.device)).double()[:, None] * (float(base) ** (-2.0 * j / d))
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob, tokens that rounding in 64 bits could give instead) of one row, numpy long doubles."""
    x = np.asarray(logits, np.longdouble)
    x = np.where(np.isnan(x), -np.inf, x)
    if not len(x) or x.max() == -np.inf:
        return -1, -math.inf, {-1}
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not temperature > 0:
        return int(order[0]), 0.0, {int(order[0])}
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        e = np.where(x[order] == x[order[0]], 0.0, (x[order] - x[order[0]]) / np.longdouble(np.float32(temperature)))
    w = np.exp(e)
    if top_p < 1:
        want = np.longdouble(np.float32(top_p)) * w.sum()
        n = max(1, min(len(w), int(np.searchsorted(np.cumsum(w), want * (1 - np.longdouble(1e-15)))) + 1))
        order, w, e = order[:n], w[:n], e[:n]
    keep = w >= min(np.longdouble(np.float32(min_p)), 1) if min_p > 0 else w >= 0
    order, w, e = order[keep], w[keep], e[keep]
    by = np.argsort(order)
    order, w, e = order[by], w[by], e[by]
    sums = np.cumsum(w)
    target = np.longdouble(np.float32(u)) * sums[-1]
    at = [min(int(np.searchsorted(sums, target + s * sums[-1] * np.longdouble(1e-12), side="right")), len(w) - 1) for s in (0, -1, 1)]
    return int(order[at[0]]), float(e[at[0]] - np.log(sums[-1])), {int(order[i]) for i in at}
