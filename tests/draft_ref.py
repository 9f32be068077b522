"""Plain float64 forms of the operators for drafted tokens and of drawing tokens,
row by row from their definitions.  The bounds of tree attention are those of
paged_ref: its scores and sums are the same, only which slots a row sees and how
far away they are is not."""

import math
from fractions import Fraction

import numpy as np
import torch

from paged_ref import E, gather, half_step


def closure(parents):
    """bool [n, n]: node j is node i or an ancestor of it."""
    n = len(parents)
    a = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            a[i] = a[p]
        a[i, i] = True
    return a


def pack(family, words):
    """Rows of bits as int64 words; columns past them are dropped."""
    out = np.zeros((len(family), words), np.uint64)
    for i, row in enumerate(family):
        for j in np.flatnonzero(row):
            if j < 64 * words:
                out[i, j // 64] |= np.uint64(1 << int(j % 64))
    return torch.from_numpy(out.view(np.int64))


def tree_attention(q, k, v, table, lens, families, cu, *, scale, softcap=0.0, slopes=None, window=0, prefix=None):
    """families: bool [n, >= n] of each sequence.  (out, lse, bound of out, bound of lse)."""
    T, H, D = q.shape
    KVH = k.shape[1]
    g, u = H // KVH, half_step(q.dtype)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    ob = torch.full((T, H, D), 2.0**-25, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    lb = torch.zeros(T, H, dtype=torch.float64)
    for s in range(table.shape[0]):
        start, n, total = int(cu[s]), int(cu[s + 1]) - int(cu[s]), int(lens[s])
        off = total - n
        fam = torch.as_tensor(np.asarray(families[s])[:, :n]).long() if n else torch.zeros(0, 0, dtype=torch.long)
        j = torch.arange(total)
        for i in range(n):
            bits = fam[i]
            above = bits.sum() - bits.cumsum(0)          # set bits over node x
            pos = off - 1 + int(bits.sum())
            away = pos - j
            see = torch.ones(total, dtype=torch.bool)
            for x in range(n):                            # the chunk's slots that exist
                if off + x >= 0:
                    away[off + x] = above[x]
                    see[off + x] = bool(bits[x])
            if window:
                see &= away < window
            if prefix is not None:
                see |= (j < int(prefix[s])) & (j < off)
            for kv in range(KVH):
                kk, ok = gather(k, table[s], total, kv)
                vv, _ = gather(v, table[s], total, kv)
                vis = see & ok
                hs = slice(kv * g, (kv + 1) * g)
                qq = q[start + i, hs].double().cpu()
                if not bool(vis.any()):
                    continue
                x = qq @ kk[vis].t() * scale
                size = torch.nan_to_num(qq.abs() @ kk[vis].abs().t() * scale, nan=0.0, posinf=0.0)
                dx = (D + 4) * E * float(size.max())
                if softcap:
                    x = torch.tanh(x / softcap) * softcap
                    dx += 8 * softcap * E
                if slopes is not None:
                    bias = slopes[hs].double().cpu()[:, None] * away[vis].abs().double()
                    x = x - bias
                    dx += 4 * E * float(bias.max())
                dx += 4 * E * float(torch.nan_to_num(x.abs(), nan=0.0, posinf=0.0).max())
                top = x.amax(-1, keepdim=True)
                p = torch.exp(x - top)
                l = p.sum(-1, keepdim=True)
                w = p / l
                o, a = w @ vv[vis], torch.nan_to_num(w) @ torch.nan_to_num(vv[vis]).abs()
                vmax = float(torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0).abs().max())
                out[start + i, hs] = o
                ob[start + i, hs] += u * (a + o.abs()) + (2 * dx + 2 * (total + 8) * E) * a + total * 2.0**-32 * vmax
                r = (top + torch.log(l)).squeeze(-1)
                lse[start + i, hs] = r
                lb[start + i, hs] = dx + (total + 8) * E + 2 * E * torch.nan_to_num(r).abs()
    return out, lse, ob, lb


def accept(drawn, drafted, parents, steps):
    """(path, tokens) of one tree."""
    path = [0] if len(parents) else []
    while path and len(path) < steps:
        child = [i for i, p in enumerate(parents) if p == path[-1] and i > p and drafted[i] == drawn[p]]
        if not child:
            break
        path.append(child[0])
    return path, [drawn[i] for i in path]


def passes(w, n, u):
    """Whether the first n weights add up to more than u times all of them, exactly."""
    add = lambda a: sum(Fraction(float(v)) * int(m) for v, m in zip(*np.unique(a, return_counts=True)))  # noqa: E731
    return add(w[:n]) > Fraction(u) * add(w)


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share) of one row of float64 logits; settings as float32 holds them."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    f = lambda v: float(np.float32(v))  # noqa: E731
    u = f(u)
    u = min(u, 1 - 2.0**-24) if u > 0 else 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, -math.inf
    if not f(temperature) > 0:
        return int(order[0]), 0.0
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        z = np.where(x[order] == top, 0.0, (x[order] - top) / f(temperature))
    w = np.exp(z)
    if top_k > 0:
        order, w, z = order[:top_k], w[:top_k], z[:top_k]
    if f(top_p) < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < f(top_p) * w.sum()).sum()))
        order, w, z = order[:n], w[:n], z[:n]
    least = min(f(min_p), 1.0) if f(min_p) > 0 else 0.0
    stay = w >= least
    order, w, z = order[stay], w[stay], z[stay]
    by = np.argsort(order)
    order, w, z = order[by], w[by], z[by]
    c = np.cumsum(w)
    i = int(np.searchsorted(c, u * c[-1], side="right"))
    # A running sum that is the aim but for this sum's own rounding (few values: halves of a row that hold the same
    # ones) is compared once more, as the fraction that its weights add up to.
    while i > 0 and abs(c[i - 1] - u * c[-1]) < 1e-12 * c[-1] and passes(w, i, u):
        i -= 1
    while i + 1 < len(w) and abs(c[i] - u * c[-1]) < 1e-12 * c[-1] and not passes(w, i + 1, u):
        i += 1
    return int(order[i]), float(z[i] - math.log(c[-1]))
