"""Plain float64 forms of the paged-cache operators, row by row from their
definitions, and the error bounds that the tests hold the kernels to.

Bounds: u = eps(type) / 2 is half a rounding step of the tensors' type, e =
2^-24 that of fp32.  A score sums D products in fp32: off by at most (D + 4) e
S, S = scale * max sum_i |q_i k_i|; a cap's exp and reciprocal (1 ulp each) add
8 cap e, a distance bias 4 e of its size, the change to units of log 2 and exp2's
argument 4 e |x|.  Call that dx.  A weight is then off by dx + 4 e of itself, and
once more by u where it is rounded for the product with v; sums of N terms add
N e.  With A = sum_j p_j |v_j| (p normalised):
  |out - o| <= u (A + |o|) + (2 dx + 2 (N + 8) e) A + tiny
  |lse - log l| <= dx + (N + 8) e + 2 e |lse|
tiny: weights under fp16's range (2^-32 of the row's largest each) and outputs
under it (2^-25)."""

import torch

E = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def chunk_of(s, rows, cu):
    return (s, 1) if cu is None else (int(cu[s]), int(cu[s + 1]) - int(cu[s]))


def gather(cache, table_row, total, kv):
    """Slots of one sequence and head, float64, absent ones as zeros, and which exist."""
    P, _, ps, D = cache.shape
    j = torch.arange(total)
    page = table_row.long().cpu()[j // ps] if total else torch.zeros(0, dtype=torch.long)
    ok = (page >= 0) & (page < P)
    x = cache[page.clamp(0, P - 1).to(cache.device), kv, (j % ps).to(cache.device)].double().cpu()
    x[~ok] = 0
    return x, ok


def seq_scores(q, k, table, lens, cu, s, kv, *, scale, softcap=0.0, slopes=None, window=0, prefix=None):
    """Scores [g, n, total] with -inf where hidden, and their fp32 error bound dx."""
    H, D = q.shape[1:]
    g = H // k.shape[1]
    start, n = chunk_of(s, q.shape[0], cu)
    total = int(lens[s])
    kk, ok = gather(k, table[s], total, kv)
    qq = q[start:start + n, kv * g:(kv + 1) * g].double().cpu().transpose(0, 1)
    x = torch.matmul(qq, kk.t().contiguous()) * scale
    fin = torch.nan_to_num(torch.matmul(qq.abs(), kk.abs().t().contiguous()) * scale, nan=0.0, posinf=0.0)
    dx = (D + 4) * E * float(fin.max()) if fin.numel() else 0.0
    if softcap:
        x = torch.tanh(x / softcap) * softcap
        dx += 8 * softcap * E
    p = torch.arange(total - n, total)[:, None]
    j = torch.arange(total)[None]
    if slopes is not None:
        bias = slopes[kv * g:(kv + 1) * g].double().cpu()[:, None, None] * (p - j).abs().double()
        x = x - bias
        dx += 4 * E * (float(bias.max()) if bias.numel() else 0.0)
    fin = torch.nan_to_num(x.abs(), nan=0.0, posinf=0.0)
    dx += 4 * E * (float(fin.max()) if fin.numel() else 0.0)
    see = j <= p
    if window:
        see = see & (j > p - window)
    if prefix is not None:
        see = see | (j < int(prefix[s]))
    see = see & ok[None]
    return torch.where(see, x, torch.full_like(x, float("-inf"))), dx, see, (start, n, total)


def attention(q, k, v, table, lens, cu=None, **how):
    """(out, lse, bound of out, bound of lse), float64 on the CPU."""
    T, H, D = q.shape
    g = H // k.shape[1]
    u = half_step(q.dtype)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    ob = torch.full((T, H, D), 2.0**-25, dtype=torch.float64)
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64)
    lb = torch.zeros(T, H, dtype=torch.float64)
    for s in range(table.shape[0]):
        for kv in range(k.shape[1]):
            x, dx, see, (start, n, total) = seq_scores(q, k, table, lens, cu, s, kv, **how)
            if n == 0 or total == 0:
                continue
            vv, _ = gather(v, table[s], total, kv)
            top = x.amax(-1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(x - top)
            l = p.sum(-1, keepdim=True)
            w = torch.where(l == 0, torch.zeros_like(p), p / l)
            # a hidden slot takes no part, whatever it holds
            hidden = ~see[None]
            o = torch.zeros(g, n, D, dtype=torch.float64)
            for i in range(n):
                vis = see[i]
                o[:, i] = torch.matmul(w[:, i][:, vis], vv[vis])
            a = torch.matmul(torch.nan_to_num(torch.where(hidden, torch.zeros_like(w), w)), torch.nan_to_num(vv).abs())
            hs = slice(kv * g, (kv + 1) * g)
            rows = slice(start, start + n)
            out[rows, hs] = o.transpose(0, 1)
            vmax = float(torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0).abs().max())
            ob[rows, hs] += (u * (a + o.abs()) + (2 * dx + 2 * (total + 8) * E) * a + total * 2.0**-32 * vmax).transpose(0, 1)
            r = (top + torch.log(l)).squeeze(-1)
            lse[rows, hs] = r.t()
            lb[rows, hs] = (dx + (total + 8) * E + 2 * E * torch.nan_to_num(r, neginf=0.0).abs()).t()
    return out, lse, ob, lb


def mass(q, k, table, lens, lse, cu=None, **how):
    """(mass, bound): weights off by dx + 4 e (1 + |lse|) each, sums of r rows by 2 (r^(1/2) + 40) e: 16 rows, then
    16 blocks, then all."""
    H = q.shape[1]
    b, kvh, ps = table.shape[0], k.shape[1], k.shape[2]
    g = H // kvh
    m = torch.zeros(b, kvh, table.shape[1] * ps, dtype=torch.float64)
    bound = torch.zeros_like(m)
    for s in range(b):
        for kv in range(kvh):
            x, dx, see, (start, n, total) = seq_scores(q, k, table, lens, cu, s, kv, **how)
            if n == 0 or total == 0:
                continue
            given = lse[start:start + n, kv * g:(kv + 1) * g].double().cpu().t()
            w = torch.exp(x - given[..., None])
            w = torch.where(see[None] & (given[..., None] > float("-inf")), w, torch.zeros_like(w))
            t = w.sum((0, 1))
            m[s, kv, :total] = t
            far = float(torch.nan_to_num(given, neginf=0.0).abs().max())
            bound[s, kv, :total] = t * (dx + (4 * (1 + far) + 4 * (n * g) ** 0.5 + 80) * E)
    return m, bound + 2.0**-120


def keep(mass_row, total, budget, recent):
    """Slots that stay of one head's `total`, ascending."""
    if total <= budget:
        return list(range(total))
    old = max(0, total - recent)

    def key(j):
        x = float(mass_row[j])
        return (0, 0.0, j) if x != x else (1, -x, j)

    return sorted(sorted(range(old), key=key)[:budget - (total - old)]) + list(range(old, total))
