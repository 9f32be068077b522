"""Performance cases of the operators that serve a model from a paged key/value cache.

Kinds of case (``case["op"]``), each with an entry point of ``metal_native.paged``:

* ``rope``   -- rotary positions with one or several axes (time, height, width) for the rows of a
  fused q/k/v projection, the keys and values written into the pages of their sequences;
* ``attn``   -- attention of the newest tokens of every sequence (one token each, or a ragged chunk)
  over its pages: causal, or with a tanh cap on the scores, a bias that falls with distance, a
  sliding window and a prefix that every row sees;
* ``mass``   -- the attention weight that every cached key got from these tokens, summed over the
  rows and query heads that share the key;
* ``evict``  -- the cache cut down to a budget: per key/value head the newest slots and the slots of
  most accumulated weight move, in order, to other pages.

Caches are ``[pages, kv_heads, page_size, head_dim]`` with the pages of all sequences in random
order.  Inputs are made on the GPU from the seed alone: queries, keys and values N(0, 1) (what
normalised activations leave after a projection), accumulated weights with the heavy tail that
softmax rows sum to, many of them exactly zero.  How long the sequences are follows from the case
itself, so that its work does not depend on the seed.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False
DEVICE = "cuda:0"
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, dtype, heads, kv_heads, dim, page, b, lmin, lmax, nmin, nmax, mix=1, **more):
    """``b`` sequences of ``lmin..lmax`` cached tokens, the last ``nmin..nmax`` of them new (0: one
    each, a decode batch); ``mix`` picks the lengths in between."""
    c = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "b": b,
         "lmin": lmin, "lmax": lmax, "nmin": nmin, "nmax": nmax, "mix": mix, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token of a 7B decoder (28 query and 4 key/value heads) behind its 512-token cache: latency
        _case("rope_decode_b1", "rope", "fp16", 28, 4, 128, 16, 1, 513, 513, 0, 0, axes=1),
        # prompts with pictures: three axes, frequencies 16/24/24, ragged, about 8000 tokens at once
        _case("rope_axes_ragged", "rope", "bf16", 28, 4, 128, 16, 7, 300, 2300, 300, 2300, mix=4, axes=3),
        # the decode step that the framework's decoder runs: one token, 513 keys: latency
        _case("attn_decode_b1", "attn", "fp16", 28, 4, 128, 16, 1, 513, 513, 0, 0),
        # a serving batch of 48 conversations from a few tokens to 8000, with the rows' log sums kept
        _case("attn_decode_ragged_b48", "attn", "bf16", 32, 8, 128, 16, 48, 1, 8000, 0, 0, lse=True),
        # four long documents being continued: the cache is all there is to read
        _case("attn_decode_long", "attn", "fp16", 28, 4, 128, 64, 4, 90001, 131072, 0, 0),
        # fresh prompts of a batch, every token new
        _case("attn_prompts", "attn", "bf16", 28, 4, 128, 16, 7, 301, 2048, 301, 2048, mix=3, fresh=True),
        # one 4096-token chunk of a long prompt behind 28672 tokens that are cached
        _case("attn_chunk_long", "attn", "fp16", 28, 4, 128, 64, 1, 32768, 32768, 4096, 4096),
        # chunks of a small model with capped scores, distance bias, window and a shared prefix
        _case("attn_masked_chunks", "attn", "fp16", 14, 2, 64, 32, 5, 700, 3500, 33, 517, mix=2,
              softcap=30.0, bias=True, window=1000, prefix=77),
        # a decode batch that keeps track of which keys are used
        _case("mass_decode_b8", "mass", "fp16", 28, 4, 128, 16, 8, 2000, 16000, 0, 0),
        # the same for a chunk of 1500 tokens of two prompts
        _case("mass_chunk", "mass", "bf16", 28, 4, 128, 16, 2, 5000, 8191, 1100, 1500),
        # one conversation cut from 1100 slots to 512
        _case("evict_b1", "evict", "fp16", 28, 4, 128, 16, 1, 1100, 1100, 0, 0, budget=512, recent=64),
        # eight long ones cut to a quarter
        _case("evict_b8_long", "evict", "bf16", 32, 8, 128, 64, 8, 20011, 32768, 0, 0, budget=8192, recent=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "attn", "attn", "attn", "mass", "evict"))
    heads, kv_heads, dim = rng.choice(((28, 4, 128), (32, 8, 128), (14, 2, 64), (16, 16, 128), (24, 8, 64), (8, 1, 128)))
    dtype, page, mix = rng.choice(("fp16", "bf16")), rng.choice((16, 32, 64, 128)), rng.randrange(1 << 20)
    if op == "rope":
        n = _log(rng, 1, 2000)
        b = rng.randint(1, max(1, min(16, 8000 // n)))
        top = n + rng.randrange(1000)
        if rng.random() < 0.3:
            return _case(None, op, dtype, heads, kv_heads, dim, page, rng.randint(1, 100), 1, top, 0, 0, mix, axes=rng.choice((1, 2, 3)))
        return _case(None, op, dtype, heads, kv_heads, dim, page, b, n, top, max(1, n // 3), n, mix, axes=rng.choice((1, 2, 3)))
    if op == "evict":
        top = _log(rng, 200, 32768)
        budget = rng.randint(top // 8 + 1, top)
        b = rng.randint(1, max(1, min(8, 400_000_000 // (budget * kv_heads * dim * 8))))
        return _case(None, op, dtype, heads, kv_heads, dim, page, b, max(1, top // 3), top, 0, 0, mix,
                     budget=budget, recent=rng.randint(0, budget // 2))
    more = {}
    if op == "attn" and rng.random() < 0.5:
        more["lse"] = True
    if rng.random() < 0.4:
        more.update(softcap=rng.choice((0.0, 20.0, 50.0)), bias=rng.random() < 0.5,
                    window=rng.choice((0, rng.randint(1, 3000))), prefix=rng.choice((0, rng.randint(1, 400))))
    if rng.random() < 0.5:   # a decode batch
        top = _log(rng, 1, 65536)
        b = rng.randint(1, max(1, min(64, 900_000_000 // (top * kv_heads * dim * 4))))
        return _case(None, op, dtype, heads, kv_heads, dim, page, b, max(1, top // rng.choice((1, 3, 50))), top, 0, 0, mix, **more)
    n = _log(rng, 2, 2048)    # chunks
    top = n + _log(rng, 1, 8192)
    b = rng.randint(1, max(1, min(8, 4096 // n)))
    if rng.random() < 0.3:
        return _case(None, op, dtype, heads, kv_heads, dim, page, b, max(1, n // 4), n, max(1, n // 4), n, mix, fresh=True, **more)
    return _case(None, op, dtype, heads, kv_heads, dim, page, b, max(n, top // 2), top, max(1, n // 4), n, mix, **more)


def _spread(rng, n, lo, hi):
    """``n`` lengths over the logarithm of ``lo..hi``, both ends among them."""
    got = [_log(rng, lo, hi) for _ in range(n)]
    got[rng.randrange(n)] = lo
    got[rng.randrange(n)] = hi
    return got


def _lengths(case):
    """(cached tokens, new tokens) of each sequence; both from the case alone."""
    rng = random.Random(case["mix"])
    total = _spread(rng, case["b"], case["lmin"], case["lmax"])
    if case["nmax"] == 0:
        return total, [1] * case["b"]
    if case.get("fresh") or case["op"] == "rope" and case["lmin"] == case["nmin"]:
        return total, list(total)
    return total, [min(n, t) for n, t in zip(_spread(rng, case["b"], case["nmin"], case["nmax"]), total)]


def _sections(dim, axes):
    """Frequencies per axis: time gets a quarter, the others share the rest."""
    half = dim // 2
    return {1: (half,), 2: (half // 4, half - half // 4), 3: (half // 4, 3 * half // 8, half - half // 4 - 3 * half // 8)}[axes]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    h, kh, d, ps, b = case["heads"], case["kv_heads"], case["dim"], case["page"], case["b"]
    total, new = _lengths(case)
    pages = [-(-t // ps) for t in total]
    target = -(-case["budget"] // ps) if case["op"] == "evict" else 0
    pool = sum(pages) + b * target + 3
    order = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    rn = lambda *s: torch.randn(*s, device=DEVICE, generator=gen, dtype=torch.float32).to(dt)  # noqa: E731
    wide = max(pages)
    table = torch.full((b, wide), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    s = {"case": dict(case), "k": rn(pool, kh, ps, d), "v": rn(pool, kh, ps, d), "table": table,
         "lens": torch.tensor(total, dtype=torch.int32, device=DEVICE), "cu": None, "rows": sum(new), "most": max(new)}
    if case["nmax"]:
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
    t = s["rows"]
    if case["op"] == "rope":
        s["sections"] = _sections(d, case["axes"])
        s["axis"] = torch.tensor([a for a, n in enumerate(s["sections"]) for _ in range(n)], device=DEVICE)
        s["qkv"] = rn(t, (h + 2 * kh) * d)
        far = case["lmax"] + 1
        inv = 1.0e6 ** (-torch.arange(d // 2, device=DEVICE, dtype=torch.float64) / (d // 2))
        angle = torch.outer(torch.arange(far, device=DEVICE, dtype=torch.float64), inv)
        s["cos"] = torch.cat([angle.cos()] * 2, 1).float()
        s["sin"] = torch.cat([angle.sin()] * 2, 1).float()
        first = torch.cat([torch.arange(a - n, a, device=DEVICE) for a, n in zip(total, new)])
        s["pos"] = first if case["axes"] == 1 else torch.stack(
            [first] + [torch.randint(0, far, (t,), device=DEVICE, generator=gen) for _ in range(case["axes"] - 1)])
    elif case["op"] == "evict":
        u = torch.rand(b, kh, wide * ps, device=DEVICE, generator=gen)
        s["mass"] = torch.where(u < 0.2, torch.zeros_like(u), 3.0 * u ** 8)
        s["to"] = order[at:at + b * target].reshape(b, target).contiguous()
        s["budget"], s["recent"] = case["budget"], case["recent"]
    else:
        s["q"] = rn(t, h, d)
        s["scale"] = 1.0 / math.sqrt(d)
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEVICE, dtype=torch.float32) / h)
                       if case.get("bias") else None)
        s["prefix"] = (torch.full((b,), case["prefix"], dtype=torch.int32, device=DEVICE) if case.get("prefix") else None)
        if case["op"] == "mass":   # what attention left for these rows
            s["lse"] = _softmax_parts(s)[1]
    return s


def _tokens(s):
    """(sequence, index in its chunk) of every row."""
    row = torch.arange(s["rows"], device=DEVICE)
    if s["cu"] is None:
        return row, torch.zeros_like(row)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    return seq, row - s["cu"].long()[seq]


def _dense(cache, table):
    """The slots of every sequence side by side: fp32 ``[b, kv_heads, slots, dim]``."""
    x = cache[table.long().clamp(min=0)]
    b, p, kh, ps, d = x.shape
    return x.float().permute(0, 2, 1, 3, 4).reshape(b, kh, p * ps, d)


def _scores(s):
    """Masked scores fp32 ``[b, kv_heads, group, rows, slots]`` of the padded chunks, and which of them count."""
    c, n = s["case"], s["most"]
    kh, d = c["kv_heads"], c["dim"]
    g = c["heads"] // kh
    k = _dense(s["k"], s["table"])
    b, _, slots, _ = k.shape
    count = s["cu"].diff().long() if s["cu"] is not None else torch.ones(b, dtype=torch.int64, device=DEVICE)
    start = s["cu"][:-1].long() if s["cu"] is not None else torch.arange(b, device=DEVICE)
    i = torch.arange(n, device=DEVICE)
    q = s["q"][(start[:, None] + i).clamp(max=s["rows"] - 1)].float()
    q = q.reshape(b, n, kh, g, d).permute(0, 2, 3, 1, 4).reshape(b, kh, g * n, d)
    x = torch.matmul(q, k.transpose(2, 3)).reshape(b, kh, g, n, slots) * s["scale"]
    if c.get("softcap"):
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    lens = s["lens"].long()
    place = (lens - count)[:, None, None] + i[:, None]
    j = torch.arange(slots, device=DEVICE)
    away = place - j
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(kh, g, 1, 1) * away.abs().float()[:, None, None]
    seen = away >= 0
    if c.get("window"):
        seen = seen & (away < c["window"])
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"].long()[:, None, None])
    seen = seen & (j < lens[:, None, None]) & (i[:, None] < count[:, None, None])
    return x.masked_fill(~seen[:, None, None], -math.inf)


def _softmax_parts(s, values=None):
    """(output rows or None, log sums ``[rows, heads]``) of softmax attention."""
    c, (seq, at) = s["case"], _tokens(s)
    x = _scores(s)
    top = x.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)[seq, :, :, at].reshape(-1, c["heads"])
    if values is None:
        return None, lse
    b, kh, g, n, slots = p.shape
    o = torch.matmul(p.reshape(b, kh, g * n, slots), values).reshape(b, kh, g, n, -1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o[seq, :, :, at].reshape(len(seq), c["heads"], c["dim"]).to(s["q"].dtype), lse


def _plain_rope(s):
    c, (seq, at) = s["case"], _tokens(s)
    h, kh, d = c["heads"], c["kv_heads"], c["dim"]
    half = d // 2
    pos = s["pos"].reshape(c["axes"], -1)[s["axis"]].t()
    f = torch.arange(half, device=DEVICE)
    cos, sin = s["cos"][pos, f].unsqueeze(1), s["sin"][pos, f].unsqueeze(1)
    x = s["qkv"].reshape(-1, h + 2 * kh, d)
    lo, hi = x[:, :h + kh, :half].float(), x[:, :h + kh, half:].float()
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], 2).to(x.dtype)
    count = s["cu"].diff().long() if s["cu"] is not None else torch.ones_like(s["lens"]).long()
    slot = s["lens"].long()[seq] - count[seq] + at
    page = s["table"].long()[seq, slot // c["page"]]
    s["k"][page, :, slot % c["page"]] = turned[:, h:]
    s["v"][page, :, slot % c["page"]] = x[:, h + kh:]
    return turned[:, :h].contiguous(), s["k"], s["v"]


def _plain_mass(s):
    c, (seq, at) = s["case"], _tokens(s)
    x = _scores(s)
    b, kh, g, n, slots = x.shape
    lse = torch.zeros(b, n, kh, g, device=DEVICE)
    lse[seq, at] = s["lse"].reshape(-1, kh, g)
    return torch.exp(x - lse.permute(0, 2, 3, 1).unsqueeze(-1)).sum((2, 3))


def _plain_evict(s):
    c = s["case"]
    ps, d, budget = c["page"], c["dim"], s["budget"]
    mass, lens = s["mass"], s["lens"].long()
    b, kh, slots = mass.shape
    j = torch.arange(slots, device=DEVICE)
    free, live = j < (lens - s["recent"])[:, None, None], j < lens[:, None, None]
    rank = torch.where(free, mass, torch.where(live, math.inf, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :budget]
    order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]))
    kept_n = lens.clamp(max=budget)
    r = torch.arange(budget, device=DEVICE)
    live = (r < kept_n[:, None, None]).expand(b, kh, budget)
    kept = torch.sort(torch.where(live, order, slots), -1)[0]
    src = torch.where(live, kept, 0)
    row = torch.arange(b, device=DEVICE)[:, None, None]
    head = torch.arange(kh, device=DEVICE)[None, :, None]
    to = s["to"].long()[row, r // ps]
    old = s["table"].long()[row, src // ps].clamp(min=0)
    for cache in (s["k"], s["v"]):
        cache[to, head, r % ps] = torch.where(live[..., None], cache[old, head, src % ps], cache[to, head, r % ps])
    left = torch.zeros(b, kh, s["to"].shape[1] * ps, device=DEVICE)
    left[..., :budget] = torch.where(live, mass.gather(-1, src), 0.0)
    return torch.where(live, kept, -1).int(), kept_n.int(), left, s["k"], s["v"]


def _own(s):
    if os.path.join(_ROOT, "metal-native_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "metal-native_amd"))
    from metal_native import paged

    c, op = s["case"], s["case"]["op"]
    if op == "rope":
        q = paged.rope_kv(s["qkv"], s["cos"], s["sin"], s["pos"], s["k"], s["v"], s["table"], s["lens"], s["cu"],
                          sections=s["sections"])
        return q, s["k"], s["v"]
    if op == "evict":
        kept, lens, left = paged.evict(s["k"], s["v"], s["table"], s["lens"], s["mass"], s["to"], s["budget"],
                                       recent=s["recent"])
        return kept, lens, left, s["k"], s["v"]
    how = {"scale": s["scale"], "softcap": c.get("softcap", 0.0), "slopes": s["slopes"], "window": c.get("window", 0),
           "prefix_lens": s["prefix"], "max_q": s["most"]}
    if op == "mass":
        return paged.attention_mass(s["q"], s["k"], s["table"], s["lens"], s["lse"], s["cu"], **how)
    return paged.attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], return_lse=bool(c.get("lse")), **how)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rope":
        return _plain_rope(state)
    if op == "mass":
        return _plain_mass(state)
    if op == "evict":
        return _plain_evict(state)
    out, lse = _softmax_parts(state, _dense(state["v"], state["table"]))
    return (out, lse) if state["case"].get("lse") else out


def _visible(case):
    """(key slots that some row of a sequence sees, pairs of a row and a slot that it sees), over all sequences."""
    total, new = _lengths(case)
    window, prefix = case.get("window", 0), case.get("prefix", 0)
    slots = pairs = 0
    for t, n in zip(total, new):
        first = 0 if not window else max(0, t - n - window + 1)
        slots += t - first + min(prefix, first)
        if not window and not prefix:
            pairs += n * (t - n) + n * (n + 1) // 2
        else:
            for p in range(t - n, t):
                lo = 0 if not window else max(0, p - window + 1)
                pairs += p + 1 - lo + min(prefix, lo) + max(0, min(prefix, t) - p - 1)
    return slots, pairs


def work(case):
    total, new = _lengths(case)
    h, kh, d, t = case["heads"], case["kv_heads"], case["dim"], sum(new)
    if case["op"] == "rope":
        # rows in, q out, k and v into their pages; the angles of each row
        return {"bytes": 2 * t * (h + 2 * kh) * d * 2 + t * (d // 2) * 8 + 8 * t * case["axes"], "flops": 6 * t * (h + kh) * (d // 2)}
    if case["op"] == "evict":
        kept = sum(min(a, case["budget"]) for a in total) * kh
        return {"bytes": 4 * kh * sum(total) + kept * (2 * 2 * 2 * d + 8), "flops": 0}
    slots, pairs = _visible(case)
    if case["op"] == "mass":
        return {"bytes": 2 * t * h * d + 4 * t * h + 2 * slots * kh * d + 4 * sum(total) * kh, "flops": 2 * pairs * h * d}
    return {"bytes": 4 * t * h * d + 4 * slots * kh * d + (4 * t * h if case.get("lse") else 0), "flops": 4 * pairs * h * d}


def _rows64(s, b, kv, total, n, start):
    """Keys, values and masked scores of one sequence and key/value head in 64 bits."""
    c = s["case"]
    g, ps = c["heads"] // c["kv_heads"], c["page"]
    ids = s["table"][b, :-(-total // ps)].long()
    k = s["k"][ids, kv].reshape(-1, c["dim"])[:total].double()
    v = s["v"][ids, kv].reshape(-1, c["dim"])[:total].double()
    x = torch.einsum("ngd,jd->gnj", s["q"][start:start + n, kv * g:(kv + 1) * g].double(), k) / math.sqrt(c["dim"])
    if c.get("softcap"):
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    p = torch.arange(total - n, total, device=DEVICE)[:, None]
    j = torch.arange(total, device=DEVICE)[None]
    if s["slopes"] is not None:
        x = x - s["slopes"][kv * g:(kv + 1) * g].double()[:, None, None] * (p - j).abs().double()
    hidden = j > p
    if c.get("window"):
        hidden = hidden | (j <= p - c["window"])
    if c.get("prefix"):
        hidden = hidden & (j >= c["prefix"])
    x.masked_fill_(hidden, -math.inf)
    return x, v


def exact(case, seed):
    s = prepare(case, seed)
    total, new = _lengths(case)
    h, kh, d, ps, b = case["heads"], case["kv_heads"], case["dim"], case["page"], case["b"]
    g, t = h // kh, sum(new)
    start = [sum(new[:i]) for i in range(b)]
    if case["op"] == "rope":
        half = d // 2
        x = s["qkv"].double().reshape(t, h + 2 * kh, d)
        pos = s["pos"].reshape(case["axes"], t)
        z = torch.empty(t, half, dtype=torch.complex128, device=DEVICE)
        f = 0
        for a, width in enumerate(s["sections"]):
            z[:, f:f + width] = torch.complex(s["cos"][pos[a], f:f + width].double(), s["sin"][pos[a], f:f + width].double())
            f += width
        turned = torch.complex(x[:, :h + kh, :half].contiguous(), x[:, :h + kh, half:].contiguous()) * z[:, None]
        turned = torch.cat([turned.real, turned.imag], -1)
        k, v = s["k"].double(), s["v"].double()
        for i in range(b):
            slot = torch.arange(total[i] - new[i], total[i], device=DEVICE)
            page, rows = s["table"][i].long()[slot // ps], slice(start[i], start[i] + new[i])
            k[page, :, slot % ps] = turned[rows, h:]
            v[page, :, slot % ps] = x[rows, h + kh:]
        return turned[:, :h], k, v
    if case["op"] == "evict":
        mass = s["mass"].double().cpu().numpy()
        k, v = s["k"].double(), s["v"].double()
        kept = torch.full((b, kh, case["budget"]), -1, dtype=torch.int32)
        left = torch.zeros(b, kh, s["to"].shape[1] * ps, dtype=torch.float64)
        for i in range(b):
            for a in range(kh):
                row, n = mass[i, a], total[i]
                old = max(0, n - case["recent"])
                if n <= case["budget"]:
                    keep = list(range(n))
                else:
                    best = sorted(range(old), key=lambda j: (-row[j], j))[:case["budget"] - (n - old)]
                    keep = sorted(best) + list(range(old, n))
                src, dst = torch.tensor(keep), torch.arange(len(keep))
                kept[i, a, :len(keep)] = src.int()
                left[i, a, :len(keep)] = torch.from_numpy(row)[src]
                src, dst = src.to(DEVICE), dst.to(DEVICE)
                for cache in (k, v):
                    cache[s["to"][i].long()[dst // ps], a, dst % ps] = cache[s["table"][i].long()[src // ps], a, src % ps]
        return kept, torch.tensor([min(n, case["budget"]) for n in total], dtype=torch.int32), left, k, v
    out = torch.zeros(t, h, d, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(t, h, dtype=torch.float64, device=DEVICE)
    mass = torch.zeros(b, kh, s["table"].shape[1] * ps, dtype=torch.float64, device=DEVICE)
    for i in range(b):
        for a in range(kh):
            x, v = _rows64(s, i, a, total[i], new[i], start[i])
            rows, hs = slice(start[i], start[i] + new[i]), slice(a * g, (a + 1) * g)
            if case["op"] == "mass":
                given = s["lse"][rows, hs].double()
                mass[i, a, :total[i]] = torch.exp(x - given.t()[..., None]).sum((0, 1))
                continue
            log = torch.logsumexp(x, -1)
            lse[rows, hs] = log.t()
            out[rows, hs] = torch.einsum("gnj,jd->ngd", torch.exp(x - log[..., None]), v)
    if case["op"] == "mass":
        return mass
    return (out, lse) if case.get("lse") else out
