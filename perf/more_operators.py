"""Performance cases of the operators that answer with drafted tokens and random numbers.

A server that drafts runs a small tree of guessed tokens through the model in one step, draws a token
behind every node of it, and keeps the path whose guesses were drawn.  Kinds of case (``case["op"]``):

* ``ancestors`` -- which nodes of its tree every drafted token descends from, as bits
  (``metal_native.paged.ancestors``);
* ``tree``      -- attention of such a tree, whose nodes are the newest slots of their sequence, over the
  sequence's pages: every older slot and the node's own ancestors are seen, with or without a tanh cap,
  a bias that falls with distance, a sliding window and a prefix (``metal_native.paged.tree_attention``);
* ``sample``    -- tokens drawn from logits by given random numbers, with temperature, top-k, top-p and
  min-p, one setting for all rows or one for each (``metal_native.sampling.sample``);
* ``accept``    -- the path through the tree whose drafted tokens are the drawn ones, its slots moved
  together in the caches of all layers (``metal_native.paged.accept``).

A sequence's chunk is its tree: node 0, the root, is the newest token that is settled, every other node
names an earlier one as its parent.  Caches are ``[pages, kv_heads, page_size, head_dim]`` with the pages
of all sequences in random order, with a dimension of layers before them for ``accept``.  Inputs are made
on the GPU from the seed alone: queries, keys and values N(0, 1), logits N(0, spread) with a few high ones
as a language model's have, random numbers uniform in [0, 1).  Lengths and the shapes of the trees follow
from the case itself, so that its work does not depend on the seed.
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
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _tree(name, dtype, heads, kv_heads, dim, page, b, lmin, lmax, nmin, nmax, mix=1, **more):
    """``b`` sequences of ``lmin..lmax`` cached tokens, the last ``nmin..nmax`` of them a tree."""
    c = {"op": "tree", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "b": b,
         "lmin": lmin, "lmax": lmax, "nmin": nmin, "nmax": nmax, "mix": mix, **more}
    return {"name": name, **c} if name else c


def _ancestors(name, b, nmin, nmax, mix=1):
    c = {"op": "ancestors", "b": b, "nmin": nmin, "nmax": nmax, "mix": mix}
    return {"name": name, **c} if name else c


def _sample(name, dtype, rows, vocab, spread, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, each=False, logprob=False):
    """``each``: settings drawn for every row in place of the given ones."""
    c = {"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "spread": spread, "temperature": temperature,
         "top_k": top_k, "top_p": top_p, "min_p": min_p, "each": each, "logprob": logprob}
    return {"name": name, **c} if name else c


def _accept(name, dtype, layers, kv_heads, dim, page, b, lmin, lmax, nmin, nmax, words, mix=1):
    """``words``: how many different tokens are drafted and drawn; few make long paths."""
    c = {"op": "accept", "dtype": dtype, "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page, "b": b,
         "lmin": lmin, "lmax": lmax, "nmin": nmin, "nmax": nmax, "words": words, "mix": mix}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the tree of one conversation: latency
        _ancestors("ancestors_b1", 1, 16, 16),
        # wide trees of a full serving batch
        _ancestors("ancestors_b64", 64, 100, 512, mix=3),
        # one conversation behind the framework's decoder cache of 512 tokens, 16 nodes: latency
        _tree("tree_b1", "fp16", 28, 4, 128, 16, 1, 528, 528, 16, 16),
        # a serving batch of 24 conversations, trees of 4 to 26 nodes, with the rows' log sums kept
        _tree("tree_ragged_b24", "bf16", 32, 8, 128, 16, 24, 200, 8000, 4, 26, mix=2, lse=True),
        # four long documents, 64 nodes each: reading the cache is most of the work
        _tree("tree_long", "fp16", 28, 4, 128, 64, 4, 90001, 131072, 64, 64),
        # wide trees of a small model with capped scores, distance bias, window and a shared prefix
        _tree("tree_masked_wide", "fp16", 14, 2, 64, 32, 5, 700, 3500, 60, 257, mix=2, softcap=30.0, bias=True, window=1000,
              prefix=77),
        # the next token of one conversation, the usual settings of a chat: latency
        _sample("sample_b1", "fp16", 1, 152064, 2.0, temperature=0.7, top_k=50, top_p=0.9),
        # every node of 16 trees of 26: nucleus alone
        _sample("sample_nodes", "fp16", 416, 152064, 2.0, temperature=0.8, top_p=0.95),
        # a batch in which every request has its own settings, log probabilities kept
        _sample("sample_each_b64", "bf16", 64, 152064, 2.0, each=True, logprob=True),
        # a small vocabulary (odd) in fp32, flat, cut by min-p
        _sample("sample_fp32", "fp32", 48, 32003, 1.0, temperature=1.3, min_p=0.05),
        # one conversation's 16 nodes in the 28 layers of a 7B decoder: latency
        _accept("accept_b1", "fp16", 28, 4, 128, 16, 1, 528, 528, 16, 16, 2),
        # 48 conversations with trees of up to 64 nodes
        _accept("accept_b48", "bf16", 28, 4, 128, 16, 48, 300, 2000, 20, 64, 2, mix=5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ancestors", "tree", "tree", "tree", "sample", "sample", "sample", "accept"))
    mix = rng.randrange(1 << 20)
    if op == "ancestors":
        n = _log(rng, 1, 512)
        return _ancestors(None, _log(rng, 1, 64), max(1, n // rng.choice((1, 2, 5))), n, mix)
    if op == "sample":
        vocab = _log(rng, 100, 152064)
        rows = _log(rng, 1, max(1, min(416, 60_000_000 // vocab)))
        return _sample(None, rng.choice(("fp16", "bf16", "fp32")), rows, vocab, rng.choice((0.5, 1.0, 2.0, 4.0)),
                       temperature=rng.choice((0.0, 0.4, 0.8, 1.0, 1.7)), top_k=rng.choice((0, 0, 1, _log(rng, 2, vocab))),
                       top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.99)), min_p=rng.choice((0.0, 0.0, 0.01, 0.1)),
                       each=rng.random() < 0.4, logprob=rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice(((28, 4, 128), (32, 8, 128), (14, 2, 64), (16, 16, 128), (24, 8, 64), (8, 1, 128)))
    dtype, page = rng.choice(("fp16", "bf16")), rng.choice((16, 32, 64, 128))
    if op == "accept":
        n = _log(rng, 1, 128)
        layers = rng.choice((1, 4, 28))
        return _accept(None, dtype, layers, kv_heads, dim, page, _log(rng, 1, 48 if layers < 28 else 16), n + rng.randrange(50),
                       n + _log(rng, 50, 1500), max(1, n // 3), n, rng.choice((1, 2, 4, 50)), mix)
    more = {}
    if rng.random() < 0.5:
        more["lse"] = True
    if rng.random() < 0.4:
        more.update(softcap=rng.choice((0.0, 20.0, 50.0)), bias=rng.random() < 0.5,
                    window=rng.choice((0, rng.randint(1, 3000))), prefix=rng.choice((0, rng.randint(1, 400))))
    n = _log(rng, 1, 300)
    top = n + _log(rng, 1, 65536)
    b = rng.randint(1, max(1, min(32, 900_000_000 // (top * kv_heads * dim * 4), 8_000_000 // (top * n))))
    return _tree(None, dtype, heads, kv_heads, dim, page, b, max(n, top // rng.choice((1, 3, 20))), top, max(1, n // 4), n, mix, **more)


def _spread(rng, n, lo, hi):
    """``n`` lengths over the logarithm of ``lo..hi``, both ends among them."""
    got = [_log(rng, lo, hi) for _ in range(n)]
    got[rng.randrange(n)] = lo
    got[rng.randrange(n)] = hi
    return got


def _shapes(case, seed=0):
    """(cached tokens, nodes) of each sequence, from the case alone, and each tree's parents; those of ``tree``
    too, as the pairs of a node and what it sees follow from them."""
    rng = random.Random(case["mix"])
    total = _spread(rng, case["b"], case["lmin"], case["lmax"]) if "lmin" in case else None
    nodes = _spread(rng, case["b"], case["nmin"], case["nmax"])
    if total:
        nodes = [min(n, t) for n, t in zip(nodes, total)]
    if case["op"] != "tree":
        rng.seed(1_000_003 * case["mix"] + seed)
    parents = []
    for n in nodes:   # mostly one of the newest nodes, sometimes any: paths of several nodes, and bushes
        parents.append([-1] + [rng.randrange(i) if rng.random() < 0.2 else max(0, i - 1 - int(rng.expovariate(0.5)))
                               for i in range(1, n)])
    return total, nodes, parents


def _bits(nodes, parents, words):
    """Ancestor bits (its own among them) of every node, as Python integers cut into 64-bit words."""
    rows = []
    for tree in parents:
        of = []
        for i, p in enumerate(tree):
            of.append((of[p] if p >= 0 else 0) | 1 << i)
        rows += of
    out = []
    for x in rows:
        part = [(x >> 64 * w) & (2**64 - 1) for w in range(words)]
        out.append([p - 2**64 if p >= 2**63 else p for p in part])
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = _TYPES[case["dtype"]] if "dtype" in case else None
    s = {"case": dict(case)}
    if case["op"] == "sample":
        rows, v = case["rows"], case["vocab"]
        x = torch.randn(rows, v, device=DEVICE, generator=gen) * case["spread"]
        high = torch.randint(0, v, (rows, 12), device=DEVICE, generator=gen)
        x.scatter_add_(1, high, 5.0 * case["spread"] * torch.rand(rows, 12, device=DEVICE, generator=gen))
        s["logits"] = x.to(dt)
        s["u"] = torch.rand(rows, device=DEVICE, generator=gen)
        for key, kind, some in (("temperature", torch.float32, (0.0, 0.5, 0.8, 1.0, 1.5)), ("top_k", torch.int32, (0, 0, 1, 20, 50, 1000)),
                                ("top_p", torch.float32, (1.0, 1.0, 0.5, 0.9, 0.95)), ("min_p", torch.float32, (0.0, 0.0, 0.05, 0.2))):
            if case["each"]:
                pick = torch.randint(0, len(some), (rows,), device=DEVICE, generator=gen)
                s[key] = torch.tensor(some, dtype=kind, device=DEVICE)[pick]
            else:
                s[key] = case[key]
        return s
    total, nodes, parents = _shapes(case, seed)
    b, t, most = case["b"], sum(nodes), max(nodes)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    s.update(rows=t, most=most, cu=torch.tensor(cu, dtype=torch.int32, device=DEVICE))
    s["parents"] = torch.tensor([p for x in parents for p in x], dtype=torch.int32, device=DEVICE)
    if case["op"] == "ancestors":
        return s
    kh, d, ps = case["kv_heads"], case["dim"], case["page"]
    pages = [-(-x // ps) for x in total]
    pool = sum(pages) + 3
    order = torch.randperm(pool, device=DEVICE, generator=gen).to(torch.int32)
    table = torch.full((b, max(pages)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    rn = lambda *z: torch.randn(*z, device=DEVICE, generator=gen, dtype=torch.float32).to(dt)  # noqa: E731
    s.update(table=table, lens=torch.tensor(total, dtype=torch.int32, device=DEVICE))
    if case["op"] == "accept":
        layers = case["layers"]
        kv = torch.empty(layers, 2, pool, kh, ps, d, dtype=dt, device=DEVICE)
        for i in range(layers):
            kv[i] = rn(2, pool, kh, ps, d)
        s.update(k=kv[:, 0], v=kv[:, 1])
        for key in ("drawn", "drafted"):
            s[key] = torch.randint(0, case["words"], (t,), device=DEVICE, generator=gen)
        s["steps"] = min(most, 32)
        return s
    h = case["heads"]
    s.update(k=rn(pool, kh, ps, d), v=rn(pool, kh, ps, d), q=rn(t, h, d), scale=1.0 / math.sqrt(d))
    s["bits"] = torch.tensor(_bits(nodes, parents, -(-most // 64)), dtype=torch.int64, device=DEVICE)
    s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, h + 1, device=DEVICE, dtype=torch.float32) / h) if case.get("bias") else None)
    s["prefix"] = torch.full((b,), case["prefix"], dtype=torch.int32, device=DEVICE) if case.get("prefix") else None
    return s


def _tokens(s):
    """(sequence, index in its chunk) of every row."""
    row = torch.arange(s["rows"], device=DEVICE)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    return seq, row - s["cu"].long()[seq]


def _closure(s):
    """Whether node j is node i or one of its ancestors: ``[b, most, most]``, by squaring the parent relation."""
    seq, at = _tokens(s)
    n, b = s["most"], s["cu"].numel() - 1
    reach = torch.zeros(b, n, n, device=DEVICE)
    up = s["parents"].long()
    reach[seq, at, up.clamp(min=0)] = (up >= 0).float()
    reach[seq, at, at] = 1.0
    far = 1
    while far < n:
        reach = (torch.matmul(reach, reach) > 0).float()
        far *= 2
    return reach > 0


def _plain_ancestors(s):
    seq, at = _tokens(s)
    rows = _closure(s)[seq, at].long()
    words = -(-s["most"] // 64)
    rows = torch.nn.functional.pad(rows, (0, 64 * words - s["most"])).reshape(-1, words, 64)
    return (rows << torch.arange(64, device=DEVICE)).sum(-1)


def _dense(cache, table):
    """The slots of every sequence side by side: fp32 ``[b, kv_heads, slots, dim]``."""
    x = cache[table.long().clamp(min=0)]
    b, p, kh, ps, d = x.shape
    return x.float().permute(0, 2, 1, 3, 4).reshape(b, kh, p * ps, d)


def _plain_tree(s):
    c, n, (seq, at) = s["case"], s["most"], _tokens(s)
    kh, d = c["kv_heads"], c["dim"]
    g = c["heads"] // kh
    k, v = _dense(s["k"], s["table"]), _dense(s["v"], s["table"])
    b, _, slots, _ = k.shape
    count, start, lens = s["cu"].diff().long(), s["cu"][:-1].long(), s["lens"].long()
    i = torch.arange(n, device=DEVICE)
    rows = (start[:, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"][rows].float().reshape(b, n, kh, g, d).permute(0, 2, 3, 1, 4).reshape(b, kh, g * n, d)
    x = torch.matmul(q, k.transpose(2, 3)).reshape(b, kh, g, n, slots) * s["scale"]
    if c.get("softcap"):
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    # the bits of every row as truth values by node, and how many of them are set up to each
    mine = ((s["bits"][rows].unsqueeze(-1) >> torch.arange(64, device=DEVICE)) & 1).reshape(b, n, -1)
    upto = mine.cumsum(-1)
    depth = upto[..., -1:] - 1
    j = torch.arange(slots, device=DEVICE)
    node = (j - (lens - count)[:, None])[:, None].expand(b, n, slots)   # negative: an older slot
    which = node.clamp(0, mine.shape[-1] - 1)
    away = torch.where(node < 0, depth - node, depth + 1 - upto.gather(-1, which))
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(kh, g, 1, 1) * away.abs().float()[:, None, None]
    seen = (node < 0) | (mine.gather(-1, which) == 1)
    if c.get("window"):
        seen = seen & (away < c["window"])
    if s["prefix"] is not None:
        seen = seen | ((node < 0) & (j < s["prefix"].long()[:, None, None]))
    seen = seen & (j < lens[:, None, None]) & (i[:, None] < count[:, None, None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = torch.exp(x - top)
    sums = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, kh, g * n, slots), v).reshape(b, kh, g, n, d)
    o = torch.where(sums > 0, o / sums, torch.zeros_like(o))[seq, :, :, at].reshape(-1, c["heads"], d).to(s["q"].dtype)
    if not c.get("lse"):
        return o
    return o, (top + torch.log(sums)).squeeze(-1)[seq, :, :, at].reshape(-1, c["heads"])


def _setting(s, key, dtype):
    """One value for each row, at the precision that the setting has (32 bits)."""
    x = s[key]
    x = x if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.int32 if key == "top_k" else torch.float32, device=DEVICE)
    return x.to(dtype).expand(s["case"]["rows"]).unsqueeze(1)


def _plain_sample(s):
    """Weights, their sums and the comparisons with a border in 64 bits: a token is drawn, not approximated."""
    logits = s["logits"].float()
    rows, v = logits.shape
    x, order = torch.sort(logits, dim=1, descending=True, stable=True)
    rank = torch.arange(v, device=DEVICE)
    temperature, k = _setting(s, "temperature", torch.float64), _setting(s, "top_k", torch.int64)
    top_p, min_p = _setting(s, "top_p", torch.float64), _setting(s, "min_p", torch.float64)
    greedy = temperature <= 0
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, temperature))
    w = torch.where((k > 0) & (rank >= k), 0.0, w)
    w = torch.where(greedy & (rank > 0), 0.0, w)
    before = w.cumsum(1) - w
    keep = (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0)
    w = torch.where(keep & (w >= min_p), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.cumsum(1)
    aim = s["u"].double().unsqueeze(1) * total[:, -1:]
    token = (total <= aim).sum(1)
    if not s["case"]["logprob"]:
        return token
    return token, torch.log(w.gather(1, token.unsqueeze(1)) / total[:, -1:]).squeeze(1).float()


def _plain_accept(s):
    n, (seq, at), ps = s["most"], _tokens(s), s["case"]["page"]
    b, steps = s["lens"].numel(), s["steps"]
    up = s["parents"].long()
    hit = (up < 0) | (s["drafted"] == s["drawn"][s["cu"].long()[seq] + up.clamp(min=0)])
    wide = lambda x, fill: torch.full((b, n), fill, dtype=x.dtype, device=DEVICE).index_put_((seq, at), x)  # noqa: E731
    ups, hits = wide(up, -2), wide(hit, False)
    i = torch.arange(n, device=DEVICE)
    earlier = (ups[:, :, None] == ups[:, None, :]) & hits[:, None, :] & (i[None, :] < i[:, None])   # a sibling drawn before
    good = hits & ~earlier.any(-1)
    reach = _closure(s)
    on = good & ~(reach & ~good[:, None, :]).any(-1)
    path = torch.sort(torch.where(on, i, n), 1)[0][:, :steps]
    live = path < n
    path = torch.where(live, path, 0)
    count = live.sum(1)
    tokens = torch.where(live, s["drawn"][s["cu"][:-1].long()[:, None] + path], -1)
    old = s["lens"].long() - s["cu"].diff().long()
    row = torch.arange(b, device=DEVICE)[:, None]
    src, dst = old[:, None] + path, old[:, None] + torch.arange(path.shape[1], device=DEVICE)
    dst = torch.where(live, dst, src)   # past the path: left where it is
    page = lambda x: s["table"].long()[row, x // ps]  # noqa: E731
    for cache in (s["k"], s["v"]):
        cache[:, page(dst)[live], :, (dst % ps)[live]] = cache[:, page(src)[live], :, (src % ps)[live]]
    return torch.where(live, path, -1).int(), tokens, count.int(), (old + count).int(), s["k"], s["v"]


def _own(s):
    if os.path.join(_ROOT, "metal-native_amd") not in sys.path:
        sys.path.insert(0, os.path.join(_ROOT, "metal-native_amd"))
    from metal_native import paged, sampling

    c, op = s["case"], s["case"]["op"]
    if op == "ancestors":
        return paged.ancestors(s["parents"], s["cu"], s["most"])
    if op == "tree":
        return paged.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["bits"], s["cu"], scale=s["scale"],
                                    softcap=c.get("softcap", 0.0), slopes=s["slopes"], window=c.get("window", 0),
                                    prefix_lens=s["prefix"], max_q=s["most"], return_lse=bool(c.get("lse")))
    if op == "sample":
        return sampling.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"], return_logprob=c["logprob"])
    path, tokens, count, lens = paged.accept(s["k"], s["v"], s["table"], s["lens"], s["drawn"], s["drafted"], s["parents"],
                                             s["cu"], steps=s["steps"])
    return path, tokens, count, lens, s["k"], s["v"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "ancestors":
        return _plain_ancestors(state)
    if op == "tree":
        return _plain_tree(state)
    if op == "sample":
        return _plain_sample(state)
    return _plain_accept(state)


def _depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def work(case):
    if case["op"] == "sample":
        rows, v = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": rows * (v * size + 4 + 8 + (4 if case["logprob"] else 0) + (16 if case["each"] else 0)), "flops": 3 * rows * v}
    total, nodes, parents = _shapes(case)
    t, words = sum(nodes), -(-max(nodes) // 64)
    if case["op"] == "ancestors":
        return {"bytes": 4 * t + 4 * (case["b"] + 1) + 8 * words * t, "flops": words * t}
    kh, d = case["kv_heads"], case["dim"]
    if case["op"] == "accept":
        # a path of about log(nodes) tokens, more where few different ones are drafted; each slot read and written
        moved = sum(min(n, 1 + math.log2(n)) for n in nodes) * (1.0 if case["words"] <= 2 else 0.3)
        return {"bytes": 20 * t + moved * case["layers"] * kh * d * 8, "flops": 0}
    h = case["heads"]
    window, prefix = case.get("window", 0), case.get("prefix", 0)
    slots = pairs = 0
    for length, n, p in zip(total, nodes, parents):
        old, depths = length - n, _depths(p)
        first = max(0, old - window) if window else 0
        slots += old - first + min(prefix, first) + n
        for x in depths:
            lo = max(0, old + x - window + 1) if window else 0
            pairs += max(0, old - lo) + min(prefix, lo, old) + min(x + 1, window or x + 1)
    return {"bytes": 4 * t * h * d + 4 * slots * kh * d + 8 * words * t + (4 * t * h if case.get("lse") else 0), "flops": 4 * pairs * h * d}


def _exact_sample(s):
    import numpy as np

    rows, v = s["logits"].shape
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    value = {}
    for key in ("temperature", "top_k", "top_p", "min_p"):
        x = s[key]
        value[key] = x.double().cpu().numpy() if isinstance(x, torch.Tensor) else np.full(rows, float(np.float32(x)))
    tokens, logs = np.zeros(rows, np.int64), np.zeros(rows)
    for r in range(rows):
        z, heat = logits[r], value["temperature"][r]
        if heat <= 0:
            tokens[r] = int(np.argmax(z))
            continue
        order = np.argsort(-z, kind="stable")
        if value["top_k"][r] > 0:
            order = order[:int(value["top_k"][r])]
        w = np.exp((z[order] - z[order[0]]) / heat)
        if value["top_p"][r] < 1:
            run_up = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int(np.searchsorted(run_up, value["top_p"][r] * w.sum(), side="left")))
            order, w = order[:n], w[:n]
        few = w >= value["min_p"][r]
        order, w = order[few], w[few]
        by = np.argsort(order)
        order, w = order[by], w[by]
        run_up = np.cumsum(w)
        i = int(np.searchsorted(run_up, u[r] * run_up[-1], side="right"))
        tokens[r], logs[r] = order[i], math.log(w[i] / run_up[-1])
    token = torch.from_numpy(tokens)
    return (token, torch.from_numpy(logs)) if s["case"]["logprob"] else token


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    total, nodes, parents = _shapes(case)
    if case["op"] in ("ancestors", "accept"):   # whole numbers and copies
        return None
    h, kh, d, ps, b = case["heads"], case["kv_heads"], case["dim"], case["page"], case["b"]
    g, t = h // kh, sum(nodes)
    out = torch.zeros(t, h, d, dtype=torch.float64, device=DEVICE)
    lse = torch.zeros(t, h, dtype=torch.float64, device=DEVICE)
    start = 0
    for i in range(b):
        n, old = nodes[i], total[i] - nodes[i]
        depths = torch.tensor(_depths(parents[i]), device=DEVICE)
        family = torch.zeros(n, n, dtype=torch.bool)
        for x, p in enumerate(parents[i]):
            if p >= 0:
                family[x] = family[p]
            family[x, x] = True
        family = family.to(DEVICE)
        away = torch.cat([old + depths[:, None] - torch.arange(old, device=DEVICE)[None], depths[:, None] - depths[None]], 1)
        hidden = torch.cat([torch.zeros(n, old, dtype=torch.bool, device=DEVICE), ~family], 1)
        if case.get("window"):
            hidden = hidden | (away >= case["window"])
        if case.get("prefix"):
            hidden[:, :min(old, case["prefix"])] = False
        ids = s["table"][i, :-(-total[i] // ps)].long()
        for a in range(kh):
            hs = slice(a * g, (a + 1) * g)
            k = s["k"][ids, a].reshape(-1, d)[:total[i]].double()
            v = s["v"][ids, a].reshape(-1, d)[:total[i]].double()
            q = s["q"][start:start + n, hs].double().transpose(0, 1).reshape(g * n, d)
            x = torch.mm(q, k.t()).reshape(g, n, -1) / math.sqrt(d)
            if case.get("softcap"):
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            if s["slopes"] is not None:
                x = x - s["slopes"][hs].double()[:, None, None] * away.double()
            x.masked_fill_(hidden, -math.inf)
            log = torch.logsumexp(x, -1)
            lse[start:start + n, hs] = log.t()
            w = torch.exp(x - log[..., None]).reshape(g * n, -1)
            out[start:start + n, hs] = torch.mm(w, v).reshape(g, n, d).transpose(0, 1)
        start += n
    return (out, lse) if case.get("lse") else out
