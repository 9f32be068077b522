"""Operators for trees of drafted tokens against their definitions: ancestor bits, tree attention (bounds in
paged_ref), accepted paths."""

import math
import random

import numpy as np
import pytest
import torch

import draft_ref as ref
from paged_ref import half_step
from test_paged import DT, HEADS, build

pytestmark = pytest.mark.gpu


def random_tree(rng, n, kind="mixed"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    return ([-1] + [rng.randrange(i) if rng.random() < 0.3 else max(0, i - 1 - int(rng.expovariate(0.7))) for i in range(1, n)])[:n]


def trees(gpu, counts, seed=0, kind="mixed"):
    rng = random.Random(seed)
    parents = [random_tree(rng, n, kind) for n in counts]
    cu = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=gpu)
    flat = torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=gpu)
    return parents, flat, cu


# ---- ancestors ----
@pytest.mark.parametrize("kind", ["mixed", "chain", "star"])
@pytest.mark.parametrize("counts", [[1], [64], [65, 1, 0, 63], [16, 130, 3, 300], [0, 0, 5], [1000, 2, 2500]])
def test_ancestors(gpu, kind, counts):
    from metal_native import paged

    parents, flat, cu = trees(gpu, counts, len(counts), kind)
    most = max(counts)
    for max_q in {most, most + 64, max(1, most // 2), 1}:
        words = -(-max_q // 64)
        want = torch.cat([ref.pack(ref.closure(p), words) for p in parents])
        got = paged.ancestors(flat, cu, max_q)
        assert got.dtype == torch.int64 and torch.equal(got.cpu(), want)
    assert paged.ancestors(flat, cu).shape == (sum(counts), -(-sum(counts) // 64))


def test_ancestors_of_odd_parents_and_rows_of_no_sequence(gpu):
    from metal_native import paged

    flat = torch.tensor([9, 9, -1, 0, 7, 1, -(2**31), 2**31 - 1, 3, 4, 5, 5], dtype=torch.int32, device=gpu)
    cu = torch.tensor([2, 6, 6, 10], dtype=torch.int32, device=gpu)   # two rows before the first tree, two past the last
    want = torch.zeros(12, 1, dtype=torch.int64)
    for s in range(3):
        a, b = int(cu[s]), int(cu[s + 1])
        if b > a:
            want[a:b] = ref.pack(ref.closure(flat[a:b].tolist()), 1)
    assert torch.equal(paged.ancestors(flat, cu, 4).cpu(), want)
    assert torch.equal(paged.ancestors(flat).cpu()[:, 0], torch.ones(12, dtype=torch.int64))   # one token for each sequence
    for wild in ([-5, 3, 10**6, 10**6], [7, 3, 1, 12], [2**31 - 1, -(2**31), 5, 6]):   # any offsets: nothing past the rows
        assert paged.ancestors(flat, torch.tensor(wild, dtype=torch.int32, device=gpu), 64).shape == (12, 1)
    assert paged.ancestors(flat[::2], cu // 2, 4).shape == (6, 1)
    assert paged.ancestors(flat[:0], torch.zeros(2, dtype=torch.int32, device=gpu), 8).shape == (0, 1)


@pytest.mark.parametrize("n", [511, 512, 513, 577])
def test_ancestors_around_512_nodes(gpu, n):
    """Where trees no longer have a thread for each node; deep ones, wide ones, and words for fewer and more nodes."""
    from metal_native import paged

    for kind in ("mixed", "chain", "star"):
        parents, flat, cu = trees(gpu, [n, 3, n], n, kind)
        for max_q in (n, 512, 513, 64, 1000):
            want = torch.cat([ref.pack(ref.closure(p), -(-max_q // 64)) for p in parents])
            assert torch.equal(paged.ancestors(flat, cu, max_q).cpu(), want)


def test_ancestors_of_any_offsets(gpu):
    """The ends of what an offset can hold: rows of no tree have no bits, and nothing past the rows is touched."""
    from metal_native import paged

    flat = torch.arange(-1, 11, dtype=torch.int32, device=gpu)
    big = 2**31 - 1
    for cu, rows in (([0, 5, big], 12), ([3, 9, -big], 0), ([big, big, big], 0), ([-big, -5, -1], 0), ([-4, 12, big], 12), ([12, 12, 12], 0)):
        got = paged.ancestors(flat, torch.tensor(cu, dtype=torch.int32, device=gpu), 64).cpu()
        assert got.shape == (12, 1) and (int((got != 0).sum()) == rows or cu[0] == 3)


# ---- attention ----
def check_tree(c, families, bits, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None, max_q=None):
    from metal_native import paged

    s = scale or 1.0 / math.sqrt(c["q"].shape[2])
    out, lse = paged.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], bits, c["cu"], scale=s, softcap=softcap, slopes=slopes,
                                    window=window, prefix_lens=prefix, max_q=max_q, return_lse=True)
    o, l, ob, lb = ref.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], families, c["cu"], scale=s, softcap=softcap,
                                      slopes=slopes, window=window, prefix=prefix)
    got, gl = out.double().cpu(), lse.double().cpu()
    assert bool((torch.isnan(got) == torch.isnan(o)).all())
    fin = ~torch.isnan(o)
    assert bool(((got == o) | ((got - o).abs() <= ob))[fin].all()), float(((got - o).abs() / ob)[fin].nan_to_num().max())
    assert bool(((gl == l) | (torch.isnan(gl) & torch.isnan(l)) | ((gl - l).abs() <= lb)).all())
    return out, lse


def tree_case(gpu, dt, H, KVH, D, ps, lens, counts, seed=0, kind="mixed", words=None, **how):
    parents, flat, cu = trees(gpu, counts, seed, kind)
    c = build(gpu, dt, H, KVH, D, ps, lens, counts, seed=seed, **how)
    families = [ref.closure(p) for p in parents]
    words = words or max(1, -(-max(counts) // 64))
    bits = torch.cat([ref.pack(f, words) for f in families]).to(gpu)
    return c, families, bits


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("ps", [8, 64])
def test_trees(gpu, dtype, H, KVH, D, ps):
    lens, counts = [1, 40, 0, 64, 300, 129, 77, 33], [1, 3, 0, 64, 65, 0, 30, 33]
    c, families, bits = tree_case(gpu, DT[dtype], H, KVH, D, ps, lens, counts, seed=D + ps)
    check_tree(c, families, bits)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_trees_in_blocks_of_256_rows(gpu, dtype, D, masked):
    """Enough rows for the other kernel, in one part and (one long sequence) in several."""
    for lens, counts in (([700, 240, 513, 1, 200, 0], [140, 200, 90, 1, 70, 0]), ([4000], [65])):
        c, families, bits = tree_case(gpu, DT[dtype], 32, 4, D, 16, lens, counts, seed=D)
        how = {}
        if masked:
            how = dict(softcap=15.0, slopes=torch.rand(32, device=gpu, generator=c["gen"]) * 0.1, window=150,
                       prefix=torch.tensor([90, 3, 0, 0, 10**6, 1][:len(lens)], dtype=torch.int32, device=gpu))
        check_tree(c, families, bits, **how)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D,lens,counts,width", [(28, 4, 128, [20003], [5], 2048), (14, 2, 64, [9000, 300, 17, 0], [14, 60, 17, 0], 1024),
                                                       (32, 8, 128, [300, 9, 8192], [40, 9, 1], 512), (8, 1, 64, [30011, 64], [9, 64], 4096)])
def test_few_trees_behind_tables_of_many_slots(gpu, dtype, H, KVH, D, lens, counts, width):
    """Blocks of 256 rows, most of them empty, in up to 64 parts, most of those past the sequence."""
    c, families, bits = tree_case(gpu, DT[dtype], H, KVH, D, 16, lens, counts, seed=width, width=width)
    check_tree(c, families, bits)
    check_tree(c, families, bits, prefix=torch.tensor([100, 3, 10**6, 0][:len(lens)], dtype=torch.int32, device=gpu), window=9000)


@pytest.mark.parametrize("window,prefix", [(0, True), (1, False), (3, True), (7, False), (64, True), (100, False), (1000, True)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("kind", ["mixed", "chain"])
def test_tree_masks_and_scores(gpu, window, prefix, softcap, bias, kind):
    lens, counts = [200, 75, 330, 1, 128], [9, 65, 130, 1, 20]
    c, families, bits = tree_case(gpu, torch.float16, 14, 2, 64, 32, lens, counts, seed=window, kind=kind, amp=2.0)
    slopes = torch.rand(14, device=gpu, generator=c["gen"]) if bias else None
    pre = torch.tensor([0, 70, 33, 5, 500], dtype=torch.int32, device=gpu) if prefix else None
    check_tree(c, families, bits, softcap=softcap, slopes=slopes, window=window, prefix=pre)


@pytest.mark.parametrize("H,KVH,D", [(28, 4, 128), (14, 2, 64)])
def test_a_chain_is_a_chunk_in_order(gpu, H, KVH, D):
    """The same masks as attention's: the same numbers, but for where a window or a bias takes another way to them."""
    from metal_native import paged

    lens, counts = [300, 70, 5], [70, 64, 5]
    c, families, bits = tree_case(gpu, torch.float16, H, KVH, D, 16, lens, counts, kind="chain")
    out, lse = check_tree(c, families, bits)
    a, la = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True)
    u = half_step(torch.float16)
    assert float((out.float() - a.float()).abs().max()) <= 8 * u * float(c["v"][c["v"].isfinite()].abs().max())
    assert float((lse - la).abs().max()) <= 1e-4


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("window", [0, 11])
def test_any_bits(gpu, n, window):
    """Bits of no tree: later nodes, not the row's own, none at all, set past the chunk; fewer words than nodes; a row
    that sees nothing."""
    rng = np.random.default_rng(n)
    lens, counts = [n + 100, n, 7], [n, n, 7]
    c = build(gpu, torch.bfloat16, 8, 2, 64, 16, lens, counts, seed=n)
    words = -(-n // 64)
    families = [rng.random((m, 64 * words)) < 0.2 for m in counts]
    families[0][3] = families[1][5] = families[2][0] = False
    families[1][6] = True
    bits = torch.cat([ref.pack(f, words) for f in families]).to(gpu)
    slopes = torch.rand(8, device=gpu) * 0.05
    check_tree(c, families, bits, window=window, slopes=slopes)
    out, lse = check_tree(c, families, bits, window=window)
    assert float(out[n + 5].abs().max()) == 0 and bool((lse[n + 5] == -math.inf).all())
    wide = torch.nn.functional.pad(bits, (0, 3), value=-1)[:, :words + 1]   # a row stride of its own; junk past the nodes
    assert torch.equal(paged_tree(c, wide), paged_tree(c, bits))
    if words > 1:
        for f in families:
            f[:, 64:] = False
        check_tree(c, families, bits[:, :1], window=window)


def paged_tree(c, bits, **how):
    from metal_native import paged

    return paged.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], bits, c["cu"], **how)


@pytest.mark.parametrize("many", [False, True])
def test_hidden_infinities_absent_pages_and_short_caches(gpu, many):
    """What a row does not see leaves it alone, whatever it holds; what it sees is seen."""
    H, KVH, lens, counts = (32, 4, [700, 300], [140, 60]) if many else (8, 2, [90, 50], [33, 20])
    c, families, bits = tree_case(gpu, torch.float16, H, KVH, 64, 16, lens, counts, seed=2)
    for s, node in ((0, 5), (0, 31), (1, 17)):
        slot = lens[s] - counts[s] + node
        page = c["table"][s, slot // 16].long()
        c["v"][page, :, slot % 16, 3] = math.inf if node == 5 else math.nan
    check_tree(c, families, bits)
    t = c["table"]
    t[0, 1], t[1, 0], t[0, (lens[0] - 3) // 16] = -1, 10**6, -(2**31)
    check_tree(c, families, bits)
    c["lens"][:] = torch.tensor([counts[0] - 7, 3], device=gpu)   # fewer slots than nodes
    check_tree(c, families, bits, window=4, prefix=torch.tensor([2, 0], dtype=torch.int32, device=gpu))
    t[1, :] = -1
    check_tree(c, families, bits)


def test_tree_layouts_and_rows_of_no_sequence(gpu):
    from metal_native import paged

    c, families, bits = tree_case(gpu, torch.float16, 8, 2, 64, 16, [50, 90], [12, 20], seed=7)
    want = paged_tree(c, bits)
    kv = torch.stack([c["k"], c["v"]], 1)
    q2 = c["q"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged.tree_attention(q2, kv[:, 0], kv[:, 1], c["table"], c["lens"], bits, c["cu"]), want)
    odd = torch.empty(32, 8, 65, dtype=torch.float16, device=gpu)[..., 1:].copy_(c["q"])   # copied
    assert torch.equal(paged.tree_attention(odd, c["k"], c["v"], c["table"], c["lens"], bits.t().contiguous().t(), c["cu"]), want)
    pad = lambda x, v: torch.nn.functional.pad(x, (0, 0) * (x.dim() - 1) + (3, 5), value=v)  # noqa: E731
    out, lse = paged.tree_attention(pad(c["q"], math.nan), c["k"], c["v"], c["table"], c["lens"], pad(bits, -1), c["cu"] + 3, return_lse=True)
    assert torch.equal(out[3:-5], want) and float(out[:3].abs().max()) == 0 and float(out[-5:].abs().max()) == 0
    assert bool((lse[:3] == -math.inf).all()) and bool((lse[-5:] == -math.inf).all())
    one = paged.tree_attention(c["q"][:2], c["k"], c["v"], c["table"], c["lens"], bits[:2] * 0 + 1)
    assert torch.equal(one, paged.attention(c["q"][:2], c["k"], c["v"], c["table"], c["lens"]))
    assert paged.tree_attention(c["q"][:0], c["k"], c["v"], c["table"], c["lens"], bits[:0], c["cu"] * 0).shape == (0, 8, 64)


# ---- accepted paths ----
def accept_case(gpu, lens, counts, *, layers=None, KVH=2, D=64, ps=16, words=2, seed=0, kind="mixed", dtype=torch.float16):
    parents, flat, cu = trees(gpu, counts, seed, kind)
    c = build(gpu, dtype, KVH, KVH, D, ps, lens, counts, seed=seed, junk=7.0)
    g = c["gen"]
    shape = c["k"].shape if layers is None else (layers, *c["k"].shape)
    k, v = (torch.randn(shape, device=gpu, generator=g).to(dtype) for _ in range(2))
    drawn, drafted = (torch.randint(0, words, (sum(counts),), device=gpu, generator=g) for _ in range(2))
    return dict(k=k, v=v, table=c["table"], lens=c["lens"], cu=cu, drawn=drawn, drafted=drafted, parents=flat, trees=parents, ps=ps)


def check_accept(c, steps, k=None, v=None):
    from metal_native import paged

    k, v = c["k"] if k is None else k, c["v"] if v is None else v
    want = [k.clone(), v.clone()]
    b = len(c["trees"])
    path, tokens = torch.full((b, steps), -1, dtype=torch.int32), torch.full((b, steps), -1)
    count, new = torch.zeros(b, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)
    pages = k.shape[-4]
    for s, tree in enumerate(c["trees"]):
        a, n = int(c["cu"][s]), len(tree)
        p, t = ref.accept(c["drawn"][a:a + n].tolist(), c["drafted"][a:a + n].tolist(), tree, steps)
        path[s, :len(p)], tokens[s, :len(p)] = torch.tensor(p, dtype=torch.int32), torch.tensor(t, dtype=torch.int64)
        count[s] = len(p)
        off = int(c["lens"][s]) - n
        new[s] = max(0, off + len(p))
        for x, y in ((off + node, off + i) for i, node in enumerate(p)):
            row = c["table"][s].tolist()
            ids = [row[z // c["ps"]] if z >= 0 else -1 for z in (x, y)]
            if x != y and all(0 <= z < pages for z in ids):
                for cache, old in zip(want, (k, v)):
                    cache[..., ids[1], :, y % c["ps"], :] = old[..., ids[0], :, x % c["ps"], :]
    k, v = (x.clone(memory_format=torch.preserve_format) if x.is_contiguous() else x for x in (k, v))
    got = paged.accept(k, v, c["table"], c["lens"], c["drawn"], c["drafted"], c["parents"], c["cu"], steps=steps)
    assert torch.equal(got[0].cpu(), path) and torch.equal(got[1].cpu(), tokens)
    assert torch.equal(got[2].cpu(), count) and torch.equal(got[3].cpu(), new)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    return path


@pytest.mark.parametrize("layers", [None, 1, 5])
@pytest.mark.parametrize("words,kind", [(1, "mixed"), (2, "mixed"), (2, "chain"), (1, "chain"), (3, "star"), (1000, "mixed")])
def test_accept(gpu, layers, words, kind):
    c = accept_case(gpu, [40, 70, 1, 90, 300, 20], [16, 64, 1, 0, 130, 20], layers=layers, words=words, kind=kind, seed=words)
    for steps in (1, 3, 64, 70, 200):
        check_accept(c, steps)


@pytest.mark.parametrize("dtype,KVH,D,ps", [("bf16", 4, 128, 16), ("fp16", 1, 64, 8), ("fp16", 3, 128, 128)])
def test_accept_layouts(gpu, dtype, KVH, D, ps):
    c = accept_case(gpu, [100, 33], [40, 33], layers=3, KVH=KVH, D=D, ps=ps, words=1, dtype=DT[dtype])
    check_accept(c, 20)
    both = torch.stack([c["k"], c["v"]], 2)                       # [layers, pages, 2, ...]
    check_accept(c, 20, both[:, :, 0], both[:, :, 1])
    far = torch.stack([c["k"], c["v"]], 0)                        # and [2, layers, ...]
    check_accept(c, 20, far[0], far[1])
    turned = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (c["k"], c["v"])]
    check_accept(c, 20, *turned)


def test_accept_of_absent_pages_and_short_caches(gpu):
    from metal_native import paged

    c = accept_case(gpu, [100, 33, 60], [64, 33, 20], words=1, kind="chain", seed=1)
    c["drawn"][10] = 5   # the chain breaks there
    c["trees"][0][5:] = [p - 1 if p > 1 else 0 for p in c["trees"][0][5:]]
    c["parents"][:64] = torch.tensor(c["trees"][0], dtype=torch.int32, device=gpu)
    check_accept(c, 64)
    t = c["table"]
    t[0, 3], t[1, 0], t[2, 3] = -1, 10**6, -7
    check_accept(c, 64)
    c["lens"][:] = torch.tensor([50, 4, 1000], device=gpu)   # fewer slots than nodes; more than the table's width: cut to it
    got = paged.accept(c["k"].clone(), c["v"].clone(), t, c["lens"], c["drawn"], c["drafted"], c["parents"], c["cu"], steps=64)
    width = t.shape[1] * 16
    assert got[3].tolist() == [max(0, 50 - 64 + int(got[2][0])), max(0, 4 - 33 + int(got[2][1])), width - 20 + int(got[2][2])]
    for wild in ([-4, 3, 10**6, 5], [9, 2, 0, 117]):
        got = paged.accept(c["k"].clone(), c["v"].clone(), t, c["lens"], c["drawn"], c["drafted"], c["parents"],
                           torch.tensor(wild, dtype=torch.int32, device=gpu), steps=8)
        assert got[0].shape == (3, 8)


def test_accept_counts_its_writes_and_refuses_gradients(gpu):
    from metal_native import MetalNativeError, paged

    c = accept_case(gpu, [40], [16], layers=2, words=1)
    call = lambda k: paged.accept(k, c["v"], c["table"], c["lens"], c["drawn"], c["drafted"], c["parents"], c["cu"], steps=4)  # noqa: E731
    before = c["k"]._version
    call(c["k"])
    assert c["k"]._version == before + 1
    with pytest.raises(MetalNativeError, match="requires a gradient"):
        call(c["k"].clone().requires_grad_())
    with pytest.raises(MetalNativeError):
        call(c["k"][:1].expand(2, -1, -1, -1, -1))   # layers that share memory
    with pytest.raises(MetalNativeError, match="same memory"):   # a slot would be moved twice
        paged.accept(c["k"], c["k"], c["table"], c["lens"], c["drawn"], c["drafted"], c["parents"], c["cu"], steps=4)


# ---- together ----
def test_a_drafted_step_as_it_is_used(gpu):
    """Chains hidden in trees: what the path's nodes saw is what the same tokens see in order, and the cache after the
    step is the one that they leave."""
    from metal_native import paged, sampling

    H, KVH, D, ps, V = 8, 2, 64, 16, 50
    lens, counts = [60, 33, 130], [21, 13, 40]
    c, families, bits = tree_case(gpu, torch.float16, H, KVH, D, ps, lens, counts, seed=4)
    parents, flat, cu = trees(gpu, counts, 4)
    assert torch.equal(paged.ancestors(flat, cu, max(counts)), bits)
    out = paged_tree(c, bits, max_q=max(counts))
    logits = out.float().reshape(sum(counts), -1)[:, :V] * 10
    drawn = sampling.sample(logits, torch.rand(sum(counts), device=gpu, generator=c["gen"]), temperature=0.7, top_k=9)
    drafted = drawn[(cu[:-1].long().repeat_interleave(torch.tensor(counts, device=gpu)) + flat.clamp(min=0)).long()].clone()
    drafted[::3] = V   # a third of the guesses is wrong
    k, v = c["k"].clone(), c["v"].clone()
    path, tokens, count, new = paged.accept(k, v, c["table"], c["lens"], drawn, drafted, flat, cu, steps=16)
    assert int(count.max()) > 1
    for s in range(3):
        p = path[s, :int(count[s])].long()
        rows = cu[s].long() + p
        assert torch.equal(tokens[s, :len(p)], drawn[rows])
        again = paged.attention(c["q"][rows], k, v, c["table"][s:s + 1], new[s:s + 1],
                                torch.tensor([0, len(p)], dtype=torch.int32, device=gpu))
        u = half_step(torch.float16)
        assert float((again.float() - out[rows].float()).abs().max()) <= 8 * u * float(v[v.isfinite()].abs().max())


def test_a_drafted_step_captured(gpu):
    """Replayed between eager calls; the caches are put back before each turn."""
    from metal_native import paged, sampling

    counts, lens = [9, 30], [70, 200]
    c, _, _ = tree_case(gpu, torch.float16, 8, 2, 64, 16, lens, counts, seed=6)
    parents, flat, cu = trees(gpu, counts, 6)
    u = torch.rand(39, device=gpu)
    drafted = torch.randint(0, 3, (39,), device=gpu)
    k0, v0 = c["k"].clone(), c["v"].clone()

    def step():
        bits = paged.ancestors(flat, cu, 30)
        out = paged.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], bits, cu, max_q=30)
        drawn = sampling.sample(out.reshape(39, -1)[:, :3], u, temperature=0.9, top_p=0.99)
        return (bits, out, drawn, *paged.accept(c["k"], c["v"], c["table"], c["lens"], drawn, drafted, flat, cu, steps=8))

    def reset(turn):
        c["k"].copy_(k0)
        c["v"].copy_(v0)
        g = torch.Generator(device=gpu)
        g.manual_seed(turn)
        u.copy_(torch.rand(39, device=gpu, generator=g))
        drafted.copy_(torch.randint(0, 3, (39,), device=gpu, generator=g))

    reset(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(4):
        reset(turn)
        graph.replay()
        kept = [t.clone() for t in got] + [c["k"].clone(), c["v"].clone()]
        reset(turn)
        want = [*step(), c["k"], c["v"]]
        same = lambda a, b: torch.equal(a.nan_to_num(), b.nan_to_num()) if a.is_floating_point() else torch.equal(a, b)  # noqa: E731
        assert all(same(a, b) for a, b in zip(kept, want))


def test_two_streams_at_once(gpu):
    """Steps of two sets of sequences side by side, each with workspaces of its own stream."""
    from metal_native import paged, sampling

    sets = []
    for seed, (lens, counts, width) in enumerate((([9000, 500], [40, 12], 1024), ([300, 77, 650], [100, 65, 200], None))):
        c, _, bits = tree_case(gpu, torch.float16, 32, 8, 128, 16, lens, counts, seed=seed, width=width)
        _, flat, cu = trees(gpu, counts, seed)
        n = sum(counts)
        sets.append((c, bits, flat, cu, torch.rand(n, device=gpu), torch.randint(0, 3, (n,), device=gpu)))

    def step(c, bits, flat, cu, u, drafted):
        k, v = c["k"].clone(), c["v"].clone()
        out = paged.tree_attention(c["q"], k, v, c["table"], c["lens"], bits, c["cu"])
        drawn = sampling.sample(out.reshape(len(u), -1)[:, :3], u, temperature=0.9, top_p=0.99)
        wide = sampling.sample(out.reshape(len(u), -1), u, top_p=0.9)
        return (out, drawn, wide, *paged.accept(k, v, c["table"], c["lens"], drawn, drafted, flat, cu, steps=8), k, v)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(6):
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(step(*s))
    torch.cuda.synchronize()
    same = lambda a, b: torch.equal(a.nan_to_num(), b.nan_to_num()) if a.is_floating_point() else torch.equal(a, b)  # noqa: E731
    for i, g in enumerate(got):
        assert all(same(a, b) for a, b in zip(g, want[i % 2])), i


# ---- offsets of any kind: where results and memory end ----
WILD = [[-5, 3, 10**6, 10**6], [7, 3, 1, 12], [2**31 - 1, -(2**31), 5, 6], [3, 9, 9, -(2**31)], [0, 5, 2**31 - 1, 4], [-4, 12, 12, 2**31 - 1], [9, 2, 0, 11]]


def c_entry(name, *args):
    from metal_native import _lib

    L = _lib.load()
    args = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    rc = getattr(L, name)(*args, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, L.mq_last_error().decode()


@pytest.mark.parametrize("wild", WILD)
@pytest.mark.parametrize("words", [1, 9])
def test_ancestors_of_wild_offsets(gpu, wild, words):
    """A row has the bits of a tree that claims it, or none where rows of no tree begin; each row is written, and nothing
    around them."""
    rows = 12
    flat = torch.tensor([9, 9, -1, 0, 7, 1, -(2**31), 2**31 - 1, 3, 4, 5, 5], dtype=torch.int32, device=gpu)
    cu = torch.tensor(wild, dtype=torch.int32, device=gpu)
    cut = lambda x: max(0, min(x, rows))  # noqa: E731
    may = [set() for _ in range(rows)]
    for r in range(rows):
        if r < cut(wild[0]) or r >= cut(wild[-1]):
            may[r].add((0,) * words)
    for a, b in zip(wild, wild[1:]):
        a, b = cut(a), cut(b)
        for r, line in enumerate(ref.pack(ref.closure(flat[a:b].tolist()), words).tolist() if a < b else [], a):
            may[r].add(tuple(line))
    assert all(may)
    out = torch.full((rows + 8, words), -7, dtype=torch.int64, device=gpu)
    c_entry("mq_paged_ancestors", flat, cu, 3, rows, words, out[4:])
    got = out.cpu()
    assert bool((got[:4] == -7).all()) and bool((got[-4:] == -7).all())
    assert all(tuple(x) in m for x, m in zip(got[4:-4].tolist(), may)), got[4:-4, 0]


@pytest.mark.parametrize("wild", WILD)
def test_accept_of_wild_offsets(gpu, wild):
    """Slots move inside the pages of the tables alone, paths and tokens are a tree's, and nothing around the outputs is
    written."""
    import ctypes

    from test_paged_host import Cache

    steps, b, rows, ps, D, KVH, pages = 5, 3, 12, 16, 64, 2, 7
    drawn, drafted = torch.ones(rows, dtype=torch.int64, device=gpu), torch.ones(rows, dtype=torch.int64, device=gpu)
    parents = torch.tensor([-1, 0, 0, 1, 2, 2, 0, 5, 6, 2, 9, 1], dtype=torch.int32, device=gpu)
    cu = torch.tensor(wild, dtype=torch.int32, device=gpu)
    table = torch.tensor([[3, 4], [5, -1], [9, 6]], dtype=torch.int32, device=gpu)   # pages 3 to 6 of seven; 9 is none
    lens = torch.tensor([20, 9, 32], dtype=torch.int32, device=gpu)
    kv = torch.randn(2, pages + 2, KVH, ps, D, device=gpu).half()
    before = kv.clone()
    k, v = kv[0, 1:-1], kv[1, 1:-1]
    path, count, new = (torch.full(n, -7, dtype=torch.int32, device=gpu) for n in ((b + 2, steps), (b + 2,), (b + 2,)))
    tokens = torch.full((b + 2, steps), -7, dtype=torch.int64, device=gpu)
    c = Cache(k=k.data_ptr(), v=v.data_ptr(), k_page=k.stride(0), k_head=k.stride(1), k_slot=k.stride(2), v_page=v.stride(0), v_head=v.stride(1),
              v_slot=v.stride(2), pages=pages, kv_heads=KVH, page_size=ps, head_dim=D, dtype=0, table=table.data_ptr(), ld_table=2, width=2,
              batch=b, lens=lens.data_ptr())
    c_entry("mq_paged_accept", ctypes.byref(c), 1, 0, 0, drawn, drafted, parents, cu, rows, steps, path[1:], tokens[1:], count[1:], new[1:])
    for out in (path, tokens, count, new):
        assert bool((out[0] == -7).all()) and bool((out[-1] == -7).all())
    cut = lambda x: max(0, min(x, rows))  # noqa: E731
    want, at = before.clone(), [path[1:-1].tolist(), tokens[1:-1].tolist(), count[1:-1].tolist(), new[1:-1].tolist()]
    for s, (a, e) in enumerate(zip(wild, wild[1:])):
        a, e = cut(a), max(cut(a), cut(e))
        n, row = e - a, table[s].tolist()
        p, t = ref.accept([1] * n, [1] * n, parents[a:e].tolist(), steps)
        assert at[0][s] == p + [-1] * (steps - len(p)) and at[1][s] == t + [-1] * (steps - len(p)) and at[2][s] == len(p)
        off = int(lens[s]) - n
        assert at[3][s] == max(0, off + len(p))
        for i, node in enumerate(p):
            x, y = off + node, off + i
            ids = [row[z // ps] if z >= 0 else -1 for z in (x, y)]
            if x != y and all(0 <= z < pages for z in ids):
                want[:, 1 + ids[1], :, y % ps] = before[:, 1 + ids[0], :, x % ps]
    assert torch.equal(kv, want)
