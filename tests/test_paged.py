"""Paged-cache operators against float64 forms of their definitions."""

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def build(dev, dt, H, KVH, D, ps, lens, new=None, seed=0, extra=3, width=None, amp=1.0, junk=float("nan")):
    """Caches whose slots past every length hold `junk`, pages in random order."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    pages = [-(-t // ps) for t in lens]
    pool = sum(pages) + extra
    rn = lambda *s: (torch.randn(*s, device=dev, generator=g) * amp).to(dt)  # noqa: E731
    k, v = torch.full((pool, KVH, ps, D), junk, device=dev, dtype=dt), torch.full((pool, KVH, ps, D), junk, device=dev, dtype=dt)
    order = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    table = torch.full((len(lens), width or max(max(pages), 1)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
        for p in range(n):
            m = min(ps, lens[i] - p * ps)
            k[table[i, p].long(), :, :m] = rn(KVH, m, D)
            v[table[i, p].long(), :, :m] = rn(KVH, m, D)
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu, rows = None, len(lens)
    if new is not None:
        cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
        rows = sum(new)
    q = rn(rows, H, D)
    free = order[at:]
    return dict(q=q, k=k, v=v, table=table, lens=lt, cu=cu, free=free, gen=g)


def check_attention(c, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None, max_q=None):
    from metal_native import paged

    s = scale or 1.0 / math.sqrt(c["q"].shape[2])
    out, lse = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], scale=s, softcap=softcap,
                               slopes=slopes, window=window, prefix_lens=prefix, max_q=max_q, return_lse=True)
    o, l, ob, lb = ref.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], scale=s, softcap=softcap,
                                 slopes=slopes, window=window, prefix=prefix)
    got = out.double().cpu()
    assert bool((torch.isnan(got) == torch.isnan(o)).all())
    fin = ~torch.isnan(o)
    assert bool(((got == o) | ((got - o).abs() <= ob))[fin].all()), float(((got - o).abs() / ob)[fin].nan_to_num().max())
    gl = lse.double().cpu()
    assert bool(((gl == l) | (torch.isnan(gl) & torch.isnan(l)) | ((gl - l).abs() <= lb)).all())
    return out, lse, s


HEADS = [(28, 4, 128), (14, 2, 64), (8, 8, 128), (8, 1, 128), (6, 2, 64)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("ps", [8, 16, 128])
def test_attention_of_single_tokens(gpu, dtype, H, KVH, D, ps):
    lens = [1, 0, 31, 32, 33, 64, 65, 127, 128, 129, 513, 700, 2, 16]
    check_attention(build(gpu, DT[dtype], H, KVH, D, ps, lens, seed=D + ps))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
def test_attention_of_chunks(gpu, dtype, H, KVH, D):
    lens, new = [1, 40, 0, 64, 300, 129, 77], [1, 3, 0, 64, 65, 0, 77]
    check_attention(build(gpu, DT[dtype], H, KVH, D, 16, lens, new, seed=D), max_q=77)


@pytest.mark.parametrize("H,KVH,D", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,prefix", [(0, True), (1, False), (7, True), (64, True), (100, False), (1000, True)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (20.0, True)])
def test_masks_and_scores(gpu, H, KVH, D, window, prefix, softcap, bias):
    lens, new = [200, 65, 330, 1, 128], [9, 65, 130, 1, 1]
    c = build(gpu, torch.float16, H, KVH, D, 32, lens, new, seed=window + H, amp=2.0)
    slopes = torch.rand(H, device=gpu, generator=c["gen"]) if bias else None
    pre = torch.tensor([0, 70, 33, 5, 500], dtype=torch.int32, device=gpu) if prefix else None
    check_attention(c, softcap=softcap, slopes=slopes, window=window, prefix=pre)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,masked", [(128, False), (64, True)])
def test_attention_of_many_rows(gpu, dtype, D, masked):
    """Enough rows for the kernel whose workgroups take 128 of them."""
    lens, new = [700, 64, 513, 1, 200, 0], [600, 64, 500, 1, 130, 0]
    c = build(gpu, DT[dtype], 32, 4, D, 16, lens, new, seed=D)
    how = {}
    if masked:
        how = dict(softcap=15.0, slopes=torch.rand(32, device=gpu) * 0.1, window=150,
                   prefix=torch.tensor([90, 3, 0, 0, 10**6, 1], dtype=torch.int32, device=gpu))
    check_attention(c, **how)


def test_chunk_longer_than_the_cache_and_rows_of_no_sequence(gpu):
    """Positions before slot 0 see nothing, or the prefix; rows past the last chunk are left to nobody."""
    from metal_native import paged

    c = build(gpu, torch.float16, 8, 2, 64, 16, [3, 20], [10, 20], seed=5)
    check_attention(c)
    check_attention(c, prefix=torch.tensor([2, 0], dtype=torch.int32, device=gpu))
    wild = torch.tensor([-5, 10, 10**6], dtype=torch.int32, device=gpu)   # cut to 0, 10, 30
    a = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], wild)
    assert torch.equal(a, paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"]))


@pytest.mark.parametrize("many", [False, True])
def test_pages_outside_the_cache_do_not_exist(gpu, many):
    lens, new = ([600, 300], [512, 300]) if many else ([600, 300], [5, 1])
    c = build(gpu, torch.float16, 32, 8, 128, 16, lens, new, seed=3)
    t = c["table"]
    t[0, 3], t[0, 30], t[1, 0], t[1, 18] = -1, 10**6, c["k"].shape[0], -2**31
    check_attention(c)
    t[1, :] = -1   # a sequence without a slot
    check_attention(c)


@pytest.mark.parametrize("many", [False, True])
def test_what_hidden_slots_hold_does_not_matter(gpu, many):
    """Infinities and NaN in slots that some rows of a tile see and others do not."""
    lens, new = ([600, 300], [512, 300]) if many else ([600, 300], [9, 40])
    c = build(gpu, torch.float16, 32, 8, 128, 16, lens, new, seed=4, junk=float("inf"))
    for pos, what in ((595, float("nan")), (598, float("inf"))):
        c["v"][c["table"][0, pos // 16].long(), 0, pos % 16, 5] = what
        c["k"][c["table"][0, pos // 16].long(), 1, pos % 16, 7] = what
    c["v"][c["table"][1, 290 // 16].long(), :, 290 % 16] = float("nan")
    check_attention(c)
    check_attention(c, window=3)


def test_scores_far_apart(gpu):
    """Rows whose largest score grows along the cache, weights far under it, and infinite scores."""
    c = build(gpu, torch.float16, 8, 2, 64, 16, [500, 400, 300], [4, 1, 2], seed=6)
    for s, p in ((0, 30), (0, 20), (1, 24), (1, 2)):
        c["k"][c["table"][s, p].long()] *= 30
    check_attention(c)
    check_attention(c, scale=1e-3)
    c = build(gpu, torch.bfloat16, 8, 2, 64, 16, [32, 33], seed=6)
    c["q"][0] = 3e38
    c["k"][c["table"][0, 1].long()] = -3e38   # overflows to -inf: no weight
    c["k"][c["table"][0, 0].long()] = 1e-37
    check_attention(c)


def test_weights_under_the_range_of_fp16_together_count(gpu):
    """One key ahead of 2^16 equal ones by 17 in the exponent: half a percent of the sum."""
    from metal_native import paged

    n, ps, D = 65537, 128, 64
    pages = -(-n // ps)
    k = torch.zeros(pages, 1, ps, D, device=gpu, dtype=torch.float16)
    v = torch.ones(pages, 1, ps, D, device=gpu, dtype=torch.float16)
    k[0, 0, 0, 0], v[0, 0, 0] = 17.0, 0.0
    q = torch.zeros(1, 1, D, device=gpu, dtype=torch.float16)
    q[..., 0] = 1.0
    table = torch.arange(pages, device=gpu, dtype=torch.int32)[None]
    out = paged.attention(q, k, v, table, torch.tensor([n], dtype=torch.int32, device=gpu), scale=1.0)
    w = (n - 1) * math.exp(-17.0)
    want = w / (1 + w)
    # every weight off by at most half of 2^-24 / 2^7 = 2^-32, or 2^-11 of itself, whichever is more
    assert float((out.double() - want).abs().max()) <= want * 2.0**-10 + n * 2.0**-32 + 2.0**-25


def test_strides_streams_and_repeats(gpu):
    """Caches interleaved or with heads inside slots, queries out of a fused row, another stream: the same bits."""
    from metal_native import paged

    c = build(gpu, torch.bfloat16, 28, 4, 128, 16, [300, 41, 700], [40, 1, 7], seed=7)
    want = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"])
    P, KVH, ps, D = c["k"].shape
    both = torch.stack([c["k"], c["v"]], 1)
    flat_k, flat_v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (c["k"], c["v"]))
    T, H, _ = c["q"].shape
    fused = torch.zeros(T, H + 8, D, device=gpu, dtype=torch.bfloat16)
    fused[:, :H] = c["q"]
    wide = torch.full((3, c["table"].shape[1] + 5), 10**8, dtype=torch.int32, device=gpu)
    wide[:, :-5] = c["table"]
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    for k, v in ((both[:, 0], both[:, 1]), (flat_k, flat_v)):
        assert torch.equal(want, paged.attention(fused[:, :H], k, v, wide[:, :-5], c["lens"], c["cu"]))
        with torch.cuda.stream(side):
            got = paged.attention(c["q"].transpose(0, 1).contiguous().transpose(0, 1), k, v, c["table"], c["lens"], c["cu"])
        side.synchronize()
        assert torch.equal(want, got)
    odd = torch.zeros(T * H * D + 1, device=gpu, dtype=torch.bfloat16)[1:].view(T, H, D)   # not 16-byte aligned
    assert torch.equal(want, paged.attention(odd.copy_(c["q"]), c["k"], c["v"], c["table"], c["lens"].flip(0).flip(0), c["cu"]))


def test_offsets_past_32_bits(gpu):
    """Pages that start more than 2^32 bytes into the cache, and a table that names the same page twice."""
    from metal_native import paged

    pages, KVH, ps, D = 40000, 4, 128, 128   # 5.2 GB
    k = torch.empty(pages, KVH, ps, D, device=gpu, dtype=torch.float16)
    v = torch.empty_like(k)
    ids = [39999, 2, 33000, 2, 16384, 39998]
    small_k = torch.randn(len(ids), KVH, ps, D, device=gpu).half()
    small_v = torch.randn(len(ids), KVH, ps, D, device=gpu).half()
    small_k[3], small_v[3] = small_k[1], small_v[1]
    for i, p in enumerate(ids):
        k[p], v[p] = small_k[i], small_v[i]
    q = torch.randn(3, 8, D, device=gpu).half()
    lens = torch.tensor([700], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=gpu)
    far = torch.tensor([ids], dtype=torch.int32, device=gpu)
    near = torch.arange(len(ids), dtype=torch.int32, device=gpu)[None]
    a, la = paged.attention(q, k, v, far, lens, cu, return_lse=True)
    b, lb = paged.attention(q, small_k, small_v, near, lens, cu, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert torch.equal(paged.attention_mass(q, k, far, lens, la, cu), paged.attention_mass(q, small_k, near, lens, la, cu))
    to = torch.tensor([[39000, 20000]], dtype=torch.int32, device=gpu)
    mass = torch.rand(1, KVH, 6 * ps, device=gpu)
    kept, n, _ = paged.evict(k, v, far, lens, mass, to, 200, recent=10)
    j = kept[0, 2].long()
    got = torch.cat([k[39000, 2], k[20000, 2]])[:200]
    assert int(n) == 200 and torch.equal(got, small_k[j // ps, 2, j % ps])


def check_mass(c, **how):
    from metal_native import paged

    _, lse, s = check_attention(c, **how)
    prefix = how.pop("prefix", None)
    kw = {k: x for k, x in how.items() if k != "scale"}
    got = paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], lse, c["cu"], scale=s, prefix_lens=prefix, **kw)
    want, bound = ref.mass(c["q"], c["k"], c["table"], c["lens"], lse, c["cu"], scale=s, prefix=prefix,
                           **{k: x for k, x in kw.items() if k != "max_q"})
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("chunk", [False, True])
def test_mass(gpu, dtype, H, KVH, D, chunk):
    lens, new = [1, 0, 255, 256, 257, 700, 40], [1, 0, 3, 100, 257, 17, 40]
    check_mass(build(gpu, DT[dtype], H, KVH, D, 16, lens, new if chunk else None, seed=D))


@pytest.mark.parametrize("window,prefix", [(0, True), (5, False), (300, True)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (20.0, True)])
def test_mass_masks(gpu, window, prefix, softcap, bias):
    c = build(gpu, torch.float16, 14, 2, 64, 32, [900, 65, 330], [300, 65, 1], seed=window)
    slopes = torch.rand(14, device=gpu, generator=c["gen"]) * 0.2 if bias else None
    pre = torch.tensor([0, 70, 33], dtype=torch.int32, device=gpu) if prefix else None
    check_mass(c, window=window, prefix=pre, softcap=softcap, slopes=slopes)


def test_mass_of_many_rows_in_parts_and_absent_slots(gpu):
    c = build(gpu, torch.float16, 8, 1, 128, 16, [300, 1100], [300, 900], seed=9)
    c["table"][1, 4], c["table"][1, 60] = -1, 10**7
    got = check_mass(c, max_q=900)
    assert float(got[1, :, 64:80].abs().max()) == 0 and float(got[1, :, 960:976].abs().max()) == 0
    # each row's weights sum to one: all of them to the number of rows, up to the sums' rounding
    assert abs(float(got.double().sum()) - 1200 * 8) <= 9600 * 2.0**-14


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", HEADS)
@pytest.mark.parametrize("sections", [None, (0.25, 0.375, 0.375), "odd"])
@pytest.mark.parametrize("chunk", [False, True])
def test_rope(gpu, dtype, H, KVH, D, sections, chunk):
    from metal_native import paged

    lens, new = [1, 40, 0, 64, 300, 129], [1, 3, 0, 64, 65, 0]
    if not chunk:
        lens, new = [1, 40, 64, 300], None
    c = build(gpu, DT[dtype], H, KVH, D, 16, lens, new, seed=D, junk=7.0)
    rows, half = c["q"].shape[0], D // 2
    sec = None if sections is None else ((5, 0, half - 12, 7) if sections == "odd" else tuple(int(x * half) for x in sections))
    axes = 1 if sec is None else len(sec)
    ang = torch.rand(400, D, device=gpu, generator=c["gen"]) * 6.3
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(-3, 410, (axes, rows), device=gpu, generator=c["gen"])
    qkv = torch.randn(rows, (H + 2 * KVH) * D, device=gpu, generator=c["gen"]).to(DT[dtype])
    k0, v0 = c["k"].clone(), c["v"].clone()
    q = paged.rope_kv(qkv, cos, sin, pos if axes > 1 else pos[0], c["k"], c["v"], c["table"], c["lens"], c["cu"], sections=sec)
    axis = torch.tensor([a for a, n in enumerate(sec or (half,)) for _ in range(n)], device=gpu)
    p = pos.clamp(0, 399)[axis].t()
    f = torch.arange(half, device=gpu)
    cc, ss = cos[p, f].double()[:, None], sin[p, f].double()[:, None]
    x = qkv.double().view(rows, H + 2 * KVH, D)
    lo, hi = x[:, :H + KVH, :half], x[:, :H + KVH, half:]
    want = torch.cat([lo * cc - hi * ss, hi * cc + lo * ss], 2)
    size = torch.cat([(lo * cc).abs() + (hi * ss).abs()] * 2, 2) + torch.cat([(hi * cc).abs() + (lo * ss).abs()] * 2, 2)
    bound = ref.half_step(DT[dtype]) * want.abs() + 2 * ref.E * size + 2.0**-25   # one rounding; products and sum in fp32
    assert bool(((q.double() - want[:, :H]).abs() <= bound[:, :H]).all())
    at = 0
    for s, (n_all, n) in enumerate(zip(lens, new or [1] * len(lens))):
        for i in range(n):
            j = n_all - n + i
            page = int(c["table"][s, j // 16])
            err = (c["k"][page, :, j % 16].double() - want[at, H:]).abs()
            assert bool((err <= bound[at, H:]).all())
            assert torch.equal(c["v"][page, :, j % 16], qkv.view(rows, -1, D)[at, H + KVH:])
            k0[page, :, j % 16], v0[page, :, j % 16] = c["k"][page, :, j % 16], c["v"][page, :, j % 16]
            at += 1
    assert torch.equal(k0, c["k"]) and torch.equal(v0, c["v"])   # nothing else written


def test_rope_writes_no_page_that_is_not_there(gpu):
    from metal_native import paged

    c = build(gpu, torch.float16, 8, 2, 64, 16, [5, 20, 40, 9], seed=1, junk=7.0)
    c["table"][0, 0], c["table"][1, 1], c["table"][2, 2] = -1, c["k"].shape[0], 2**31 - 1
    c["lens"][3] = 10**9   # past the table: cut to its width
    cos = torch.ones(50, 64, device=gpu)
    k0 = c["k"].clone()
    qkv = torch.randn(4, 12 * 64, device=gpu).half()
    q = paged.rope_kv(qkv, cos, 0 * cos, torch.zeros(4, dtype=torch.int64, device=gpu), c["k"], c["v"], c["table"], c["lens"])
    assert torch.equal(q.reshape(4, -1), qkv[:, :512])
    last = int(c["table"][3, -1])
    if 0 <= last < c["k"].shape[0]:
        k0[last, :, 15] = c["k"][last, :, 15]
    assert torch.equal(k0, c["k"])


def check_evict(c, mass, budget, recent, KVH, ps, lens, spread=None):
    from metal_native import paged

    b, need = len(lens), -(-budget // ps)
    to = c["free"][:b * need].reshape(b, need) if spread is None else spread
    k0, v0, m = c["k"].clone(), c["v"].clone(), mass.cpu()
    kept, n, left = paged.evict(c["k"], c["v"], c["table"], c["lens"], mass, to, budget, recent=recent)
    tab, tt = c["table"].cpu(), to.cpu()
    for s, total in enumerate(lens):
        assert int(n[s]) == min(total, budget)
        for h in range(KVH):
            want = ref.keep(m[s, h], total, budget, recent)
            row = kept[s, h].tolist()
            assert row[:len(want)] == want and row[len(want):] == [-1] * (budget - len(want))
            l = left[s, h].cpu()
            got_l, want_l = l[:len(want)], m[s, h][want] if want else l[:0]
            assert bool(((got_l == want_l) | (torch.isnan(got_l) & torch.isnan(want_l))).all())
            assert float(l[len(want):].abs().sum()) == 0
            w, d = torch.tensor(want, dtype=torch.long), torch.arange(len(want))
            dst, src = (tt[s][d // ps].long(), tab[s][w // ps].long()) if want else (d, w)
            k0[dst, h, d % ps], v0[dst, h, d % ps] = k0[src, h, w % ps], v0[src, h, w % ps]
    assert torch.equal(k0, c["k"]) and torch.equal(v0, c["v"])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,ps", [(128, 16), (64, 64), (64, 8)])
@pytest.mark.parametrize("budget,recent", [(100, 0), (100, 100), (100, 37), (1, 0), (513, 64), (2000, 5)])
def test_evict(gpu, dtype, D, ps, budget, recent):
    lens = [0, 1, 99, 100, 101, 700, 1500]
    c = build(gpu, DT[dtype], 8, 2, D, ps, lens, seed=budget + recent, extra=len(lens) * -(-budget // ps) + 2, junk=3.0)
    u = torch.rand(len(lens), 2, c["table"].shape[1] * ps, device=gpu, generator=c["gen"])
    check_evict(c, torch.where(u < 0.2, torch.zeros_like(u), 3 * u**8), budget, recent, 2, ps, lens)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "special", "close"])
def test_evict_ties_and_special_values(gpu, kind):
    lens = [3000, 64, 1025]
    c = build(gpu, torch.float16, 8, 2, 64, 16, lens, seed=2, extra=3 * 40, junk=3.0)
    shape = (3, 2, c["table"].shape[1] * 16)
    u = torch.rand(shape, device=gpu, generator=c["gen"])
    m = {"equal": torch.full(shape, 0.5, device=gpu), "few": (u * 3).floor(), "signs": (u - 0.5),
         "special": torch.where(u < 0.1, torch.full_like(u, float("nan")),
                                torch.where(u < 0.2, torch.full_like(u, float("inf")),
                                            torch.where(u < 0.5, -torch.zeros_like(u), torch.zeros_like(u)))),
         "close": 1.0 + torch.floor(u * 50) * 2.0**-23}[kind]
    check_evict(c, m, 600, 20, 2, 16, lens)


def test_evict_pages_that_are_not_there(gpu):
    from metal_native import paged

    c = build(gpu, torch.float16, 4, 1, 64, 16, [200], seed=8, extra=10, junk=3.0)
    mass = torch.arange(200 + 8, device=gpu, dtype=torch.float32).reshape(1, 1, -1)[..., :208].contiguous()
    src = c["table"].clone()
    c["table"][0, 12] = -1   # slots 192 .. 199
    to = torch.stack([c["free"][0], torch.tensor(-7, dtype=torch.int32, device=gpu)])[None]
    k0 = c["k"].clone()
    kept, n, _ = paged.evict(c["k"], c["v"], c["table"], c["lens"], mass, to, 24, recent=4)
    assert kept[0, 0].tolist() == list(range(176, 200)) and int(n) == 24
    page = int(c["free"][0])
    assert torch.equal(c["k"][page, 0], k0[src[0, 11].long(), 0])   # 176 .. 191; the rest had no page to go to
    k0[page] = c["k"][page]
    assert torch.equal(k0, c["k"])
    to = c["free"][:2][None]
    paged.evict(c["k"], c["v"], c["table"], c["lens"], mass, to, 24, recent=4)
    assert float(c["k"][int(c["free"][1]), 0, :8].abs().max()) == 0   # slots without a page move as zeros


def test_graph_of_a_step(gpu):
    """rope, attention, mass and eviction captured once, replayed among eager work of the same calls."""
    from metal_native import paged

    H, KVH, D, ps = 28, 4, 128, 16
    c = build(gpu, torch.float16, H, KVH, D, ps, [513, 33, 200], seed=11, extra=40, junk=1.0)
    cos, sin = torch.rand(600, D, device=gpu), torch.rand(600, D, device=gpu)
    qkv = torch.randn(3, (H + 2 * KVH) * D, device=gpu).half()
    to = c["free"][:18].reshape(3, 6)

    def step():
        q = paged.rope_kv(qkv, cos, sin, c["lens"].long() - 1, c["k"], c["v"], c["table"], c["lens"])
        out, lse = paged.attention(q, c["k"], c["v"], c["table"], c["lens"], return_lse=True)
        m = paged.attention_mass(q, c["k"], c["table"], c["lens"], lse)
        return (q, out, lse, m, *paged.evict(c["k"], c["v"], c["table"], c["lens"], m, to, 96, recent=8))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        qkv.copy_(torch.randn(3, (H + 2 * KVH) * D, device=gpu))
        c["lens"].copy_(torch.tensor([[513, 33, 200], [100, 1, 0], [512, 32, 199], [513, 48, 7]][i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held] + [c["k"].clone(), c["v"].clone()]
        want = [*step(), c["k"], c["v"]]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b) or bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def test_many_sequences(gpu):
    """Chunks found among more sequences than a wavefront has lanes, some of no tokens."""
    n = 150
    new = [(7 * i) % 5 for i in range(n)]
    lens = [x + (11 * i) % 40 for i, x in enumerate(new)]
    check_mass(build(gpu, torch.float16, 6, 2, 64, 8, lens, new, seed=12), max_q=4)
    check_attention(build(gpu, torch.bfloat16, 28, 4, 128, 16, lens, new, seed=13))
    check_attention(build(gpu, torch.float16, 32, 8, 128, 16, [x + 20 for x in lens] * 7, seed=14))   # single tokens


@pytest.mark.parametrize("ps", [8, 64, 128])
def test_many_rows_of_other_pages_and_masks(gpu, ps):
    c = build(gpu, torch.float16, 32, 8, 64, ps, [900, 640, 129], [700, 500, 129], seed=ps)
    check_attention(c)
    pre = torch.tensor([65, 200, 0], dtype=torch.int32, device=gpu)   # a gap between the prefix and the window
    check_attention(c, window=70, prefix=pre)
    check_attention(c, window=1)


@pytest.mark.parametrize("max_q", [1, 2, 64])
def test_a_longest_chunk_that_is_understated(gpu, max_q):
    check_mass(build(gpu, torch.float16, 14, 2, 64, 16, [400, 65], [300, 65], seed=15), max_q=max_q)


def test_a_table_far_wider_than_the_sequences(gpu):
    c = build(gpu, torch.float16, 8, 2, 64, 16, [700, 0, 33], seed=16, width=5000)
    check_mass(c)
    check_mass(c, window=40)
    c = build(gpu, torch.float16, 8, 2, 64, 16, [700, 0, 33], [50, 0, 33], seed=17, width=5000)
    check_mass(c)


@pytest.mark.parametrize("lens,width", [([9000, 20, 5001], 80), ([40000, 3, 33000], None), ([700, 0, 90], 500)])
@pytest.mark.parametrize("budget,recent", [(3000, 64), (64, 0)])
def test_evict_from_long_tables(gpu, lens, width, budget, recent):
    """Tables of 10240, 40064 and 64000 slots: weights kept in registers, and read again each time."""
    c = build(gpu, torch.bfloat16, 4, 1, 64, 128, lens, seed=18, extra=3 * 24, width=width, junk=2.0)
    u = torch.rand(3, 1, c["table"].shape[1] * 128, device=gpu, generator=c["gen"])
    check_evict(c, torch.where(u < 0.3, torch.zeros_like(u), (40 * u).floor() + u * (u > 0.7)), budget, recent, 1, 128, lens)


def test_single_tokens_of_very_many_sequences(gpu):
    """More row blocks than a grid holds along z, and many rows that are all single tokens."""
    from metal_native import paged

    for n, H, KVH in ((1500, 32, 8), (40000, 64, 1)):
        c = build(gpu, torch.float16, H, KVH, 64, 8, [3, 17, 40], seed=n)
        rows = torch.arange(n, device=gpu) % 3
        q = torch.randn(3, H, 64, device=gpu).half()
        table, lens = c["table"][rows], c["lens"][rows]
        out, lse = paged.attention(q[rows], c["k"], c["v"], table, lens, return_lse=True)
        o, l, ob, lb = ref.attention(q, c["k"], c["v"], c["table"], c["lens"], scale=0.125)
        at = rows.cpu()
        assert bool(((out.double().cpu() - o[at]).abs() <= ob[at]).all())
        assert bool(((lse.double().cpu() - l[at]).abs() <= lb[at]).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", [(14, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("masked", [False, True])
def test_chunks_behind_long_caches(gpu, dtype, H, KVH, D, masked):
    """Many rows whose slots are dealt out to several workgroups, sequences of fewer parts among them."""
    c = build(gpu, DT[dtype], H, KVH, D, 16, [3200, 40, 1000, 0], [600, 40, 33, 0], seed=D)
    how = {}
    if masked:
        how = dict(softcap=15.0, slopes=torch.rand(H, device=gpu) * 0.01, window=2500,
                   prefix=torch.tensor([90, 3, 0, 0], dtype=torch.int32, device=gpu))
    check_attention(c, **how)
    first = c["table"][0]
    first[3], first[100] = -1, 10**6
    c["v"][first[150].long(), :, 5] = float("nan")   # slot 2405: seen by all rows; 3195: by the last few
    c["v"][first[199].long(), 0, 11] = float("inf")
    check_attention(c, **how)


def test_chunks_behind_long_caches_repeat(gpu):
    from metal_native import paged

    c = build(gpu, torch.float16, 28, 4, 128, 16, [5000, 3000], [300, 200], seed=3)
    a, la = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True)
    for _ in range(3):
        b, lb = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
