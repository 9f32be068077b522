"""Which attention kernel a paged call takes, and the kernel of 256-row blocks at the masks where it can go wrong."""

import ctypes

import pytest
import torch

from test_paged import DT, build, check_attention
from test_paged_host import Cache, Mask


def plan(rows, heads, kv_heads, dim, page, batch, width, *, chunks=True, window=0, softcap=0.0, slopes=False, prefix=False):
    """(rows of a block, most parts)."""
    from metal_native import _lib

    c = Cache(k=4096, v=4096, pages=1 << 20, kv_heads=kv_heads, page_size=page, head_dim=dim, dtype=0, table=4096, ld_table=width,
              width=width, batch=batch, lens=4096, **{f"{t}_{n}": x for t in "kv" for n, x in
                                                      (("page", kv_heads * page * dim), ("head", page * dim), ("slot", dim))})
    m = Mask(scale=0.1, softcap=softcap, slopes=4096 if slopes else None, window=window, prefix_lens=4096 if prefix else None,
             cu_q=4096 if chunks else None, max_q=0)
    block, parts = ctypes.c_int32(), ctypes.c_int32()
    rc = _lib.load().mq_paged_attention_plan(ctypes.byref(c), ctypes.byref(m), rows, heads, ctypes.byref(block), ctypes.byref(parts))
    assert rc == 0
    return block.value, parts.value


def test_plans():
    assert plan(1, 28, 4, 128, 16, 1, 33, chunks=False) == (32, 5)
    assert plan(48, 32, 8, 128, 16, 48, 500, chunks=False)[0] == 32
    assert plan(1280, 32, 8, 128, 16, 1280, 40, chunks=False)[0] == 32   # single tokens, however many
    assert plan(4096, 28, 4, 128, 64, 1, 512) == (256, 1)
    assert plan(512, 28, 4, 128, 16, 1, 512)[0] == 256 and plan(512, 28, 4, 128, 16, 1, 512)[1] > 1
    assert plan(20, 28, 4, 128, 16, 1, 38)[0] == 32
    for extra in (dict(softcap=30.0), dict(slopes=True)):   # a softmax that weighs more needs more work to pay
        assert plan(160, 28, 4, 128, 16, 4, 64, **extra)[0] == 32
        assert plan(512, 28, 4, 128, 16, 1, 512, **extra)[0] == 256


def test_plan_refuses():
    from metal_native import _lib

    L, n = _lib.load(), ctypes.c_int32()
    assert L.mq_paged_attention_plan(None, None, 1, 1, ctypes.byref(n), ctypes.byref(n)) == 4


# H, KVH, D, lens, new, parts (whether more than one), mask
SPREAD = ([700, 64, 513, 1, 200, 0], [600, 64, 500, 1, 130, 0])
SHORT = ([330, 400, 258, 320, 512, 300, 340, 290, 321, 65], [320, 300, 258, 310, 400, 300, 320, 280, 300, 65])
LONG = ([8000, 40, 1000, 0], [600, 40, 33, 0])
MANY = {
    "cap": (32, 4, 128, *SPREAD, False, dict(softcap=15.0)),
    "bias": (32, 4, 128, *SPREAD, False, dict(bias=True)),
    "both, a prefix": (32, 4, 64, *SPREAD, False, dict(softcap=15.0, bias=True, prefix=[90, 3, 0, 0, 10**6, 1])),
    "a window of one": (64, 2, 64, *SHORT, False, dict(softcap=9.0, window=1)),
    "a window under a tile": (64, 2, 64, *SHORT, False, dict(bias=True, window=40)),
    "a gap behind the prefix": (64, 2, 64, *SHORT, False, dict(softcap=9.0, bias=True, window=70, prefix=[65, 200, 0, 1, 130, 64, 63, 0, 5, 65])),
    "in parts": (14, 2, 128, *LONG, True, dict(softcap=15.0, bias=True)),
    "a window and a prefix in parts": (14, 2, 64, *LONG, True, dict(bias=True, window=5000, prefix=[200, 3, 0, 0])),
    "plain": (32, 4, 128, *SPREAD, False, {}),
    "a plain window": (32, 4, 128, *SPREAD, False, dict(window=150, prefix=[90, 3, 0, 0, 10**6, 1])),
}


def table_width(lens, wide):
    return max(-(-max(lens) // 16), wide)


@pytest.mark.parametrize("name", list(MANY))
def test_the_cases_below_take_blocks_of_256_rows(name):
    """By half as much work again at least: the rule may move a little without their going elsewhere unseen."""
    H, KVH, D, lens, new, parts, how = MANY[name]
    rows = 2 * sum(new) // 3
    got = plan(rows, H, KVH, D, 16, len(lens), table_width(lens, 100), window=how.get("window", 0), softcap=how.get("softcap", 0.0),
               slopes=how.get("bias", False), prefix="prefix" in how)
    assert got[0] == 256, got
    got = plan(sum(new), H, KVH, D, 16, len(lens), table_width(lens, 100), window=how.get("window", 0), softcap=how.get("softcap", 0.0),
               slopes=how.get("bias", False), prefix="prefix" in how)
    assert got[0] == 256 and (got[1] > 1) == parts, got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("name", list(MANY))
def test_many_rows_masked(gpu, dtype, name):
    H, KVH, D, lens, new, _, how = MANY[name]
    how = dict(how)
    c = build(gpu, DT[dtype], H, KVH, D, 16, lens, new, seed=len(name), width=table_width(lens, 100))
    if how.pop("bias", False):
        how["slopes"] = torch.rand(H, device=gpu, generator=c["gen"]) * 0.1
    if "prefix" in how:
        how["prefix"] = torch.tensor(how["prefix"], dtype=torch.int32, device=gpu)
    check_attention(c, **how)


@pytest.mark.gpu
def test_absent_pages_at_the_end_of_the_longest_sequence(gpu):
    """2^31 - 32 slots, whose last tile of 64 ends past 32 bits: 600 tokens that see the last 300 slots, one page of them absent."""
    from metal_native import paged

    H, D, ps, n, window, width = 16, 64, 32, 600, 300, 2**26 - 1
    assert plan(n, H, 1, D, ps, 1, width, window=window)[0] == 256
    g = torch.Generator(device=gpu)
    g.manual_seed(2)
    tail = 40   # pages whose slots these tokens may see
    k, v = (torch.randn(tail, 1, ps, D, device=gpu, generator=g).half() for _ in range(2))
    far = torch.zeros(1, width, dtype=torch.int32, device=gpu)
    far[0, -tail:] = torch.arange(tail, device=gpu)
    for absent in (None, 1, 2, 9):
        near = torch.arange(tail, dtype=torch.int32, device=gpu)[None].clone()
        far[0, -tail:] = near[0]
        if absent:
            near[0, -absent] = far[0, -absent] = -1
        q = torch.randn(n, H, D, device=gpu, generator=g).half()
        cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        end = torch.tensor([width * ps], dtype=torch.int32, device=gpu)
        a, la = paged.attention(q, k, v, far, end, cu, window=window, return_lse=True)
        b, lb = paged.attention(q, k, v, near, torch.tensor([tail * ps], dtype=torch.int32, device=gpu), cu, window=window, return_lse=True)
        # the same slots in other tiles: two results, each within the bounds of one
        e = torch.finfo(torch.float16).eps / 2
        assert bool(((la - lb).abs() <= 2 * ((D + 4) * 60 + n) * 2.0**-24).all())
        assert bool(((a - b).float().abs() <= 4 * e * v.float().abs().max()).all())
