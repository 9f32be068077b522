"""Operators for drafted tokens on the host: bits of a row, refused arguments."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from test_paged_host import BAD_CACHE, BAD_MASK, BAD_QUERY, BAD_V, BIG, CACHE, CU, LIBRARY, MASK, P, ROOT, ROWS, V, Cache, Mask
from test_paged_host import arguments as paged_arguments


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_bits_of_a_row(tmp_path):
    """Every 64 of them, from in front of the row to past it, read inside it alone (bounds trapped)."""
    src = tmp_path / "bits.cpp"
    src.write_text('''
#include <cstdio>
#include <vector>
#include "mq_paged.hpp"
int main() {
  long bad = 0;
  for (int words = 1; words <= 4; ++words) {
    std::vector<uint64_t> row(words);
    for (int w = 0; w < words; ++w) row[w] = 0x9E3779B97F4A7C15ull * (w + 3) ^ (0xD1B54A32D192ED03ull >> w);
    for (int64_t d = -200; d <= 64 * words + 200; ++d) {
      uint64_t want = 0;
      for (int i = 0; i < 64; ++i) {
        const int64_t at = d + i;
        if (at >= 0 && at < 64 * words) want |= (row[at / 64] >> (at % 64) & 1) << i;
      }
      bad += mq::paged_tree_bits(row.data(), words, d) != want;
    }
    for (int64_t d : {-(int64_t{1} << 40), int64_t{1} << 40, -(int64_t{1} << 31), int64_t{1} << 31}) bad += mq::paged_tree_bits(row.data(), words, d) != 0;
  }
  std::printf("bad %ld\\n", bad);
}
''')
    exe = tmp_path / "bits"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{os.path.join(ROOT, 'metal-native_amd', 'csrc')}", str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env={k: v for k, v in os.environ.items() if k != "LD_PRELOAD"})
    assert out.returncode == 0 and "bad 0" in out.stdout, out.stdout + out.stderr


def arguments(dev):
    h = paged_arguments(dev)["attention"]
    i = dict(dtype=torch.int32, device=dev)
    cache = {n: h[n] for n in ("k_cache", "v_cache", "table", "lens")}
    return {
        "ancestors": dict(parents=torch.zeros(ROWS, **i), cu=h["cu"], max_q=3),
        "tree_attention": dict(h, tree=torch.ones(ROWS, 1, dtype=torch.int64, device=dev)),
        "accept": dict(cache, drawn=torch.zeros(ROWS, dtype=torch.int64, device=dev), drafted=torch.zeros(ROWS, dtype=torch.int64, device=dev),
                       parents=torch.zeros(ROWS, **i), cu=h["cu"], steps=2),
    }


INT64 = [None, lambda x: x.int(), lambda x: x[:-1], lambda x: x[None]]
CHANGES = {
    "ancestors": {"parents": [None, lambda x: x.long(), lambda x: x[None]], "cu": [lambda x: x[:1], lambda x: x.long(), lambda x: x[None]],
                  "max_q": [lambda _: -1, lambda _: 2**31]},
    "tree_attention": {**CACHE, **V, **CU, **MASK, "tree": [None, lambda x: x.int(), lambda x: x[:-1], lambda x: x[:, :0], lambda x: x[:, 0]]},
    "accept": {**CACHE, **V, **CU, "drawn": INT64, "drafted": INT64, "parents": [None, lambda x: x.long(), lambda x: x[1:]],
               "steps": [lambda _: 0, lambda _: -3, lambda _: 2**31]},
}
# the caches of accept may have a dimension of layers, in which case both have it
LAYERS = [lambda k, v: (k[None], v), lambda k, v: (k, v[None]), lambda k, v: (k[None][:0], v[None][:0]), lambda k, v: (k.expand(2, -1, -1, -1, -1), v[None]),
          lambda k, v: (k[None, None], v[None, None])]
REFUSED = [(op, name, i) for op, by in CHANGES.items() for name, how in by.items() for i in range(len(how))]


def call(op, name, i, dev):
    from metal_native import paged

    kw = arguments(dev)[op]
    change = CHANGES[op][name][i]
    value = None if change is None else change(kw.get(name))
    kw[name] = value.to(dev) if isinstance(value, torch.Tensor) and value.device != dev and name in ("slopes", "prefix_lens") else value
    return getattr(paged, op)(**kw)


@pytest.fixture
def stand_in(monkeypatch):
    """CPU tensors stand in for the GPU's: no call gets past the checks."""
    from metal_native import MetalNativeError, paged

    def tensor(t, what, op):
        if not isinstance(t, torch.Tensor):
            raise MetalNativeError(f"{op}: {what} must be a torch.Tensor")

    monkeypatch.setattr(paged, "_require_cuda", tensor)


@pytest.mark.parametrize("op,name,i", [r for r in REFUSED if r[1] not in LIBRARY])
def test_refused_before_the_library(op, name, i, stand_in):
    from metal_native import MetalNativeError

    with pytest.raises(MetalNativeError, match=f"paged.{op}: "):
        call(op, name, i, torch.device("cpu"))


@pytest.mark.parametrize("how", LAYERS)
def test_layers_refused(how, stand_in):
    from metal_native import MetalNativeError, paged

    kw = arguments(torch.device("cpu"))["accept"]
    kw["k_cache"], kw["v_cache"] = how(kw["k_cache"], kw["v_cache"])
    with pytest.raises(MetalNativeError, match="paged.accept: "):
        paged.accept(**kw)


@pytest.mark.parametrize("op", list(CHANGES))
def test_cpu_tensors_are_refused(op):
    from metal_native import MetalNativeError, paged

    with pytest.raises(MetalNativeError, match="GPU tensor"):
        getattr(paged, op)(**arguments(torch.device("cpu"))[op])


@pytest.mark.gpu
@pytest.mark.parametrize("op", list(CHANGES))
def test_refused(gpu, op):
    from metal_native import MetalNativeError, paged

    getattr(paged, op)(**arguments(gpu)[op])
    for name, how in CHANGES[op].items():
        for i in range(len(how)):
            with pytest.raises(MetalNativeError):
                call(op, name, i, gpu)
    for name in [n for n, x in arguments(gpu)[op].items() if isinstance(x, torch.Tensor)]:
        with pytest.raises(MetalNativeError):   # one tensor on the host
            getattr(paged, op)(**{n: x.cpu() if n == name else x for n, x in arguments(gpu)[op].items()})
    if op == "accept":
        for how in LAYERS:
            kw = arguments(gpu)[op]
            kw["k_cache"], kw["v_cache"] = how(kw["k_cache"], kw["v_cache"])
            with pytest.raises(MetalNativeError):
                paged.accept(**kw)
        kw = arguments(gpu)[op]
        kw["k_cache"] = kw["k_cache"][:, :1].expand(-1, 2, -1, -1)   # heads that share memory
        with pytest.raises(MetalNativeError):
            paged.accept(**kw)
    getattr(paged, op)(**arguments(gpu)[op])


# ---- the C entries: pointers that no refused call follows ----
def c_call(op, cache=None, mask=None, **other):
    from metal_native import _lib

    L = _lib.load()
    c = Cache(**{**dict(k=P, v=P, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, pages=6, kv_heads=2,
                        page_size=16, head_dim=64, dtype=0, table=P, ld_table=3, width=3, batch=2, lens=P), **(cache or {})})
    m = Mask(**{**dict(scale=0.125, softcap=0.0, slopes=None, window=0, prefix_lens=None, cu_q=P, max_q=0), **(mask or {})})
    o = dict(q=P, q_token=512, q_head=64, rows=5, heads=8, out=P, lse=P, ws=None, ws_bytes=0, parents=P, cu=P, batch=2, words=1, tree=P,
             ld_tree=1, layers=1, k_layer=0, v_layer=0, drawn=P, drafted=P, steps=4, path=P, tokens=P, count=P, new_lens=P)
    assert set(other) <= set(o)
    o.update(other)
    names, first = {"ancestors": ("parents cu batch rows words tree", []),
                    "tree_attention": ("tree ld_tree words q q_token q_head rows heads out lse ws ws_bytes", [ctypes.byref(c), ctypes.byref(m)]),
                    "accept": ("layers k_layer v_layer drawn drafted parents cu rows steps path tokens count new_lens", [ctypes.byref(c)])}[op]
    rc = getattr(L, f"mq_paged_{op}")(*first, *[o[n] for n in names.split()], None)
    return rc, L.mq_last_error().decode()


C_REFUSED = [("ancestors", b) for b in (dict(parents=None), dict(tree=None), dict(tree=P + 4), dict(batch=0), dict(batch=BIG), dict(rows=-1),
                                        dict(rows=2**31 - 1), dict(words=0), dict(words=2**26), dict(cu=None))] + \
    [(op, dict(cache=b)) for op in ("tree_attention", "accept") for b in BAD_CACHE + BAD_V] + \
    [("tree_attention", dict(mask=b)) for b in BAD_MASK] + [("tree_attention", b) for b in BAD_QUERY] + \
    [("tree_attention", b) for b in (dict(out=None), dict(out=P + 8), dict(tree=None), dict(tree=P + 4), dict(words=0), dict(words=BIG), dict(ld_tree=-1))] + \
    [("accept", b) for b in (dict(layers=0), dict(layers=BIG), dict(k_layer=-8), dict(v_layer=-8), dict(k_layer=4), dict(v_layer=12), dict(drawn=None),
                             dict(drafted=None), dict(parents=None), dict(cu=None), dict(rows=-1), dict(rows=2**31), dict(steps=0), dict(steps=BIG),
                             dict(path=None), dict(tokens=None), dict(count=None), dict(new_lens=None))]


@pytest.mark.parametrize("op,how", C_REFUSED, ids=lambda x: x if isinstance(x, str) else str(x))
def test_c_entries_refuse(op, how):
    rc, text = c_call(op, **how)
    assert rc == 4 and text.startswith(f"paged.{op}: "), (rc, text)


def test_c_entries_of_null_structs_and_no_rows():
    from metal_native import _lib

    assert _lib.load().mq_paged_tree_attention_workspace_size(None, None, 1, 1) == -1
    assert c_call("tree_attention", rows=0, q=None, out=None)[0] == 0
    assert c_call("ancestors", rows=0, parents=None, tree=None)[0] == 0


def test_tree_plans():
    """(rows of a block, most parts): few trees behind many slots in blocks of 256 rows, many or short ones as chunks are."""
    from metal_native import _lib

    def plan(rows, heads, kv_heads, dim, batch, slots, window=0, softcap=0.0, op="tree_attention"):
        c = Cache(k=P, v=P, pages=1 << 20, kv_heads=kv_heads, page_size=16, head_dim=dim, dtype=0, table=P, ld_table=slots // 16, width=slots // 16,
                  batch=batch, lens=P, **{f"{t}_{n}": x for t in "kv" for n, x in (("page", kv_heads * 16 * dim), ("head", 16 * dim), ("slot", dim))})
        m = Mask(scale=0.1, softcap=softcap, slopes=None, window=window, prefix_lens=None, cu_q=P, max_q=0)
        block, parts = ctypes.c_int32(), ctypes.c_int32()
        assert getattr(_lib.load(), f"mq_paged_{op}_plan")(ctypes.byref(c), ctypes.byref(m), rows, heads, ctypes.byref(block), ctypes.byref(parts)) == 0
        return block.value, parts.value

    assert plan(5, 28, 4, 128, 1, 32768)[0] == 256 and 16 < plan(5, 28, 4, 128, 1, 32768)[1] <= 64
    assert plan(14, 14, 2, 64, 2, 16384)[0] == 256 and plan(14, 14, 2, 64, 2, 16384, op="attention")[0] == 32
    for other in (plan(4, 28, 4, 128, 1, 32768), plan(20, 28, 4, 128, 4, 8176), plan(100, 28, 4, 128, 9, 32768), plan(14, 14, 2, 64, 2, 16384, window=100),
                  plan(14, 14, 2, 64, 2, 16384, softcap=2.0)):   # a block of 32 holds the tree; short; many; a window; a cap
        assert other[0] == 32
    assert plan(4096, 28, 4, 128, 1, 32768) == plan(4096, 28, 4, 128, 1, 32768, op="attention")
    n = ctypes.c_int32()
    assert _lib.load().mq_paged_tree_attention_plan(None, None, 1, 1, ctypes.byref(n), ctypes.byref(n)) == 4


# ---- caches that share memory ----
@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_whether_arrays_share_an_element(tmp_path):
    """Against every element of both, for strides that nest, interleave, differ and overlap."""
    src = tmp_path / "share.cpp"
    src.write_text('''
#include <cstdio>
#include <random>
#include <set>
#include "mq_paged.hpp"
int main() {
  std::mt19937 rng(1);
  long bad = 0, shared = 0, apart_ones = 0;
  for (int turn = 0; turn < 60000; ++turn) {
    const int dims = 1 + rng() % 4;
    int64_t size[4], x[4], y[4];
    for (int64_t* s : {x, y}) {   // nested, in an order of its own, with gaps
      int order[4] = {0, 1, 2, 3};
      if (s == x) for (int d = 0; d < dims; ++d) size[d] = 1 + rng() % 4;
      if (s == x || turn % 3) for (int d = dims - 1; d > 0; --d) std::swap(order[d], order[rng() % (d + 1)]);
      int64_t step = 1;
      for (int d = 0; d < dims; ++d) {
        s[order[d]] = step;
        step *= size[order[d]] * (rng() % 3 ? 1 : 1 + rng() % 3);
      }
    }
    if (turn % 2) for (int d = 0; d < dims; ++d) y[d] = x[d];
    const int64_t apart = (int64_t)(rng() % 81) - 40;
    auto all = [&](const int64_t* s, int64_t from) {
      std::set<int64_t> r{from};
      for (int d = 0; d < dims; ++d) {
        std::set<int64_t> next;
        for (int64_t v : r) for (int64_t i = 0; i < size[d]; ++i) next.insert(v + i * s[d]);
        r = next;
      }
      return r;
    };
    bool want = false;
    const auto a = all(x, 0), b = all(y, apart);
    for (int64_t v : b) want |= a.count(v) != 0;
    (want ? shared : apart_ones)++;
    bad += mq::paged_share(dims, size, x, y, apart) != want;
  }
  // the largest there are: no overflow, and an end
  const int64_t huge[5] = {INT64_C(1) << 30, INT64_C(1) << 31, 65535, 65536, 128}, s[5] = {INT64_C(1) << 61, INT64_C(1) << 30, 8, 128, 1}, z[5] = {8, 8, 8, 136, 1};
  for (int64_t apart : {INT64_C(0), INT64_MAX / 2, INT64_MIN / 2, INT64_C(8)}) mq::paged_share(5, huge, s, z, apart), mq::paged_share(5, huge, s, s, apart);
  std::printf("bad %ld of %ld and %ld\\n", bad, shared, apart_ones);
  return shared < 10000 || apart_ones < 10000;
}
''')
    exe = tmp_path / "share"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                    f"-I{os.path.join(ROOT, 'metal-native_amd', 'csrc')}", str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env={k: v for k, v in os.environ.items() if k != "LD_PRELOAD"})
    assert out.returncode == 0 and "bad 0 " in out.stdout, out.stdout + out.stderr


# a page is 2 heads of 16 slots of 64 halves: 4096 bytes; 6 pages a layer, one layer after the other
@pytest.mark.parametrize("how", [dict(v=P), dict(v=P + 4096), dict(v=P + 5 * 4096), dict(v=P - 16), dict(v=P + 3 * 24576, layers=4), dict(v=P + 24576, layers=2),
                                 dict(v=P + 64, k_slot=128, v_slot=128, k_head=2048, v_head=2048, k_page=4096, v_page=4096)])
def test_keys_and_values_that_share_memory_are_refused(how):
    layers = how.get("layers", 1)
    rc, text = c_call("accept", cache={n: x for n, x in how.items() if n != "layers"}, layers=layers, k_layer=12288, v_layer=12288)
    assert rc == 4 and text == "paged.accept: keys and values must not share memory: a slot would be moved twice", (rc, text)


@pytest.mark.gpu
def test_layers_shifted_by_one_are_refused(gpu):
    from metal_native import MetalNativeError, paged

    kw = arguments(gpu)["accept"]
    both = kw["k_cache"].new_zeros(4, *kw["k_cache"].shape)
    wide = kw["k_cache"].new_zeros(2, 9, *kw["k_cache"].shape[1:])
    for k, v in ((both[:-1], both[1:]), (both[1:], both[:-1]), (wide[:, :6], wide[:, 3:])):
        with pytest.raises(MetalNativeError, match="share memory"):
            paged.accept(**{**kw, "k_cache": k, "v_cache": v})
    paged.accept(**{**kw, "k_cache": both[::2], "v_cache": both[1::2]})   # layers in turn


# ---- tangents of forward mode ----
def every(dev):
    return {**paged_arguments(dev), **arguments(dev)}


def with_tangent(kw, name):
    from torch.autograd import forward_ad

    return {**kw, name: forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))}


FLOATS = [(op, name) for op, kw in every(torch.device("cpu")).items() for name, x in kw.items()
          if isinstance(x, torch.Tensor) and x.is_floating_point()]


@pytest.mark.parametrize("op,name", FLOATS)
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(op, name, grad, stand_in):
    from torch.autograd import forward_ad

    from metal_native import MetalNativeError, paged

    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(MetalNativeError, match=f"paged.{op}: .*tangent"):
            getattr(paged, op)(**with_tangent(every(torch.device("cpu"))[op], name))


@pytest.mark.gpu
@pytest.mark.parametrize("op,name", FLOATS)
def test_a_tangent_is_not_lost(gpu, op, name):
    from torch.autograd import forward_ad

    from metal_native import MetalNativeError, paged

    kw = every(gpu)[op]
    for grad in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            with pytest.raises(MetalNativeError, match=f"paged.{op}: .*tangent"):
                getattr(paged, op)(**with_tangent(kw, name))
    getattr(paged, op)(**kw)
