"""Paged-cache operators on the host: addressing arithmetic, refused arguments."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_addressing(tmp_path):
    """Built with a host compiler from the kernels' own header, undefined behaviour and bounds trapped."""
    exe = tmp_path / "paged_check"
    cmd = ["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
           f"-I{os.path.join(ROOT, 'metal-native_amd', 'csrc')}",
           os.path.join(ROOT, "tests", "native", "paged_check.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env={k: v for k, v in os.environ.items() if k != "LD_PRELOAD"})
    assert out.returncode == 0 and "bad 0" in out.stdout, out.stdout + out.stderr


H, KVH, D, PS, PAGES, B, W, ROWS = 8, 2, 64, 16, 6, 2, 3, 5


def arguments(dev):
    """Keyword arguments that each operator takes."""
    h = dict(dtype=torch.float16, device=dev)
    i = dict(dtype=torch.int32, device=dev)
    cache = dict(k_cache=torch.zeros(PAGES, KVH, PS, D, **h), v_cache=torch.zeros(PAGES, KVH, PS, D, **h),
                 table=torch.arange(6, **i).view(B, W), lens=torch.tensor([9, 30], **i))
    cu = torch.tensor([0, 2, 5], **i)
    cos = torch.ones(50, D, device=dev)
    q = torch.zeros(ROWS, H, D, **h)
    keys = {k: x for k, x in cache.items() if k != "v_cache"}
    return {
        "rope_kv": dict(cache, qkv=torch.zeros(ROWS, (H + 2 * KVH) * D, **h), cos=cos, sin=cos.clone(),
                        pos=torch.zeros(ROWS, dtype=torch.int64, device=dev), cu=cu, sections=None),
        "attention": dict(cache, q=q, cu=cu),
        "attention_mass": dict(keys, q=q, lse=torch.zeros(ROWS, H, device=dev), cu=cu),
        "evict": dict(cache, mass=torch.zeros(B, KVH, W * PS, device=dev), to=torch.tensor([[0], [1]], **i), budget=8, recent=2),
    }


CACHE = {
    "k_cache": [None, lambda x: x.float(), lambda x: x[0], lambda x: x[..., :48], lambda x: x[:, :, :12], lambda x: x[:, :, :4],
                lambda x: x[:0], lambda x: x.transpose(2, 3)],
    "table": [None, lambda x: x.long(), lambda x: x[0], lambda x: x[:, :0]],
    "lens": [None, lambda x: x.long(), lambda x: x[:1], lambda x: x[None]],
}
V = {"v_cache": [None, lambda x: x.bfloat16(), lambda x: x[:-1], lambda x: x.transpose(2, 3)]}
CU = {"cu": [None, lambda x: x[:2], lambda x: x.long()]}
MASK = dict(q=[None, lambda x: x.bfloat16(), lambda x: x[:, :7], lambda x: x[:, :, :32], lambda x: x[0]],
            slopes=[lambda _: torch.zeros(H - 1), lambda _: torch.zeros(H, dtype=torch.float64), lambda _: 1.0],
            prefix_lens=[lambda _: torch.zeros(B + 1, dtype=torch.int32), lambda _: torch.zeros(B, dtype=torch.int64)],
            scale=[lambda _: 0.0, lambda _: -1.0, lambda _: float("nan"), lambda _: float("inf")],
            softcap=[lambda _: -1.0, lambda _: float("inf"), lambda _: float("nan")], window=[lambda _: -1])
CHANGES = {
    "rope_kv": {**CACHE, **V, **CU,
                "qkv": [None, lambda x: x.bfloat16(), lambda x: x[:, :-8], lambda x: x[:, :4 * D], lambda x: x[:, :-D], lambda x: x[0]],
                "cos": [None, lambda x: x.half(), lambda x: x[:, :32], lambda x: x[:0], lambda x: x[:40]],
                "sin": [None, lambda x: x.double()],
                "pos": [None, lambda x: x.int(), lambda x: x[:-1], lambda x: x[None].expand(2, -1)],
                "sections": [lambda _: (), lambda _: (32, 0), lambda _: (16,), lambda _: (40, -8), lambda _: (4,) * 9]},
    "attention": {**CACHE, **V, **CU, **MASK},
    "attention_mass": {**CACHE, **CU, **MASK, "lse": [None, lambda x: x.half(), lambda x: x[:, :4], lambda x: x[:-1]]},
    "evict": {**CACHE, **V, "mass": [None, lambda x: x.half(), lambda x: x[..., :-1], lambda x: x[:1]],
              "to": [None, lambda x: x.long(), lambda x: x[:1], lambda x: x[0], lambda x: x[:, :0]],
              "budget": [lambda _: 0, lambda _: -3, lambda _: 17], "recent": [lambda _: -1, lambda _: 9]},
}
REFUSED = [(op, name, i) for op, by in CHANGES.items() for name, how in by.items() for i in range(len(how))]
LIBRARY = ("scale", "softcap", "window")   # refused by the library's entry, not before it


def call(op, name, i, dev):
    from metal_native import paged

    kw = arguments(dev)[op]
    change = CHANGES[op][name][i]
    value = None if change is None else change(kw.get(name))
    kw[name] = value.to(dev) if isinstance(value, torch.Tensor) and value.device != dev and name in ("slopes", "prefix_lens") else value
    return getattr(paged, op)(**kw)


@pytest.mark.parametrize("op,name,i", [r for r in REFUSED if r[1] not in LIBRARY])
def test_refused_before_the_library(op, name, i, monkeypatch):
    """The checks' own answers: CPU tensors stand in for the GPU's, and no call gets past the checks."""
    from metal_native import MetalNativeError, paged

    def tensor(t, what, op):
        if not isinstance(t, torch.Tensor):
            raise MetalNativeError(f"{op}: {what} must be a torch.Tensor")

    monkeypatch.setattr(paged, "_require_cuda", tensor)
    with pytest.raises(MetalNativeError, match=f"paged.{op}: "):
        call(op, name, i, torch.device("cpu"))


@pytest.mark.parametrize("op", list(CHANGES))
def test_cpu_tensors_are_refused(op):
    from metal_native import MetalNativeError, paged

    with pytest.raises(MetalNativeError, match="GPU tensor"):
        getattr(paged, op)(**arguments(torch.device("cpu"))[op])


@pytest.mark.gpu
@pytest.mark.parametrize("op", list(CHANGES))
def test_refused(gpu, op):
    """Every change through the public entry, and the unchanged call between them."""
    from metal_native import MetalNativeError, paged

    getattr(paged, op)(**arguments(gpu)[op])
    for name, how in CHANGES[op].items():
        for i in range(len(how)):
            with pytest.raises(MetalNativeError):
                call(op, name, i, gpu)
    for name in [n for n, x in arguments(gpu)[op].items() if isinstance(x, torch.Tensor)]:
        with pytest.raises(MetalNativeError):   # one tensor on the host
            getattr(paged, op)(**{n: x.cpu() if n == name else x for n, x in arguments(gpu)[op].items()})
    kw = arguments(gpu)[op]
    if op in ("rope_kv", "evict"):   # written: heads that share memory are refused
        kw["k_cache"] = kw["k_cache"][:, :1].expand(-1, KVH, -1, -1)
        with pytest.raises(MetalNativeError):
            getattr(paged, op)(**kw)
    getattr(paged, op)(**arguments(gpu)[op])


# ---- the C entries: pointers that no refused call follows ----
class Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + \
        [(n, ctypes.c_int64) for n in ("k_page", "k_head", "k_slot", "v_page", "v_head", "v_slot", "pages")] + \
        [(n, ctypes.c_int32) for n in ("kv_heads", "page_size", "head_dim", "dtype")] + \
        [("table", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("ld_table", "width", "batch")] + [("lens", ctypes.c_void_p)]


class Mask(ctypes.Structure):
    _fields_ = [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("slopes", ctypes.c_void_p), ("window", ctypes.c_int64),
                ("prefix_lens", ctypes.c_void_p), ("cu_q", ctypes.c_void_p), ("max_q", ctypes.c_int64)]


P = 4096   # never followed


def c_call(op, cache=None, mask=None, **other):
    from metal_native import _lib

    L = _lib.load()
    c = Cache(**{**dict(k=P, v=P, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024, v_slot=64, pages=6, kv_heads=2,
                        page_size=16, head_dim=64, dtype=0, table=P, ld_table=3, width=3, batch=2, lens=P), **(cache or {})})
    m = Mask(**{**dict(scale=0.125, softcap=0.0, slopes=None, window=0, prefix_lens=None, cu_q=P, max_q=0), **(mask or {})})
    sections = other.pop("sections", None)
    o = dict(q=P, q_token=512, q_head=64, rows=5, heads=8, out=P, lse=P, ws=None, ws_bytes=0, qkv=P, ld_qkv=768, cos=P, ld_cos=64,
             sin=P, ld_sin=64, table_rows=50, pos=P, ld_pos=5, axes=1, cu=P, mass=P, mass_b=96, mass_h=48, to=P, ld_to=1, to_width=1,
             budget=8, recent=2, kept=P, new_lens=P, left=P)
    assert set(other) <= set(o)
    o.update(other)
    sec = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    names = {"rope_kv": ("qkv ld_qkv cos ld_cos sin ld_sin table_rows pos ld_pos axes", sec, "cu rows heads out"),
             "attention": ("", ctypes.byref(m), "q q_token q_head rows heads out lse ws ws_bytes"),
             "attention_mass": ("", ctypes.byref(m), "q q_token q_head rows heads lse mass ws ws_bytes"),
             "evict": ("mass mass_b mass_h to ld_to to_width budget recent kept new_lens left", 0, "")}[op]
    args = [ctypes.byref(c)] + [o[n] for n in names[0].split()] + ([] if names[1] == 0 else [names[1]]) + \
        [o[n] for n in names[2].split()] + [None]
    rc = getattr(L, f"mq_paged_{op}")(*args)
    return rc, L.mq_last_error().decode()


BIG = 2**62
BAD_CACHE = [dict(k=None), dict(table=None), dict(lens=None), dict(head_dim=96), dict(dtype=2), dict(page_size=4),
             dict(page_size=24), dict(page_size=1 << 17), dict(kv_heads=0), dict(kv_heads=65536), dict(pages=0), dict(pages=2**31),
             dict(batch=0), dict(batch=65536), dict(width=0), dict(width=2**27), dict(width=BIG), dict(ld_table=2), dict(ld_table=-3),
             dict(ld_table=-1, width=1), dict(k=P + 8), dict(k_page=2044), dict(k_head=-1024), dict(k_slot=56), dict(k_slot=60),
             dict(k_slot=2**27), dict(k_page=2**31), dict(k_page=-2048), dict(k_slot=2**16 + 64, page_size=65536)]
BAD_V = [dict(v=None), dict(v=P + 2), dict(v_slot=0), dict(v_page=BIG), dict(v_head=4)]
BAD_MASK = [dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(window=-1), dict(cu_q=None)]
BAD_QUERY = [dict(q=None), dict(q=P + 8), dict(q_token=-8), dict(q_token=60), dict(q_token=2**40), dict(q_head=2**40), dict(q_token=BIG), dict(q_head=BIG), dict(q_head=4),
             dict(rows=-1), dict(heads=0), dict(heads=7), dict(rows=2**28), dict(rows=BIG)]
C_REFUSED = [(op, dict(cache=b)) for op in CHANGES for b in BAD_CACHE + ([] if op == "attention_mass" else BAD_V)] + \
    [(op, dict(mask=b)) for op in ("attention", "attention_mass") for b in BAD_MASK] + \
    [(op, b) for op in ("attention", "attention_mass") for b in BAD_QUERY] + \
    [("attention", dict(out=None)), ("attention", dict(out=P + 8)), ("attention_mass", dict(lse=None)), ("attention_mass", dict(mass=None))] + \
    [("rope_kv", b) for b in (
        dict(qkv=None), dict(cos=None), dict(sin=None), dict(pos=None), dict(out=None), dict(qkv=P + 8), dict(ld_qkv=760),
        dict(ld_qkv=772), dict(cos=P + 4), dict(ld_cos=62), dict(ld_sin=-64), dict(table_rows=0), dict(axes=0), dict(axes=9),
        dict(axes=2), dict(axes=2, sections=[16, 16], ld_pos=-5), dict(axes=2, sections=[16, 8]), dict(axes=2, sections=[40, -8]),
        dict(sections=[31]), dict(cu=None), dict(heads=0), dict(heads=3), dict(rows=-1), dict(rows=2**31), dict(heads=2**31 - 2))] + \
    [("evict", b) for b in (
        dict(mass=None), dict(to=None), dict(kept=None), dict(new_lens=None), dict(left=None), dict(budget=0), dict(budget=17),
        dict(budget=BIG), dict(recent=-1), dict(recent=9), dict(to_width=0), dict(to_width=BIG), dict(mass_b=-1), dict(mass_h=-1),
        dict(ld_to=0))]


@pytest.mark.parametrize("op,how", C_REFUSED, ids=lambda x: x if isinstance(x, str) else str(x))
def test_c_entries_refuse(op, how):
    rc, text = c_call(op, **how)
    assert rc == 4 and text.startswith(f"paged.{op}: "), (rc, text)


def test_c_entries_of_null_structs_and_no_rows():
    from metal_native import _lib

    L = _lib.load()
    assert L.mq_paged_attention_workspace_size(None, None, 1, 1) == -1
    assert L.mq_paged_attention_mass_workspace_size(None, None, 1, 1) == -1
    assert c_call("attention", rows=0, q=None, out=None)[0] == 0
    assert c_call("rope_kv", rows=0)[0] == 0
