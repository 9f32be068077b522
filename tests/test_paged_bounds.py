"""Paged-cache operators where values, masks or tables stand at their ends."""

import math
import os
import re
import shutil
import subprocess

import pytest
import torch

import paged_ref as ref
from test_paged import DT, build, check_attention

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_rows_of_a_block_of_slots(tmp_path):
    """Built with a host compiler from the kernels' own header, undefined behaviour and bounds trapped."""
    exe = tmp_path / "paged_rows_check"
    cmd = ["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
           f"-I{os.path.join(ROOT, 'metal-native_amd', 'csrc')}",
           os.path.join(ROOT, "tests", "native", "paged_rows_check.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env={k: v for k, v in os.environ.items() if k != "LD_PRELOAD"})
    assert out.returncode == 0 and "bad 0" in out.stdout, out.stdout + out.stderr


@pytest.mark.gpu
def test_mass_of_short_sequences_in_a_table_of_far_more_slots(gpu):
    """128 heads and a table of 2^24 + 128 slots: rows numbered by the table's slots would pass 32 bits."""
    from metal_native import paged

    H, D, ps, width = 128, 64, 128, (1 << 17) + 1
    g = torch.Generator(device=gpu)
    g.manual_seed(1)
    k, v = (torch.randn(8, 1, ps, D, device=gpu, generator=g).half() for _ in range(2))
    wide = torch.full((2, width), -1, dtype=torch.int32, device=gpu)
    wide[0, :3] = torch.tensor([5, 1, 7])
    wide[1, 0] = 2
    lens = torch.tensor([300, 9], dtype=torch.int32, device=gpu)
    for cu, rows in ((None, 2), (torch.tensor([0, 4, 9], dtype=torch.int32, device=gpu), 9)):
        q = torch.randn(rows, H, D, device=gpu, generator=g).half()
        near = wide[:, :3].contiguous()
        _, lse = paged.attention(q, k, v, near, lens, cu, return_lse=True)
        want = paged.attention_mass(q, k, near, lens, lse, cu)
        got = paged.attention_mass(q, k, wide, lens, lse, cu)
        assert got.shape == (2, 1, width * ps)
        # the far table's call may add the rows up in other parts: two sums of weights, each within 2 (r^1/2 + 40) e
        r = rows * H
        assert bool(((got[..., :3 * ps] - want).abs() <= want * 4 * (math.sqrt(r) + 40) * 2.0**-24).all())
        assert float(got[..., 3 * ps:].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("parts", [False, True])
def test_infinite_values_that_every_row_sees(gpu, dtype, D, parts):
    """Blocks of 256 rows, their slots in one part or several: an infinity in each tile of 64 slots, the first of a
    block and of a part among them, and both signs in one column."""
    H, KVH, lens, new = (14, 2, [3200, 40], [600, 40]) if parts else (32, 8, [900, 300], [512, 300])
    c = build(gpu, DT[dtype], H, KVH, D, 16, lens, new, seed=D)
    seen = (lens[0] - new[0]) // 64   # tiles that every row of the first sequence sees whole
    assert seen >= 6
    for t in range(seen):
        slot = 64 * t + 5 * t % 64
        c["v"][c["table"][0, slot // 16].long(), :, slot % 16, t] = float("inf") if t % 2 else -float("inf")
    last = c["table"][0, (64 * seen - 1) // 16].long()
    c["v"][last, :, 15, 1] = -float("inf")   # +inf stands in tile 1: NaN
    out, _, _ = check_attention(c)
    first = out[:new[0]].float()
    assert bool(first[..., 1].isnan().all()) and bool((first[..., 3:seen:2] == float("inf")).all())
    assert bool((first[..., 0:seen:2] == -float("inf")).all()) and bool(first[..., seen:].isfinite().all())


def test_refilled_buffers_have_been_read(tmp_path):
    """The few-row kernel fills a wave's key and value buffers again as soon as its products have read them: in its
    assembly no LDS read is outstanding where a load into LDS starts."""
    import importlib.util

    spec = importlib.util.spec_from_file_location("mq_build", os.path.join(ROOT, "metal-native_amd", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    try:
        hipcc = b._hipcc()
    except RuntimeError:
        pytest.skip("needs hipcc")
    src, asm = "mq_pattn.hip", tmp_path / "pattn.s"
    subprocess.run([hipcc, *b.HIP_FLAGS, *b.SOURCE_FLAGS[src], "-x", "hip", "-S", "--cuda-device-only", os.path.join(b.CSRC, src),
                    "-o", str(asm)], check=True, capture_output=True, timeout=600)
    loads, name, reads = {}, "", 0
    for line in asm.read_text().splitlines():
        label = re.match(r"(_Z\w+):", line)
        if label:
            name, reads = label.group(1), 0
        if "paged_split_kernel" not in name:
            continue
        line = line.strip()
        wait = re.search(r"s_waitcnt.*lgkmcnt\((\d+)\)", line)
        if line.startswith(("ds_", "s_load")):
            reads += 1
        elif wait:
            reads = min(reads, int(wait.group(1)))
        elif line.startswith("buffer_load_dwordx4") and line.endswith("lds"):
            loads[name] = loads.get(name, 0) + 1
            assert reads == 0, (name, line)
    assert len(loads) == 8 and min(loads.values()) >= 8, loads   # two types, two widths, with and without caps and biases


class Marked(torch.Tensor):
    pass


def step_of(gpu):
    """The four operators on inputs of their own: the same outputs each time."""
    from metal_native import paged

    def run(form=lambda t: t):
        c = build(gpu, torch.float16, 8, 2, 64, 16, [40, 100], [3, 1], seed=21, extra=12, junk=1.0)
        qkv = torch.randn(4, 12 * 64, device=gpu, generator=c["gen"]).half()
        ang = torch.rand(128, 64, device=gpu, generator=c["gen"])
        pos = torch.tensor([37, 38, 39, 99], device=gpu)
        k, v, table, lens, cu = (form(c[n]) for n in ("k", "v", "table", "lens", "cu"))
        q = paged.rope_kv(form(qkv), form(ang.cos()), form(ang.sin()), form(pos), k, v, table, lens, cu)
        slopes, prefix = form(torch.full((8,), 0.01, device=gpu)), form(torch.tensor([2, 0], dtype=torch.int32, device=gpu))
        how = dict(slopes=slopes, prefix_lens=prefix, window=50)
        out, lse = paged.attention(form(q), k, v, table, lens, cu, return_lse=True, **how)
        m = paged.attention_mass(form(q), k, table, lens, form(lse), cu, **how)
        to = form(c["free"][:4].reshape(2, 2).contiguous())
        return [torch.Tensor(x) if type(x) is Marked else x for x in
                (q, out, lse, m, *paged.evict(k, v, table, lens, form(m), to, 32, recent=4), k, v)]

    return run


@pytest.mark.gpu
def test_modes_and_tensor_subclasses_make_no_difference(gpu):
    """A default device is a function mode; profilers and counters are dispatch modes."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    run = step_of(gpu)
    want = run()

    def same(got):
        assert len(got) == len(want) and all(type(b) is torch.Tensor and torch.equal(a, b) for a, b in zip(want, got))

    for mode in (torch.device("cuda"), torch.device("cpu"), Function(), Dispatch(), torch.inference_mode(), torch.no_grad()):
        with mode:
            same(run())
    same(run(lambda t: t.as_subclass(Marked)))


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_serving_under_a_default_device(gpu, device):
    from metal_native.serving import PagedServer
    from test_serving import PROMPTS, model_of

    m = model_of(gpu)

    def run():
        server = PagedServer(m, 24, 4, chunk=24, budget=20, recent=6, slack=5)
        return [server.start(PROMPTS)] + [server.step() for _ in range(8)]

    want = run()
    with torch.device(device):
        assert run() == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("H,KVH,D", [(14, 2, 64), (28, 4, 128), (6, 6, 64)])
@pytest.mark.parametrize("lens,new,before,after", [
    ([40, 9, 100], [3, 0, 17], 0, 1), ([40, 9, 100], [3, 9, 1], 5, 70), ([40, 9], [0, 0], 0, 40), ([900, 700], [700, 600], 3, 600)])
def test_rows_of_no_chunk(gpu, dtype, H, KVH, D, lens, new, before, after):
    """Rows before the first chunk and past the last, as a batch padded for a graph has them: zeros and -inf, the others
    as without them.  The last case fills blocks of 256 rows."""
    from metal_native import paged

    c = build(gpu, DT[dtype], H, KVH, D, 16, lens, new, seed=before + after)
    rows = before + sum(new) + after
    q = torch.randn(rows, H, D, device=gpu, generator=c["gen"]).to(DT[dtype])
    q[before:before + sum(new)] = c["q"]
    for _ in range(2):   # what the outputs' memory held before
        junk = [torch.full((rows, H, D), float("nan"), dtype=DT[dtype], device=gpu), torch.full((rows, H), float("nan"), device=gpu)]
    del junk
    out, lse = paged.attention(q, c["k"], c["v"], c["table"], c["lens"], c["cu"] + before, return_lse=True)
    want, wl, ob, lb = ref.attention(q, c["k"], c["v"], c["table"], c["lens"], c["cu"] + before, scale=D**-0.5)
    unused = torch.ones(rows, dtype=torch.bool)
    unused[before:before + sum(new)] = False
    assert bool((out[unused.to(gpu)] == 0).all()) and bool((lse[unused.to(gpu)] == -float("inf")).all())
    assert bool(((out.double().cpu() - want).abs() <= ob).all())
    gl = lse.double().cpu()
    assert bool(((gl == wl) | ((gl - wl).abs() <= lb)).all())


@pytest.mark.parametrize("op", ["rope_kv", "evict"])
@pytest.mark.parametrize("name", ["k_cache", "v_cache"])
def test_written_caches_may_not_require_gradients(op, name, monkeypatch):
    from metal_native import MetalNativeError, paged
    from test_paged_host import arguments

    monkeypatch.setattr(paged, "_require_cuda", lambda *a: None)
    kw = arguments(torch.device("cpu"))[op]
    kw[name].requires_grad_()
    with pytest.raises(MetalNativeError, match="written in place"):
        getattr(paged, op)(**kw)


@pytest.mark.gpu
def test_gradients_are_refused_not_lost(gpu):
    from metal_native import MetalNativeError, paged
    from test_paged_host import arguments

    floats = {"rope_kv": ("qkv", "cos", "sin"), "attention": ("q", "k_cache", "v_cache", "slopes"),
              "attention_mass": ("q", "k_cache", "lse", "slopes"), "evict": ("mass",)}
    for op, names in floats.items():
        def call(**other):
            kw = arguments(gpu)[op]
            if "q" in kw:
                kw["q"] = torch.randn(kw["q"].shape, device=gpu, generator=torch.Generator(gpu).manual_seed(1)).half()
                kw["slopes"] = torch.full((kw["q"].shape[1],), 0.1, device=gpu)
            kw.update({n: form(kw[n]) for n, form in other.items()})
            r = getattr(paged, op)(**kw)
            return r if isinstance(r, tuple) else (r,)

        want = call()
        assert not any(x.requires_grad for x in want)
        for name in names:
            got = call(**{name: lambda t: t.detach().clone().requires_grad_()})
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(want, got))
            out = [x for x in got if x.is_floating_point()]
            assert all(x.requires_grad for x in out)
            for x in out:
                with pytest.raises(MetalNativeError, match=f"paged.{op}: has no backward pass"):
                    x.float().sum().backward()
            with torch.no_grad():
                assert not any(x.requires_grad for x in call(**{name: lambda t: t.detach().clone().requires_grad_()}))
        if op in ("rope_kv", "evict"):
            for name in ("k_cache", "v_cache"):
                with pytest.raises(MetalNativeError, match="written in place"):
                    call(**{name: lambda t: t.requires_grad_()})
                with torch.no_grad():
                    call(**{name: lambda t: t.requires_grad_()})


@pytest.mark.gpu
def test_autograd_sees_that_caches_were_written(gpu):
    """A product that saved a cache for its own gradient notices the write; caches of inference mode have no counter."""
    from metal_native import paged
    from test_paged_host import arguments

    for op, other in (("rope_kv", {}), ("evict", {})):
        kw = arguments(gpu)[op]
        w = torch.ones((), device=gpu, dtype=torch.float16, requires_grad=True)
        before = (kw["k_cache"]._version, kw["v_cache"]._version)
        y = (kw["k_cache"] * w).sum()
        getattr(paged, op)(**kw)
        assert kw["k_cache"]._version > before[0] and kw["v_cache"]._version > before[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():
            kw = arguments(gpu)[op]
        getattr(paged, op)(**kw)
    for op in ("attention", "attention_mass"):   # only read
        kw = arguments(gpu)[op]
        getattr(paged, op)(**kw)
        assert kw["k_cache"]._version == 0


@pytest.mark.gpu
@pytest.mark.parametrize("flag", [True, 1, "yes", False, 0, None])
def test_return_lse_is_a_truth_value(gpu, flag):
    from metal_native import paged
    from test_paged_host import arguments

    r = paged.attention(**arguments(gpu)["attention"], return_lse=flag)
    assert (isinstance(r, tuple) and len(r) == 2) if flag else isinstance(r, torch.Tensor)


def test_sections_that_are_not_whole_numbers(monkeypatch):
    from metal_native import MetalNativeError, paged
    from test_paged_host import arguments

    monkeypatch.setattr(paged, "_require_cuda", lambda *a: None)
    kw = arguments(torch.device("cpu"))["rope_kv"]
    kw["pos"] = kw["pos"].expand(2, -1)
    for sections in ((16.5, 15.5), [16.5, 16.5]):
        with pytest.raises(MetalNativeError, match="whole numbers"):
            paged.rope_kv(**{**kw, "sections": sections})


@pytest.mark.gpu
def test_sections_of_any_integer_type(gpu):
    import numpy as np

    from metal_native import paged
    from test_paged_host import arguments

    for sections in ((20, 12), [20, 12], (np.int64(20), np.int32(12)), np.array([20, 12]), torch.tensor([20, 12]), (20.0, 12)):
        kw = arguments(gpu)["rope_kv"]
        kw["pos"] = kw["pos"].expand(2, -1).contiguous()
        assert paged.rope_kv(**{**kw, "sections": sections}).shape == (5, 8, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("cap", [1e-40, 0.5, 8.0, 50.0, 1e4, 1e6, 3e38])
def test_caps_of_every_size(gpu, cap, many):
    """A cap far above the scores leaves them as they are.  Bounds: with S = scale max sum |q k| and X the largest score
    in size, dx = (D + 4) e S + 32 e X + 4 e X (a product of D terms; the cap, 22 e at most; units of log 2): a weight is
    off by 2 dx of itself, by u where it is rounded, an output by u again; the log sum by dx + (n + 8) e + 2 e of itself."""
    from metal_native import paged

    H, KVH, D, ps = 14, 2, 64, 16
    lens, new = ([2000, 40, 1700], [1100, 40, 900]) if many else ([300, 1, 77, 130], [1, 1, 20, 130])
    c = build(gpu, torch.float16, H, KVH, D, ps, lens, new, seed=3, amp=1.5)
    cap = float(torch.tensor(cap, dtype=torch.float32))
    how = dict(scale=0.2, softcap=cap)
    out, lse = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True, **how)
    m = paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], lse, c["cu"], **how)
    E, n = ref.E, max(lens)
    at = torch.zeros(3 if many else 4, KVH, c["table"].shape[1] * ps, dtype=torch.float64)
    for s in range(len(lens)):
        for kv in range(KVH):
            x, _, see, (start, n_new, total) = ref.seq_scores(c["q"], c["k"], c["table"], c["lens"], c["cu"], s, kv, **how)
            plain, _, _, _ = ref.seq_scores(c["q"], c["k"], c["table"], c["lens"], c["cu"], s, kv, scale=0.2)
            kk, _ = ref.gather(c["k"], c["table"][s], total, kv)
            vv, _ = ref.gather(c["v"], c["table"][s], total, kv)
            qq = c["q"][start:start + n_new, 7 * kv:7 * kv + 7].double().cpu()
            S = 0.2 * float(torch.matmul(qq.abs(), kk.abs().t()).max())
            X = float(torch.where(see, plain, torch.zeros_like(plain)).abs().max())
            dx = (D + 4) * E * S + 36 * E * X
            l = torch.logsumexp(x, -1)
            w = torch.exp(x - l[..., None])
            o = torch.matmul(w, vv)
            a = torch.matmul(w, vv.abs())
            u = ref.half_step(torch.float16)
            ob = u * (a + o.abs()) + (2 * dx + 2 * (total + 8) * E) * a + total * 2.0**-32 * float(vv.abs().max()) + 2.0**-25
            rows, hs = slice(start, start + n_new), slice(7 * kv, 7 * kv + 7)
            err = (out[rows, hs].double().cpu().transpose(0, 1) - o).abs()
            assert bool((err <= ob).all()), float((err / ob).max())
            err, lb = (lse[rows, hs].double().cpu().t() - l).abs(), dx + (total + 8) * E + 2 * E * l.abs()
            assert bool((err <= lb).all()), float((err / lb).max())
            # the mass against the log sums that the call was given: dx + 4 e (1 + |lse|) a weight, and the sums
            given = lse[rows, hs].double().cpu().t()
            t = torch.where(see, torch.exp(x - given[..., None]), torch.zeros_like(x)).sum((0, 1))
            at[s, kv, :total] = t
            mb = t * (dx + (4 * (1 + float(given.abs().max())) + 4 * (n_new * 7) ** 0.5 + 80) * E) + 2.0**-120
            err = (m[s, kv, :total].double().cpu() - t).abs()
            assert bool((err <= mb).all()), float((err / mb).max())
    assert float(m.double().cpu().sub(at).abs().max()) < 1   # and nothing past the sequences


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_mass_of_infinite_keys_and_rows_left_out(gpu, dtype, chunk, cap):
    """A key of -inf under positive queries has no weight, also where a block of rows is not full; rows whose log sum is
    -inf add nothing, whatever their queries hold."""
    from metal_native import paged

    lens, new = [300, 70, 200], ([40, 1, 130] if chunk else None)
    c = build(gpu, DT[dtype], 8, 2, 64, 16, lens, new, seed=5)
    c["q"][..., 3] = c["q"][..., 3].abs() + 0.5
    for s, slot in ((0, 17), (0, 150), (1, 69), (2, 0)):
        c["k"][c["table"][s, slot // 16].long(), :, slot % 16, 3] = -float("inf")
    how = dict(softcap=cap)
    if not cap:   # with a cap an infinite score is a weight like others
        _, lse, scale = check_attention(c)
        got = paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], lse, c["cu"], scale=scale)
        want, bound = ref.mass(c["q"], c["k"], c["table"], c["lens"], lse, c["cu"], scale=scale)
        assert bool(((got.double().cpu() - want).abs() <= bound).all())
        assert float(got[0, :, 17].abs().max()) == 0 and float(got[1, :, 69].abs().max()) == 0
    c = build(gpu, DT[dtype], 8, 2, 64, 16, lens, new, seed=6)
    _, lse = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True, **how)
    out = torch.rand(lse.shape, device=gpu, generator=c["gen"]) < 0.3
    want = paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], lse.masked_fill(out, -float("inf")), c["cu"], **how)
    for junk in (float("nan"), float("inf")):
        q = c["q"].masked_fill(out[..., None], junk)
        assert torch.equal(want, paged.attention_mass(q, c["k"], c["table"], c["lens"], lse.masked_fill(out, -float("inf")), c["cu"], **how))


@pytest.mark.parametrize("op", ["attention", "attention_mass"])
def test_a_window_past_the_table_is_no_window(op):
    """The same plan (its workspace) as without one, up to the largest number."""
    import ctypes

    from metal_native import _lib
    from test_paged_host import Cache, Mask

    size = getattr(_lib.load(), f"mq_paged_{op}_workspace_size")
    for rows, width in ((4096, 512), (64, 512), (512, 512), (1, 4096)):
        c = Cache(k=4096, v=4096, k_page=8192, k_head=2048, k_slot=128, v_page=8192, v_head=2048, v_slot=128, pages=600, kv_heads=4,
                  page_size=16, head_dim=128, dtype=0, table=4096, ld_table=width, width=width, batch=1, lens=4096)

        def need(window):
            m = Mask(scale=0.1, softcap=0.0, slopes=None, window=window, prefix_lens=None, cu_q=4096, max_q=rows)
            return size(ctypes.byref(c), ctypes.byref(m), rows, 28)

        want = need(0)
        assert want >= 0
        for window in (width * 16, width * 16 + 1, 2**31 - 257, 2**31 - 1, 2**31, 2**62):
            assert need(window) == want, window


@pytest.mark.gpu
@pytest.mark.parametrize("window", [800, 2**31 - 1, 2**40])
def test_windows_past_the_table(gpu, window):
    from metal_native import paged

    c = build(gpu, torch.float16, 28, 4, 128, 16, [790, 40, 513], [300, 40, 1], seed=9)
    a, la = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], return_lse=True)
    b, lb = paged.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], window=window, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    assert torch.equal(paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], la, c["cu"]),
                       paged.attention_mass(c["q"], c["k"], c["table"], c["lens"], la, c["cu"], window=window))


@pytest.mark.gpu
@pytest.mark.parametrize("budget", [None, 20])
def test_serving_asks_for_log_sums_only_where_it_cuts(gpu, monkeypatch, budget):
    from metal_native import paged
    from metal_native.serving import PagedServer
    from test_serving import PROMPTS, model_of

    asked, attention = [], paged.attention
    monkeypatch.setattr(paged, "attention", lambda *a, **how: asked.append(bool(how.get("return_lse"))) or attention(*a, **how))
    server = PagedServer(model_of(gpu), 24, 4, chunk=24, **({} if budget is None else dict(budget=budget, recent=6, slack=5)))
    server.start(PROMPTS)
    server.step()
    assert set(asked) == {budget is not None}
