"""Drawing tokens against the definition in 64 bits, row by row."""

import math

import numpy as np
import pytest
import torch

import draft_ref as ref

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# (temperature, top_k, top_p, min_p)
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.5, 0.0), (0.8, 0, 0.95, 0.02), (1.0, 1, 1.0, 0.0), (2.5, 7, 1.0, 0.3),
            (0.0, 5, 0.2, 0.0), (1.0, 3000, 0.999, 0.0), (0.3, 0, 1.0, 1e-4)]


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One setting, or a list with one for each row."""
    from metal_native import sampling

    rows, V = x.shape
    each = lambda v: list(v) if isinstance(v, (list, tuple)) else [v] * rows  # noqa: E731
    dev = x.device
    give = lambda v, t: torch.tensor(v, dtype=t, device=dev) if isinstance(v, (list, tuple)) else v  # noqa: E731
    how = dict(temperature=give(temperature, torch.float32), top_k=give(top_k, torch.int32), top_p=give(top_p, torch.float32),
               min_p=give(min_p, torch.float32))
    token, log = sampling.sample(x, u, return_logprob=True, **how)
    assert token.dtype == torch.int64 and log.dtype == torch.float32
    assert torch.equal(token, sampling.sample(x, u, **how))
    got, logs, xs, us = token.tolist(), log.double().tolist(), x.double().cpu().numpy(), u.cpu().tolist()
    # a weight is a multiple of 2^-44 or less (V <= 2^18) and the sum at least 1; then the rounding to fp32
    for r, (t, k, p, m) in enumerate(zip(each(temperature), each(top_k), each(top_p), each(min_p))):
        want, share = ref.sample(xs[r], us[r], t, k, p, m)
        assert got[r] == want, (r, V, t, k, p, m, got[r], want)
        if math.isfinite(share):
            assert abs(logs[r] - share) <= abs(share) * 2.0**-23 + V * 2.0**-44 + 2.0**-40, (r, logs[r], share)
        else:
            assert logs[r] == share
    return token


def logits(gpu, rows, V, dtype, seed, spread=2.0):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    x = torch.randn(rows, V, device=gpu, generator=g) * spread
    x[:, :: max(1, V // 5)] += 3 * spread * torch.rand(rows, len(range(0, V, max(1, V // 5))), device=gpu, generator=g)
    return x.to(DT[dtype]), torch.rand(rows, device=gpu, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [1, 2, 7, 64, 65, 1000, 2049, 8193, 32003, 152064])
def test_settings(gpu, dtype, V):
    x, u = logits(gpu, len(SETTINGS), V, dtype, V)
    for s in SETTINGS:
        check(x, u, *s)
    check(x, u, *(list(c) for c in zip(*SETTINGS)))   # one for each row


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40, 300])
@pytest.mark.parametrize("spread", [0.0, 0.3, 8.0])
def test_rows_and_spreads(gpu, rows, spread):
    x, u = logits(gpu, rows, 5003, "bf16", rows, spread)
    check(x, u, 0.9, 0, 0.9, 0.0)
    check(x, u, 0.9, 0, 1.0, 0.0)
    check(x, u, 0.9, 400, 0.97, 1e-3)
    one = check(x[rows // 2:rows // 2 + 1], u[rows // 2:rows // 2 + 1], 0.9, 400, 0.97, 1e-3)
    assert int(one) == int(check(x, u, 0.9, 400, 0.97, 1e-3)[rows // 2])   # whatever else is in the batch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [12, 3001, 40000])
def test_ties_are_cut_by_index(gpu, dtype, V):
    """Three values only, so every cut falls among thousands of equal tokens; one value only."""
    g = torch.Generator(device=gpu)
    g.manual_seed(V)
    x = torch.randint(0, 3, (6, V), device=gpu, generator=g).to(DT[dtype])
    x[5] = 1.0
    x[4, ::2] = -0.0
    x[4, 1::2] = 0.0
    u = torch.tensor([0.0, 0.3, 0.999999, 0.5, 0.71, 0.25], device=gpu)
    for k in (0, 1, 2, V // 7 + 1, V // 2, V - 1, V, V + 5):
        for p in (1.0, 0.5, 0.01, 0.25):
            check(x, u, 1.0, k, p, 0.0)
    check(x, u, 1.0, 0, 1.0, 0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [9, 700, 20011])
def test_masks_infinities_and_nan(gpu, dtype, V):
    low = torch.finfo(DT[dtype]).min
    x, _ = logits(gpu, 12, V, dtype, V)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :V - 1] = -math.inf          # one token alone
    x[3] = low                        # masked by the type's lowest value, all of them
    x[4, 1:] = low
    x[5, ::3] = math.nan
    x[6, ::3] = math.inf              # several infinite ones share the weight
    x[7, ::2], x[7, 1::2] = math.nan, -math.inf
    x[8, V // 2] = math.inf
    x[9] = math.inf
    x[10, 2:] = -math.inf
    x[11, ::2] = -math.inf
    for u in (0.0, 0.4, 0.9999):
        us = torch.full((12,), u, device=gpu)
        for s in SETTINGS:
            check(x, us, *s)


@pytest.mark.gpu
def test_settings_at_their_ends(gpu):
    inf, nan = math.inf, math.nan
    x, u = logits(gpu, 1, 3000, "fp16", 3)
    ends = [(t, k, p, m) for t in (1e-4, 1e30, inf, -1.0, nan, 1.0) for k, p, m in
            ((0, 1.0, 0.0), (-7, 2.0, -1.0), (2**31 - 1, 0.0, 0.0), (10, -0.5, 0.0), (0, nan, nan), (5, 0.9, 1.0), (0, 1.0, 2.0), (0, 1e-30, 0.0))]
    n = len(ends)
    check(x.expand(n, -1), u.expand(n).contiguous(), *(list(c) for c in zip(*ends)))
    for end in ends:
        check(x, u, *end)
    us = torch.tensor([0.0, -0.0, -3.0, 1.0, 7.5, inf, -inf, nan, 1 - 2.0**-24, 1e-38, 2.0**-140], device=gpu)
    for s in SETTINGS:
        check(x.expand(len(us), -1), us, *s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [("fp16", 2**18), ("bf16", 2**18 + 1), ("fp32", 2**18 + 1027), ("bf16", 2**20 + 3), ("fp32", 2**22)])
def test_large_vocabularies(gpu, dtype, V):
    """A row's parts grow past 2^18 tokens in more than one workgroup's; 2^22 is the most."""
    x, u = logits(gpu, 2, V, dtype, V, 1.0)
    for s in ((0.9, 0, 0.9, 0.0), (1.1, 300, 1.0, 0.0), (1.0, 5000, 0.99, 0.0), (1.5, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.01)):
        check(x, u, *s)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [5, 700])
def test_many_rows(gpu, V):
    """More than a thousand rows go in several turns, settings of each row with them."""
    x, u = logits(gpu, 2051, V, "fp16", V)
    check(x, u, 0.9, 0, 0.9, 0.0)
    every = [SETTINGS[r % len(SETTINGS)] for r in range(2051)]
    check(x, u, *(list(c) for c in zip(*every)))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [63, 64, 65, 511, 512, 513, 1024, 1025])
def test_borders_of_the_short_lists(gpu, k):
    """Around the lengths at which lists change their place and way; nearly equal and many equal logits among them."""
    for dtype, spread in (("bf16", 0.05), ("fp32", 1e-5), ("fp16", 3.0)):
        x, u = logits(gpu, 3, 20000, dtype, k, spread)
        for p, m in ((1.0, 0.0), (0.9, 0.0), (0.5, 1e-3)):
            check(x, u, 0.8, k, p, m)
            check(x, u, [0.8] * 3, [k, k, 1], [p] * 3, [m] * 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_strides_and_alignment(gpu, dtype):
    wide, _ = logits(gpu, 8, 6007, dtype, 1)
    u = torch.rand(8, device=gpu)
    for a, b in ((0, 6007), (1, 6007), (2, 6000), (3, 5000), (5, 4101), (7, 8)):
        check(wide[:, a:b], u, 0.8, 0, 0.9, 0.0)
    check(wide[::2], u[:4], 0.8, 30, 1.0, 0.0)
    check(wide[:4].t()[:4].t(), u[:4], 0.8, 0, 0.9, 0.0)
    check(wide.t().contiguous().t(), u, 0.8, 0, 0.9, 0.0)      # copied
    check(wide[3:4].expand(8, -1), u, 1.0, 0, 1.0, 0.0)
    check(wide, torch.rand(16, device=gpu)[::2], 1.0, 0, 1.0, 0.0)


@pytest.mark.gpu
def test_every_share_of_the_unit_interval(gpu):
    """4096 evenly spaced numbers: each token as often as its part of the sum holds such numbers."""
    x, _ = logits(gpu, 1, 300, "fp32", 8)
    u = (torch.arange(4096, device=gpu) + 0.5) / 4096
    for s in ((1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0)):
        check(x.expand(4096, -1), u, *s)


@pytest.mark.gpu
def test_captured_and_on_other_streams(gpu):
    """Replayed with new inputs between eager calls, two graphs in turn, and eager calls on two streams at once."""
    from metal_native import sampling

    shapes = [(5, 40000, dict(temperature=0.8, top_p=0.9)), (70, 3000, dict(top_k=20, min_p=0.01))]
    held, graphs = [], []
    for i, (rows, V, how) in enumerate(shapes):
        x, u = logits(gpu, rows, V, "fp16", i)
        sampling.sample(x, u, **how)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = sampling.sample(x, u, return_logprob=True, **how)
        held.append((x, u, how, out))
        graphs.append(g)
    for turn in range(4):
        for (x, u, how, out), g in zip(held, graphs):
            nx, nu = logits(gpu, *x.shape, "fp16", 10 + turn)
            x.copy_(nx)
            u.copy_(nu)
            g.replay()
            want = sampling.sample(x, u, return_logprob=True, **how)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(gpu) for _ in range(2)], [[], []]
    for _ in range(5):
        for i, (s, (x, u, how, _)) in enumerate(zip(streams, held)):
            with torch.cuda.stream(s):
                outs[i].append(sampling.sample(x, u, **how))
    torch.cuda.synchronize()
    for (x, u, how, _), got in zip(held, outs):
        want = sampling.sample(x, u, **how)
        assert all(torch.equal(t, want) for t in got)


@pytest.mark.gpu
def test_no_rows_subclasses_and_gradients(gpu):
    from metal_native import MetalNativeError, sampling

    x, u = logits(gpu, 4, 100, "fp32", 2)
    assert sampling.sample(x[:0], u[:0]).shape == (0,)
    want = sampling.sample(x, u)

    class Marked(torch.Tensor):
        pass

    assert torch.equal(sampling.sample(x.as_subclass(Marked), u), want)
    assert torch.equal(sampling.sample(torch.nn.Parameter(x), u).detach(), want)
    with torch.device(gpu):
        assert torch.equal(sampling.sample(x, u), want)
    t, log = sampling.sample(x.clone().requires_grad_(), u, return_logprob=True)
    assert torch.equal(t, want)
    with pytest.raises(MetalNativeError, match="no backward pass"):
        log.sum().backward()


@pytest.mark.gpu
def test_top_k_of_any_size(gpu):
    from metal_native import sampling

    x, u = logits(gpu, 3, 500, "fp16", 4)
    for k, same in ((10**30, 0), (2**63, 0), (2**31, 0), (-(10**30), 0), (True, 1)):
        assert torch.equal(sampling.sample(x, u, top_k=k), sampling.sample(x, u, top_k=same)), k


@pytest.mark.gpu
def test_tangents(gpu):
    """Lost by a log share, so refused; a token has none."""
    from torch.autograd import forward_ad

    from metal_native import MetalNativeError, sampling

    kw = dict(arguments(gpu), logits=logits(gpu, 3, 50, "fp32", 6)[0])
    want = sampling.sample(**kw)
    for name, x in kw.items():
        if x.is_floating_point():
            for grad in (True, False):
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    dual = {**kw, name: forward_ad.make_dual(x, torch.ones_like(x))}
                    with pytest.raises(MetalNativeError, match="tangent"):
                        sampling.sample(**dual, return_logprob=True)
                    got = sampling.sample(**dual)
                    assert torch.equal(got, want) and not got.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("V,top_k,unit", [(2, 0, -50), (32, 0, -50), (1000, 7, -50), (33, 0, -44), (1000, 600, -44), (2**18, 0, -44), (2**18 + 1, 0, -43),
                                          (2**20 + 1, 0, -41), (2**22, 0, -40)])
def test_the_smallest_weight_that_is_drawn(gpu, V, top_k, unit):
    """Half of the unit that sums go by; u = 0 draws the first token that weighs one."""
    from metal_native import sampling

    x = torch.full((2, V), -math.inf, device=gpu)
    x[:, 1] = 0.0
    x[0, 0], x[1, 0] = (unit - 0.9) * math.log(2), (unit - 1.1) * math.log(2)
    if top_k == 600:
        x[:, 2:602] = -80.0
    assert sampling.sample(x, torch.zeros(2, device=gpu), top_k=top_k).tolist() == [0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("first", [True, False])
def test_a_cut_far_under_the_largest_weight(gpu, first):
    """150 thousand weights around 2^-29 of the largest, of which top_p = 0.9999 leaves some two thirds: the cut lies under 2^-28.  Sums go by units
    of 2^-44, half a unit off for each token, so the aim may lie that much beside a token's share; so may the cut."""
    from metal_native import sampling

    V, n = 152064, 48
    g = torch.Generator(device=gpu)
    g.manual_seed(11)
    x = torch.randn(1, V, device=gpu, generator=g) * 0.3 - 20.0
    top = 0 if first else V - 1
    x[0, top] = 0.0
    off = torch.linspace(2e-6, 1.9e-4, n, device=gpu)
    u = 1 - off if first else off
    got = sampling.sample(x.expand(n, -1), u, top_p=0.9999).tolist()
    w = np.exp(x[0].double().cpu().numpy())
    order = np.argsort(-w, kind="stable")
    before = np.cumsum(w[order]) - w[order]
    keep = order[:int((before < float(np.float32(0.9999)) * w.sum()).sum())]
    err = V * 2.0**-45
    assert 0.4 * V < len(keep) < 0.9 * V
    least = w[keep].min()
    assert least < 2.0**-28
    kept = np.zeros(V)
    kept[keep] = w[keep]
    c = np.cumsum(kept)
    for t, share in zip(got, u.double().tolist()):
        aim, slack = share * c[-1], 2 * err + 2 * least
        # a cut that lies `err` beside its place takes or leaves tokens of about the least weight that stays
        assert w[t] >= least * 0.999
        assert c[t] + slack > aim and c[t] - kept[t] - slack <= aim, (t, share)
    assert len(set(got)) > n // 2


def arguments(dev):
    return dict(logits=torch.zeros(3, 50, device=dev), u=torch.zeros(3, device=dev), temperature=torch.ones(3, device=dev),
                top_k=torch.zeros(3, dtype=torch.int32, device=dev), top_p=torch.ones(3, device=dev), min_p=torch.zeros(3, device=dev))


CHANGES = {"logits": [None, lambda x: x.double(), lambda x: x[0], lambda x: x[:, :0], lambda x: x[None], lambda x: x.int()],
           "u": [None, 0.5, lambda x: x.half(), lambda x: x[:2], lambda x: x[None]],
           "temperature": [None, "hot", lambda x: x.half(), lambda x: x[:1], lambda x: x[:, None]],
           "top_k": [None, 1.5, float("nan"), float("inf"), lambda x: x.long(), lambda x: x[:2]],
           "top_p": [None, [1.0], lambda x: x.double(), lambda x: x[:2]],
           "min_p": [None, 1j, lambda x: x.bfloat16(), lambda x: x[:0]]}
REFUSED = [(n, i) for n, how in CHANGES.items() for i in range(len(how))]


def changed(name, i, dev):
    kw, change = arguments(dev), CHANGES[name][i]
    kw[name] = change(kw[name]) if callable(change) else change
    return kw


@pytest.mark.parametrize("name,i", REFUSED)
def test_refused_on_the_host(name, i, monkeypatch):
    """CPU tensors stand in for the GPU's; no call gets past the checks."""
    from metal_native import MetalNativeError, sampling

    def tensor(t, what, op):
        if not isinstance(t, torch.Tensor):
            raise MetalNativeError(f"{op}: {what} must be a torch.Tensor")

    monkeypatch.setattr(sampling, "_require_cuda", tensor)
    with pytest.raises(MetalNativeError, match="sampling.sample: "):
        sampling.sample(**changed(name, i, torch.device("cpu")))


def test_cpu_tensors_are_refused():
    from metal_native import MetalNativeError, sampling

    with pytest.raises(MetalNativeError, match="GPU tensor"):
        sampling.sample(**arguments(torch.device("cpu")))


@pytest.mark.gpu
def test_refused(gpu):
    from metal_native import MetalNativeError, sampling

    sampling.sample(**arguments(gpu))
    for name, i in REFUSED:
        with pytest.raises(MetalNativeError):
            sampling.sample(**changed(name, i, gpu))
    for name in arguments(gpu):
        with pytest.raises(MetalNativeError):
            sampling.sample(**{n: x.cpu() if n == name else x for n, x in arguments(gpu).items()})
    sampling.sample(**arguments(gpu))


def test_c_entry_refuses():
    import ctypes

    from metal_native import _lib

    class Sampling(ctypes.Structure):
        _fields_ = [("temperatures", ctypes.c_void_p), ("top_ps", ctypes.c_void_p), ("min_ps", ctypes.c_void_p), ("top_ks", ctypes.c_void_p),
                    ("temperature", ctypes.c_float), ("top_p", ctypes.c_float), ("min_p", ctypes.c_float), ("top_k", ctypes.c_int32)]

    L, how, P = _lib.load(), Sampling(temperature=1.0, top_p=1.0), 4096   # never followed

    def call(logits=P, ld=100, rows=3, vocab=100, dtype=0, u=P, settings=ctypes.byref(how), token=P, ws=None, ws_bytes=0):
        rc = L.mq_sample(logits, ld, rows, vocab, dtype, u, settings, token, None, ws, ws_bytes, None)
        return rc, L.mq_last_error().decode()

    for bad in (dict(logits=None), dict(u=None), dict(token=None), dict(settings=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1),
                dict(rows=2**31), dict(vocab=0), dict(vocab=2**28 + 1), dict(vocab=2**62), dict(ld=-1), dict(ld=2**62), dict(logits=P + 1),
                dict(logits=P + 2, dtype=2)):
        rc, text = call(**bad)
        assert rc == 4 and text.startswith("sampling.sample: "), (bad, rc, text)
    assert call(rows=0, logits=None)[0] == 0
    assert L.mq_sample_workspace_size(3, 0, 0, ctypes.byref(how)) == -1
    assert L.mq_sample_workspace_size(3, 100, 0, None) == -1


def test_workspace_follows_what_top_k_leaves():
    """Small vocabularies, whose rows go by the lanes' largest logits whether top_k says so or leaves all: the workspace
    has a place for these."""
    import ctypes

    from metal_native import _lib

    class Sampling(ctypes.Structure):
        _fields_ = [("temperatures", ctypes.c_void_p), ("top_ps", ctypes.c_void_p), ("min_ps", ctypes.c_void_p), ("top_ks", ctypes.c_void_p),
                    ("temperature", ctypes.c_float), ("top_p", ctypes.c_float), ("min_p", ctypes.c_float), ("top_k", ctypes.c_int32)]

    def size(top_k, vocab, top_p=1.0):
        return _lib.load().mq_sample_workspace_size(7, vocab, 0, ctypes.byref(Sampling(temperature=1.0, top_p=top_p, top_k=top_k)))

    for vocab in (2, 20, 32):
        assert size(vocab, vocab) >= 3 * 256 + 7 * 64 * 4   # of each part, of each row, the subs' sums; 64 lanes of each row
        for top_k in (0, -5, vocab + 1, 1000, 2**31 - 1):
            for top_p in (1.0, 0.9):
                assert size(top_k, vocab, top_p) == size(vocab, vocab, top_p), (vocab, top_k, top_p)


def test_the_largest_vocabulary_of_the_c_entry():
    """One more than 2^22 is refused: shared memory and the number of parts go by it."""
    import ctypes

    from metal_native import _lib

    how = (ctypes.c_char * 64)()
    for vocab, refused in ((2**22, False), (2**22 + 1, True)):
        size = _lib.load().mq_sample_workspace_size(1, vocab, 0, how)
        assert (size == -1) == refused and (refused or size > 0)
    assert _lib.load().mq_sample(4096, 2**22 + 1, 1, 2**22 + 1, 0, 4096, how, 4096, None, None, 0, None) == 4
