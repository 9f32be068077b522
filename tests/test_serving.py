"""Generation over a paged cache: against the one-sequence decoder, and each
paged operator against its float64 form at the states that generation makes."""

from dataclasses import replace

import pytest
import torch

import paged_ref as ref
from test_decoder import tiny

pytestmark = pytest.mark.gpu
PROMPTS = [list(range(1, 38)), [5], list(range(400, 470)), list(range(16))]


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda:0")


def model_of(gpu, max_len=160):
    from metal_native.decoder import SyntheticDecoder

    return SyntheticDecoder(replace(tiny(), max_len=max_len), gpu, seed=3, prefilled=0)


def test_same_logits_as_the_decoder(gpu, monkeypatch):
    """Chunks and packed steps against one token at a time on the contiguous cache."""
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    server = PagedServer(m, 40, 4, chunk=16)
    logits = []
    real = PagedServer._forward
    monkeypatch.setattr(PagedServer, "_forward", lambda self, *a: logits.append(real(self, *a)) or logits[-1])
    got = server.start(PROMPTS)
    assert sorted(got) == [0, 1, 2, 3]
    logits.clear()
    feed = [dict(server.last)]
    for _ in range(3):
        feed.append(server.step())
    for s, prompt in enumerate(PROMPTS):
        line = prompt + [f[s] for f in feed]
        for i, t in enumerate(line[:-1]):
            _, want = m.step(torch.tensor([t], device=gpu), torch.tensor([i], device=gpu), return_logits=True)
            step = i - len(prompt)
            if step >= 0:   # both within 1e-2 + 1e-3 |x| of exact logits
                err = (logits[step][s].float() - want[0].float()).abs()
                assert bool((err <= 2e-2 + 2e-3 * want[0].float().abs()).all()), float(err.max())


def test_a_budget_that_is_never_reached_changes_nothing(gpu):
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    a, b = PagedServer(m, 40, 4, chunk=32), PagedServer(m, 40, 4, chunk=32, budget=150, slack=10)
    assert a.start(PROMPTS) == b.start(PROMPTS)
    for _ in range(4):
        assert a.step() == b.step()
    for s, n in enumerate(a.lens):
        for j in range(n):
            p = int(a.table[s, j // 16])
            assert p == int(b.table[s, j // 16])
    assert torch.equal(a.kv, b.kv)


def test_generation_under_a_budget(gpu, monkeypatch):
    """Every attention and eviction on the way is checked, then the pages."""
    from metal_native import paged
    from metal_native.serving import PagedServer

    calls = {"attention": 0, "evict": 0}
    attention, evict = paged.attention, paged.evict

    def checked_attention(q, k, v, table, lens, cu=None, **how):
        out, lse = attention(q, k, v, table, lens, cu, **how)
        o, l, ob, lb = ref.attention(q, k, v, table, lens, cu, scale=64**-0.5)
        assert bool(((out.double().cpu() - o).abs() <= ob).all()) and bool(((lse.double().cpu() - l).abs() <= lb).all())
        calls["attention"] += 1
        return out, lse

    def checked_evict(k, v, table, lens, mass, to, budget, *, recent):
        m, k0, v0 = mass.cpu(), k.clone(), v.clone()
        kept, n, left = evict(k, v, table, lens, mass, to, budget, recent=recent)
        for s in range(len(lens)):
            for h in range(k.shape[1]):
                want = torch.tensor(ref.keep(m[s, h], int(lens[s]), budget, recent))
                assert kept[s, h].tolist() == want.tolist()
                d = torch.arange(len(want))
                src, dst = table[s].cpu()[want // 16].long(), to[s].cpu()[d // 16].long()
                assert torch.equal(k[dst, h, d % 16], k0[src, h, want % 16])
                assert torch.equal(v[dst, h, d % 16], v0[src, h, want % 16])
        calls["evict"] += 1
        return kept, n, left

    monkeypatch.setattr(paged, "attention", checked_attention)
    monkeypatch.setattr(paged, "evict", checked_evict)
    m = model_of(gpu)
    server = PagedServer(m, 24, 4, chunk=24, budget=20, recent=6, slack=5)
    server.start(PROMPTS)
    for _ in range(12):
        server.step()
        assert all(n < 25 for n in server.lens)
        held = [p for h in server.held for p in h]
        assert sorted(held + server.free) == list(range(24))
    assert server.seen == [49, 13, 82, 28] and calls["evict"] >= 8 and calls["attention"] >= 26
    server.finish(2)
    assert server.start([[7, 8, 9]]).keys() == {2} and server.lens[2] == 3
    for s in range(4):
        server.finish(s)
    assert sorted(server.free) == list(range(24)) and float(server.mass.abs().max()) == 0 and server.step() == {}


def test_refusals_leave_the_server_as_it_was(gpu):
    from metal_native.serving import PagedServer

    m = model_of(gpu, max_len=48)
    server = PagedServer(m, 4, 2)
    for bad in ([[]], [[1] * 49], [[1]] * 3, [[1] * 40, [2] * 30]):   # empty, past max_len, too many, too few pages
        with pytest.raises(ValueError):
            server.start(bad)
        assert len(server.free) == 4 and server.lens == [0, 0] and not server.last
    server.start([[1] * 48])
    with pytest.raises(ValueError, match="48 positions"):
        server.step()
    assert server.lens[0] == 48
