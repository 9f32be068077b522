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


# ---- drawing and drafting ----
def lines_of(server, prompts, n, drafted):
    """n tokens behind every prompt, and how many passes they took."""
    lines = {s: [t] for s, t in server.start(prompts).items()}
    passes = 0
    while server.last:
        passes += 1
        for s, t in (server.step_drafted() if drafted else server.step()).items():
            lines[s] += t if drafted else [t]
            if len(lines[s]) >= n:
                server.finish(s)
    return [lines[s][:n] for s in sorted(lines)], passes


def exact(monkeypatch):
    """Logits that depend on the row's token alone, so that how rows were grouped rounds nothing."""
    from metal_native.serving import PagedServer

    real = PagedServer._forward

    def forward(self, flat, pos, rows, table, lens, cu, max_q, last, tree=None):
        out = real(self, flat, pos, rows, table, lens, cu, max_q, last, tree)
        flat = flat if last is None else flat[last]   # mostly one token behind another: text that repeats
        x = torch.full(out.shape, -4.0, dtype=out.dtype, device=out.device)
        for i, step in enumerate((7, 11, 30)):
            x[torch.arange(len(flat), device=x.device), (flat * step + i) % 23] += (6.0, 4.0, 1.0)[i]
        return x

    monkeypatch.setattr(PagedServer, "_forward", forward)


@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.8, top_k=5, seed=3), dict(temperature=1.3, top_p=0.9, min_p=0.01)])
def test_drafts_change_no_token(gpu, monkeypatch, settings):
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    exact(monkeypatch)
    plain, _ = lines_of(PagedServer(m, 60, 4, chunk=32, **settings), PROMPTS, 60, False)
    for draft in (1, 6, 40):
        server = PagedServer(m, 60, 4, chunk=32, draft=draft, **settings)
        got, passes = lines_of(server, PROMPTS, 60, True)
        assert got == plain and passes < 59
    other, _ = lines_of(PagedServer(m, 60, 4, chunk=32, **{**settings, "seed": 5}), PROMPTS, 60, False)
    assert (other == plain) == (not settings)


def test_a_sequence_draws_the_same_in_other_company(gpu, monkeypatch):
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    exact(monkeypatch)
    how = dict(temperature=1.0, seed=9)
    both, _ = lines_of(PagedServer(m, 40, 4, **how), PROMPTS[:2], 20, False)
    one, _ = lines_of(PagedServer(m, 40, 4, **how), PROMPTS[:1], 20, False)
    assert one[0] == both[0]


def test_drafted_caches_and_logits(gpu, monkeypatch):
    """After drafted steps the cache holds what the kept tokens leave when they run one at a time, and the logits of
    the path are theirs."""
    from metal_native import paged
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    server = PagedServer(m, 60, 4, chunk=32, draft=12)
    logits, paths = [], []
    real_forward, real_accept = PagedServer._forward, paged.accept
    monkeypatch.setattr(PagedServer, "_forward", lambda self, *a: logits.append(real_forward(self, *a)) or logits[-1])

    def agree(k, v, table, lens, drawn, drafted, parents, cu=None, *, steps):
        """Takes a guess wherever there is one: random weights hardly repeat themselves."""
        drawn = drawn.clone()
        ends = [0, *range(1, len(drawn) + 1)] if cu is None else cu.tolist()
        up, tokens = parents.tolist(), drafted.tolist()
        for lo, hi in zip(ends, ends[1:]):
            for i in range(hi - 1, lo, -1):
                drawn[lo + up[i]] = tokens[i]
        out = real_accept(k, v, table, lens, drawn, drafted, parents, cu, steps=steps)
        paths.append((ends, out[0].tolist(), out[2].tolist()))
        return out

    monkeypatch.setattr(paged, "accept", agree)
    prompts = [[3, 4, 5, 6] * 9, [5], [9, 8, 7, 9, 8, 1, 9, 8], list(range(16))]
    lines = {s: p + [t] for (s, t), p in zip(server.start(prompts).items(), prompts)}
    logits.clear()
    firsts = {s: len(line) - 1 for s, line in lines.items()}
    rows = {s: [] for s in lines}
    for turn in range(5):
        for s, t in server.step_drafted().items():
            lines[s] += t
        ends, path, count = paths[-1]
        for s in lines:
            rows[s] += [logits[-1][ends[s] + i] for i in path[s][:count[s]]]
    assert max(max(c) for _, _, c in paths) > 3
    for s, line in lines.items():
        assert server.lens[s] == server.seen[s] == len(line) - 1 and server.last[s] == line[-1]
        for i, t in enumerate(line[:-1]):
            _, want = m.step(torch.tensor([t], device=gpu), torch.tensor([i], device=gpu), return_logits=True)
            if i >= firsts[s]:   # both within 1e-2 + 1e-3 |x| of exact logits
                got = rows[s][i - firsts[s]].float()
                err = (got - want[0].float()).abs()
                assert bool((err <= 2e-2 + 2e-3 * want[0].float().abs()).all()), (s, i, float(err.max()))
        n = len(line) - 1
        slots = torch.tensor([server.held[s][i // 16] * 16 + i % 16 for i in range(n)], device=gpu)
        kv = server.kv.permute(0, 1, 3, 2, 4, 5).flatten(3, 4)[:, :, :, slots]
        want = m.kv[:, :, :, :n]
        assert bool(((kv.float() - want.float()).abs() <= 2e-2 + 2e-3 * want.float().abs()).all())


def test_drafts_where_pages_and_positions_are_short(gpu, monkeypatch):
    from metal_native.serving import PagedServer

    m = model_of(gpu, max_len=48)
    exact(monkeypatch)
    prompts = [[1, 2, 3] * 5, [4, 5] * 7]
    plain, _ = lines_of(PagedServer(m, 6, 2), prompts, 30, False)
    server = PagedServer(m, 6, 2, draft=30)   # three pages a sequence: all that 48 positions need
    got, _ = lines_of(server, prompts, 30, True)
    assert got == plain
    assert sorted(server.free) == list(range(6)) and not server.history

    server = PagedServer(m, 3, 2, draft=30)
    server.start([[1, 2, 3] * 5, [4]])   # 15 slots and 1: a page each, guesses take the third
    before = dict(server.last)
    server.step_drafted()
    assert before.keys() == server.last.keys()
    server.finish(1)
    assert sum(len(h) for h in server.held) + len(server.free) == 3
    while server.seen[0] < 48:
        server.step_drafted()
    with pytest.raises(ValueError, match="48 positions"):
        server.step_drafted()


def test_logits_with_nothing_to_draw(gpu, monkeypatch):
    """The server stays as it was: the embedding has no row for -1."""
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    server = PagedServer(m, 40, 4, temperature=1.0, draft=3)
    server.start(PROMPTS)
    kept = dict(server.last), list(server.lens), list(server.seen)
    real = PagedServer._forward
    monkeypatch.setattr(PagedServer, "_forward", lambda self, *a: torch.full_like(real(self, *a), float("nan")))
    for step in (server.step, server.step_drafted):
        with pytest.raises(RuntimeError, match="nothing above"):
            step()
        assert (dict(server.last), list(server.lens), list(server.seen)) == kept
    monkeypatch.setattr(PagedServer, "_forward", real)
    assert server.step().keys() == kept[0].keys()


def test_greedy_steps_pass_over_nan(gpu, monkeypatch):
    """A logit that is no number is never the largest, with drafts or without; a row of nothing else is refused."""
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    exact(monkeypatch)
    even = PagedServer._forward

    def forward(self, *a):
        x = even(self, *a)
        x[:, 5] = float("nan")
        return x

    monkeypatch.setattr(PagedServer, "_forward", forward)
    plain, _ = lines_of(PagedServer(m, 60, 4, chunk=32), PROMPTS, 40, False)
    assert not any(5 in line for line in plain)
    assert lines_of(PagedServer(m, 60, 4, chunk=32, draft=6), PROMPTS, 40, True)[0] == plain
    server = PagedServer(m, 60, 4, chunk=32)
    server.start(PROMPTS)
    kept = dict(server.last), list(server.lens), list(server.seen)
    monkeypatch.setattr(PagedServer, "_forward", lambda self, *a: torch.full_like(even(self, *a), float("nan")))
    with pytest.raises(RuntimeError, match="nothing above"):
        server.step()
    assert (dict(server.last), list(server.lens), list(server.seen)) == kept


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_logits_inside_a_prompt_draw_nothing(gpu, monkeypatch, temperature):
    """What stands behind a chunk that is not a prompt's last may hold nothing above -inf."""
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    real, calls = PagedServer._forward, []

    def forward(self, *a):
        x = real(self, *a)
        calls.append(len(calls))
        return torch.full_like(x, -float("inf")) if calls[-1] < bad else x

    monkeypatch.setattr(PagedServer, "_forward", forward)
    bad = 0
    want = PagedServer(m, 60, 4, chunk=16, temperature=temperature).start([PROMPTS[0], PROMPTS[2]])
    calls.clear()
    bad = 2   # of three chunks and of five
    server = PagedServer(m, 60, 4, chunk=16, temperature=temperature)
    assert server.start([PROMPTS[0], PROMPTS[2]]) == want
    calls.clear()
    bad = 3
    server = PagedServer(m, 60, 4, chunk=16, temperature=temperature)
    with pytest.raises(RuntimeError, match="nothing above"):
        server.start([PROMPTS[0], PROMPTS[2]])
    assert not server.last and sorted(server.free) == list(range(60)) and server.lens == [0] * 4


def test_drafted_steps_are_sized_by_what_the_cache_holds(gpu, monkeypatch):
    """The operators see the pages in use, not the widest table there can be: launches go by its width."""
    from metal_native import paged
    from metal_native.serving import PagedServer

    m = model_of(gpu)
    widths = []
    real = paged.tree_attention
    monkeypatch.setattr(paged, "tree_attention", lambda q, k, v, table, *a, **how: widths.append(table.shape[1]) or real(q, k, v, table, *a, **how))
    server = PagedServer(m, 60, 4, draft=6)
    server.start([[1, 2, 3] * 3, [4] * 20])
    while server.seen[1] < 120:
        widths.clear()
        server.step_drafted()
        assert len(set(widths)) == 1 and -(-max(server.seen) // 16) <= widths[0] <= max(len(h) for h in server.held)
    server.finish(1)
    server.step_drafted()
    assert -(-server.seen[0] // 16) <= widths[-1] <= len(server.held[0])
