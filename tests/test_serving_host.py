"""What PagedServer refuses before anything reaches the GPU."""

from types import SimpleNamespace

import pytest
import torch


def model(max_len=48):
    cfg = SimpleNamespace(max_len=max_len, layers=1, kv_heads=1, head_dim=64, vocab=100)
    return SimpleNamespace(cfg=cfg, device=torch.device("cpu"))


def server(**how):
    from metal_native.serving import PagedServer

    s = PagedServer(model(), 8, 2, **how)
    s._run = lambda tokens: pytest.fail("reached the model")
    return s


@pytest.mark.parametrize("prompts", [[[100]], [[-1]], [[1, 2, 10**9]], [[5], [99, 100]], [[2**63]], [[1.5]], [["a"]], [[None]], [[torch.tensor(3.0)]]])
def test_prompts_of_tokens_outside_the_vocabulary(prompts):
    """The embedding's rows are read on the GPU, where an index past them ends the process."""
    s = server()
    with pytest.raises(ValueError, match="token"):
        s.start(prompts)
    assert len(s.free) == 8 and s.lens == [0, 0] and not s.last


def test_tokens_of_any_integer_type():
    import numpy as np

    s = server()
    asked = []
    s._run = lambda tokens: asked.append(tokens) or {i: 7 for i in tokens}
    assert s.start([[0, 99], np.array([5, 98])]) == {0: 7, 1: 7}
    assert {i: [int(t) for t in part] for i, part in asked[0].items()} == {0: [0, 99], 1: [5, 98]}


@pytest.mark.parametrize("how", [dict(recent=33), dict(recent=-1), dict(page_size=12), dict(page_size=4),
                                 dict(page_size=0), dict(page_size=1 << 17)])
def test_servers_that_could_not_cut_or_write(how):
    """Otherwise the first cut, or the first call, fails with pages taken and lengths moved."""
    with pytest.raises(ValueError, match="recent|page_size"):
        server(**{**dict(budget=32), **how})


def test_the_ends_of_the_allowed_range():
    for recent in (0, 32, None):
        assert server(budget=32, recent=recent).recent == (16 if recent is None else recent)
    assert server(page_size=8).width == 6 and server(page_size=64).width == 1


# ---- drawing and drafting ----
@pytest.mark.parametrize("how", [dict(temperature=-1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature="a"),
                                 dict(top_k=-1), dict(top_k=2**31), dict(top_k=1.5), dict(top_p=0), dict(top_p=1.1), dict(min_p=-0.1),
                                 dict(min_p=2), dict(seed=0.5), dict(draft=-1), dict(draft=1.5), dict(draft=4, budget=32)])
def test_settings_refused(how):
    with pytest.raises(ValueError, match="temperature|top_p|draft"):
        server(**how)


def test_drafts_need_a_server_that_drafts():
    s = server()
    assert s.step_drafted() == {}
    s.last[0] = 1
    with pytest.raises(ValueError, match="without draft"):
        s.step_drafted()


def test_what_is_guessed():
    from metal_native.serving import _History

    h = _History()
    h.extend([1, 2, 3, 4, 1, 2, 3, 5, 9, 2, 3])
    # after 2 3: 5 9 2 (newest), 4 1 2; after 3 alone: the same ones
    assert h.draft(16, 3) == ([3, 5, 9, 2, 4, 1, 2], [-1, 0, 1, 2, 0, 4, 5], [0, 1, 2, 3, 1, 2, 3])
    assert h.draft(4, 2) == ([3, 5, 9, 4], [-1, 0, 1, 0], [0, 1, 2, 1])
    assert h.draft(1, 2) == ([3], [-1], [0])
    h.extend([7])
    assert h.draft(16, 3) == ([7], [-1], [0])
    one = _History()
    one.extend([5])
    assert one.draft(8, 4) == ([5], [-1], [0])
    one.extend([5] * 6)   # places whose continuation is shorter than the depth
    tokens, parents, depths = one.draft(8, 4)
    assert tokens == [5] * len(tokens) and parents == list(range(-1, len(tokens) - 1)) and depths == list(range(len(tokens)))


def test_guesses_are_trees_of_what_followed():
    import random

    from metal_native.serving import _History

    rng = random.Random(1)
    line = [rng.randrange(3) for _ in range(200)]
    h = _History()
    for i, t in enumerate(line):
        h.extend([t])
        nodes, deepest = rng.randrange(1, 12), rng.randrange(1, 5)
        tokens, parents, depths = h.draft(nodes, deepest)
        assert tokens[0] == t and len(tokens) == len(parents) == len(depths) <= nodes and max(depths) <= deepest
        assert all(0 <= p < j and depths[j] == depths[p] + 1 for j, p in enumerate(parents) if j)
        assert len({(p, x) for p, x in zip(parents, tokens)}) == len(tokens)   # children of one node differ
        for j in range(1, len(tokens)):
            path, node = [], j
            while node >= 0:
                path.insert(0, tokens[node])
                node = parents[node]
            assert any(line[a:a + len(path)] == path for a in range(i - len(path) + 2))


def test_random_numbers_of_tokens():
    """By seed, order of starting and position; spread over the unit interval."""
    from metal_native import serving

    seen = []
    for seed in range(-1, 3):
        s = server(temperature=1.0, seed=seed)
        s._run = lambda tokens: {i: 7 for i in tokens}
        for turn in range(3):
            s.start([[1], [2]])
            seen += s.key
            s.finish(0), s.finish(1)
    assert len(set(seen)) == len(seen) == 24
    grabbed = []
    real, serving.sampling = serving.sampling, SimpleNamespace(sample=lambda x, u, **how: grabbed.append((u, how)))
    try:
        s._draws(torch.zeros(1), [0, 1] * 2000, [p for p in range(2000) for _ in range(2)])
    finally:
        serving.sampling = real
    u, how = grabbed[0]
    assert how == dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    assert u.dtype == torch.float32 and 0 <= float(u.min()) < 0.01 and 0.99 < float(u.max()) < 1 and abs(float(u.mean()) - 0.5) < 0.03
    assert u.unique().numel() > 3990
