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
