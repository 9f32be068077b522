"""Greedy generation of many sequences over one paged key/value cache, with the
layers of ``SyntheticDecoder`` (int4 ``dequant_matmul``) and the operators of
``paged``: prompts run in chunks, every later step adds one token to each
sequence, and a sequence that outgrows its budget keeps, per layer and
key/value head, its newest slots and those that gathered the most attention.
No reference counterpart.

Pages are handed out by the host, one numbering for all layers; lengths live on
the host and go to the device as one small copy a call.
"""

from __future__ import annotations

from operator import index

import torch

from . import ops, paged
from .decoder import SyntheticDecoder

__all__ = ["PagedServer", "serve_tokens_per_second"]


class PagedServer:
    """``pages`` pages of ``page_size`` slots, at most ``batch`` sequences.

    ``budget``: slots that a sequence is cut back to once it holds ``slack``
    more, ``recent`` of them its newest (default half); ``None``: never cut, a
    sequence ends at the model's ``max_len`` positions.
    """

    def __init__(self, model: SyntheticDecoder, pages: int, batch: int, *, page_size: int = 16, chunk: int = 512,
                 budget: int | None = None, recent: int | None = None, slack: int = 64):
        cfg = model.cfg
        if min(pages, batch, chunk) < 1 or (budget is not None and (budget < 1 or slack < 1)):
            raise ValueError("PagedServer: pages, batch, chunk, budget and slack must be positive")
        if budget is not None and recent is not None and not 0 <= recent <= budget:
            raise ValueError(f"PagedServer: recent must be 0 .. budget, got {recent} of {budget}")
        if not 8 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError(f"PagedServer: page_size must be a power of two from 8 to 65536, got {page_size}")
        self.model, self.page_size, self.chunk, self.budget, self.slack = model, page_size, chunk, budget, slack
        self.recent = budget // 2 if budget is not None and recent is None else recent
        most = cfg.max_len if budget is None else min(cfg.max_len, budget + slack + chunk)
        self.width = -(-most // page_size)
        dev = model.device
        self.kv = torch.zeros((cfg.layers, 2, pages, cfg.kv_heads, page_size, cfg.head_dim), dtype=torch.float16, device=dev)
        self.table = torch.full((batch, self.width), -1, dtype=torch.int32, device=dev)
        self.mass = None
        if budget is not None:
            self.mass = torch.zeros((cfg.layers, batch, cfg.kv_heads, self.width * page_size), device=dev)
        self.free = list(range(pages - 1, -1, -1))
        self.held: list[list[int]] = [[] for _ in range(batch)]   # pages of each sequence, in order
        self.lens = [0] * batch                                   # slots
        self.seen = [0] * batch                                   # positions; more than slots after a cut
        self.last: dict[int, int] = {}                            # the token each live sequence goes on from

    def start(self, prompts: list[list[int]]) -> dict[int, int]:
        """Runs the prompts, all together and in chunks; returns the next token
        of each by the number that its sequence got."""
        idle = [s for s in range(len(self.lens)) if s not in self.last]
        if len(prompts) > len(idle) or any(not 0 < len(p) <= self.model.cfg.max_len for p in prompts):
            raise ValueError("PagedServer.start: more prompts than idle sequences, or one empty or past max_len")
        try:   # the embedding is read on the GPU, where an index past its rows ends the process
            prompts = [[index(t) for t in p] for p in prompts]
        except TypeError as e:
            raise ValueError(f"PagedServer.start: a token is not a whole number ({e})") from None
        if any(not 0 <= t < self.model.cfg.vocab for p in prompts for t in p):
            raise ValueError(f"PagedServer.start: a token outside the vocabulary of {self.model.cfg.vocab}")
        ids, at, out = idle[:len(prompts)], 0, {}
        try:
            while any(len(p) > at for p in prompts):
                part = {s: p[at:at + self.chunk] for s, p in zip(ids, prompts) if len(p) > at}
                out.update(self._run(part))
                at += self.chunk
        except Exception:
            for s in ids:
                self.finish(s)
            raise
        self.last.update(out)
        return out

    def step(self) -> dict[int, int]:
        """One more token for every live sequence."""
        if not self.last:
            return {}
        out = self._run({s: [t] for s, t in self.last.items()})
        self.last.update(out)
        return out

    def finish(self, s: int) -> None:
        """Ends sequence ``s``; its pages go back."""
        self.last.pop(s, None)
        self.free += self.held[s]
        self.held[s], self.lens[s], self.seen[s] = [], 0, 0
        self.table[s].fill_(-1)
        if self.mass is not None:
            self.mass[:, s].zero_()

    def _take(self, n: int) -> list[int]:
        return [self.free.pop() for _ in range(n)]

    def _run(self, tokens: dict[int, list[int]]) -> dict[int, int]:
        cfg, dev, ps = self.model.cfg, self.model.device, self.page_size
        ids, new = list(tokens), [len(t) for t in tokens.values()]
        need = [-(-(self.lens[s] + n) // ps) - len(self.held[s]) for s, n in zip(ids, new)]
        if any(self.seen[s] + n > cfg.max_len for s, n in zip(ids, new)):
            raise ValueError(f"PagedServer: a sequence would pass the model's {cfg.max_len} positions")
        pages = sum(need)
        if self.budget is not None and any(self.lens[s] + n >= self.budget + self.slack for s, n in zip(ids, new)):
            pages += -(-self.budget // ps)   # a cut moves to new pages first
        if pages > len(self.free):
            raise ValueError(f"PagedServer: {pages} pages needed, {len(self.free)} free")
        for s, n in zip(ids, need):
            if n:
                got = self._take(n)
                self.table[s, len(self.held[s]):len(self.held[s]) + n] = torch.tensor(got, dtype=torch.int32)
                self.held[s] += got
        pos = torch.tensor([self.seen[s] + i for s, n in zip(ids, new) for i in range(n)], device=dev)
        for s, n in zip(ids, new):
            self.lens[s] += n
            self.seen[s] += n
        rows = torch.tensor(ids, device=dev)
        table = self.table.index_select(0, rows)
        ends = torch.tensor(new).cumsum(0)
        lens = torch.tensor([self.lens[s] for s in ids], dtype=torch.int32, device=dev)
        single = len(pos) == len(ids)
        cu = None if single else torch.cat([ends.new_zeros(1), ends]).to(dev, torch.int32)
        flat = torch.tensor([t for part in tokens.values() for t in part], device=dev)
        logits = self._forward(flat, pos, rows, table, lens, cu, max(new), ends.to(dev) - 1)
        if self.budget is not None:
            self._cut([s for s in ids if self.lens[s] >= self.budget + self.slack])
        return dict(zip(ids, logits.float().argmax(-1).tolist()))

    def _forward(self, flat, pos, rows, table, lens, cu, max_q, last):
        m = self.model
        x, delta = m.embed.index_select(0, flat), None
        for li, layer in enumerate(m.layers):
            k, v = self.kv[li, 0], self.kv[li, 1]
            qkv = layer["qkv"](ops.add_rmsnorm(x, delta, layer["ln1"], m.cfg.eps))
            q = paged.rope_kv(qkv, m.cos, m.sin, pos, k, v, table, lens, cu)
            if self.mass is None:
                a = paged.attention(q, k, v, table, lens, cu, max_q=max_q)
            else:
                a, lse = paged.attention(q, k, v, table, lens, cu, max_q=max_q, return_lse=True)
                self.mass[li].index_add_(0, rows, paged.attention_mass(q, k, table, lens, lse, cu, max_q=max_q))
            o = layer["o"](a.reshape(a.shape[0], -1))
            delta = layer["down"](layer["gate_up"](ops.add_rmsnorm(x, o, layer["ln2"], m.cfg.eps), "swiglu"))
        h = ops.add_rmsnorm(x, delta, m.norm, m.cfg.eps)
        return m.lm_head(h.index_select(0, last))

    def _cut(self, ids: list[int]) -> None:
        """Cuts these sequences to the budget, in every layer."""
        if not ids:
            return
        need, dev = -(-self.budget // self.page_size), self.model.device
        if need * len(ids) > len(self.free):   # one after the other: each gives back no fewer than it takes
            for s in ids:
                self._cut([s])
            return
        pages = [self._take(need) for _ in ids]
        rows = torch.tensor(ids, device=dev)
        to = torch.full((len(ids), self.width), -1, dtype=torch.int32)
        to[:, :need] = torch.tensor(pages, dtype=torch.int32)
        to = to.to(dev)
        table = self.table.index_select(0, rows)
        lens = torch.tensor([self.lens[s] for s in ids], dtype=torch.int32, device=dev)
        for li in range(len(self.model.layers)):
            mass = self.mass[li].index_select(0, rows)
            _, _, left = paged.evict(self.kv[li, 0], self.kv[li, 1], table, lens, mass, to, self.budget, recent=self.recent)
            self.mass[li].index_copy_(0, rows, left)
        self.table.index_copy_(0, rows, to)
        for s, got in zip(ids, pages):
            self.free += self.held[s]
            self.held[s], self.lens[s] = got, self.budget


def serve_tokens_per_second(model: SyntheticDecoder, batch: int = 8, prompt: int = 700, tokens: int = 64, *,
                            budget: int | None = 512, page_size: int = 16) -> dict:
    """Runs ``batch`` random prompts and ``tokens`` steps; returns tokens/s of
    the prompts and of the steps."""
    room = -(-(prompt + tokens) // page_size) + (0 if budget is None else -(-budget // page_size))
    server = PagedServer(model, batch * room, batch, page_size=page_size, budget=budget)
    gen = torch.Generator("cpu")
    gen.manual_seed(0)
    asked = torch.randint(0, model.cfg.vocab, (batch, prompt), generator=gen, device="cpu").tolist()
    t = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    for timed in (False, True):
        for s in list(server.last):
            server.finish(s)
        t[0].record()
        server.start(asked)
        t[1].record()
        for _ in range(tokens if timed else 2):
            server.step()
        t[2].record()
    torch.cuda.synchronize(model.device)
    return {"prompt_tokens_per_s": batch * prompt / t[0].elapsed_time(t[1]) * 1e3,
            "tokens_per_s": batch * tokens / t[1].elapsed_time(t[2]) * 1e3}


if __name__ == "__main__":
    import argparse

    from .decoder import qwen25_7b

    ap = argparse.ArgumentParser(description="Prompts and greedy steps over a paged cache (random weights).")
    for name, value in (("batch", 8), ("prompt", 700), ("tokens", 64), ("budget", 512)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args()
    decoder = SyntheticDecoder(qwen25_7b(max_len=args.prompt + args.tokens), "cuda:0", prefilled=0)
    print(serve_tokens_per_second(decoder, args.batch, args.prompt, args.tokens, budget=args.budget or None))
