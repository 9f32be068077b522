"""Generation of many sequences over one paged key/value cache, with the
layers of ``SyntheticDecoder`` (int4 ``dequant_matmul``) and the operators of
``paged`` and ``sampling``: prompts run in chunks, every later step adds one
token to each sequence, or with drafts as many as the model agrees to, and a
sequence that outgrows its budget keeps, per layer and key/value head, its
newest slots and those that gathered the most attention.
No reference counterpart.

Pages are handed out by the host, one numbering for all layers; lengths live on
the host and go to the device as one small copy a call.
"""

from __future__ import annotations

from operator import index

import torch

from . import ops, paged, sampling
from .decoder import SyntheticDecoder

__all__ = ["PagedServer", "serve_tokens_per_second"]

_MASK = 2**64 - 1


def _mixed(x: int) -> int:
    """64 bits in which every bit of ``x`` counts: the mixing function of SplitMix64 (Steele, Lea and Flood, 2014)."""
    x = (x ^ x >> 30) * 0xBF58476D1CE4E5B9 & _MASK
    x = (x ^ x >> 27) * 0x94D049BB133111EB & _MASK
    return x ^ x >> 31


class _History:
    """A sequence's tokens, and where each run of 1 to 3 of them was seen last."""

    RUNS, KEPT = 3, 4

    def __init__(self):
        self.tokens: list[int] = []
        self.behind: dict[tuple, list[int]] = {}   # run -> indexes of the tokens that followed it, newest last

    def extend(self, tokens) -> None:
        for t in tokens:
            at = len(self.tokens)
            for n in range(1, min(self.RUNS, at) + 1):
                seen = self.behind.setdefault(tuple(self.tokens[at - n:]), [])
                seen.append(at)
                del seen[:-self.KEPT]
            self.tokens.append(t)

    def draft(self, nodes: int, deepest: int) -> tuple[list[int], list[int], list[int]]:
        """What followed the newest run earlier, as a tree of at most ``nodes`` nodes
        and that depth, its root the newest token: tokens, parents, depths."""
        tokens, parents, depths = [self.tokens[-1]], [-1], [0]
        child: dict[tuple, int] = {}
        for n in range(min(self.RUNS, len(self.tokens)), 0, -1):
            for at in reversed(self.behind.get(tuple(self.tokens[-n:]), ())):
                node = 0
                for t in self.tokens[at:at + deepest]:
                    nxt = child.get((node, t))
                    if nxt is None:
                        if len(tokens) >= nodes:
                            return tokens, parents, depths
                        nxt = child[node, t] = len(tokens)
                        tokens.append(t)
                        parents.append(node)
                        depths.append(depths[node] + 1)
                    node = nxt
        return tokens, parents, depths


class PagedServer:
    """``pages`` pages of ``page_size`` slots, at most ``batch`` sequences.

    ``budget``: slots that a sequence is cut back to once it holds ``slack``
    more, ``recent`` of them its newest (default half); ``None``: never cut, a
    sequence ends at the model's ``max_len`` positions.

    ``temperature``, ``top_k``, ``top_p``, ``min_p``: how tokens are drawn, as in
    ``sampling.sample``; at temperature 0 the largest logit is taken.  The random
    number of a token comes from ``seed``, from how many sequences were started
    before its own and from its position, not from what else runs or is drafted.

    ``draft``: the most tokens that ``step_drafted`` guesses for a sequence, from
    what followed its last tokens earlier in it; not with a budget.
    """

    def __init__(self, model: SyntheticDecoder, pages: int, batch: int, *, page_size: int = 16, chunk: int = 512,
                 budget: int | None = None, recent: int | None = None, slack: int = 64, temperature: float = 0.0,
                 top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, seed: int = 0, draft: int = 0):
        cfg = model.cfg
        if min(pages, batch, chunk) < 1 or (budget is not None and (budget < 1 or slack < 1)):
            raise ValueError("PagedServer: pages, batch, chunk, budget and slack must be positive")
        if budget is not None and recent is not None and not 0 <= recent <= budget:
            raise ValueError(f"PagedServer: recent must be 0 .. budget, got {recent} of {budget}")
        if not 8 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError(f"PagedServer: page_size must be a power of two from 8 to 65536, got {page_size}")
        try:
            temperature, top_k, top_p, min_p, seed, draft = float(temperature), index(top_k), float(top_p), float(min_p), index(seed), index(draft)
        except (TypeError, ValueError) as e:
            raise ValueError(f"PagedServer: temperature, top_p and min_p must be numbers, top_k, seed and draft whole ones ({e})") from None
        if not 0 <= temperature < float("inf") or not 0 <= top_k < 2**31 or not 0 < top_p <= 1 or not 0 <= min_p <= 1:
            raise ValueError("PagedServer: temperature and top_k must not be negative, top_p in (0, 1], min_p in [0, 1]")
        if draft < 0 or (draft and budget is not None):
            raise ValueError("PagedServer: draft must not be negative, and a budget has none")
        self.settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        self.seed, self.draft, self.started = seed, draft, 0
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
        self.key = [0] * batch                                    # of the random numbers
        self.history: dict[int, _History] = {}                    # with drafts

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
        for i, s in enumerate(ids):
            self.key[s] = _mixed(_mixed(self.seed & _MASK) + self.started + i + 1 & _MASK)
        try:
            while any(len(p) > at for p in prompts):
                part = {s: p[at:at + self.chunk] for s, p in zip(ids, prompts) if len(p) > at}
                out.update(self._run(part))
                at += self.chunk
            self._drawn(out)
        except Exception:
            for s in ids:
                self.finish(s)
            raise
        self.started += len(ids)
        if self.draft:
            for s, p in zip(ids, prompts):
                self.history[s] = _History()
                self.history[s].extend(p)
        self._goes_on({s: [t] for s, t in out.items()})
        return out

    def step(self) -> dict[int, int]:
        """One more token for every live sequence."""
        if not self.last:
            return {}
        out = self._run({s: [t] for s, t in self.last.items()})
        self._goes_on({s: [t] for s, t in out.items()})
        return out

    def step_drafted(self) -> dict[int, list[int]]:
        """One or more tokens for every live sequence, at most ``draft + 1``, in one
        pass of the model: those that ``step`` would give, up to the rounding of logits.

        Guessed tokens run behind the newest one as a tree, one is drawn behind
        every node of it, and the path of guesses that were drawn stays.  Where
        positions or pages are short, fewer are guessed."""
        if not self.last:
            return {}
        if not self.draft:
            raise ValueError("PagedServer.step_drafted: the server was made without draft")
        most, deepest = self.draft + 1, self._deepest()
        trees = {s: self.history[s].draft(max(1, min(most, self.model.cfg.max_len - self.seen[s])), deepest) for s in self.last}
        if self._pages({s: len(t[0]) for s, t in trees.items()}) > len(self.free):
            self._trim()
        if self._pages({s: len(t[0]) for s, t in trees.items()}) > len(self.free):
            trees = {s: ([t], [-1], [0]) for s, t in self.last.items()}
        out = self._run({s: t[0] for s, t in trees.items()}, trees)
        self._goes_on(out)
        return out

    def _deepest(self) -> int:
        """Half of the guesses go to the newest place that matches, the others to
        where older and shorter ones differ from it."""
        return -(-self.draft // 2)

    def _goes_on(self, out: dict[int, list[int]]) -> None:
        for s, tokens in out.items():
            self.last[s] = tokens[-1]
            if self.draft:
                self.history[s].extend(tokens)

    def finish(self, s: int) -> None:
        """Ends sequence ``s``; its pages go back."""
        self.last.pop(s, None)
        self.history.pop(s, None)
        self.free += self.held[s]
        self.held[s], self.lens[s], self.seen[s] = [], 0, 0
        self.table[s].fill_(-1)
        if self.mass is not None:
            self.mass[:, s].zero_()

    def _take(self, n: int) -> list[int]:
        return [self.free.pop() for _ in range(n)]

    def _pages(self, new: dict[int, int]) -> int:
        """How many pages these sequences lack for so many more slots."""
        return sum(max(0, -(-(self.lens[s] + n) // self.page_size) - len(self.held[s])) for s, n in new.items())

    def _trim(self) -> None:
        """Takes back the pages that only guesses reached."""
        for s, held in enumerate(self.held):
            keep = -(-self.lens[s] // self.page_size)
            if keep < len(held):
                self.table[s, keep:len(held)] = -1
                self.free += held[keep:]
                del held[keep:]

    def _draws(self, logits, ids, pos) -> torch.Tensor:
        """A token for each row; row i stands at position ``pos[i]`` of sequence ``ids[i]``."""
        if self.settings["temperature"] == 0:
            return sampling.sample(logits, torch.zeros(len(pos), device=logits.device), temperature=0)
        u = [(_mixed(self.key[s] + _mixed(p + 1) & _MASK) >> 40) * 2.0**-24 for s, p in zip(ids, pos)]
        return sampling.sample(logits, torch.tensor(u, dtype=torch.float32, device=logits.device), **self.settings)

    def _run(self, tokens: dict[int, list[int]], trees=None):
        """The next token of each sequence; with its tree in ``trees``, those of the path that was drawn."""
        cfg, dev, ps = self.model.cfg, self.model.device, self.page_size
        ids, new = list(tokens), [len(t) for t in tokens.values()]
        if any(self.seen[s] + n > cfg.max_len for s, n in zip(ids, new)):
            raise ValueError(f"PagedServer: a sequence would pass the model's {cfg.max_len} positions")
        pages = self._pages(dict(zip(ids, new)))
        if self.draft and pages > len(self.free):
            self._trim()
            pages = self._pages(dict(zip(ids, new)))
        if self.budget is not None and any(self.lens[s] + n >= self.budget + self.slack for s, n in zip(ids, new)):
            pages += -(-self.budget // ps)   # a cut moves to new pages first
        if pages > len(self.free):
            raise ValueError(f"PagedServer: {pages} pages needed, {len(self.free)} free")
        for s, n in zip(ids, new):
            n = -(-(self.lens[s] + n) // ps) - len(self.held[s])
            if n > 0:
                got = self._take(n)
                self.table[s, len(self.held[s]):len(self.held[s]) + n] = torch.tensor(got, dtype=torch.int32)
                self.held[s] += got
        at = [self.seen[s] + i for s, n in zip(ids, new) for i in (range(n) if trees is None else trees[s][2])]
        pos = torch.tensor(at, device=dev)
        rows = torch.tensor(ids, device=dev)
        table = self.table.index_select(0, rows)
        ends = torch.tensor(new).cumsum(0)
        lens = torch.tensor([self.lens[s] + n for s, n in zip(ids, new)], dtype=torch.int32, device=dev)
        single = len(pos) == len(ids)
        cu = None if single else torch.cat([ends.new_zeros(1), ends]).to(dev, torch.int32)
        flat = torch.tensor([t for part in tokens.values() for t in part], device=dev)
        if trees is not None:
            # launches are sized by the table's width, not by lengths that only the device knows: no more columns than are used
            table = table[:, :max(-(-(self.lens[s] + n) // ps) for s, n in zip(ids, new))]
            parents = torch.tensor([p for t in trees.values() for p in t[1]], dtype=torch.int32, device=dev)
            tree = paged.ancestors(parents, cu, max(new))
            logits = self._forward(flat, pos, rows, table, lens, cu, max(new), None, tree)
            drawn = self._draws(logits, [s for s, n in zip(ids, new) for _ in range(n)], at)
            _, got, count, _ = paged.accept(self.kv[:, 0], self.kv[:, 1], table, lens, drawn, flat, parents, cu,
                                            steps=1 + max(max(t[2]) for t in trees.values()))
            out = {s: line[:n] for s, line, n in zip(ids, got.tolist(), count.tolist())}
            self._drawn({s: line[-1] for s, line in out.items()})
            for s, line in out.items():
                self.lens[s] += len(line)
                self.seen[s] += len(line)
            return out
        logits = self._forward(flat, pos, rows, table, lens, cu, max(new), ends.to(dev) - 1)
        out = dict(zip(ids, self._draws(logits, ids, [self.seen[s] + n - 1 for s, n in zip(ids, new)]).tolist()))
        self._drawn({s: t for s, t in out.items() if s in self.last})   # of a prompt only what its last chunk gives counts
        for s, n in zip(ids, new):
            self.lens[s] += n
            self.seen[s] += n
        if self.budget is not None:
            self._cut([s for s in ids if self.lens[s] >= self.budget + self.slack])
        return out

    def _drawn(self, out: dict[int, int]) -> None:
        """Before anything counts as generated: a row with nothing to draw gives -1, which the embedding has no row for."""
        empty = [s for s, t in out.items() if t < 0]
        if empty:
            raise RuntimeError(f"PagedServer: the logits of sequence {empty[0]} hold nothing above -inf")

    def _forward(self, flat, pos, rows, table, lens, cu, max_q, last, tree=None):
        m = self.model
        x, delta = m.embed.index_select(0, flat), None
        for li, layer in enumerate(m.layers):
            k, v = self.kv[li, 0], self.kv[li, 1]
            qkv = layer["qkv"](ops.add_rmsnorm(x, delta, layer["ln1"], m.cfg.eps))
            q = paged.rope_kv(qkv, m.cos, m.sin, pos, k, v, table, lens, cu)
            if tree is not None:
                a = paged.tree_attention(q, k, v, table, lens, tree, cu, max_q=max_q)
            elif self.mass is None:
                a = paged.attention(q, k, v, table, lens, cu, max_q=max_q)
            else:
                a, lse = paged.attention(q, k, v, table, lens, cu, max_q=max_q, return_lse=True)
                self.mass[li].index_add_(0, rows, paged.attention_mass(q, k, table, lens, lse, cu, max_q=max_q))
            o = layer["o"](a.reshape(a.shape[0], -1))
            delta = layer["down"](layer["gate_up"](ops.add_rmsnorm(x, o, layer["ln2"], m.cfg.eps), "swiglu"))
        h = ops.add_rmsnorm(x, delta, m.norm, m.cfg.eps)
        return m.lm_head(h if last is None else h.index_select(0, last))

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
                            budget: int | None = 512, page_size: int = 16, temperature: float = 0.0, draft: int = 0) -> dict:
    """Runs ``batch`` random prompts and ``tokens`` steps, or with ``draft`` as many
    as give every sequence that many tokens; returns tokens/s of the prompts and of
    the steps, and tokens a step of a sequence."""
    room = -(-(prompt + tokens) // page_size) + (0 if budget is None else -(-budget // page_size))
    server = PagedServer(model, batch * room, batch, page_size=page_size, budget=budget, temperature=temperature, draft=draft)
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
        made, steps, lines = 0, 0, {s: 0 for s in server.last}
        for _ in range(tokens if timed else 2):
            steps += len(server.last)
            for s, n in [(s, len(line)) for s, line in server.step_drafted().items()] if draft else [(s, 1) for s in server.step()]:
                made, lines[s] = made + n, lines[s] + n
                if draft and lines[s] >= tokens:
                    server.finish(s)
        t[2].record()
    torch.cuda.synchronize(model.device)
    return {"prompt_tokens_per_s": batch * prompt / t[0].elapsed_time(t[1]) * 1e3,
            "tokens_per_s": made / t[1].elapsed_time(t[2]) * 1e3, "tokens_per_step": made / steps}


if __name__ == "__main__":
    import argparse

    from .decoder import qwen25_7b

    ap = argparse.ArgumentParser(description="Prompts and steps over a paged cache (random weights).")
    for name, value in (("batch", 8), ("prompt", 700), ("tokens", 64), ("budget", 512), ("draft", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--temperature", type=float, default=0.0)
    args = ap.parse_args()
    decoder = SyntheticDecoder(qwen25_7b(max_len=args.prompt + args.tokens), "cuda:0", prefilled=0)
    print(serve_tokens_per_second(decoder, args.batch, args.prompt, args.tokens, budget=args.budget or None,
                                  temperature=args.temperature, draft=args.draft))
