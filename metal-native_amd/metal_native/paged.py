"""Serving from a paged key/value cache: rotary positions, attention, the
attention weight that keys gathered, eviction by it.  No reference counterpart.

Shapes, for all four operators:

* caches ``k_cache``, ``v_cache``: ``[pages, kv_heads, page_size, head_dim]``,
  Float16 or BFloat16, ``page_size`` a power of two from 8, ``head_dim`` 64 or
  128, unit stride along ``head_dim`` and 16-byte aligned slots, otherwise any
  strides (``kv[:, 0]`` and ``kv[:, 1]`` of one ``[pages, 2, ...]`` tensor);
* ``table`` int32 ``[batch, width]``: slot ``j`` of sequence ``s`` (its token at
  position ``j``) lies in page ``table[s, j // page_size]``;
* ``lens`` int32 ``[batch]``: slots per sequence, those of this call's tokens
  among them;
* ``cu`` int32 ``[batch + 1]``, not decreasing: the call's packed tokens
  ``cu[s]:cu[s + 1]`` are the newest of sequence ``s``; ``None``: one token per
  sequence.  Tokens before ``cu[0]`` or past ``cu[batch]`` (a batch padded for a
  graph) belong to no sequence: ``rope_kv`` turns their queries and writes no
  slot, ``attention`` gives zeros and -inf, ``attention_mass`` counts none.

The index tensors are device memory that no call looks at on the host, so a
step of a decode loop is capturable in a graph.  Whatever they hold, no kernel
leaves the tensors it was given: a slot whose page number is no page of the
cache does not exist (not written, not attended to), lengths past the table's
width are cut to it, positions past the rotary tables to their last row.

Every call launches HIP kernels of libmetal_native_amd.so on the current stream
and returns without synchronising; workspaces come from torch's allocator on
that stream.  None has a backward pass: where autograd follows an input, going
back through the outputs raises, and a cache that is written may not require a
gradient.
"""

from __future__ import annotations

import torch

from .ops import _check, _invalid, _mq_torch, _raw_stream, _require_cuda

__all__ = ["rope_kv", "attention", "attention_mass", "evict"]


def _plain(*tensors):
    """Tensors of other classes as ordinary ones over the same memory; anything else as it is."""
    odd = [isinstance(t, torch.Tensor) and type(t) not in (torch.Tensor, torch.nn.Parameter) for t in tensors]
    if not any(odd):
        return tensors
    with torch._C.DisableTorchFunctionSubclass():
        return tuple(t.as_subclass(torch.Tensor) if o else t for t, o in zip(tensors, odd))


def _cache(op, k, v, table, lens, keys_only=False):
    """Raises for what no kernel takes; returns table and lens as the kernels
    read them.  The caches themselves are never copied."""
    for t, what in ((k, "k_cache"), (v, "v_cache"), (table, "table"), (lens, "lens")):
        if keys_only and what == "v_cache":
            continue
        _require_cuda(t, what, op)
        if t.device != k.device:
            _invalid(f"{op}: {what} must be on the cache's device")
    for t, what in ((k, "k_cache"), (v, "v_cache")):
        if t is None:
            continue
        if t.dim() != 4 or t.numel() == 0:
            _invalid(f"{op}: {what} must be [pages, kv_heads, page_size, head_dim]")
        if t.dtype not in (torch.float16, torch.bfloat16) or t.dtype != k.dtype:
            _invalid(f"{op}: the caches must both be Float16 or both BFloat16")
        if t.shape != k.shape:
            _invalid(f"{op}: k_cache and v_cache must have the same shape")
        if t.stride(3) != 1 or t.data_ptr() % 16 or any(n > 1 and (s % 8 or s < 0) for n, s in zip(t.shape[:3], t.stride())):
            _invalid(f"{op}: {what} must have unit stride along head_dim and 16-byte aligned slots")
    ps, d = k.shape[2:]
    if d not in (64, 128):
        _invalid(f"{op}: head_dim must be 64 or 128, got {d}")
    if ps < 8 or ps > 65536 or ps & (ps - 1):
        _invalid(f"{op}: page_size must be a power of two from 8 to 65536, got {ps}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.numel() == 0:
        _invalid(f"{op}: table must be Int32 [batch, width]")
    if lens.dtype != torch.int32 or tuple(lens.shape) != (table.shape[0],):
        _invalid(f"{op}: lens must be Int32 [batch] = [{table.shape[0]}]")
    return table.contiguous(), lens.contiguous()


def _chunks(op, cu, table, rows):
    if cu is None:
        if rows != table.shape[0]:
            _invalid(f"{op}: without cu there must be one row per sequence ({table.shape[0]}), got {rows}")
        return None
    _require_cuda(cu, "cu", op)
    if cu.dtype != torch.int32 or tuple(cu.shape) != (table.shape[0] + 1,) or cu.device != table.device:
        _invalid(f"{op}: cu must be Int32 [batch + 1] = [{table.shape[0] + 1}] on the cache's device")
    return cu.contiguous()


class _NoGradient(torch.autograd.Function):
    """Outputs that autograd refuses to go back through."""

    @staticmethod
    def forward(ctx, op, out, *inputs):
        ctx.op = op
        return out

    @staticmethod
    def backward(ctx, *grads):
        _invalid(f"{ctx.op}: has no backward pass (call it under torch.no_grad(), or detach what goes in)")


def _tracked(op, read, written=()):
    """The inputs that autograd follows; raises where one of them is written."""
    if not torch.is_grad_enabled():
        return []
    for t in written:
        if t.requires_grad:
            _invalid(f"{op}: a cache that requires a gradient is written in place (call it under torch.no_grad())")
    return [t for t in read if isinstance(t, torch.Tensor) and t.requires_grad]


def _finish(op, r, tracked=()):
    if r is None:
        _invalid(f"{op}: arguments not supported (memory overlaps, strides out of range, or a tensor without memory of its own)")
    if type(r) is int:
        _check(r)
    return _NoGradient.apply(op, r, *tracked) if tracked else r


def rope_kv(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, k_cache: torch.Tensor,
            v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, cu: torch.Tensor | None = None, *,
            sections=None) -> torch.Tensor:
    """Rotary positions for fused rows ``qkv [rows, (heads + 2 kv_heads) *
    head_dim]``: returns q turned, ``[rows, heads, head_dim]``, and writes k
    (turned) and v into the slots of their tokens.

    ``cos``, ``sin``: fp32 ``[positions, head_dim]`` as ``rope_tables`` makes
    them (rotate-half: frequency f turns elements f and f + head_dim / 2; the
    second half of the columns is not read).  ``pos``: int64 ``[rows]``, the row
    of the tables, or ``[axes, rows]`` with ``sections``, the number of
    frequencies that each axis (time, height, width) turns, in order.
    """
    op = "paged.rope_kv"
    if sections is not None and (type(sections) is not tuple or any(type(n) is not int for n in sections)):
        given, sections = tuple(sections), tuple(int(n) for n in sections)
        if given != sections:
            _invalid(f"{op}: sections must be whole numbers, got {given}")
    if type(qkv) is torch.Tensor and qkv.is_cuda:
        r = _mq_torch.paged_rope_kv(qkv, cos, sin, pos, k_cache, v_cache, table, lens, cu, sections,
                                    _raw_stream(qkv.get_device()))
        if r is not None:
            return _finish(op, r)
    qkv, cos, sin, pos, k_cache, v_cache, table, lens, cu = _plain(qkv, cos, sin, pos, k_cache, v_cache, table, lens, cu)
    table, lens = _cache(op, k_cache, v_cache, table, lens)
    kvh, d = k_cache.shape[1], k_cache.shape[3]
    for t, what in ((qkv, "qkv"), (cos, "cos"), (sin, "sin"), (pos, "pos")):
        _require_cuda(t, what, op)
        if t.device != k_cache.device:
            _invalid(f"{op}: {what} must be on the cache's device")
    if qkv.dtype != k_cache.dtype or qkv.dim() != 2 or qkv.shape[1] % d or qkv.shape[1] // d <= 2 * kvh \
            or (qkv.shape[1] // d) % kvh:
        _invalid(f"{op}: qkv must be [rows, (heads + 2 kv_heads) * head_dim] of the cache's type")
    for t, what in ((cos, "cos"), (sin, "sin")):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != d or t.shape[0] < 1 or t.shape != cos.shape:
            _invalid(f"{op}: {what} must be Float32 [positions, head_dim]")
    rows, axes = qkv.shape[0], 1 if sections is None else len(sections)
    if sections is not None and (not 1 <= axes <= 8 or min(sections) < 0 or sum(sections) != d // 2):
        _invalid(f"{op}: sections must be one to eight numbers of frequencies that add up to head_dim / 2")
    if pos.dtype != torch.int64 or tuple(pos.shape) not in (((axes, rows), (rows,)) if axes == 1 else ((axes, rows),)):
        _invalid(f"{op}: pos must be Int64 [rows], or [axes, rows] with sections")
    cu = _chunks(op, cu, table, rows)
    tracked = _tracked(op, (qkv, cos, sin), (k_cache, v_cache))
    with torch.no_grad(), torch.cuda.device(qkv.device):
        for copied in (False, True):   # as they are, then laid out anew
            if copied:
                qkv, cos, sin, pos = (t.clone(memory_format=torch.contiguous_format) for t in (qkv, cos, sin, pos))
            r = _mq_torch.paged_rope_kv(qkv, cos, sin, pos, k_cache, v_cache, table, lens, cu, sections,
                                        _raw_stream(qkv.get_device()))
            if r is not None:
                break
    return _finish(op, r, tracked)


def _mask(op, q, k_cache, table, cu, scale, softcap, slopes, window, prefix_lens, max_q):
    """Checks of the queries and the mask; the tensors as the kernels read them."""
    _require_cuda(q, "q", op)
    kvh, d = k_cache.shape[1], k_cache.shape[3]
    if q.device != k_cache.device or q.dtype != k_cache.dtype or q.dim() != 3 or q.shape[2] != d or q.shape[1] < 1 \
            or q.shape[1] % kvh:
        _invalid(f"{op}: q must be [rows, heads, head_dim] of the cache's type and device, heads a multiple of kv_heads")
    cu = _chunks(op, cu, table, q.shape[0])
    if slopes is not None:
        _require_cuda(slopes, "slopes", op)
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (q.shape[1],) or slopes.device != q.device:
            _invalid(f"{op}: slopes must be Float32 [heads] = [{q.shape[1]}]")
        slopes = slopes.contiguous()
    if prefix_lens is not None:
        _require_cuda(prefix_lens, "prefix_lens", op)
        if prefix_lens.dtype != torch.int32 or tuple(prefix_lens.shape) != (table.shape[0],) or prefix_lens.device != q.device:
            _invalid(f"{op}: prefix_lens must be Int32 [batch] = [{table.shape[0]}]")
        prefix_lens = prefix_lens.contiguous()
    return cu, float(scale), float(softcap), slopes, int(window), prefix_lens, int(max_q)


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
              cu: torch.Tensor | None = None, *, scale: float | None = None, softcap: float = 0.0,
              slopes: torch.Tensor | None = None, window: int = 0, prefix_lens: torch.Tensor | None = None,
              max_q: int | None = None, return_lse: bool = False):
    """Attention of the newest tokens ``q [rows, heads, head_dim]`` over the
    cache, their own keys and values included: ``[rows, heads, head_dim]``, with
    ``return_lse`` also the log of each row's exponential sum, fp32 ``[rows,
    heads]``.

    Scores are ``scale * q . k`` (``scale`` default ``head_dim ** -0.5``), capped
    to ``softcap * tanh(x / softcap)`` where ``softcap`` is not 0, less ``slopes
    [heads] * distance``.  A row at position p sees slot j where ``j <= p``, with
    a ``window`` only the last ``window`` of those, and always the first
    ``prefix_lens [batch]`` slots.  A row that sees nothing gives zeros and -inf.
    Sums and log sums are held in 32 bits; the weights are rounded to the cache's
    type for their product with the values (half a step of it, next to the
    output's own rounding), and an infinite value under a weight that rounds to
    zero gives NaN where a whole tile of slots is seen.
    ``max_q``: the longest chunk where it is known (it sizes launches, no more).
    """
    op = "paged.attention"
    if scale is None:
        scale = q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    if max_q is None:
        max_q = 0
    if type(q) is torch.Tensor and q.is_cuda:
        r = _mq_torch.paged_attention(q, k_cache, v_cache, table, lens, cu, scale, softcap, slopes, window, prefix_lens,
                                      max_q, return_lse, _raw_stream(q.get_device()))
        if r is not None:
            return _finish(op, r)
    q, k_cache, v_cache, table, lens, cu, slopes, prefix_lens = _plain(q, k_cache, v_cache, table, lens, cu, slopes, prefix_lens)
    table, lens = _cache(op, k_cache, v_cache, table, lens)
    tracked = _tracked(op, (q, k_cache, v_cache, slopes))
    how = _mask(op, q, k_cache, table, cu, scale, softcap, slopes, window, prefix_lens, max_q)
    with torch.no_grad(), torch.cuda.device(q.device):
        for copied in (False, True):   # as it is, then laid out anew
            r = _mq_torch.paged_attention(q.clone(memory_format=torch.contiguous_format) if copied else q, k_cache, v_cache,
                                          table, lens, *how, bool(return_lse), _raw_stream(q.get_device()))
            if r is not None:
                break
    return _finish(op, r, tracked)


def attention_mass(q: torch.Tensor, k_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, lse: torch.Tensor,
                   cu: torch.Tensor | None = None, *, scale: float | None = None, softcap: float = 0.0,
                   slopes: torch.Tensor | None = None, window: int = 0, prefix_lens: torch.Tensor | None = None,
                   max_q: int | None = None) -> torch.Tensor:
    """The attention weight that every slot got from these rows: fp32 ``[batch,
    kv_heads, width * page_size]``, the sum of ``exp(x - lse)`` over the
    sequence's tokens of this call and the query heads that share the key/value
    head, zero past ``lens``.  ``lse`` is what ``attention`` returned for the
    same arguments; rows of ``-inf`` add nothing.  What ``evict`` takes is the
    running sum of these.
    """
    op = "paged.attention_mass"
    if scale is None:
        scale = q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0
    if max_q is None:
        max_q = 0
    if type(q) is torch.Tensor and q.is_cuda:
        r = _mq_torch.paged_attention_mass(q, k_cache, table, lens, lse, cu, scale, softcap, slopes, window, prefix_lens,
                                           max_q, _raw_stream(q.get_device()))
        if r is not None:
            return _finish(op, r)
    q, k_cache, table, lens, lse, cu, slopes, prefix_lens = _plain(q, k_cache, table, lens, lse, cu, slopes, prefix_lens)
    table, lens = _cache(op, k_cache, None, table, lens, keys_only=True)
    tracked = _tracked(op, (q, k_cache, lse, slopes))
    how = _mask(op, q, k_cache, table, cu, scale, softcap, slopes, window, prefix_lens, max_q)
    _require_cuda(lse, "lse", op)
    if lse.dtype != torch.float32 or tuple(lse.shape) != tuple(q.shape[:2]) or lse.device != q.device:
        _invalid(f"{op}: lse must be Float32 [rows, heads] = {list(q.shape[:2])}")
    with torch.no_grad(), torch.cuda.device(q.device):
        for copied in (False, True):
            r = _mq_torch.paged_attention_mass(q.clone(memory_format=torch.contiguous_format) if copied else q, k_cache, table, lens,
                                               lse.contiguous(), *how, _raw_stream(q.get_device()))
            if r is not None:
                break
    return _finish(op, r, tracked)


def evict(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, mass: torch.Tensor,
          to: torch.Tensor, budget: int, *, recent: int = 0):
    """Cut every sequence to ``budget`` slots per key/value head: the newest
    ``recent`` and, of the older, those of largest ``mass`` (fp32 ``[batch,
    kv_heads, width * page_size]``; NaN above all, ties to the lowest slot),
    moved in their order to the pages ``to`` (int32 ``[batch, pages]``), none of
    which may be a page of ``table``.  A sequence within the budget moves whole.

    Returns ``(kept, lens, mass)``: the slots that stay, int32 ``[batch, kv_heads,
    budget]``, -1 past the sequence's end; the new lengths; and the mass of what
    stayed, fp32 ``[batch, kv_heads, to.shape[1] * page_size]``, zero past it.
    Slot numbers no longer are positions afterwards, and a head's slot j is no
    longer another's: causal attention of single tokens and of chunks over the
    shortened cache stays right (every slot is older than the new tokens),
    windows, prefixes and distance biases do not.
    """
    op = "paged.evict"
    if type(k_cache) is torch.Tensor and k_cache.is_cuda:
        r = _mq_torch.paged_evict(k_cache, v_cache, table, lens, mass, to, budget, recent,
                                  _raw_stream(k_cache.get_device()))
        if r is not None:
            return _finish(op, r)
    k_cache, v_cache, table, lens, mass, to = _plain(k_cache, v_cache, table, lens, mass, to)
    table, lens = _cache(op, k_cache, v_cache, table, lens)
    b, kvh, ps = table.shape[0], k_cache.shape[1], k_cache.shape[2]
    for t, what in ((mass, "mass"), (to, "to")):
        _require_cuda(t, what, op)
        if t.device != k_cache.device:
            _invalid(f"{op}: {what} must be on the cache's device")
    if mass.dtype != torch.float32 or tuple(mass.shape) != (b, kvh, table.shape[1] * ps):
        _invalid(f"{op}: mass must be Float32 [batch, kv_heads, width * page_size] = [{b}, {kvh}, {table.shape[1] * ps}]")
    if to.dtype != torch.int32 or to.dim() != 2 or to.shape[0] != b:
        _invalid(f"{op}: to must be Int32 [batch, pages]")
    budget, recent = int(budget), int(recent)
    if not (budget >= 1 and 0 <= recent <= budget):
        _invalid(f"{op}: budget must be positive and recent 0 .. budget, got {budget} and {recent}")
    if to.shape[1] * ps < budget:
        _invalid(f"{op}: {to.shape[1]} pages of {ps} slots cannot hold {budget}")
    tracked = _tracked(op, (mass,), (k_cache, v_cache))
    with torch.no_grad(), torch.cuda.device(k_cache.device):
        r = _mq_torch.paged_evict(k_cache, v_cache, table, lens, mass.contiguous(), to.contiguous(), budget, recent,
                                  _raw_stream(k_cache.get_device()))
    return _finish(op, r, tracked)
