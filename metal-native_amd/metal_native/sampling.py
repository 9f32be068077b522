"""Drawing tokens from logits by given random numbers.  No reference counterpart.

The call launches HIP kernels of libmetal_native_amd.so on the current stream
and returns without synchronising; workspaces come from torch's allocator on
that stream, and no tensor is looked at on the host, so a step of a decode loop
is capturable in a graph.  There is no derivative: where autograd follows an
input, going back through the outputs raises, and log shares refuse tangents of
forward mode.
"""

from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual

from .ops import _invalid, _mq_torch, _raw_stream, _require_cuda
from .paged import _dual, _finish, _plain, _tracked

__all__ = ["sample"]


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprob: bool = False):
    """One token for each row of ``logits [rows, vocab]`` (Float16, BFloat16 or
    Float32): int64 ``[rows]``, with ``return_logprob`` also the log of its share
    among the tokens it was drawn from, fp32 ``[rows]``.

    Tokens have weights ``exp((logit - largest) / temperature)`` and an order, the
    largest logit first and ties by index.  Of it stay the first ``top_k`` (0 or
    less: all), of those the ones before which less than ``top_p`` of their sum
    has gone (1 or more: all; 0 or less: the first), of those the ones of weight
    at least ``min_p`` (of 1 where it is more).  ``u`` (fp32 ``[rows]``, uniform in [0, 1); what lies
    outside is cut to it) picks, in order of index, the first of them with which
    their running sum passes ``u`` times their sum: the same call gives the same
    tokens on every run, and what else is in the batch does not matter to a row, but
    for a cut by ``top_p`` that falls within the rounding of its sums.

    Each setting is a number, or a tensor ``[rows]`` (fp32; int32 for ``top_k``).  A
    temperature of 0 or less takes the first token; a NaN is such a temperature, and
    as another setting cuts nothing.  NaN logits count as -inf,
    which is never drawn; of infinite ones each counts as much as another.  A row
    with nothing above -inf gives token -1 and -inf.

    Weights and their sums are held in 64 bits: a token is right or wrong, and rows
    of 150 thousand have as many borders between two of them.  What is drawn goes by
    whole multiples of a unit, and tokens of less than half of one are never drawn: of
    2^-44 of the largest weight up to 2^18 tokens, 2^-40 at 2^22, and of 2^-50 where
    ``top_k`` leaves at most 512 (and 32 for each 1024 of the vocabulary).

    A row with very many equal logits at a cut is slow (152064 tokens 0.8 to 1 ms where 15 to
    40 us are usual): mask tokens with -inf, not with the type's lowest value.
    """
    op = "sampling.sample"
    if type(logits) is torch.Tensor and logits.is_cuda:
        r = _mq_torch.sample(logits, u, temperature, top_k, top_p, min_p, return_logprob, _raw_stream(logits.get_device()))
        if r is not None:
            return _finish(op, r)
    logits, u, temperature, top_k, top_p, min_p = _plain(logits, u, temperature, top_k, top_p, min_p)
    _require_cuda(logits, "logits", op)
    if logits.dtype not in (torch.float16, torch.bfloat16, torch.float32) or logits.dim() != 2 or not 1 <= logits.shape[1] <= 2**22:
        _invalid(f"{op}: logits must be Float16, BFloat16 or Float32 [rows, vocab], the vocabulary 1 to 2^22")
    rows = logits.shape[0]
    _require_cuda(u, "u", op)
    if u.dtype != torch.float32 or tuple(u.shape) != (rows,) or u.device != logits.device:
        _invalid(f"{op}: u must be Float32 [rows] = [{rows}] on the logits' device")
    given = []
    for x, what in ((temperature, "temperature"), (top_k, "top_k"), (top_p, "top_p"), (min_p, "min_p")):
        if isinstance(x, torch.Tensor):
            _require_cuda(x, what, op)
            dtype = torch.int32 if what == "top_k" else torch.float32
            if x.dtype != dtype or tuple(x.shape) != (rows,) or x.device != logits.device:
                _invalid(f"{op}: {what} must be a number, or {'Int32' if what == 'top_k' else 'Float32'} [rows] = [{rows}] on the logits' device")
            x = x.contiguous()
        else:
            try:
                if what == "top_k":
                    if int(x) != x:
                        _invalid(f"{op}: top_k must be a whole number, got {x}")
                    x = min(max(int(x), 0), 2**31 - 1)   # past any vocabulary
                else:
                    x = float(x)
            except (TypeError, ValueError, OverflowError):
                _invalid(f"{op}: {what} must be a number or a tensor, got {x!r}")
        given.append(x)
    if not return_logprob:   # a token has no tangent to lose
        logits, u, *given = (unpack_dual(x).primal if _dual(x) else x for x in (logits, u, *given))
    tracked = _tracked(op, (logits, u, *given))
    with torch.no_grad(), torch.cuda.device(logits.device):
        for copied in (False, True):   # as it is, then laid out anew
            r = _mq_torch.sample(logits.clone(memory_format=torch.contiguous_format) if copied else logits, u.contiguous(), *given,
                                 bool(return_logprob), _raw_stream(logits.get_device()))
            if r is not None:
                break
    return _finish(op, r, tracked)
