"""The next token of each row of logits, from given random numbers (``csrc/sample.cu``)."""
from __future__ import annotations

import math
import numbers
import operator

import torch

from . import native

MAX_VOCAB = 1 << 18
UNIT = 2.0 ** 42            # weights are multiples of 1 / UNIT of the largest one's


def _whole(top_k):
    """A number of tokens as an int: a float of one is taken."""
    try:
        return operator.index(top_k)
    except TypeError:
        if not isinstance(top_k, numbers.Real):
            raise TypeError(f"sample: top_k is a number of tokens, not {top_k!r}") from None
    if not top_k >= 0:
        raise ValueError(f"sample: top_k of 0 or more required, not {top_k}")
    if math.isinf(top_k) or top_k != int(top_k):
        raise TypeError(f"sample: top_k is a number of tokens, not {top_k}")
    return int(top_k)


def _check(logits, uniform, settings):
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"sample: logits [..., vocabulary] of 1 to {MAX_VOCAB} tokens required, not "
                         f"{tuple(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"sample: bf16, fp16 or fp32 required, not {logits.dtype}")
    if uniform.dtype != torch.float32:
        raise TypeError(f"sample: random numbers of fp32 required, not {uniform.dtype}")
    rows = logits.numel() // logits.shape[-1]
    if uniform.numel() != rows:
        raise ValueError(f"sample: one random number for each of the {rows} rows required, not {tuple(uniform.shape)}")
    for name, (value, dtype, most) in settings.items():
        if torch.is_tensor(value):
            if value.dtype != dtype:
                raise TypeError(f"sample: {name} of {dtype} required, not {value.dtype}")
            if value.numel() != rows:
                raise ValueError(f"sample: one {name} for each of the {rows} rows required")
        elif not (value >= 0 and (most is None or value <= most)):
            raise ValueError(f"sample: {name} of 0 or more{'' if most is None else ' and at most 1'} required, "
                             f"not {value}")


def sample_reference(logits, uniform, temperature, top_k, top_p, min_p):
    """:func:`sample` by sorting, weights in fp64 (the oracle)."""
    x = logits.detach().float().reshape(-1, logits.shape[-1])
    b, vocab = x.shape
    x = torch.where(x > -float("inf"), x, -float("inf"))        # (NaN: not there)

    def each(v, dtype):
        if torch.is_tensor(v):
            return v.reshape(b, 1).to(dtype)
        if dtype == torch.float64:          # (a number of the kernel's width)
            v = float(torch.tensor(v, dtype=torch.float32))
        return torch.full((b, 1), v, dtype=dtype, device=x.device)

    temperature, top_p, min_p = (each(v, torch.float64) for v in (temperature, top_p, min_p))
    top_k = each(top_k, torch.int64)
    min_p = torch.fmin(min_p, torch.ones_like(min_p))        # (the largest is kept, and its equals)
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    there = value > -float("inf")
    value = value.double()
    gap = torch.where(value == value[:, :1], 0.0, value - value[:, :1])
    greedy = ~(temperature > 0) | (top_k == 1)
    share = torch.where(there, torch.exp(gap / torch.where(greedy, 1.0, temperature)), 0.0)
    rank = torch.arange(vocab, device=x.device)
    w = torch.where((rank < top_k) | (top_k <= 0), (share * UNIT).round().long(), 0)
    before = w.cumsum(1) - w
    limit = torch.ceil(top_p * w.sum(1, keepdim=True)).long().clamp(min=1)
    keep = ((before < limit) | ~(top_p < 1.0)) & (share >= min_p)
    keep = torch.where(greedy, rank == 0, keep | (rank == 0)) & there
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0))
    total = kept.cumsum(1)
    target = torch.floor(uniform.reshape(b, 1).double().clamp(min=0.0) * total[:, -1:]).long()
    token = (total <= torch.minimum(target, total[:, -1:] - 1)).sum(1)
    return torch.where(there[:, 0], token, -1).reshape(logits.shape[:-1])


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The next token of each row of ``logits [..., vocabulary]``, int64 ``[...]``.

    Of the logits over ``temperature`` the ``top_k`` largest are kept (0: all; equals in the order of their
    indices), of these the shortest beginning of their order that holds a share ``top_p`` of their mass, of
    these what has at least ``min_p`` times the largest one's probability.  ``uniform``: a random number in
    [0, 1) for each row, fp32; the token is the first one kept, in the order of indices, at which the sum of
    probabilities passes it.  Temperature 0 takes the largest, the first of equals.

    Each setting is one number, or a tensor of one for each row (fp32; ``top_k`` int32).  A logit of -inf or
    NaN is no token; a row of nothing else gives -1.  Weights are computed in fp64 and held as multiples of
    2^-42 of the largest one's, their sums are exact: the same call gives the same token."""
    if type(top_k) is not int and not torch.is_tensor(top_k):
        top_k = _whole(top_k)
    if torch.is_tensor(logits) and logits.is_cuda:
        fn = native.direct("sample")
        out = None if fn is None else fn(logits, uniform, temperature, top_k, top_p, min_p)
        if out is not None:
            return out
    settings = {"temperature": (temperature, torch.float32, None), "top_k": (top_k, torch.int32, None),
                "top_p": (top_p, torch.float32, 1.0), "min_p": (min_p, torch.float32, 1.0)}
    _check(logits, uniform, settings)
    from . import functional as NF

    if NF._native_ok(logits):
        args = []
        for value, dtype, _ in settings.values():
            tensor = torch.is_tensor(value)
            args += [0 if tensor else value, value if tensor else None]
        return NF._nodes().sample(logits, uniform, *args)
    return sample_reference(logits, uniform, temperature, top_k, top_p, min_p)
