"""Rotation of queries and keys by their positions (``csrc/rotary.cu``).

A pair ``(a, b)`` of a head at position ``p`` becomes ``(a cos - b sin, b cos + a sin)``, with cosine and
sine from row ``p`` of a table ``[positions, rotated / 2, 2]`` in fp32, in which the base, a stretched
context and a factor are.  Pairs are the halves of the rotated part of a head, or neighbours
(``interleaved``); what lies behind that part stays.  The rotation is computed in fp32 and rounded once; its
gradient is the transposed rotation, so that nothing is kept but the positions.
"""
from __future__ import annotations

import math

import torch
from torch import nn

from . import native


def rotary_table(rotary_dim, positions, base=10000.0, scaling=None, device=None):
    """Cosines and sines ``[positions, rotary_dim / 2, 2]`` in fp32, computed in fp64.

    ``scaling``, for contexts longer than the trained one: ``{"type": "linear", "factor": f}`` (positions
    divided by the factor), ``{"type": "ntk", "factor": f}`` (a larger base, so that the slowest pair is
    stretched by the factor and the fastest one not at all), or ``{"type": "yarn", "factor": f,
    "original_positions": n}`` (pairs that turn more than ``fast`` = 32 times in the trained context as they
    are, those that turn less than ``slow`` = 1 time stretched, a ramp between; cosine and sine times
    ``attention_factor`` = ``0.1 ln(factor) + 1``)."""
    if rotary_dim < 2 or rotary_dim % 2 or positions < 0:
        raise ValueError(f"an even number of rotated values and a number of positions required, not {rotary_dim} "
                         f"and {positions}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = base ** (-i / rotary_dim)
    factor = 1.0
    if scaling is not None:
        known = {"linear": {"type", "factor"}, "ntk": {"type", "factor"},
                 "yarn": {"type", "factor", "original_positions", "fast", "slow", "attention_factor"}}
        kind = scaling.get("type")
        if kind not in known or set(scaling) - known[kind] or not scaling.get("factor", 0) >= 1:
            raise ValueError(f"scaling: type 'linear', 'ntk' or 'yarn' with its values and a factor of 1 or more "
                             f"required, not {scaling}")
        by = float(scaling["factor"])
        if kind == "linear":
            freq = freq / by
        elif kind == "ntk":
            if rotary_dim == 2:
                raise ValueError("scaling 'ntk' needs more than one pair")
            freq = (base * by ** (rotary_dim / (rotary_dim - 2.0))) ** (-i / rotary_dim)
        else:
            trained = scaling.get("original_positions")
            if not trained or trained < 1:
                raise ValueError("scaling 'yarn' needs the trained context, original_positions")
            # the pair that turns so many times in the trained context
            low, high = (rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
                         for turns in (scaling.get("fast", 32.0), scaling.get("slow", 1.0)))
            low, high = max(math.floor(low), 0), min(math.ceil(high), rotary_dim - 1)
            ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
            freq = freq * (1.0 - ramp) + freq / by * ramp
            factor = scaling.get("attention_factor", 0.1 * math.log(by) + 1.0)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], -1) * factor).float().to(device)


def _check(q, k, table, positions):
    packed = k is None
    if q.dim() != (5 if packed else 4) or (packed and q.shape[3] != 3):
        raise ValueError(f"rotary: {'[B, S, H, 3, D]' if packed else '[B, S, H, D]'} required, not {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16, torch.float32, torch.float64):
        raise TypeError(f"rotary: bf16, fp16 or fp32 required, not {q.dtype}")
    if not packed:
        if k.dtype != q.dtype:
            raise TypeError("rotary: q and k of one type required")
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise ValueError(f"rotary: k [B, S, heads, D] of q's tokens and width required: {tuple(k.shape)} and "
                             f"{tuple(q.shape)}")
    if table.dtype != torch.float32:
        raise TypeError(f"rotary: a table of fp32 required, not {table.dtype}")
    if table.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary: the table has no gradient")
    if table.dim() != 3 or table.shape[2] != 2 or not 1 <= table.shape[1] <= q.shape[-1] // 2:
        raise ValueError(f"rotary: a table [positions, rotated / 2, 2] of at most the head's {q.shape[-1]} values "
                         f"required, not {tuple(table.shape)}")
    if torch.is_tensor(positions):
        if positions.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"rotary: positions of int64 or int32 required, not {positions.dtype}")
        if tuple(positions.shape) not in ((q.shape[1],), (1, q.shape[1]), (q.shape[0], q.shape[1])):
            raise ValueError(f"rotary: positions [S], [1, S] or [B, S] required, not {tuple(positions.shape)}")
    elif positions is not None and (isinstance(positions, bool) or not isinstance(positions, int)):
        raise TypeError(f"rotary: positions are a tensor, the first one's number or None, not {positions!r}")


def turn_reference(x, table, pos, interleaved):
    """``x [B, S, ..., D]`` rotated in fp32; ``pos [S]`` or ``[B, S]``.  Positions outside of the table:
    zeros."""
    pos = pos.long()
    known = (pos >= 0) & (pos < table.shape[0])
    if table.shape[0]:
        rows = table[torch.where(known, pos, torch.zeros_like(pos))]
    else:
        rows = table.new_zeros(*pos.shape, *table.shape[1:])
    shape = ((1,) if pos.dim() == 1 else ()) + tuple(pos.shape) + (1,) * (x.dim() - 3)
    cos, sin = (rows[..., j].reshape(shape + (table.shape[1],)) for j in (0, 1))
    known = known.reshape(shape + (1,))
    half = table.shape[1]
    y = x if x.dtype == torch.float64 else x.float()
    r, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        a, b = r[..., ::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    out = torch.cat([r, rest], -1)
    return torch.where(known, out, torch.zeros_like(out)).to(x.dtype)


def _positions(q, positions):
    if torch.is_tensor(positions):
        return positions
    start = positions or 0
    return torch.arange(start, start + q.shape[1], device=q.device)


def _rotary(q, k, table, positions, interleaved):
    if torch.is_tensor(q) and q.is_cuda:
        fn = native.direct("rotary")
        out = None if fn is None else fn(q, k, table, positions, interleaved)
        if out is not None:
            return out
    from . import functional as NF

    _check(q, k, table, positions)
    if NF._native_ok(q):
        tensor = torch.is_tensor(positions)
        return NF._nodes().rotary(q, k, table, positions if tensor else None, 0 if tensor else positions or 0,
                                  bool(interleaved))
    pos = _positions(q, positions)
    if k is None:
        turned = turn_reference(q[..., :2, :], table, pos, interleaved)
        return torch.cat([turned, q[..., 2:, :]], 3), None
    return turn_reference(q, table, pos, interleaved), turn_reference(k, table, pos, interleaved)


def rotary(q, k, table, positions=None, interleaved=False):
    """Queries ``[B, S, H, D]`` and keys ``[B, S, heads, D]`` rotated by their positions: two new tensors.

    ``table``: :func:`rotary_table`, of the rotated part of the head; ``positions``: those of the tokens,
    ``[S]``, ``[1, S]`` or ``[B, S]``, the first one's number, or None for 0, 1, ....  A token whose position lies
    outside of the table (padding: -1) gets zeros and no gradient."""
    return _rotary(q, k, table, positions, interleaved)


def rotary_qkvpacked(qkv, table, positions=None, interleaved=False):
    """:func:`rotary` on a packed projection ``[B, S, H, 3, D]``, whose values are copied: one new tensor, for
    attention on packed projections, and one gradient."""
    return _rotary(qkv, None, table, positions, interleaved)[0]


class RotaryEmbedding(nn.Module):
    """What :class:`~slapo_b200.ops.attention.FlashAttention` rotates its queries and keys by: a table of
    ``max_positions`` for the first ``rotary_dim`` values of a head (``base``, ``scaling``:
    :func:`rotary_table`).

    Tokens that follow one another - their first position is a number, or none is given - have to fit the table: more
    are refused.  Positions in a tensor are not looked at: outside of the table they give zeros
    (:func:`rotary`).

    The table is no parameter and no buffer: it stays in fp32 whatever the model is cast to, and is made on
    a device when that is first used (before a capture, as a model's first pass is)."""

    traceable = False

    def __init__(self, rotary_dim, max_positions, base=10000.0, interleaved=False, scaling=None):
        super().__init__()
        self.rotary_dim, self.max_positions = rotary_dim, max_positions
        self.base, self.interleaved, self.scaling = base, interleaved, scaling
        rotary_table(rotary_dim, 0, base, scaling)      # (refuses what it does not know)
        self._tables = {}

    def table(self, device):
        device = torch.device(device)
        if device not in self._tables:
            with torch.inference_mode(False):      # (a table of inference could not be kept for a gradient)
                self._tables[device] = rotary_table(self.rotary_dim, self.max_positions, self.base,
                                                    self.scaling, device)
        return self._tables[device]

    def __getstate__(self):
        return {**self.__dict__, "_tables": {}}

    def check_positions(self, tokens, what):
        """Refuses a sequence of more tokens than the table has positions."""
        if tokens > self.max_positions:
            raise ValueError(f"{what}: {tokens} tokens, a rotation of {self.max_positions} positions")

    def _check(self, x, positions):
        if x.dim() > 1 and x.shape[1] > 0 and (positions is None or isinstance(positions, int)):
            self.check_positions((positions or 0) + x.shape[1], "RotaryEmbedding")

    def forward(self, q, k, positions=None):
        self._check(q, positions)
        return rotary(q, k, self.table(q.device), positions, self.interleaved)

    def forward_packed(self, qkv, positions=None):
        self._check(qkv, positions)
        return rotary_qkvpacked(qkv, self.table(qkv.device), positions, self.interleaved)

    def extra_repr(self):
        scaling = "" if self.scaling is None else f", scaling={self.scaling}"
        return f"{self.rotary_dim}, {self.max_positions}, interleaved={self.interleaved}" + scaling
