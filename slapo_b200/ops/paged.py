"""A paged key / value cache in 8 bits, what appends to it and attention over it (``csrc/paged_append.cu``,
``csrc/paged_attn.cu``).

``pages [P, 2, H, T, W]`` of ``float8_e4m3fn``: for keys and values and each head the ``T`` tokens of a page
(16, 32, 64 or 128), ``W`` the head's width up to a multiple of 16.  ``scales [P, 2, H]`` in fp32: a power
of two for each page, side and head, the smallest with which the largest value fits (448 times it), at least
2^-100. ``block_table [B, pages]`` (int32) names a sequence's pages in their order, ``lengths [B]`` (int32)
counts its tokens, new ones among them.  Of ``n`` new tokens a sequence brings all, or the first
``counts[b]``: they are its last ones.

All of it is in device memory and read there, so that a captured step serves whatever it holds at a replay.
"""
from __future__ import annotations

import math

import torch

from . import native
from .rotary import turn_reference

PAGE_SIZES = (16, 32, 64, 128)
LARGEST = 448.0                # of e4m3
LEAST_EXPONENT = -100          # of a scale


def page_width(head_dim):
    """Values that a token of a head has in a page: a multiple of 16."""
    return (head_dim + 15) // 16 * 16


def _check(pages, scales, block_table, lengths, counts, x, what):
    if x.dim() != 4:
        raise ValueError(f"{what}: [B, n, heads, D] required, not {tuple(x.shape)}")
    if pages.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{what}: pages of float8_e4m3fn required, not {pages.dtype}")
    if scales.dtype != torch.float32:
        raise TypeError(f"{what}: scales of fp32 required, not {scales.dtype}")
    d = x.shape[3]
    if not (8 <= d <= 128 and d % 8 == 0):
        raise ValueError(f"{what}: heads of 8 to 128 values, a multiple of 8, required, not {d}")
    if pages.dim() != 5 or pages.shape[0] < 1 or pages.shape[1] != 2 or not pages.is_contiguous():
        raise ValueError(f"{what}: contiguous pages [pages, 2, heads, tokens, width] required, not {tuple(pages.shape)}")
    if pages.shape[3] not in PAGE_SIZES:
        raise ValueError(f"{what}: pages of {PAGE_SIZES} tokens required, not {pages.shape[3]}")
    if pages.shape[4] != page_width(d):
        raise ValueError(f"{what}: pages of {page_width(d)} values a token for heads of {d} required, not "
                         f"{pages.shape[4]}")
    if scales.shape != pages.shape[:3] or not scales.is_contiguous():
        raise ValueError(f"{what}: contiguous scales [pages, 2, heads] required, not {tuple(scales.shape)}")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError(f"{what}: block_table and lengths of int32 required")
    b = x.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != b or not block_table.is_contiguous():
        raise ValueError(f"{what}: a contiguous block_table [{b}, pages] required, not {tuple(block_table.shape)}")
    for name, t in (("lengths", lengths), ("counts", counts)):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError(f"{what}: {name} of int32 required, not {t.dtype}")
        if t.shape != (b,) or not t.is_contiguous():
            raise ValueError(f"{what}: contiguous {name} [{b}] required, not {tuple(t.shape)}")


def _check_no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


def _new_tokens(lengths, counts, n):
    """The new tokens of each sequence and the position of the first."""
    count = torch.full_like(lengths, n) if counts is None else counts.clamp(0, n)
    return count, lengths - count


def paged_append_reference(pages, scales, k, v, block_table, lengths, counts=None, q=None, rotary_table=None,
                           interleaved=False):
    """:func:`paged_append` in plain PyTorch (the oracle)."""
    b, n, _, d = k.shape
    t = pages.shape[3]
    count, start = _new_tokens(lengths.long(), counts, n)
    pos = start[:, None] + torch.arange(n, device=k.device)
    there = (torch.arange(n, device=k.device) < count[:, None]) & (pos >= 0)
    new_k, new_v, new_q = k.float(), v.float(), q
    if rotary_table is not None:
        new_k = turn_reference(new_k, rotary_table, pos, interleaved)
        new_q = None if q is None else turn_reference(q, rotary_table, pos, interleaved)
    if q is not None:
        new_q = torch.where(there[:, :, None, None], new_q, torch.zeros_like(new_q))
    finite = torch.finfo(torch.float32).max
    for i in range(b):
        first, end = max(int(start[i]), 0), int(start[i] + count[i])
        while first < end and first // t < block_table.shape[1]:
            last = min(end, (first // t + 1) * t)
            page, held = int(block_table[i, first // t]), first % t
            at = slice(first - int(start[i]), last - int(start[i]))
            if 0 <= page < pages.shape[0]:
                new = torch.stack([new_k[i, at], new_v[i, at]]).transpose(1, 2)         # [2, H, tokens, D]
                size = new.abs()
                top = torch.where(size <= finite, size, torch.zeros_like(size)).amax((2, 3))
                part, e = torch.frexp(top)
                e = torch.where(part <= 0.875, e - 9, e - 8).clamp(min=LEAST_EXPONENT)
                need = torch.exp2(torch.where(top == 0, LEAST_EXPONENT, e).float())
                scale = torch.maximum(scales[page], need) if held else need
                new = torch.where(size <= finite, new, float("nan")) / scale[..., None, None]
                if held:
                    old = pages[page, :, :, :held].float() * (scales[page] / scale)[..., None, None]
                    pages[page, :, :, :held] = old.to(pages.dtype)
                wide = torch.zeros(*new.shape[:3], pages.shape[4], device=new.device)
                wide[..., :d] = new
                pages[page, :, :, held:held + last - first] = wide.to(pages.dtype)
                scales[page] = scale
            first = last
    return new_q


def paged_append(pages, scales, k, v, block_table, lengths, counts=None, q=None, rotary_table=None,
                 interleaved=False):
    """New tokens' keys and values ``[B, n, H, D]`` (bf16, fp16 or fp32; slices of a packed projection are
    read in place) into the cache, in place; returns their queries, a new tensor (or None).

    ``rotary_table``: keys - and ``q [B, n, heads, D]`` - are rotated by their positions on the way
    (:func:`slapo_b200.ops.functional.rotary`); without one they stay as they are.  New tokens have
    positions ``lengths[b] - counts[b]`` on; those before position 0 (left padding), behind the block
    table's end or in a page that there is not are not kept, a query that is none (behind ``counts[b]``,
    before position 0) is zeros, and so are a query and a key behind the rotation's table.  A page takes
    tokens of one sequence: pages that several share have to be full.

    A value is off by at most 2^-4 of itself, or half of 2^-9 of its page's scale if it is small; values
    that are not finite are held as NaN.  A page's first token sets its scale anew; where a later one is too
    large for it, the page's codes are rounded to the larger scale."""
    if torch.is_tensor(k) and k.is_cuda:
        fn = native.direct("paged_append")
        out = None if fn is None else fn(pages, scales, k, v, block_table, lengths, counts, q, rotary_table, interleaved)
        if out is not None:
            return None if q is None else out
    from . import functional as NF
    from .rotary import _check as check_rotary

    _check(pages, scales, block_table, lengths, counts, k, "paged_append")
    if k.shape != v.shape or k.shape[2] != pages.shape[2]:
        raise ValueError(f"paged_append: k and v [B, n, {pages.shape[2]}, D] required, not {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"paged_append: k and v of bf16, fp16 or fp32 required, not {k.dtype} and {v.dtype}")
    if q is not None:
        if q.dtype != k.dtype:
            raise TypeError("paged_append: q of k's type required")
        if q.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
            raise ValueError(f"paged_append: q [B, n, heads, D] of k's tokens and width required: {tuple(q.shape)} "
                             f"and {tuple(k.shape)}")
    if rotary_table is not None:
        check_rotary(k, k, rotary_table, None)
    _check_no_gradient("paged_append", k, v, q)
    if NF._native_ok(k):
        out = NF._nodes().paged_append(pages, scales, k, v, block_table, lengths, counts, q, rotary_table,
                                       bool(interleaved))
        return None if q is None else out
    return paged_append_reference(pages, scales, k, v, block_table, lengths, counts, q, rotary_table, interleaved)


def paged_attention_reference(q, pages, scales, block_table, lengths, counts=None, scale=None, window=None):
    """:func:`paged_attention` in plain PyTorch (the oracle): fp32, or fp64 for queries in it."""
    b, n, h, d = q.shape
    kv, t = pages.shape[2], pages.shape[3]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    real = torch.float64 if q.dtype == torch.float64 else torch.float32
    count, start = _new_tokens(lengths.long(), counts, n)
    out = torch.zeros(b, n, h, d, dtype=real, device=q.device)
    for i in range(b):
        keys = min(max(int(lengths[i]), 0), block_table.shape[1] * t)
        ids = block_table[i, :(keys + t - 1) // t].long()
        known = (ids >= 0) & (ids < pages.shape[0])
        if not keys or not int(count[i]) or not bool(known.any()):
            continue
        at = torch.where(known, ids, torch.zeros_like(ids))
        got = pages[at].to(real) * scales[at].to(real)[..., None, None]
        got = torch.where(known[:, None, None, None, None], got, torch.zeros_like(got))
        k, v = got[..., :d].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, d)[:, :, :keys]
        pos = start[i] + torch.arange(n, device=q.device)
        key = torch.arange(keys, device=q.device)
        seen = (key <= pos[:, None]) & known.repeat_interleave(t)[:keys]
        if window is not None:
            seen = seen & (key > pos[:, None] - window)
        seen = seen & (torch.arange(n, device=q.device) < count[i])[:, None]            # [n, keys]
        x = torch.einsum("nhgd,hkd->hgnk", q[i].to(real).view(n, kv, h // kv, d), k) * scale
        x = x.masked_fill(~seen, -float("inf"))
        empty = ~seen.any(-1)[:, None]
        p = torch.softmax(x.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)
        out[i] = torch.einsum("hgnk,hkd->nhgd", p, v).reshape(n, h, d)
    return out.to(q.dtype)


def paged_attention(q, pages, scales, block_table, lengths, counts=None, scale=None, window=None):
    """Attention of the newest tokens' queries ``[B, n, heads, D]`` (bf16 or fp16) over the cache, which has
    their own keys already: causal, ``heads`` a multiple of the cache's, which its neighbours share.

    The query of new token ``t`` has position ``lengths[b] - counts[b] + t`` and sees the keys up to it,
    with a ``window`` that many.  A query without a key - behind ``counts[b]``, before position 0, in an
    empty sequence - has an output of 0; pages that there are not are not seen.  What is cached has to be
    finite.

    Keys are dealt out evenly over the GPU whatever the lengths; made for few tokens at a time (their keys
    are read again for every 32 rows of heads and tokens): a prompt's first tokens go through
    :func:`slapo_b200.ops.functional.flash_attention`.  fp32 queries run the PyTorch reference, which reads lengths
    on the host: not in a capture."""
    if window is not None and (isinstance(window, bool) or not isinstance(window, int) or window < 1):
        raise ValueError(f"a window is a number of keys, 1 and more, not {window!r}")
    if torch.is_tensor(q) and q.is_cuda:
        fn = native.direct("paged_attention")
        out = None if fn is None else fn(q, pages, scales, block_table, lengths, counts, scale, window)
        if out is not None:
            return out
    from . import functional as NF

    _check(pages, scales, block_table, lengths, counts, q, "paged_attention")
    if q.dtype not in (torch.bfloat16, torch.float16, torch.float32, torch.float64):
        raise TypeError(f"paged_attention: bf16 or fp16 required, not {q.dtype}")
    if q.shape[2] % pages.shape[2] if pages.shape[2] else q.shape[2]:
        raise ValueError(f"paged_attention: a multiple of the cache's {pages.shape[2]} heads required, not {q.shape[2]}")
    _check_no_gradient("paged_attention", q)
    if q.dtype in (torch.bfloat16, torch.float16) and NF._native_ok(q):
        return NF._nodes().paged_attention(q, pages, scales, block_table, lengths, counts, scale, window or 0)
    if q.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"paged_attention: {q.dtype} queries are not captured, bf16 and fp16 are")
    return paged_attention_reference(q, pages, scales, block_table, lengths, counts, scale, window)


class PagedKVCache:
    """Keys and values of ``layers`` attention layers for up to ``batch`` sequences of ``max_tokens`` in
    ``pages`` pages.

    A step: :meth:`add` makes room for the new tokens of each sequence, then every layer appends and attends
    (``FlashAttention(..., layer_past=cache.layer(i))``); :meth:`free` gives a sequence's pages back.  The
    tables on the device keep their addresses, and layers read from them how many tokens a sequence brings: their
    work can be captured and replayed after each :meth:`add`, of whatever kind, that brings a sequence at
    most as many tokens as the captured step is wide.  A captured step attends over the pages, a prompt's first
    tokens among it."""

    @torch.inference_mode(False)        # (tensors of inference could not be written outside of it)
    def __init__(self, layers, pages, heads, head_dim, batch, max_tokens, page=64, device=None):
        if page not in PAGE_SIZES:
            raise ValueError(f"pages of {PAGE_SIZES} tokens, not {page}")
        if not (8 <= head_dim <= 128 and head_dim % 8 == 0):
            raise ValueError(f"heads of 8 to 128 values, a multiple of 8, required, not {head_dim}")
        self.page, self.batch, self.max_tokens, self.head_dim = page, batch, max_tokens, head_dim
        shape = (pages, 2, heads, page, page_width(head_dim))
        self.pages = [torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device) for _ in range(layers)]
        self.scales = [torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(layers)]
        per = (max_tokens + page - 1) // page
        self.block_table = torch.full((batch, per), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._counts = torch.zeros(batch, dtype=torch.int32, device=device)     # of the step
        self._each = 0              # what all of them are, None: a list's
        self.counts = None          # of the step: None where each sequence brings all of its tokens
        self.fresh = False          # the step's tokens are the first ones of all sequences
        self.width = 0              # of the step: its most new tokens of a sequence
        self._tables = torch.full((batch, per), -1, dtype=torch.int32)      # the host's copies
        self._tokens = [0] * batch
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    def tokens(self, sequence):
        """Tokens of a sequence."""
        return self._tokens[sequence]

    def add(self, counts):
        """Room for a step's new tokens: the same number for every sequence, or a list of one for each (0:
        none in this step; the step's tensors are then as wide as the largest, right-padded).  Refused, with
        nothing changed, where pages or a sequence's ``max_tokens`` do not suffice."""
        each = [counts] * self.batch if isinstance(counts, int) else [int(c) for c in counts]
        if len(each) != self.batch or min(each, default=0) < 0:
            raise ValueError(f"a number of new tokens for each of {self.batch} sequences required, not {counts}")
        need = []
        for i, c in enumerate(each):
            if self._tokens[i] + c > self.max_tokens:
                raise ValueError(f"sequence {i} would have {self._tokens[i] + c} tokens of at most {self.max_tokens}")
            need.append((self._tokens[i] + c + self.page - 1) // self.page - len(self._owned[i]))
        if sum(need) > len(self._free):
            raise RuntimeError(f"the step needs {sum(need)} pages, {len(self._free)} are free")
        self.fresh, self.width = not any(self._tokens), max(each, default=0)
        for i, c in enumerate(each):
            for _ in range(need[i]):
                self._tables[i, len(self._owned[i])] = self._free[-1]
                self._owned[i].append(self._free.pop())
            self._tokens[i] += c
        if any(need):
            self.block_table.copy_(self._tables)
        if isinstance(counts, int):
            self.counts = None
            self.lengths.add_(counts)
            if self._each != counts:
                self._counts.fill_(counts)
                self._each = counts
        else:
            self.counts, self._each = self._counts, None
            both = torch.tensor([self._tokens, each], dtype=torch.int32).to(self.lengths.device)
            self.lengths.copy_(both[0])
            self._counts.copy_(both[1])

    def free(self, sequence):
        """A sequence's pages back to the others; it is empty then."""
        self._free.extend(reversed(self._owned[sequence]))
        self._owned[sequence] = []
        self._tokens[sequence] = 0
        self._tables[sequence] = -1
        self.block_table[sequence] = -1
        self.lengths[sequence] = 0

    def layer(self, index):
        """What attention layer ``index`` takes as its ``layer_past``."""
        return PagedLayer(self, index)


class PagedLayer:
    """One layer of a :class:`PagedKVCache`.  Its calls always pass the counts' tensor: a captured one has to serve steps
    in which sequences bring all of its tokens and others."""

    def __init__(self, cache, index):
        self.cache, self.index = cache, index

    @property
    def fresh(self):
        """Whether the step's tokens may attend over its own keys alone: the first ones of all sequences, and no
        capture, whose replays may come when sequences have others."""
        return self.cache.fresh and not (self.cache.lengths.is_cuda and torch.cuda.is_current_stream_capturing())

    def append(self, k, v, q=None, rotary_table=None, interleaved=False):
        """The step's keys and values; returns its queries, which stay as they are without a rotation."""
        c = self.cache
        if k.shape[:2] != (c.batch, c.width):
            raise ValueError(f"the step has room for {c.width} tokens of {c.batch} sequences, not {tuple(k.shape[:2])}")
        turned = paged_append(c.pages[self.index], c.scales[self.index], k, v, c.block_table, c.lengths, c._counts,
                              None if rotary_table is None else q, rotary_table, interleaved)
        return q if rotary_table is None else turned

    def attend(self, q, scale=None, window=None):
        c = self.cache
        return paged_attention(q, c.pages[self.index], c.scales[self.index], c.block_table, c.lengths, c._counts,
                               scale, window)
