"""Rotation by positions, the paged 8-bit cache, attention over it and sampling on the GPU, against 64
bits."""
import math

import pytest
import torch

from slapo_b200.op import FlashAttention, PagedKVCache, RotaryEmbedding
from slapo_b200.ops import functional as NF
from slapo_b200.ops import native
from slapo_b200.ops.paged import paged_attention_reference
from slapo_b200.ops.sampling import sample_reference
from test_generation_cpu import (CHUNKS, append_case, make_cache, paged_refusals,
                                 rotary_refusals, sample_refusals, turned)

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


# ---------------------------------------------------------------------- #
# refusals first: nothing is launched
@pytest.mark.parametrize("which,index", [(0, i) for i in range(15)] + [(1, i) for i in range(41)]
                         + [(2, i) for i in range(14)])
def test_refusals(which, index):
    error, call = list((rotary_refusals, paged_refusals, sample_refusals)[which]("cuda"))[index]
    with pytest.raises(error):
        call()


def test_operands_on_the_host_are_refused():
    table = NF.rotary_table(8, 4, device="cuda")
    q = torch.zeros(1, 2, 1, 8, device="cuda", dtype=torch.float16)
    for call in (lambda: NF.rotary(q, q.cpu(), table), lambda: NF.rotary(q, q, table.cpu()),
                 lambda: NF.rotary(q, q, table, torch.zeros(2, dtype=torch.long)),
                 lambda: NF.sample(torch.zeros(1, 4, device="cuda"), torch.zeros(1)),
                 lambda: NF.sample(torch.zeros(1, 4, device="cuda"), torch.zeros(1, device="cuda"),
                         torch.ones(1))):
        with pytest.raises(ValueError, match="must be on"):
            call()
    pages, scales, tab = make_cache(1, 1, 1, 8, 16, "cuda")
    lengths = torch.ones(1, dtype=torch.int32, device="cuda")
    for i in range(4):
        args = [pages, scales, tab, lengths]
        args[i] = args[i].cpu()
        with pytest.raises(ValueError, match="must be on"):
            NF.paged_append(args[0], args[1], q, q, args[2], args[3])
        with pytest.raises(ValueError, match="must be on"):
            NF.paged_attention(q, args[0], args[1], args[2], args[3])


def test_transforms_are_refused():
    table = NF.rotary_table(8, 4, device="cuda")
    q = torch.zeros(3, 1, 2, 1, 8, device="cuda")
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: NF.rotary(x, x, table)[0])(q)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: NF.sample(x, torch.zeros(2, device="cuda")))(q[:, 0, :, 0])


# ---------------------------------------------------------------------- #
# rotation
def _rotation_bound(x, want, half):
    """Two products and a sum in fp32, then one rounding (below the type's normal numbers its steps stay)."""
    size = x.double().abs().amax(-1, keepdim=True)
    return want.abs() * half * (1 + 2.0 ** -10) + size * 4 * 2.0 ** -24 + 2.0 ** -24 * half


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,s,heads,kv,dim,rotated", [(1, 1, 1, 1, 2, 2), (2, 3, 5, 1, 8, 8), (3, 17, 16,
        16, 128, 128),
                                                      (2, 33, 8, 2, 80, 40), (1, 100, 3, 3, 72, 72), (1, 5,
                                                              2, 1, 256, 256),
                                                      (2, 7, 40, 8, 96, 20), (1, 9, 300, 1, 24, 10), (5, 2,
                                                              4, 4, 7, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation(b, s, heads, kv, dim, rotated, interleaved, dtype):
    table = NF.rotary_table(rotated, 500, device="cuda")
    q = torch.randn(b, s, heads, dim, device="cuda").to(dtype).requires_grad_()
    k = torch.randn(b, s, kv, dim, device="cuda").to(dtype).requires_grad_()
    pos = torch.randint(0, 500, (b, s), device="cuda")
    half = HALF[dtype]
    for at in (None, 7, pos, pos[0].int()):
        where = torch.arange(s, device="cuda") + (at or 0) if not torch.is_tensor(at) else at.long()
        got = NF.rotary(q, k, table, at, interleaved)
        want = [turned(x.detach(), table, where, interleaved) for x in (q, k)]
        for x, y, z in zip((q, k), got, want):
            assert y.dtype == dtype and y.is_contiguous()
            assert bool(((y.detach().double() - z).abs() <= _rotation_bound(x.detach(), z, half)).all())
        # the gradient: <dy, R x> = <R^T dy, x> as R^T is the rotation by the table with its sines negated
        dy = [torch.randn_like(y) for y in got]
        dx = torch.autograd.grad(got, (q, k), dy)
        back = table * torch.tensor([1.0, -1.0], device="cuda")
        for g, y in zip(dx, dy):
            z = turned(y, back, where, interleaved)
            assert bool(((g.double() - z).abs() <= _rotation_bound(y, z, half)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,s,heads,dim,rotated", [(1, 1, 1, 16, 16), (2, 50, 12, 64, 64), (1, 33, 4, 80,
        40), (2, 5, 3, 10, 4)])
def test_packed_rotation(b, s, heads, dim, rotated, dtype):
    table = NF.rotary_table(rotated, 100, device="cuda")
    qkv = torch.randn(b, s, heads, 3, dim, device="cuda").to(dtype).requires_grad_()
    got = NF.rotary_qkvpacked(qkv, table, 5)
    q, k = NF.rotary(qkv[..., 0, :], qkv[..., 1, :], table, 5)
    assert torch.equal(got, torch.stack([q, k, qkv[..., 2, :]], 3)) and got.is_contiguous()
    dy = torch.randn_like(got)
    dx = torch.autograd.grad(got, qkv, dy)[0]
    dq, dk = torch.autograd.grad((q, k), qkv, (dy[..., 0, :], dy[..., 1, :]))[0].unbind(3)[:2]
    assert torch.equal(dx, torch.stack([dq, dk, dy[..., 2, :]], 3))


def test_rotation_strides_and_second_derivatives():
    table = NF.rotary_table(16, 64, device="cuda")
    base = torch.randn(3, 40, 6, 24, device="cuda")
    for view in (base, base.transpose(0, 1), base[:, ::3], base[:, :, ::2], base.flip(1), base[..., 3:19],
            base[..., 4:20],
                 base.expand(2, 3, 40, 6, 24)[:, 0], base.transpose(2, 3)[:, :,
                         :16].contiguous().transpose(2, 3)):
        for x in (view, view.bfloat16() if view is base else view):
            got = NF.rotary(x, x[:, :, :1], table, 2)
            assert torch.equal(got[0], NF.rotary(x.contiguous(), x[:, :, :1].contiguous(), table, 2)[0])
            assert torch.equal(got[0][:, :, :1], got[1])
    pos = torch.arange(80, device="cuda").view(2, 40).t()[:, 0] % 64
    assert torch.equal(NF.rotary(base, base, table, pos)[0], NF.rotary(base, base, table,
            pos.contiguous())[0])
    x = torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True)
    g = torch.randn(1, 3, 2, 16, device="cuda", requires_grad=True)
    dx = torch.autograd.grad(NF.rotary(x, x.detach(), table)[0], x, g, create_graph=True)[0]
    h = torch.randn_like(dx)
    assert torch.allclose(torch.autograd.grad(dx, g, h)[0], NF.rotary(h, h, table)[0], atol=1e-6)
    # only one of the two outputs is used
    k = torch.randn(1, 3, 1, 16, device="cuda", requires_grad=True)
    dk = torch.autograd.grad(NF.rotary(x, k, table)[1].sum(), (x, k), allow_unused=True)
    assert bool((dk[0] == 0).all()) and bool((dk[1] != 0).any())


def test_positions_outside_of_the_table():
    table = NF.rotary_table(8, 6, device="cuda")
    for dtype in TYPES:
        q = torch.randn(2, 3, 2, 16, device="cuda").to(dtype).requires_grad_()
        pos = torch.tensor([[-1, 0, 5], [6, 2 ** 40, -(2 ** 40)]], device="cuda")
        got, other = NF.rotary(q, q, table, pos)
        hidden = torch.tensor([[True, False, False], [True, True, True]], device="cuda")
        assert bool((got[hidden] == 0).all()) and bool((got[~hidden] != 0).any())
        dx = torch.autograd.grad(got.sum(), q)[0]
        assert bool((dx[hidden] == 0).all()) and bool((dx[~hidden] != 0).any())
    assert bool((NF.rotary(q, q, table[:0])[0] == 0).all())
    e = q.detach()[:0]
    assert NF.rotary(e, e, table)[0].shape == e.shape


# ---------------------------------------------------------------------- #
# append
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("chunks,b", CHUNKS)
@pytest.mark.parametrize("page,dim,rotated,interleaved", [(16, 8, 0, False), (32, 24, 24, False), (16, 80,
        40, True),
                                                          (64, 128, 128, False), (128, 128, 50, True), (64,
                                                                  72, 20, False)])
def test_append(chunks, b, page, dim, rotated, interleaved, dtype):
    append_case(chunks, b, page, dim, rotated, interleaved, dtype, "cuda")


def test_append_is_the_oracle_to_the_bit_without_rotation():
    from slapo_b200.ops.paged import paged_append_reference

    g = torch.Generator().manual_seed(5)
    for page, dim in ((16, 40), (128, 128), (64, 64)):
        size = torch.exp2(torch.randint(-130, 100, (2, 150, 1, 1), generator=g).float())
        k = (torch.randn(2, 150, 3, dim, generator=g) * size).cuda()
        k[0, 7, 1, 3], k[1, 140, 0, 0] = float("inf"), float("nan")
        mine, oracle = (make_cache(2, 10, 3, dim, page, "cuda") for _ in range(2))
        done = 0
        for n in (100, 1, 1, 13, 35):
            done += n
            lengths = torch.full((2,), done, dtype=torch.int32, device="cuda")
            part = k[:, done - n:done]
            NF.paged_append(mine[0], mine[1], part, -part, mine[2], lengths)
            paged_append_reference(oracle[0], oracle[1], part, -part, oracle[2], lengths)
            assert torch.equal(mine[1].nan_to_num(-1.0), oracle[1].nan_to_num(-1.0))
            a, b = mine[0].float(), oracle[0].float()
            assert bool(((a == b) | (a.isnan() & b.isnan())).all())


def test_append_ragged_slices_and_bad_pages():
    # a packed projection's slices, heads in another order, one sequence that brings nothing
    qkv = torch.randn(3, 40, 2, 3, 64, device="cuda").bfloat16()
    rot = NF.rotary_table(64, 200, device="cuda")
    lengths = torch.tensor([7, 140, 100], dtype=torch.int32, device="cuda")
    counts = torch.tensor([7, 40, 0], dtype=torch.int32, device="cuda")
    results = []
    for q, k, v in ([qkv[..., i, :] for i in range(3)], [qkv[..., i, :].contiguous() for i in range(3)],
                    [qkv[..., i, :].transpose(1, 2).contiguous().transpose(1, 2) for i in range(3)],
                    [torch.empty(3, 40, 2, 65, device="cuda", dtype=torch.bfloat16)[..., 1:].copy_(qkv[...,
                            i, :])
                     for i in range(3)]):
        pages, scales, table = make_cache(3, 9, 2, 64, 16, "cuda", poison=False)
        table[1, 7] = 1000
        out = NF.paged_append(pages, scales, k, v, table, lengths, counts, q=q, rotary_table=rot)
        results.append((out, pages.float(), scales))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    out, pages, scales = results[0]
    assert bool((out[0, 7:] == 0).all()) and bool((out[2] == 0).all())
    touched = (pages != 0).flatten(1).any(1).nonzero().flatten().tolist()
    table = make_cache(3, 9, 2, 64, 16, "cpu", poison=False)[2]
    assert sorted(touched) == sorted([int(table[0, 0]), int(table[1, 6]), int(table[1, 8])])
    # (100 .. 139: pages 6, 7 - which there is not - and 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rotated,interleaved", [(64, 64, False), (80, 40, True), (24, 20, False)])
def test_append_rotates_as_rotary_does(dim, rotated, interleaved, dtype):
    """To the bit: queries beside a cache and without one."""
    pages, scales, table = make_cache(2, 2, 1, dim, 64, "cuda")
    rot = NF.rotary_table(rotated, 100, device="cuda")
    k = torch.randn(2, 50, 1, dim, device="cuda").to(dtype)
    q = torch.randn(2, 50, 5, dim, device="cuda").to(dtype)
    lengths = torch.tensor([50, 70], dtype=torch.int32, device="cuda")
    got = NF.paged_append(pages, scales, k, k, table, lengths, q=q, rotary_table=rot, interleaved=interleaved)
    pos = torch.stack([torch.arange(50), torch.arange(20, 70)]).cuda()
    want, turned_k = NF.rotary(q, k, rot, pos, interleaved)
    assert torch.equal(got, want)
    if dtype == torch.float32:
        other = make_cache(2, 2, 1, dim, 64, "cuda")
        NF.paged_append(other[0], other[1], turned_k, k, table, lengths)
        assert torch.equal(pages.view(torch.uint8), other[0].view(torch.uint8))


@pytest.mark.parametrize("page,dim,rotated,interleaved", [(64, 128, 128, False), (64, 64, 64, True), (16, 128, 128, False),
                                                          (32, 80, 40, True), (128, 64, 32, False)])
def test_a_table_that_starts_anywhere(page, dim, rotated, interleaved):
    """A table on 8 bytes, not on 16: whole pages, their queries and the rotation alone."""
    table = NF.rotary_table(rotated, 600, device="cuda")
    odd = torch.empty(table.numel() + 2, device="cuda")[2:].view(table.shape).copy_(table)
    assert odd.data_ptr() % 16 == 8
    k, v = (torch.randn(2, 600, 2, dim, device="cuda").half() for _ in range(2))
    q = torch.randn(2, 600, 4, dim, device="cuda").half()
    results = []
    for rot in (table, odd):
        for n in (600, 60):
            cache = make_cache(2, 38, 2, dim, page, "cuda", poison=False)
            lengths = torch.full((2,), n, dtype=torch.int32, device="cuda")
            out = NF.paged_append(cache[0], cache[1], k[:, :n], v[:, :n], cache[2], lengths, None, q[:, :n], rot,
                                  interleaved)
            results.append((out, cache[0].float(), cache[1], *NF.rotary(q, k, rot, None, interleaved)))
    for a, b in zip(results[:2], results[2:]):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rotated", [(96, 128), (128, 96), (95, 128), (97, 128), (127, 96), (300, 96), (128, 94),
                                       (128, 98), (300, 128)])
def test_a_pages_rotation_of_any_size_in_shared_memory(n, rotated, dtype):
    """Keys of pages of 128 as those turned before, to the bit; 47 to 64 KB of the table for a page."""
    rot = NF.rotary_table(rotated, 320, device="cuda")
    k, v = (torch.randn(2, n, 3, 128, device="cuda").to(dtype) for _ in range(2))
    lengths = torch.tensor([n, n + 7], dtype=torch.int32, device="cuda")
    pos = torch.stack([torch.arange(n), torch.arange(7, n + 7)]).cuda()
    mine, other = (make_cache(2, 3, 3, 128, 128, "cuda") for _ in range(2))
    NF.paged_append(mine[0], mine[1], k, v, mine[2], lengths, rotary_table=rot)
    turned_k = NF.rotary(k.float(), k.float(), rot, pos)[1]
    NF.paged_append(other[0], other[1], turned_k, v.float(), other[2], lengths)
    assert torch.equal(mine[0].view(torch.uint8), other[0].view(torch.uint8))
    assert torch.equal(mine[1].nan_to_num(-1.0), other[1].nan_to_num(-1.0))


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_many_tokens_is_the_oracle(interleaved):
    """Ragged, on top of what is there, some behind the rotation's table: queries by a launch of their own."""
    from slapo_b200.ops.paged import paged_append_reference

    rot = NF.rotary_table(40, 900, device="cuda")
    k, v = (torch.randn(3, 700, 2, 80, device="cuda").half() for _ in range(2))
    q = torch.randn(3, 700, 6, 80, device="cuda").half()
    mine, oracle = (make_cache(3, 32, 2, 80, 32, "cuda") for _ in range(2))
    for lengths, counts in (([5, 300, 1], [5, 300, 1]), ([705, 950, 1], [700, 650, 0])):
        lengths, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts))
        got = NF.paged_append(mine[0], mine[1], k, v, mine[2], lengths, counts, q, rot, interleaved)
        want = paged_append_reference(oracle[0], oracle[1], k, v, oracle[2], lengths, counts, q, rot,
                interleaved)
        # products and sum in fp32 in another order, then fp16; e4m3: another side of a border now and then
        assert bool(((got.float() - want.float()).abs() <= 2.0 ** -10 * want.float().abs() + 2.0 ** -22).all())
        a, b = mine[0].float(), oracle[0].float()
        assert torch.equal(a.isnan(), b.isnan())
        a, b = a.nan_to_num(0.0), b.nan_to_num(0.0)
        assert bool(((a - b).abs() <= 2.0 ** -3 * b.abs() + 2.0 ** -9).all()) and float((a != b).float().mean()) < 1e-3
        assert torch.equal(mine[1].nan_to_num(0.0), oracle[1].nan_to_num(0.0))


# ---------------------------------------------------------------------- #
# attention
def _filled(b, lengths, kv, dim, page, seed=0, spread=1.0):
    """A cache of given lengths with values of about one; what nobody may see is NaN."""
    g = torch.Generator().manual_seed(seed)
    per = max(1, (max(lengths) + page - 1) // page)
    pages, scales, table = make_cache(b, per, kv, dim, page, "cpu", seed)
    for i, n in enumerate(lengths):
        for p in range((n + page - 1) // page):
            rows = min(page, n - p * page)
            id = int(table[i, p])
            s = torch.exp2(torch.randint(-9, -4, (2, kv), generator=g).float())
            x = torch.randn(2, kv, rows, dim, generator=g) * spread / s[..., None, None]
            pages[id, :, :, :rows, :dim] = x.clamp(-448, 448).to(pages.dtype)
            pages[id, :, :, :rows, dim:] = 0.0
            scales[id] = s
    return [t.cuda() for t in (pages, scales, table)]


def _attention_bound(q, want, cache, lengths, counts, scale, window):
    """How far an output may be off.  A score's sum in fp32 is off by 2^-20 of its terms' sizes at most
    (some 130 additions), which changes a weight and the weights' sum by as much of themselves, exp2 by
    2^-20 more; weights are rounded to fp16: 2^-11 of themselves, or 2^-25 where they are small, the largest
    being one; sums in fp32; one rounding to the type."""
    pages, scales, table = cache
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    sizes = pages.clone()
    sizes[:, 1] = pages[:, 1].float().abs().to(pages.dtype)
    size = paged_attention_reference(q.double(), sizes, scales, table, lengths, counts, scale, window)
    values = (pages.float().nan_to_num(0.0).abs() * scales.nan_to_num(0.0)[..., None, None]).amax((0,
            3))       # [2, H, W]
    group = q.shape[2] // pages.shape[2]
    k, v = (x[:, :q.shape[3]].repeat_interleave(group, 0).double() for x in values)
    scores = (q.double().abs() * k).sum(-1, keepdim=True) * scale
    half = HALF[q.dtype]
    return (want.abs() * half * (1 + 2.0 ** -6) + size * (2.0 ** -11 + 2.0 ** -13 + 2 * scores * 2.0 ** -20)
            + lengths.max() * 2.0 ** -25 * v + 2.0 ** -25)


def _attend(q, cache, lengths, counts=None, scale=None, window=None):
    pages, scales, table = cache
    got = NF.paged_attention(q, pages, scales, table, lengths, counts, scale, window)
    want = paged_attention_reference(q.double(), pages, scales, table, lengths, counts, scale, window)
    bound = _attention_bound(q, want, cache, lengths, counts, scale, window)
    assert got.dtype == q.dtype and got.shape == q.shape
    assert not got.isnan().any()
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    return got


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("kv,group", [(1, 1), (3, 1), (2, 4), (1, 8), (2, 12), (1, 33)])
@pytest.mark.parametrize("dim", [8, 16, 64, 72, 80, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_of_a_token(kv, group, dim, page, dtype):
    lengths = [1, 2, 15, 16, 17, 0, 63, 64, 65, 300, 1111]
    cache = _filled(len(lengths), lengths, kv, dim, page)
    q = torch.randn(len(lengths), 1, kv * group, dim, device="cuda").to(dtype)
    out = _attend(q, cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    assert bool((out[5] == 0).all())


@pytest.mark.parametrize("window", [None, 1, 7, 16, 100, 5000])
@pytest.mark.parametrize("n,group", [(2, 1), (5, 3), (16, 1), (17, 2), (70, 1)])
def test_attention_of_some_tokens(n, group, window):
    lengths = [n, n + 1, 100, 129, 1000, 3]
    counts = [n, n, 1, 0, n - 1, 3]
    cache = _filled(6, lengths, 2, 80, 32, seed=n)
    q = torch.randn(6, n, 2 * group, 80, device="cuda").half()
    lengths, counts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, counts))
    _attend(q, cache, lengths, counts, 0.3, window)
    _attend(q, cache, lengths, None, None, window)


@pytest.mark.parametrize("b,length", [(1, 20000), (3, 5001), (200, 40), (700, 3)])
def test_attention_over_long_and_many(b, length):
    cache = _filled(b, [max(1, length - 7 * i) for i in range(b)], 1 if b < 5 else 4, 64, 128)
    lengths = torch.tensor([max(1, length - 7 * i) for i in range(b)], dtype=torch.int32, device="cuda")
    q = torch.randn(b, 1, 4, 64, device="cuda").bfloat16()
    first = _attend(q, cache, lengths)
    for _ in range(3):        # the same every time
        assert torch.equal(first, NF.paged_attention(q, cache[0], cache[1], cache[2], lengths))


def test_attention_of_large_small_and_empty_values():
    """Scores far apart, queries of any size, all-zero queries, pages that there are not."""
    cache = _filled(4, [200, 200, 200, 200], 2, 128, 16, spread=3.0)
    lengths = torch.full((4,), 200, dtype=torch.int32, device="cuda")
    for size in (0.0, 1e-30, 1e-3, 1.0, 30.0):
        q = (torch.randn(4, 1, 2, 128, device="cuda") * size).bfloat16()
        _attend(q, cache, lengths, scale=0.5)
    big = (torch.randn(4, 1, 2, 128, device="cuda") * 1e30).bfloat16()
    _attend(big, cache, lengths, scale=1e-31)
    cache[2][0, 3], cache[2][1, :] = -1, 10 ** 6
    q = torch.randn(4, 1, 4, 128, device="cuda").bfloat16()
    out = _attend(q, cache, lengths)
    assert bool((out[1] == 0).all()) and bool((out[0] != 0).any())
    # a table that ends before the length
    _attend(q, [cache[0], cache[1], cache[2][:, :5].contiguous()], lengths)


def test_attention_queries_in_other_strides():
    cache = _filled(3, [50, 60, 70], 2, 64, 16)
    lengths = torch.tensor([50, 60, 70], dtype=torch.int32, device="cuda")
    qkv = torch.randn(3, 2, 4, 3, 64, device="cuda").half()
    want = _attend(qkv[..., 0, :].contiguous(), cache, lengths)
    for q in (qkv[..., 0, :], qkv[..., 0, :].transpose(1, 2).contiguous().transpose(1, 2),
              torch.empty(3, 2, 4, 67, device="cuda", dtype=torch.float16)[..., 3:].copy_(qkv[..., 0, :])):
        assert torch.equal(want, NF.paged_attention(q, cache[0], cache[1], cache[2], lengths))


def test_a_cache_beyond_32_bits():
    """Pages whose bytes lie behind the first 2^32."""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("a cache of 5 GB")
    small = make_cache(2, 5, 4, 128, 128, "cuda", poison=False)
    total = (5 << 30) // (2 * 4 * 128 * 128)
    pages = torch.empty(total, 2, 4, 128, 128, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(total, 2, 4, device="cuda")
    far = small[2] + (total - 12)
    k = torch.randn(2, 600, 4, 128, device="cuda").half()
    lengths = torch.full((2,), 600, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 1, 8, 128, device="cuda").half()
    outs = []
    for p, s, t in (small, (pages, scales, far)):
        NF.paged_append(p, s, k, k, t, lengths)
        outs.append(NF.paged_attention(q, p, s, t, lengths))
    assert torch.equal(*outs)


# ---------------------------------------------------------------------- #
# sampling
SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05),
            dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=3.0, top_p=0.5),
            dict(top_k=10 ** 9, top_p=0.999), dict(temperature=1e-3), dict(top_p=0.0), dict(temperature=1e30)]


def _sample(x, u, **kw):
    got = NF.sample(x, u, **kw)
    want = sample_reference(x, u, **{**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw})
    assert torch.equal(got, want), (got, want)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 33), (5, 511), (2, 2047), (3, 2048), (4, 5000),
        (2, 50304),
                                        (1, 128001), (300, 700), (1, 262144)])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_sampling(rows, vocab, setting, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab + setting)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    u = torch.rand(rows, generator=g, device="cuda")
    _sample(x, u, **SETTINGS[setting])


@pytest.mark.parametrize("vocab", [40, 3000, 60000])
@pytest.mark.parametrize("kind", ["equal", "two", "masked", "nan", "all_masked", "inf", "huge", "one_left"])
def test_sampling_of_odd_rows(kind, vocab):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, vocab, generator=g, device="cuda")
    if kind == "equal":
        x.zero_()
    elif kind == "two":
        x = (x > 0).float()
    elif kind == "masked":
        x[:, ::3] = -float("inf")
    elif kind == "nan":
        x[:, ::2] = float("nan")
    elif kind == "all_masked":
        x[::2] = -float("inf")
        x[1] = float("nan")
    elif kind == "inf":
        x[:, 5::7] = float("inf")
    elif kind == "huge":
        x *= 1e38
    else:
        x.fill_(-float("inf"))
        x[:, vocab - 1] = -5.0
    u = torch.tensor([0.0, 0.2, 0.5, 0.77, 0.999, 1.0 - 2.0 ** -24], device="cuda")
    for kw in SETTINGS + [dict(top_k=20, top_p=0.6), dict(top_k=vocab - 1), dict(top_k=vocab // 2,
            top_p=0.7)]:
        got = _sample(x, u, **kw)
        if kind == "all_masked":
            assert got[::2].eq(-1).all() and got[1] == -1
        if kind == "one_left":
            assert got.eq(vocab - 1).all()


def test_sampling_rows_of_their_own_and_strides():
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(8, 5000, generator=g, device="cuda") * 4
    u = torch.rand(8, generator=g, device="cuda")
    t = torch.tensor([0.0, 0.5, 1.0, 2.0] * 2, device="cuda")
    k = torch.tensor([0, 1, 5, 100, 4999, 5000, 6000, 3], dtype=torch.int32, device="cuda")
    p = torch.tensor([1.0, 0.1, 0.5, 0.9, 0.99, 0.0, 1.0, 0.7], device="cuda")
    m = torch.tensor([0.0, 0.5, 0.1, 0.01, 0.0, 1.0, 0.2, 0.0], device="cuda")
    want = _sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert torch.equal(NF.sample(x.view(2, 4, 5000), u.view(2, 4), t, k, p, m), want.view(2, 4))
    wide = torch.empty(8, 5003, device="cuda")[:, 1:5001].copy_(x)
    assert torch.equal(NF.sample(wide, u, t, k, p, m), want)
    assert torch.equal(NF.sample(x.t().contiguous().t(), u, t, k, p, m), want)
    for more in ((t, k, p + 1, m), (t, -k, p, m + 1), (-t, k, p, m), (t, k, -p, m)):
        _sample(x, u, **dict(zip(("temperature", "top_k", "top_p", "min_p"), more)))
    assert NF.sample(x[:0], u[:0]).shape == (0,)
    assert int(NF.sample(x[3], u[3], 0.0)) == int(x[3].argmax())


def test_sampled_shares():
    """Drawn 20 000 times, tokens come as often as their probability says."""
    x = torch.log(torch.tensor([0.05, 0.4, 0.15, 0.3, 0.1], device="cuda")).repeat(20000, 1)
    u = (torch.arange(20000, device="cuda") + 0.5) / 20000
    got = torch.bincount(NF.sample(x, u, top_k=3), minlength=5).cpu().double() / 20000
    want = torch.tensor([0, 0.4, 0.15, 0.3, 0], dtype=torch.float64) / 0.85
    # (evenly spaced numbers: off by one of them at each border, and by logits' rounding)
    assert bool(((got - want).abs() <= 2 / 20000).all())


# ---------------------------------------------------------------------- #
# together
def _layers(dim, heads, window=None, dtype=torch.bfloat16):
    torch.manual_seed(0)
    rot = RotaryEmbedding(dim, 4096)
    blocks = [FlashAttention(dim * heads, heads, fused_qkv=True, causal=True, window=window,
            rotary=rot) for _ in range(2)]
    head = torch.nn.Linear(dim * heads, 1000)
    emb = torch.nn.Embedding(1000, dim * heads)
    return [m.to("cuda", dtype).eval() for m in (*blocks, head, emb)]


def test_generation_step_captured_and_replayed():
    """Prompts, then tokens by a captured step: the same as eager steps."""
    *blocks, head, emb = _layers(64, 4)
    u = torch.rand(40, 2, device="cuda")

    def start():
        cache = PagedKVCache(2, 20, 4, 64, batch=2, max_tokens=200, page=32, device="cuda")
        ids = torch.arange(60, device="cuda").view(2, 30) % 1000
        cache.add([30, 17])
        h = emb(ids)
        for i, block in enumerate(blocks):
            h = h + block(h, layer_past=cache.layer(i), use_cache=True)[0]
        last = h[torch.arange(2), torch.tensor([29, 16])]
        return cache, NF.sample(head(last), u[0], 0.9, 40, 0.95)

    def step(cache, token, number):
        h = emb(token[:, None])
        for i, block in enumerate(blocks):
            h = h + block(h, layer_past=cache.layer(i), use_cache=True)[0]
        return NF.sample(head(h[:, 0]), number, 0.9, 40, 0.95)

    with torch.no_grad():
        cache, token = start()
        eager = [token]
        for i in range(1, 40):
            cache.add(1)
            eager.append(step(cache, eager[-1], u[i]))
        cache, token = start()
        token, number = token.clone(), u[1].clone()
        cache.add(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(cache, token, number)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, token, number)
        got = [token.clone()]
        for i in range(1, 40):
            if i > 1:
                cache.add(1)
            token.copy_(got[-1])
            number.copy_(u[i])
            graph.replay()
            got.append(out.clone())
        assert torch.equal(torch.stack(eager), torch.stack(got))
    assert len(set(torch.stack(got)[:, 0].tolist())) > 5


def test_generation_is_near_the_layer_without_a_cache():
    *blocks, head, emb = _layers(64, 4, window=50, dtype=torch.float16)
    block = blocks[0]
    x = torch.randn(3, 200, 256, device="cuda").half()
    with torch.no_grad():
        want, _ = block(x)
        cache = PagedKVCache(1, 60, 4, 64, batch=3, max_tokens=256, page=16, device="cuda")
        outs = []
        for n in (90, 1, 1, 3, 40, 1, 64):
            t = sum(o.shape[1] for o in outs)
            cache.add(n)
            outs.append(block(x[:, t:t + n], layer_past=cache.layer(0), use_cache=True)[0])
    got = torch.cat(outs, 1).float()
    assert (got - want.float()).norm() <= 0.1 * want.float().norm()      # (what 8 bits lose)
    assert (got[:, :90] - want[:, :90].float()).norm() <= 2.0 ** -9 * want.float().norm()


def test_training_with_rotation_has_its_gradients():
    """A rotated layer against the same by the oracles, in fp32 through the packed path and in bf16."""
    rot = RotaryEmbedding(32, 128, interleaved=True, scaling={"type": "yarn", "factor": 4,
            "original_positions": 32})
    layer = FlashAttention(256, 4, fused_qkv=True, causal=True, rotary=rot).to("cuda", torch.bfloat16)
    x = torch.randn(2, 100, 256, device="cuda").bfloat16().requires_grad_()
    out, _ = layer(x)
    dy = torch.randn_like(out)
    got = torch.autograd.grad(out, [x, layer.qkv.weight], dy)

    def plain(x, w):
        qkv = torch.nn.functional.linear(x, w, layer.qkv.bias.double()).view(2, 100, 4, 3, 64)
        q, k = NF.rotary(qkv[..., 0, :].cpu(), qkv[..., 1, :].cpu(), rot.table("cpu"), None, True)
        s = torch.einsum("bqhd,bkhd->bhqk", q.cuda(), k.cuda()) / 8
        s = s.masked_fill(~torch.ones(100, 100, dtype=torch.bool, device="cuda").tril(), -math.inf)
        c = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), qkv[..., 2, :]).reshape(2, 100, 256)
        return torch.nn.functional.linear(c, layer.out_proj.weight.double(), layer.out_proj.bias.double())

    xd, wd = x.detach().double().requires_grad_(), layer.qkv.weight.detach().double().requires_grad_()
    want_out = plain(xd, wd)
    want = torch.autograd.grad(want_out, (xd, wd), dy.double())
    # about eight roundings to bf16 on the way, 2^-9 in the mean each
    for a, b in zip((out, *got), (want_out, *want)):
        assert (a.double() - b).norm() <= 8 * 2.0 ** -9 * b.norm()


def test_inference_mode_and_training_in_turn():
    layer = FlashAttention(128, 2, fused_qkv=True, causal=True, rotary=RotaryEmbedding(64, 64)).to(
        "cuda", torch.bfloat16).eval()
    x = torch.randn(2, 40, 128, device="cuda").bfloat16()
    with torch.inference_mode():
        cache = PagedKVCache(1, 8, 2, 64, batch=2, max_tokens=64, page=16, device="cuda")
        cache.add(39)
        layer(x[:, :39], layer_past=cache.layer(0))
    out, _ = layer(x, position_ids=torch.arange(40, device="cuda")[None])
    assert torch.equal(out, layer(x)[0])
    assert torch.autograd.grad(out.sum(), layer.qkv.weight)[0].abs().sum() > 0
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            cache.add(1)
            one, _ = layer(x[:, 39:], layer_past=cache.layer(0))
            assert bool(one.isfinite().all())


def test_prompts_captured_and_replayed():
    """Append with its queries by a launch of their own, and attention of many rows, from a graph."""
    rot = NF.rotary_table(64, 900, device="cuda")
    k, v = (torch.randn(2, 400, 2, 64, device="cuda").half() for _ in range(2))
    q = torch.randn(2, 400, 4, 64, device="cuda").half()
    lengths = torch.tensor([400, 450], dtype=torch.int32, device="cuda")
    cache = make_cache(2, 20, 2, 64, 32, "cuda", poison=False)

    def step():
        turned_q = NF.paged_append(cache[0], cache[1], k, v, cache[2], lengths, q=q, rotary_table=rot)
        return turned_q, NF.paged_attention(turned_q, *cache, lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for more in (0, 37):
        lengths.add_(more)
        cache[0].zero_()
        cache[1].zero_()
        want = step()
        pages, scales = cache[0].clone(), cache[1].clone()
        cache[0].zero_()
        cache[1].zero_()
        graph.replay()
        for a, b in zip((*want, pages.float(), scales), (*got, cache[0].float(), cache[1])):
            assert torch.equal(a, b)


def test_streams_of_their_own():
    """Calls on a stream that is not the default one, while the default one is busy."""
    cache = _filled(4, [500] * 4, 4, 64, 64)
    lengths = torch.full((4,), 500, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 1, 8, 64, device="cuda").half()
    x, u = torch.randn(4, 9000, device="cuda"), torch.rand(4, device="cuda")
    want = NF.paged_attention(q, *cache, lengths), NF.sample(x, u, top_p=0.9)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        busy = busy @ busy * 1e-3
        with torch.cuda.stream(side):
            got = NF.paged_attention(q, *cache, lengths), NF.sample(x, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_kernels_are_counted():
    before = native.launch_count()
    q = torch.randn(1, 2, 2, 16, device="cuda")
    NF.rotary(q, q, NF.rotary_table(16, 4, device="cuda"))
    NF.sample(torch.randn(1, 9, device="cuda"), torch.rand(1, device="cuda"))
    assert native.launch_count() == before + 2
