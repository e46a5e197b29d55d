"""Rotation by positions, the paged 8-bit cache and sampling on the CPU: the oracles against definitions
written apart from them, refusals, the cache's bookkeeping, generation through ``FlashAttention``."""
import copy
import math

import pytest
import torch

from slapo_b200.op import FlashAttention, PagedKVCache, RotaryEmbedding
from slapo_b200.ops import functional as NF


# ---------------------------------------------------------------------- #
# rotation
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(8, 8), (16, 6), (10, 2), (64, 64)])
def test_rotation_is_a_complex_product(dim, rotated, interleaved):
    table = NF.rotary_table(rotated, 50)
    q, k = torch.randn(2, 7, 3, dim, dtype=torch.float64), torch.randn(2, 7, 1, dim, dtype=torch.float64)
    pos = torch.randint(0, 50, (2, 7))
    got = NF.rotary(q, k, table, pos, interleaved)
    for x, y in zip((q, k), got):
        part = x[..., :rotated]
        pairs = part.view(*part.shape[:-1], -1, 2) if interleaved else part.view(*part.shape[:-1], 2,
                -1).transpose(-1, -2)
        z = torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(table.double()[pos])[:, :, None]
        z = torch.view_as_real(z)
        want = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
        # two products and a sum in fp64
        assert (y[..., :rotated] - want).abs().max() <= 4 * 2.0 ** -52 * x.abs().max() * 2
        assert torch.equal(y[..., rotated:], x[..., rotated:])


def test_rotation_keeps_distances_and_has_its_gradient():
    table = NF.rotary_table(8, 64).double().float()
    q = torch.randn(1, 4, 2, 12, dtype=torch.float64, requires_grad=True)
    k = torch.randn(1, 4, 1, 12, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a, b: NF.rotary(a, b, table, 3, True), (q, k))
    qkv = torch.randn(1, 3, 2, 3, 8, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda a: NF.rotary_qkvpacked(a, table, torch.tensor([5, 0, 63])), qkv)
    a, b = torch.randn(2, 8, dtype=torch.float64)
    dots = []
    for p in (0, 11, 40):
        x, y = NF.rotary(a.view(1, 1, 1, 8), b.view(1, 1, 1, 8), table, p)[0], \
            NF.rotary(a.view(1, 1, 1, 8), b.view(1, 1, 1, 8), table, p + 5)[1]
        dots.append(float((x * y).sum()))
    # (the table's entries are off by 2^-25 of 1 each)
    assert max(dots) - min(dots) <= 8 * 4 * 2.0 ** -24 * float(a.abs().max() * b.abs().max())


def test_positions_outside_of_the_table_give_zeros():
    table = NF.rotary_table(4, 6)
    q = torch.randn(2, 3, 1, 8)
    pos = torch.tensor([[-1, 0, 5], [6, 2 ** 40, -(2 ** 40)]])
    got, _ = NF.rotary(q, q, table, pos)
    hidden = torch.tensor([[True, False, False], [True, True, True]])
    assert bool((got[hidden] == 0).all()) and bool((got[~hidden] != 0).any())
    assert bool((NF.rotary(q, q, table, 6)[0] == 0).all())


def test_tables():
    # written out: the angle of pair i at position p
    t = NF.rotary_table(8, 20, base=100.0)
    for p in (0, 3, 19):
        for i in range(4):
            angle = p * 100.0 ** (-2 * i / 8)
            assert abs(float(t[p, i, 0]) - math.cos(angle)) <= 2.0 ** -24
            assert abs(float(t[p, i, 1]) - math.sin(angle)) <= 2.0 ** -24
    linear = NF.rotary_table(8, 20, scaling={"type": "linear", "factor": 4})
    assert torch.equal(linear[4::4][:4], NF.rotary_table(8, 5)[1:])
    ntk = NF.rotary_table(8, 20, scaling={"type": "ntk", "factor": 4})
    assert torch.equal(ntk[:, 0], NF.rotary_table(8, 20)[:, 0])          # the fastest pair as it is
    angle = 19 * 1e4 ** (-6 / 8) / 4                                      # the slowest one stretched by the factor
    assert abs(float(ntk[19, 3, 1]) - math.sin(angle)) <= 2.0 ** -23
    yarn = NF.rotary_table(64, 4096, scaling={"type": "yarn", "factor": 4, "original_positions": 1024})
    plain, stretched = NF.rotary_table(64, 4096), NF.rotary_table(64, 4096, scaling={"type": "linear",
            "factor": 4})
    m = 0.1 * math.log(4) + 1
    assert torch.allclose(yarn[:, 0], plain[:, 0] * m, rtol=2.0 ** -22, atol=2.0 ** -22)
    assert torch.allclose(yarn[:, -1], stretched[:, -1] * m, rtol=2.0 ** -22, atol=2.0 ** -22)


def test_table_refusals():
    for args in ((3, 4), (0, 4), (4, -1)):
        with pytest.raises(ValueError):
            NF.rotary_table(*args)
    for scaling in ({"type": "other"}, {"factor": 2}, {"type": "linear", "factor": 0.5}, {"type": "linear"},
                    {"type": "yarn", "factor": 2}, {"type": "linear", "factor": 2, "base": 3}):
        with pytest.raises(ValueError):
            NF.rotary_table(4, 4, scaling=scaling)
    with pytest.raises(ValueError):
        NF.rotary_table(2, 4, scaling={"type": "ntk", "factor": 2})


def rotary_refusals(device):
    def t(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype, device=device)

    table = NF.rotary_table(8, 4, device=device)
    q = t(2, 3, 4, 8)
    yield ValueError, lambda: NF.rotary(t(2, 3, 8), t(2, 3, 8), table)
    yield ValueError, lambda: NF.rotary(q, t(2, 4, 4, 8), table)
    yield ValueError, lambda: NF.rotary(q, t(2, 3, 4, 16), table)
    yield TypeError, lambda: NF.rotary(q, t(2, 3, 4, 8, dtype=torch.float32), table)
    yield TypeError, lambda: NF.rotary(q.int(), q.int(), table)
    yield TypeError, lambda: NF.rotary(q, q, table.double())
    yield ValueError, lambda: NF.rotary(q[..., :6], q[..., :6], table)
    yield ValueError, lambda: NF.rotary(q, q, table[:, :, 0])
    yield ValueError, lambda: NF.rotary(q, q, table.clone().requires_grad_())
    yield ValueError, lambda: NF.rotary(q, q, table, torch.zeros(2, dtype=torch.long, device=device))
    yield ValueError, lambda: NF.rotary(q, q, table, torch.zeros(3, 3, dtype=torch.long, device=device))
    yield TypeError, lambda: NF.rotary(q, q, table, torch.zeros(3, device=device))
    yield TypeError, lambda: NF.rotary(q, q, table, 1.5)
    yield ValueError, lambda: NF.rotary_qkvpacked(q, table)
    yield ValueError, lambda: NF.rotary_qkvpacked(t(2, 3, 4, 2, 8), table)


@pytest.mark.parametrize("index", range(15))
def test_rotary_refusals(index):
    error, call = list(rotary_refusals("cpu"))[index]
    with pytest.raises(error):
        call()


# ---------------------------------------------------------------------- #
# the paged cache
def make_cache(b, per, heads, dim, page, device="cpu", seed=0, poison=True, spare=2):
    """An empty cache, its pages in no order, and a table; ``poison``: codes are NaN until they are
    written."""
    g = torch.Generator().manual_seed(seed)
    total = b * per + spare
    width = (dim + 15) // 16 * 16
    pages = torch.full((total, 2, heads, page, width),
            float("nan") if poison else 0.0).to(torch.float8_e4m3fn).to(device)
    scales = torch.full((total, 2, heads), float("nan") if poison else 0.0, device=device)
    table = torch.randperm(total, generator=g)[:b * per].view(b, per).int().to(device)
    return pages, scales, table


def read_cache(pages, scales, table, b, tokens, dim):
    """Keys and values ``[2, tokens, H, D]`` that sequence ``b`` has, in fp64, and the scale of each."""
    page = pages.shape[3]
    ids = table[b, :(tokens + page - 1) // page].long()
    got = pages[ids].double() * scales[ids].double()[..., None, None]
    step = scales[ids].double()[..., None].expand(*scales[ids].shape, page)
    flat = got.permute(1, 0, 3, 2, 4).reshape(2, -1, pages.shape[2], pages.shape[4])
    return flat[:, :tokens, :, :dim], step.permute(1, 0, 3, 2).reshape(2, -1, pages.shape[2])[:, :tokens]


def check_cache(pages, scales, table, want, grown=0):
    """The cache against ``want``: for each sequence keys and values ``[2, tokens, H, D]`` in fp64.  A value
    is rounded to e4m3, off by 2^-4 of itself or half of 2^-9 of its scale; each growth of its scale can
    round it again in the last way alone (a power of two)."""
    page = pages.shape[3]
    for b, x in enumerate(want):
        tokens, dim = x.shape[1], x.shape[3]
        got, scale = read_cache(pages, scales, table, b, tokens, dim)
        bound = torch.maximum(x.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10) + grown * scale[...,
                None] * 2.0 ** -10
        assert bool(((got - x).abs() <= bound * (1 + 2.0 ** -10)).all())
        # scales: the smallest power of two for the page's largest value (of rounded ones: with their slack)
        for p in range((tokens + page - 1) // page):
            top = x[:, p * page:(p + 1) * page].abs().amax((1, 3))
            s = scale[:, p * page]
            assert bool((torch.frexp(s)[0] == 0.5).all())
            assert bool((top <= 448 * s * (1 + 2.0 ** -20)).all())
            small = (top > 224 * s * (1 - 2.0 ** -20)) | (s == 2.0 ** -100)
            assert bool(small.all())


def append_all(chunks, k, v, q, cache, table_rot, interleaved, counts=None):
    """Chunks of new tokens one after the other; queries as they come back."""
    pages, scales, table = cache
    b = k.shape[0]
    done = torch.zeros(b, dtype=torch.int32, device=k.device)
    out = []
    at = 0
    for i, n in enumerate(chunks):
        c = None if counts is None else counts[i]
        done = done + (n if c is None else c)
        part = [None if x is None else x[:, at:at + n] for x in (k, v, q)]
        got = NF.paged_append(pages, scales, part[0], part[1], table, done, c, q=part[2],
                rotary_table=table_rot,
                              interleaved=interleaved)
        out.append(got)
        at += n
    return out, done


def turned(x, rot, pos, interleaved):
    """In fp64, written apart: by complex numbers."""
    x = x.double().clone()
    if rot is None:
        return x
    r = 2 * rot.shape[1]
    part = x[..., :r]
    pairs = part.reshape(*part.shape[:-1], -1, 2) if interleaved else \
        part.reshape(*part.shape[:-1], 2, -1).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(rot.double()[pos])[..., None, :]
    z = torch.view_as_real(z)
    x[..., :r] = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return x


CHUNKS = [([1], 1), ([5], 2), ([40], 1), ([33, 1, 1, 1], 2), ([1] * 20, 3), ([16, 16, 3], 2), ([200, 7, 64],
        1)]


def append_case(chunks, b, page, dim, rotated, interleaved, dtype, device="cpu"):
    g = torch.Generator().manual_seed(sum(chunks) + dim)
    n, heads, q_heads = sum(chunks), 2, 4
    # values whose size jumps, so that scales grow within pages
    size = torch.exp2(torch.randint(-3, 4, (b, n, 1, 1), generator=g).float())
    k, v, q = ((torch.randn(b, n, h, dim, generator=g) * size).to(dtype).to(device) for h in (heads, heads,
            q_heads))
    cache = make_cache(b, (n + page - 1) // page, heads, dim, page, device)
    rot = NF.rotary_table(rotated, n, device=device) if rotated else None
    out, lengths = append_all(chunks, k, v, q, cache, rot, interleaved)
    pos = torch.arange(n, device=device)
    want = [torch.stack([turned(k[i], rot, pos, interleaved), v[i].double()]) for i in range(b)]
    check_cache(*cache, want, grown=min(len(chunks) - 1, 6))
    got = torch.cat(out, 1)
    wish = torch.stack([turned(q[i], rot, pos, interleaved) for i in range(b)])
    half = torch.finfo(dtype).eps / 2
    # products and sum in fp32 (two roundings of |a| + |b|), then one to the type
    bound = wish.abs() * half * (1 + 2.0 ** -10) + q.double().abs().amax(-1, keepdim=True) * 4 * 2.0 ** -24
    assert bool(((got.double() - wish).abs() <= bound).all())
    # nothing behind the last token, no other page
    pages, scales, table = cache
    used = torch.zeros(pages.shape[0], page, dtype=torch.bool, device=device)
    for i in range(b):
        for p in range(0, n, page):
            used[table[i, p // page].long(), :min(page, n - p)] = True
    rest = pages.permute(0, 3, 1, 2, 4)[~used].float()
    assert bool(rest.isnan().all())
    return cache, lengths


@pytest.mark.parametrize("chunks,b", CHUNKS)
@pytest.mark.parametrize("page,dim,rotated,interleaved", [(16, 8, 0, False), (32, 24, 24, False), (16, 80,
        40, True),
                                                          (64, 64, 20, False)])
def test_append(chunks, b, page, dim, rotated, interleaved):
    append_case(chunks, b, page, dim, rotated, interleaved, torch.float32)


def test_append_ragged_and_bad_pages():
    pages, scales, table = make_cache(3, 3, 1, 8, 16)
    table[1, 1], table[2, 0] = 99, -1
    k = torch.randn(3, 40, 1, 8)
    lengths = torch.tensor([7, 40, 20], dtype=torch.int32)
    counts = torch.tensor([7, 40, 20], dtype=torch.int32)
    rot = NF.rotary_table(8, 30)
    q = NF.paged_append(pages, scales, k, k, table, lengths, counts, q=k, rotary_table=rot)
    for i, c in enumerate((7, 30, 20)):        # (behind the rotation's table: none)
        assert bool((q[i, c:] == 0).all()) and bool((q[i, :c] != 0).any(-1).all())
    assert not pages[table[0, 0].long(), :, :, :7].float().isnan().any()
    assert pages[table[0, 0].long(), :, :, 7:].float().isnan().all()
    assert pages[table[0, 1:].long()].float().isnan().all() and pages[table[2,
            2].long()].float().isnan().all()
    assert not pages[table[1, 0].long()].float().isnan().any() and not pages[table[1, 2].long(), :, :,
            :8].float().isnan().any()
    assert not pages[table[2, 1].long(), :, :, :4].float().isnan().any()
    # left padding, a table that is too short, no sequences, no tokens
    pages, scales, table = make_cache(1, 1, 1, 8, 16)
    NF.paged_append(pages, scales, k[:1, :5], k[:1, :5], table, torch.tensor([2], dtype=torch.int32))
    got, _ = read_cache(pages, scales, table, 0, 2, 8)
    assert bool(((got - k[0, 3:5].double()).abs() <= k[0, 3:5].abs() * 2.0 ** -4 + 2.0 ** -8).all())
    NF.paged_append(pages, scales, k[:1, :40], k[:1, :40], table, torch.tensor([40], dtype=torch.int32))
    NF.paged_append(pages, scales, k[:0], k[:0], table[:0], lengths[:0])
    NF.paged_append(pages, scales, k[:1, :0], k[:1, :0], table, lengths[:1])


def test_append_values_that_are_not_finite():
    pages, scales, table = make_cache(1, 1, 1, 8, 16)
    k = torch.ones(1, 3, 1, 8)
    k[0, 1, 0, 2], k[0, 2, 0, 5] = float("inf"), float("nan")
    NF.paged_append(pages, scales, k, k, table, torch.tensor([3], dtype=torch.int32))
    got, _ = read_cache(pages, scales, table, 0, 3, 8)
    assert bool((got.isnan() == ~k[0].isfinite()).all()) and bool((got[got.isfinite()] == 1).all())
    big = torch.full((1, 1, 1, 8), torch.finfo(torch.float32).max)
    zero = torch.zeros(1, 1, 1, 8)
    NF.paged_append(pages, scales, big, zero, table, torch.tensor([1], dtype=torch.int32))
    s = scales[table[0, 0].long()]
    assert float(s[0]) == 2.0 ** 120 and float(s[1]) == 2.0 ** -100


def test_attention_over_the_cache_is_attention():
    """Against the framework's own attention on the values that the cache holds."""
    for n, window, q_heads in ((1, None, 2), (4, None, 6), (5, 3, 4), (30, 7, 2), (3, 100, 2)):
        (pages, scales, table), lengths = append_case([30, 9], 2, 16, 16, 16, False, torch.float32)
        q = torch.randn(2, n, q_heads, 16)
        got = NF.paged_attention(q, pages, scales, table, lengths, window=window)
        kv = torch.stack([read_cache(pages, scales, table, i, 39, 16)[0] for i in range(2)], 1).float()
        k, v = (x.repeat_interleave(q_heads // 2, 2) for x in kv)
        want = NF.attention_reference(q, k, v, causal=True, window=window)
        assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)      # (sums of 39 in fp32, two orders)


def test_attention_rows_without_a_key():
    (pages, scales, table), _ = append_case([20], 3, 16, 8, 0, False, torch.float32)
    q = torch.randn(3, 4, 2, 8)
    lengths = torch.tensor([0, 2, 20], dtype=torch.int32)
    out = NF.paged_attention(q, pages, scales, table, lengths)
    assert bool((out[0] == 0).all()) and bool((out[1, :2] == 0).all()) and bool((out[1,
            2:] != 0).any(-1).all())
    counts = torch.tensor([0, 2, 9], dtype=torch.int32)
    out = NF.paged_attention(q, pages, scales, table, lengths, counts)
    assert bool((out[1, 2:] == 0).all()) and bool((out[1, 0] != 0).any(-1).all())
    table[2, 0] = -5                                   # a page that there is not
    first = NF.paged_attention(q, pages, scales, table, lengths, counts)[2]
    only = NF.paged_attention(q[2:], pages, scales, table[2:], lengths[2:], counts[2:], window=4)
    assert torch.allclose(first[3], only[0, 3],
            atol=1e-6)         # 17 .. 20 of 20: what the second page holds


def paged_refusals(device):
    pages, scales, table = make_cache(2, 2, 2, 16, 16, device)
    lengths = torch.full((2,), 3, dtype=torch.int32, device=device)
    k = torch.randn(2, 3, 2, 16, device=device).half()
    q = torch.randn(2, 3, 4, 16, device=device).half()

    def append(**kw):
        a = dict(pages=pages, scales=scales, k=k, v=k, block_table=table, lengths=lengths)
        return lambda: NF.paged_append(**{**a, **kw})

    def attend(**kw):
        a = dict(q=q, pages=pages, scales=scales, block_table=table, lengths=lengths)
        return lambda: NF.paged_attention(**{**a, **kw})

    for call in (append, attend):
        yield TypeError, call(pages=pages.float())
        yield TypeError, call(scales=scales.half())
        yield ValueError, call(pages=pages[:, :, :, :8].contiguous())
        yield ValueError, call(pages=pages[..., :8])
        yield ValueError, call(pages=pages[:, :1])
        yield ValueError, call(scales=scales[:3])
        yield TypeError, call(block_table=table.long())
        yield ValueError, call(block_table=table[:1])
        yield ValueError, call(block_table=table[:, 0])
        yield TypeError, call(lengths=lengths.long())
        yield ValueError, call(lengths=lengths[:1])
        yield TypeError, call(counts=lengths.float())
        yield ValueError, call(counts=lengths[:1])
    yield ValueError, append(v=k[:, :2])
    yield TypeError, append(v=k.float())
    yield ValueError, append(k=k[:, :, :1], v=k[:, :, :1])
    yield TypeError, append(k=k.double(), v=k.double())
    yield ValueError, append(k=k[..., :4], v=k[..., :4])
    yield TypeError, append(q=q.float(), rotary_table=NF.rotary_table(4, 4, device=device))
    yield ValueError, append(q=q[:, :2], rotary_table=NF.rotary_table(4, 4, device=device))
    yield ValueError, append(rotary_table=NF.rotary_table(18, 4, device=device))
    yield RuntimeError, append(k=k.clone().requires_grad_())
    yield ValueError, attend(q=q[:, :, :3])
    yield ValueError, attend(q=q[:, 0])
    yield ValueError, attend(window=0)
    yield ValueError, attend(window=1.5)
    yield TypeError, attend(q=q.int())
    yield RuntimeError, attend(q=q.clone().requires_grad_())


@pytest.mark.parametrize("index", range(41))
def test_paged_refusals(index):
    error, call = list(paged_refusals("cpu"))[index]
    with pytest.raises(error):
        call()


def test_refusals_are_all_tested():
    assert len(list(paged_refusals("cpu"))) == 41 and len(list(rotary_refusals("cpu"))) == 15
    assert len(list(sample_refusals("cpu"))) == 14


# ---------------------------------------------------------------------- #
# sampling
def test_sampling_by_hand():
    x = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]]))

    def take(u, **kw):
        return int(NF.sample(x, torch.tensor([u]), **kw))

    assert [take(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.99)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [take(u, top_k=2) for u in (0.0, 0.56, 0.58, 0.99)] == [1, 1, 3, 3]
    assert [take(u, top_p=0.65) for u in (0.0, 0.56, 0.58, 0.99)] == [1, 1, 3, 3]
    assert [take(u, top_p=0.75) for u in (0.0, 0.46, 0.65, 0.68)] == [1, 2, 2, 3]
    assert [take(u, min_p=0.6) for u in (0.0, 0.56, 0.58)] == [1, 1, 3]
    # top_p is a share of what top_k kept: 0.4 / 0.7 of it suffices for 0.57
    assert [take(u, top_k=2, top_p=0.57) for u in (0.0, 0.99)] == [1, 1]
    assert [take(u, temperature=0.0) for u in (0.0, 0.99)] == [1, 1]
    assert [take(u, top_p=0.0) for u in (0.0, 0.99)] == [1, 1]


def test_sampling_ties_masks_and_empty_rows():
    inf = float("inf")
    x = torch.zeros(1, 8)
    assert [int(NF.sample(x, torch.tensor([u]), top_k=3)) for u in (0.0, 0.5, 0.99)] == [0, 1, 2]
    assert [int(NF.sample(x, torch.tensor([u]), top_p=0.26)) for u in (0.0, 0.5, 0.99)] == [0, 1, 2]
    assert int(NF.sample(x, torch.tensor([0.9]), temperature=0.0)) == 0
    x = torch.tensor([[-inf, 1.0, -inf, float("nan")], [-inf] * 4, [float("nan")] * 4, [inf, 1.0, inf, 0.0]])
    got = NF.sample(x, torch.tensor([0.99, 0.5, 0.5, 0.7]))
    assert got.tolist() == [1, -1, -1, 2] and got.dtype == torch.int64
    assert NF.sample(torch.zeros(2, 3, 5), torch.zeros(2, 3)).shape == (2, 3)
    assert NF.sample(torch.zeros(0, 5), torch.zeros(0)).shape == (0,)
    assert int(NF.sample(torch.zeros(1), torch.tensor(0.5))) == 0


def test_sampling_settings_for_each_row():
    x = torch.log(torch.tensor([0.1, 0.4, 0.2, 0.3])).repeat(4, 1)
    u = torch.tensor([0.05, 0.05, 0.99, 0.05])
    got = NF.sample(x, u, torch.tensor([1.0, 0.0, 1.0, 1.0]), torch.tensor([0, 0, 2, 0], dtype=torch.int32),
                    torch.tensor([1.0, 1.0, 1.0, 0.1]), torch.tensor([0.0, 0.0, 0.9, 0.0]))
    assert got.tolist() == [0, 1, 1, 1]
    # settings beyond their range, which a tensor of them can have: all there is, or the largest
    one = torch.ones(4)
    got = NF.sample(x, u, one, torch.full((4,), -3, dtype=torch.int32), 2 * one, -one)
    assert got.tolist() == [0, 0, 3, 0]
    for args in ((one, torch.zeros(4, dtype=torch.int32), -one, 0 * one), (one, torch.zeros(4,
            dtype=torch.int32), one, 2 * one),
                 (-one, torch.zeros(4, dtype=torch.int32), one, 0 * one)):
        assert NF.sample(x, u, *args).tolist() == [1, 1, 1, 1]


def sample_refusals(device):
    x, u = torch.zeros(2, 5, device=device), torch.zeros(2, device=device)
    yield ValueError, lambda: NF.sample(x[:, :0], u)
    yield ValueError, lambda: NF.sample(torch.zeros(2, (1 << 18) + 1, device=device), u)
    yield TypeError, lambda: NF.sample(x.double(), u)
    yield TypeError, lambda: NF.sample(x, u.double())
    yield ValueError, lambda: NF.sample(x, u[:1])
    yield ValueError, lambda: NF.sample(x, u, -1.0)
    yield ValueError, lambda: NF.sample(x, u, float("nan"))
    yield ValueError, lambda: NF.sample(x, u, 1.0, -1)
    yield ValueError, lambda: NF.sample(x, u, 1.0, 0, 1.5)
    yield ValueError, lambda: NF.sample(x, u, 1.0, 0, 1.0, -0.1)
    yield TypeError, lambda: NF.sample(x, u, 1.0, u)
    yield TypeError, lambda: NF.sample(x, u, u.double())
    yield ValueError, lambda: NF.sample(x, u, u[:1])
    yield TypeError, lambda: NF.sample(x, u, 1.0, 1.5)


@pytest.mark.parametrize("index", range(14))
def test_sample_refusals(index):
    error, call = list(sample_refusals("cpu"))[index]
    with pytest.raises(error):
        call()


# ---------------------------------------------------------------------- #
# the cache's bookkeeping, and generation through a layer
def test_bookkeeping():
    c = PagedKVCache(2, 7, 2, 16, batch=3, max_tokens=40, page=16)
    assert c.pages[0].shape == (7, 2, 2, 16, 16) and c.block_table.shape == (3, 3) and len(c.pages) == 2
    c.add([17, 0, 16])
    assert c.fresh and c.free_pages == 4 and c.lengths.tolist() == [17, 0, 16] and c.counts.tolist() == [17,
            0, 16]
    c.add(1)
    assert not c.fresh and c.counts is None and c.lengths.tolist() == [18, 1, 17] and c.free_pages == 2
    used = c.block_table[c.block_table >= 0].tolist()
    assert len(used) == len(set(used)) == 5
    for bad, error in (([1, 40, 1], ValueError), ([1, 1], ValueError), ([1, -1, 1], ValueError), ([16, 16,
            16], RuntimeError)):
        before = (c.block_table.clone(), c.lengths.clone(), c.free_pages, [c.tokens(i) for i in range(3)])
        with pytest.raises(error):
            c.add(bad)
        assert torch.equal(before[0], c.block_table) and torch.equal(before[1], c.lengths)
        assert before[2:] == (c.free_pages, [c.tokens(i) for i in range(3)])
    c.free(0)
    assert c.free_pages == 4 and c.lengths.tolist() == [0, 1, 17] and c.block_table[0].tolist() == [-1] * 3
    c.add([33, 0, 0])
    assert c.free_pages == 1 and c.tokens(0) == 33
    for kw in ({"page": 20}, {"head_dim": 12}, {"head_dim": 136}):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(layers=1, pages=1, heads=1, head_dim=16, batch=1, max_tokens=16), **kw})


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("window", [None, 5])
def test_generation_over_pages_is_generation(fused, window):
    """Token by token over the 8-bit cache against the layer without one: off by what 8 bits lose."""
    torch.manual_seed(3)
    rot = RotaryEmbedding(8, 64, interleaved=True)
    layer = FlashAttention(32, 2, fused_qkv=fused, causal=True, window=window, rotary=rot).eval()
    x = torch.randn(2, 20, 32)
    with torch.no_grad():
        want, _ = layer(x)
        cache = PagedKVCache(1, 8, 2, 16, batch=2, max_tokens=32, page=16)
        cache.add(11)
        first, present = layer(x[:, :11], layer_past=cache.layer(0), use_cache=True)
        assert torch.allclose(first, want[:, :11],
                atol=1e-5)        # a prompt's first tokens: keys as they are
        for t in range(11, 20):
            cache.add(1)
            out, present = layer(x[:, t:t + 1], layer_past=present, use_cache=True)
            # values off by 2^-4 of themselves at most, by an eighth of that in the mean of many; weights by
            # the keys'
            assert (out[:, 0] - want[:, t]).norm() <= 0.1 * want[:, t].norm()
        # the same over a cache of tensors, which keeps rotated keys
        past = None
        for t in range(20):
            out, past = layer(x[:, t:t + 1], layer_past=past, use_cache=True)
            assert torch.allclose(out[:, 0], want[:, t], atol=1e-5)
    with pytest.raises(NotImplementedError):
        layer(x[:, :1], attention_mask=torch.ones(2, 1), layer_past=present)
    with pytest.raises(NotImplementedError):
        FlashAttention(32, 2, causal=False)(x[:, :1], layer_past=present)
    with pytest.raises(NotImplementedError):
        FlashAttention(32, 2, causal=True, attn_pdrop=0.1).train()(x[:, :1], layer_past=present)
    with pytest.raises(NotImplementedError):
        FlashAttention(32, 2, causal=True, window=3, sinks=1)(x[:, :1], layer_past=present)
    with pytest.raises(RuntimeError):
        layer(x[:, :1], layer_past=present)
    for other in (x[:, :2], x[:1, :1]):              # the step has room for one token of two sequences
        with pytest.raises(ValueError), torch.no_grad():
            layer(other, layer_past=present)
    with pytest.raises(ValueError):
        FlashAttention(32, 2, rotary=RotaryEmbedding(18, 8))


def test_inference_mode_and_training_in_turn():
    layer = FlashAttention(32, 2, fused_qkv=True, causal=True, rotary=RotaryEmbedding(16, 64)).eval()
    x = torch.randn(2, 6, 32)
    with torch.inference_mode():
        cache = PagedKVCache(1, 4, 2, 16, batch=2, max_tokens=32, page=16)
        cache.add(5)
        layer(x[:, :5], layer_past=cache.layer(0))
    out, _ = layer(x)                                  # the table that inference has made
    assert torch.autograd.grad(out.sum(), layer.qkv.weight)[0].abs().sum() > 0
    with torch.no_grad():                              # the cache that inference has made
        cache.add(1)
        layer(x[:, 5:], layer_past=cache.layer(0))
    with torch.inference_mode():
        cache.add(1)
        layer(x[:, 5:], layer_past=cache.layer(0))
    assert cache.lengths.tolist() == [7, 7]


def test_rotated_layer_takes_positions_and_copies():
    layer = FlashAttention(32, 2, fused_qkv=True, causal=True, rotary=RotaryEmbedding(16, 64))
    x = torch.randn(1, 6, 32)
    pos = torch.arange(10, 16)
    a, _ = layer(x, position_ids=pos)
    b, _ = layer(x)
    assert torch.allclose(a, b, atol=1e-5)             # (distances alone count)
    both = torch.cat([x, x])                           # one row of positions for all sequences
    assert torch.equal(layer(both, position_ids=pos[None])[0], layer(both, position_ids=pos)[0])
    c, _ = layer(x, position_ids=torch.tensor([0, 1, 2, 3, 4, 9]))
    assert not torch.allclose(a[:, -1], c[:, -1], atol=1e-3)
    twin = copy.deepcopy(layer).bfloat16()
    assert twin.rotary.table("cpu").dtype == torch.float32 and not list(twin.rotary.parameters())
    assert "rotary" not in "".join(layer.state_dict())
