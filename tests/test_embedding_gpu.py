"""Token table on the GPU: lookup and gradient against 64 bits, over lengths, widths, types and repeated
ids."""
import pytest
import torch

from slapo_b200.op import FusedEmbedding
from slapo_b200.ops import functional as NF
from slapo_b200.ops import native

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _ids(n, vocab, kind, dtype=torch.int64):
    if kind == "one":
        ids = torch.full((n,), vocab - 1)
    elif kind == "order":
        ids = torch.arange(n) % vocab
    else:        # frequent small ids, a few rare large ones
        ids = (vocab ** torch.rand(n, dtype=torch.float64)).long() - 1
        ids = ids.clamp(0, vocab - 1)
    return ids.to("cuda", dtype)


def _check(ids, w, dy, scale, padding=None, start=0):
    """Output and gradient against the definition in 64 bits."""
    w = w.detach().requires_grad_()
    out = NF.embedding(ids, w, padding_idx=padding, scale=scale, vocab_start=start)
    got = torch.autograd.grad(out, w, dy)[0]
    assert got.dtype == w.dtype and got.shape == w.shape and got.is_contiguous()
    row = ids.long().reshape(-1) - start
    own = (row >= 0) & (row < w.shape[0])
    want = torch.zeros(row.numel(), w.shape[1], dtype=torch.float64, device="cuda")
    want[own] = w.detach().double()[row[own]] * scale
    half = HALF[w.dtype]
    tiny = torch.finfo(w.dtype).smallest_normal * half     # (below it steps stay as they are)
    assert bool(((out.detach().double().view_as(want) - want).abs()
                 <= want.abs() * half * (1 + 2.0 ** -20) + want.abs() * 2.0 ** -23 + tiny).all())
    if padding is not None:
        own &= ids.reshape(-1) != padding
    rows = dy.double().reshape(-1, w.shape[1])[own]
    total = torch.zeros(w.shape, dtype=torch.float64, device="cuda").index_add_(0, row[own], rows)
    size = torch.zeros_like(total).index_add_(0, row[own], rows.abs())
    count = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda").index_add_(
        0, row[own], torch.ones_like(row[own], dtype=torch.float64))
    # a sum of c terms in fp32 is off by at most (c - 1) half steps of the sum of their absolute values, the
    # factor by one more, and the result is rounded once
    bound = scale * size * (count[:, None] + 1) * 2.0 ** -24 + tiny
    bound += (total * scale).abs() * half * (1 + 2.0 ** -20)
    assert bool(((got.double() - total * scale).abs() <= bound).all())
    assert bool((got[count == 0] == 0).all())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 8), (1, 5, 1), (31, 7, 33), (33, 255, 64), (200, 256, 100),
                                          (777, 257, 8), (2049, 1000, 128), (5000, 65536, 16),
                                          (4100, 70001, 7)])
def test_lengths_and_widths(n, vocab, cols, dtype):
    for kind in ("order", "zipf", "one"):
        ids = _ids(n, vocab, kind)
        _check(ids, torch.randn(vocab, cols, device="cuda", dtype=dtype),
               torch.randn(n, cols, device="cuda", dtype=dtype), 3.25)


@pytest.mark.parametrize("n", [16384, 20001, 70000])
@pytest.mark.parametrize("kind", ["zipf", "one"])
def test_many_tokens(n, kind):
    ids = _ids(n, 3001, kind, torch.int32).view(1, -1)
    _check(ids, torch.randn(3001, 48, device="cuda", dtype=torch.bfloat16),
           torch.randn(1, n, 48, device="cuda", dtype=torch.bfloat16), 1.0)


def test_padding_and_other_shards_ids():
    ids = torch.randint(0, 900, (6, 301), device="cuda")
    ids[:, 200:] = 350
    ids[0, 0] = -5
    w = torch.randn(400, 24, device="cuda", dtype=torch.float16)
    dy = torch.randn(6, 301, 24, device="cuda", dtype=torch.float16)
    got = _check(ids, w, dy, 0.5, padding=350, start=300)
    assert bool((got[50] == 0).all())


def test_no_tokens_and_no_rows():
    w = torch.randn(9, 16, device="cuda", requires_grad=True)
    out = NF.embedding(torch.zeros(0, dtype=torch.long, device="cuda"), w)
    assert out.shape == (0, 16)
    assert torch.equal(torch.autograd.grad(out.sum(), w)[0], torch.zeros(9, 16, device="cuda"))
    empty = torch.randn(0, 16, device="cuda", requires_grad=True)
    out = NF.embedding(torch.tensor([0, 3], device="cuda"), empty)
    assert torch.equal(out, torch.zeros(2, 16, device="cuda"))
    assert torch.autograd.grad(out.sum(), empty)[0].shape == (0, 16)


def test_strides_and_alignment():
    base = torch.randn(300, 81, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn(50, 64, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(0, 300, (100,), device="cuda")[::2]
    for w in (base[:, :64], base[:, 1:65], torch.randn(64, 300, device="cuda", dtype=torch.bfloat16).t()):
        _check(ids, w, dy, 1.5)
    flat = torch.randn(50 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    for g in (flat[1:].view(50, 64), dy[:, :1].expand(50, 64), dy.t().contiguous().t()):
        _check(ids, base[:, :64], g, 1.0)


def test_same_result_every_time():
    ids = _ids(30000, 500, "zipf")
    dy = torch.randn(30000, 40, device="cuda")
    first = native.ops().embedding_bwd(dy, ids, 500, 0, None, 1.0)
    for _ in range(5):
        assert torch.equal(native.ops().embedding_bwd(dy, ids, 500, 0, None, 1.0), first)


def test_gradient_against_differences():
    w = torch.randn(11, 6, device="cuda", requires_grad=True)
    ids = torch.randint(0, 11, (40,), device="cuda")
    c = torch.randn(40, 6, device="cuda")
    f = lambda t: (NF.embedding(ids, t, scale=2.0).double() * c.double()).sum()      # noqa: E731
    grad = torch.autograd.grad(f(w), w)[0]
    step = torch.randn_like(w)
    # linear in the table: a difference of any length has no error but rounding, 2^-24 of each of 240 terms
    diff = (f(w.detach() + step) - f(w.detach() - step)) / 2
    want = (grad.double() * step.double()).sum()
    size = (2 * (w.detach().abs().amax() + step.abs().amax()) * c.abs().sum()).double()
    assert abs(float(diff - want)) <= float(size) * 4 * 2.0 ** -24


def test_captured_and_on_another_stream():
    emb = FusedEmbedding(1000, 64, padding_idx=0, scale=8.0, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(0, 1000, (4, 100), device="cuda")
    dy = torch.randn(4, 100, 64, device="cuda", dtype=torch.bfloat16)

    def both():
        out = emb(ids)
        return out, torch.autograd.grad(out, emb.weight, dy)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = both()
    for seed in range(3):
        torch.manual_seed(seed)
        ids.copy_(torch.randint(0, 1000, (4, 100), device="cuda"))
        dy.normal_()
        graph.replay()
        want, want_grad = both()
        assert torch.equal(out, want) and torch.equal(grad, want_grad)


def test_refusals():
    w = torch.randn(10, 8, device="cuda")
    ids = torch.tensor([1, 2], device="cuda")
    with pytest.raises(RuntimeError, match="device"):
        NF.embedding(ids.cpu(), w)
    with pytest.raises(RuntimeError, match="one row"):
        native.ops().embedding_bwd(torch.randn(3, 8, device="cuda"), ids, 10, 0, None, 1.0)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        native.ops().embedding_fwd(ids.short(), w, 0, 1.0)


@pytest.mark.parametrize("padding", [None, 3])
def test_second_derivatives(padding):
    """Lookup and gradient are each other's derivative: as indexing the table in 64 bits, to the roundings of
    the chain (2^-24 each, sums of fewer than 64 terms)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(9, 8, device="cuda", generator=g).requires_grad_()
    x = torch.randn(40, 8, device="cuda", generator=g).requires_grad_()
    ids = torch.randint(-1, 10, (40,), device="cuda", generator=g)      # (two of them outside of the table)

    def third(w, x, lookup):
        out = lookup(w)
        (dw,) = torch.autograd.grad((out ** 3 * x).sum(), w, create_graph=True)
        dw2, dx2 = torch.autograd.grad((dw ** 2).sum(), (w, x), create_graph=True)
        return [dw, dw2, dx2, *torch.autograd.grad((dw2 * dw).sum() + (dx2 ** 2).sum(), (w, x))]

    def plain(w):
        own = (ids >= 0) & (ids < 9)
        rows = w[ids.clamp(0, 8)]
        if padding is not None:
            rows = torch.where((ids != padding)[:, None], rows, rows.detach())
        return torch.where(own[:, None], rows, 0.0) * 1.5

    got = third(w, x, lambda w: NF.embedding(ids, w, padding_idx=padding, scale=1.5))
    w64, x64 = (t.detach().double().requires_grad_() for t in (w, x))
    want = third(w64, x64, plain)
    for a, b in zip(got, want):
        assert bool(((a.double() - b).abs() <= 256 * 2.0 ** -24 * b.abs().max()).all())


def test_offsets_beyond_32_bits():
    """A table and a gradient of more than 2^31 elements, each row by one token."""
    rows, cols = 270_000, 8192
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randperm(rows, device="cuda", generator=g)
    w = torch.randn(rows, 1, device="cuda", generator=g).to(torch.bfloat16)
    w = (w * torch.linspace(1, 2, cols, device="cuda", dtype=torch.bfloat16)).requires_grad_()
    out = NF.embedding(ids, w)
    assert torch.equal(out.detach(), w.detach()[ids])
    (dw,) = torch.autograd.grad(out, w, out.detach())
    assert torch.equal(dw, w.detach())


def test_the_same_row_as_parameter_of_two_lookups():
    """A table that is looked up twice in a step: gradients add up."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(50, 16, device="cuda", generator=g).requires_grad_()
    a, b = (torch.randint(0, 50, (n,), device="cuda", generator=g) for n in (30, 70))
    (NF.embedding(a, w).sum() + NF.embedding(b, w, scale=2.0).sum()).backward()
    want = torch.bincount(a, minlength=50) + 2 * torch.bincount(b, minlength=50)
    assert torch.equal(w.grad, want[:, None].float().expand(50, 16))


def test_more_tokens_than_the_sort_numbers():
    """Refused before anything is allocated or copied (ids and gradient are one element each, seen many times)."""
    ids = torch.zeros(1, device="cuda", dtype=torch.int32)
    dy = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16)
    held, launches = torch.cuda.memory_allocated(), native.launch_count()
    for n in (2 ** 31 - 8191, 2 ** 31 - 256, 2 ** 31, 2 ** 33):
        with pytest.raises(RuntimeError, match="at most 2147475456 ids"):
            native.ops().embedding_bwd(dy.expand(n, 1), ids.expand(n), 4, 0, None, 1.0)
    assert torch.cuda.memory_allocated() == held and native.launch_count() == launches


# (94208 tokens are the last whose sort stays in shared memory: eight CTAs' slices of 11776)
@pytest.mark.parametrize("n", [94208, 94209, 150001])
@pytest.mark.parametrize("kind", ["zipf", "one"])
def test_sort_through_global_memory(n, kind):
    """Repeated ids, rows over many stretches, a padding id and ids of other shards, in one and two passes."""
    for vocab in (200, 3001):
        ids = _ids(n, vocab + 20, kind)
        ids[n // 2:n // 2 + 1000] = 40
        got = _check(ids, torch.randn(vocab, 24, device="cuda", dtype=torch.bfloat16),
                     torch.randn(n, 24, device="cuda", dtype=torch.bfloat16), 0.5, padding=40, start=10)
        assert bool((got[30] == 0).all())


@pytest.mark.parametrize("rows", [30, 300, 12500, 20000])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_tokens_of_a_row_stay_in_their_order(rows, dtype):
    """Eight tokens to each row: a warp adds up one row's, so that the result has the order of the tokens, to
    the bit.  (The sort goes through shared memory for the first two, through global memory for the others.)"""
    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = torch.arange(8 * rows, device="cuda")[torch.randperm(8 * rows, device="cuda", generator=g)] % rows
    dy = torch.randn(8 * rows, 12, device="cuda", generator=g)
    got = native.ops().embedding_bwd(dy, ids.to(dtype), rows, 0, None, 1.0)
    of_row = dy[torch.argsort(ids, stable=True)].view(rows, 8, 12)
    want = torch.zeros(rows, 12, device="cuda")
    for i in range(8):
        want = want + of_row[:, i]
    other = torch.zeros(rows, 12, device="cuda")
    for i in reversed(range(8)):
        other = other + of_row[:, i]
    assert torch.equal(got, want) and not torch.equal(got, other)


def test_after_a_function_transform():
    """A transform that is over does not keep calls from the entry without the dispatcher, nor makes a node."""
    torch.func.vmap(lambda x: x + 1)(torch.zeros(2, device="cuda"))
    w = torch.randn(10, 8, device="cuda")
    ids = torch.tensor([1, 2], device="cuda")
    assert torch.equal(native.direct("embedding")(ids, w, 0, None, 1.0), w[ids])
    q = torch.randn(1, 1, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert native.direct("flash")(q, q, q, None, True, None, 4, 0) is not None

    def inside(x):
        assert native.direct("embedding")(ids, w, 0, None, 1.0) is None
        return x + 1

    torch.func.vmap(inside)(torch.zeros(2, device="cuda"))
    # (inside, the operator's node says that it does not take transforms)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: NF.embedding(ids, t).sum())(w)
