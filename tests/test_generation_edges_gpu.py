"""Generation over a paged cache at its edges, on the GPU: captured steps of every kind, weights far below the largest,
values that are not finite beside rotated ones, windows of more than 2^30 keys, settings of any kind."""
import pytest
import torch

from slapo_b200.op import FlashAttention, PagedKVCache, RotaryEmbedding
from slapo_b200.ops import functional as NF
from slapo_b200.ops.paged import paged_append_reference
from test_generation_cpu import make_cache
from test_generation_edges_cpu import (numbers_from_tables, queries_without_rotation, query_refusals,
                                       tables_in_other_strides, whole_numbers)

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ---------------------------------------------------------------------- #
# captured steps
def _layers(rotated, window=None):
    torch.manual_seed(0)
    rot = RotaryEmbedding(64, 256) if rotated else None
    blocks = [FlashAttention(256, 4, fused_qkv=True, causal=True, window=window, rotary=rot) for _ in range(2)]
    return [b.to("cuda", torch.bfloat16).eval() for b in blocks]


def _run(blocks, cache, x):
    for i, block in enumerate(blocks):
        x = x + block(x, layer_past=cache.layer(i), use_cache=True)[0]
    return x


def _captured(step):
    """A graph of a step, its output, and what the step gave before it was captured."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out, before


def _same(cache, other):
    for a, b in zip((*cache.pages, *cache.scales), (*other.pages, *other.scales)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(cache.lengths, other.lengths) and torch.equal(cache.block_table, other.block_table)


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("kept,steps", [(1, [1, [1, 0, 1], [0, 1, 1], 1, [0, 0, 0], 1]),
                                        ([1, 0, 1], [[1, 0, 1], 1, [0, 1, 0], 1]),
                                        (3, [3, [1, 3, 0], [3, 2, 1], 3]),
                                        ([3, 0, 2], [[3, 0, 2], 3, [0, 3, 3], 1])])
def test_a_captured_step_serves_every_kind_of_step(kept, steps, rotated):
    """Replayed after steps of every kind: the same as eager ones, codes and scales among it."""
    blocks = _layers(rotated)
    width = kept if isinstance(kept, int) else max(kept)
    prompt = torch.randn(3, 30, 256, device="cuda").bfloat16()
    xs = torch.randn(len(steps), 3, width, 256, device="cuda").bfloat16()

    def start():
        cache = PagedKVCache(2, 30, 4, 64, batch=3, max_tokens=128, page=16, device="cuda")
        cache.add([30, 17, 1])
        _run(blocks, cache, prompt)
        return cache

    with torch.no_grad():
        cache, other = start(), start()
        x = xs[0].clone()
        cache.add(kept)
        graph, out, _ = _captured(lambda: _run(blocks, cache, x))
        for i, step in enumerate(steps):
            if i > 0:
                cache.add(step)
            x.copy_(xs[i])
            graph.replay()
            other.add(step)
            other.width = width         # (a narrower step, padded: projections of other sizes round in other orders)
            want = _run(blocks, other, xs[i])
            each = [step] * 3 if isinstance(step, int) else step
            for b, n in enumerate(each):
                assert torch.equal(out[b, :n], want[b, :n])
            _same(cache, other)


@pytest.mark.parametrize("window", [None, 9])
def test_a_captured_step_of_an_empty_cache_serves_later_ones(window):
    blocks = _layers(True, window)
    xs = torch.randn(4, 2, 20, 256, device="cuda").bfloat16()

    def start():
        return PagedKVCache(2, 20, 4, 64, batch=2, max_tokens=128, page=16, device="cuda")

    with torch.no_grad():
        cache, other = start(), start()
        x = xs[0].clone()
        cache.add(20)
        graph, out, eager = _captured(lambda: _run(blocks, cache, x))
        for i, step in enumerate((20, 20, [7, 20])):
            if i > 0:
                cache.add(step)
            x.copy_(xs[i])
            graph.replay()
            other.add(step)
            want = _run(blocks, other, xs[i])
            if i == 0:          # a prompt's first tokens: over keys as they are where a call is eager, else in 8 bits
                assert torch.equal(want, eager)
                assert (out.float() - want.float()).norm() <= 0.1 * want.float().norm()
                # (what the second layer has kept follows from the first one's output: taken over)
                for a, b in zip((*other.pages, *other.scales), (*cache.pages, *cache.scales)):
                    a.copy_(b)
                continue
            for b, n in enumerate([step] * 2 if isinstance(step, int) else step):
                assert torch.equal(out[b, :n], want[b, :n])
            _same(cache, other)


def test_queries_in_32_bits_are_not_captured():
    layer = FlashAttention(64, 2, fused_qkv=True, causal=True, output_proj=False).cuda().eval()
    cache = PagedKVCache(1, 4, 2, 32, batch=2, max_tokens=32, page=16, device="cuda")
    x = torch.randn(2, 3, 64, device="cuda")
    with torch.no_grad():
        cache.add(3)
        want, _ = layer(x, layer_past=cache.layer(0))
        with pytest.raises(RuntimeError, match="not captured"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            layer(x, layer_past=cache.layer(0))
        assert torch.equal(layer(x, layer_past=cache.layer(0))[0], want)


# ---------------------------------------------------------------------- #
# queries beside an append, settings of any kind
def test_queries_without_rotation():
    queries_without_rotation("cuda")


def test_queries_of_many_tokens_without_rotation():
    q = torch.randn(3, 700, 6, 80, device="cuda").half()
    k = torch.randn(3, 700, 2, 80, device="cuda").half()
    lengths = torch.tensor([700, 650, 960], dtype=torch.int32, device="cuda")
    mine, oracle = (make_cache(3, 32, 2, 80, 32, "cuda", poison=False) for _ in range(2))
    got = NF.paged_append(mine[0], mine[1], k, k, mine[2], lengths, q=q)
    assert torch.equal(got, paged_append_reference(oracle[0], oracle[1], k, k, oracle[2], lengths, q=q))
    assert bool((got[1, :50] == 0).all()) and torch.equal(mine[0].view(torch.uint8), oracle[0].view(torch.uint8))


@pytest.mark.parametrize("index", range(5))
def test_query_refusals(index):
    error, call = list(query_refusals("cuda"))[index]
    with pytest.raises(error):
        call()


def test_whole_numbers():
    whole_numbers("cuda")


def test_numbers_from_tables():
    numbers_from_tables("cuda")


def test_tables_in_other_strides():
    tables_in_other_strides("cuda")


# ---------------------------------------------------------------------- #
# values beside the rotated ones
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dim,rotated", [(24, 4), (24, 20), (128, 100), (80, 40)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_behind_the_rotated_ones_stay(interleaved, dim, rotated, n):
    """Infinities and NaN behind the rotated part do not reach their neighbours."""
    rot = NF.rotary_table(rotated, 64, device="cuda")
    k, q = (torch.randn(2, n, h, dim, device="cuda") for h in (2, 3))
    for x in (k, q):
        x[0, 0, 0, rotated], x[1, n - 1, 1, rotated + 3], x[1, 0, 0, rotated + 1] = float("inf"), float("nan"), -float("inf")
    lengths = torch.tensor([n, n + 9], dtype=torch.int32, device="cuda")
    mine, oracle = (make_cache(2, 4, 2, dim, 16, "cuda", poison=False) for _ in range(2))
    got = NF.paged_append(mine[0], mine[1], k, k, mine[2], lengths, q=q, rotary_table=rot, interleaved=interleaved)
    want = paged_append_reference(oracle[0], oracle[1], k, k, oracle[2], lengths, q=q, rotary_table=rot, interleaved=interleaved)
    assert torch.equal(got[..., rotated:].nan_to_num(5.0), q[..., rotated:].nan_to_num(5.0))
    assert torch.equal(got.isnan(), want.isnan())
    a, b = mine[0].float(), oracle[0].float()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(mine[1], oracle[1])


# ---------------------------------------------------------------------- #
# attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 12, 40])
def test_weights_far_below_the_largest_count(n, dtype):
    """A first key far ahead whose value is zero, and a long row of equal ones: their values by their exact weights.

    So many items that a warp has whole sequences, under one maximum.  A weight is rounded to fp16, 2^-11 of itself
    whatever its size; a score (up to 19) is off by 2^-20 of itself, and exp2 and the sums in fp32 are far better than
    2^-12; the output is rounded once."""
    batch, kv, dim, page, length = 64, 32, 64, 64, 12001
    per = (length + page - 1) // page
    pages = torch.zeros(per, 2, kv, page, dim, device="cuda")
    pages[0, 0, :, 0] = 64.0                                          # keys: the first one, as 1
    g = torch.Generator(device="cuda").manual_seed(n)
    pages[:, 1] = torch.rand(per, kv, page, dim, generator=g, device="cuda") * 64.0 + 32.0
    pages[0, 1, :, 0] = 0.0
    pages = pages.to(torch.float8_e4m3fn)
    scales = torch.full((per, 2, kv), 2.0 ** -6, device="cuda")
    table = torch.arange(per, dtype=torch.int32, device="cuda").repeat(batch, 1)      # (full pages, but for the last: shared)
    lengths = torch.full((batch,), length, dtype=torch.int32, device="cuda")
    size = torch.tensor([2.0, 2.0625, 2.125, 2.25, 2.375], device="cuda")[torch.arange(batch, device="cuda") % 5]
    q = size[:, None, None, None].expand(batch, n, kv, dim).to(dtype)
    got = NF.paged_attention(q, pages, scales, table, lengths).double()
    values = (pages[:, 1].double() * 2.0 ** -6).transpose(1, 2).reshape(-1, kv, dim)[:length].cumsum(0)[length - n:]
    others = torch.arange(length - n, length, device="cuda").double()                  # beside the first
    for b in range(5):
        score = float(size[b]) * 8.0
        want = values / (others + torch.tensor(score, dtype=torch.float64).exp().item())[:, None, None]
        off = ((got[b::5] - want) / want).abs().max()
        assert float(off) <= HALF[dtype] + 2.0 ** -11 + 2.0 ** -12 + score * 2.0 ** -20, float(off)


@pytest.mark.parametrize("group,length", [(1, 100), (4, 100), (20, 100), (1, 3)])
def test_values_near_the_types_largest(group, length):
    """The mean of equal values of 2^120."""
    pages, scales, table = make_cache(2, 4, 2, 64, 32, "cuda", poison=False)
    pages[:, 1] = torch.full_like(pages[:, 1].float(), 256.0).to(pages.dtype)
    scales[:, 0], scales[:, 1] = 1.0, 2.0 ** 112
    q = torch.zeros(2, 1, 2 * group, 64, device="cuda", dtype=torch.bfloat16)
    got = NF.paged_attention(q, pages, scales, table, torch.tensor([length, 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(got.float(), torch.full_like(got, 2.0 ** 120, dtype=torch.float32))


def test_a_window_of_more_than_two_to_the_thirty_keys():
    """One page in all places of the table but the first, whose first key outweighs all others."""
    length, page = (1 << 30) + 1000, 128
    pages = torch.zeros(2, 2, 1, page, 16, device="cuda")
    pages[1, 0, 0, 0], pages[1, 1, 0, 0] = 4.0, 1.0
    pages = pages.to(torch.float8_e4m3fn)
    scales = torch.ones(2, 2, 1, device="cuda")
    table = torch.zeros(1, (length + page - 1) // page, dtype=torch.int32, device="cuda")
    table[0, 0] = 1
    lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
    q = torch.full((1, 1, 1, 8), 8.0, device="cuda", dtype=torch.bfloat16)
    for window in (length, length + 5, (1 << 31) - 1, 1 << 40, None):
        assert bool((NF.paged_attention(q, pages, scales, table, lengths, window=window) == 1).all()), window
    assert bool((NF.paged_attention(q, pages, scales, table, lengths, window=length - 1) == 0).all())
