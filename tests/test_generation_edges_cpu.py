"""Generation over a paged cache at its edges, on the CPU: steps that are run again as a graph would, queries that
are no tokens, sequences longer than the rotation's table, settings of any kind."""
import pytest
import torch

from slapo_b200.op import FlashAttention, PagedKVCache, RotaryEmbedding
from slapo_b200.ops import functional as NF
from slapo_b200.ops import paged
from test_generation_cpu import make_cache


# ---------------------------------------------------------------------- #
# steps of one kind run again after a step of another
def frozen_calls(monkeypatch, layer, x, cache):
    """The calls of a layer's step on a cache, as a graph keeps them: with the tensors (and what is None) that they had,
    outputs among them."""
    calls = []
    for name in ("paged_append", "paged_attention"):
        def call(*args, _f=getattr(paged, name), **kw):
            out = _f(*args, **kw)
            calls.append(lambda: _f(*args, **kw) if out is None else out.copy_(_f(*args, **kw)))
            return out

        monkeypatch.setattr(paged, name, call)
    layer(x, layer_past=cache.layer(0))
    monkeypatch.undo()
    assert len(calls) == 2
    return calls


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("kept,now", [(1, [1, 0, 1]), ([1, 0, 1], 1), ([0, 1, 1], [1, 0, 1]), (1, [0, 0, 0])])
def test_a_steps_calls_serve_every_kind_of_step(monkeypatch, kept, now, rotated):
    torch.manual_seed(0)
    rot = RotaryEmbedding(16, 64) if rotated else None
    layer = FlashAttention(32, 2, fused_qkv=True, causal=True, output_proj=False, rotary=rot).eval()
    prompt, x = torch.randn(3, 7, 32), torch.randn(3, 1, 32)

    def start():
        cache = PagedKVCache(1, 9, 2, 16, batch=3, max_tokens=48, page=16)
        cache.add([7, 5, 1])
        layer(prompt, layer_past=cache.layer(0))
        return cache

    with torch.no_grad():
        cache = start()
        cache.add(kept)
        calls = frozen_calls(monkeypatch, layer, x, cache)
        cache.add(now)
        for call in calls:
            got = call()
        other = start()
        for step in (kept, now):
            other.add(step)
            if other.width:                 # (a step of nothing is not run)
                want, _ = layer(x, layer_past=other.layer(0))
    assert torch.equal(got.flatten(2), want if other.width else torch.zeros_like(want))
    for a, b in ((cache.pages[0].view(torch.uint8), other.pages[0].view(torch.uint8)),
                 (cache.scales[0], other.scales[0]), (cache.lengths, other.lengths),
                 (cache.block_table, other.block_table)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------- #
# queries beside an append
def queries_without_rotation(device):
    """Queries that are none are zeros, with and without counts; the others as they are, in a tensor of their own."""
    k, q = torch.randn(3, 4, 2, 8, device=device).half(), torch.randn(3, 4, 6, 8, device=device).half()
    lengths = torch.tensor([1, 4, 9], dtype=torch.int32, device=device)
    counts = torch.tensor([1, 4, 2], dtype=torch.int32, device=device)
    token = torch.arange(4, device=device)
    for each, there in ((None, lengths[:, None] - 4 + token >= 0), (counts, token < counts[:, None])):
        cache = make_cache(3, 1, 2, 8, 16, device)
        got = NF.paged_append(cache[0], cache[1], k, k, cache[2], lengths, each, q=q)
        assert got.data_ptr() != q.data_ptr()
        assert torch.equal(got, torch.where(there[:, :, None, None], q, torch.zeros_like(q)))
    assert NF.paged_append(cache[0], cache[1], k, k, cache[2], lengths) is None


def query_refusals(device):
    k, q = torch.randn(2, 3, 2, 16, device=device).half(), torch.randn(2, 3, 4, 16, device=device).half()
    pages, scales, table = make_cache(2, 2, 2, 16, 16, device)
    lengths = torch.full((2,), 3, dtype=torch.int32, device=device)

    def append(q):
        return lambda: NF.paged_append(pages, scales, k, k, table, lengths, q=q)

    yield TypeError, append(q.float())
    yield ValueError, append(q[:, :2])
    yield ValueError, append(q[..., :8])
    yield ValueError, append(q[:, 0])
    yield RuntimeError, append(q.clone().requires_grad_())


def test_queries_without_rotation():
    queries_without_rotation("cpu")


@pytest.mark.parametrize("index", range(5))
def test_query_refusals(index):
    error, call = list(query_refusals("cpu"))[index]
    with pytest.raises(error):
        call()


# ---------------------------------------------------------------------- #
# sequences longer than the rotation's table
@pytest.mark.parametrize("fused", [False, True])
def test_a_sequence_longer_than_the_rotations_table_is_refused(fused):
    layer = FlashAttention(32, 2, fused_qkv=fused, causal=True, rotary=RotaryEmbedding(16, 8)).eval()
    x = torch.randn(2, 12, 32)
    with torch.no_grad():
        layer(x[:, :8])
        layer(x, position_ids=torch.arange(12).clamp(max=7))       # (positions on the device: zeros behind the table)
        with pytest.raises(ValueError, match="8 positions"):
            layer(x)
        past = layer(x[:, :8], use_cache=True)[1]
        with pytest.raises(ValueError, match="8 positions"):
            layer(x[:, 8:9], layer_past=past)
        # a cache whose sequences can get longer, whatever they have now: a captured step is not asked again
        cache = PagedKVCache(1, 4, 2, 16, batch=2, max_tokens=9, page=16)
        cache.add(1)
        with pytest.raises(ValueError, match="8 positions"):
            layer(x[:, :1], layer_past=cache.layer(0))
        cache = PagedKVCache(1, 4, 2, 16, batch=2, max_tokens=8, page=16)
        for n in (7, 1):
            cache.add(n)
            layer(x[:, :n], layer_past=cache.layer(0))


def test_rotation_of_no_tokens():
    table = NF.rotary_table(8, 4)
    q, qkv = torch.randn(2, 3, 2, 16), torch.randn(2, 3, 2, 3, 16)
    for part in (slice(0), (slice(None), slice(0))):
        for got in NF.rotary(q[part], q[part][:, :, :1], table):
            assert got.shape[:2] == q[part].shape[:2] and got.shape[3] == 16
        assert NF.rotary_qkvpacked(qkv[part], table, 9).shape == qkv[part].shape


def test_a_rotation_past_the_end_of_its_table_is_refused():
    rot = RotaryEmbedding(8, 8)
    q = torch.randn(1, 3, 2, 8)
    rot(q, q, 5), rot(q, q, -2), rot(q[:, :0], q[:, :0], 8)
    rot.forward_packed(torch.randn(1, 8, 2, 3, 8))
    for call in (lambda: rot(q, q, 6), lambda: rot(torch.randn(1, 9, 1, 8), torch.randn(1, 9, 1, 8)),
                 lambda: rot.forward_packed(torch.randn(1, 9, 2, 3, 8))):
        with pytest.raises(ValueError, match="8 positions"):
            call()


# ---------------------------------------------------------------------- #
# settings and tables of any kind: the same on the CPU and the GPU
def whole_numbers(device):
    x, u = torch.randn(2, 50, device=device), torch.rand(2, device=device)
    assert torch.equal(NF.sample(x, u, top_k=5.0), NF.sample(x, u, top_k=5))
    for bad, error in ((1.5, TypeError), (-1.0, ValueError), (float("nan"), ValueError), (float("inf"), TypeError),
                       ("5", TypeError)):
        with pytest.raises(error):
            NF.sample(x, u, top_k=bad)


def numbers_from_tables(device):
    """Random numbers and settings that are columns of a table."""
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(6, 70, generator=g) * 3).to(device)
    u = torch.rand(6, 9, generator=g).to(device)
    t, p, m = (torch.rand(6, 2, generator=g).to(device) for _ in range(3))
    k = torch.randint(0, 70, (6, 2), generator=g).int().to(device)
    for i in range(2):
        got = NF.sample(x, u[:, i], t[:, i], k[:, i], p[:, i], m[:, i])
        assert torch.equal(got, NF.sample(x, *(a[:, i].contiguous() for a in (u, t, k, p, m))))
    assert torch.equal(NF.sample(x, u[:1, :1].expand(6, 1)), NF.sample(x, u[:1, 0].repeat(6)))


def tables_in_other_strides(device):
    """A rotation's table as a slice of a wider one, transposed, and on 4 bytes."""
    table = NF.rotary_table(8, 40, device=device)
    wide = torch.empty(40, 6, 3, device=device)[:, 1:5, 1:].copy_(table)
    turned = table.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    odd = torch.empty(table.numel() + 1, device=device)[1:].view(table.shape).copy_(table)
    x = torch.randn(2, 9, 3, 8, device=device).half()
    lengths = torch.tensor([9, 30], dtype=torch.int32, device=device)
    results = []
    for rot in (table, wide, turned, odd):
        a, b = (x.clone().requires_grad_() for _ in range(2))
        y, z = NF.rotary(a, b[:, :, :1], rot, 3)
        grads = torch.autograd.grad((y, z), (a, b), (x, x[:, :, :1]))
        pages, scales, tab = make_cache(2, 2, 3, 8, 16, device, poison=False)
        q = NF.paged_append(pages, scales, x, x, tab, lengths, q=x, rotary_table=rot)
        results.append((y, z, *grads, NF.rotary_qkvpacked(torch.stack([x, x, x], 3), rot, 3), q, pages.float(), scales))
    for other in results[1:]:
        for got, want in zip(other, results[0]):
            assert torch.equal(got, want)


def test_whole_numbers():
    whole_numbers("cpu")


def test_numbers_from_tables():
    numbers_from_tables("cpu")


def test_tables_in_other_strides():
    tables_in_other_strides("cpu")
