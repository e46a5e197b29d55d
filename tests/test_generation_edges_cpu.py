"""Generation over a paged cache at its edges, on the CPU: steps that are run again as a graph would, queries that
are no tokens, sequences longer than the rotation's table, settings of any kind."""
import pytest
import torch

from slapo_b200.op import FlashAttention, PagedKVCache, RotaryEmbedding
from slapo_b200.ops import paged


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
