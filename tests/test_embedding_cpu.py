"""Token table: the plain form against nn.Embedding, what it does with ids of other shards, and refusals."""
import pytest
import torch

from slapo_b200.op import FusedEmbedding
from slapo_b200.ops import functional as NF


def test_is_nn_embedding_with_a_factor():
    emb = torch.nn.Embedding(50, 12, padding_idx=3)
    fused = FusedEmbedding.from_embedding(emb, scale=2.5)
    assert fused.weight is emb.weight
    ids = torch.randint(0, 50, (4, 9))
    ids[:, 2] = 3
    out, ref = fused(ids), emb(ids) * 2.5
    torch.testing.assert_close(out, ref, rtol=2.0 ** -23, atol=0)
    dy = torch.randn(4, 9, 12)
    got = torch.autograd.grad(out, fused.weight, dy)[0]
    want = torch.autograd.grad(ref, emb.weight, dy)[0]
    # sums of up to 36 terms in another order, and the factor before or after
    torch.testing.assert_close(got, want, rtol=2.0 ** -20, atol=40 * 2.0 ** -22)
    assert bool((got[3] == 0).all())


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_shards_add_up_to_the_table(dtype):
    w = torch.randn(40, 6)
    ids = torch.randint(0, 40, (5, 7), dtype=dtype)
    parts = []
    for lo in (0, 10, 30):
        shard = w[lo:lo + (20 if lo == 10 else 10)].clone().requires_grad_()
        out = NF.embedding(ids, shard, vocab_start=lo)
        out.sum().backward()
        count = torch.stack([(ids == lo + r).sum() for r in range(shard.shape[0])]).float()
        assert torch.equal(shard.grad, count[:, None].expand(-1, 6))
        parts.append(out)
    assert torch.equal(sum(parts), w[ids.long()])


def test_ids_outside_give_zeros():
    w = torch.randn(4, 3)
    out = NF.embedding(torch.tensor([-1, 0, 3, 4, 2 ** 40]), w)
    assert torch.equal(out, torch.stack([w[0] * 0, w[0], w[3], w[0] * 0, w[0] * 0]))
    assert NF.embedding(torch.zeros(0, dtype=torch.long), w).shape == (0, 3)
    assert torch.equal(NF.embedding(torch.tensor([0, 1]), torch.zeros(0, 3)), torch.zeros(2, 3))


def test_refusals():
    w = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="2-D"):
        NF.embedding(torch.tensor([0]), torch.zeros(4))
    with pytest.raises(TypeError, match="int64"):
        NF.embedding(torch.tensor([0.0]), w)
    with pytest.raises(ValueError, match="padding_idx"):
        NF.embedding(torch.tensor([0]), w, padding_idx=-1)
    for kw in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(ValueError, match="not supported"):
            FusedEmbedding.from_embedding(torch.nn.Embedding(4, 3, **kw))
