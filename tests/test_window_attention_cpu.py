"""Attention with a window and sinks, plain form: against the definition key by key, its module forms over a
cache, rows that see nothing and refusals."""
import math

import pytest
import torch

from slapo_b200.op import FlashAttention, FlashAttentionOp
from slapo_b200.ops import functional as NF
from slapo_b200.ops.flash_attn import flash_attention_qkvpacked


def _by_key(q, k, v, window, sinks, bias):
    """Every query on its own, in 64 bits."""
    b, sq, h, d = q.shape
    sk = k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for n in range(b):
        for i in range(sq):
            pos = i + sk - sq
            see = [j for j in range(sk) if j <= pos and (j > pos - window or j < sinks)
                   and (bias is None or bias[n, j] >= -1e30)]
            if not see:
                continue
            for m in range(h):
                s = k[n, see, m].double() @ q[n, i, m].double() / math.sqrt(d)
                if bias is not None:
                    s = s + bias[n, see].double()
                out[n, i, m] = torch.softmax(s, 0) @ v[n, see, m].double()
    return out


@pytest.mark.parametrize("sq,sk,window,sinks", [(9, 9, 1, 0), (9, 9, 3, 0), (9, 9, 3, 2), (7, 12, 4, 1),
                                                (1, 12, 5, 3), (12, 7, 2, 1), (9, 9, 50, 0),
                                                (9, 9, 2, 50), (1, 1, 1, 1)])
@pytest.mark.parametrize("mask", [None, "finite", "lowest", "inf"])
def test_against_the_definition(sq, sk, window, sinks, mask):
    g = torch.Generator().manual_seed(sq * 100 + sk)
    q = torch.randn(2, sq, 2, 8, generator=g)
    k, v = (torch.randn(2, sk, 2, 8, generator=g) for _ in range(2))
    bias = None
    if mask is not None:
        low = {"finite": -3.0, "lowest": torch.finfo(torch.float32).min, "inf": -math.inf}[mask]
        bias = torch.where(torch.rand(2, sk, generator=g) < 0.5, low, 0.0)
        bias[1] = low
    got = NF.flash_attention(q, k, v, bias, causal=True, window=window, sinks=sinks)
    want = _by_key(q, k, v, window, sinks, bias)
    torch.testing.assert_close(got.double(), want, rtol=2.0 ** -18, atol=2.0 ** -18)


def test_rows_that_see_nothing_have_no_gradient():
    q = torch.randn(1, 5, 1, 8, requires_grad=True)
    k, v = (torch.randn(1, 3, 1, 8, requires_grad=True) for _ in range(2))
    out = NF.flash_attention(q, k, v, causal=True, window=2)     # the first two queries precede all keys
    assert bool((out[0, :2] == 0).all())
    out.square().sum().backward()
    assert bool((q.grad[0, :2] == 0).all()) and all(bool(torch.isfinite(t.grad).all()) for t in (q, k, v))


def test_wide_window_is_causal_attention():
    q, k, v = (torch.randn(2, 17, 3, 8) for _ in range(3))
    wide = NF.flash_attention(q, k, v, causal=True, window=17)
    want = NF.flash_attention(q, k, v, causal=True)
    torch.testing.assert_close(wide, want, rtol=2.0 ** -20, atol=2.0 ** -20)


@pytest.mark.parametrize("sinks", [0, 2])
def test_generation_over_a_cache(sinks):
    """Token by token over a growing cache = the whole sequence at once."""
    torch.manual_seed(0)
    block = FlashAttention(32, 4, fused_qkv=True, output_proj=True, causal=True, window=5, sinks=sinks).eval()
    x = torch.randn(2, 14, 32)
    with torch.no_grad():
        want, _ = block(x)
        past, got = None, []
        for t in range(14):
            out, past = block(x[:, t:t + 1], layer_past=past, use_cache=True)
            got.append(out)
    torch.testing.assert_close(torch.cat(got, 1), want, rtol=2.0 ** -16, atol=2.0 ** -16)


def test_general_bias_and_reference_name():
    q, k, v = (torch.randn(1, 6, 2, 8) for _ in range(3))
    bias = torch.zeros(1, 2, 6, 6)
    want = NF.flash_attention(q, k, v, causal=True, window=3, sinks=1)
    for op in (FlashAttentionOp(apply_causal_mask=True, window=3, sinks=1),
               FlashAttentionOp("reference", apply_causal_mask=True, window=3, sinks=1)):
        assert torch.equal(op(q, k, v), want)
        assert torch.equal(op(q, k, v, bias), want)
    assert "window=3" in repr(op)


@pytest.mark.parametrize("disable", [False, True])
def test_local_layers_of_gpt_neo(disable):
    """A configuration's local layers, in the plain model and under the recipe."""
    import slapo_b200 as slapo
    from slapo_b200.model_schedule import apply_schedule
    from slapo_b200.models import GPT2LMHeadModel, GPTConfig, GPTNeoForCausalLM

    kw = dict(vocab_size=64, n_positions=32, hidden_size=32, num_layers=3, num_heads=4, resid_dropout=0.0,
              embed_dropout=0.0, attention_dropout=0.0, model_type="gpt_neo", window_size=4)
    torch.manual_seed(1)
    plain = GPTNeoForCausalLM(GPTConfig(**kw)).eval()
    config = GPTConfig(**kw, attention_layers=("global", "local", "global"))
    local = GPTNeoForCausalLM(config).eval()
    local.load_state_dict(plain.state_dict())
    ids = torch.randint(0, 64, (2, 20))
    with torch.no_grad():
        a, b = plain(ids)["logits"], local(ids)["logits"]
        torch.testing.assert_close(a[:, :4], b[:, :4])          # four tokens see the same
        assert not torch.allclose(a[:, 4:], b[:, 4:], atol=1e-4)
        sch = apply_schedule(local, "gpt_neo", model_config=config, disable_flash_attn=disable, group=False)
        model, _ = slapo.build(sch, init_weights=False)
        torch.testing.assert_close(model(ids)["logits"], b, rtol=2.0 ** -14, atol=2.0 ** -14)
    for layers, cls in ((("local",), GPTNeoForCausalLM), (("near",) * 3, GPTNeoForCausalLM),
                        (("local",) * 3, GPT2LMHeadModel)):
        with pytest.raises(ValueError):
            cls(GPTConfig(**kw, attention_layers=layers))


def test_local_layers_of_hugging_face():
    transformers = pytest.importorskip("transformers")
    import slapo_b200 as slapo
    from slapo_b200.model_schedule import apply_schedule

    config = transformers.GPTNeoConfig(num_layers=2, hidden_size=32, num_heads=4, vocab_size=50,
                                       window_size=4, attention_types=[[["global", "local"], 1]],
                                       max_position_embeddings=64, resid_dropout=0.0, embed_dropout=0.0,
                                       attention_dropout=0.0)
    torch.manual_seed(1)
    model = transformers.GPTNeoForCausalLM(config).eval()
    ids = torch.randint(0, 50, (2, 20))
    with torch.no_grad():
        want = model(ids, use_cache=False).logits
        sch = apply_schedule(model, "gpt_neo", model_config=config, local_attention=True, group=False)
        built, _ = slapo.build(sch, init_weights=False)
        got = built(ids, use_cache=False).logits
    torch.testing.assert_close(got, want, rtol=2.0 ** -14, atol=2.0 ** -14)


def test_refusals():
    q = torch.randn(1, 4, 2, 8)
    for kw in (dict(window=0), dict(window=-1), dict(window=1.5), dict(window=True), dict(window=2, sinks=-1),
               dict(window=2, sinks=1.0), dict(sinks=1), dict(window=2, causal=False),
               dict(window=2, rel_bias_table=torch.zeros(32, 2))):
        kw = {"causal": True, **kw}
        with pytest.raises(ValueError):
            NF.flash_attention(q, q, q, **kw)
        with pytest.raises(ValueError):
            NF.attention_reference(q, q, q, **kw)
    with pytest.raises(ValueError):
        FlashAttentionOp(apply_causal_mask=False, window=2)
    with pytest.raises(ValueError):
        FlashAttention(32, 4, output_proj=False, window=2)
    with pytest.raises(ValueError):
        flash_attention_qkvpacked(torch.randn(1, 4, 2, 3, 8), causal=False, window=2)


@pytest.mark.parametrize("general", [False, True])
def test_the_lowest_value_of_a_16bit_mask(general):
    """A mask in fp16 hides with -65504 as one in bf16 or fp32 with its lowest value: rows whose keys are all
    masked are zeros, in the key-padding form and with a bias for each pair.  Without a window it is a number."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 9, 2, 8, generator=g) for _ in range(3))
    pad = torch.zeros(2, 1, 1, 9, dtype=torch.bool)
    pad[0, ..., 6:] = True
    pad[1, ..., :5] = True       # (the window of the first queries is all padding)
    want = None
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        mask = torch.zeros(2, 1, 1, 9, dtype=dtype).masked_fill(pad, torch.finfo(dtype).min)
        if general:
            mask = mask.expand(2, 2, 9, 9)
        got = FlashAttentionOp(apply_causal_mask=True, window=3)(q, k, v, mask)
        want = got if want is None else want
        assert torch.equal(got, want) and bool((got[1, :5] == 0).all()) and not bool((got[1, 5:] == 0).any())
        plain = FlashAttentionOp(apply_causal_mask=True)(q, k, v, mask)
        assert not bool((plain[1, :5] == 0).any())
