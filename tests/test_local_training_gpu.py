"""Lookup, local attention, their gradients and the optimizer as a program uses them together: a training step
of a small GPT-Neo with local layers, the same captured, and generation token by token."""
import copy

import pytest
import torch

import slapo_b200 as slapo
from slapo_b200.model_schedule import apply_schedule
from slapo_b200.models import GPTConfig, GPTNeoForCausalLM
from slapo_b200.op import FlashAttention, FusedAdamW, FusedEmbedding
from slapo_b200.ops import native
from slapo_b200.ops.adamw import _reference_step, dequantize_moment

pytestmark = pytest.mark.gpu

VOCAB, HIDDEN, SEQ = 512, 128, 300


def _config():
    return GPTConfig(vocab_size=VOCAB, n_positions=SEQ, hidden_size=HIDDEN, num_layers=3, num_heads=2,
                     resid_dropout=0.0, embed_dropout=0.0, attention_dropout=0.0, model_type="gpt_neo",
                     attention_layers=("global", "local", "local"), window_size=50)


def _plain():
    torch.manual_seed(4)
    return GPTNeoForCausalLM(_config()).init_weights()


def _fused(dtype):
    model = _plain().cuda()
    sch = apply_schedule(model, "gpt_neo", model_config=_config(), bf16=dtype == torch.bfloat16, group=False)
    model, _ = slapo.build(sch, init_weights=False)
    model = model.cuda()
    model.transformer.wte = FusedEmbedding.from_embedding(model.transformer.wte)
    model.transformer.wpe = FusedEmbedding.from_embedding(model.transformer.wpe)
    return model


def _ids(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, VOCAB, (2, SEQ), generator=g, device="cuda")


def _table(model):
    return model.transformer.wte.weight


def test_gradients_of_a_step():
    fused, plain = _fused(torch.bfloat16), _plain().cuda().double()
    ids = _ids(0)
    before = native.launch_count()
    fused(ids, labels=ids)["loss"].backward()
    assert native.launch_count() - before > 20 and native.ops().device_status() == 0
    plain(ids, labels=ids)["loss"].backward()
    pairs = [(_table(fused), _table(plain)), (fused.transformer.wpe.weight, plain.transformer.wpe.weight),
             (fused.transformer.ln_f.weight, plain.transformer.ln_f.weight)]
    for got, want in pairs:
        err = (got.grad.double() - want.grad).norm() / want.grad.norm()
        # three layers forward and backward, some twenty roundings of at most 2^-8 between a weight and the
        # loss and as many back
        assert float(err) <= 40 * 2.0 ** -8, float(err)
        assert float(err) > 0


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_with_the_optimizer(bits):
    model = _fused(torch.bfloat16)
    decay = [p for p in model.parameters() if p.dim() > 1]
    rest = [p for p in model.parameters() if p.dim() <= 1]
    opt = FusedAdamW([{"params": decay, "weight_decay": 0.1}, {"params": rest, "weight_decay": 0.0}], lr=1e-3,
                     state_bits=bits)
    for step in range(1, 4):
        ids = _ids(step)
        opt.zero_grad()
        model(ids, labels=ids)["loss"].backward()
        state = {p: copy.deepcopy(opt.state[p]) for p in model.parameters()}
        old = {p: p.detach().clone() for p in model.parameters()}
        opt.step()
        for p in model.parameters():
            s, new = state[p], opt.state[p]
            if step == 1:
                s = {k: torch.zeros_like(v) for k, v in new.items() if torch.is_tensor(v)}
                s["master"] = old[p].float()
            _reference_step(old[p], p.grad, s["master"], s["exp_avg"], s["exp_avg_sq"],
                            s.get("exp_avg_scale"), s.get("exp_avg_sq_scale"), 1e-3,
                            0.1 if p.dim() > 1 else 0.0, (0.9, 0.999), 1e-8, step, None)
            # an update of some 1e-3 at most (m / sqrt(v), up to 3), off by a few 2^-23 of it
            torch.testing.assert_close(new["master"], s["master"], rtol=2.0 ** -22,
                                       atol=1e-3 * 64 * 2.0 ** -23)
            assert torch.equal(p, new["master"].to(p.dtype))
            if bits == 8:
                assert torch.equal(dequantize_moment(new["exp_avg"], new["exp_avg_scale"]),
                                   dequantize_moment(s["exp_avg"], s["exp_avg_scale"]))


def test_a_captured_step_is_the_eager_one():
    eager, captured = _fused(torch.bfloat16), _fused(torch.bfloat16)
    ids = _ids(0).clone()

    def step(model, opt):
        opt.zero_grad(set_to_none=False)
        model(ids, labels=ids)["loss"].backward()
        opt.step()

    opts = [FusedAdamW(m.parameters(), lr=1e-3, state_bits=8, capturable=m is captured)
            for m in (eager, captured)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(captured, opts[1])
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(2):
        step(eager, opts[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(captured, opts[1])
    for seed in range(1, 4):
        ids.copy_(_ids(seed))
        graph.replay()
        step(eager, opts[0])
        for p, q in zip(eager.parameters(), captured.parameters()):
            assert torch.equal(p, q)


def test_generation_with_sinks():
    """Lookup and attention of single tokens over a growing cache against the whole sequence in 64 bits."""
    torch.manual_seed(2)
    emb = FusedEmbedding(VOCAB, HIDDEN, scale=HIDDEN ** 0.5, device="cuda", dtype=torch.float16)
    block = FlashAttention(HIDDEN, 2, fused_qkv=True, output_proj=True, causal=True, window=20, sinks=3,
                           attn_op_name="auto").cuda().half().eval()
    ids = _ids(9)[:, :90]
    exact = copy.deepcopy(block).double()
    with torch.no_grad():
        past, outs = None, []
        for t in range(90):
            out, past = block(emb(ids[:, t:t + 1]) / HIDDEN ** 0.5, layer_past=past, use_cache=True)
            outs.append(out)
        want, _ = exact(emb.weight.double()[ids])
    err = (torch.cat(outs, 1).double() - want).norm() / want.norm()
    # the lookup's factor and its inverse, the projections, probabilities, output and second projection: some
    # eight roundings of 2^-11, those of queries and keys with a score's size of a few in front
    assert float(err) <= 30 * 2.0 ** -11, float(err)
