"""AdamW over many tensors: the plain form against the formula in 64 bits and against torch.optim.AdamW, the
8-bit moments' format, the optimizer's bookkeeping and what it refuses."""
import copy
import math

import pytest
import torch

from slapo_b200.op import FusedAdamW, dequantize_moment, multi_tensor_adamw, quantize_moment
from slapo_b200.ops.adamw import STATE_BLOCK, state_blocks


def _model():
    torch.manual_seed(3)
    return torch.nn.Sequential(torch.nn.Linear(13, 7), torch.nn.LayerNorm(7), torch.nn.Linear(7, 5))


def _grads(model, seed):
    g = torch.Generator().manual_seed(seed)
    for p in model.parameters():
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype)


def test_follows_torch_adamw():
    a, b = _model(), _model()
    groups = lambda m: [{"params": [m[0].weight, m[2].weight], "weight_decay": 0.1},    # noqa: E731
                        {"params": [m[0].bias, m[2].bias, *m[1].parameters()], "weight_decay": 0.0,
                         "lr": 3e-3}]
    mine = FusedAdamW(groups(a), lr=1e-2, betas=(0.8, 0.95))
    ref = torch.optim.AdamW(groups(b), lr=1e-2, betas=(0.8, 0.95))
    for step in range(5):
        _grads(a, step)
        _grads(b, step)
        mine.step()
        ref.step()
    for p, q in zip(a.parameters(), b.parameters()):
        # (a step moves a weight by at most about lr; a few roundings of 2^-24 of it and of the weight)
        torch.testing.assert_close(p, q, rtol=16 * 2.0 ** -24, atol=5 * 1e-2 * 16 * 2.0 ** -24)


@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
def test_8bit_moments_keep_their_precision(n, second):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g))
    if second:
        x = x * x
    codes, scale = quantize_moment(x, second)
    assert codes.dtype == torch.float8_e4m3fn and scale.shape == (state_blocks(n),)
    mantissa, _ = torch.frexp(scale)
    assert bool((mantissa == 0.5).all())                      # powers of two
    held = x.double().sqrt() if second else x.double()
    value = codes.double() * scale.double().repeat_interleave(STATE_BLOCK)[:n]
    factor = scale.double().repeat_interleave(STATE_BLOCK)[:n]
    # half a step: 2^-4 of the value, or 2^-10 of the factor (the square root itself is rounded to 2^-24);
    # what would be rounded to zero is held as 2^-9 of it
    least = factor * (2.0 ** -9 if second else 2.0 ** -10)
    bound = torch.maximum(held.abs() * 2.0 ** -4, least) * (1 + 2.0 ** -22)
    assert bool(((value - held).abs() <= bound).all())
    assert bool((codes.float().abs() <= 448).all())
    if second:
        assert bool((value[held > 0] > 0).all())
    again, scale2 = quantize_moment(dequantize_moment(codes, scale, second), second)
    assert torch.equal(again.float(), codes.float()) or not torch.equal(scale, scale2)


def test_8bit_factor_is_the_smallest_that_fits():
    for top, want in ((448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (1.0, 2.0 ** -8), (0.0, 2.0 ** -126),
                      (2.0 ** -130, 2.0 ** -126)):
        x = torch.zeros(300)
        x[7] = -top
        _, scale = quantize_moment(x)
        assert scale.tolist() == [want, 2.0 ** -126], (top, scale)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_round_trip(bits, dtype):
    a = _model().to(dtype)
    opt = FusedAdamW(a.parameters(), lr=1e-2, state_bits=bits)
    for step in range(3):
        _grads(a, step)
        opt.step()
    b = copy.deepcopy(a)
    other = FusedAdamW(b.parameters(), lr=5.0, state_bits=bits)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for p, q in zip(a.parameters(), b.parameters()):
        for name, value in opt.state[p].items():
            got = other.state[q][name]
            if torch.is_tensor(value):
                assert got.dtype == value.dtype and torch.equal(got.float(), value.float()), name
                assert got.data_ptr() != value.data_ptr()
            else:
                assert got == value
    _grads(a, 9)
    _grads(b, 9)
    opt.step()
    other.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
    with pytest.raises(ValueError, match="bits"):
        FusedAdamW(b.parameters(), state_bits=40 - bits).load_state_dict(opt.state_dict())


@pytest.mark.parametrize("saved,wanted", [(True, False), (False, True)])
def test_state_of_an_optimizer_with_other_masters(saved, wanted):
    """Masters that were not saved begin at the parameters; those that are not wanted are left out.  Refused
    states leave the optimizer as it was."""
    a = _model().to(torch.bfloat16)
    opt = FusedAdamW(a.parameters(), lr=1e-2, master_weights=saved)
    _grads(a, 0)
    opt.step()
    b = copy.deepcopy(a)
    other = FusedAdamW(b.parameters(), lr=1e-2, master_weights=wanted)
    other.load_state_dict(opt.state_dict())
    for p in b.parameters():
        assert ("master" in other.state[p]) == wanted
        if wanted:
            assert torch.equal(other.state[p]["master"], p.float())
    _grads(b, 1)
    other.step()
    fresh = FusedAdamW(_model().parameters(), state_bits=8)
    with pytest.raises(ValueError, match="bits"):
        fresh.load_state_dict(opt.state_dict())
    assert not fresh.state


def test_parameters_without_a_gradient_are_left_alone():
    m = _model()
    opt = FusedAdamW(m.parameters(), lr=1e-2)
    _grads(m, 0)
    m[2].weight.grad = None
    before = m[2].weight.detach().clone()
    opt.step()
    assert torch.equal(before, m[2].weight) and m[2].weight not in opt.state
    _grads(m, 1)
    opt.step()
    assert opt.state[m[2].weight]["step"] == 1 and opt.state[m[0].weight]["step"] == 2


def test_closure_and_grad_scale():
    a, b = _model(), _model()
    x = torch.randn(4, 13)
    one, two = FusedAdamW(a.parameters(), lr=1e-2), FusedAdamW(b.parameters(), lr=1e-2)

    def closure():
        one.zero_grad()
        loss = a(x).square().sum()
        loss.backward()
        return loss

    loss = one.step(closure)
    assert loss.requires_grad
    (b(x).square().sum() * 4.0).backward()
    two.step(grad_scale=torch.full((1,), 0.25))
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=2.0 ** -20, atol=1e-2 * 2.0 ** -18)


def test_masters_keep_what_the_type_loses():
    p = torch.nn.Parameter(torch.ones(8, dtype=torch.bfloat16))
    q = torch.nn.Parameter(torch.ones(8, dtype=torch.bfloat16))
    keep, lose = FusedAdamW([p], lr=1e-4, weight_decay=0.0), FusedAdamW([q], lr=1e-4, weight_decay=0.0,
                                                                      master_weights=False)
    for _ in range(100):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
        keep.step()
        lose.step()
    assert bool((q == 1).all()) and bool((p < 1).all())
    # 100 differences just below 1, each rounded by up to 2^-25, and updates of 1e-4 off by some 2^-22 of it
    torch.testing.assert_close(keep.state[p]["master"], torch.full((8,), 0.99), rtol=0,
                               atol=100 * 2.0 ** -25 + 100 * 1e-4 * 2.0 ** -22)


def test_refusals():
    w = torch.nn.Parameter(torch.zeros(4, 4))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8),
               dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            FusedAdamW([w], **kw)
    t = torch.nn.Parameter(torch.zeros(4, 3).t())
    t.grad = torch.zeros_like(t)
    with pytest.raises(ValueError, match="contiguous"):
        FusedAdamW([t]).step()
    w.grad = torch.zeros(4, 4).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        FusedAdamW([w]).step()
    z = lambda: [torch.zeros(3)]     # noqa: E731
    with pytest.raises(ValueError, match="both"):
        multi_tensor_adamw(z(), z(), z(), z(), lr=1.0, step=1, exp_avg_scales=z())
    with pytest.raises(ValueError, match="count from 1"):
        multi_tensor_adamw(z(), z(), z(), z(), lr=1.0, step=0)
    with pytest.raises(ValueError, match="values required"):
        multi_tensor_adamw(z(), z(), z(), z(), lr=[1.0, 2.0], step=1)
    with pytest.raises(ValueError, match="gradients"):
        multi_tensor_adamw(z(), [], z(), z(), lr=1.0, step=1)
    with pytest.raises(ValueError, match="own masters"):
        multi_tensor_adamw(z(), z(), z(), z(), lr=1.0, step=1, masters=z())
    multi_tensor_adamw([], [], [], [], lr=1.0, step=1)
    assert math.isfinite(float(w.sum()))


def test_the_entry_for_lists_refuses_other_things():
    from slapo_b200.ops import native
    if not native.available():
        pytest.skip("extension not built")
    call = native.direct("multi_adamw")
    p = [torch.zeros(3)]
    rest = (p, p, [], p, p, [], [], [0.1], [0.1], 0.9, 0.99, 1e-8, 1, None, None)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        call(*rest)
    for at, value in ((0, tuple(p)), (1, [None]), (7, [1]), (7, ["x"]), (9, "x"), (12, 1.5), (13, 3),
                      (14, [])):
        bad = list(rest)
        bad[at] = value
        with pytest.raises((TypeError, RuntimeError)):
            call(*bad)
    with pytest.raises(TypeError):
        call(*rest[:-1])


def test_the_kernel_refuses_an_eps_that_8bit_moments_do_not_bear():
    """What counts as zero in 8 bits has a corrected root of up to 2^-63 / sqrt(1 - beta2): eps must not be
    less.  (The check comes before the one that CPU tensors do not pass.)"""
    from slapo_b200.ops import native
    if not native.available():
        pytest.skip("extension not built")
    p = [torch.zeros(3)]
    codes, scale = quantize_moment(p[0])

    def call(eps, bits, b2=0.999):
        factors = [scale] if bits == 8 else []
        m = [codes] if bits == 8 else p
        native.direct("multi_adamw")(p, p, [], m, m, factors, factors, [0.1], [0.1], 0.9, b2, eps, 1, None, None)

    least = 2.0 ** -63 / math.sqrt(1 - 0.999)
    for eps in (0.0, 1e-30, least * 0.999):
        with pytest.raises(RuntimeError, match="8-bit moments need eps"):
            call(eps, 8)
    for eps, bits in ((least * 1.001, 8), (1e-8, 8), (0.0, 32)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call(eps, bits)
    with pytest.raises(RuntimeError, match="8-bit moments need eps"):
        call(least * 1.001, 8, 0.9999)


def test_the_entry_for_lists_after_a_function_transform():
    """A transform that is at work has to see the call (False, nothing done); one that is over is none."""
    from slapo_b200.ops import native
    if not native.available():
        pytest.skip("extension not built")
    p = [torch.zeros(3)]

    def call():
        return native.direct("multi_adamw")(p, p, [], p, p, [], [], [0.1], [0.1], 0.9, 0.99, 1e-8, 1, None, None)

    def inside(x):
        assert call() is False
        return x + 1

    torch.func.vmap(inside)(torch.zeros(2))
    torch.func.grad(lambda x: inside(x).sum())(torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        call()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_changes_nothing(bits):
    """Neither states nor their number of steps, for what is refused and for what comes before it."""
    good, other = torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(4, 3).t())
    opt = FusedAdamW([good, other], lr=1e-2, state_bits=bits, capturable=True)
    good.grad, other.grad = torch.ones(5), torch.ones(4, 3).t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert not opt.state and bool((good == 1).all())
    other.grad = None
    opt.step()
    assert opt.state[good]["step"] == 1 and other not in opt.state
    held = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state[good].items()}
    weights = good.detach().clone()
    other.grad = torch.ones(4, 3).t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    good.grad = torch.ones(5).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        opt.step()
    good.grad = torch.ones(5)
    other.grad = None
    with pytest.raises(AttributeError):
        opt.step(grad_scale="not a tensor")
    assert list(opt.state) == [good] and torch.equal(good, weights)
    for name, value in opt.state[good].items():
        assert torch.equal(value.float(), held[name].float()) if torch.is_tensor(value) else value == held[name]
    # a state that something else has begun, without values, is none
    assert opt.state[other] == {}
    opt.step()
    again = FusedAdamW([good, other], state_bits=bits)
    again.load_state_dict(opt.state_dict())
    assert again.state[good]["step"] == 2
    again.step()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("how", ["deepcopy", "save"])
def test_a_copied_optimizer_goes_on(how, bits, tmp_path):
    """A copy, and one that was saved whole, keep their options and states, and step as the original does."""
    model = _model().to(torch.bfloat16)
    opt = FusedAdamW(model.parameters(), lr=1e-2, state_bits=bits, master_weights=bits == 32)
    _grads(model, 0)
    opt.step()
    if how == "deepcopy":
        other = copy.deepcopy(opt)
    else:
        torch.save(opt, tmp_path / "opt.pt")
        other = torch.load(tmp_path / "opt.pt", weights_only=False)
    assert (other.state_bits, other.master_weights, other.capturable) == (bits, bits == 32, False)
    copies = other.param_groups[0]["params"]
    for i, p in enumerate(model.parameters()):
        g = torch.full_like(p, 0.5 + i)
        p.grad, copies[i].grad = g, g.clone()
    opt.step()
    other.step()
    for p, q in zip(model.parameters(), copies):
        assert p is not q and torch.equal(p, q)
        assert other.state[q]["step"] == 2 and ("master" in other.state[q]) == (bits == 32)
