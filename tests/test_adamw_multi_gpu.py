"""AdamW over many tensors on the GPU: against the formula in 64 bits, 8-bit moments to the bit against the
plain form, odd lengths and addresses, captured steps and refusals."""
import copy

import pytest
import torch

from slapo_b200.op import FusedAdamW, dequantize_moment, multi_tensor_adamw, quantize_moment
from slapo_b200.ops import native
from slapo_b200.ops.adamw import _reference_step, state_blocks

pytestmark = pytest.mark.gpu

SIZES = [1, 7, 8, 255, 256, 257, 2047, 2048, 2049, 5000, 0, 70001]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _tensors(sizes, dtype, bits, master, offset=0, seed=0):
    """Lists of a step's tensors; each begins ``offset`` elements into memory of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def make(values):
        at = torch.empty(values.numel() + offset, device="cuda", dtype=values.dtype)
        at = at[offset:]
        at.copy_(values.reshape(-1))
        return at

    t = {"params": [], "grads": [], "exp_avgs": [], "exp_avg_sqs": []}
    if master:
        t["masters"] = []
    if bits == 8:
        t["exp_avg_scales"], t["exp_avg_sq_scales"] = [], []
    for n in sizes:
        w = torch.randn(n, generator=g, device="cuda") * 0.05
        m = torch.randn(n, generator=g, device="cuda") * 1e-3
        v = (m * 1.5) ** 2 + 1e-8
        t["params"].append(make(w.to(dtype)))
        t["grads"].append(make((torch.randn(n, generator=g, device="cuda") * 2e-3).to(dtype)))
        if master:
            t["masters"].append(make(w))
        for name, x, second in (("exp_avgs", m, False), ("exp_avg_sqs", v, True)):
            if bits == 8:
                codes, scale = quantize_moment(x, second)
                t[name].append(make(codes))
                t[name[:-1] + "_scales"].append(scale)
            else:
                t[name].append(make(x))
    return t


def _copy(t):
    return {k: [x.clone() for x in v] for k, v in t.items()}


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("dtype,master", [(torch.bfloat16, True), (torch.bfloat16, False),
                                          (torch.float16, True), (torch.float16, False),
                                          (torch.float32, False)])
@pytest.mark.parametrize("bits", [32, 8])
def test_against_64_bits(bits, dtype, master, offset):
    t = _tensors(SIZES, dtype, bits, master, offset)
    old = _copy(t)
    lrs = [1e-2 * (1 + i) for i in range(len(SIZES))]
    decays = [0.1 * (i % 3) for i in range(len(SIZES))]
    b1, b2, eps, step = 0.9, 0.99, 1e-6, 3
    gs = torch.full((1,), 0.5, device="cuda")
    multi_tensor_adamw(**t, lr=lrs, betas=(b1, b2), eps=eps, weight_decay=decays, step=step, grad_scale=gs)
    for i, n in enumerate(SIZES):
        g = old["grads"][i].double() * 0.5
        if bits == 8:
            m = dequantize_moment(old["exp_avgs"][i], old["exp_avg_scales"][i]).double()
            v = dequantize_moment(old["exp_avg_sqs"][i], old["exp_avg_sq_scales"][i], second=True).double()
        else:
            m, v = old["exp_avgs"][i].double(), old["exp_avg_sqs"][i].double()
        size = m.abs() * b1 + g.abs() * (1 - b1)
        m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
        w = (old["masters"] if master else old["params"])[i].double()
        denom = (v / (1 - b2 ** step)).sqrt() + eps
        update = m / (1 - b1 ** step) / denom + decays[i] * w
        want = w - lrs[i] * update
        # the moment: three roundings of 2^-24 and the constants' two; the quotient: some ten of 2^-23 more
        # (__fdividef is within 2 of them); then one of the product and one of the weight
        slack = lrs[i] * ((size / (1 - b1 ** step) / denom) * 8 + update.abs() * 16) * 2.0 ** -23
        bound = slack + (w.abs() * lrs[i] * decays[i] + want.abs()) * 2.0 ** -23
        if master:
            assert bool(((t["masters"][i].double() - want).abs() <= bound).all())
            assert torch.equal(t["params"][i], t["masters"][i].to(dtype))
        else:
            tiny = torch.finfo(dtype).smallest_normal * HALF[dtype]
            half = HALF[dtype] if dtype != torch.float32 else 0.0
            assert bool(((t["params"][i].double() - want).abs()
                         <= bound * 2 + want.abs() * half * (1 + 2.0 ** -8) + tiny).all())
        if bits == 32:
            assert bool(((t["exp_avgs"][i].double() - m).abs() <= size * 5 * 2.0 ** -24).all())
            assert bool(((t["exp_avg_sqs"][i].double() - v).abs() <= v * 6 * 2.0 ** -24).all())
        assert torch.equal(t["grads"][i], old["grads"][i])


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_8bit_moments_are_those_of_the_plain_form(dtype, offset):
    """Products and sums are rounded one by one on both sides: the same first moments, to the bit.  The
    square roots of the second are a unit in the last place apart at most (2^-23 of them), so that only next
    to the middle between two 8-bit numbers another one may come out."""
    t = _tensors(SIZES, dtype, 8, False, offset, seed=5)
    gs = torch.full((1,), 0.7, device="cuda")
    for step in range(1, 4):
        r = _copy(t)
        held = [dequantize_moment(c, s, second=True)
                for c, s in zip(r["exp_avg_sqs"], r["exp_avg_sq_scales"])]
        multi_tensor_adamw(**t, lr=1e-3, step=step, grad_scale=gs)
        for i in range(len(SIZES)):
            _reference_step(r["params"][i], r["grads"][i], None, r["exp_avgs"][i], r["exp_avg_sqs"][i],
                            r["exp_avg_scales"][i], r["exp_avg_sq_scales"][i], 1e-3, 0.01,
                            (0.9, 0.999), 1e-8, step, gs)
            assert torch.equal(t["exp_avgs"][i].view(torch.uint8), r["exp_avgs"][i].view(torch.uint8))
            for scales in ("exp_avg_scales", "exp_avg_sq_scales"):
                assert torch.equal(t[scales][i], r[scales][i])
            _same_roots(t["exp_avg_sqs"][i], r["exp_avg_sqs"][i], r["exp_avg_sq_scales"][i],
                        held[i] * 0.999 + (r["grads"][i].float() * 0.7).square() * (1 - 0.999))


def _same_roots(got, want, scale, v):
    """8-bit square roots of ``v``, equal but next to the middle between two."""
    # (below the smallest normal number a second moment counts as zero)
    none = (v > 0) & (v < 2.0 ** -126)
    assert bool((got.float()[none] == 0).all())
    other = (got.view(torch.uint8) != want.view(torch.uint8)) & ~none
    assert float(other.float().mean()) <= 1e-3 if other.numel() > 1000 else int(other.sum()) <= 1
    a, b = got.float()[other].double(), want.float()[other].double()
    at = scale.double().repeat_interleave(256)[:v.numel()][other]
    root = v.double().sqrt()[other] / at
    assert bool(((root - (a + b) / 2).abs() <= root * 2.0 ** -21).all())


def test_8bit_extremes():
    """Blocks of zeros, of very small and of very large values, and a NaN that stays in its place."""
    n = 256 * 6
    g = torch.zeros(n, device="cuda")
    g[256:512] = 1e-25
    g[512:768] = 1e15 * torch.linspace(-1, 1, 256, device="cuda")
    g[768:1024] = torch.logspace(-30, 3, 256, device="cuda")
    g[1030] = float("nan")
    w = torch.zeros(n, device="cuda")
    m, ms = quantize_moment(torch.zeros(n, device="cuda"))
    v, vs = quantize_moment(torch.zeros(n, device="cuda"), second=True)
    m2, ms2, v2, vs2, w2 = m.clone(), ms.clone(), v.clone(), vs.clone(), w.clone()
    multi_tensor_adamw([w], [g], [m], [v], lr=1e-3, step=1, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    ok = torch.arange(n, device="cuda") // 256 != 4
    _reference_step(w2, torch.where(ok, g, torch.zeros_like(g)), None, m2, v2, ms2, vs2, 1e-3, 0.01,
                    (0.9, 0.999), 1e-8, 1, None)
    assert torch.equal(m.view(torch.uint8)[ok], m2.view(torch.uint8)[ok])
    assert torch.equal(vs, vs2)
    _same_roots(v[ok], v2[ok], vs[[0, 1, 2, 3, 5]], (g[ok].square() * (1 - 0.999)))
    assert bool((dequantize_moment(v, vs, True)[768:1024][g[768:1024].square() > 0] >= 0).all())
    assert bool(torch.isnan(w[1030])) and int(torch.isnan(w).sum()) == 1
    assert bool(torch.isnan(m.float()[1030])) and int(torch.isnan(m.float()).sum()) == 1


@pytest.mark.parametrize("count", [1, 48, 49, 360, 361, 800])
def test_number_of_tensors(count):
    sizes = [(i * 37) % 301 for i in range(count)]
    t = _tensors(sizes, torch.bfloat16, 8, True)
    r = _copy(t)
    before = native.launch_count()
    multi_tensor_adamw(**t, lr=1e-3, step=2)
    assert native.launch_count() - before <= -(-count // 360)
    for i in range(count):
        _reference_step(r["params"][i], r["grads"][i], r["masters"][i], r["exp_avgs"][i], r["exp_avg_sqs"][i],
                        r["exp_avg_scales"][i], r["exp_avg_sq_scales"][i], 1e-3, 0.01, (0.9, 0.999), 1e-8,
                        2, None)
        assert torch.equal(t["exp_avgs"][i].view(torch.uint8), r["exp_avgs"][i].view(torch.uint8))
        # (an update is at most some lr, off by a few 2^-23 of it)
        torch.testing.assert_close(t["masters"][i], r["masters"][i], rtol=2.0 ** -22,
                                   atol=1e-3 * 32 * 2.0 ** -23)


def test_neighbours_are_left_alone():
    """Memory before and behind each tensor, and factors of other tensors, keep their values."""
    for bits in (8, 32):
        t = _tensors([300, 1000], torch.bfloat16, bits, True)
        guarded = {}
        for k, v in t.items():
            guarded[k] = []
            for x in v:
                whole = torch.full((x.numel() + 64,), 3.0, device="cuda").to(x.dtype)
                whole[32:-32].copy_(x)
                guarded[k].append(whole)
        multi_tensor_adamw(**{k: [x[32:-32] for x in v] for k, v in guarded.items()}, lr=1e-3, step=1)
        multi_tensor_adamw(**t, lr=1e-3, step=1)
        for k, v in guarded.items():
            for whole, x in zip(v, t[k]):
                assert torch.equal(whole[32:-32].float(), x.float()), k
                assert bool((whole[:32].float() == 3).all()) and bool((whole[-32:].float() == 3).all()), k


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_go_on_counting(bits):
    torch.manual_seed(0)
    a = torch.nn.Linear(40, 30, device="cuda").to(torch.bfloat16)
    b = copy.deepcopy(a)
    one = FusedAdamW(a.parameters(), lr=1e-2, state_bits=bits, capturable=True)
    two = FusedAdamW(b.parameters(), lr=1e-2, state_bits=bits)
    for m in (a, b):
        for p in m.parameters():
            p.grad = torch.zeros_like(p)

    def grads(seed):
        for m in (a, b):
            g = torch.Generator(device="cuda").manual_seed(seed)
            for p in m.parameters():
                p.grad.normal_(generator=g)

    fresh = FusedAdamW(copy.deepcopy(a).parameters(), lr=1e-2, capturable=True)
    grads(0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        one.step()
    torch.cuda.current_stream().wait_stream(stream)
    two.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.step()
    for step in range(1, 5):
        grads(step)
        graph.replay()
        two.step()
        for p, q in zip(a.parameters(), b.parameters()):
            # (1 - beta^t is formed in 64 bits on both sides and rounded)
            assert torch.equal(p, q)
            assert int(one.state[p]["step"]) == two.state[q]["step"] == step + 1
    one.load_state_dict(copy.deepcopy(two.state_dict()))
    grads(9)
    one.step()
    two.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
    a.bias.grad = None
    with pytest.raises(RuntimeError, match="together"):
        one.step()
    for p in fresh.param_groups[0]["params"]:
        p.grad = torch.zeros_like(p)
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()
    torch.cuda.synchronize()


def test_saved_parameters_are_noticed():
    w = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = FusedAdamW([w], lr=1e-2)
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_refusals():
    def call(**kw):
        t = _tensors([300, 40], torch.bfloat16, 32, True)
        t.update(lr=1e-3, step=1)
        t.update({k: v(t) if callable(v) else v for k, v in kw.items()})
        multi_tensor_adamw(**t)

    call()
    bad = [("entry", dict(masters=lambda t: t["masters"][:1])),
           ("values required", dict(grads=lambda t: t["grads"][::-1])),
           ("contiguous", dict(grads=lambda t: [torch.zeros(600, device="cuda", dtype=torch.bfloat16)[::2],
                                                t["grads"][1]])),
           ("must be", dict(grads=lambda t: [g.float() for g in t["grads"]])),
           ("must be", dict(exp_avgs=lambda t: [x.half() for x in t["exp_avgs"]])),
           ("CUDA tensors", dict(masters=lambda t: [x.cpu() for x in t["masters"]])),
           ("share memory", dict(params=lambda t: [t["params"][0], t["params"][0][:40]])),
           ("share memory", dict(exp_avgs=lambda t: [t["exp_avgs"][0], t["exp_avgs"][0][260:]])),
           ("count from 1", dict(step=0)), ("betas", dict(betas=(0.9, 1.0))),
           ("must be", dict(step=torch.ones(1, device="cuda"))),
           ("values required", dict(grad_scale=torch.ones(2, device="cuda"))),
           ("own masters", dict(params=lambda t: [p.float() for p in t["params"]],
                                grads=lambda t: [p.float() for p in t["grads"]])),
           ("must be", dict(params=lambda t: [p.double() for p in t["params"]],
                            grads=lambda t: [p.double() for p in t["grads"]]))]
    for message, kw in bad[:-1]:
        with pytest.raises((RuntimeError, ValueError), match=message):
            call(**kw)
    with pytest.raises(RuntimeError, match="bf16, fp16 or fp32"):
        call(**bad[-1][1])
    t = _tensors([300], torch.bfloat16, 8, True)
    t["exp_avg_scales"][0] = torch.ones(state_blocks(300) + 1, device="cuda")
    with pytest.raises(RuntimeError, match="factors"):
        multi_tensor_adamw(**t, lr=1e-3, step=1)
    t = _tensors([300, 40], torch.bfloat16, 32, False)
    t["grads"][1].untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="no memory"):
        multi_tensor_adamw(**t, lr=1e-3, step=1)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_operator_and_the_lists_agree(bits):
    """The registered operator, and the entry that reads Python lists in place; the latter leaves tensors that
    the dispatcher has to see to the former, which has no form for tensors without values."""
    a = _tensors([300, 4100, 40], torch.bfloat16, bits, True)
    b = _copy(a)
    multi_tensor_adamw(**a, lr=[1e-3, 2e-3, 3e-3], weight_decay=0.1, step=3)
    native.ops().multi_adamw(b["params"], b["grads"], b["masters"], b["exp_avgs"], b["exp_avg_sqs"],
                             b.get("exp_avg_scales", []), b.get("exp_avg_sq_scales", []), [1e-3, 2e-3, 3e-3],
                             [0.1] * 3, 0.9, 0.999, 1e-8, 3, None, None)
    for name in a:
        for x, y in zip(a[name], b[name]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        fake = [torch.zeros(8, device="cuda") for _ in range(4)]
    before = native.launch_count()
    with pytest.raises(Exception):
        multi_tensor_adamw([fake[0]], [fake[1]], [fake[2]], [fake[3]], lr=1e-3, step=1)
    assert native.launch_count() == before


def test_another_stream():
    a = _tensors([70001, 300], torch.bfloat16, 8, True)
    b = _copy(a)
    multi_tensor_adamw(**a, lr=1e-3, step=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        multi_tensor_adamw(**b, lr=1e-3, step=1)
    torch.cuda.current_stream().wait_stream(side)
    for name in a:
        for x, y in zip(a[name], b[name]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_beyond_32_bits(bits):
    """A parameter of more than 2^31 elements: its end as that part alone, and zeros stay zeros."""
    n, tail = 2 ** 31 + 812, 812
    small = _tensors([tail], torch.bfloat16, bits, False)
    large = {k: [torch.zeros(n if "scale" not in k else state_blocks(n), device="cuda",
                             dtype=torch.uint8 if v[0].dtype == torch.float8_e4m3fn else v[0].dtype)]
             for k, v in small.items()}
    for name, (x,) in large.items():
        if "scale" in name:
            x.fill_(2.0 ** -126)
        if x.dtype == torch.uint8:
            large[name][0] = x.view(torch.float8_e4m3fn)
        x[-small[name][0].numel():].copy_(small[name][0].view(x.dtype))
    for t in (small, large):
        multi_tensor_adamw(**t, lr=1e-3, step=2)
    for name, (x,) in large.items():
        end = small[name][0].numel()
        assert torch.equal(x[-end:].view(torch.uint8), small[name][0].view(torch.uint8)), name
    assert int(torch.count_nonzero(large["params"][0][:-tail])) == 0


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30])
def test_32bit_moments_with_hardly_any_eps(eps, offset):
    """Second moments and divisors below the smallest normal number count: the first step moves each weight by
    lr g / (|g| + eps), whatever the gradient's size."""
    n = 5000
    g = torch.logspace(-20.5, 3, n, device="cuda") * (1 - 2 * (torch.arange(n, device="cuda") % 2))
    t = [torch.zeros(n + offset, device="cuda")[offset:] for _ in range(4)]
    t[1].copy_(g)
    lr, b1, b2 = 1e-3, 0.9, 0.999
    multi_tensor_adamw([t[0]], [t[1]], [t[2]], [t[3]], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, step=1)
    # v = g^2 (1 - b2) in fp32: below 2^-126 steps are 2^-149, so that the product is off by half of one and
    # by (1 - b2) of the square's half: 2^-150 * 1.001 = e v in all, e < 0.08.  The root is off by
    # 1 - sqrt(1 - e) < 0.52 e, its inverse by less than 0.57 e
    v = g.double().square() * (1 - b2)
    off = 2.0 ** -150 / v + 32 * 2.0 ** -24
    assert float(off.max()) < 0.2
    want = -lr * g.double() / (g.double().abs() + torch.tensor(eps, dtype=torch.float32).double().item())
    assert bool(((t[0].double() - want).abs() <= want.abs() * off).all())


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_does_not_count(capturable, bits):
    """A gradient without memory is refused by the kernel's checks: weights, moments and the number of steps,
    on the host or on the device, are as before; so after a first step under a capture."""
    torch.manual_seed(1)
    a = torch.nn.Linear(40, 30, device="cuda").to(torch.bfloat16)
    b = copy.deepcopy(a)
    one = FusedAdamW(a.parameters(), lr=1e-2, state_bits=bits, capturable=capturable)
    two = FusedAdamW(b.parameters(), lr=1e-2, state_bits=bits, capturable=capturable)
    grad = torch.randn(30, 40, device="cuda").to(torch.bfloat16)

    def grads(m):
        m.weight.grad, m.bias.grad = grad.clone(), torch.ones(30, device="cuda").to(torch.bfloat16)

    def refused():
        grads(a)
        a.bias.grad.untyped_storage().resize_(0)
        with pytest.raises(RuntimeError, match="no memory"):
            one.step()

    if capturable:
        grads(a)
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                one.step()
        torch.cuda.synchronize()
    refused()
    assert not one.state
    for step in range(1, 4):
        grads(a)
        grads(b)
        one.step()
        two.step()
        refused()
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.equal(p, q) and int(one.state[p]["step"]) == int(two.state[q]["step"]) == step
            for name, value in one.state[p].items():
                assert not torch.is_tensor(value) or torch.equal(value.float(), two.state[q][name].float())


def test_what_was_updated_before_a_refusal_counts():
    """Two types are two kernels: the first is through when the second is refused."""
    a = torch.nn.Parameter(torch.ones(8, device="cuda"))
    b = torch.nn.Parameter(torch.ones(8, device="cuda", dtype=torch.bfloat16))
    opt = FusedAdamW([a, b], lr=1e-2)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    b.grad.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="no memory"):
        opt.step()
    assert opt.state[a]["step"] == 1 and b not in opt.state and bool((a < 1).all())
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1


@pytest.mark.parametrize("steps", [0, 1])
def test_a_step_that_counts_on_the_host_is_not_captured(steps):
    """Its replays would keep the bias corrections of the one that was captured."""
    w = torch.nn.Parameter(torch.ones(300, device="cuda"))
    w.grad = torch.ones_like(w)
    opt = FusedAdamW([w], lr=1e-2)
    for _ in range(steps):
        opt.step()
    torch.cuda.synchronize()
    before = native.launch_count()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert native.launch_count() == before and len(opt.state) == steps
    opt.step()
    assert opt.state[w]["step"] == steps + 1


@pytest.mark.parametrize("which", ["params", "masters", "grads"])
def test_weights_that_a_step_changes_are_noticed(which):
    """Autograd refuses a backward that has saved weights which a step has written; gradients are only read."""
    t = _tensors([300, 40], torch.bfloat16, 8, True)
    x = t[which][1]
    loss = (torch.ones_like(x, requires_grad=True) * x).sum()
    multi_tensor_adamw(**t, lr=1e-3, step=1)
    if which == "grads":
        loss.backward()
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


@pytest.mark.parametrize("dtype,master", [(torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
def test_8bit_moments_of_more_than_the_resident_warps_take(dtype, master):
    """Every warp has several units, of several tensors, in one sweep and in more: first moments to the bit,
    weights to some roundings of 2^-23 of an update, as the plain form; the rest of a tensor's memory is left."""
    sizes = [3_000_001, 77, 2_500_000, 511, 4_000_003]
    t = _tensors(sizes, dtype, 8, master, seed=7)
    r = _copy(t)
    multi_tensor_adamw(**t, lr=1e-3, step=2)
    for i in range(len(sizes)):
        _reference_step(r["params"][i], r["grads"][i], r["masters"][i] if master else None, r["exp_avgs"][i],
                        r["exp_avg_sqs"][i], r["exp_avg_scales"][i], r["exp_avg_sq_scales"][i], 1e-3, 0.01,
                        (0.9, 0.999), 1e-8, 2, None)
        assert torch.equal(t["exp_avgs"][i].view(torch.uint8), r["exp_avgs"][i].view(torch.uint8))
        assert torch.equal(t["exp_avg_scales"][i], r["exp_avg_scales"][i])
        w, want = (x["masters" if master else "params"][i].float() for x in (t, r))
        # (an update is at most some 30 lr, off by 2^-19 of it; what a type has in between goes up or down)
        step = 0.0 if master or dtype == torch.float32 else 2 * HALF[dtype]
        assert bool(((w - want).abs() <= want.abs() * (step + 2.0 ** -22) + 30e-3 * 2.0 ** -19).all())
