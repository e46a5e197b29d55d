"""Attention with a window and sinks on the GPU: output and gradients against 64 bits within bounds that are
computed from the roundings the kernels make, over lengths, windows, sinks, masks, types and layouts."""
import math

import pytest
import torch

from slapo_b200.op import FlashAttention
from slapo_b200.ops import functional as NF
from slapo_b200.ops import native
from slapo_b200.ops.flash_attn import dropout_keep_mask, effective_dropout_p, flash_attention_qkvpacked

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _seen(sq, sk, window, sinks, bias):
    i = torch.arange(sq, device="cuda")[:, None] + (sk - sq)
    j = torch.arange(sk, device="cuda")[None]
    seen = ((j <= i) & ((j > i - window) | (j < sinks)))[None, None]
    return seen if bias is None else seen & (bias >= -1e30)[:, None, None]


def _check(got, q, k, v, do, window, sinks, bias=None, scale=None, keep=None, p_drop=0.0):
    """``got``: output and gradients (or the output alone).  Roundings of half a step h of the type: of the
    probabilities before the products, of the output, of dS and of the gradients; the output's again in the
    row term of dS.  Scores are sums of D products in fp32."""
    dtype, h = q.dtype, HALF[q.dtype]
    b, sq, n, d = q.shape
    sk = k.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, k, v = (t.detach().transpose(1, 2).double() for t in (q, k, v))
    seen = _seen(sq, sk, window, sinks, bias)
    s = q @ k.transpose(-1, -2) * scale
    size = q.abs() @ k.abs().transpose(-1, -2) * abs(scale)
    if bias is not None:
        s = s + bias.double()[:, None, None]
        size = size + bias.double().abs().clamp(max=1e30)[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    empty = ~seen.expand(b, n, sq, sk).any(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(empty, 0.0), -1).masked_fill(empty | ~seen, 0.0)
    # relative error of a probability: of its score (D + 4 roundings of 2^-24), of the row's sum likewise, and
    # 2^-21 for the exponential and the rest
    off = torch.where(seen, size, torch.zeros_like(size)).amax(-1, keepdim=True)
    off = off * (d + 4) * 2.0 ** -23 + 2.0 ** -21
    m = 1.0 if keep is None else keep.double() / (1.0 - p_drop)
    out = (p * m) @ v
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0     # steps of fp16 below 2^-14
    room = (p * m * (h + off)) @ v.abs() + tiny * seen.double().sum(-1, keepdim=True).amax()
    bound = room * (1 + 2.0 ** -8) + out.abs() * h * (1 + 2.0 ** -6) + tiny
    pairs = [("out", got[0], out, bound)]
    if len(got) > 1:
        do = do.detach().transpose(1, 2).double()
        dp = (do @ v.transpose(-1, -2)) * m
        delta = (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # dS is formed as p (dP - delta): what delta and dP are off by, times p, and p's own error
        off_delta = (do.abs() * bound).sum(-1, keepdim=True) + (do.abs() @ v.abs().transpose(-1, -2)) * m \
            * (d + 4) * 2.0 ** -24
        off_ds = p * off_delta + ds.abs() * (h + off) + p * (dp.abs() + delta.abs()) * off + tiny
        for name, x, want, room in (
                ("dq", got[1], ds @ k * scale, off_ds @ k.abs() * abs(scale)),
                ("dk", got[2], ds.transpose(-1, -2) @ q * scale,
                 off_ds.transpose(-1, -2) @ q.abs() * abs(scale)),
                ("dv", got[3], (p * m).transpose(-1, -2) @ do,
                 (p * m * (h + off) + tiny).transpose(-1, -2) @ do.abs())):
            pairs.append((name, x, want, room * (1 + 2.0 ** -6) + want.abs() * h * (1 + 2.0 ** -6) + tiny))
    for name, x, want, bound in pairs:
        assert x.dtype == dtype
        err = (x.detach().transpose(1, 2).double() - want).abs()
        most = float((err / bound.clamp(min=1e-30)).max())
        assert bool((err <= bound).all()), f"{name}: {most:.3f} of its bound"
    return pairs


def _run(q, k, v, do, window, sinks, bias=None, **kw):
    out = NF.flash_attention(q, k, v, bias, causal=True, window=window, sinks=sinks, **kw)
    got = [out, *torch.autograd.grad(out, (q, k, v), do)]
    assert native.ops().device_status() == 0, "a bounded wait inside the kernel ran out"
    return got


def _tensors(b, sq, sk, n, d, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda s: torch.randn(b, s, n, d, generator=g, device="cuda").to(dtype)      # noqa: E731
    q, k, v, do = make(sq), make(sk), make(sk), make(sq)
    return q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), do


LENGTHS = [(1, 1), (2, 2), (64, 64), (127, 127), (129, 129), (257, 257), (700, 700), (130, 513), (60, 700),
           (5, 300), (300, 130), (200, 1)]


@pytest.mark.parametrize("sq,sk", LENGTHS)
@pytest.mark.parametrize("window", [1, 2, 65, 128, 200, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 70, 140])
def test_lengths_windows_sinks(sq, sk, window, sinks):
    q, k, v, do = _tensors(2, sq, sk, 3, 64, torch.bfloat16)
    _check(_run(q, k, v, do, window, sinks), q, k, v, do, window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 40, 64, 80, 128])
@pytest.mark.parametrize("sq,sk,window,sinks", [(333, 333, 100, 5), (1100, 1100, 256, 0), (90, 600, 130, 3)])
def test_types_and_head_dims(sq, sk, window, sinks, d, dtype):
    q, k, v, do = _tensors(2, sq, sk, 4, d, dtype, seed=d)
    _check(_run(q, k, v, do, window, sinks), q, k, v, do, window, sinks)


@pytest.mark.parametrize("low", [-10000.0, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min,
                                 -math.inf, -4.0])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,sk", [(300, 300), (1, 300), (40, 520)])
def test_masks(sq, sk, d, low):
    """Right and left padding, a sequence of nothing but padding, queries whose window is all padding."""
    q, k, v, do = _tensors(4, sq, sk, 2, d, torch.bfloat16, seed=3)
    at = torch.arange(sk, device="cuda")
    pad = torch.stack([at >= sk - 120, at < sk // 2, at >= 0, (at > 20) & (at < sk - 3)])
    bias = torch.zeros(4, sk, device="cuda").masked_fill(pad, low)
    for window, sinks in ((33, 0), (150, 6)):
        _check(_run(q, k, v, do, window, sinks, bias), q, k, v, do, window, sinks, bias)


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("sk,window,sinks", [(1, 1, 0), (1, 9, 9), (7, 3, 1), (300, 256, 4),
                                             (1501, 256, 4), (1501, 1, 0), (5000, 2048, 130),
                                             (4097, 4000, 300), (900, 900, 0)])
def test_one_query(sk, window, sinks, d):
    with torch.no_grad():
        for b, n, dtype in ((1, 2, torch.bfloat16), (8, 16, torch.float16), (3, 100, torch.bfloat16)):
            q, k, v, _ = _tensors(b, 1, sk, n, d, dtype, seed=sk)
            # (a cache with room behind it and heads before tokens, as programs keep them)
            cache = torch.full((b, n, sk + 9, 2, d), float("nan"), device="cuda", dtype=dtype)
            cache[:, :, :sk, 0].copy_(k.transpose(1, 2))
            cache[:, :, :sk, 1].copy_(v.transpose(1, 2))
            ck, cv = (cache[:, :, :sk, i].transpose(1, 2) for i in range(2))
            out = NF.flash_attention(q, ck, cv, causal=True, window=window, sinks=sinks)
            _check([out], q, k, v, None, window, sinks)


def test_keys_outside_of_the_window_are_not_read():
    """NaN and infinities where no query looks: whole tiles of them for many queries, any place for one."""
    for sq in (1, 200):
        q, k, v, _ = _tensors(2, sq, 1000, 2, 64, torch.bfloat16)
        with torch.no_grad():
            want = NF.flash_attention(q, k, v, causal=True, window=100, sinks=3)
            lo, hi = (3, 1000 - 100) if sq == 1 else (128, 640)
            k[:, lo:hi], v[:, lo:hi] = float("nan"), float("inf")
            assert torch.equal(NF.flash_attention(q, k, v, causal=True, window=100, sinks=3), want)


@pytest.mark.parametrize("shape,window,sinks", [((2, 384, 4, 64), 100, 0), ((1, 700, 2, 128), 256, 70),
                                                ((2, 130, 3, 80), 40, 2)])
def test_packed_is_the_same(shape, window, sinks):
    b, s, n, d = shape
    qkv = torch.randn(b, s, n, 3, d, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    do = torch.randn(b, s, n, d, device="cuda", dtype=torch.bfloat16)
    out = flash_attention_qkvpacked(qkv, causal=True, window=window, sinks=sinks)
    dqkv = torch.autograd.grad(out, qkv, do)[0]
    q, k, v = qkv.detach().unbind(3)
    _check([out, *dqkv.unbind(3)], q, k, v, do, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,sk,window,sinks", [(300, 300, 90, 0), (300, 300, 90, 5), (64, 500, 200, 130),
                                                (1200, 1200, 128, 1)])
def test_dropout(sq, sk, window, sinks, d):
    p = 0.25
    q, k, v, do = _tensors(2, sq, sk, 2, d, torch.bfloat16)
    torch.cuda.manual_seed(5)
    keep = dropout_keep_mask(2, 2, sq, sk, p)
    got = _run(q, k, v, do, window, sinks, dropout_p=p)
    _check(got, q, k, v, do, window, sinks, keep=keep, p_drop=effective_dropout_p(p))


@pytest.mark.parametrize("d", [64, 128])
def test_dropout_with_keep_bits_in_memory(d):
    """Many heads: both passes of the backward in launches of their own, keep bits handed over in pieces."""
    q, k, v, do = _tensors(2, 500, 500, 6, d, torch.bfloat16)
    p, window, sinks = 0.5, 150, 3
    torch.cuda.manual_seed(6)
    keep = dropout_keep_mask(2, 6, 500, 500, p)
    rng = native.ops().philox_reserve(2 * 6 * 500 * 500)
    ops, scale = native.ops(), 1.0 / math.sqrt(d)
    with torch.no_grad():
        out, lse = ops.flash_attn_fwd(q, k, v, None, None, True, scale, p, rng, window, sinks)
        for words in (1, 16 * 512 * 5):
            dq, dk, dv, _ = ops.flash_attn_bwd(do, q, k, v, out, lse, None, None, True, scale, p, rng, False,
                                               words, window, sinks)
            _check([out, dq, dk, dv], q, k, v, do, window, sinks, keep=keep, p_drop=0.5)


def test_negative_and_other_scales():
    q, k, v, do = _tensors(1, 270, 270, 2, 64, torch.bfloat16)
    for scale in (1.0, -0.2, 0.01):
        _check(_run(q, k, v, do, 77, 2, scale=scale), q, k, v, do, 77, 2, scale=scale)


def test_a_window_over_everything_is_causal_attention():
    q, k, v, do = _tensors(2, 400, 400, 2, 128, torch.bfloat16)
    want = NF.flash_attention(q, k, v, causal=True)
    want = [want, *torch.autograd.grad(want, (q, k, v), do)]
    for a, b in zip(_run(q, k, v, do, 400, 0), want):
        assert torch.equal(a, b)


def test_same_result_every_time():
    q, k, v, do = _tensors(2, 900, 900, 4, 64, torch.bfloat16)
    first = _run(q, k, v, do, 200, 150)
    for _ in range(5):
        for a, b in zip(first, _run(q, k, v, do, 200, 150)):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    q, k, v, do = _tensors(1, 150, 150, 1, 64, torch.float16)
    got = _run(q, k, v, do, 40, 3)
    # the loss along a direction, by the plain form in 32 bits
    g = torch.Generator(device="cuda").manual_seed(9)
    for i, t in enumerate((q, k, v)):
        u = torch.randn(t.shape, generator=g, device="cuda") * 1e-2

        def loss(sign):
            args = [x.detach().double() for x in (q, k, v)]
            args[i] = args[i] + sign * u.double()
            s = torch.einsum("bihd,bjhd->bhij", args[0], args[1]) / 8.0
            s = s.masked_fill(~_seen(150, 150, 40, 3, None), -math.inf)
            return (torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), args[2]) * do.double()).sum()

        diff = (loss(1.0) - loss(-1.0)) / 2
        want = (got[1 + i].double() * u.double()).sum()
        size = (got[1 + i].double() * u.double()).abs().sum()
        # gradients are rounded to 2^-11 (dS and P within them likewise, and the output in the row term); the
        # difference's own error is of third order in steps of 1e-2
        assert abs(float(diff - want)) <= float(size) * 4 * 2.0 ** -11 + 1e-3 * float(size)


def test_captured():
    q, k, v, do = _tensors(2, 500, 500, 4, 64, torch.bfloat16)
    cache_q = torch.randn(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16)

    def work():
        got = _grads()
        with torch.no_grad():
            return [*got, NF.flash_attention(cache_q, k, v, causal=True, window=60, sinks=2)]

    def _grads():
        out = NF.flash_attention(q, k, v, causal=True, window=60, sinks=2)
        return [out, *torch.autograd.grad(out, (q, k, v), do)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for seed in range(2):
        with torch.no_grad():
            for t, new in zip((q, k, v, do), _tensors(2, 500, 500, 4, 64, torch.bfloat16, seed + 20)):
                t.copy_(new)
        graph.replay()
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("sinks", [0, 4])
def test_generation_over_a_cache(sinks):
    """Token by token over a growing cache = the whole sequence at once, up to the roundings of either."""
    torch.manual_seed(0)
    block = FlashAttention(256, 4, fused_qkv=True, output_proj=True, causal=True, window=20,
                           sinks=sinks).cuda().to(torch.bfloat16).eval()
    x = torch.randn(2, 70, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want, _ = block(x)
        past, got = None, []
        for t in range(70):
            out, past = block(x[:, t:t + 1], layer_past=past, use_cache=True)
            got.append(out)
    err = (torch.cat(got, 1).double() - want.double()).norm() / want.double().norm()
    # heads' outputs rounded twice (2^-8 at most each), the projection's result again
    assert float(err) <= 4 * 2.0 ** -8


def test_refusals():
    q = torch.randn(1, 8, 2, 64, device="cuda", dtype=torch.bfloat16)
    ops = native.ops()
    for causal, rel, window, sinks in ((False, None, 4, 0), (True, None, 0, 2), (True, None, -1, 0),
                                       (True, None, 4, -1), (True, torch.zeros(2, 15, device="cuda"), 4, 0)):
        with pytest.raises(RuntimeError, match="window"):
            ops.flash_attn_fwd(q, q, q, None, rel, causal, 1.0, 0.0, None, window, sinks)
        with pytest.raises(RuntimeError, match="window"):
            ops.flash_attn_bwd(q, q, q, q, q, torch.zeros(1, 2, 8, device="cuda"), None, rel, causal, 1.0,
                               0.0, None, False, 0, window, sinks)
    with pytest.raises(ValueError):
        NF.flash_attention(q, q, q, causal=True, window=0)
    huge = NF.flash_attention(q, q, q, causal=True, window=2 ** 40, sinks=2 ** 40)
    assert torch.equal(huge, NF.flash_attention(q, q, q, causal=True))


@pytest.mark.parametrize("sq,window,sinks", [(1, 500, 4), (40, 300, 0), (40, 300, 130)])
def test_offsets_beyond_32_bits(sq, window, sinks):
    """A cache of more than 2^31 elements: as over the keys alone that any query sees."""
    b, sk, n, d = 2, 600_000, 16, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(b, sq, n, d, generator=g, device="cuda").to(torch.bfloat16)
    do = torch.randn(b, sq, n, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.empty(b, sk, n, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g) for _ in "kv")
    kept = torch.cat((torch.arange(sinks), torch.arange(sk - window - sq + 1, sk))).cuda()
    if sq == 1:
        _check([NF.flash_attention(q, k, v, causal=True, window=window, sinks=sinks)], q, k[:, kept],
               v[:, kept], None, window, sinks)
        return
    out, dq, dk, dv = _run(*(t.requires_grad_() for t in (q, k, v)), do, window, sinks)
    _check([out, dq, dk[:, kept], dv[:, kept]], q, k[:, kept], v[:, kept], do, window, sinks)
    rest = torch.ones(sk, dtype=torch.bool, device="cuda")
    rest[kept] = False
    for t in (dk, dv):
        assert int(t.ne(0).view(b, sk, -1).any(-1)[:, rest].sum()) == 0


def test_two_streams_at_once():
    """Calls in flight together share nothing."""
    q, k, v, do = _tensors(2, 700, 700, 4, 64, torch.bfloat16)
    want = _run(q, k, v, do, 200, 130)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_run(q, k, v, do, 200, 130))
    torch.cuda.synchronize()
    for one in got:
        for a, b in zip(one, want):
            assert torch.equal(a, b)


def test_modes_see_the_operators():
    """Calls go past the dispatcher only where nobody watches it, with the same results."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class WatchFunctions(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    q, k, v, _ = (t.detach() for t in _tensors(2, 1, 300, 4, 64, torch.bfloat16))
    ids = torch.arange(5, device="cuda")
    bias = torch.zeros(2, 300, device="cuda")
    for b in (None, bias, bias.to(torch.bfloat16)):       # (the last is converted in Python)
        plain = NF.flash_attention(q, k, v, b, causal=True, window=200, sinks=3)
        for mode in (Watch, WatchFunctions):
            seen.clear()
            with mode():
                watched = NF.flash_attention(q, k, v, b, causal=True, window=200, sinks=3)
            # (a dispatch mode sees what the operator allocates, as of every operator of the extension)
            assert any(("flash" if mode is WatchFunctions else "empty") in name for name in seen)
            assert torch.equal(plain, watched)
    table = q.reshape(8, 64)
    plain = NF.embedding(ids, table, scale=2.0)
    seen.clear()
    with WatchFunctions():
        watched = NF.embedding(ids, table, scale=2.0)
    assert any("embedding" in name for name in seen) and torch.equal(plain, watched)


def test_tensors_that_calls_do_not_take_as_they_are():
    """Subclasses, odd strides, parameters, another default for the scale: the same as contiguous tensors."""
    class Sub(torch.Tensor):
        pass

    q, k, v, do = _tensors(2, 130, 130, 4, 64, torch.bfloat16)
    want = _run(q, k, v, do, 100, 3)
    got = _run(*(torch.nn.Parameter(t.detach()) for t in (q, k, v)), do, 100, 3, scale=0.125)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    out = NF.flash_attention(*(t.detach().as_subclass(Sub) for t in (q, k, v)), causal=True, window=100,
                             sinks=3)
    assert torch.equal(out.as_subclass(torch.Tensor), want[0].detach())
    with pytest.raises(Exception, match="Expected|sizes|size"):
        NF.flash_attention(q, k.detach()[:, :, :2], v, causal=True, window=100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s,d", [(3, 64), (100, 40), (128, 128), (300, 64), (300, 80), (777, 128)])
def test_what_the_output_loses_by_rounding(s, d, dtype):
    """With q = 0 and a window of two keys the output is the mean of two values, exact in fp32: a byte holds
    the next eight bits, so that less than one of their last (2^8 or 2^5 of fp32's 2^-23 of the value) stays
    lost.  Nothing is held of ties and what begins like one, nor of fp16's denormals."""
    _, _, v, do = _tensors(2, s, s, 3, d, dtype)
    v = v.detach()
    q = torch.zeros_like(v)
    ops = native.ops()
    out, lse, rest = ops.flash_attn_fwd_rest(q, v, v, None, None, True, 1.0, 0.0, None, 2, 0)
    x = v.double()
    x[:, 1:] = (x[:, 1:] + x[:, :-1]) / 2
    assert torch.equal(out, x.to(dtype))
    byte = rest.view(torch.int8).int()
    lost = out.float().view(torch.int32) + byte * (32 if dtype == torch.float16 else 256)
    left_out = byte == 0
    if dtype == torch.float16:
        left_out |= out.abs() < 2.0 ** -14
    assert int((byte == -128).sum()) == 0
    got = torch.where(left_out, out.float(), lost.view(torch.float32)).double()
    step = 2.0 ** (-18 if dtype == torch.float16 else -15)
    room = torch.where(left_out, HALF[dtype], step) * x.abs() * (1 + HALF[dtype])
    assert bool(((got - x).abs() <= room.clamp(min=2.0 ** -25)).all())
    args = (do, q, v, v, out, lse, None, None, True, 1.0, 0.0, None, False, 0, 2, 0)
    for given in (rest, rest[:0], None):
        assert all(bool(t.isfinite().all()) for t in ops.flash_attn_bwd(*args, given)[:3])
    for bad in (rest[:, :, :1], rest.view(torch.int8), rest.cpu(), rest.flatten()[1:]):
        with pytest.raises(RuntimeError, match="byte"):
            ops.flash_attn_bwd(*args, bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_carry_two_roundings(dtype):
    """dQ and dK: dS and the result are rounded to the type, each an independent error of the same size (a
    factor of sqrt 2 over the result's alone).  The output in the row term comes without its rounding; that of
    the probabilities in it, with many rows that see few keys, measured in 64 bits, adds 0.3 of one: 1.45."""
    b, s, n, d, window, sinks = 4, 1000, 4, 80, 201, 5
    q, k, v, do = _tensors(b, s, s, n, d, dtype)
    bias = torch.zeros(b, s, device="cuda")
    for i in range(b):
        bias[i, 500 + 100 * i:] = -10000.0
    got = _run(q, k, v, do, window, sinks, bias)
    q64, k64, v64 = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    p = q64 @ k64.transpose(-1, -2) / math.sqrt(d) + bias.double()[:, None, None]
    p = torch.softmax(p.masked_fill(~_seen(s, s, window, sinks, bias), -math.inf), -1)
    dp = do.double().transpose(1, 2) @ v64.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
    for x, want in ((got[1], ds @ k64), (got[2], ds.transpose(-1, -2) @ q64)):
        want = want.transpose(1, 2)
        rounding = (want.to(dtype).double() - want).norm()
        assert float((x.double() - want).norm() / rounding) < 1.5


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("packed", [True, False])
def test_nothing_is_kept_for_a_backward_that_will_not_be(packed, p):
    """Without a gradient: the output (and row sums while the call runs), not a byte for each of its values
    besides; the output is that of a call with a gradient."""
    b, s, h, d = 2, 500, 4, 64
    qkv = torch.randn(b, s, h, 3, d, device="cuda", dtype=torch.bfloat16)
    bias = torch.zeros(b, s, device="cuda")
    bias[:, 400:] = -10000.0

    def call(qkv):
        torch.manual_seed(3)
        if packed:
            return flash_attention_qkvpacked(qkv, bias, True, p=p, window=64, sinks=2)
        return NF.flash_attention(*qkv.unbind(3), bias, True, dropout_p=p, window=64, sinks=2)

    want = call(qkv.clone().requires_grad_())
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            got = call(qkv)             # (not a leaf that wants one)
            assert torch.equal(got, want) and got.grad_fn is None
            del got
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            held = torch.cuda.memory_allocated()
            got = call(qkv)
            kept = torch.cuda.max_memory_allocated() - held
            # output, log sums, the generator's place; each rounded up to 512 bytes
            assert kept <= b * s * h * (2 * d + 4) + 4 * 512, kept
            del got


@pytest.mark.parametrize("s,n,window,sinks,d", [(8192, 1, 256, 4, 128), (8000, 1, 256, 4, 64), (4096, 3, 128, 1, 64),
                                                (3001, 1, 65, 300, 32), (2600, 2, 1, 129, 128)])
def test_shares_of_the_sinks_queries(s, n, window, sinks, d):
    """Few heads and many queries: the sinks' are dealt out to many work items, some of one half tile more."""
    q, k, v, do = _tensors(1, s, s, n, d, torch.bfloat16, seed=s)
    _check(_run(q, k, v, do, window, sinks), q, k, v, do, window, sinks)


@pytest.mark.multigpu
@pytest.mark.parametrize("sq", [1, 130])
def test_a_bias_on_another_device_is_refused(sq):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    q = torch.randn(1, sq, 2, 64, device="cuda:0", dtype=torch.bfloat16)
    k = torch.randn(1, 200, 2, 64, device="cuda:0", dtype=torch.bfloat16)
    bias = torch.zeros(1, 200, device="cuda:1")
    for window in (None, 64):
        with pytest.raises(RuntimeError, match="device of the queries"):
            NF.flash_attention(q, k, k, bias, causal=True, window=window)
    with pytest.raises(RuntimeError, match="one device"):
        NF.flash_attention(q, k.to("cuda:1"), k, None, causal=True, window=64)


@pytest.mark.parametrize("sq,sk", [(300, 300), (1, 300)])
def test_the_lowest_value_of_a_16bit_mask(sq, sk):
    """-65504 of an fp16 mask hides a key as -inf does, in all entries."""
    q, k, v, do = _tensors(3, sq, sk, 2, 64, torch.float16, seed=4)
    at = torch.arange(sk, device="cuda")
    pad = torch.stack([at >= sk - 120, at < sk // 2, at >= 0])
    low, inf = (torch.zeros(3, sk, device="cuda", dtype=t).masked_fill(pad, x)
                for t, x in ((torch.float16, -65504.0), (torch.float32, -math.inf)))
    got = _run(q, k, v, do, 33, 2, low)
    for a, b in zip(got, _run(q, k, v, do, 33, 2, inf)):
        assert torch.equal(a, b)
    _check(got, q, k, v, do, 33, 2, inf)
    assert bool((got[0][2] == 0).all())
    if sq == sk:
        qkv = torch.stack((q, k, v), 3).detach()
        assert torch.equal(flash_attention_qkvpacked(qkv, low, True, window=33, sinks=2), got[0])


@pytest.mark.parametrize("sq,sk", [(1, 700), (60, 700), (700, 700), (300, 130), (200, 1)])
@pytest.mark.parametrize("window,sinks", [(700, 0), (650, 50), (1, 699), (900, 900)])
def test_what_reaches_over_all_keys_is_no_window(sq, sk, window, sinks):
    """Output and gradients to the bit, queries before all keys (zeros) among them; and with a bias, whose
    masked keys then count as with a window, rows of nothing but such keys are zeros."""
    q, k, v, do = _tensors(2, sq, sk, 2, 64, torch.bfloat16, seed=sq)
    out = NF.flash_attention(q, k, v, causal=True)
    want = [out, *torch.autograd.grad(out, (q, k, v), do)]
    got = _run(q, k, v, do, window, sinks)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    _check(got, q, k, v, do, window, sinks)
    bias = torch.zeros(2, sk, device="cuda")
    bias[1] = torch.finfo(torch.float32).min
    got = _run(q, k, v, do, window, sinks, bias)
    _check(got, q, k, v, do, window, sinks, bias)
    assert bool((got[0][1] == 0).all()) and all(bool((g[1] == 0).all()) for g in got[1:])
