"""The operators around a decoder's layers, as cases that can be timed and compared.

Three operators that a training step of a GPT-Neo-like decoder has besides its plain layers, and what
generation needs of them: the token table's lookup (scaled, with a padding id) and its gradient by sorted
tokens; attention in which a token sees a window of tokens before it and a few first ones (sinks), its
gradients, and its form for one new token over a cache; the AdamW step over all tensors of a model at once,
with moments in 32 bits or in 8.  Sizes are those of this repository's BERT, ALBERT, GPT-Neo and OPT
configurations, or generic.

With ``own`` set, ``run`` calls the framework; without, it computes the same in elementary torch operations.

The 8-bit moments of AdamW are blocks of 256 values of a tensor in row order: e4m3 numbers and one power of
two per block, the smallest with which the block's largest value fits (448), and at least 2^-126.  The first
moment is held itself, the second as its square root, which never becomes zero by rounding.  They are returned
as the e4m3 values they are, beside their blocks' factors.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256
HIDDEN = -1e30      # a key with a bias below this is not seen at all


def listed():
    return [
        # BERT-large's word table in the benchmark's step: 32 right-padded sequences of 512
        {"name": "embed_bert_large", "kind": "embed", "batch": 32, "seq": 512, "vocab": 30528,
         "hidden": 1024, "pad": True, "hot": 0.0, "scale": 1.0, "train": True, "dtype": "bf16",
         "ids": "int64"},
        # GPT-Neo-1.3B's padded vocabulary, a micro-batch of 4 x 2048, the table scaled by sqrt(hidden)
        {"name": "embed_gpt_neo", "kind": "embed", "batch": 4, "seq": 2048, "vocab": 50304,
         "hidden": 2048, "pad": False, "hot": 0.15, "scale": 45.25, "train": True, "dtype": "bf16",
         "ids": "int64"},
        # ALBERT's factorised table on one short odd sequence, 32-bit weights: launches count
        {"name": "embed_albert_short", "kind": "embed", "batch": 1, "seq": 201, "vocab": 30000,
         "hidden": 128, "pad": True, "hot": 0.0, "scale": 1.0, "train": True, "dtype": "fp32",
         "ids": "int64"},
        # the tokens that eight sequences of OPT-2.7B have just generated
        {"name": "embed_decode", "kind": "embed", "batch": 8, "seq": 1, "vocab": 50272, "hidden":
         2560, "pad": False, "hot": 0.0, "scale": 1.0, "train": False, "dtype": "fp16", "ids":
         "int64"},
        # GPT-Neo-1.3B's local layers at their full context: packed projections, window 256
        {"name": "window_gpt_neo", "kind": "attn", "batch": 4, "sq": 2048, "sk": 2048, "heads": 16,
         "dim": 128, "window": 256, "sinks": 0, "packed": True, "mask": "none", "train": True,
         "dtype": "bf16"},
        # a long document: window 1024 and four sinks, heads of 64
        {"name": "window_long_sinks", "kind": "attn", "batch": 1, "sq": 8192, "sk": 8192, "heads":
         12, "dim": 64, "window": 1024, "sinks": 4, "packed": False, "mask": "none", "train": True,
         "dtype": "bf16"},
        # OPT-2.7B's heads of 80 on right-padded prompts, odd length, odd window, a few sinks
        {"name": "window_ragged", "kind": "attn", "batch": 4, "sq": 1000, "sk": 1000, "heads": 32,
         "dim": 80, "window": 201, "sinks": 5, "packed": False, "mask": "pad", "train": True,
         "dtype": "fp16"},
        # one generated token of GPT-Neo-1.3B's local layers for eight sequences, sinks kept
        {"name": "window_decode", "kind": "attn", "batch": 8, "sq": 1, "sk": 1501, "heads": 16,
         "dim": 128, "window": 256, "sinks": 4, "packed": False, "mask": "none", "train": False,
         "dtype": "bf16"},
        # all tensors of a 12-layer model of BERT-large's width: 16-bit weights, 32-bit masters and moments
        {"name": "adamw_12_layers", "kind": "adamw", "layers": 12, "hidden": 1024, "vocab": 30528,
         "tensors": 0, "largest": 0, "bits": 32, "master": True, "dtype": "bf16", "step": 100},
        # the same with moments in 8 bits
        {"name": "adamw_12_layers_8bit", "kind": "adamw", "layers": 12, "hidden": 1024, "vocab":
         30528, "tensors": 0, "largest": 0, "bits": 8, "master": True, "dtype": "bf16", "step": 100},
        # four layers of GPT-Neo-1.3B's width and its table, moments in 8 bits, no masters
        {"name": "adamw_wide_8bit", "kind": "adamw", "layers": 4, "hidden": 2048, "vocab": 50304,
         "tensors": 0, "largest": 0, "bits": 8, "master": False, "dtype": "bf16", "step": 7},
        # the many small tensors of adapters and norms in 32 bits: launches count
        {"name": "adamw_small", "kind": "adamw", "layers": 0, "hidden": 0, "vocab": 0, "tensors":
         50, "largest": 20000, "bits": 32, "master": False, "dtype": "fp32", "step": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "attn", "attn", "adamw"])
    if kind == "embed":
        hidden = rng.choice([64, 100, 128, 333, 512, 768, 1024, 1600, 2048, 2560])
        vocab = _log(rng, 500, 50304)
        seq = _log(rng, 1, 2048)
        batch = _log(rng, 1, max(1, min(64, 16384 * 1024 // (seq * hidden))))
        return {"kind": "embed", "batch": batch, "seq": seq, "vocab": vocab, "hidden": hidden,
                "pad": rng.random() < 0.4, "hot": rng.choice([0.0, 0.0, 0.2, 1.0]),
                "scale": rng.choice([1.0, round(math.sqrt(hidden), 2)]), "train": rng.random() < 0.8,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "ids": rng.choice(["int64", "int64", "int32"])}
    if kind == "attn":
        train = rng.random() < 0.65
        dim = rng.choice([32, 64, 64, 80, 128, 128])
        heads = rng.choice([4, 8, 12, 16, 20])
        sk = _log(rng, 20, 8192)
        one = not train and rng.random() < 0.7
        packed = train and rng.random() < 0.4
        sq = 1 if one else sk if packed or rng.random() < 0.6 else rng.randint(1, sk)
        heads = min(heads, max(1, int(8.0e8 / (sq * sk))))
        most = max(1, int(8.0e8 / (heads * sq * sk)))
        return {"kind": "attn", "batch": rng.randint(1, min(8, most)), "sq": sq, "sk": sk, "heads": heads,
                "dim": dim, "window": _log(rng, 1, 2048), "sinks": rng.choice([0, 0, 1, 4, 7, 64, 200]),
                "packed": packed, "mask": rng.choice(["none", "none", "pad", "lowest"]), "train": train,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = {"kind": "adamw", "layers": 0, "hidden": 0, "vocab": 0, "tensors": 0, "largest": 0,
            "bits": rng.choice([8, 32]), "master": dtype != "fp32" and rng.random() < 0.6, "dtype": dtype,
            "step": _log(rng, 1, 20000)}
    if rng.random() < 0.5:
        case.update(layers=rng.randint(1, 8), hidden=rng.choice([256, 512, 1024]),
                    vocab=_log(rng, 500, 50304))
    else:
        case.update(tensors=_log(rng, 1, 400), largest=_log(rng, 10, 400000))
    return case


# --------------------------------------------------------------------------- #
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(gen, shape, std, dtype):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _sizes(case):
    """Elements of the step's tensors, and which of them weight decay leaves alone (vectors)."""
    h, sizes = case["hidden"], []
    if case["layers"]:
        sizes = [(case["vocab"] * h, True), (512 * h, True)]
        for _ in range(case["layers"]):
            sizes += [(h * h, True), (h, False)] * 4 + [(h, False)] * 4
            sizes += [(4 * h * h, True), (4 * h, False), (4 * h * h, True), (h, False)]
        return sizes + [(h, False), (h, False)]
    # sizes between 1 and `largest`, spread over their logarithm
    n, top = case["tensors"], math.log(case["largest"])
    for i in range(n):
        size = int(round(math.exp(top * ((i * 0.6180339887 + 0.5) % 1.0)))) if i else case["largest"]
        sizes.append((size, i % 3 != 1))
    return sizes


def prepare(case, seed):
    gen = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "embed":
        shape = (case["batch"], case["seq"])
        v, h = case["vocab"], case["hidden"]
        # token ids by falling frequency: the k-th has a share of about 1 / k
        u = torch.rand(shape, generator=gen, device=DEV, dtype=torch.float64)
        ids = (torch.exp(u * math.log(v)).floor().long() - 1).clamp(0, v - 1)
        if case["hot"]:
            some = torch.rand(shape, generator=gen, device=DEV) < case["hot"]
            ids[some] = v // 3
        if case["pad"]:
            length = torch.randint((shape[1] + 1) // 2, shape[1] + 1, (shape[0], 1), generator=gen,
                                   device=DEV)
            ids[torch.arange(shape[1], device=DEV)[None] >= length] = 0
        s = {"case": case, "ids": ids.to(torch.int32 if case["ids"] == "int32" else torch.int64),
             "weight": _normal(gen, (v, h), 0.02, dtype)}
        if case["train"]:
            s["dy"] = _normal(gen, shape + (h,), 1e-3, dtype)
            s["weight"].requires_grad_()
        return s
    if case["kind"] == "attn":
        b, sq, sk, n, d = (case[k] for k in ("batch", "sq", "sk", "heads", "dim"))
        s = {"case": case}
        if case["packed"]:
            s["qkv"] = _normal(gen, (b, sq, n, 3, d), 1.0, dtype)
        else:
            s["q"] = _normal(gen, (b, sq, n, d), 1.0, dtype)
            s["k"] = _normal(gen, (b, sk, n, d), 1.0, dtype)
            s["v"] = _normal(gen, (b, sk, n, d), 1.0, dtype)
        s["bias"] = None
        if case["mask"] != "none":
            length = torch.randint((sk + 1) // 2, sk + 1, (b, 1), generator=gen, device=DEV)
            pad = torch.arange(sk, device=DEV)[None] >= length
            low = -10000.0 if case["mask"] == "pad" else torch.finfo(torch.float32).min
            s["bias"] = torch.zeros(b, sk, device=DEV).masked_fill(pad, low)
        if case["train"]:
            s["dout"] = _normal(gen, (b, sq, n, d), 1.0, dtype)
            for name in ("qkv", "q", "k", "v"):
                if name in s:
                    s[name].requires_grad_()
        return s
    sizes = _sizes(case)
    at, total = [], 0
    for size, _ in sizes:       # (each tensor begins a block of its own)
        at.append(total)
        total += -(-size // BLOCK) * BLOCK
    real, decay = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    for (size, decays), a in zip(sizes, at):
        real[a:a + size] = 1.0
        decay[a:a + size] = 0.01 if decays else 0.0
    weights = torch.randn(total, generator=gen, device=DEV) * 0.02 * real
    grad = torch.randn(total, generator=gen, device=DEV) * real
    # a few rows have much larger gradients than the others
    spread = torch.exp(2.0 * torch.randn(total // BLOCK, 1, generator=gen, device=DEV))
    grad = (grad.view(-1, BLOCK) * spread * 1e-3).view(-1)
    m = torch.randn(total, generator=gen, device=DEV) * 3e-4 * real
    u = (m.abs() + 1e-3 * torch.rand(total, generator=gen, device=DEV)) * real
    s = {"case": case, "param": weights.to(dtype), "grad": grad.to(dtype), "master": None, "decay": decay,
         "grad_scale": torch.full((1,), 0.75, device=DEV), "sizes": sizes, "at": at}
    if case["master"]:
        s["master"] = weights
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _to_8bit(m, False)
        s["v"], s["v_scale"] = _to_8bit(u, True)
    else:
        s["m"], s["v"] = m, u * u
    cut = [(a, a + size) for (size, _), a in zip(sizes, at)]
    for name in ("param", "grad", "master", "m", "v"):
        if s[name] is not None:
            s[name + "s"] = [s[name][a:e] for a, e in cut]
    if case["bits"] == 8:
        for name in ("m_scale", "v_scale"):
            s[name + "s"] = [s[name][a // BLOCK:-(-e // BLOCK)] for a, e in cut]
    s["decays"] = [0.01 if decays else 0.0 for _, decays in sizes]
    return s


def _to_8bit(x, keep_above_zero):
    """Values (a multiple of BLOCK) as e4m3 numbers and their blocks' factors."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True).clamp(min=2.0 ** -126)
    mant, exp = torch.frexp(top)
    exp = torch.where(mant > 0.875, exp - 8, exp - 9).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(top), exp)
    y = torch.ldexp(x, -exp).to(torch.float8_e4m3fn)
    if keep_above_zero:
        y = torch.where((x > 0) & (y.float() == 0), torch.full_like(x, 2.0 ** -9), y.float())
        y = y.to(torch.float8_e4m3fn)
    return y.view(-1), scale.view(-1)


LR, BETAS, EPS = 1e-4, (0.9, 0.999), 1e-8


# --------------------------------------------------------------------------- #
def run(state):
    if own:
        return _run_own(state)
    return {"embed": _embed, "attn": _attn, "adamw": _adamw}[state["case"]["kind"]](state)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "embed":
        from slapo_b200.ops import functional as NF

        out = NF.embedding(s["ids"], s["weight"], padding_idx=0 if c["pad"] else None,
                           scale=c["scale"])
        if not c["train"]:
            return out
        return out.detach(), torch.autograd.grad(out, s["weight"], s["dy"])[0]
    if c["kind"] == "attn":
        from slapo_b200.ops import functional as NF
        from slapo_b200.ops.flash_attn import flash_attention_qkvpacked

        more = {"causal": True, "window": c["window"], "sinks": c["sinks"]}
        if c["packed"]:
            out = flash_attention_qkvpacked(s["qkv"], s["bias"], **more)
            inputs = [s["qkv"]]
        else:
            out = NF.flash_attention(s["q"], s["k"], s["v"], s["bias"], **more)
            inputs = [s["q"], s["k"], s["v"]]
        if not c["train"]:
            return out
        return [out.detach(), *torch.autograd.grad(out, inputs, s["dout"])]
    from slapo_b200.op import multi_tensor_adamw

    more = {"masters": s["masters"]} if c["master"] else {}
    if c["bits"] == 8:
        more.update(exp_avg_scales=s["m_scales"], exp_avg_sq_scales=s["v_scales"])
    multi_tensor_adamw(s["params"], s["grads"], s["ms"], s["vs"], lr=LR, betas=BETAS, eps=EPS,
                       weight_decay=s["decays"], step=c["step"], grad_scale=s["grad_scale"], **more)
    return _adamw_outputs(s)


def _embed(s):
    c, ids, w = s["case"], s["ids"].long(), s["weight"].detach()
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return out
    dy = s["dy"].float()
    if c["pad"]:
        dy = dy * (ids != 0)[..., None]
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, ids.view(-1), dy.view(-1, w.shape[1]))
    return out, (dw * c["scale"]).to(w.dtype)


def _seen(c, bias, device):
    """[1 or B, 1, Sq, Sk]: which keys a query sees."""
    i = torch.arange(c["sq"], device=device)[:, None] + (c["sk"] - c["sq"])
    j = torch.arange(c["sk"], device=device)[None]
    seen = (j <= i) & ((j > i - c["window"]) | (j < c["sinks"]))
    seen = seen[None, None]
    return seen if bias is None else seen & (bias >= HIDDEN)[:, None, None]


def _attn(s):
    c = s["case"]
    q, k, v = (s["qkv"].detach().unbind(3) if c["packed"] else (s[n].detach() for n in "qkv"))
    dtype, scale = q.dtype, 1.0 / math.sqrt(c["dim"])
    q, k, v = (t.transpose(1, 2).float() for t in (q, k, v))
    hidden = ~_seen(c, s["bias"], q.device)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if s["bias"] is not None:
        p += s["bias"][:, None, None]
    p.masked_fill_(hidden, float("-inf"))
    top = p.amax(-1, keepdim=True).clamp(min=-3e38)     # (a row that sees no key: its probabilities are 0)
    p.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p, v)
    if not c["train"]:
        return out.transpose(1, 2).to(dtype)
    do = s["dout"].transpose(1, 2).float()
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds.sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    out, dq, dk, dv = (t.transpose(1, 2).to(dtype) for t in (out, dq, dk, dv))
    return [out, torch.stack((dq, dk, dv), 3)] if c["packed"] else [out, dq, dk, dv]


def _adamw(s):
    """Every product and sum in 32 bits, each rounded by itself; all tensors of a kind lie in one buffer."""
    c, (b1, b2) = s["case"], BETAS
    g = s["grad"].float() * s["grad_scale"]
    if c["bits"] == 8:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g * g * (1.0 - b2)
    u = v.sqrt()
    w = s["master"] if c["master"] else s["param"].float()
    step = (m / (1.0 - b1 ** c["step"])) / (u / math.sqrt(1.0 - b2 ** c["step"]) + EPS)
    w = w - LR * (step + s["decay"] * w)
    if c["master"]:
        s["master"].copy_(w)
    s["param"].copy_(w)
    if c["bits"] == 8:
        for name, x in (("m", m), ("v", u)):
            y, scale = _to_8bit(x, name == "v")
            s[name].copy_(y)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {n: s[n] for n in ("param", "master", "m", "v", "m_scale", "v_scale") if s.get(n) is not None}


# --------------------------------------------------------------------------- #
def work(case):
    c = case
    e = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    if c["kind"] == "embed":
        n, row = c["batch"] * c["seq"], c["hidden"] * e
        size = n * (8 if c["ids"] == "int64" else 4) + min(n, c["vocab"]) * row + n * row
        flops = n * c["hidden"]
        if c["train"]:
            size += n * row + c["vocab"] * row
            flops *= 2
        return {"bytes": size, "flops": flops}
    if c["kind"] == "attn":
        first, w, sinks = c["sk"] - c["sq"], c["window"], c["sinks"]
        pairs = keys = 0
        for i in range(first, c["sk"]):
            pairs += min(w, i + 1) + min(sinks, max(0, i + 1 - w))
        keys = c["sk"] - max(0, first - w + 1) + min(sinks, max(0, first - w + 1))
        tokens = c["batch"] * c["heads"] * c["dim"] * e
        q, kv = c["sq"] * tokens, keys * tokens
        pairs *= c["batch"] * c["heads"]
        if not c["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * c["dim"]}
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * c["dim"]}
    n = sum(size for size, _ in _sizes(c))
    weights = (8 + e) if c["master"] else 2 * e
    moments = 16 if c["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (e + weights + moments), "flops": 20 * n}


# --------------------------------------------------------------------------- #
def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "embed":
        ids, w = s["ids"].reshape(-1).long(), s["weight"].detach().double()
        out = torch.empty(*s["ids"].shape, case["hidden"], dtype=torch.float64, device=DEV)
        torch.index_select(w, 0, ids, out=out.view(-1, case["hidden"]))
        out *= case["scale"]
        if not case["train"]:
            return out
        dy = s["dy"].double().reshape(ids.numel(), -1)
        order = torch.argsort(ids, stable=True)
        if case["pad"]:
            order = order[ids[order] != 0]
        total = torch.cat([dy.new_zeros(1, dy.shape[1]), dy[order].cumsum(0)])
        row, count = torch.unique_consecutive(ids[order], return_counts=True)
        end = count.cumsum(0)
        dw = torch.zeros_like(w)
        dw[row] = total[end] - total[end - count]
        return out, dw * case["scale"]
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    return _exact_adamw(case, s)


def _exact_attn(c, s):
    parts = s["qkv"].unbind(3) if c["packed"] else [s[n] for n in "qkv"]
    q, k, v = (t.detach().double() for t in parts)
    do = s["dout"].double() if c["train"] else None
    outs = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)]
    pos_q = torch.arange(c["sk"] - c["sq"], c["sk"], device=DEV)
    pos_k = torch.arange(c["sk"], device=DEV)
    back = pos_q[:, None] - pos_k[None, :]
    for b in range(c["batch"]):
        near = (back < c["window"]) | (pos_k[None] < c["sinks"])
        add = torch.where((back >= 0) & near, 0.0, -math.inf).double()
        if s["bias"] is not None:
            add = add + torch.where(s["bias"][b] < HIDDEN, -math.inf, s["bias"][b].double())
        for h in range(c["heads"]):
            x = q[b, :, h] @ k[b, :, h].T / math.sqrt(c["dim"]) + add
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
            outs[0][b, :, h] = p @ v[b, :, h]
            if c["train"]:
                g = do[b, :, h]
                dp = g @ v[b, :, h].T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(c["dim"])
                outs[1][b, :, h] = ds @ k[b, :, h]
                outs[2][b, :, h] = ds.T @ q[b, :, h]
                outs[3][b, :, h] = p.T @ g
    if not c["train"]:
        return outs[0]
    return [outs[0], torch.stack(outs[1:], 3)] if c["packed"] else outs


def _exact_8bit(x, keep_above_zero):
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    # the smallest power of two that the largest value fits under 448 times
    exp = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=-126.0)
    exp = torch.where(top > 448.0 * torch.exp2(exp), exp + 1, exp)
    exp = torch.where((exp > -126) & (top <= 448.0 * torch.exp2(exp - 1)), exp - 1, exp)
    y = x / torch.exp2(exp)
    # three bits behind the leading one, steps of 2^-9 below 2^-6; ties to even
    ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.round(y / ulp) * ulp
    if keep_above_zero:
        y = torch.where((x > 0) & (y == 0), 2.0 ** -9, y)
    return y.view(-1), torch.exp2(exp).view(-1)


def _exact_adamw(c, s):
    g = s["grad"].double() * s["grad_scale"].double()
    m, u = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["m_scale"].double()[:, None]).view(-1)
        u = (u.view(-1, BLOCK) * s["v_scale"].double()[:, None]).view(-1)
        v = u * u
    else:
        v = u
    t = c["step"]
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    w = (s["master"] if c["master"] else s["param"]).double()
    decay = torch.where(s["decay"] > 0, 0.01, 0.0).double()
    w = w * (1 - LR * decay) - LR * (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
    got = {"param": w, "m": m, "v": v}
    if c["master"]:
        got["master"] = w.clone()
    if c["bits"] == 8:
        got["m"], got["m_scale"] = _exact_8bit(m, False)
        got["v"], got["v_scale"] = _exact_8bit(torch.sqrt(v), True)
    return got
