"""Generation over a paged cache in 8 bits, as cases that can be timed and compared.

Four operators: the rotation of queries and keys by their positions (with its gradient, as training needs it);
new tokens' keys and values appended to a cache of pages in 8 bits, rotated on the way; attention of the newest
tokens over that cache; the next token drawn from the logits by a given random number.  Sizes are those of this
repository's GPT-2, GPT-Neo, OPT and BERT configurations, or generic.

With ``own`` set, ``run`` calls the framework; without, it computes the same in elementary torch operations.

Rotation: a table ``[positions, rotary / 2, 2]`` of cosines and sines in 32 bits; the pair ``(a, b)`` of a head
becomes ``(a cos - b sin, b cos + a sin)``.  Pairs are the halves of the rotated part (``half``) or neighbours
(``pairs``); what lies behind the rotated part stays.

Cache: ``pages [P, 2, H, T, D']`` of e4m3 numbers (keys and values, a head's T tokens in a row, D' the head's
width up to a multiple of 16), ``scales [P, 2, H]`` in 32 bits: a power of two for each page, side and head, the
smallest with which the largest value fits (448), and at least 2^-100.  ``block_table [B, pages]`` names a
sequence's pages in their order; ``lengths [B]`` counts its tokens, the new ones among them; of ``n`` new ones
a sequence brings the first ``counts[b]``, its last tokens.  A page's scale only grows while tokens are added,
and the codes that are there are then rounded to the new one.

Sampling: logits over the temperature; the ``top_k`` largest, ties in the order of their indices; of their mass
the shortest row of largest ones that holds ``top_p`` of it; of those, what has ``min_p`` of the largest one's
probability; then the first token, in the order of the indices, at which the sum passes the random number times
the kept mass.  Temperature 0: the largest, the first one of equals.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
TOP = 448.0
LEAST = -100


def listed():
    return [
        # GPT-Neo-1.3B's heads in a training step of 4 x 2048: rotation inside of a packed projection, its gradient
        {"name": "rotary_gpt_neo", "kind": "rotary", "batch": 4, "seq": 2048, "heads": 16, "kv_heads": 16,
         "dim": 128, "rotary": 128, "layout": "half", "packed": True, "scaling": "none", "table": 2048,
         "start": 0, "by_token": False, "train": True, "dtype": "bf16"},
        # a long document of odd length, OPT-2.7B's heads of 80 with a few shared key heads: neighbours in half of
        # the head, the table stretched for four times its context
        {"name": "rotary_long_part", "kind": "rotary", "batch": 1, "seq": 12001, "heads": 32, "kv_heads": 4,
         "dim": 80, "rotary": 40, "layout": "pairs", "packed": False, "scaling": "yarn", "table": 16384,
         "start": 4000, "by_token": False, "train": True, "dtype": "fp16"},
        # one token each of eight sequences at their own positions: launches count
        {"name": "rotary_token", "kind": "rotary", "batch": 8, "seq": 1, "heads": 16, "kv_heads": 16,
         "dim": 128, "rotary": 128, "layout": "half", "packed": False, "scaling": "ntk", "table": 8192,
         "start": 0, "by_token": True, "train": False, "dtype": "fp32"},
        # a generated token of eight sequences of GPT-Neo-1.3B
        {"name": "append_token", "kind": "append", "batch": 8, "n": 1, "heads": 16, "kv_heads": 16, "dim": 128,
         "page": 64, "past": 1500, "ragged": True, "rotary": 128, "layout": "half", "dtype": "bf16"},
        # prompts of four sequences, right-padded to an odd length, on top of what is there; OPT-2.7B's heads
        {"name": "append_prompts", "kind": "append", "batch": 4, "n": 1001, "heads": 32, "kv_heads": 32, "dim":
         80, "page": 32, "past": 301, "ragged": True, "rotary": 40, "layout": "pairs", "dtype": "fp16"},
        # eight whole contexts of GPT-Neo-1.3B into an empty cache
        {"name": "append_contexts", "kind": "append", "batch": 8, "n": 2048, "heads": 16, "kv_heads": 16, "dim":
         128, "page": 64, "past": 0, "ragged": False, "rotary": 128, "layout": "half", "dtype": "bf16"},
        # a generated token of eight sequences of GPT-Neo-1.3B, each head with its own cache
        {"name": "attend_token", "kind": "attend", "batch": 8, "n": 1, "heads": 16, "kv_heads": 16, "dim": 128,
         "page": 64, "length": 1501, "ragged": True, "window": 0, "dtype": "bf16"},
        # long sequences of very different lengths, eight query heads to a cached one: the largest
        {"name": "attend_long", "kind": "attend", "batch": 16, "n": 1, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 64, "length": 32001, "ragged": True, "window": 0, "dtype": "bf16"},
        # a few tokens at once (a guess that is checked), OPT-2.7B's heads, a window over an odd number of tokens
        {"name": "attend_few_window", "kind": "attend", "batch": 4, "n": 5, "heads": 32, "kv_heads": 32, "dim":
         80, "page": 16, "length": 2003, "ragged": True, "window": 1001, "dtype": "fp16"},
        # the next tokens of eight sequences, GPT-Neo's padded vocabulary
        {"name": "sample_eight", "kind": "sample", "batch": 8, "vocab": 50304, "temperature": 0.8, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "mixed": False, "dtype": "bf16"},
        # a full server's batch, OPT's vocabulary, each request with settings of its own
        {"name": "sample_mixed", "kind": "sample", "batch": 256, "vocab": 50272, "temperature": 0.7, "top_k":
         200, "top_p": 0.9, "min_p": 0.05, "mixed": True, "dtype": "fp32"},
        # one sequence, BERT's padded vocabulary, nothing cut off
        {"name": "sample_one", "kind": "sample", "batch": 1, "vocab": 30528, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "mixed": False, "dtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "sample":
        return {"kind": kind, "batch": _log(rng, 1, 256), "vocab": _log(rng, 1000, 50300),
                "temperature": rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]), "top_k": rng.choice([0, 1, 40, 50, 500]),
                "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.02, 0.1]),
                "mixed": rng.random() < 0.4, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 4, 8]) if kv < 8 else kv * rng.choice([1, 2])
    dim = rng.choice([64, 72, 80, 96, 128])
    rotary = rng.choice([dim, dim, dim // 2, 32])
    layout = rng.choice(["half", "pairs"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "rotary":
        packed = rng.random() < 0.4
        token = not packed and rng.random() < 0.3
        heads = kv if packed else heads
        batch = _log(rng, 1, 16)
        seq = 1 if token else min(_log(rng, 2, 12000), max(2, 16_000_000 // (batch * (heads + 2 * kv) * dim)))
        start = 0 if packed else rng.randrange(0, 3000)
        return {"kind": kind, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv, "dim": dim, "rotary":
                rotary, "layout": layout, "packed": packed, "scaling": rng.choice(["none", "linear", "ntk",
                "yarn"]), "table": 16384, "start": start, "by_token": token or rng.random() < 0.3, "train":
                not token, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "append":
        batch = _log(rng, 1, 32)
        n = 1 if rng.random() < 0.4 else min(_log(rng, 2, 4000), max(2, 24_000_000 // (batch * (heads + 2 * kv) * dim)))
        return {"kind": kind, "batch": batch, "n": n, "heads": heads, "kv_heads": kv, "dim": dim, "page": page,
                "past": rng.choice([0, _log(rng, 1, 3000)]), "ragged": rng.random() < 0.7, "rotary":
                rng.choice([0, rotary, rotary]), "layout": layout, "dtype": dtype}
    batch = _log(rng, 1, 64)
    n = 1 if rng.random() < 0.6 else rng.randrange(2, 17)
    length = max(n, min(_log(rng, 1, 32000), 100_000_000 // (batch * kv * dim)))
    return {"kind": kind, "batch": batch, "n": n, "heads": heads, "kv_heads": kv, "dim": dim, "page": page,
            "length": length, "ragged": rng.random() < 0.7, "window": rng.choice([0, 0, _log(rng, 1, 4000)]),
            "dtype": dtype}


# --------------------------------------------------------------------------- #
def _pitch(dim):
    return (dim + 15) // 16 * 16


def _table(rotary, positions, scaling):
    """Cosines and sines ``[positions, rotary / 2, 2]``, computed in 64 bits; a context four times the trained one."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    freq = 10000.0 ** (-i / rotary)
    factor = 1.0
    if scaling == "linear":
        freq = freq / 4.0
    elif scaling == "ntk":
        freq = (10000.0 * 4.0 ** (rotary / (rotary - 2.0))) ** (-i / rotary)
    elif scaling == "yarn":
        # turns within the trained context: above 32 as trained, below 1 stretched, between them a ramp
        edge = [rotary * math.log(positions / 4.0 / (t * 2 * math.pi)) / (2 * math.log(10000.0)) for t in (32.0, 1.0)]
        low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rotary - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / 4.0 * ramp
        factor = 0.1 * math.log(4.0) + 1.0
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq[None]
    return (torch.stack([angle.cos(), angle.sin()], -1) * factor).float().to(DEV)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(gen, batch, most, least, ragged):
    if not ragged:
        return torch.full((batch,), most, dtype=torch.int32, device=DEV)
    u = torch.rand(batch, generator=gen, device=DEV)
    u[0] = 1.0
    low = max(least, most // 16, 1)
    if most <= low:
        return torch.full((batch,), most, dtype=torch.int32, device=DEV)
    return (low * (most / low) ** u).round().int().clamp(max=most)


def _pages(gen, c, tokens):
    """A cache with room for ``tokens`` per sequence, values of about one in all places, pages in no order."""
    per = (tokens + c["page"] - 1) // c["page"]
    total = c["batch"] * per + 3
    shape = (total, 2, c["kv_heads"], c["page"], _pitch(c["dim"]))
    codes = torch.empty(shape, dtype=E4M3, device=DEV)
    for at in range(0, total, 256):
        part = torch.randn((min(256, total - at),) + shape[1:], generator=gen, device=DEV) * 64.0
        part[..., c["dim"]:] = 0.0
        codes[at:at + 256] = part.clamp(-TOP, TOP).to(E4M3)
    scales = torch.exp2(torch.randint(-8, -4, shape[:3], generator=gen, device=DEV).float())
    table = torch.randperm(total, generator=gen, device=DEV)[:c["batch"] * per].view(c["batch"], per).int()
    return codes, scales, table


def prepare(case, seed):
    c, gen = case, _generator(seed)
    dtype = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype)

    s = {"case": c}
    if c["kind"] == "rotary":
        b, n, d = c["batch"], c["seq"], c["dim"]
        s["table"] = _table(c["rotary"], c["table"], c["scaling"])
        if c["by_token"]:
            first = torch.randint(0, c["table"] - n + 1, (b, 1), generator=gen, device=DEV)
            s["positions"] = first + torch.arange(n, device=DEV)
        else:
            s["positions"] = c["start"]
        names = {"qkv": (b, n, c["heads"], 3, d)} if c["packed"] else \
            {"q": (b, n, c["heads"], d), "k": (b, n, c["kv_heads"], d)}
        for name, shape in names.items():
            s[name] = randn(*shape).requires_grad_(c["train"])
            if c["train"]:
                s["d" + name] = randn(*shape)
        return s
    if c["kind"] == "append":
        b, n = c["batch"], c["n"]
        past = _lengths(gen, b, c["past"], 0, c["ragged"])
        s["counts"] = None
        new = torch.full((b,), n, dtype=torch.int32, device=DEV)
        if c["ragged"] and n > 1:
            s["counts"] = new = _lengths(gen, b, n, 1, True)
        s["lengths"] = past + new
        s["pages"], s["scales"], s["block_table"] = _pages(gen, c, c["past"] + n)
        s["q"] = randn(b, n, c["heads"], c["dim"])
        s["k"] = randn(b, n, c["kv_heads"], c["dim"])
        s["v"] = randn(b, n, c["kv_heads"], c["dim"])
        s["table"] = _table(c["rotary"], c["past"] + n, "none") if c["rotary"] else None
        return s
    if c["kind"] == "attend":
        s["lengths"] = _lengths(gen, c["batch"], c["length"], c["n"], c["ragged"])
        s["pages"], s["scales"], s["block_table"] = _pages(gen, c, c["length"])
        s["q"] = randn(c["batch"], c["n"], c["heads"], c["dim"])
        return s
    # logits with a few tokens far ahead, as a model's are
    b, vocab = c["batch"], c["vocab"]
    x = torch.randn(b, vocab, generator=gen, device=DEV) * 2.5
    ahead = torch.randint(0, vocab, (b, 20), generator=gen, device=DEV)
    x.scatter_(1, ahead, torch.rand(b, 20, generator=gen, device=DEV) * 10.0 + 6.0)
    s["logits"] = x.to(dtype)
    s["uniform"] = torch.rand(b, generator=gen, device=DEV)
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = c[name]
    if c["mixed"]:
        def pick(values, dtype):
            at = torch.randint(0, len(values), (b,), generator=gen, device=DEV)
            return torch.tensor(values, dtype=dtype, device=DEV)[at]

        s["temperature"] = pick([0.0, 0.5, 0.7, 1.0, c["temperature"]], torch.float32)
        s["top_k"] = pick([0, 1, 20, c["top_k"]], torch.int32)
        s["top_p"] = pick([1.0, 0.5, c["top_p"]], torch.float32)
        s["min_p"] = pick([0.0, 0.1, c["min_p"]], torch.float32)
    return s


# --------------------------------------------------------------------------- #
def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend,
                "sample": _plain_sample}[s["case"]["kind"]](s)


def _run_own(s):
    from slapo_b200.ops import functional as NF

    c = s["case"]
    if c["kind"] == "rotary":
        pairs = c["layout"] == "pairs"
        if c["packed"]:
            out = NF.rotary_qkvpacked(s["qkv"], s["table"], s["positions"], interleaved=pairs)
            return out, torch.autograd.grad(out, s["qkv"], s["dqkv"])[0]
        out = NF.rotary(s["q"], s["k"], s["table"], s["positions"], interleaved=pairs)
        return (*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))) if c["train"] else out
    if c["kind"] == "append":
        q = NF.paged_append(s["pages"], s["scales"], s["k"], s["v"], s["block_table"], s["lengths"], s["counts"],
                            q=s["q"], rotary_table=s["table"], interleaved=c["layout"] == "pairs")
        return {"pages": s["pages"], "scales": s["scales"], "q": q}
    if c["kind"] == "attend":
        return NF.paged_attention(s["q"], s["pages"], s["scales"], s["block_table"], s["lengths"],
                                  window=c["window"] or None)
    return NF.sample(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _turn(x, cos, sin, rotary, layout):
    """``x [..., D]`` rotated in 32 bits; cos and sin broadcast to ``[..., rotary / 2]``."""
    x = x.float()
    r, rest = x[..., :rotary], x[..., rotary:]
    if layout == "half":
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., ::2], r[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    pos = s["positions"]
    if not torch.is_tensor(pos):
        pos = torch.arange(pos, pos + c["seq"], device=DEV)
    cos, sin = s["table"][pos][..., None, :, 0], s["table"][pos][..., None, :, 1]
    dtype = DTYPES[c["dtype"]]

    def turn(x, sign):
        return _turn(x, cos, sign * sin, c["rotary"], c["layout"]).to(dtype)

    if c["packed"]:
        cos, sin = cos[..., None, :], sin[..., None, :]

        def packed(x, sign):
            return torch.cat([turn(x[..., :2, :], sign), x[..., 2:, :]], 3)

        return packed(s["qkv"], 1.0), packed(s["dqkv"], -1.0)
    if not c["train"]:
        return turn(s["q"], 1.0), turn(s["k"], 1.0)
    return turn(s["q"], 1.0), turn(s["k"], 1.0), turn(s["dq"], -1.0), turn(s["dk"], -1.0)


def _plain_append(s):
    c = s["case"]
    b, n, t, h, d = c["batch"], c["n"], c["page"], c["kv_heads"], c["dim"]
    counts = torch.full((b,), n, device=DEV) if s["counts"] is None else s["counts"].long()
    start = s["lengths"].long() - counts
    pos = start[:, None] + torch.arange(n, device=DEV)              # [B, n]
    q, k, v = s["q"], s["k"].float(), s["v"].float()
    if s["table"] is not None:
        at = pos.clamp(max=s["table"].shape[0] - 1)
        cos, sin = s["table"][at][:, :, None, :, 0], s["table"][at][:, :, None, :, 1]
        q = _turn(q, cos, sin, c["rotary"], c["layout"]).to(q.dtype)
        k = _turn(k, cos, sin, c["rotary"], c["layout"])
    valid = torch.arange(n, device=DEV) < counts[:, None]
    if s["counts"] is not None:
        q = torch.where(valid[:, :, None, None], q, torch.zeros_like(q))
    # the pages that new tokens touch, in the layout of the cache
    m = (n + t - 2) // t + 1
    slots = torch.arange(m * t, device=DEV)
    first = start // t
    token = first[:, None] * t + slots - start[:, None]             # [B, m t]: which of the new ones
    fresh = (token >= 0) & (token < counts[:, None])
    pick = token.clamp(0, n - 1)[:, :, None, None].expand(-1, -1, h, d)
    new = torch.stack([torch.gather(k, 1, pick), torch.gather(v, 1, pick)], 2)      # [B, m t, 2, H, D]
    new = new.view(b, m, t, 2, h, d).permute(0, 1, 3, 4, 2, 5)                      # [B, m, 2, H, T, D]
    fresh = fresh.view(b, m, t)
    old = ((token < 0) & (first[:, None] * t + slots >= 0)).view(b, m, t)
    number = first[:, None] + torch.arange(m, device=DEV)
    touched = fresh.any(2)
    ids = torch.gather(s["block_table"].long(), 1, number.clamp(max=s["block_table"].shape[1] - 1))
    ids, fresh, old, new = ids[touched], fresh[touched], old[touched], new[touched]
    codes, scale = s["pages"][ids].float(), s["scales"][ids]
    mask = fresh[:, None, None, :, None]
    part, exponent = torch.frexp(torch.where(mask, new, torch.zeros_like(new)).abs().amax((3, 4)))
    exponent = torch.where(part <= 0.875, exponent - 9, exponent - 8).clamp(min=LEAST)
    need = torch.exp2(torch.where(part == 0, LEAST, exponent).float())
    has_old = old.any(1)[:, None, None]
    grown = torch.where(has_old, torch.maximum(scale, need), need)
    kept = torch.where(old[:, None, None, :, None], codes * (scale / grown)[..., None, None], codes)
    kept[..., :d] = torch.where(mask, new / grown[..., None, None], kept[..., :d])
    s["pages"][ids] = kept.to(E4M3)
    s["scales"][ids] = grown
    return {"pages": s["pages"], "scales": s["scales"], "q": q}


def _plain_attend(s):
    c = s["case"]
    b, n, h, kv, d = c["batch"], c["n"], c["heads"], c["kv_heads"], c["dim"]
    ids = s["block_table"].long()
    got = s["pages"][ids].float()[..., :d] * s["scales"][ids][..., None, None]       # [B, m, 2, H, T, D]
    k, v = got.permute(2, 0, 3, 1, 4, 5).reshape(2, b, kv, -1, d)
    q = s["q"].float().view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
    key = torch.arange(k.shape[2], device=DEV)
    pos = s["lengths"].long()[:, None] - n + torch.arange(n, device=DEV)             # [B, n]
    seen = key <= pos[..., None]
    if c["window"]:
        seen = seen & (key > pos[..., None] - c["window"])
    x = x.view(b, kv, h // kv, n, -1).masked_fill(~seen[:, None, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    out = torch.matmul(x.view(b, kv, -1, key.numel()), v).view(b, kv, h // kv, n, d)
    out = out / x.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"]
    b, vocab = x.shape

    def each(v):
        return v[:, None].double() if torch.is_tensor(v) else torch.full((b, 1), float(v), dtype=torch.float64,
                                                                         device=DEV)

    # (numbers of the operator's own width: 32 bits)
    temperature, top_p, min_p = (each(s[n]).float().double() for n in ("temperature", "top_p", "min_p"))
    top_k = each(s["top_k"]).long()
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    gap = value.double() - value[:, :1].double()
    greedy = temperature <= 0
    w = torch.exp(gap / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device=DEV)
    kept = torch.where((rank < top_k) | (top_k <= 0), w, 0.0)
    before = kept.cumsum(1) - kept
    mass = kept.sum(1, keepdim=True)
    keep = (kept > 0) & ((before < top_p * mass) | (top_p >= 1.0)) & (w >= min_p)
    keep = torch.where(greedy, rank == 0, keep | (rank == 0))
    ordered = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    total = ordered.cumsum(1)
    return (total <= s["uniform"].double()[:, None] * total[:, -1:]).sum(1)


# --------------------------------------------------------------------------- #
def _spread_sum(most, least, batch, ragged):
    """About what ``_lengths`` adds up to."""
    low = max(least, most // 16, 1)
    if not ragged or most <= low:
        return batch * most
    return most + (batch - 1) * (most - low) / math.log(most / low)


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "sample":
        return {"bytes": c["batch"] * (c["vocab"] * e + 12), "flops": 4 * c["batch"] * c["vocab"]}
    if c["kind"] == "rotary":
        rows = c["batch"] * c["seq"]
        width = (3 * c["heads"] if c["packed"] else c["heads"] + c["kv_heads"]) * c["dim"]
        ways = 4 if c["train"] else 2
        entries = min(rows, c["table"]) if c["by_token"] else c["seq"]
        return {"bytes": ways * rows * width * e + entries * c["rotary"] * 4,
                "flops": ways // 2 * 3 * rows * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if c["kind"] == "append":
        tokens = _spread_sum(c["n"], 1, c["batch"], c["ragged"] and c["n"] > 1)
        width = (2 * c["heads"] + 2 * c["kv_heads"]) * e * c["dim"] + 2 * c["kv_heads"] * c["dim"]
        return {"bytes": tokens * width, "flops": tokens * (c["heads"] + 3 * c["kv_heads"]) * c["dim"] * 3}
    tokens = _spread_sum(c["length"], c["n"], c["batch"], c["ragged"])
    if c["window"]:
        tokens = min(tokens, c["batch"] * (c["window"] + c["n"]))
    return {"bytes": tokens * c["kv_heads"] * 2 * c["dim"] + 2 * c["batch"] * c["n"] * c["heads"] * c["dim"] * e,
            "flops": 4 * tokens * c["n"] * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------- #
def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend,
                "sample": _exact_sample}[case["kind"]](case, s)


def _matrix(table, pos, dim, layout):
    """``[S, D, D]`` would be the rotations; here their entries: for each place of a head its own factor, its
    partner's place and factor."""
    half = table.shape[1]
    i = torch.arange(dim, device=DEV)
    partner, mine = i.clone(), torch.zeros(dim, dtype=torch.long, device=DEV)
    sign = torch.zeros(dim, dtype=torch.float64, device=DEV)
    if layout == "half":
        partner[:half], partner[half:2 * half] = i[half:2 * half], i[:half]
        mine[:half], mine[half:2 * half] = i[:half], i[:half]
        sign[:half], sign[half:2 * half] = -1.0, 1.0
    else:
        partner[:2 * half] = i[:2 * half] ^ 1
        mine[:2 * half] = i[:2 * half] // 2
        sign[:2 * half] = torch.where(i[:2 * half] % 2 == 0, -1.0, 1.0).double()
    rows = table.double()[pos]
    cos = torch.where(sign != 0, rows[..., mine, 0], 1.0)
    sin = rows[..., mine, 1] * sign
    return cos[..., None, :], sin[..., None, :], partner


def _exact_rotary(c, s):
    pos = s["positions"]
    pos = pos if torch.is_tensor(pos) else torch.arange(pos, pos + c["seq"], device=DEV)
    cos, sin, partner = _matrix(s["table"], pos, c["dim"], c["layout"])

    def forward(x):
        x = x.detach().double()
        return x * cos + x[..., partner] * sin

    def backward(g):       # the transposed rotation
        g = g.double()
        return g * cos + (g * sin)[..., partner]

    if c["packed"]:
        def each(x, f):
            return torch.stack([f(x[:, :, :, 0]), f(x[:, :, :, 1]), x[:, :, :, 2].detach().double()], 3)

        return each(s["qkv"], forward), each(s["dqkv"], backward)
    out = [forward(s["q"]), forward(s["k"])]
    return (*out, backward(s["dq"]), backward(s["dk"])) if c["train"] else tuple(out)


def _nearest_e4m3(x):
    # three bits behind the leading one, steps of 2^-9 below 2^-6; ties to even
    ulp = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / ulp) * ulp


def _exact_append(c, s):
    pages, scales = s["pages"].double(), s["scales"].double()
    counts = [c["n"]] * c["batch"] if s["counts"] is None else s["counts"].tolist()
    lengths, table, t, d = s["lengths"].tolist(), s["block_table"].tolist(), c["page"], c["dim"]
    q = torch.zeros_like(s["q"], dtype=torch.float64)
    for b, count in enumerate(counts):
        start = lengths[b] - count
        new = torch.stack([s["k"][b, :count].double(), s["v"][b, :count].double()])     # [2, count, H, D]
        q[b, :count] = s["q"][b, :count].double()
        if s["table"] is not None:
            pos = torch.arange(start, start + count, device=DEV)
            cos, sin, partner = _matrix(s["table"], pos, d, c["layout"])
            for x in (q[b, :count], new[0]):
                x.copy_(x * cos + x[..., partner] * sin)
        for page in range(start // t, (lengths[b] - 1) // t + 1):
            lo, hi = max(start, page * t), min(lengths[b], page * t + t)
            mine = new[:, lo - start:hi - start].transpose(1, 2)                        # [2, H, tokens, D]
            largest = mine.abs().amax((2, 3))
            power = torch.ceil(torch.log2(largest.clamp(min=1e-300) / TOP)).clamp(min=LEAST)
            scale = torch.exp2(power)
            scale = torch.where(largest > TOP * scale, 2 * scale, scale)
            scale = torch.where((largest <= TOP * scale / 2) & (power > LEAST), scale / 2, scale)
            p, held = table[b][page], lo - page * t
            if held:
                scale = torch.maximum(scale, scales[p])
                pages[p, :, :, :held] = _nearest_e4m3(pages[p, :, :, :held] * (scales[p] / scale)[..., None, None])
            pages[p, :, :, held:held + hi - lo, :d] = _nearest_e4m3(mine / scale[..., None, None])
            scales[p] = scale
    return {"pages": pages, "scales": scales, "q": q}


def _exact_attend(c, s):
    b, n, h, kv, d = c["batch"], c["n"], c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros(b, n, h, d, dtype=torch.float64, device=DEV)
    for i, length in enumerate(s["lengths"].tolist()):
        ids = s["block_table"][i, :(length + c["page"] - 1) // c["page"]].long()
        got = s["pages"][ids].double() * s["scales"][ids].double()[..., None, None]
        k, v = got[..., :d].permute(1, 2, 0, 3, 4).reshape(2, kv, -1, d)[:, :, :length]
        for t in range(n):
            last = length - n + t + 1
            first = max(0, last - c["window"]) if c["window"] else 0
            x = torch.einsum("hgd,hkd->hgk", s["q"][i, t].double().view(kv, -1, d), k[:, first:last])
            p = torch.softmax(x / math.sqrt(d), -1)
            out[i, t] = torch.einsum("hgk,hkd->hgd", p, v[:, first:last]).reshape(h, d)
    return out


def _exact_sample(c, s):
    import numpy as np

    x = s["logits"].double().cpu().numpy()
    u = s["uniform"].double().cpu().numpy()

    def each(v):
        return np.broadcast_to(v.double().cpu().numpy() if torch.is_tensor(v) else np.float64(np.float32(v)),
                               (c["batch"],))

    temperature, top_k, top_p, min_p = (each(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    got = np.zeros(c["batch"], dtype=np.int64)
    for i in range(c["batch"]):
        if temperature[i] <= 0:
            got[i] = int(np.argmax(x[i]))
            continue
        order = np.argsort(-x[i], kind="stable")
        w = np.exp((x[i] - x[i].max()) / temperature[i])
        if top_k[i] > 0:
            order = order[:int(top_k[i])]
        row = np.cumsum(w[order])
        if top_p[i] < 1:
            order = order[:int(np.searchsorted(row, top_p[i] * row[-1])) + 1]
        order = order[w[order] >= min_p[i]]
        chosen = np.sort(order)
        row = np.cumsum(w[chosen])
        got[i] = chosen[int(np.searchsorted(row, u[i] * row[-1], side="right"))]
    return torch.from_numpy(got)
