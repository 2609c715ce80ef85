"""The operators of the 4-bit key/value cache as a program that embeds them calls them, as timed cases.

append: one layer's queries, keys and values of a batch come out of their projections; each head is (optionally biased and
        RMS-)normed and rotated to its position, the queries are handed back, the keys and values are stored in 4 bits in the
        pages of their sequences. The rows just stored are then read back as the values they stand for.
attend: queries of a batch over the cached keys and values of their sequences, causal, optionally inside a sliding window.

The cache holds each head's row in blocks of 32 values: a scale d of 8 significant bits, kept as f16, and 32 numbers of four
bits, n - 8 times d each. Byte j of a block holds value j below and value j + 16 above, as a Q4_0 block does.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# query heads, key/value heads, head size and rotation of the model shapes that this repository benchmarks
SHAPES = {
    "qwen3-0.6b": {"heads": 16, "kv_heads": 8, "dim": 128, "layout": "half", "base": 1e6, "norm": True, "scaled": False, "window": 0},
    "llama-3.2-1b": {"heads": 32, "kv_heads": 8, "dim": 64, "layout": "adjacent", "base": 5e5, "norm": False, "scaled": True, "window": 0},
    "bitnet-2b4t": {"heads": 20, "kv_heads": 5, "dim": 128, "layout": "half", "base": 5e5, "norm": False, "scaled": False, "window": 0},
    "mistral-7b": {"heads": 32, "kv_heads": 8, "dim": 128, "layout": "adjacent", "base": 1e6, "norm": False, "scaled": False, "window": 0},
    "gemma3-1b": {"heads": 4, "kv_heads": 1, "dim": 256, "layout": "half", "base": 1e4, "norm": True, "scaled": False, "window": 512},
}
MOST_SCORES = 4096 * 4096 * 32  # of the largest listed case, padded


def _case(op, model, type, sequences, tokens, context, ragged=False, page=64, bias=False, width=0, window=None):
    c = {"op": op, "type": type, "sequences": sequences, "tokens": tokens, "context": context, "ragged": ragged, "page": page,
         "bias": bias, "width": width, **SHAPES[model]}
    if window is not None:
        c["window"] = window
    return c


def listed():
    def named(name, *a, **kw):
        return {"name": name, **_case(*a, **kw)}

    return [
        # One token of one conversation: the smallest calls, between two multiplies of a layer.
        named("append-token", "append", "qwen3-0.6b", "f32", 1, 1, 517),
        named("attend-token", "attend", "qwen3-0.6b", "f32", 1, 1, 517),
        # A server's step: one token of each of 64 conversations of all lengths.
        named("append-step", "append", "mistral-7b", "bf16", 64, 1, 8000, ragged=True),
        named("attend-step", "attend", "mistral-7b", "bf16", 64, 1, 8000, ragged=True),
        # A conversation at the end of a long context, one token.
        named("attend-long", "attend", "mistral-7b", "f16", 1, 1, 32767),
        # The verify step of speculative decoding: the carried token and eight drafted ones.
        named("attend-verify", "attend", "mistral-7b", "f32", 1, 9, 2064),
        # A prompt of one batch, projections with biases.
        named("append-prompt", "append", "qwen3-0.6b", "f32", 1, 512, 0, bias=True),
        named("attend-prompt", "attend", "qwen3-0.6b", "f32", 1, 512, 0),
        # Prompts of many users, ragged, part of each head rotated, small pages.
        named("append-prompts", "append", "bitnet-2b4t", "bf16", 13, 1023, 700, ragged=True, page=16, width=96),
        # A later part of a document, long-context divisors, narrow heads.
        named("attend-chunk", "attend", "llama-3.2-1b", "f16", 3, 777, 3001, ragged=True, page=32),
        # Sliding-window layers with heads of 256 values.
        named("attend-sliding", "attend", "gemma3-1b", "bf16", 2, 600, 1500, ragged=True),
        # A long document as one prompt.
        named("attend-document", "attend", "mistral-7b", "bf16", 1, 4096, 0),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    model = rng.choice(sorted(SHAPES))
    op = rng.choice(["append", "attend", "attend"])
    type = rng.choice(sorted(TYPES))
    kind = rng.choice(["token", "step", "verify", "prompt"])
    sequences = {"token": 1, "verify": 1, "step": _between(rng, 2, 64), "prompt": _between(rng, 1, 13)}[kind]
    tokens = {"token": 1, "step": 1, "verify": _between(rng, 2, 24), "prompt": _between(rng, 25, 4096 if sequences == 1 else 1023)}[kind]
    context = _between(rng, 1, {"token": 32767, "step": 8000, "verify": 8000, "prompt": 4096}[kind]) - 1
    s = SHAPES[model]
    width = rng.choice([0, 0, s["dim"] // 2, s["dim"] * 3 // 4]) if s["layout"] == "half" else 0
    window = s["window"] or rng.choice([0, 0, 0, _between(rng, 16, 2048)])
    rest = {"ragged": rng.random() < 0.7, "page": rng.choice([16, 32, 64, 128]), "bias": rng.random() < 0.3, "width": width, "window": window}
    most = [work(c) for c in listed()]
    case = _case(op, model, type, sequences, tokens, context, **rest)
    while not all(work(case)[x] <= max(w[x] for w in most) for x in ("bytes", "flops")) or sequences * tokens * (context + tokens) * s["heads"] > MOST_SCORES:
        sequences, tokens, context = max(1, sequences * 3 // 4), (tokens * 3 + 3) // 4, context * 3 // 4
        case = _case(op, model, type, sequences, tokens, context, **rest)
    return case


# ---- the batch of a case ----------------------------------------------------------------------------------------------


def _lengths(case):
    """Positions before the batch and tokens of the batch, of each sequence."""
    n = case["sequences"]
    if not case["ragged"]:
        return [case["context"]] * n, [case["tokens"]] * n
    share = [1.0 - (s * 0.6180339887) % 1.0 for s in range(n)]  # the first sequence is the longest
    context = [int(case["context"] * f) for f in share]
    tokens = [case["tokens"] if case["tokens"] == 1 else int(case["tokens"] * f) for f in reversed(share)]
    return context, tokens


def work(case):
    context, tokens = _lengths(case)
    heads, kv, dim, size, rows = case["heads"], case["kv_heads"], case["dim"], SIZES[case["type"]], sum(_lengths(case)[1])
    cached = kv * 2 * (dim // 2 + dim // 32 * 2)  # a position's keys and values
    if case["op"] == "append":
        # q, k, v in; q out; the cache rows; the rows as values
        return {"bytes": rows * (size * dim * (heads + 2 * kv + heads + 2 * kv) + cached), "flops": rows * dim * (6 * (heads + kv) + 4 * 2 * kv)}
    window = case["window"] or 1 << 30
    read = pairs = 0
    for c, t in zip(context, tokens):
        read += min(c + t, t + window - 1) if t else 0
        full = max(0, min(t, c + t - window))  # tokens that see a whole window
        pairs += full * window + (t - full) * c + (t - full) * (t - full + 1) // 2
    return {"bytes": read * cached + 2 * rows * heads * dim * size, "flops": 4 * pairs * heads * dim}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _pack(x):
    """Rows of [..., dim] 64-bit values as [..., dim / 2] bytes and [..., dim / 32] scales."""
    b = x.double().unflatten(-1, (-1, 32))
    high, low = b.amax(-1), b.amin(-1)
    d = torch.where(high >= -low, high, low) / -8.0  # the value of the largest magnitude becomes -8; of two the positive one
    mantissa, exponent = torch.frexp(d)
    d = torch.ldexp(torch.round(mantissa * 256.0), exponent - 8).clamp(-65280.0, 65280.0).half()
    wide = d.double().unsqueeze(-1)
    n = torch.floor(b / torch.where(wide == 0, 1.0, wide) + 8.5).clamp(0, 15)
    n = torch.where(wide == 0, 8.0, n).to(torch.uint8)
    return (n[..., :16] | (n[..., 16:] << 4)).flatten(-2), d


def _unpack(quants, scales, dtype):
    q = quants.unflatten(-1, (-1, 16))
    n = torch.cat((q & 15, q >> 4), -1).to(dtype) - 8.0
    return (n * scales.to(dtype).unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    context, tokens = _lengths(case)
    heads, kv, dim, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    n, rows = case["sequences"], sum(tokens)
    longest = max(c + t for c, t in zip(context, tokens))
    columns = -(-longest // page)
    pages = n * columns + 3

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    # Keys have channels of their own strength, as trained ones do; what no sequence has written yet holds other rows.
    strength = torch.exp(0.5 * normal(kv, 1, dim))
    k_quants = torch.empty((pages, kv, page, dim // 2), dtype=torch.uint8, device="cuda")
    v_quants = torch.empty_like(k_quants)
    k_scales = torch.empty((pages, kv, page, dim // 32), dtype=torch.float16, device="cuda")
    v_scales = torch.empty_like(k_scales)
    step = max(1, (1 << 25) // (kv * page * dim))
    for p in range(0, pages, step):
        part = slice(p, min(pages, p + step))
        count = part.stop - p
        k_quants[part], k_scales[part] = _pack(normal(count, kv, page, dim) * strength)
        v_quants[part], v_scales[part] = _pack(normal(count, kv, page, dim))
    table = torch.randperm(pages, generator=gen, device="cuda")[:n * columns].reshape(n, columns).int()
    start = torch.tensor([0, *torch.tensor(tokens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    # one buffer of q, k and v rows side by side, as a fused projection leaves them
    qkv = (normal(rows, (heads + 2 * kv) * dim) * 1.3).to(dtype)
    s = {"case": case, "context": torch.tensor(context, dtype=torch.int32, device="cuda"), "start": start, "table": table, "rows": rows,
         "longest": longest, "most": max(tokens), "k_quants": k_quants, "k_scales": k_scales, "v_quants": v_quants, "v_scales": v_scales,
         "q": qkv[:, :heads * dim].unflatten(1, (heads, dim)), "k": qkv[:, heads * dim:(heads + kv) * dim].unflatten(1, (kv, dim)),
         "v": qkv[:, (heads + kv) * dim:].unflatten(1, (kv, dim)), "q_norm": None, "k_norm": None, "q_bias": None, "k_bias": None,
         "v_bias": None, "factors": None}
    if case["op"] == "attend":
        s["q"] = s["q"].contiguous()
    if case["norm"]:
        s["q_norm"], s["k_norm"] = 1.0 + 0.2 * normal(dim), 1.0 + 0.2 * normal(dim)
    if case["bias"]:
        s["q_bias"], s["k_bias"], s["v_bias"] = 0.3 * normal(heads * dim), 0.3 * normal(kv * dim), 0.3 * normal(kv * dim)
    if case["scaled"]:  # divisors of the angles: the fast pairs keep theirs, the slow ones turn 8 times slower
        s["factors"] = 1.0 + 7.0 * torch.linspace(0, 1, _width(case) // 2, device="cuda").square()
    if own:
        from brisk_llm_b200 import cache4

        s["cache"] = cache4.PagedCache(k_quants, k_scales, v_quants, v_scales)
        s["batch"] = cache4.Batch(s["context"], rows, page_table=table, query_start=start, max_tokens=s["most"], max_length=longest)
        s["rotary"] = cache4.Rotary(dim, case["base"], layout=case["layout"], width=case["width"], factors=s["factors"], device="cuda")
    return s


def _width(case):
    return case["width"] or case["dim"]


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(state):
    if state["case"]["op"] == "append":
        return _append(state)
    return _attend(state)


def _append(s):
    if own:
        cache, batch = s["cache"], s["batch"]
        q = cache.append(batch, s["q"], s["k"], s["v"], rotary=s["rotary"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6,
                         q_bias=s["q_bias"], k_bias=s["k_bias"], v_bias=s["v_bias"])
        k, v = cache.read(batch, s["q"].dtype)
        return {"q": q, "k": k, "v": v}
    sequence, position = _rows(s)
    page, slot = s["table"][sequence, position // s["case"]["page"]].long(), position % s["case"]["page"]
    q = _rotated(s, s["q"].float(), s["q_bias"], s["q_norm"], position)
    # keys in 64 bits: their values fall next to the borders between two steps of the four bits
    k = _rotated(s, s["k"].double(), s["k_bias"], s["k_norm"], position)
    v = s["v"].double()
    if s["v_bias"] is not None:
        v = v + s["v_bias"].double().view(v.shape[1:])
    s["k_quants"][page, :, slot], s["k_scales"][page, :, slot] = _pack(k)
    s["v_quants"][page, :, slot], s["v_scales"][page, :, slot] = _pack(v)
    stored = [_unpack(s[x + "_quants"][page, :, slot], s[x + "_scales"][page, :, slot], torch.float32).to(s["q"].dtype) for x in ("k", "v")]
    return {"q": q.to(s["q"].dtype), "k": stored[0], "v": stored[1]}


def _rows(s):
    """Sequence and position of every row of the batch."""
    row = torch.arange(s["rows"], device="cuda")
    sequence = torch.bucketize(row, s["start"][1:].long(), right=True)
    return sequence, s["context"][sequence].long() + row - s["start"][sequence].long()


def _rotated(s, x, bias, norm, position):
    """[rows, heads, dim] + bias, each head over its root mean square times `norm`, rotated."""
    case, width = s["case"], _width(s["case"])
    if bias is not None:
        x = x + bias.to(x.dtype).view(x.shape[1:])
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * norm.to(x.dtype)
    pair = torch.arange(width // 2, dtype=torch.float64, device="cuda")
    turn = torch.pow(case["base"], -2.0 * pair / width)  # angles in 64 bits: those of far positions are large
    if s["factors"] is not None:
        turn = turn / s["factors"].double()
    angle = (position.double()[:, None] * turn)[:, None, :]
    c, z = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    if case["layout"] == "half":
        a, b, rest = x[..., :width // 2], x[..., width // 2:width], x[..., width:]
        return torch.cat((a * c - b * z, a * z + b * c, rest), -1)
    a, b, rest = x[..., 0:width:2], x[..., 1:width:2], x[..., width:]
    return torch.cat((torch.stack((a * c - b * z, a * z + b * c), -1).flatten(-2), rest), -1)


def _attend(s):
    case = s["case"]
    if own:
        return s["cache"].attention(s["batch"], s["q"], window=case["window"])
    heads, kv, dim, most = case["heads"], case["kv_heads"], case["dim"], s["most"]
    table, context, start = s["table"].long(), s["context"].long(), s["start"].long()
    # [sequences, kv heads, positions, dim], padded to whole pages of the longest
    k = _unpack(s["k_quants"][table], s["k_scales"][table], torch.float32).transpose(1, 2).flatten(2, 3)
    v = _unpack(s["v_quants"][table], s["v_scales"][table], torch.float32).transpose(1, 2).flatten(2, 3)
    sequence, position = _rows(s)
    at = torch.arange(s["rows"], device="cuda") - start[sequence]
    q = torch.zeros((case["sequences"], most, heads, dim), device="cuda")
    q[sequence, at] = s["q"].float()
    q = q.unflatten(2, (kv, heads // kv)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [sequences, kv heads, group x tokens, dim]
    scores = ((q @ k.transpose(-1, -2)) / math.sqrt(dim)).unflatten(2, (heads // kv, most))
    key = torch.arange(k.shape[2], device="cuda")
    last = context[:, None] + torch.arange(most, device="cuda")  # the position of each token
    hidden = key > last[..., None]
    if case["window"]:
        hidden = hidden | (key <= last[..., None] - case["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (heads // kv, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[sequence, at].to(s["q"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------


def _stood_for(block, scale):
    """What a block of 32 values is stored as: the nearest of sixteen steps, by its borders."""
    d = scale.double()[..., None]
    borders = torch.arange(-7.5, 7.0, 1.0, dtype=torch.float64, device="cuda")  # between the steps -8 .. 7
    sign = torch.where(d < 0, -1.0, 1.0)
    n = (block[..., None] * sign[..., None] >= borders * d.abs()[..., None]).sum(-1) - 8.0
    return torch.where(d == 0, torch.zeros_like(block), n * d)


def _scale_of(block):
    """-1/8 of the value of the largest magnitude, to 8 significant bits, as f16."""
    peak = block.abs().max(-1).values
    top = torch.where((block == peak[..., None]).any(-1), peak, -peak)
    exact = top / -8.0
    unit = torch.exp2(torch.floor(torch.log2(exact.abs().clamp_min(1e-300))) - 7)
    return (torch.round(exact / unit) * unit).clamp(-65280.0, 65280.0).to(torch.float16)


def exact(case, seed):
    s = prepare(case, seed)
    context, tokens = _lengths(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv
    if case["op"] == "append":
        position = torch.cat([torch.arange(c, c + t) for c, t in zip(context, tokens)]).cuda().double()
        width = _width(case)
        i = torch.arange(width // 2, dtype=torch.float64, device="cuda")
        theta = torch.exp(-2.0 * i / width * math.log(case["base"]))
        if s["factors"] is not None:
            theta = theta / s["factors"].double()
        turn = torch.polar(torch.ones_like(theta).expand(len(position), -1), position[:, None] * theta)[:, None]

        def turned(x, bias, norm):
            x = x.double()
            if bias is not None:
                x = x + bias.double().reshape(1, -1, dim)
            if norm is not None:
                x = x * (x.pow(2).sum(-1, keepdim=True) / dim + 1e-6).rsqrt() * norm.double()
            first, second = (slice(0, width // 2), slice(width // 2, width)) if case["layout"] == "half" else (slice(0, width, 2), slice(1, width, 2))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        def stored(x):
            block = x.reshape(*x.shape[:-1], dim // 32, 32)
            return _stood_for(block, _scale_of(block)).reshape(x.shape)

        v = s["v"].double() if s["v_bias"] is None else s["v"].double() + s["v_bias"].double().reshape(1, kv, dim)
        return {"q": turned(s["q"], s["q_bias"], s["q_norm"]), "k": stored(turned(s["k"], s["k_bias"], s["k_norm"])), "v": stored(v)}
    out = torch.zeros((s["rows"], heads, dim), dtype=torch.float64, device="cuda")
    row = 0
    for n, (c, t) in enumerate(zip(context, tokens)):
        if t == 0:
            continue
        pages = s["table"][n, :-(-(c + t) // page)].long()

        def rows_of(name, h):
            q = s[name + "_quants"][pages, h].reshape(-1, dim // 32, 16)[:c + t].int()
            return ((torch.cat((q % 16, q // 16), -1) - 8).double() * s[name + "_scales"][pages, h].reshape(-1, dim // 32, 1)[:c + t].double()).reshape(-1, dim)

        for h in range(kv):
            key, value = rows_of("k", h), rows_of("v", h)
            for begin in range(0, t, 512):
                end = min(t, begin + 512)
                q = s["q"][row + begin:row + end, h * group:(h + 1) * group].double()
                score = torch.einsum("tgd,kd->gtk", q, key) * dim ** -0.5
                seen = c + torch.arange(begin, end, device="cuda")[:, None] - torch.arange(c + t, device="cuda")
                mask = (seen < 0) | (seen >= (case["window"] or 1 << 30))
                score = score.masked_fill(mask, -math.inf).log_softmax(-1).exp()
                out[row + begin:row + end, h * group:(h + 1) * group] = torch.einsum("gtk,kd->tgd", score, value)
        row += t
    return out
