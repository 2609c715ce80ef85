"""The 4-bit key/value cache on the device against its definition in 64 bits (cache4_oracle.py).

Tolerances. Stored bytes and scales, and values read back: none, they are equal (bf16: the stored value rounded once). Queries that
append returns, f32: the mean of squares of up to 256 values, a root, two products and a rotation, 2 half-ulps each and the sum's
8 + 5 steps: 24 * 2^-24 of the row's largest value; other types half a step of theirs more. Attention: see tolerance().
"""
import numpy as np
import pytest

import cache4_oracle as O
import helpers as H  # noqa: F401  (puts the repository on sys.path)

pytestmark = pytest.mark.gpu
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def torch_types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class World:
    """A cache of random pages with a batch over it, on the host and on the device."""

    def __init__(self, seed, kv_heads, dim, context, tokens, page=64, even=False, table=True, pad=0, extra_pages=3, garbage=False, spare_columns=1):
        import torch
        from brisk_llm_b200 import cache4
        self.rng = rng = np.random.default_rng(seed)
        self.kv, self.dim, self.page, self.context, self.tokens = kv_heads, dim, page, context, tokens
        n = len(context)
        longest = max(c + t for c, t in zip(context, tokens))
        self.columns = max(1, -(-longest // page)) + spare_columns
        pages = n * self.columns + extra_pages
        rows = rng.standard_normal((pages, kv_heads, page, dim)) * np.exp(0.5 * rng.standard_normal(dim))
        self.kq, self.ks = O.quantise(rows)
        self.vq, self.vs = O.quantise(rng.standard_normal(rows.shape))
        ids = rng.permutation(pages)[:n * self.columns] if table else np.arange(n * self.columns)
        self.table = ids.reshape(n, self.columns).astype(np.int32)
        if garbage:  # what no sequence has written holds scales that are not numbers
            for planes in (self.ks, self.vs):
                written = np.zeros(planes.shape, bool)
                for s in range(n):
                    for p in range(context[s] + tokens[s]):
                        written[self.table[s, p // page], :, p % page] = True
                planes[~written] = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float16), size=int((~written).sum()))
        self.start = np.concatenate(([0], np.cumsum(tokens))).astype(np.int32)
        self.rows = int(self.start[-1]) + pad
        self.device = torch.device("cuda", 0)
        self.cache = cache4.PagedCache(*(torch.from_numpy(x.copy()).to(self.device) for x in (self.kq, self.ks, self.vq, self.vs)))
        self.batch = cache4.Batch(self.dev(np.asarray(context, np.int32)), self.rows, page_table=self.dev(self.table) if table else None,
                                  query_start=None if even else self.dev(self.start), columns=self.columns, max_tokens=max(tokens), max_length=longest)

    def dev(self, x):
        import torch
        return torch.from_numpy(np.ascontiguousarray(x)).to(self.device)

    def positions(self):
        return np.concatenate([np.arange(c, c + t) for c, t in zip(self.context, self.tokens)] or [np.zeros(0)]).astype(np.int64)

    def sequences(self):
        return np.repeat(np.arange(len(self.tokens)), self.tokens)

    def values(self, s, count):
        p = np.arange(count)
        at = (self.table[s, p // self.page], slice(None), p % self.page)
        return O.values(self.kq[at], self.ks[at]), O.values(self.vq[at], self.vs[at])

    def planes(self):
        c = self.cache
        return [t.cpu().numpy() for t in (c.k_quants, c.k_scales, c.v_quants, c.v_scales)]


def rounded(x, type):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch_types()[type])


def same_scales(a, b):
    return np.array_equal(a.view(np.uint16), b.view(np.uint16))


# ---- append and read ------------------------------------------------------------------------------------------------------

APPENDS = [
    # heads, kv, dim, type, context, tokens, page, layout, width, norm, bias
    (16, 8, 128, "f32", [517], [1], 64, "half", 0, True, False),
    (4, 4, 64, "f16", [0], [1], 16, "adjacent", 0, False, False),
    (4, 1, 256, "bf16", [511, 0, 33], [3, 0, 40], 32, "half", 0, True, True),
    (6, 2, 128, "f32", [0, 15, 16, 9], [17, 1, 33, 0], 16, "half", 96, False, True),
    (5, 5, 64, "bf16", [100, 1], [70, 2], 128, "adjacent", 32, True, False),
    (8, 1, 256, "f32", [30000], [5], 256, "adjacent", 0, True, False),
    (3, 1, 128, "f16", [7] * 33, [1] * 33, 64, "half", 2, False, False),
    (20, 5, 128, "bf16", [3, 0], [600, 41], 64, None, 0, True, False),
    (0, 2, 64, "f32", [5], [9], 16, "half", 64, False, False),
]


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c[:4])))
def test_append_stores_what_the_definition_says(case, fused):
    import torch
    from brisk_llm_b200 import cache4
    heads, kv, dim, type, context, tokens, page, layout, width, norm, bias = case
    w = World(1, kv, dim, context, tokens, page=page, pad=3)
    rng, rows = w.rng, w.rows
    wide = heads + 2 * kv
    # fused: q, k and v in one buffer whose rows have an odd stride, from an odd value on (no vector access fits)
    spare = 1 if fused else 0
    flat = rounded(rng.standard_normal((rows, wide * dim + spare)) * 2, type).to(w.device)
    x = flat[:, spare:]
    q, k, v = (x[:, a * dim:b * dim].unflatten(1, (b - a, dim)) if b > a else None for a, b in ((0, heads), (heads, heads + kv), (heads + kv, wide)))
    if not fused:
        q, k, v = (None if t is None else t.contiguous() for t in (q, k, v))
    qn, kn = (1 + 0.3 * rng.standard_normal(dim), 1 + 0.3 * rng.standard_normal(dim)) if norm else (None, None)
    qb, kb, vb = (rng.standard_normal(heads * dim), rng.standard_normal(kv * dim), rng.standard_normal(kv * dim)) if bias else (None, None, None)
    f32 = [None if t is None else t.astype(np.float32) for t in (qn, kn, qb, kb, vb)]
    factors = np.linspace(1, 9, (width or dim) // 2).astype(np.float32)
    rotary = None if layout is None else cache4.Rotary(dim, 1e6, layout=layout, width=width, scale=0.5, factors=factors, attn_factor=1.25, device="cuda")
    turns = None if layout is None else 0.5 * 1e6 ** (-2.0 * np.arange(len(factors)) / (width or dim)) / factors / (2 * np.pi)
    before = w.planes()
    out = torch.full((rows, heads, dim), 77.0, dtype=k.dtype, device=w.device) if heads else None
    got = w.cache.append(w.batch, q, k, v, rotary=rotary, q_norm=None if not norm else w.dev(f32[0]), k_norm=None if not norm else w.dev(f32[1]), eps=1e-5,
                         q_bias=None if not bias or not heads else w.dev(f32[2]), k_bias=None if not bias else w.dev(f32[3]),
                         v_bias=None if not bias else w.dev(f32[4]), out=out)
    used, position, sequence = int(w.start[-1]), w.positions(), w.sequences()
    eps = float(np.float32(1e-5))
    def host(t):
        return t[:used].float().cpu().numpy().astype(np.float64)
    turn = dict(turns=turns, adjacent=layout == "adjacent", attn_factor=1.25)
    want = [p.copy() for p in before]
    at = (w.table[sequence, position // page], slice(None), position % page)
    want[0][at], want[1][at] = O.quantise(O.rotated(host(k), position, f32[3], f32[1], eps, **turn))
    want[2][at], want[3][at] = O.quantise(host(v) if not bias else host(v) + f32[4].astype(np.float64).reshape(kv, dim))
    after = w.planes()
    for name, a, b in zip(("k", "k scales", "v", "v scales"), after, want):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), name  # every page, those that nothing was appended to among them
    if heads:
        ref = O.rotated(host(q), position, f32[2], f32[0], eps, **turn)
        err = np.abs(host(got) - ref)
        assert (err <= HALF_STEP[type] * np.abs(ref) + 24 * 2.0 ** -24 * np.abs(ref).max(-1, keepdims=True) + 1e-7).all(), err.max()
        assert (got[used:] == 77.0).all()  # rows behind the last sequence stay as they were
    kk, vv = w.cache.read(w.batch, dtype=k.dtype, k_out=torch.full((rows, kv, dim), 5.0, dtype=k.dtype, device=w.device),
                          v_out=torch.full((rows, kv, dim), 5.0, dtype=k.dtype, device=w.device))
    assert torch.equal(kk[:used].cpu(), rounded(O.values(want[0][at], want[1][at]), type))
    assert torch.equal(vv[:used].cpu(), rounded(O.values(want[2][at], want[3][at]), type))
    assert (kk[used:] == 5.0).all() and (vv[used:] == 5.0).all()


def test_values_on_the_borders_and_off_the_scale():
    """Blocks of exact ties, zeros, one value, the smallest and largest numbers, infinities and NaN."""
    import torch
    w = World(2, 1, 64, [0], [12], page=16)
    x = np.zeros((12, 2, 32), np.float32)
    x[0, 0] = np.arange(-16, 16) / 2.0          # d = 1: every second value lies on a border
    x[0, 1] = -x[0, 0]
    x[1, 0, 5] = -3.0
    x[1, 1, 31] = 1e-8                          # d rounds to nothing
    x[2] = 1e-6 * np.arange(-32, 32).reshape(2, 32)   # d below the smallest normal f16
    x[3, 0, 0], x[3, 1, 0] = 1e30, -1e30        # d is held to the largest f16 of 8 bits
    x[4, 0, :3], x[4, 1, 7] = (np.nan, 1.0, -2.0), np.inf
    x[5, 0, 0], x[5, 0, 1], x[5, 1, :] = np.inf, -np.inf, np.nan
    x[6, 0, :2], x[6, 1, :2] = (4.0, -4.0), (-4.0, 4.0)  # two values of the largest magnitude
    x[7:] = w.rng.standard_normal((5, 2, 32)).astype(np.float32)
    x[7, 0] = np.float32(2.0) ** -149
    x[8, 1] *= 1e-38
    x = x.reshape(12, 1, 64)
    w.cache.append(w.batch, None, w.dev(x), w.dev(x))
    q, d = O.quantise(x)
    pages, slots = w.table[0, np.arange(12) // 16], np.arange(12) % 16
    for planes in (w.planes()[:2], w.planes()[2:]):
        assert same_scales(planes[1][pages, :, slots], d)
        assert np.array_equal(planes[0][pages, :, slots], q)
    k, v = w.cache.read(w.batch)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


# ---- attention ------------------------------------------------------------------------------------------------------------


def tolerance(q, k, v, ref, type, scale, n):
    """A score's products carry 2^-22 (an f32 query as two f16 parts) and its sum dim * 2^-24 at most; exp passes a score's error on as a
    relative one of the weight, in numerator and denominator; weights are two f16 parts for f32 and one, 2^-12, otherwise; the sums over n
    positions carry at most n * 2^-24, far less as they are split; the result is rounded once."""
    size = scale * (np.abs(q).sum(-1).max() * np.abs(k).max())
    score = size * (2.0 ** -22 + q.shape[-1] * 2.0 ** -24)
    weight = 2.0 ** -22 if type == "f32" else 2.0 ** -12
    return np.abs(v).max() * (2 * score + 2 * weight + (16 + n / 8) * 2.0 ** -24) + HALF_STEP[type] * np.abs(ref) + 1e-7


def check_attention(w, heads, type, window=0, scale=0.0, odd=False, stretch=1.0):
    import torch
    rng = w.rng
    width = heads * w.dim + (1 if odd else 0)
    q = rounded(rng.standard_normal((w.rows, width)) * stretch, type).to(w.device)[:, width - heads * w.dim:].unflatten(1, (heads, w.dim))
    out = torch.full((w.rows, heads * w.dim + (3 if odd else 0)), 9.0, dtype=q.dtype, device=w.device)[:, :heads * w.dim].unflatten(1, (heads, w.dim))
    before = w.planes()
    got = w.cache.attention(w.batch, q, scale=scale, window=window, out=out)
    for a, b in zip(before, w.planes()):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    used = int(w.start[-1])
    assert (got[used:] == 9.0).all()
    real = scale or w.dim ** -0.5
    for s, (c, t) in enumerate(zip(w.context, w.tokens)):
        if t == 0:
            continue
        rows = slice(int(w.start[s]), int(w.start[s]) + t)
        k, v = w.values(s, c + t)
        qs = q[rows].float().cpu().numpy().astype(np.float64)
        ref = O.attention(qs, k, v, c, real, window)
        err = np.abs(got[rows].float().cpu().numpy() - ref)
        assert np.isfinite(err).all()
        assert (err <= tolerance(qs, k, v, ref, type, real, c + t)).all(), (s, err.max())
        rel = np.linalg.norm(err) / np.linalg.norm(ref)
        assert rel <= {"f32": 1e-5, "f16": 1e-3, "bf16": 5e-3}[type], (s, rel)  # errors of both signs average: far inside the bound of each value
    return got


ATTENDS = [
    # heads, kv, dim, context, tokens, page, window
    (16, 8, 128, [517], [1], 64, 0),
    (8, 1, 128, [0], [1], 16, 0),
    (4, 4, 64, [0, 1, 62, 63, 64, 127, 1000], [1] * 7, 64, 0),
    (32, 8, 64, [15, 0, 300], [5, 0, 9], 32, 0),
    (20, 5, 128, [2047, 3], [9, 24], 64, 0),
    (12, 4, 128, [77], [130], 16, 0),
    (4, 1, 256, [511, 600, 0], [1, 3, 70], 32, 512),
    (10, 2, 256, [33], [40], 128, 0),
    (7, 1, 64, [100], [300], 64, 17),
    (16, 1, 64, [40, 9], [2, 33], 64, 1),
    (48, 2, 128, [129], [11], 256, 0),
    (16, 8, 128, [0], [512], 64, 0),
    (8, 2, 128, [1500, 0, 700], [333, 257, 1], 64, 400),
    (32, 4, 64, [255], [520], 128, 0),
    (4, 4, 128, [9000], [1], 64, 0),
    # rows enough for the kernel of many, and for two tiles of them to a CTA
    (21, 3, 64, [100], [300], 16, 0),
    (32, 8, 128, [0, 100, 5], [256, 200, 301], 32, 0),
    (56, 8, 64, [31, 0], [290, 150], 64, 70),
    # positions enough for two or four CTAs to share them; of a short sequence some of these have none
    (8, 2, 128, [2500], [300], 64, 0),
    (7, 1, 64, [3100], [260], 32, 0),
    (16, 2, 128, [1999], [280], 64, 1200),
    (16, 2, 128, [3000, 0, 0], [150, 1, 20], 16, 0),
    (48, 3, 64, [2600, 0, 700], [70, 0, 33], 128, 0),
]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3][0]}-{c[4][0]}-w{c[6]}")
def test_attention_is_the_definition_s(case, type):
    heads, kv, dim, context, tokens, page, window = case
    w = World(3, kv, dim, context, tokens, page=page, pad=2, garbage=True)
    check_attention(w, heads, type, window=window, odd=type == "f16")


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [1, 40, 300, 700])
def test_attention_of_large_scores(type, tokens):
    """Scores of some hundreds: one position has all the weight, and the running maximum moves often."""
    w = World(4, 2, 128, [500], [tokens])
    check_attention(w, 8, type, scale=1.0, stretch=3.0)


def test_even_batches_without_a_table():
    w = World(5, 2, 128, [70, 0, 130], [4, 4, 4], even=True, table=False, extra_pages=0)
    check_attention(w, 8, "f32")


@pytest.mark.parametrize("tokens", [1, 200, 1300])
def test_a_sequence_that_sees_nothing_and_pages_outside_the_pool(tokens):
    import torch
    w = World(6, 2, 64, [100, 40], [tokens, tokens])
    w.table[0, 1] = -1          # positions 64 .. 127 of the first sequence: rows of zeros
    w.table[1, 0] = 10 ** 6
    w.batch.page_table.copy_(w.dev(w.table))
    for s, page in ((0, 1), (1, 0)):
        w.table[s, page] = len(w.kq)  # the oracle's page of zeros
    for name in ("kq", "ks", "vq", "vs"):
        old = getattr(w, name)
        setattr(w, name, np.concatenate((old, np.full_like(old[:1], 0x88 if old.dtype == np.uint8 else 0))))
    planes = w.planes()
    q = torch.randn((w.rows, 4, 64), device=w.device)
    got = w.cache.attention(w.batch, q).cpu().numpy()
    for s in range(2):
        rows = slice(s * tokens, (s + 1) * tokens)
        k, v = w.values(s, w.context[s] + tokens)
        qs = q[rows].cpu().numpy().astype(np.float64)
        ref = O.attention(qs, k, v, w.context[s], 64 ** -0.5)
        assert (np.abs(got[rows] - ref) <= tolerance(qs, k, v, ref, "f32", 0.125, len(k))).all()
    # appending writes nothing for them, reading gives zeros
    x = torch.randn((w.rows, 2, 64), device=w.device)
    w.cache.append(w.batch, None, x, x)
    k, _ = w.cache.read(w.batch)
    after = w.planes()
    position, sequence = w.positions(), w.sequences()
    bad = w.table[sequence, position // 64] == len(planes[0])
    assert (k.cpu().numpy()[bad] == 0).all()
    good = ~bad
    at = (w.table[sequence[good], position[good] // 64], slice(None), position[good] % 64)
    want = planes[0].copy()
    want[at] = O.quantise(x.cpu().numpy()[good])[0]
    assert np.array_equal(after[0], want)
    # nothing before the batch and no positions held: a context below zero, as a host may leave it for an idle slot
    w.batch.context.copy_(w.dev(np.array([-tokens, 40], np.int32)))
    got = w.cache.attention(w.batch, q)
    assert (got[:tokens] == 0).all() and torch.isfinite(got).all()


@pytest.mark.parametrize("heads", [2, 128])
def test_positions_past_the_columns_are_not_seen(heads):
    import torch
    w = World(7, 1, 128, [60], [40], spare_columns=0)  # two columns hold 128 positions
    w.batch.context.copy_(w.dev(np.array([100], np.int32)))  # ... and 12 of the 40 tokens stand past them
    q = torch.randn((40, heads, 128), device=w.device)
    planes = w.planes()
    got = w.cache.attention(w.batch, q).cpu().numpy()
    k, v = w.values(0, 128)
    qs = q.cpu().numpy().astype(np.float64)
    ref = O.attention(qs, k, v, 100, 128 ** -0.5)
    assert (np.abs(got - ref) <= tolerance(qs, k, v, ref, "f32", 128 ** -0.5, 128)).all()
    w.cache.append(w.batch, None, q[:, :1].contiguous(), q[:, :1].contiguous())
    after = w.planes()
    touched = np.zeros(after[0].shape[:1] + after[0].shape[2:3], bool)
    for p in range(100, 128):
        touched[w.table[0, p // 64], p % 64] = True
    assert np.array_equal(after[0].transpose(0, 2, 1, 3)[~touched], planes[0].transpose(0, 2, 1, 3)[~touched])


@pytest.mark.parametrize("tokens", [1, 3, 150, 400])
def test_bounds_that_are_not_given_change_nothing(tokens):
    import torch
    from brisk_llm_b200 import cache4
    w = World(8, 2, 128, [900, 10], [tokens, tokens])
    q = torch.randn((w.rows, 8, 128), device=w.device, dtype=torch.bfloat16)
    loose = cache4.Batch(w.batch.context, w.rows, page_table=w.batch.page_table, query_start=w.batch.query_start)
    a, b = w.cache.attention(w.batch, q).float(), w.cache.attention(loose, q).float()
    assert ((a - b).abs() <= 2.0 ** -7 * a.abs() + 2.0 ** -10 * 8).all()


# ---- together, as they are used -----------------------------------------------------------------------------------------------


def test_a_prompt_at_once_and_token_by_token():
    """A prompt appended whole, and the same token by token with the attention of each: the caches are equal byte for byte, the results
    as near as two orders of the same sums are."""
    import torch
    from brisk_llm_b200 import cache4
    n, heads, kv, dim = 77, 8, 2, 128
    gen = torch.Generator("cuda").manual_seed(9)
    q, k, v = (torch.randn((n, h, dim), generator=gen, device="cuda") for h in (heads, kv, kv))
    rotary = cache4.Rotary(dim, 1e6)
    norm = torch.rand(dim, generator=gen, device="cuda") + 0.5
    caches = [cache4.PagedCache.allocate(8, kv, dim, page_size=16) for _ in range(2)]
    whole = cache4.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), n, columns=8, max_length=n)
    a = caches[0].attention(whole, caches[0].append(whole, q, k, v, rotary=rotary, q_norm=norm, k_norm=norm))
    context = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = cache4.Batch(context, 1, columns=8)
    b = []
    for i in range(n):
        context.fill_(i)
        b.append(caches[1].attention(one, caches[1].append(one, q[i:i + 1], k[i:i + 1], v[i:i + 1], rotary=rotary, q_norm=norm, k_norm=norm)))
    for x in ("k_quants", "k_scales", "v_quants", "v_scales"):
        assert torch.equal(getattr(caches[0], x), getattr(caches[1], x))
    assert (a - torch.cat(b)).abs().max() <= 2e-5 * a.abs().max()


@pytest.mark.parametrize("tokens", [1, 140, 320])
def test_captured_and_replayed_on_two_streams(tokens):
    """A captured append and attention, replayed for other positions and pages; two graphs at a time on two streams."""
    import torch
    from brisk_llm_b200 import cache4
    worlds = [World(10 + i, 2, 128, [300, 40], [tokens, tokens]) for i in range(2)]
    rotary = cache4.Rotary(128, 1e4, layout="adjacent")
    runs = []
    for w in worlds:
        x = [torch.randn((w.rows, h, 128), device="cuda", dtype=torch.float16) for h in (8, 2, 2)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            w.cache.attention(w.batch, w.cache.append(w.batch, *x, rotary=rotary))
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                out = w.cache.attention(w.batch, w.cache.append(w.batch, *x, rotary=rotary))
        runs.append((w, x, stream, graph, out))
    torch.cuda.synchronize()
    for shift in (0, 1, 60):
        for w, x, stream, graph, out in runs:
            w.batch.context.copy_(w.dev(np.array([300 - shift, 40 - shift // 2], np.int32)))
            w.batch.page_table.copy_(w.dev(np.roll(w.table, shift, axis=0)))
        torch.cuda.synchronize()
        for _ in range(3):
            for w, x, stream, graph, out in runs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for w, x, stream, graph, out in runs:
            want = w.cache.attention(w.batch, w.cache.append(w.batch, *x, rotary=rotary))
            assert torch.equal(want, out)  # the same call on the same data: bit for bit


def test_calls_of_several_threads_at_once():
    """Each thread with a stream and a batch of its own, over one cache that they read and pages of their own that they append to."""
    import threading

    import torch
    from brisk_llm_b200 import cache4
    worlds = [World(20 + i, 2, 128, [400 + 10 * i, 30], [t, t]) for i, t in enumerate((1, 9, 340, 1))]
    rotary = cache4.Rotary(128, 1e6)
    inputs = [[torch.randn((w.rows, h, 128), device="cuda") for h in (8, 2, 2)] for w in worlds]
    want = [w.cache.attention(w.batch, w.cache.append(w.batch, *x, rotary=rotary)) for w, x in zip(worlds, inputs)]
    torch.cuda.synchronize()
    got = [None] * len(worlds)

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = worlds[i].cache.attention(worlds[i].batch, worlds[i].cache.append(worlds[i].batch, *inputs[i], rotary=rotary))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(worlds))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_results_do_not_depend_on_the_run():
    import torch
    for tokens in (1, 9, 300):
        w = World(12, 2, 128, [2000, 130], [tokens, tokens])
        q = torch.randn((w.rows, 16, 128), device="cuda")
        first = w.cache.attention(w.batch, q)
        for _ in range(4):
            assert torch.equal(first, w.cache.attention(w.batch, q))


def test_a_cache_past_two_to_the_31_bytes_and_values():
    """The last pages of a pool of 3.2 GB a plane: offsets past 32 bits."""
    import torch
    from brisk_llm_b200 import cache4
    pages, kv, dim, page = 25000, 8, 256, 128
    cache = cache4.PagedCache.allocate(pages, kv, dim, page_size=page)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    x = torch.randn((300, kv, dim), device="cuda", dtype=torch.bfloat16)
    batch = cache4.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), 300, page_table=table)
    cache.append(batch, None, x, x)
    k, v = cache.read(batch)
    kq, ks = O.quantise(x.float().cpu().numpy())
    assert np.array_equal(k.cpu().numpy(), O.values(kq, ks).astype(np.float32)) and torch.equal(k, v)
    for tokens in (1, 200):
        q = torch.randn((tokens, kv, dim), device="cuda")
        last = cache4.Batch(torch.full((1,), 300 - tokens, dtype=torch.int32, device="cuda"), tokens, page_table=table)
        got = cache.attention(last, q).cpu().numpy()
        kk = k.cpu().numpy().astype(np.float64)
        qs = q.cpu().numpy().astype(np.float64)
        ref = O.attention(qs, kk, kk, 300 - tokens, dim ** -0.5)
        assert (np.abs(got - ref) <= tolerance(qs, kk, kk, ref, "f32", dim ** -0.5, 300)).all()


def test_the_wrapper_refuses_what_does_not_fit():
    import torch
    from brisk_llm_b200 import cache4
    cache = cache4.PagedCache.allocate(4, 2, 64)
    batch = cache4.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), 3, columns=2)
    x = torch.zeros((3, 2, 64), device="cuda")
    for call in (
        lambda: cache.append(batch, x, x, x[:2]), lambda: cache.append(batch, x, x.half(), x), lambda: cache.append(batch, x.cpu(), x, x),
        lambda: cache.append(batch, x, x[..., :32], x), lambda: cache.append(batch, x, x, x, q_norm=torch.ones(63, device="cuda")),
        lambda: cache.attention(batch, x.double()), lambda: cache.attention(batch, x, out=x), lambda: cache.attention(batch, x, window=-1),
        lambda: cache.attention(batch, x.transpose(1, 2)), lambda: cache.attention(batch, torch.zeros((3, 3, 64), device="cuda")),
        lambda: cache.read(batch, torch.int8), lambda: cache.read(batch, torch.float32, k_out=x.half()),
        lambda: cache4.Batch(torch.zeros(1, dtype=torch.int64, device="cuda"), 1), lambda: cache4.Batch(torch.zeros(1, dtype=torch.int32), 1),
        lambda: cache4.Rotary(64, 1e4, layout="both"), lambda: cache4.Rotary(64, 1e4, width=66), lambda: cache4.Rotary(64, 1e4, factors=[1.0]),
        lambda: cache4.PagedCache(cache.k_quants, cache.k_scales, cache.v_quants, cache.v_scales.float()),
        lambda: cache4.PagedCache.allocate(4, 2, 64, page_size=24).attention(batch, x),
    ):
        with pytest.raises(RuntimeError, match="^cuda: "):
            call()
    assert cache.attention(cache4.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), 0, columns=2), x[:0]).shape == (0, 2, 64)
