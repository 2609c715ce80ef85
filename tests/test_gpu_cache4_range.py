"""The 4-bit cache's operators at the ends of their range: weights far below a row's largest, keys, values and queries past what an f16 holds,
rows whose squares leave 32 bits. Against the definition, both kernels of the attention: few rows and many."""
import numpy as np
import pytest

import cache4_oracle as O
import helpers as H  # noqa: F401  (puts the repository on sys.path)
from test_gpu_cache4 import HALF_STEP, World, rounded, same_scales

pytestmark = pytest.mark.gpu


def torch_type(name):
    from test_gpu_cache4 import torch_types
    return torch_types()[name]


@pytest.mark.parametrize("type,dim,sequences,tokens,context,nats", [
    ("f32", 128, 8, 300, 2000, 10.0), ("f32", 128, 8, 300, 2000, 12.5), ("f32", 64, 8, 300, 2000, 12.5), ("f32", 128, 8, 300, 2000, 17.05),
    ("f16", 128, 8, 300, 60000, 17.05), ("f16", 64, 8, 300, 60000, 17.05), ("bf16", 128, 8, 300, 2000, 17.05),
    ("f32", 64, 128, 1, 16000, 10.0), ("f32", 128, 128, 1, 16000, 12.5), ("f32", 256, 128, 1, 16000, 12.5), ("f16", 128, 128, 1, 16000, 17.05)])
def test_heavy_positions_and_a_long_even_tail(type, dim, sequences, tokens, context, nats):
    """Heavy positions (values -1) are `nats` above all others (values 1), whose weights are equal, so that whatever each of them loses
    all lose, and nothing averages out. Sequences enough that no cluster shares a row's positions; with few rows a heavy position for each
    of the warps that do.

    The result is (tail - heavy) / (tail + heavy) of the weights' sums. By arithmetic: a heavy weight is off by its score's roundings (an f32
    query's parts 2^-22, the sum, the factor and the difference 2^-24 each, of `nats`) and exp2's 2^-21, which moves the result by twice
    its share times the tail's; a tail's weight by 2^-22 or 2^-11 of itself, or 2^-37 or 2^-32 of a heavy one; a running sum by 2^-24 with
    each of its steps: 11 or 19 for a tile of 64 or 128 positions of the many-rows kernel and one for every 16 positions of the product,
    6 for 32 positions of a warp of the other (eight warps, heads of 256 four)."""
    import torch
    from brisk_llm_b200 import cache4
    heads, page, many = 8, 64, tokens > 1
    heavy = 1 if many else 8
    columns = -(-(context + tokens) // page)
    cache = cache4.PagedCache.allocate(columns, 1, dim, page_size=page)
    cache.k_quants.fill_(0x88)  # zeros
    cache.v_scales.fill_(-0.125)  # (0 - 8) * -1/8
    for p in range(0, 32 * heavy, 32):
        cache.k_scales[p // page, 0, p % page, 0] = -1.0
        cache.k_quants[p // page, 0, p % page, 0] = 0x80  # 8 in dim 0
        cache.v_scales[p // page, 0, p % page] = 0.125
    table = torch.arange(columns, dtype=torch.int32, device="cuda").expand(sequences, columns).contiguous()
    batch = cache4.Batch(torch.full((sequences,), context, dtype=torch.int32, device="cuda"), sequences * tokens, page_table=table,
                         max_tokens=tokens, max_length=context + tokens)
    q = torch.zeros((sequences * tokens, heads, dim))
    q[:, :, 0] = rounded([nats * dim ** 0.5 / 8.0], type)
    got = cache.attention(batch, q.to(torch_type(type)).cuda()).double().cpu().numpy()
    score = float(q[0, 0, 0]) * 8.0 / dim ** 0.5
    others = np.tile(context + np.arange(tokens) + 1 - heavy, sequences)[:, None, None]
    tail = others * np.exp(-score)
    want = (tail - heavy) / (tail + heavy)
    share = heavy / (tail + heavy)
    small, floor = (2.0 ** -22, 2.0 ** -37) if type == "f32" else (2.0 ** -11, 2.0 ** -32)
    n = context + tokens
    steps = (n / 64 * 11 + n / 256 + 32 if type == "f32" else n / 128 * 19 + n / 16) if many else n / (32 * (4 if dim == 256 else 8)) * 6 + 32
    bound = 2 * share * (1 - share) * (score * (2.0 ** -22 + 3 * 2.0 ** -24) + 2.0 ** -21) + 2 * (1 - share) * share * small + 2 * others / heavy * floor
    bound = bound + steps * 2.0 ** -24 + HALF_STEP[type] * np.abs(want)
    err = np.abs(got - want)
    assert (err <= bound).all(), (err.max(), bound.min())


def bound(q, k, v, ref, type, scale, context):
    """As test_gpu_cache4's tolerance(), but of each row by what that row sees - its own largest score and value - so that a position behind
    it widens nothing. Scores: the products' magnitudes carry 2^-22 and their sum dim * 2^-24; a part of an f32 query is at least
    2^-35 of the row's largest wide. A weight has 2^-22 (f32) or 2^-12 of itself, and is not known below 2^-37 (2^-32) of the largest."""
    n, dim, group = k.shape[0], k.shape[2], q.shape[1] // k.shape[1]
    out = np.empty_like(ref)
    small, floor = (2.0 ** -22, 2.0 ** -37) if type == "f32" else (2.0 ** -12, 2.0 ** -32)
    for h in range(q.shape[1]):
        kh, vh = np.abs(k[:, h // group]), np.abs(v[:, h // group]).max(1)
        size = np.abs(q[:, h]) @ kh.T * (2.0 ** -22 + dim * 2.0 ** -24) + np.abs(q[:, h]).max(1)[:, None] * 2.0 ** -35 * kh.sum(1)
        for r in range(len(q)):
            sees = context + r + 1
            out[r, h] = vh[:sees].max() * (2 * scale * size[r, :sees].max() + 2 * small + (16 + n / 8) * 2.0 ** -24 + sees * floor)
    return out + HALF_STEP[type] * np.abs(ref) + 1e-7


def compare(got, q, k, v, type, context):
    scale = q.shape[2] ** -0.5
    ref = O.attention(q, k, v, context, scale)
    err = np.abs(got - ref)
    assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:4]
    assert (err <= bound(q, k, v, ref, type, scale, context)).all(), err.max()
    return err, ref


LARGE = {"f32": [1e5, np.inf, -65504.0, 3e38, -np.inf], "bf16": [1e5, np.inf, -65504.0, 3e38, -np.inf], "f16": [65504.0, np.inf, -65504.0, 65408.0, -np.inf]}


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (128, 3), (256, 3), (64, 200), (128, 200), (256, 60), (128, 420)])
def test_values_past_an_f16(dim, tokens, type):
    """Values of up to 522 240 and infinities, appended among others: rows before them are as if they were not there, rows behind them are
    what the stored values give."""
    heads, kv, context = 8 if tokens < 100 else 32, 2, 400
    n = context + tokens
    w = World(31, kv, dim, [0], [n])
    k, v = (w.rng.standard_normal((n, kv, dim)) for _ in range(2))
    for i, x in enumerate(LARGE[type]):
        v[n - tokens // 2 - 1 - 37 * (i % 2), i % kv, (11 * i) % dim] = x
    v[130, 0, 3] = 1e-5  # a small one in a block of its own
    v[130, 0, 4:32], v[130, 0, :3] = 0.0, 0.0
    k, v = (rounded(x, type).to(w.device) for x in (k, v))
    w.cache.append(w.batch, None, k, v)
    kk, vv = (O.values(*O.quantise(x.float().cpu().numpy())) for x in (k, v))
    from brisk_llm_b200 import cache4
    batch = cache4.Batch(w.dev(np.array([context], np.int32)), tokens, page_table=w.batch.page_table, max_length=n)
    q = rounded(w.rng.standard_normal((tokens, heads, dim)), type).to(w.device)
    got = w.cache.attention(batch, q, out=q.new_empty(q.shape)).double().cpu().numpy()
    ref = O.attention(q.double().cpu().numpy(), kk, vv, context, dim ** -0.5)
    tops = {"f16": 65504.0}.get(type, np.inf)  # what an f16 result cannot hold is not asked for
    here = np.abs(ref) < tops * 0.99
    err = np.abs(got - ref)
    assert here.mean() > 0.5 and np.isfinite(got[here]).all(), np.argwhere(~np.isfinite(got) & here)[:4]
    assert (err <= bound(q.double().cpu().numpy(), kk, vv, ref, type, dim ** -0.5, context))[here].all()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (128, 3), (256, 3), (64, 200), (128, 200), (256, 60), (128, 420)])
def test_keys_past_an_f16(dim, tokens, type):
    """Keys of up to 522 240 and infinities in dims that the queries have next to nothing in: their scores are of ordinary size."""
    heads, kv, context = 8 if tokens < 100 else 32, 2, 400
    n = context + tokens
    w = World(32, kv, dim, [0], [n])
    k, v = (w.rng.standard_normal((n, kv, dim)) for _ in range(2))
    q = w.rng.standard_normal((tokens, heads, dim))
    q[:, :, :32] *= 2e-5
    for i, x in enumerate(LARGE[type]):
        k[n - tokens // 2 - 1 - 37 * (i % 2), i % kv, 3 + 5 * i] = x
    k, v, q = (rounded(x, type).to(w.device) for x in (k, v, q))
    w.cache.append(w.batch, None, k, v)
    kk, vv = (O.values(*O.quantise(x.float().cpu().numpy())) for x in (k, v))
    from brisk_llm_b200 import cache4
    batch = cache4.Batch(w.dev(np.array([context], np.int32)), tokens, page_table=w.batch.page_table, max_length=n)
    got = w.cache.attention(batch, q).double().cpu().numpy()
    compare(got, q.double().cpu().numpy(), kk, vv, type, context)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (128, 3), (256, 3), (128, 200), (64, 200)])
def test_queries_near_the_end_of_32_bits(dim, tokens, type):
    """Scores of 10^35: one position of every row has all the weight."""
    heads, kv, context = 4 if tokens < 100 else 32, 2, 300
    n = context + tokens
    w = World(33, kv, dim, [context], [tokens])
    q = rounded(w.rng.standard_normal((tokens, heads, dim)) * 1e35, type).to(w.device)
    got = w.cache.attention(w.batch, q).double().cpu().numpy()
    k, v = w.values(0, n)
    qs = q.double().cpu().numpy()
    ref = O.attention(qs, k, v, context, dim ** -0.5)
    for h in range(heads):  # no two scores of a row are within the rounding of one
        s = np.sort(np.where(np.arange(n) <= context + np.arange(tokens)[:, None], qs[:, h] @ k[:, h * kv // heads].T, -np.inf), axis=1)
        sure = s[:, -1] - s[:, -2] > dim * 2.0 ** -20 * np.abs(s).max(initial=0, where=np.isfinite(s))
        assert sure.mean() > 0.9
        assert (np.abs(got[:, h] - ref[:, h])[sure] <= HALF_STEP[type] * np.abs(ref[:, h])[sure] + 2.0 ** -11 * np.abs(v).max()).all()


@pytest.mark.parametrize("type,size", [("f32", 1e25), ("f32", 3e37), ("bf16", 1e30), ("f32", 1e-25), ("bf16", 1e-30), ("f16", 6e-8)])
@pytest.mark.parametrize("dim,layout", [(64, "half"), (128, "adjacent"), (256, None)])
def test_norms_of_rows_whose_squares_leave_32_bits(dim, layout, type, size):
    import torch
    from brisk_llm_b200 import cache4
    w = World(34, 2, dim, [7], [9])
    rng = w.rng
    q, k, v = (rounded(rng.standard_normal((w.rows, h, dim)) * size, type).to(w.device) for h in (4, 2, 2))
    q[3], k[3] = q[3] / size if size < 1e4 else q[3] * 0, k[3] * 0  # among rows of ordinary size and of zeros
    qn, kn = (1 + 0.3 * rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    rotary = None if layout is None else cache4.Rotary(dim, 1e4, layout=layout)
    turns = None if layout is None else 1e4 ** (-2.0 * np.arange(dim // 2) / dim) / (2 * np.pi)
    got = w.cache.append(w.batch, q, k, v, rotary=rotary, q_norm=w.dev(qn), k_norm=w.dev(kn), eps=0.0)
    position, at = w.positions(), None
    with np.errstate(divide="ignore", invalid="ignore"):
        wanted = [O.rotated(x.double().cpu().numpy(), position, norm=n, turns=turns, adjacent=layout == "adjacent") for x, n in ((q, qn), (k, kn))]
    at = (w.table[0, position // w.page], slice(None), position % w.page)
    kq, ks = O.quantise(wanted[1])
    planes = w.planes()
    assert same_scales(planes[1][at], ks) and np.array_equal(planes[0][at], kq)
    here = ~np.isnan(wanted[0])
    err = np.abs(got.double().cpu().numpy() - wanted[0])
    top = np.abs(np.where(here, wanted[0], 0)).max(-1, keepdims=True)
    assert (err <= HALF_STEP[type] * np.abs(wanted[0]) + 24 * 2.0 ** -24 * top + 1e-7)[here].all() and here.mean() > 0.8
    assert not torch.isinf(got.float()).any()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,scale", [(0, 0.0), (90, 0.0), (0, -0.05)])
def test_large_values_and_keys_where_no_cluster_shares_a_row(window, scale, dim, type):
    """CTAs enough for all SMs: each computes its rows alone, those that met a large scale twice. Two ragged sequences, one without any large
    one; a window that leaves them behind; a scale below zero."""
    from brisk_llm_b200 import cache4
    heads, kv, context, tokens = 32, 8, [100, 31], [300, 120]
    w = World(35, kv, dim, [0, 0], [c + t for c, t in zip(context, tokens)])
    k, v = (w.rng.standard_normal((w.rows, kv, dim)) for _ in range(2))
    q = w.rng.standard_normal((sum(tokens), heads, dim))
    q[:, :, :32] *= 2e-5
    for i, x in enumerate(LARGE[type]):
        v[150 + i, 3, 7 * i] = x
        k[170 + 11 * i, i + 1, 5 * i] = x
    k, v, q = (rounded(x, type).to(w.device) for x in (k, v, q))
    w.cache.append(w.batch, None, k, v)
    batch = cache4.Batch(w.dev(np.array(context, np.int32)), sum(tokens), page_table=w.batch.page_table,
                         query_start=w.dev(np.array([0, tokens[0], sum(tokens)], np.int32)), max_tokens=max(tokens), max_length=400)
    got = w.cache.attention(batch, q, scale=scale, window=window).double().cpu().numpy()
    kk, vv = (O.values(*O.quantise(x.float().cpu().numpy())) for x in (k, v))
    qs, real = q.double().cpu().numpy(), scale or dim ** -0.5
    for s in range(2):
        rows, at = slice(sum(tokens[:s]), sum(tokens[:s + 1])), slice(int(w.start[s]), int(w.start[s + 1]))
        ref = O.attention(qs[rows], kk[at], vv[at], context[s], real, window)
        here = np.abs(ref) < (65504.0 * 0.99 if type == "f16" else np.inf)
        err = np.abs(got[rows] - ref)
        assert here.mean() > 0.9 and np.isfinite(got[rows][here]).all()
        assert (err <= bound(qs[rows], kk[at], vv[at], ref, type, abs(real), context[s]))[here].all(), s
