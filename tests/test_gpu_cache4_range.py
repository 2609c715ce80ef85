"""The 4-bit cache's operators at the ends of their range: weights far below a row's largest. Against the definition, both kernels of the
attention: few rows and many."""
import numpy as np
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from test_gpu_cache4 import HALF_STEP, rounded

pytestmark = pytest.mark.gpu


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


def torch_type(name):
    from test_gpu_cache4 import torch_types
    return torch_types()[name]
