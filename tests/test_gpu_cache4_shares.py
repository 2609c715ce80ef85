"""What a rank of a tensor-parallel session with the 4-bit cache holds and computes: its share of the key/value heads and their queries. On one
device, share by share: the stored bytes are the whole's, and the results as near to the definition as the whole's are."""
import numpy as np
import pytest

import cache4_oracle as O
import helpers as H  # noqa: F401  (puts the repository on sys.path)
from test_gpu_cache4 import tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ranks", [2, 4, 8])
@pytest.mark.parametrize("tokens", [1, 9, 300])
def test_shares_of_the_heads_are_parts_of_the_whole(tokens, ranks):
    import torch
    from brisk_llm_b200 import cache4
    heads, kv, dim, context = 32, 8, 128, 200
    gen = torch.Generator("cuda").manual_seed(50)
    rotary, norm = cache4.Rotary(dim, 1e6), torch.rand(dim, generator=gen, device="cuda") + 0.5
    rows = [[torch.randn((n, h, dim), generator=gen, device="cuda") for h in (heads, kv, kv)] for n in (context, tokens)]

    def run(rank, of):
        cache = cache4.PagedCache.allocate(8, kv // of, dim)
        for at, part in ((0, rows[0]), (context, rows[1])):
            batch = cache4.Batch(torch.full((1,), at, dtype=torch.int32, device="cuda"), len(part[0]), columns=8, max_length=at + len(part[0]))
            q, k, v = (x[:, rank * x.shape[1] // of:(rank + 1) * x.shape[1] // of].contiguous() for x in part)
            q = cache.append(batch, q, k, v, rotary=rotary, q_norm=norm, k_norm=norm)
        return cache, q, cache.attention(batch, q)

    whole, q, out = run(0, 1)
    every = cache4.Batch(torch.zeros(1, dtype=torch.int32, device="cuda"), context + tokens, columns=8)
    k, v = (x.double().cpu().numpy() for x in whole.read(every))
    qs = q.double().cpu().numpy()
    ref = O.attention(qs, k, v, context, dim ** -0.5)
    bound = tolerance(qs, k, v, ref, "f32", dim ** -0.5, len(k))
    assert (np.abs(out.double().cpu().numpy() - ref) <= bound).all()
    for rank in range(ranks):
        cache, _, part = run(rank, ranks)
        mine, heads_at = slice(rank * kv // ranks, (rank + 1) * kv // ranks), slice(rank * heads // ranks, (rank + 1) * heads // ranks)
        for name in ("k_quants", "k_scales", "v_quants", "v_scales"):
            assert torch.equal(getattr(cache, name), getattr(whole, name)[:, mine]), name
        assert (np.abs(part.double().cpu().numpy() - ref[:, heads_at]) <= bound[:, heads_at]).all()
