"""The bounds of a batch (max_tokens, max_length) decide how the work of the 4-bit cache's attention is split, not what comes out: given tightly,
loosely and not at all, each against the definition in 64 bits with the tolerances of test_gpu_cache4.py."""
import numpy as np
import pytest

import cache4_oracle as O
import helpers as H  # noqa: F401  (puts the repository on sys.path)
from test_gpu_cache4 import World, rounded, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,tokens", [(128, 1), (64, 3), (256, 70), (128, 150), (64, 400)])
def test_whatever_bounds_are_given_the_result_is_the_definition_s(dim, tokens, type):
    from brisk_llm_b200 import cache4
    context, heads = [900, 10], 16
    w = World(40, 2, dim, context, [tokens, tokens], spare_columns=9)
    q = rounded(w.rng.standard_normal((w.rows, heads, dim)), type).to(w.device)
    refs = []
    for s in range(2):
        k, v = w.values(s, context[s] + tokens)
        qs = q[s * tokens:(s + 1) * tokens].double().cpu().numpy()
        ref = O.attention(qs, k, v, context[s], dim ** -0.5)
        refs.append((ref, tolerance(qs, k, v, ref, type, dim ** -0.5, len(k))))
    for bounds in (dict(max_tokens=tokens, max_length=900 + tokens), dict(), dict(max_tokens=2 * tokens), dict(max_length=901 + 2 * tokens), dict(max_tokens=tokens, max_length=1)):
        batch = cache4.Batch(w.batch.context, w.rows, page_table=w.batch.page_table, query_start=w.batch.query_start, **bounds)
        got = w.cache.attention(batch, q).double().cpu().numpy()
        for s, (ref, bound) in enumerate(refs):
            err = np.abs(got[s * tokens:(s + 1) * tokens] - ref)
            assert (err <= bound).all(), (bounds, s, err.max())
            assert np.linalg.norm(err) <= {"f32": 1e-5, "f16": 1e-3, "bf16": 5e-3}[type] * np.linalg.norm(ref), (bounds, s)
