"""Sessions whose key/value cache is held in 4 bits (BRISK_CUDA_FLAG_CACHE_4BIT).

The attention of a layer is compared with the definition in 64 bits (cache4_oracle.py) on the session's own queries, keys and values: in
these models a layer's key projection is made of the query projection's rows, so that the queries a session shows are the keys it
stored, and a second session without norm and rotation shows the values.
"""
import dataclasses

import numpy as np
import pytest

import cache4_oracle as O
import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi, engine, synth

pytestmark = pytest.mark.gpu
FLAG = abi.FLAG_CACHE_4BIT


def shared_projections(spec, seed):
    """A model whose keys and values are projected by rows of the query projection: query head h of a group has its key head's."""
    model = synth.generate(spec, seed=seed)
    t = dict(model.tensors)
    group = spec.heads // spec.kv_heads
    for i in range(spec.layers):
        fmt, (rows, cols), data = t[f"blk.{i}.attn_k.weight"]
        heads = data.reshape(spec.kv_heads, -1)
        t[f"blk.{i}.attn_v.weight"] = t[f"blk.{i}.attn_k.weight"]
        t[f"blk.{i}.attn_q.weight"] = (fmt, (rows * group, cols), np.ascontiguousarray(np.repeat(heads, group, axis=0)).reshape(-1))
    return synth.HostModel(spec, t, model.rope_factors)


def plain(model):
    """The same without per-head norm and rotation: its queries are the projection itself."""
    m = synth.HostModel(model.spec, model.tensors, model.rope_factors)
    for layer in m._keep[-1]:
        layer.no_rope, layer.q_norm, layer.k_norm = 1, None, None
    return m


ONE_LAYER = {
    "qwen3": synth.tiny(synth.QWEN3_0_6B, layers=1, vocab=512, context=1500),
    "llama": synth.tiny(synth.LLAMA_3_2_1B, layers=1, vocab=512, context=1500),
    "bitnet": synth.tiny(synth.BITNET_2B, layers=1, vocab=512, context=700),
    "gemma3": synth.tiny(synth.GEMMA3_1B, layers=1, vocab=512, context=1500, sliding_window=100),
    "phi3": synth.tiny(synth.MISTRAL_7B, arch="phi3", layers=1, vocab=512, context=700, hidden=1024, heads=8, kv_heads=8, ffn=2048, rope_dim=96,
                       rope_attn_factor=1.19, rope_original_context=512),
}


@pytest.mark.parametrize("family", sorted(ONE_LAYER))
def test_a_layer_attends_as_the_definition_says(family):
    spec = ONE_LAYER[family]
    model = shared_projections(spec, seed=3)
    dim, heads, kv, group = spec.head_dim, spec.heads, spec.kv_heads, spec.heads // spec.kv_heads
    tokens = synth.random_tokens(spec, 1300, seed=4)
    keys, values, at = [], [], 0
    window = spec.sliding_window if spec.layer_slides(0) else 0
    with engine.CudaSession(model, flags=FLAG) as s, engine.CudaSession(plain(model), flags=FLAG) as p:
        assert "4 bits" in s.step_path()
        for n in (1, 1, 9, 70, 1, 24, 400, 1, 1, 130, 3, 1):
            if at + n > spec.context:
                break
            s.eval(tokens[at:at + n])
            p.eval(tokens[at:at + n])
            query = s.debug_buffer("query", n * heads * dim).reshape(n, heads, dim)
            keys.append(query[:, ::group])
            values.append(p.debug_buffer("query", n * heads * dim).reshape(n, heads, dim)[:, ::group])
            got = s.debug_buffer("attended", n * heads * dim).reshape(n, heads, dim)
            k, v = (O.values(*O.quantise(np.concatenate(x))) for x in (keys, values))
            ref = O.attention(query.astype(np.float64), k, v, at, dim ** -0.5, window)
            # f32 throughout, as the operators' tests have it; a key that the session rounds from 64 bits and this test from its f32 copy may
            # fall on the other side of a border: of at most 2^-22 of the values, each moving one result in `at` by a step
            assert np.linalg.norm(got - ref) <= 1e-3 * np.linalg.norm(ref), (n, at)
            at += n


FAMILIES = dict(ONE_LAYER, smollm3=synth.tiny(synth.LLAMA_3_2_1B, arch="smollm3", layers=4, vocab=512, context=700, llama3_rope=None),
                biased=synth.tiny(synth.QWEN3_0_6B, layers=2, vocab=512, context=700, qkv_bias=True))


@pytest.mark.parametrize("family", sorted(FAMILIES))
def test_the_ways_of_a_step_agree_bit_for_bit(family):
    """Replayed, launched kernel by kernel, through the batched kernels, and in the device's own greedy loop, across 512 positions where the
    replayed form changes."""
    spec = dataclasses.replace(FAMILIES[family], layers=max(2, FAMILIES[family].layers))
    model = synth.perturb_norms(synth.generate(spec, seed=5))
    tokens = synth.random_tokens(spec, 520, seed=6)
    runs = {}
    for name, flags in (("graph", 0), ("kernels", abi.FLAG_NO_GRAPH), ("batched", abi.FLAG_NO_MEGAKERNEL)):
        with engine.CudaSession(model, flags=FLAG | flags) as s:
            rows = [s.eval(tokens[:505]).copy()]
            for i in range(505, 520):
                rows.append(s.eval(tokens[i:i + 1]).copy())
            s.rollback(510)
            ids, logits = s.generate_greedy(int(tokens[510]), 6, want_logits=True)
            runs[name] = np.concatenate((np.stack(rows), logits))
            assert np.isfinite(runs[name]).all()
            assert list(ids) == [int(np.argmax(r)) for r in logits]
            assert np.array_equal(logits[0], rows[6])  # the step after position 510 once more
    for name in ("kernels", "batched"):
        assert np.array_equal(runs["graph"], runs[name]), name


def test_rollback_verify_and_scoring():
    spec = synth.tiny(synth.QWEN3_0_6B, layers=2, vocab=512, context=700)
    model = synth.perturb_norms(synth.generate(spec, seed=7))
    tokens = synth.random_tokens(spec, 300, seed=8)
    with engine.CudaSession(model, flags=FLAG) as s:
        s.eval(tokens[:200])
        first = s.eval_all(tokens[200:209]).copy()
        s.rollback(200)
        assert np.array_equal(first, s.eval_all(tokens[200:209]))
        s.rollback(0)
        s.eval(tokens[:200])
        assert np.array_equal(first, s.eval_all(tokens[200:209]))
        ids, values = s.eval_topk(tokens[209:210], 5)
        s.rollback(209)
        row = s.eval(tokens[209:210])
        assert list(ids) == list(np.argsort(-row, kind="stable")[:5]) and np.array_equal(values, row[ids])
        s.rollback(0)
        total = s.log_likelihood(tokens[:64])
        s.rollback(0)
        rows = s.eval_all(tokens[:63]).astype(np.float64)
        logp = rows - rows.max(1, keepdims=True)
        logp -= np.log(np.exp(logp).sum(1, keepdims=True))
        # 64 and 63 tokens of one batch: the same kernels and orders, the last row apart
        assert abs(total - logp[np.arange(63), tokens[1:64]].sum()) <= 63 * 2.0 ** -20 * np.abs(logp).max()


def test_what_a_session_holds():
    spec = synth.tiny(synth.QWEN3_0_6B, layers=2, vocab=512, context=640)
    model = synth.generate(spec, seed=9)
    wide, four = engine.estimate_memory(model), engine.estimate_memory(model, flags=FLAG)
    assert four["cache"] * 32 == wide["cache"] * 9 and four["scratch"] < wide["scratch"] and four["weights"] == wide["weights"]
    with engine.CudaSession(model, flags=FLAG) as s, engine.CudaSession(model) as w:
        s.eval([1, 2, 3])
        w.eval([1, 2, 3])
        assert s.stats()["kv_bytes"] == four["cache"] and w.stats()["kv_bytes"] == wide["cache"]
    with engine.CudaSession(model, max_context=70, flags=FLAG) as s:  # not whole pages
        s.eval(np.arange(69))
        s.eval([5])
        with pytest.raises(RuntimeError, match="context length exceeded"):
            s.eval([5])
        assert engine.estimate_memory(model, max_context=70, flags=FLAG)["cache"] == s.stats()["kv_bytes"]


def test_sessions_of_both_kinds_side_by_side():
    """A 4-bit session leaves one with the f16 cache as it is, bit for bit."""
    spec = synth.tiny(synth.QWEN3_0_6B, layers=2, vocab=512, context=256)
    model = synth.perturb_norms(synth.generate(spec, seed=10))
    tokens = synth.random_tokens(spec, 60, seed=11)
    with engine.CudaSession(model) as w:
        alone = [w.eval(tokens[:50]).copy()] + [w.eval(tokens[i:i + 1]).copy() for i in range(50, 60)]
    with engine.CudaSession(model) as w, engine.CudaSession(model, flags=FLAG) as s:
        both = []
        for part in [tokens[:50]] + [tokens[i:i + 1] for i in range(50, 60)]:
            s.eval(part)
            both.append(w.eval(part).copy())
    assert all(np.array_equal(a, b) for a, b in zip(alone, both))
