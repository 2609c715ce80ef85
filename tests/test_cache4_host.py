"""What a session with the key/value cache in 4 bits asks for, alone and as a rank of several."""
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi, engine, synth

SHAPES = {"qwen3": synth.tiny(synth.QWEN3_0_6B, layers=3, vocab=512, context=640, hidden=512, ffn=512), "llama": synth.tiny(synth.MISTRAL_7B, layers=2, vocab=512, context=1000, hidden=512, heads=8, kv_heads=4, ffn=512),
          "gemma3": synth.tiny(synth.QWEN3_0_6B, arch="gemma3", layers=7, vocab=1024, hidden=512, heads=8, kv_heads=4, ffn=512, context=512, sliding_window=16,
                               rope_scaling_factor=8.0)}


@pytest.mark.parametrize("ranks", [1, 2, 4])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_memory_of_a_cache_in_4_bits_and_of_a_rank_s_share(shape, ranks):
    spec = SHAPES[shape]
    model = synth.generate(spec, seed=0)
    four, wide = (engine.estimate_memory(model, tp_size=ranks, flags=f) for f in (abi.FLAG_CACHE_4BIT, 0))
    positions = -(-spec.context // 64) * 64  # whole pages
    assert four["cache"] == spec.layers * 2 * positions * (spec.kv_heads // ranks) * (spec.head_dim // 2 + spec.head_dim // 32 * 2)
    assert wide["cache"] == spec.layers * 2 * spec.context * (spec.kv_heads // ranks) * spec.head_dim * 2
    assert four["weights"] == wide["weights"]
    # no scores of a batch, and turns instead of tables of every position
    scores = 512 * (spec.heads // ranks) * spec.context * 4
    tables = spec.context * spec.head_dim * 4 * (2 if spec.sliding_window else 1)
    assert wide["scratch"] - four["scratch"] == scores + tables - 2 * spec.head_dim * 8
