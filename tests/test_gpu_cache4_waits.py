"""The bounded waits of the many-rows attention over a 4-bit cache (csrc/cache4_prompt.cu): one that ran out is reported by the call of the
session it belongs to. Nothing here faults or hangs: BRISK_CUDA_TEST_TC_TIMEOUT=2 + k has the kernel never widen a CTA's tile k of
positions, so that the waits for it run out after 50 us."""
import numpy as np
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi, engine, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (32, 8, 64)], ids=["positions shared by two CTAs", "one CTA"])
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
def test_a_wait_that_runs_out_is_reported_by_its_own_session(heads, kv_heads, dim, tile, monkeypatch):
    """Tiles at which nothing, one, both places of the ring have been filled and one has been filled again (tiles of 64 positions, four to
    eight to a CTA). The call raises, nothing of it is left, and another session of the process goes on with the bits it had."""
    spec = synth.tiny(synth.QWEN3_0_6B, layers=1, vocab=256, context=600, hidden=1024, heads=heads, kv_heads=kv_heads, head_dim=dim, ffn=1024)
    model = synth.perturb_norms(synth.generate(spec, seed=7))
    tokens = synth.random_tokens(spec, 512, seed=8)
    with engine.CudaSession(model, flags=abi.FLAG_CACHE_4BIT) as sound:
        want = sound.eval(tokens).copy()
        assert np.isfinite(want).all()
        monkeypatch.setenv("BRISK_CUDA_TEST_TC_TIMEOUT", str(2 + tile))
        with engine.CudaSession(model, flags=abi.FLAG_CACHE_4BIT) as failed:
            monkeypatch.delenv("BRISK_CUDA_TEST_TC_TIMEOUT")
            for _ in range(2):
                with pytest.raises(RuntimeError, match="ran out"):
                    failed.eval(tokens)
                assert failed.position() == 0
                sound.rollback(0)
                assert np.array_equal(sound.eval(tokens), want)
