"""More of what the calls of the 4-bit cache refuse: rotations without finite angles."""
import ctypes as C

import numpy as np
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi


def turns(width=8, base=1e4, scale=1.0, factors=None):
    err, out = C.create_string_buffer(512), np.full(width // 2, 7.0)
    divisors = None if factors is None else np.asarray(factors, np.float32)
    rc = abi.load_library().brisk_cuda_rope_turns(width, base, scale, None if divisors is None else divisors.ctypes.data_as(C.POINTER(C.c_float)),
                                                  out.ctypes.data_as(C.POINTER(C.c_double)), err, 512)
    return rc, err.value.decode(), out


@pytest.mark.parametrize("wrong", [0.0, -0.0, float("nan"), float("inf"), -float("inf")])
def test_divisors_without_an_angle_are_refused(wrong):
    for at in range(4):
        factors = [1.0, 2.0, 4.0, 8.0]
        factors[at] = wrong
        rc, text, _ = turns(factors=factors)
        assert rc != 0 and text.startswith("cuda: ") and "divisors" in text
    assert turns(factors=[1.0, -2.0, 4.0, 1e-30])[0] == 0


def test_angles_past_64_bits_are_refused():
    rc, text, _ = turns(base=1e-300, scale=1e200)
    assert rc != 0 and "angles are finite" in text


@pytest.mark.parametrize("factor", [0.0, float("nan"), float("inf")])
def test_a_rotary_s_factor_is_what_is_multiplied_by(factor):
    from brisk_llm_b200 import cache4
    with pytest.raises(RuntimeError, match="^cuda: .*factor"):
        cache4.Rotary(64, 1e4, attn_factor=factor, device="cpu")
    assert cache4.Rotary(64, 1e4, attn_factor=0.5, device="cpu").attn_factor == 0.5
