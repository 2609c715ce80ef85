"""More of what the calls of the 4-bit cache refuse: rotations without finite angles, outputs that overlap what is still to be
read, pointers off their boundaries."""
import ctypes as C

import numpy as np
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi
from test_cache4_refusals import P, append, attention, batch, cache, read, rows


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


# heads of 128, 4 of queries and 2 of keys and values, f16: rows of 1024 and 512 bytes; 5 tokens
FAR = 1 << 24


def refused(call, message):
    rc, text = call
    return rc != 0 and message in text


@pytest.mark.parametrize("out,q_stride,out_stride,over", [
    (P, 512, 512, True), (P + 2, 512, 512, True), (P - 1022, 512, 512, True), (P + 4 * 1024 + 1022, 512, 512, True), (P + 1024, 512, 512, True),
    (P + 5 * 1024, 512, 512, False), (P - 5 * 1024, 512, 512, False),           # behind and before
    (P + 1024, 1024, 1024, False), (P - 1024, 1024, 1024, False),               # between one another's rows
    (P + 1022, 1024, 1024, True), (P + 1026, 1024, 1024, True), (P - 1022, 1024, 1024, True), (P + 3 * 2048 + 1024, 1024, 1024, False),
    (P + 1024, 1024, 512, True), (P + 4 * 2048 + 1024, 1024, 512, False)])      # rows of two strides
def test_a_result_that_overlaps_the_queries_is_refused(out, q_stride, out_stride, over):
    call = attention(cache(), batch(), out=out, q_stride=q_stride, out_stride=out_stride)
    assert refused(call, "over the queries") == over, call  # without a device what is not refused fails later


@pytest.mark.parametrize("kw,over", [
    (dict(q=P, q_out=P, k=FAR, v=FAR), False), (dict(q=P, q_out=P, q_out_stride=1024, k=FAR, v=FAR), True), (dict(q=P, q_out=P + 1024, k=FAR, v=FAR), True),
    (dict(q=P, q_out=P + 1024, q_stride=1024, q_out_stride=1024, k=FAR, v=FAR), False)])
def test_queries_go_over_themselves_or_apart(kw, over):
    call = append(cache(), batch(), rows(**kw))
    assert refused(call, "over q itself") == over, call


@pytest.mark.parametrize("kw,over", [
    (dict(k=P + 1024, v=P + 1536, q_stride=1024, k_stride=1024, v_stride=1024, q_out_stride=1024), False),  # in one fused buffer, queries in place
    (dict(k=P + 1022, v=P + 1536, q_stride=1024, k_stride=1024, v_stride=1024, q_out_stride=1024), True),
    (dict(q=FAR, k=P, v=2 * FAR), True), (dict(q=FAR, k=2 * FAR, v=P + 5 * 1024 - 2), True), (dict(q=FAR, k=P + 5 * 1024, v=P - 5 * 512), False)])
def test_queries_over_keys_or_values_are_refused(kw, over):
    call = append(cache(), batch(), rows(**kw))
    assert refused(call, "over keys and values") == over, call


@pytest.mark.parametrize("v,k_stride,v_stride,over", [(P, 256, 256, True), (P + 5 * 512, 256, 256, False), (P + 512, 512, 512, False), (P + 510, 512, 512, True)])
def test_keys_read_over_values_are_refused(v, k_stride, v_stride, over):
    call = read(cache(), batch(), v=v, k_stride=k_stride, v_stride=v_stride)
    assert refused(call, "over its values") == over, call


@pytest.mark.parametrize("name", ["context", "page_table", "query_start"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_a_batch_off_its_boundaries_is_refused(name, off):
    """Read as they are, these would end the process's context with a misaligned address."""
    for call in (append(cache(), batch(**{name: P + off}), rows()), attention(cache(), batch(**{name: P + off})), read(cache(), batch(**{name: P + off}))):
        assert refused(call, "4-byte boundaries"), call


@pytest.mark.parametrize("name,off,message", [("rope_turns", 4, "8-byte"), ("rope_turns", 1, "8-byte")] +
                         [(n, o, "norms and biases") for n in ("q_norm", "k_norm", "q_bias", "k_bias", "v_bias") for o in (1, 2, 3)])
def test_rows_off_their_boundaries_are_refused(name, off, message):
    call = append(cache(), batch(), rows(k=FAR, v=FAR, **{name: P + off}))
    assert refused(call, message), call
