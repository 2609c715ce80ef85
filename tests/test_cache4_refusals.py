"""What the calls of the 4-bit cache refuse, and the turns of a rotation: all before a device is asked for."""
import ctypes as C

import numpy as np
import pytest

import helpers as H  # noqa: F401  (puts the repository on sys.path)
from brisk_llm_b200 import abi

P = 1 << 20  # stands for a device address; no call of this file gets as far as using it


def cache(**kw):
    f = dict(k_quants=P, k_scales=P, v_quants=P, v_scales=P, pages=4, page_size=64, kv_heads=2, head_dim=128)
    f.update(kw)
    return abi.Cache4(*f.values())


def batch(**kw):
    f = dict(context=P, page_table=P, query_start=P, sequences=2, table_columns=2, tokens=5, max_tokens=0, max_length=0)
    f.update(kw)
    return abi.Cache4Batch(*f.values())


def rows(**kw):
    r = abi.Cache4Rows(q=P, k=P, v=P, q_out=P, q_stride=512, k_stride=256, v_stride=256, q_out_stride=512, rope_turns=P, rope_dim=128, eps=1e-6, heads=4, type=1)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def append(c, b, r):
    err = C.create_string_buffer(512)
    rc = abi.load_library().brisk_cuda_cache4_append(c, b, r, None, err, 512)
    return rc, err.value.decode()


def attention(c, b, type=1, q=P, out=2 * P, q_stride=512, out_stride=512, heads=4, scale=0.0, window=0):
    err = C.create_string_buffer(512)
    rc = abi.load_library().brisk_cuda_cache4_attention(c, b, type, q, out, q_stride, out_stride, heads, scale, window, None, err, 512)
    return rc, err.value.decode()


def read(c, b, type=1, k=P, v=P, k_stride=256, v_stride=256):
    err = C.create_string_buffer(512)
    rc = abi.load_library().brisk_cuda_cache4_read(c, b, type, k, v, k_stride, v_stride, None, err, 512)
    return rc, err.value.decode()


@pytest.mark.parametrize("wrong,message", [
    (dict(head_dim=96), "head sizes"), (dict(head_dim=0), "head sizes"), (dict(kv_heads=0), "key/value heads"),
    (dict(page_size=8), "pages of 16"), (dict(page_size=48), "power of two"), (dict(page_size=8192), "pages of 16"),
    (dict(pages=0), "at least one page"), (dict(k_scales=None), "four planes"), (dict(v_quants=P + 8), "16-byte")])
def test_a_cache_that_does_not_hold_is_refused(wrong, message):
    for rc, text in (append(cache(**wrong), batch(), rows()), attention(cache(**wrong), batch()), read(cache(**wrong), batch())):
        assert rc != 0 and text.startswith("cuda: ") and message in text


@pytest.mark.parametrize("wrong,message", [
    (dict(context=None), "positions before the batch"), (dict(query_start=None), "split evenly"), (dict(table_columns=0), "columns"),
    (dict(table_columns=1 << 26), "columns"), (dict(tokens=1 << 31), "2^31"), (dict(sequences=65536), "65535 sequences")])
def test_a_batch_that_does_not_hold_is_refused(wrong, message):
    for rc, text in (append(cache(), batch(**wrong), rows()), attention(cache(), batch(**wrong)), read(cache(), batch(**wrong))):
        assert rc != 0 and message in text


@pytest.mark.parametrize("wrong,message", [
    (dict(type=2), "f32, f16 and bf16"), (dict(k=None), "keys and values"), (dict(v=P + 1), "boundaries"), (dict(heads=3), "multiple"),
    (dict(q=None), "queries"), (dict(q_out=P + 1), "queries"), (dict(q_stride=511), "strides"), (dict(q_out_stride=0), "strides"), (dict(k_stride=255), "strides"),
    (dict(v_stride=128), "strides"), (dict(rope_dim=130), "even width"), (dict(rope_dim=63), "even width"), (dict(rope_turns=None), "turns"),
    (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"), (dict(rope_attn_factor=float("inf")), "factor")])
def test_rows_that_do_not_fit_are_refused(wrong, message):
    rc, text = append(cache(), batch(), rows(**wrong))
    assert rc != 0 and message in text


@pytest.mark.parametrize("wrong,message", [
    (dict(type=8), "f32, f16 and bf16"), (dict(heads=0), "multiple"), (dict(heads=5), "multiple"), (dict(scale=float("inf")), "finite"),
    (dict(q=None), "queries"), (dict(out=P), "over the queries"), (dict(out=P + 1), "boundaries"), (dict(q_stride=100), "strides")])
def test_an_attention_that_does_not_fit_is_refused(wrong, message):
    rc, text = attention(cache(), batch(), **wrong)
    assert rc != 0 and message in text


def test_more_rows_than_an_index_holds_are_refused():
    rc, text = attention(cache(kv_heads=1, head_dim=64), batch(tokens=1 << 20), q_stride=1 << 20, out_stride=1 << 20, heads=4096)
    assert rc != 0 and "2^31" in text


def test_a_read_that_does_not_fit_is_refused():
    for wrong, message in ((dict(type=3), "f32, f16"), (dict(k=None), "outputs"), (dict(v=P + 1), "boundaries"), (dict(k_stride=1), "strides")):
        rc, text = read(cache(), batch(), **wrong)
        assert rc != 0 and message in text


def test_a_null_description_is_refused_and_a_message_needs_no_room():
    lib = abi.load_library()
    assert append(None, batch(), rows())[0] != 0
    assert append(cache(), None, rows())[0] != 0
    assert append(cache(), batch(), None)[0] != 0
    assert lib.brisk_cuda_cache4_read(None, None, 0, None, None, 0, 0, None, None, 0) != 0


def test_an_empty_batch_is_done_at_once():
    for b in (batch(sequences=0, context=None), batch(tokens=0, query_start=None)):
        assert append(cache(), b, rows()) == (0, "") and attention(cache(), b) == (0, "") and read(cache(), b) == (0, "")


@pytest.mark.parametrize("width,base,scale,factors", [(2, 1e4, 1.0, False), (128, 1e6, 0.125, False), (96, 5e5, 1.0, True)])
def test_turns_of_a_rotation(width, base, scale, factors):
    err = C.create_string_buffer(512)
    divisors = np.linspace(1.0, 32.0, width // 2).astype(np.float32)
    out = np.empty(width // 2)
    rc = abi.load_library().brisk_cuda_rope_turns(width, base, scale, divisors.ctypes.data_as(C.POINTER(C.c_float)) if factors else None,
                                                  out.ctypes.data_as(C.POINTER(C.c_double)), err, 512)
    assert rc == 0, err.value
    want = scale * base ** (-2.0 * np.arange(width // 2) / width) / (divisors if factors else 1.0) / (2 * np.pi)
    assert np.allclose(out, want, rtol=1e-15 * 8, atol=0)
    for wrong in ((3, base, scale), (0, base, scale), (width, -1.0, scale), (width, base, float("nan"))):
        assert abi.load_library().brisk_cuda_rope_turns(*wrong, None, out.ctypes.data_as(C.POINTER(C.c_double)), err, 512) != 0
