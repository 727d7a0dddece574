"""Refusals of the attention entry points, before any HIP call: no device is
needed, and the addresses are compared, never read."""
import ctypes

import numpy as np
import pytest

BUF = np.zeros(1 << 16, np.float32)
BASE = (BUF.ctypes.data + 63) // 64 * 64
BIG = 1 << 40  # an address far from the others


def _sequences(qmv, **change):
    s = qmv.make_sequences(BASE, 2, BASE + 64, BASE + 128, 4)
    for k, v in change.items():
        setattr(s, k, v)
    return s


def _cache(qmv, **change):
    c = qmv.make_paged_cache(BIG, 2 * BIG, qmv.GGML_TYPE_F16, 2, 64, 16, 8)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def _paged(qmv, seq, cache, **a):
    a = {"q": BASE, "qs": 0, "tokens": 3, "heads": 4, "scale": 0.125, "out": BASE + 65536, "os": 0, **a}
    return qmv.hip_lib().qmv_device_attention_paged_f32(a["q"], a["qs"], a["tokens"], a["heads"], a["scale"],
                                                        ctypes.byref(seq) if seq is not None else None,
                                                        ctypes.byref(cache) if cache is not None else None, a["out"], a["os"],
                                                        None, None)


def _prompt(qmv, seq, **a):
    a = {"q": BASE, "qs": 0, "k": BASE + 4096, "ks": 0, "v": BASE + 8192, "vs": 0, "tokens": 3, "heads": 4, "kv": 2, "dim": 64,
         "scale": 0.125, "out": BASE + 65536, "os": 0, **a}
    return qmv.hip_lib().qmv_device_attention_prompt_f32(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["tokens"],
                                                         a["heads"], a["kv"], a["dim"], a["scale"],
                                                         ctypes.byref(seq) if seq is not None else None, a["out"], a["os"], None)


def _rope(qmv, seq, cache, **a):
    a = {"q": BASE, "qs": 0, "heads": 4, "k": BASE + 4096, "ks": 0, "v": BASE + 8192, "vs": 0, "kv": 2, "dim": 64, "tokens": 3,
         "f": BASE + 16384, "rotary": 64, "qo": BASE + 32768, "ko": BASE + 65536, **a}
    return qmv.hip_lib().qmv_device_rope_append_f32(a["q"], a["qs"], a["heads"], a["k"], a["ks"], a["v"], a["vs"], a["kv"],
                                                    a["dim"], a["tokens"], a["f"], a["rotary"], 0,
                                                    ctypes.byref(seq) if seq is not None else None, a["qo"], a["ko"],
                                                    ctypes.byref(cache) if cache is not None else None, None, None)


SHARED = [{"tokens": 0}, {"tokens": -1}, {"tokens": (1 << 22) + 1}, {"heads": 0}, {"heads": 5}, {"heads": 65536}, {"q": None},
          {"q": BASE + 4}, {"qs": 252}, {"qs": 258}, {"qs": 1 << 31}, {"qs": -256}]
ATTENTION = [{"scale": float("nan")}, {"scale": float("inf")}, {"scale": -2e38}, {"out": None}, {"out": BASE + 8}, {"os": 255}, {"out": BASE},
             {"out": BASE + 1024}]


@pytest.mark.parametrize("change", SHARED + ATTENTION, ids=str)
def test_paged_arguments(qmv, change):
    assert _paged(qmv, _sequences(qmv), _cache(qmv), **change) == 0
    assert qmv.last_error() != ""


@pytest.mark.parametrize("change", SHARED + ATTENTION + [
    {"kv": 0}, {"kv": -2}, {"dim": 0}, {"dim": 4}, {"dim": 60}, {"dim": 136}, {"k": None}, {"v": None}, {"k": BASE + 4100},
    {"ks": 124}, {"vs": 129}, {"out": BASE + 4096}, {"out": BASE + 8192 + 512}], ids=str)
def test_prompt_arguments(qmv, change):
    assert _prompt(qmv, _sequences(qmv), **change) == 0
    assert qmv.last_error() != ""


@pytest.mark.parametrize("change", SHARED + [
    {"kv": 0}, {"dim": 12}, {"dim": 256}, {"k": None}, {"v": None}, {"f": None}, {"f": BASE + 4}, {"rotary": 66}, {"rotary": -8},
    {"rotary": 72}, {"rotary": 4}, {"qo": None}, {"qo": BASE + 4}, {"ko": BASE + 12}, {"qo": BASE + 256}, {"ko": BASE + 4096 + 256},
    {"qo": BASE + 4096}, {"ko": BASE + 8192}, {"ko": BASE}, {"qo": BIG}, {"ko": 2 * BIG}, {"kv": 4, "heads": 4}, {"ko": BASE + 32768}],
    ids=str)
def test_rope_arguments(qmv, change):
    assert _rope(qmv, _sequences(qmv), _cache(qmv), **change) == 0
    assert qmv.last_error() != ""


def test_rope_without_any_output_for_keys(qmv):
    assert _rope(qmv, _sequences(qmv), None, ko=None) == 0


@pytest.mark.parametrize("change", [{"starts": None}, {"count": 0}, {"count": -1}, {"count": 65536}, {"lengths": None},
                                    {"pages": None}, {"table_stride": 0}, {"table_stride": 1 << 28}], ids=str)
def test_sequences(qmv, change):
    assert _paged(qmv, _sequences(qmv, **change), _cache(qmv)) == 0
    assert _rope(qmv, _sequences(qmv, **change), _cache(qmv)) == 0
    if change.keys() & {"starts", "count"}:
        assert _prompt(qmv, _sequences(qmv, **change)) == 0
        assert _rope(qmv, _sequences(qmv, **change), None) == 0
    assert _paged(qmv, None, _cache(qmv)) == 0 and _prompt(qmv, None) == 0 and _rope(qmv, None, _cache(qmv)) == 0


@pytest.mark.parametrize("change", [{"keys": None}, {"values": None}, {"keys": BIG + 8}, {"type": 2}, {"type": 8}, {"kv_heads": 0},
                                    {"kv_heads": 3}, {"head_dim": 20}, {"head_dim": 136}, {"page_size": 0}, {"page_size": -16},
                                    {"page_size": 1 << 30}, {"pages": 0}, {"page_stride": 32}, {"head_stride": 60},
                                    {"token_stride": 0}, {"token_stride": 68}, {"page_stride": 1 << 62}], ids=str)
def test_cache(qmv, change):
    assert _paged(qmv, _sequences(qmv), _cache(qmv, **change)) == 0
    assert _rope(qmv, _sequences(qmv), _cache(qmv, **change)) == 0
    assert _paged(qmv, _sequences(qmv), None) == 0
    assert qmv.last_error() != ""


def test_output_over_the_cache(qmv):
    last = BIG + 2 * (8 * 2048 - 8)  # in the last row of the keys
    assert _paged(qmv, _sequences(qmv), _cache(qmv), out=last // 16 * 16) == 0


def test_python_raises(qmv):
    with pytest.raises(qmv.QmvError):
        qmv.device_attention_paged(BASE, 0, 4, 0.125, _sequences(qmv), _cache(qmv), BASE + 65536)
    with pytest.raises(qmv.QmvError):
        qmv.device_attention_prompt(BASE, BASE, BASE, 3, 4, 3, 64, 0.125, _sequences(qmv), BASE + 65536)
    with pytest.raises(qmv.QmvError):
        qmv.device_rope_append(BASE, 4, BASE, BASE, 2, 63, 3, BASE, 32, _sequences(qmv), BASE)
