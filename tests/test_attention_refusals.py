"""Calls of the attention entry points that are refused for what they are as a
whole, before any HIP call: no device is needed, and no address is read."""
import pytest

FAR = 1 << 44  # between addresses


def _prompt(qmv, tokens, heads, kv_heads, dim, count):
    seq = qmv.make_sequences(FAR, count)
    assert qmv.hip_lib().qmv_device_attention_prompt_f32(2 * FAR, 0, 3 * FAR, 0, 4 * FAR, 0, tokens, heads, kv_heads, dim, 0.1,
                                                         seq, 5 * FAR, 0, None) == 0
    return qmv.last_error()


@pytest.mark.parametrize("tokens,heads,dim,count", [(16384, 65535, 8, 16384), (16384, 65535, 128, 16384), (40000, 16384, 64, 3000)])
def test_more_threads_than_a_launch_has(qmv, tokens, heads, dim, count):
    """Within each limit by itself: 2^22 tokens, 65535 heads and sequences, 2^30
    rows."""
    assert "too many" in _prompt(qmv, tokens, heads, heads, dim, count)
    seq = qmv.make_sequences(FAR, count, FAR, FAR, 4)
    cache = qmv.make_paged_cache(3 * FAR, 4 * FAR, qmv.GGML_TYPE_F16, heads, dim, 16, 8)
    assert qmv.hip_lib().qmv_device_attention_paged_f32(2 * FAR, 0, tokens, heads, 0.1, seq, cache, 5 * FAR, 0, None, None) == 0
    assert "too many" in qmv.last_error()


def test_rows_of_a_call(qmv):
    """2^30 rows of a token and a head are the most (that this is no error of
    the arguments shows in the one that follows it)."""
    assert "rows" in _prompt(qmv, 1 << 22, 257, 257, 8, 1)
    assert "rows" not in _prompt(qmv, 1 << 22, 256, 256, 8, 60000)


def _rope(qmv, cache, q, qs, k, ks, v, vs, qo, ko, tokens=3, heads=4, kv_heads=2, dim=64):
    """The error of a call; "hip..." where it got as far as the device"""
    seq = qmv.make_sequences(FAR, 2, FAR, FAR, 4)
    ok = qmv.hip_lib().qmv_device_rope_append_f32(q, qs, heads, k, ks, v, vs, kv_heads, dim, tokens, FAR, dim, 0, seq, qo, ko, cache,
                                                  None, None)
    assert ok == 0
    return qmv.last_error()


@pytest.fixture
def no_device(qmv):
    """Calls that pass the host's rules end at the device, which must not be
    there: their addresses are not."""
    if qmv.hip_lib().qmv_device_count() > 0:
        pytest.skip("checks on addresses alone, for a machine without a GPU")


def test_rope_rows_that_share_floats(qmv, no_device):
    """In place, too: values that are the keys' rows would be stored half
    turned."""
    cache = qmv.make_paged_cache(8 * FAR, 9 * FAR, qmv.GGML_TYPE_F16, 2, 64, 16, 8)
    q, k, v = FAR, 2 * FAR, 3 * FAR
    for a in ((q, 0, k, 0, k, 0, q, k), (q, 0, k, 0, q, 0, q, k), (q, 0, k, 0, v, 0, q, v), (q, 0, k, 0, v, 0, k, q),
              (q, 0, q, 0, v, 0, q, q), (q, 512, q + 4 * 192, 512, v, 0, q, q + 4 * 192), (q, 512, q + 4 * 448, 512, v, 0, q, q + 4 * 448),
              (q, 512, q + 4 * 256, 512, q + 4 * 320, 512, q, q + 4 * 256), (q, 0, k, 0, k + 4 * 64, 256, q, k)):
        assert "overlaps rows" in _rope(qmv, cache, *a), a
    same = qmv.make_paged_cache(8 * FAR, 8 * FAR, qmv.GGML_TYPE_F16, 2, 64, 16, 8)
    assert "one place" in _rope(qmv, same, q, 0, k, 0, v, 0, q, k)


def test_rope_rows_side_by_side(qmv, no_device):
    """One buffer for q, k and v, in place or into another such buffer; values
    of the keys' own buffer."""
    cache = qmv.make_paged_cache(8 * FAR, 9 * FAR, qmv.GGML_TYPE_F16, 2, 64, 16, 8)
    q, k, v, out = FAR, FAR + 4 * 256, FAR + 4 * 384, 2 * FAR
    for a in ((q, 512, k, 512, v, 512, q, k), (q, 512, k, 512, v, 512, out, out + 4 * 256), (q, 512, k, 512, v, 512, q, 3 * FAR),
              (q, 0, out, 256, out + 4 * 128, 256, q, out)):
        assert "hip" in _rope(qmv, cache, *a), a


@pytest.mark.parametrize("change", [{"starts": FAR + 2}, {"lengths": FAR + 1}, {"pages": FAR + 3}, {"status": FAR + 2}], ids=str)
def test_unaligned_ints(qmv, no_device, change):
    a = {"starts": FAR, "lengths": FAR, "pages": FAR, "status": FAR, **change}
    seq = qmv.make_sequences(a["starts"], 2, a["lengths"], a["pages"], 4)
    cache = qmv.make_paged_cache(8 * FAR, 9 * FAR, qmv.GGML_TYPE_F16, 2, 64, 16, 8)
    assert qmv.hip_lib().qmv_device_attention_paged_f32(FAR, 0, 3, 4, 0.1, seq, cache, 5 * FAR, 0, a["status"], None) == 0
    assert "unaligned" in qmv.last_error()
    assert qmv.hip_lib().qmv_device_rope_append_f32(FAR, 0, 4, 2 * FAR, 0, 3 * FAR, 0, 2, 64, 3, FAR, 64, 0, seq, FAR, 2 * FAR, cache,
                                                    a["status"], None) == 0
    assert "unaligned" in qmv.last_error()
    if "starts" in change:
        assert qmv.hip_lib().qmv_device_attention_prompt_f32(FAR, 0, 2 * FAR, 0, 3 * FAR, 0, 3, 4, 2, 64, 0.1, seq, 5 * FAR, 0, None) == 0
        assert "unaligned" in qmv.last_error()
