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
