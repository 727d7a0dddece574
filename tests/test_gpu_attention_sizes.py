"""Attention over keys and values of unlike sizes: blocks of zeros or of small
values beside large ones, one large channel, scores too large for an exponent
beside them. Each tile height, prompts, images and a cache.

The bound. What tests/_attention.py:attention64 allows, and for what the limbs
hold less of than of values of like sizes:
  - a weight is held to 2^-22 of itself or to 2^-25 of the row's largest;
  - a value (fp32, bf16) to 2^-22 of itself or to 2^-39 of the largest of the
    16 consecutive tokens it is among (2^-125 where that is less);
  - products of weight and value below 2^-60 of a row's largest may be left out,
    here with 2^3 for references in whole powers of two and the 2^4 that they
    may lag, each of the row's keys once.
The first two count twice where attention64's bound counts numerator and
denominator alike; the denominator has none of them."""
import numpy as np
import pytest

import _attention as A
from _attention_plan import plan, plan_of
from test_gpu_attention import _check, _paged, _prompt, _rand, hip  # noqa: F401

pytestmark = pytest.mark.gpu


def _reference(q, k, v, scale, positions):
    """As attention64, with the bound above"""
    o, bound = A.attention64(q, k, v, scale, positions)
    group = q.shape[1] // k.shape[1]
    size = np.abs(v).astype(np.float64)
    n = len(size)
    largest = np.zeros_like(size)
    for j in range(0, n, 16):
        largest[j:j + 16] = size[j:j + 16].max(axis=(0, 2), keepdims=True)
    for i, last in enumerate(positions):
        for h in range(q.shape[1]):
            s = scale * (k[:last + 1, h // group].astype(np.float64) @ q[i, h].astype(np.float64))
            p = np.exp(s - s.max())
            p /= p.sum()
            a, b = size[:last + 1, h // group], largest[:last + 1, h // group]
            held = 2.0 ** -22 * p + 2.0 ** -25 * p.max()
            bound[i, h] += held @ a + p @ (2.0 ** -22 * a + 2.0 ** -39 * b) + 2.0 ** -125
            bound[i, h] += (last + 1) * 2.0 ** -53 * np.max(p[:, None] * a)
    return o, bound


def _values(kind, rng, n, heads, dim):
    """Values of unlike sizes"""
    v = _rand(rng, n, heads, dim)
    at = np.arange(n)
    if kind == "zeros_then_large":
        v[at < n // 2 // 16 * 16 + 16] = 0
        v *= np.float32(1e30)
    elif kind == "large_then_zeros":
        v[at >= n // 2 // 16 * 16] = 0
        v *= np.float32(1e30)
    elif kind == "zeros_between":  # every second block of 16
        v[at // 16 % 2 == 0] = 0
        v *= np.float32(1e24)
    elif kind.startswith("channel") and n:  # one channel of one block
        v[min(n // 3 // 16 * 16 + 5, n - 1), :, 3] = 2.0 ** int(kind[7:])
    elif kind == "blocks":  # each block of a size of its own, 2^-30 to 2^30
        v *= (2.0 ** rng.integers(-30, 31, -(-n // 16)))[at // 16][:, None, None].astype(np.float32)
    elif kind == "wild":  # 2^-90 to 2^110
        v *= (2.0 ** rng.integers(-90, 111, -(-n // 16)))[at // 16][:, None, None].astype(np.float32)
    return v


KINDS = ["zeros_then_large", "large_then_zeros", "zeros_between", "channel20", "channel30", "channel60", "blocks", "wild"]


def _some(n):
    return sorted({i for i in (0, 1, 15, 16, 17, 33, 48, 63, 64, 65, 130, 255, 256, n // 3, n // 2, n - 1) if 0 <= i < n} | set(range(0, n, 89)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim,new,rows,images", [
    (2, 1, 64, [64], 16, False),
    (4, 2, 128, [100], 16, False),
    (8, 8, 64, [333, 1, 0, 200], 128, False),
    (4, 4, 128, [100, 1, 150] * 9, 128, False),
    (4, 1, 128, [300, 500], 256, False),
    (4, 2, 128, [1100, 1030], 256, True),
    (16, 2, 64, [1200, 900], 256, True),
])
def test_prompt_values_of_unlike_sizes(qmv, hip, kind, heads, kv_heads, dim, new, rows, images):  # noqa: F811
    chosen = plan(sum(new), heads, kv_heads, dim, len(new))
    assert (chosen.rows, chosen.images > 0) == (rows, images)
    rng = np.random.default_rng(len(kind) + dim)
    T = sum(new)
    q, k = _rand(rng, T, heads, dim, wide=2), _rand(rng, T, kv_heads, dim, wide=3)
    v = np.concatenate([_values(kind, rng, n, kv_heads, dim) for n in new])
    o = _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, dim ** -0.5)
    t = 0
    for s, n in enumerate(new[:4]):
        if n:
            at = _some(n)
            ref, bound = _reference(q[t:t + n][at], k[t:t + n], v[t:t + n], dim ** -0.5, at)
            _check(o[t:t + n][at], ref, bound, f"{kind} sequence {s} of {n}")
        t += n


@pytest.mark.parametrize("t", [A.F32, A.BF16, A.F16], ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim,new,length,rows", [
    (14, 2, 64, [1, 1, 2], [700, 64, 129], (16,)),          # cut into pieces
    (28, 4, 128, [1], [2000], (16,)),
    (28, 4, 128, [4, 3, 5, 4] * 6, [900, 40, 41, 333] * 6, (32,)),
    (28, 4, 128, [17, 1, 40, 30] * 3, [900, 700, 41, 333] * 3, (128, 256)),
    (14, 2, 64, [17, 1, 40, 30] * 3, [900, 700, 41, 333] * 3, (128,)),
    (28, 1, 128, [45], [2200], (256,)),
])
def test_paged_values_of_unlike_sizes(qmv, hip, t, kind, heads, kv_heads, dim, new, length, rows):  # noqa: F811
    rng = np.random.default_rng(len(kind) + dim)
    b = A.Batch(new, length, 16, 5)
    assert plan_of(b, heads, kv_heads, dim, t).rows in rows
    keys = [_rand(rng, n, kv_heads, dim, wide=3) for n in length]
    values = [_values(kind, rng, n, kv_heads, dim) for n in length]
    if t == A.F16:  # which holds 2^-24 to 2^16
        values = [np.clip(v, -60000, 60000) for v in values]
    keys, values = ([A.decode(A.encode(x, t), t) for x in y] for y in (keys, values))
    q = _rand(rng, b.tokens, heads, dim, wide=2)
    o, ok = _paged(qmv, hip, b, q, A.Cache(qmv, hip, b, keys, values, t), dim ** -0.5)
    assert ok == 1
    for s, n in enumerate(new[:4]):
        if n:
            a, at = int(b.starts[s]), _some(n)
            pos = b.positions(s)
            ref, bound = _reference(q[a:a + n][at], keys[s], values[s], dim ** -0.5, [pos[i] for i in at])
            _check(o[a:a + n][at], ref, bound, f"{A.NAMES[t]} {kind} sequence {s} ({n} of {length[s]})")


@pytest.mark.parametrize("size", [1e4, 1e8, 1e15])
@pytest.mark.parametrize("heads,kv_heads,dim,new", [(2, 1, 64, [80]), (4, 4, 128, [100, 1, 150] * 9), (4, 2, 128, [1100, 1030])])
def test_prompt_equal_keys_of_any_size(qmv, hip, size, heads, kv_heads, dim, new):  # noqa: F811
    """All keys alike and large, so that the scores (up to 1e31) have no place
    for an exponent of the values beside them: a row is the mean of the values
    up to it, each held to 2^-22 of itself or 2^-39 of the largest of its block;
    the equal weights to 2^-22, and n sums rounded by n 2^-23, numerator and
    denominator."""
    rng = np.random.default_rng(7)
    T = sum(new)
    q, k = np.full((T, heads, dim), size, np.float32), np.full((T, kv_heads, dim), size, np.float32)
    v = np.concatenate([_values("blocks", rng, n, kv_heads, dim) if n > 1 else _rand(rng, n, kv_heads, dim) for n in new])
    o = _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, dim ** -0.5)
    t = 0
    for n in new[:3]:
        for i in _some(n):
            x = np.repeat(v[t:t + i + 1].astype(np.float64), heads // kv_heads, 1)
            largest = np.max(np.abs(v[t:t + n]))
            size_of = np.abs(x).mean(0)
            bound = (3 * 2.0 ** -22 + 2 * (i + 65) * 2.0 ** -23) * size_of + 2.0 ** -39 * largest
            assert (np.abs(o[t + i] - x.mean(0)) <= bound).all(), (n, i)
        t += n


def test_a_large_value_of_a_later_token(qmv, hip):  # noqa: F811
    """Rows before a token with a large value keep what they hold but for the 16
    tokens of its block (their values are held to 2^-39 of the largest there)."""
    rng = np.random.default_rng(8)
    n, dim = 200, 64
    q, k, v = _rand(rng, n, 2, dim), _rand(rng, n, 1, dim), _rand(rng, n, 1, dim)
    v[150] *= np.float32(1e25)  # the block of 144..159
    o = _prompt(qmv, hip, [n], 2, 1, dim, q, k, v, 0.125)
    ref, bound = A.attention64(q[:144], k, v, 0.125, range(144))
    _check(o[:144], ref, bound + 2.0 ** -25 * 4, "before the block")
    at = list(range(150, 200))
    ref, bound = _reference(q[at], k, v, 0.125, at)
    _check(o[150:], ref, bound, "from the token on")
