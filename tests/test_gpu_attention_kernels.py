"""Every kernel that the attention planner can choose, against 64 bits, with the
choice itself asserted: images and row tiles of several sequences, and pieces of
decoding sequences of like lengths."""
import numpy as np
import pytest

import _attention as A
from _attention_plan import plan, plan_of
from test_gpu_attention import _check, _check_paged, _paged, _paged_case, _prompt, _rand, hip  # noqa: F401

pytestmark = pytest.mark.gpu

PROMPTS = [  # heads, kv_heads, dim, new tokens, rows of a tile, through images
    (4, 2, 128, [2100, 3, 0, 2100], 256, True),
    (2, 1, 104, [1500, 1801], 256, True),
    (16, 2, 64, [1200, 5, 2500], 256, True),
    (8, 1, 40, [70, 2060, 1], 256, False),
    (4, 1, 128, [300, 500], 256, False),
    (4, 4, 128, [100, 1, 150, 0, 129] * 6, 128, False),
    (8, 8, 64, [600, 1, 0, 90], 128, False),
    (6, 2, 96, [5, 0, 1, 17, 64] * 30, 128, False),
    (28, 4, 128, [37], 16, False),
]


def _rows(n):
    """Some rows of a sequence: its ends, those of tiles, and some between"""
    return sorted({i for i in (0, 1, 15, 16, 31, 32, 63, 64, 65, 127, 128, 255, 256, 257, 511, n // 2, n - 65, n - 2, n - 1)
                   if 0 <= i < n} | set(range(0, n, 97)))


@pytest.mark.parametrize("heads,kv_heads,dim,new,rows,images", PROMPTS, ids=lambda x: None if isinstance(x, list) else str(x))
def test_prompt_kernels(qmv, hip, heads, kv_heads, dim, new, rows, images):  # noqa: F811
    chosen = plan(sum(new), heads, kv_heads, dim, len(new))
    assert (chosen.rows, chosen.images > 0) == (rows, images)
    rng = np.random.default_rng(dim + sum(new))
    T = sum(new)
    q, k, v = _rand(rng, T, heads, dim, wide=2), _rand(rng, T, kv_heads, dim, wide=3), _rand(rng, T, kv_heads, dim)
    o = _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, dim ** -0.5, extra=(4, 8, 4))
    t = 0
    for s, n in enumerate(new):
        if n:
            at = _rows(n)
            ref, bound = A.attention64(q[t:t + n][at], k[t:t + n], v[t:t + n], dim ** -0.5, at)
            _check(o[t:t + n][at], ref, bound, f"sequence {s} of {n}")
        t += n


def test_images_of_later_sequences_not_finite(qmv, hip):  # noqa: F811
    """A value that is not finite in the second sequence, which begins inside a
    tile, reaches the rows that attend it and no others."""
    new, dim = [1100, 2, 1300], 128
    assert plan(sum(new), 4, 2, dim, 3).images == 0 and plan(sum(new[::2]), 4, 2, dim, 2).images > 0
    new = new[::2]
    rng = np.random.default_rng(12)
    T, a = sum(new), new[0]
    for bad in (np.inf, np.nan):
        q, k, v = _rand(rng, T, 4, dim), _rand(rng, T, 2, dim), _rand(rng, T, 2, dim)
        v[a + 400, 0, 5] = v[a + 1299, 1, 100] = bad
        k[a + 800, 1, 3] = np.nan
        o = _prompt(qmv, hip, new, 4, 2, dim, q, k, v, 0.1)
        odd = np.zeros_like(o, bool)
        odd[a + 400:, :2, 5] = odd[a + 800:, 2:] = True
        assert not np.isfinite(o[odd]).any() and np.isfinite(o[~odd]).all()
        v[a + 400, 0, 5] = v[a + 1299, 1, 100] = k[a + 800, 1, 3] = 0
        at = [0, 399, 400, 401, 799, 800, 1298, 1299]
        ref, bound = A.attention64(q[a:][at], k[a:], v[a:], 0.1, at)
        keep = ~odd[a:][at]
        _check(np.where(keep, o[a:][at], 0), np.where(keep, ref, 0), np.where(keep, bound, 1), f"second sequence around {bad}")


PAGED = [  # heads, kv_heads, dim, new, length, rows of a tile by type
    (28, 1, 128, [45], [2200], {A.F32: 256, A.F16: 256, A.BF16: 256}),
    (28, 4, 128, [17, 1, 40, 30] * 3, [900, 1000, 41, 333] * 3, {A.F32: 256, A.F16: 128, A.BF16: 128}),
    (14, 2, 64, [17, 1, 40, 30] * 3, [900, 1000, 41, 333] * 3, {A.F32: 128, A.F16: 128, A.BF16: 128}),
    (32, 1, 40, [190, 150], [400, 1600], {A.F32: 256, A.F16: 256, A.BF16: 256}),
    (28, 4, 128, [4, 3, 5, 4] * 6, [900, 3, 41, 333] * 6, {A.F32: 32, A.F16: 32, A.BF16: 32}),
    (14, 2, 64, [4, 3, 5, 4] * 12, [900, 3, 41, 333] * 12, {A.F32: 32, A.F16: 32, A.BF16: 32}),
    (14, 2, 80, [1, 1, 0, 1, 2], [777, 64, 5, 3000, 129], {A.F32: 16, A.F16: 16, A.BF16: 16}),
]


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim,new,length,rows", PAGED, ids=lambda x: None if isinstance(x, (list, dict)) else str(x))
def test_paged_kernels(qmv, hip, t, heads, kv_heads, dim, new, length, rows):  # noqa: F811
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, 16, seed=dim + len(new))
    assert plan_of(b, heads, kv_heads, dim, t).rows == rows[t]
    o, ok = _paged(qmv, hip, b, q, cache, dim ** -0.5, 4, 8)
    assert ok == 1
    for s, n in enumerate(new):
        if n:
            a, at = int(b.starts[s]), _rows(n)
            pos = b.positions(s)
            ref, bound = A.attention64(q[a:a + n][at], keys[s], values[s], dim ** -0.5, [pos[i] for i in at])
            _check(o[a:a + n][at], ref, bound, f"{A.NAMES[t]} sequence {s} ({n} of {length[s]})")


@pytest.mark.parametrize("t", [A.F16, A.BF16], ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim,count,new,longest,rows,lists", [
    (28, 4, 128, 64, 1, 1000, 16, 0),   # several rounds of workgroups
    (28, 4, 128, 16, 1, 4000, 16, 0),   # one
    (4, 2, 64, 300, 1, 600, 16, 1),     # the pieces listed first
    (14, 2, 64, 64, 4, 700, 32, 0),     # tiles of 32 rows
    (14, 2, 64, 270, 4, 300, 32, 1),
])
def test_paged_alike(qmv, hip, t, heads, kv_heads, dim, count, new, longest, rows, lists):  # noqa: F811
    """Sequences of (nearly) one length, whose pieces are fitted to rounds of
    the workgroups that run at once; every row, and the same bits again."""
    length = [longest - i % 3 for i in range(count)]
    b, q, keys, values, cache = _paged_case(qmv, hip, [new] * count, length, heads, kv_heads, dim, t, 16, seed=31)
    chosen = plan_of(b, heads, kv_heads, dim, t)
    assert (chosen.rows, chosen.slots > 0, chosen.target > 0, chosen.lists) == (rows, True, True, lists)
    o, ok = _paged(qmv, hip, b, q, cache, dim ** -0.5)
    assert ok == 1
    for s in range(count):
        a = s * new
        ref, bound = A.attention64(q[a:a + new], keys[s], values[s], dim ** -0.5, b.positions(s))
        assert (np.abs(o[a:a + new] - ref) <= bound).all(), s
    again, _ = _paged(qmv, hip, b, q, cache, dim ** -0.5)
    assert np.array_equal(o.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("count", [24, 300])
def test_paged_graph_between_alike_and_unlike(qmv, hip, count):  # noqa: F811
    """One captured call, replayed with lengths alike and not: the device finds
    the pieces, and whatever they are, all keys are summed."""
    heads, kv_heads, dim, most = 8, 2, 64, 700
    b, q, keys, values, cache = _paged_case(qmv, hip, [1] * count, [most] * count, heads, kv_heads, dim, A.F16, 16, seed=33)
    assert plan_of(b, heads, kv_heads, dim, A.F16).slots > 0
    rng = np.random.default_rng(34)
    dq, do = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer(q.nbytes)
    seq = b.upload(qmv, hip)
    with hip.Stream() as s:
        qmv.device_attention_paged(dq.ptr, count, heads, 0.125, seq, cache.c, do.ptr, s.handle)
        s.synchronize()
        with hip.Graph(s) as g:
            g.begin()
            qmv.device_attention_paged(dq.ptr, count, heads, 0.125, seq, cache.c, do.ptr, s.handle)
            g.end()
            for step, now in enumerate([[most] * count, [1 + int(x) for x in rng.integers(0, most, count)], [most - i % 2 for i in range(count)],
                                        [1] * count, [most if i == 7 else 3 for i in range(count)]]):
                lens = np.array(now, np.int32)
                hip.check(hip.rt().hipMemcpy(b.d[1].ptr, lens.ctypes.data, lens.nbytes, hip.H2D))
                do.fill(0xFF)
                g.replay()
                s.synchronize()
                o = do.to_array(np.float32, q.shape)
                for i in range(count):
                    ref, bound = A.attention64(q[i:i + 1], keys[i], values[i], 0.125, [now[i] - 1])
                    assert (np.abs(o[i:i + 1] - ref) <= bound).all(), (step, i, now[i])
