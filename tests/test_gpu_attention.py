"""Attention over packed prompts and over a paged cache, and rotary embedding
with the cache write, against 64 bits (tests/_attention.py derives the
bounds)."""
import ctypes

import numpy as np
import pytest

import _attention as A
import _blocks as B

pytestmark = pytest.mark.gpu

MARK = np.float32(-12345.0)


def log(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def hip(qmv, gpu):
    return A.hip_module()


def _rand(rng, *shape, wide=1.0):
    x = rng.standard_normal(shape)
    return (x * np.where(rng.random(shape[-1]) < 0.1, wide, 1.0)).astype(np.float32)


def _check(o, ref, bound, what):
    err = np.abs(o.astype(np.float64) - ref)
    assert np.isfinite(o).all(), f"{what}: not finite"
    worst = np.max(err / np.maximum(bound, 1e-300))
    log(f"{what}: error {np.max(err):.2e}, {worst:.3f} of the bound")
    assert worst <= 1.0, what


def _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, scale, extra=(0, 0, 0), tail=0, stream=0, starts=None):
    """The output [T + tail, heads, dim], rows of `tail` tokens no sequence has
    among them; every row's gap is checked to stay as it was."""
    T = q.shape[0]
    ws, wk = heads * dim, kv_heads * dim
    qs, ks, os_ = ws + extra[0], wk + extra[1], ws + extra[2]
    vs = wk + 2 * extra[1]
    dq = hip.DeviceBuffer.from_array(A.pack(q.reshape(T, ws), qs, ws))
    dk, dv = (hip.DeviceBuffer.from_array(A.pack(x.reshape(T, wk), st, wk)) for x, st in ((k, ks), (v, vs)))
    do = hip.DeviceBuffer.from_array(np.full((T, os_), MARK, np.float32))
    if starts is None:
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    ds = hip.DeviceBuffer.from_array(starts)
    seq = qmv.make_sequences(ds.ptr, len(starts) - 1)
    qmv.device_attention_prompt(dq.ptr, dk.ptr, dv.ptr, T, heads, kv_heads, dim, scale, seq, do.ptr, stream, qs, ks, vs, os_)
    hip.synchronize()
    out = do.to_array(np.float32, (T, os_))
    assert (out[:, ws:] == MARK).all()
    return out[:, :ws].reshape(T, heads, dim)


@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (12, 2, 128), (28, 4, 128), (3, 3, 8), (8, 1, 40), (5, 5, 96),
                                                (16, 2, 120), (33, 1, 16)])
@pytest.mark.parametrize("new", [[1], [37], [0, 1, 65, 0, 2, 130, 17]])
def test_prompt(qmv, hip, heads, kv_heads, dim, new):
    rng = np.random.default_rng(1000 * heads + dim)
    T = sum(new)
    q, k, v = _rand(rng, T, heads, dim, wide=2), _rand(rng, T, kv_heads, dim, wide=3), _rand(rng, T, kv_heads, dim)
    scale = dim ** -0.5
    o = _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, scale, extra=(8, 4, 12))
    t = 0
    for s, n in enumerate(new):
        if n:
            ref, bound = A.attention64(q[t:t + n], k[t:t + n], v[t:t + n], scale, range(n))
            _check(o[t:t + n], ref, bound, f"prompt {heads}/{kv_heads}/{dim} sequence {s} of {n}")
        t += n


@pytest.mark.parametrize("n", [300, 515])
def test_prompt_long(qmv, hip, n):
    rng = np.random.default_rng(n)
    heads, kv_heads, dim = 4, 2, 128
    q, k, v = _rand(rng, n, heads, dim, wide=2), _rand(rng, n, kv_heads, dim, wide=3), _rand(rng, n, kv_heads, dim)
    o = _prompt(qmv, hip, [n], heads, kv_heads, dim, q, k, v, dim ** -0.5)
    ref, bound = A.attention64(q, k, v, dim ** -0.5, range(n))
    _check(o, ref, bound, f"prompt of {n}")


@pytest.mark.parametrize("heads,kv_heads,dim,new", [
    (4, 2, 128, [1100]),              # images of tiles, row tiles of 256
    (2, 1, 104, [1030, 3, 1030]),     # ... of sequences that end inside a tile
    (8, 1, 64, [1025]),               # ... of 64 elements, 8200 rows
    (2, 2, 64, [600, 1, 0, 90]),      # row tiles of 128
    (3, 1, 128, [100, 260]),          # row tiles of 256 without images
])
def test_prompt_shapes(qmv, hip, heads, kv_heads, dim, new):
    """Each kernel that the sizes choose; only some rows are checked against 64
    bits: the first and last of each sequence and of tiles."""
    rng = np.random.default_rng(dim)
    T = sum(new)
    q, k, v = _rand(rng, T, heads, dim, wide=2), _rand(rng, T, kv_heads, dim, wide=3), _rand(rng, T, kv_heads, dim)
    o = _prompt(qmv, hip, new, heads, kv_heads, dim, q, k, v, dim ** -0.5, extra=(4, 8, 4))
    t = 0
    for s, n in enumerate(new):
        if n:
            rows = sorted({i for i in (0, 1, 31, 32, 63, 64, 65, 127, 128, 255, 256, 257, 511, n // 2, n - 65, n - 2, n - 1)
                           if 0 <= i < n} | set(range(0, n, 41)))
            ref, bound = A.attention64(q[t:t + n][rows], k[t:t + n], v[t:t + n], dim ** -0.5, rows)
            _check(o[t:t + n][rows], ref, bound, f"prompt {heads}/{kv_heads}/{dim} sequence {s} of {n}")
        t += n


def test_prompt_images_not_finite(qmv, hip):
    """As test_prompt_not_finite where the keys and values are split first."""
    rng = np.random.default_rng(8)
    n = 1090
    for bad in (np.inf, np.nan):
        q, k, v = _rand(rng, n, 4, 128), _rand(rng, n, 2, 128), _rand(rng, n, 2, 128)
        v[400, 0, 5] = v[700, 0, 5] = v[1089, 1, 100] = bad
        k[800, 1, 3] = np.nan
        o = _prompt(qmv, hip, [n], 4, 2, 128, q, k, v, 0.1)
        odd = np.zeros_like(o, bool)
        odd[400:, :2, 5] = odd[800:, 2:] = True
        assert not np.isfinite(o[odd]).any() and np.isfinite(o[~odd]).all()
        v[400, 0, 5] = v[700, 0, 5] = v[1089, 1, 100] = k[800, 1, 3] = 0
        rows = [0, 399, 400, 401, 700, 799, 800, 1088, 1089]
        ref, bound = A.attention64(q[rows], k, v, 0.1, rows)
        keep = ~odd[rows]
        _check(np.where(keep, o[rows], 0), np.where(keep, ref, 0), np.where(keep, bound, 1), f"images around {bad}")


@pytest.mark.parametrize("count,longest", [(150, 9), (400, 9), (300, 60)])
def test_prompt_many_sequences(qmv, hip, count, longest):
    """As test_paged_many_sequences, some empty."""
    rng = np.random.default_rng(9)
    new = [int(x) for x in rng.integers(0, longest, count)]
    T = sum(new)
    q, k, v = _rand(rng, T, 6, 64), _rand(rng, T, 2, 64), _rand(rng, T, 2, 64)
    o = _prompt(qmv, hip, new, 6, 2, 64, q, k, v, 0.125)
    t = 0
    for n in new:
        if n:
            ref, bound = A.attention64(q[t:t + n], k[t:t + n], v[t:t + n], 0.125, range(n))
            assert (np.abs(o[t:t + n] - ref) <= bound).all()
        t += n


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_prompt_scales(qmv, hip, scale):
    rng = np.random.default_rng(3)
    q, k, v = _rand(rng, 70, 2, 64), _rand(rng, 70, 1, 64), _rand(rng, 70, 1, 64)
    o = _prompt(qmv, hip, [70], 2, 1, 64, q, k, v, scale)
    ref, bound = A.attention64(q, k, v, scale, range(70))
    _check(o, ref, bound, f"scale {scale}")


def test_prompt_leaves_rows_of_no_sequence(qmv, hip):
    """Tokens before the first start, behind the last and between none."""
    rng = np.random.default_rng(4)
    q, k, v = _rand(rng, 50, 4, 64), _rand(rng, 50, 2, 64), _rand(rng, 50, 2, 64)
    o = _prompt(qmv, hip, None, 4, 2, 64, q, k, v, 0.125, starts=np.array([3, 3, 20, 41, 41], np.int32))
    assert (o[:3] == MARK).all() and (o[41:] == MARK).all()
    for a, b in ((3, 20), (20, 41)):
        ref, bound = A.attention64(q[a:b], k[a:b], v[a:b], 0.125, range(b - a))
        _check(o[a:b], ref, bound, f"rows {a}..{b}")


def test_prompt_cuts_starts_to_the_tokens(qmv, hip):
    """Starts that leave the call's tokens, or fall, write nothing outside it."""
    rng = np.random.default_rng(5)
    q, k, v = _rand(rng, 40, 2, 64), _rand(rng, 40, 2, 64), _rand(rng, 40, 2, 64)
    o = _prompt(qmv, hip, None, 2, 2, 64, q, k, v, 0.125, starts=np.array([0, 30, 1000000], np.int32))
    ref, bound = A.attention64(q[:30], k[:30], v[:30], 0.125, range(30))
    _check(o[:30], ref, bound, "before the cut")
    ref, bound = A.attention64(q[30:], k[30:], v[30:], 0.125, range(10))
    _check(o[30:], ref, bound, "cut")


@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 3e4, 1e18, 1e36])
def test_prompt_magnitudes(qmv, hip, magnitude):
    """Values, and keys against queries, far from one; rows of other sizes in
    one tile."""
    rng = np.random.default_rng(6)
    q, k, v = _rand(rng, 90, 2, 64), _rand(rng, 90, 1, 64), _rand(rng, 90, 1, 64)
    m = np.float32(magnitude)
    o = _prompt(qmv, hip, [90], 2, 1, 64, q / m, k * m, v * m, 0.125)
    ref, bound = A.attention64(q / m, k * m, v * m, 0.125, range(90))
    _check(o, ref, bound, f"magnitude {magnitude}")
    grow = (2.0 ** np.linspace(-20, 20, 90)).astype(np.float32)[:, None, None]
    o = _prompt(qmv, hip, [90], 2, 1, 64, q, k, v * grow, 0.125)
    ref, bound = A.attention64(q, k, v * grow, 0.125, range(90))
    _check(o, ref, bound, "values that grow by the token")


def test_prompt_not_finite(qmv, hip):
    """A key or value that is not finite reaches the tokens that attend it and
    no others, nor other heads; a query only its own row."""
    rng = np.random.default_rng(7)
    for bad in (np.inf, -np.inf, np.nan):
        q, k, v = _rand(rng, 100, 4, 64), _rand(rng, 100, 2, 64), _rand(rng, 100, 2, 64)
        v[40, 0, 5] = bad
        k[70, 1, 3] = np.nan
        q[10, 3, 0] = bad
        o = _prompt(qmv, hip, [100], 4, 2, 64, q, k, v, 0.125)
        assert not np.isfinite(o[40:, :2, 5]).any()
        assert np.isnan(o[70:, 2:]).all()
        assert not np.isfinite(o[10, 3]).any()
        clean = np.ones_like(o, bool)
        clean[40:, :2, 5] = clean[70:, 2:] = clean[10, 3] = False
        q[10, 3, 0] = v[40, 0, 5] = k[70, 1, 3] = 0
        ref, bound = A.attention64(q, k, v, 0.125, range(100))
        _check(np.where(clean, o, 0), np.where(clean, ref, 0), np.where(clean, bound, 1), f"around {bad}")


def _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, page, layout="heads", seed=0, tail=0):
    rng = np.random.default_rng(seed)
    b = A.Batch(new, length, page, seed)
    keys = [_rand(rng, max(0, n), kv_heads, dim, wide=3) for n in b.length]
    values = [_rand(rng, max(0, n), kv_heads, dim) for n in b.length]
    keys, values = ([A.decode(A.encode(x, t), t) for x in y] for y in (keys, values))
    q = _rand(rng, b.tokens + tail, heads, dim, wide=2)
    cache = A.Cache(qmv, hip, b, keys, values, t, layout)
    return b, q, keys, values, cache


def _paged(qmv, hip, b, q, cache, scale, q_extra=0, out_extra=0, stream=None):
    T, heads, dim = q.shape
    w = heads * dim
    dq = hip.DeviceBuffer.from_array(A.pack(q.reshape(T, w), w + q_extra, w))
    do = hip.DeviceBuffer.from_array(np.full((T, w + out_extra), MARK, np.float32))
    status = hip.DeviceBuffer.from_array(np.array([1, 77], np.int32))
    seq = b.upload(qmv, hip)
    qmv.device_attention_paged(dq.ptr, T, heads, scale, seq, cache.c, do.ptr, stream.handle if stream else 0, w + q_extra,
                               w + out_extra, status.ptr)
    hip.synchronize()
    out = do.to_array(np.float32, (T, w + out_extra))
    assert (out[:, w:] == MARK).all()
    ok = status.to_array(np.int32, 2)
    assert ok[1] == 77
    return out[:, :w].reshape(T, heads, dim), int(ok[0])


def _check_paged(b, q, keys, values, o, scale, what):
    for s, n in enumerate(b.new):
        if n:
            a = int(b.starts[s])
            ref, bound = A.attention64(q[a:a + n], keys[s], values[s], scale, b.positions(s))
            _check(o[a:a + n], ref, bound, f"{what} sequence {s} ({n} of {b.length[s]})")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim,page,layout", [
    (14, 2, 64, 16, "heads"), (28, 4, 128, 64, "tokens"), (12, 2, 128, 1, "heads"), (6, 3, 40, 48, "wide"),
    (33, 1, 96, 7, "shared"), (4, 4, 8, 256, "tokens")])
@pytest.mark.parametrize("new,length", [([1], [1]), ([1, 1, 0, 1, 1], [300, 64, 0, 129, 2]), ([5, 1, 33, 8], [5, 77, 200, 65])])
def test_paged(qmv, hip, t, heads, kv_heads, dim, page, layout, new, length):
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, page, layout, seed=dim + page)
    o, ok = _paged(qmv, hip, b, q, cache, dim ** -0.5, 4, 8)
    assert ok == 1
    _check_paged(b, q, keys, values, o, dim ** -0.5, f"{A.NAMES[t]} {heads}/{kv_heads}/{dim} page {page} {layout}")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("new,length", [([1], [2500]), ([3, 1], [1777, 1025]), ([40], [1400])])
def test_paged_long(qmv, hip, t, new, length):
    """Few rows over a long axis: the work is cut along it."""
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, 7, 1, 128, t, 32, seed=9)
    o, ok = _paged(qmv, hip, b, q, cache, 128 ** -0.5)
    assert ok == 1
    _check_paged(b, q, keys, values, o, 128 ** -0.5, f"{A.NAMES[t]} long")
    again, _ = _paged(qmv, hip, b, q, cache, 128 ** -0.5)
    assert np.array_equal(o.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim,new,length", [
    (14, 2, 128, [190, 30], [900, 1000]),   # row tiles of 128 or 256, cut along the keys
    (28, 1, 128, [45], [700]),              # 256 rows and more of one key head
    (32, 1, 40, [140], [400]),              # row tiles of 256 of 64 elements
    (8, 8, 64, [3, 20, 1], [2000, 300, 64]),
])
def test_paged_shapes(qmv, hip, t, heads, kv_heads, dim, new, length):
    """Each kernel that the sizes choose; rows as in test_prompt_shapes."""
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, 16, seed=dim)
    o, ok = _paged(qmv, hip, b, q, cache, dim ** -0.5)
    assert ok == 1
    for s, n in enumerate(new):
        a = int(b.starts[s])
        rows = sorted({i for i in (0, 1, 17, 18, 35, 36, 37, n - 2, n - 1) if 0 <= i < n} | set(range(0, n, 23)))
        pos = b.positions(s)
        ref, bound = A.attention64(q[a:a + n][rows], keys[s], values[s], dim ** -0.5, [pos[i] for i in rows])
        _check(o[a:a + n][rows], ref, bound, f"{A.NAMES[t]} {heads}/{kv_heads}/{dim} sequence {s} ({n} of {length[s]})")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim,count,longest", [(28, 4, 128, 24, 700), (14, 2, 64, 60, 200), (6, 1, 40, 12, 5000)])
def test_paged_few_tokens_each(qmv, hip, t, heads, kv_heads, dim, count, longest):
    """Sequences of 17 to 32 rows on average, as when a few drafted tokens are
    checked at once: some idle, some of one token, some of several row tiles,
    one that stands partly before its first key, and a value that is not
    finite, which only the rows that attend it may see."""
    rng = np.random.default_rng(21)
    new = [int(x) for x in rng.choice([4, 4, 4, 3, 5, 1, 0, 9], count)]
    new[:4] = [5, 4, 9, 4]
    length = [int(n + x) for n, x in zip(new, rng.integers(0, longest, count))]
    length[0], length[1], length[2] = longest, 2, 9
    assert 17 <= sum(new) * (heads // kv_heads) / count <= 32
    b, q, keys, values, _ = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, 16, seed=22)
    odd = [x.copy() for x in values]
    odd[3][length[3] - 2, 0, 5] = np.inf  # the third of four new tokens
    o, ok = _paged(qmv, hip, b, q, A.Cache(qmv, hip, b, keys, odd, t), dim ** -0.5, 4, 8)
    assert ok == 1
    a, first = int(b.starts[3]), heads // kv_heads
    assert not np.isfinite(o[a + 2:a + 4, :first, 5]).any()
    ref, _ = A.attention64(q[a + 2:a + 4], keys[3], values[3], dim ** -0.5, b.positions(3)[2:])
    o[a + 2:a + 4, :first, 5] = ref[:, :first, 5]
    assert (o[int(b.starts[1]):int(b.starts[1]) + 2] == 0).all()
    _check_paged(b, q, keys, values, o, dim ** -0.5, f"{A.NAMES[t]} {heads}/{kv_heads}/{dim}")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,dim", [(28, 4, 128), (14, 2, 64), (6, 1, 40)])
def test_paged_decoding_beside_chunks(qmv, hip, t, heads, kv_heads, dim):
    """A step of a server: chunks of prompts and decoding sequences in one call,
    with a value that is not finite, which only the second of two tokens sees."""
    new, length = [60, 1, 0, 2, 20, 1, 1, 4], [400, 4000, 5, 700, 40, 1, 1290, 31]
    b, q, keys, values, _ = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, 16, seed=23)
    odd = [x.copy() for x in values]
    odd[3][699, 0, 5] = np.nan
    o, ok = _paged(qmv, hip, b, q, A.Cache(qmv, hip, b, keys, odd, t), dim ** -0.5, 4, 8)
    assert ok == 1
    a, group = int(b.starts[3]) + 1, heads // kv_heads
    assert np.isnan(o[a, :group, 5]).all()
    ref, _ = A.attention64(q[a:a + 1], keys[3], values[3], dim ** -0.5, [699])
    o[a, :group, 5] = ref[0, :group, 5]
    _check_paged(b, q, keys, values, o, dim ** -0.5, f"{A.NAMES[t]} {heads}/{kv_heads}/{dim}")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("heads,kv_heads,new,length", [
    (28, 4, [240] + [1] * 60, [240] + [(37 * i) % 700 + 1 for i in range(60)]),  # decoding beside a prompt
    (28, 4, [6] * 60, [500 + i % 9 for i in range(60)]),                         # all alike
    (28, 4, [600, 1, 2], [700, 2500, 1200]),                                     # tiles of 256 rows
    (28, 4, [900] + [1] * 20, [900] + [90 * i + 1 for i in range(20)]),          # of fp32 alone
    (7, 1, [5] * 300, [5 + 7 * i % 90 for i in range(300)]),                     # more than workgroups look through themselves
])
def test_paged_many_tiles(qmv, hip, t, heads, kv_heads, new, length):
    """Tiles of 128 or 256 rows that are nearly as many as the workgroups at once,
    decoding sequences among them."""
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, heads, kv_heads, 128, t, 16, seed=24)
    o, ok = _paged(qmv, hip, b, q, cache, 128 ** -0.5)
    assert ok == 1
    for s, n in enumerate(new):
        a, rows = int(b.starts[s]), sorted({0, 17, 18, 36, n // 2, n - 1} & set(range(n)))
        pos = b.positions(s)
        ref, bound = A.attention64(q[a:a + n][rows], keys[s], values[s], 128 ** -0.5, [pos[i] for i in rows])
        assert (np.abs(o[a:a + n][rows] - ref) <= bound).all(), (s, n, length[s])
    again, _ = _paged(qmv, hip, b, q, cache, 128 ** -0.5)
    assert np.array_equal(o.view(np.uint32), again.view(np.uint32))


@pytest.mark.parametrize("count,longest", [(139, 200), (257, 40), (2500, 30)])
def test_paged_many_sequences(qmv, hip, count, longest):
    """More sequences than a wave has lanes, or than workgroups look through
    themselves; some idle, one far longer."""
    rng = np.random.default_rng(18)
    length = [int(x) for x in rng.integers(1, longest, count)]
    length[70] = 1500
    new = [int(rng.random() < 0.8) for _ in length]
    b, q, keys, values, cache = _paged_case(qmv, hip, new, length, 4, 2, 64, A.F16, 16, seed=19)
    o, ok = _paged(qmv, hip, b, q, cache, 0.125)
    assert ok == 1
    for s, n in enumerate(new):
        if n:
            a = int(b.starts[s])
            ref, bound = A.attention64(q[a:a + 1], keys[s], values[s], 0.125, [length[s] - 1])
            assert (np.abs(o[a:a + 1] - ref) <= bound).all(), s


def test_starts_that_fall_stay_inside(qmv, hip):
    """Starts that do not rise: no row outside the call's is written, and the
    call ends (every index is compared with the call's sizes)."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [10, 10, 10], [50, 60, 70], 4, 2, 64, A.F16, 16, seed=20)
    table, length = b.table, b.length
    falling = [int(x) for x in np.random.default_rng(2).integers(-9, 40, 301)]
    for starts in ([0, 30, 10, 25], [-5, 100, -5, 100], [30, 20, 10, 0], falling):
        b.starts = np.array(starts, np.int32)
        times = -(-(len(starts) - 1) // 3)
        b.new, b.length, b.table = [0] * (len(starts) - 1), (length * times)[:len(starts) - 1], np.concatenate([table] * times)
        o, _ = _paged(qmv, hip, b, q, cache, 0.125, 4, 4)
        assert o.shape == q.shape
        k = _rand(np.random.default_rng(1), 30, 2, 64)
        _prompt(qmv, hip, None, 4, 2, 64, q, k, k, 0.125, extra=(4, 4, 4), starts=b.starts)


def test_paged_rows_that_attend_nothing(qmv, hip):
    """More new tokens than the length says: zeros at negative positions; idle
    sequences; tokens behind the last sequence stay as they were."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [4, 0, 3, 2], [2, 5, 0, -3], 4, 2, 64, A.F16, 16, seed=11, tail=6)
    o, ok = _paged(qmv, hip, b, q, cache, 0.125)
    assert ok == 1
    assert (o[:2] == 0).all() and (o[4:9] == 0).all() and (o[9:] == MARK).all()
    ref, bound = A.attention64(q[2:4], keys[0], values[0], 0.125, [0, 1])
    _check(o[2:4], ref, bound, "the two that stand somewhere")


@pytest.mark.parametrize("bad", [-1, 1 << 30, None])
@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
def test_paged_bad_pages(qmv, hip, bad, t):
    """A page outside the cache, or a length outside the table: the rows that
    attend it are NaN, others keep their values, and the status says so. No
    address of such a page is read: the number is compared with the cache's
    pages first (bounds that the kernel checks itself)."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [1, 40, 1], [200, 120, 50], 4, 2, 64, t, 16, seed=12)
    if bad is None:
        b.length[0] = b.columns * 16 + 500  # past the table
        b.table[0, :] = b.table[0, 0]
    else:
        b.table[0, 3] = bad
        b.table[1, 6] = bad  # positions 96..111, new tokens 16..31: 16.. attend it
    o, ok = _paged(qmv, hip, b, q, cache, 0.125)
    assert ok == 0
    assert np.isnan(o[0]).all()
    ref, bound = A.attention64(q[41:], keys[2], values[2], 0.125, b.positions(2))
    _check(o[41:], ref, bound, "another sequence")
    n = 40 if bad is None else 16
    ref, bound = A.attention64(q[1:1 + n], keys[1], values[1], 0.125, b.positions(1)[:n])
    _check(o[1:1 + n], ref, bound, "rows before the page")
    assert bad is None or np.isnan(o[17:41]).all()


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
def test_paged_not_finite(qmv, hip, t):
    """As test_prompt_not_finite, a chunk of new tokens over a cache."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [60], [150], 4, 2, 64, t, 16, seed=13)
    for bad in (np.inf, np.nan):
        k2, v2 = keys[0].copy(), values[0].copy()
        v2[120, 0, 9] = bad  # new token 30
        k2[130, 1, 0] = np.nan
        c2 = A.Cache(qmv, hip, b, [k2], [v2], t)
        o, _ = _paged(qmv, hip, b, q, c2, 0.125)
        clean = np.ones_like(o, bool)
        clean[30:, :2, 9] = clean[40:, 2:] = False
        assert not np.isfinite(o[30:, :2, 9]).any() and np.isnan(o[40:, 2:]).all()
        ref, bound = A.attention64(q, keys[0], values[0], 0.125, b.positions(0))
        _check(np.where(clean, o, 0), np.where(clean, ref, 0), np.where(clean, bound, 1), f"{A.NAMES[t]} around {bad}")


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
def test_paged_magnitudes(qmv, hip, t):
    rng = np.random.default_rng(14)
    for m in (1e-4, 1e3) if t == A.F16 else (1e-30, 1e4, 1e30):
        b = A.Batch([1, 20], [200, 100], 16, 1)
        keys = [A.decode(A.encode(_rand(rng, n, 2, 64) * np.float32(m), t), t) for n in b.length]
        values = [A.decode(A.encode(_rand(rng, n, 2, 64) * np.float32(m), t), t) for n in b.length]
        q = _rand(rng, b.tokens, 4, 64) / np.float32(m)
        cache = A.Cache(qmv, hip, b, keys, values, t)
        o, ok = _paged(qmv, hip, b, q, cache, 0.125)
        assert ok == 1
        _check_paged(b, q, keys, values, o, 0.125, f"{A.NAMES[t]} magnitude {m}")


def test_paged_shared_pages(qmv, hip):
    """Sequences that begin alike read the same pages."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [1, 2, 1], [64, 64, 64], 4, 2, 64, A.F16, 16, seed=15)
    b.table[1, :4] = b.table[0, :4]
    b.table[2, :3] = b.table[0, :3]
    keys[1], values[1] = keys[0], values[0]
    for x in (keys, values):
        x[2] = np.concatenate([x[0][:48], x[2][48:]])
    o, ok = _paged(qmv, hip, b, q, cache, 0.125)
    assert ok == 1
    _check_paged(b, q, keys, values, o, 0.125, "shared pages")


def test_paged_far_offsets(qmv, hip):
    """Pages whose elements lie beyond 2^31 of the cache's first."""
    dim, hk, page, stride = 64, 1, 16, (1 << 31) + 64
    rng = np.random.default_rng(16)
    k, v = (_rand(rng, 24, hk, dim).astype(np.float16) for _ in range(2))
    bufs = [hip.DeviceBuffer(2 * (stride + page * dim)) for _ in range(2)]
    for buf, a in zip(bufs, (k, v)):
        full = np.zeros((2, page, dim), np.float16)
        full.reshape(32, dim)[:24] = a[:, 0]
        for p, at in ((0, stride), (1, 0)):  # the sequence's first page is the far one
            part = np.ascontiguousarray(full[p])
            hip.check(hip.rt().hipMemcpy(buf.ptr + 2 * at, part.ctypes.data, part.nbytes, hip.H2D))
    b = A.Batch([2], [24], page)
    b.table = np.array([[1, 0]], np.int32)
    b.columns = 2
    seq = b.upload(qmv, hip)
    q = _rand(rng, 2, 2, dim)
    dq, do = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer(q.nbytes)
    c = qmv.make_paged_cache(bufs[0].ptr, bufs[1].ptr, A.F16, hk, dim, page, 2, stride, page * dim, dim)
    qmv.device_attention_paged(dq.ptr, 2, 2, 0.125, seq, c, do.ptr)
    hip.synchronize()
    ref, bound = A.attention64(q, k.astype(np.float32), v.astype(np.float32), 0.125, [22, 23])
    _check(do.to_array(np.float32, q.shape), ref, bound, "far pages")


def test_paged_graph_and_streams(qmv, hip):
    """A captured call, replayed with other lengths and queries between eager
    calls of the same stream; another stream at the same time."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [1, 1, 1], [900, 333, 1200], 14, 2, 64, A.F16, 16, seed=17)
    scale = 0.125
    dq, do = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer(q.nbytes)
    do2 = hip.DeviceBuffer(q.nbytes)
    seq = b.upload(qmv, hip)
    lengths = b.d[1]
    with hip.Stream() as s, hip.Stream() as other:
        qmv.device_attention_paged(dq.ptr, 3, 14, scale, seq, cache.c, do.ptr, s.handle)
        s.synchronize()
        _check_paged(b, q, keys, values, do.to_array(np.float32, q.shape), scale, "eager")
        with hip.Graph(s) as g:
            g.begin()
            qmv.device_attention_paged(dq.ptr, 3, 14, scale, seq, cache.c, do.ptr, s.handle)
            g.end()
            for step, now in enumerate([[900, 333, 1200], [1, 300, 1199], [0, 64, 65], [700, 2, 1000]]):
                b.length = now
                lens = np.array(now, np.int32)
                hip.check(hip.rt().hipMemcpy(lengths.ptr, lens.ctypes.data, lens.nbytes, hip.H2D))
                do.fill(0xFF)
                g.replay()
                qmv.device_attention_paged(dq.ptr, 3, 14, scale, seq, cache.c, do2.ptr, other.handle)
                s.synchronize()
                other.synchronize()
                o, o2 = do.to_array(np.float32, q.shape), do2.to_array(np.float32, q.shape)
                assert np.array_equal(o.view(np.uint32), o2.view(np.uint32)), f"replay {step}"
                for i in range(3):
                    if now[i] == 0:
                        assert (o[i] == 0).all()
                    else:
                        ref, bound = A.attention64(q[i:i + 1], keys[i], values[i], scale, [now[i] - 1])
                        _check(o[i:i + 1], ref, bound, f"replay {step} sequence {i}")


def test_workspace(qmv, hip):
    """A call that would have to grow its workspace in a capture is refused; a
    graph stays right after a larger call has replaced the workspace; a size that
    ran before allocates nothing."""
    b, q, keys, values, cache = _paged_case(qmv, hip, [1, 1], [700, 1300], 14, 2, 64, A.F16, 16, seed=21)
    dq, do = hip.DeviceBuffer.from_array(q), hip.DeviceBuffer(q.nbytes)
    seq = b.upload(qmv, hip)
    rng = np.random.default_rng(22)
    T = 1200
    x = [_rand(rng, T, h, 64) for h in (14, 2, 2)]
    dx = [hip.DeviceBuffer.from_array(a) for a in x]
    dxo = hip.DeviceBuffer(x[0].nbytes)
    dstarts = hip.DeviceBuffer.from_array(np.array([0, T], np.int32))
    prompt = qmv.make_sequences(dstarts.ptr, 1)
    far = [hip.DeviceBuffer(4 * 60000 * 256) for _ in range(4)]  # more than any test needs
    with hip.Stream() as s:
        with hip.Graph(s) as refused:
            refused.begin()
            with pytest.raises(qmv.QmvError, match="workspace"):
                qmv.device_attention_prompt(far[0].ptr, far[1].ptr, far[2].ptr, 60000, 2, 2, 128, 0.125, prompt, far[3].ptr,
                                            s.handle)
            refused.end()
        qmv.device_attention_paged(dq.ptr, 2, 14, 0.125, seq, cache.c, do.ptr, s.handle)
        s.synchronize()
        first = do.to_array(np.uint32, q.shape)
        with hip.Graph(s) as g:
            g.begin()
            qmv.device_attention_paged(dq.ptr, 2, 14, 0.125, seq, cache.c, do.ptr, s.handle)
            g.end()
            for i in range(3):
                qmv.device_attention_prompt(dx[0].ptr, dx[1].ptr, dx[2].ptr, T, 14, 2, 64, 0.125, prompt, dxo.ptr, s.handle)
                do.fill(0xFF)
                g.replay()
                s.synchronize()
                assert np.array_equal(do.to_array(np.uint32, q.shape), first), f"replay {i}"
                count = qmv.allocation_count() if i == 0 else count
            assert qmv.allocation_count() == count
    ref, bound = A.attention64(x[0][::97], x[1], x[2], 0.125, list(range(T))[::97])
    _check(dxo.to_array(np.float32, x[0].shape)[::97], ref, bound, "the larger call")


def test_graph_of_a_step(qmv, hip):
    """Rotary embedding, cache write and both attentions in one graph, replayed
    with other queries and positions between eager work, against eager calls on
    another stream with a cache of its own."""
    rng = np.random.default_rng(23)
    heads, kv_heads, dim, page, n = 14, 2, 64, 16, 24
    b = A.Batch([n, 1], [n, 400], page, 6)
    filled = [_rand(rng, m, kv_heads, dim) for m in (n + 40, 440)]
    big = A.Batch([0, 0], [n + 40, 440], page, 6)
    caches = [A.Cache(qmv, hip, big, filled, filled, A.BF16) for _ in range(2)]
    b.table, b.columns = big.table, big.columns
    seq = b.upload(qmv, hip)
    T = b.tokens
    d = [hip.DeviceBuffer(4 * T * w) for w in (heads * dim, kv_heads * dim, kv_heads * dim)]
    outs = [[hip.DeviceBuffer(4 * T * w) for w in (heads * dim, kv_heads * dim, heads * dim, heads * dim)] for _ in range(2)]
    f = hip.DeviceBuffer.from_array(A.frequencies(dim))

    def step(which, stream):
        q, k, o, p = (x.ptr for x in outs[which])
        qmv.device_rope_append(d[0].ptr, heads, d[1].ptr, d[2].ptr, kv_heads, dim, T, f.ptr, dim, seq, q, k, caches[which].c,
                               stream=stream.handle)
        qmv.device_attention_paged(q, T, heads, 0.125, seq, caches[which].c, o, stream.handle)
        qmv.device_attention_prompt(q, k, d[2].ptr, T, heads, kv_heads, dim, 0.125, seq, p, stream.handle)

    with hip.Stream() as s, hip.Stream() as other:
        step(0, s)
        s.synchronize()
        with hip.Graph(s) as g:
            g.begin()
            step(0, s)
            g.end()
            for i in range(4):
                for x in d:
                    a = rng.standard_normal(x.nbytes // 4).astype(np.float32)
                    hip.check(hip.rt().hipMemcpy(x.ptr, a.ctypes.data, x.nbytes, hip.H2D))
                lens = np.array([n + 10 * i, 400 + 9 * i], np.int32)
                hip.check(hip.rt().hipMemcpy(b.d[1].ptr, lens.ctypes.data, 8, hip.H2D))
                g.replay()
                step(1, other)
                s.synchronize()
                other.synchronize()
                for x, y in zip(*outs):
                    assert np.array_equal(x.to_array(np.uint32, x.nbytes // 4), y.to_array(np.uint32, y.nbytes // 4)), i
                for which in (0, 1):
                    assert np.array_equal(caches[0].read(which), caches[1].read(which))


def test_threads_on_their_own_streams(qmv, hip):
    """Two host threads with a stream each, many calls at once."""
    import threading
    cases = [_paged_case(qmv, hip, [1, 2], [900, 500 + 300 * i], 14, 2, 64, A.F16, 16, seed=30 + i) for i in range(2)]
    bufs = [(hip.DeviceBuffer.from_array(c[1]), hip.DeviceBuffer(c[1].nbytes), c[0].upload(qmv, hip)) for c in cases]
    expected, failures = [], []
    for (b, q, keys, values, cache), (dq, do, seq) in zip(cases, bufs):
        qmv.device_attention_paged(dq.ptr, 3, 14, 0.125, seq, cache.c, do.ptr)
        hip.synchronize()
        expected.append(do.to_array(np.uint32, q.shape))

    def work(i):
        try:
            (b, q, keys, values, cache), (dq, do, seq) = cases[i], bufs[i]
            with hip.Stream() as s:
                for _ in range(30):
                    do.fill(0)
                    qmv.device_attention_paged(dq.ptr, 3, 14, 0.125, seq, cache.c, do.ptr, s.handle)
                    s.synchronize()
                    if not np.array_equal(do.to_array(np.uint32, q.shape), expected[i]):
                        failures.append(i)
        except Exception as e:  # noqa: BLE001
            failures.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert failures == []


# ---- rotary embedding and the cache write ------------------------------------------

def _rope_bound(x):
    """The angle's rest is rounded to fp32 (at most 2^-22.3 absolute, see the
    kernel), sine and cosine to 2 steps of fp32, products and their sum to half
    a step each: under 2^-21 of |x| + |y|, whose largest is twice max |x|."""
    return 2.0 ** -21 * 2 * np.max(np.abs(x)) + 2.0 ** -140


@pytest.mark.parametrize("t", A.TYPES + [None], ids=lambda t: A.NAMES.get(t, "none"))
@pytest.mark.parametrize("heads,kv_heads,dim,rotary,page,layout", [
    (14, 2, 64, 64, 16, "heads"), (28, 4, 128, 128, 64, "tokens"), (3, 1, 40, 24, 1, "wide"), (5, 5, 8, 0, 7, "heads")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append(qmv, hip, t, heads, kv_heads, dim, rotary, page, layout, interleaved):
    rng = np.random.default_rng(20 + dim)
    b = A.Batch([1, 0, 5, 17, 2], [1000, 0, 5, 40, 1], page, 3)
    T = b.tokens + 4
    q, k, v = _rand(rng, T, heads, dim, wide=4), _rand(rng, T, kv_heads, dim, wide=4), _rand(rng, T, kv_heads, dim)
    f = A.frequencies(rotary)
    qs, ks = heads * dim + 4, kv_heads * dim + 8
    dq, dk, dv = (hip.DeviceBuffer.from_array(A.pack(x.reshape(T, -1), st, w)) for x, st, w in
                  ((q, qs, heads * dim), (k, ks, kv_heads * dim), (v, ks, kv_heads * dim)))
    dqo, dko = (hip.DeviceBuffer.from_array(np.full((T, st), MARK, np.float32)) for st in (qs, ks))
    df = hip.DeviceBuffer.from_array(f if rotary else np.zeros(1))
    status = hip.DeviceBuffer.from_array(np.array([1], np.int32))
    seq = b.upload(qmv, hip)
    cache = None
    if t is not None:
        blank = [np.full((max(0, n), kv_heads, dim), np.nan, np.float32) for n in b.length]
        cache = A.Cache(qmv, hip, b, blank, blank, t, layout)
        before = [cache.read(0), cache.read(1)]
    qmv.device_rope_append(dq.ptr, heads, dk.ptr, dv.ptr, kv_heads, dim, T, df.ptr if rotary else 0, rotary, seq, dqo.ptr,
                           dko.ptr, cache.c if cache else None, interleaved, status.ptr, 0, qs, ks, ks)
    hip.synchronize()
    assert status.to_array(np.int32, 1)[0] == 1
    qo, ko = dqo.to_array(np.float32, (T, qs)), dko.to_array(np.float32, (T, ks))
    assert (qo[:, heads * dim:] == MARK).all() and (ko[:, kv_heads * dim:] == MARK).all()
    assert (qo[b.tokens:] == MARK).all() and (ko[b.tokens:] == MARK).all()
    for s, n in enumerate(b.new):
        for i, pos in enumerate(b.positions(s)):
            a = int(b.starts[s]) + i
            for x, o, h in ((q[a], qo[a], heads), (k[a], ko[a], kv_heads)):
                y = o[:h * dim].reshape(h, dim)
                ref = A.rope64(x, pos, f, interleaved)
                assert np.max(np.abs(y - ref)) <= _rope_bound(x), (s, i)
                assert np.array_equal(y[:, rotary:], x[:, rotary:])
            if cache is not None and pos >= 0:
                for which, rows in ((0, ko[a, :kv_heads * dim].reshape(kv_heads, dim)), (1, v[a])):
                    for h in range(kv_heads):
                        before[which][cache.at(s, pos, h)] = A.encode(rows[h], t)
    if cache is not None:
        for which in (0, 1):
            after = cache.read(which)
            assert np.array_equal(after.view(np.uint8), before[which].view(np.uint8)), "codes, and all else as it was"


def test_rows_of_one_buffer(qmv, hip):
    """q, k and v of a token side by side in one row, turned in place, without a
    cache, and attended from there."""
    rng = np.random.default_rng(24)
    heads, kv_heads, dim, T = 6, 2, 64, 90
    wide = (heads + 2 * kv_heads) * dim
    rows = _rand(rng, T, wide)
    d = hip.DeviceBuffer.from_array(rows)
    do = hip.DeviceBuffer(4 * T * heads * dim)
    df, ds = hip.DeviceBuffer.from_array(A.frequencies(dim)), hip.DeviceBuffer.from_array(np.array([0, 30, T], np.int32))
    seq = qmv.make_sequences(ds.ptr, 2)
    k, v = d.ptr + 4 * heads * dim, d.ptr + 4 * (heads + kv_heads) * dim
    qmv.device_rope_append(d.ptr, heads, k, 0, kv_heads, dim, T, df.ptr, dim, seq, d.ptr, k, q_stride=wide, k_stride=wide)
    qmv.device_attention_prompt(d.ptr, k, v, T, heads, kv_heads, dim, 0.125, seq, do.ptr, 0, wide, wide, wide)
    hip.synchronize()
    turned, o = d.to_array(np.float32, rows.shape), do.to_array(np.float32, (T, heads, dim))
    assert np.array_equal(turned[:, (heads + kv_heads) * dim:], rows[:, (heads + kv_heads) * dim:])
    for t in range(T):
        x = rows[t, :(heads + kv_heads) * dim].reshape(-1, dim)
        ref = A.rope64(x, t if t < 30 else t - 30, A.frequencies(dim), False)
        assert np.max(np.abs(turned[t, :(heads + kv_heads) * dim].reshape(-1, dim) - ref)) <= _rope_bound(x)
    parts = turned.reshape(T, -1, dim)
    for a, b in ((0, 30), (30, T)):
        ref, bound = A.attention64(parts[a:b, :heads], parts[a:b, heads:heads + kv_heads], parts[a:b, heads + kv_heads:], 0.125,
                                   range(b - a))
        _check(o[a:b], ref, bound, f"rows {a}..{b}")


@pytest.mark.parametrize("position", [0, 131071, 4000000, 2000000000])
def test_rope_far_positions(qmv, hip, position):
    rng = np.random.default_rng(21)
    q, k = _rand(rng, 1, 2, 128), _rand(rng, 1, 1, 128)
    f = A.frequencies(128)
    dq, dk, df = (hip.DeviceBuffer.from_array(x) for x in (q, k, f))
    ds = [hip.DeviceBuffer.from_array(np.array(x, np.int32)) for x in ([0, 1], [position + 1])]
    seq = qmv.make_sequences(ds[0].ptr, 1, ds[1].ptr)
    qmv.device_rope_append(dq.ptr, 2, dk.ptr, 0, 1, 128, 1, df.ptr, 128, seq, dq.ptr, dk.ptr)  # in place
    hip.synchronize()
    for d, x in ((dq, q), (dk, k)):
        # the product position * frequency is rounded to 64 bits on both sides: 2^-53 of at most 2^31
        assert np.max(np.abs(d.to_array(np.float32, x.shape)[0] - A.rope64(x[0], position, f, False))) <= _rope_bound(x) + 2.0 ** -21


def test_rope_bad_pages(qmv, hip):
    """Nothing is stored where the page is outside the cache or the table."""
    for bad in (-1, 1 << 30, None):
        b = A.Batch([2, 1, 1], [20, 9, 9], 16, 4)
        blank = [np.full((n, 1, 64), np.nan, np.float32) for n in b.length]
        cache = A.Cache(qmv, hip, b, blank, blank, A.F32)
        before = [cache.read(0), cache.read(1)]
        if bad is None:
            b.length[0] = 16 * b.columns + 30
        else:
            b.table[0, 1] = bad
        rng = np.random.default_rng(22)
        q, k, v = _rand(rng, 4, 2, 64), _rand(rng, 4, 1, 64), _rand(rng, 4, 1, 64)
        dq, dk, dv, df = (hip.DeviceBuffer.from_array(x) for x in (q, k, v, A.frequencies(64)))
        status = hip.DeviceBuffer.from_array(np.array([1], np.int32))
        seq = b.upload(qmv, hip)
        qmv.device_rope_append(dq.ptr, 2, dk.ptr, dv.ptr, 1, 64, 4, df.ptr, 64, seq, dq.ptr, 0, cache.c, d_status=status.ptr)
        hip.synchronize()
        assert status.to_array(np.int32, 1)[0] == 0
        for s in (1, 2):
            a = int(b.starts[s])
            before[1][cache.at(s, 8, 0)] = v[a, 0]
            got = cache.read(0)[cache.at(s, 8, 0)]
            assert np.max(np.abs(got - A.rope64(k[a], 8, A.frequencies(64), False)[0])) <= _rope_bound(k[a])
            before[0][cache.at(s, 8, 0)] = got
        for which in (0, 1):
            assert np.array_equal(cache.read(which).view(np.uint32), before[which].view(np.uint32))


# ---- a run of them together ----------------------------------------------------------

@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
def test_attention_block_of_a_layer(qmv, oracle, hip, t):
    """Norm and q|k|v projections, rotary embedding into the cache, attention
    and the output projection with the residual: two sequences in chunks and
    then token by token, against 64 bits from the rows the projections wrote;
    the first chunks also as whole prompts."""
    heads, kv_heads, dim, hidden, page = 14, 2, 64, 896, 16
    shapes = [(hidden, hidden), (kv_heads * dim, hidden), (kv_heads * dim, hidden), (hidden, hidden)]
    raws = [qmv.synth_tensor(B.Q8_0, r, c, seed=50 + i) for i, (r, c) in enumerate(shapes)]
    wq, wk, wv, wo = (qmv.DeviceTensor(qmv.make_view(raw, B.Q8_0, r, c)) for raw, (r, c) in zip(raws, shapes))
    rng = np.random.default_rng(30)
    norm = hip.DeviceBuffer.from_array((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32))
    f = A.frequencies(dim)
    df = hip.DeviceBuffer.from_array(f)
    full = [61, 40]  # the lengths at the end
    whole = A.Batch([0, 0], full, page, 5)
    blank = [np.zeros((n, kv_heads, dim), np.float32) for n in full]
    cache = A.Cache(qmv, hip, whole, blank, blank, t)
    keys, values = [np.zeros((0, kv_heads, dim), np.float32)] * 2, [np.zeros((0, kv_heads, dim), np.float32)] * 2
    have = [0, 0]
    for new in ([20, 12], [11, 0], [1, 1], [28, 1], [1, 0], [0, 26]):
        for s in (0, 1):
            have[s] += new[s]
        step = A.Batch(new, list(have), page)
        step.table, step.columns = whole.table, whole.columns
        seq = step.upload(qmv, hip)
        T = step.tokens
        x = rng.standard_normal((T, hidden)).astype(np.float32)
        dx = hip.DeviceBuffer.from_array(x)
        dq, dk, dv, dn, datt = (hip.DeviceBuffer(4 * T * w) for w in (hidden, 128, 128, hidden, hidden))
        qmv.device_rms_norm_matvec_add_group([wq, wk, wv], dx.ptr, norm.ptr, 1e-6, T, None, None, [dq.ptr, dk.ptr, dv.ptr],
                                             dn.ptr)
        hip.synchronize()
        q, k, v = (d.to_array(np.float32, (T, h, dim)) for d, h in ((dq, heads), (dk, kv_heads), (dv, kv_heads)))
        qmv.device_rope_append(dq.ptr, heads, dk.ptr, dv.ptr, kv_heads, dim, T, df.ptr, dim, seq, dq.ptr, dk.ptr, cache.c)
        qmv.device_attention_paged(dq.ptr, T, heads, dim ** -0.5, seq, cache.c, datt.ptr)
        hip.synchronize()
        att = datt.to_array(np.float32, (T, heads, dim))
        qr, kr = dq.to_array(np.float32, q.shape), dk.to_array(np.float32, k.shape)
        for s in (0, 1):
            a, e = int(step.starts[s]), int(step.starts[s + 1])
            for i, pos in enumerate(step.positions(s)):
                assert np.max(np.abs(qr[a + i] - A.rope64(q[a + i], pos, f, False))) <= _rope_bound(q[a + i])
                assert np.max(np.abs(kr[a + i] - A.rope64(k[a + i], pos, f, False))) <= _rope_bound(k[a + i])
            keys[s] = np.concatenate([keys[s], A.decode(A.encode(kr[a:e], t), t)])
            values[s] = np.concatenate([values[s], A.decode(A.encode(v[a:e], t), t)])
        _check_paged(step, qr, keys, values, att, dim ** -0.5, f"{A.NAMES[t]} step {new}")
        if have == new:
            dp = hip.DeviceBuffer(att.nbytes)
            qmv.device_attention_prompt(dq.ptr, dk.ptr, dv.ptr, T, heads, kv_heads, dim, dim ** -0.5, seq, dp.ptr)
            hip.synchronize()
            p = dp.to_array(np.float32, att.shape)
            for s in (0, 1):
                a, e = int(step.starts[s]), int(step.starts[s + 1])
                ref, bound = A.attention64(qr[a:e], kr[a:e], v[a:e], dim ** -0.5, range(e - a))
                _check(p[a:e], ref, bound, f"as prompts, sequence {s}")
        qmv.device_matvec_add_group([wo], datt.ptr, T, [dx.ptr], [hidden], [dx.ptr])
        hip.synchronize()
        y = dx.to_array(np.float32, x.shape)
        for i in range(T):
            ref = oracle.matvec(raws[3], B.Q8_0, hidden, hidden, att[i].reshape(-1))
            _, absdot = oracle.row_stats(raws[3], B.Q8_0, hidden, hidden, att[i].reshape(-1))
            assert (np.abs(y[i] - (ref.astype(np.float64) + x[i])) <= 1e-5 * absdot + 2.0 ** -24 * np.abs(y[i])).all()
    for w in (wq, wk, wv, wo):
        w.close()
