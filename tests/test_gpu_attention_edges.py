"""Calls of the operators between the projections that the documentation allows
at its edges, against 64 bits."""
import threading

import numpy as np
import pytest

import _attention as A
import _blocks as B
from _attention_plan import plan
from test_gpu_attention import _paged, _paged_case, _prompt, _rand, _rope_bound, hip  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- rotary embedding ------------------------------------------------------------------


@pytest.mark.parametrize("with_lengths", [False, True])
def test_rope_cuts_starts_to_the_tokens(qmv, hip, with_lengths):  # noqa: F811
    """A first start below zero is cut to zero and a last one to the tokens, as
    attention cuts them: without lengths, positions count from the cut."""
    rng = np.random.default_rng(40)
    T, heads, dim = 12, 2, 64
    q, k = _rand(rng, T, heads, dim), _rand(rng, T, 1, dim)
    f = A.frequencies(dim)
    dq, dk, df = (hip.DeviceBuffer.from_array(x) for x in (q, k, f))
    qo, ko = hip.DeviceBuffer(q.nbytes), hip.DeviceBuffer(k.nbytes)
    ds = hip.DeviceBuffer.from_array(np.array([-3, 7, 1000], np.int32))
    dl = hip.DeviceBuffer.from_array(np.array([50, 9], np.int32))
    seq = qmv.make_sequences(ds.ptr, 2, dl.ptr if with_lengths else 0)
    qmv.device_rope_append(dq.ptr, heads, dk.ptr, 0, 1, dim, T, df.ptr, dim, seq, qo.ptr, ko.ptr)
    hip.synchronize()
    positions = [43 + t if t < 7 else 9 - 12 + t for t in range(T)] if with_lengths else [t if t < 7 else t - 7 for t in range(T)]
    for got, x in ((qo.to_array(np.float32, q.shape), q), (ko.to_array(np.float32, k.shape), k)):
        for t, p in enumerate(positions):
            assert np.max(np.abs(got[t] - A.rope64(x[t], p, f, False))) <= _rope_bound(x[t]), (t, p)


def test_rope_from_one_buffer_into_another(qmv, hip):  # noqa: F811
    """q, k and v of a token side by side; turned q and k side by side in another
    buffer; k and v into a cache."""
    rng = np.random.default_rng(45)
    heads, kv_heads, dim, b = 6, 2, 64, A.Batch([9, 4], [30, 4], 16, 2)
    T, wide, out_wide = b.tokens, 10 * 64, 10 * 64
    rows = _rand(rng, T, wide)
    f = A.frequencies(dim)
    blank = [np.full((n, kv_heads, dim), np.nan, np.float32) for n in b.length]
    cache = A.Cache(qmv, hip, b, blank, blank, A.F32)
    d, out, df = hip.DeviceBuffer.from_array(rows), hip.DeviceBuffer.from_array(np.zeros((T, out_wide), np.float32)), hip.DeviceBuffer.from_array(f)
    seq = b.upload(qmv, hip)
    k, v = 4 * heads * dim, 4 * (heads + kv_heads) * dim
    qmv.device_rope_append(d.ptr, heads, d.ptr + k, d.ptr + v, kv_heads, dim, T, df.ptr, dim, seq, out.ptr, out.ptr + k, cache.c,
                           q_stride=wide, k_stride=wide, v_stride=wide)
    hip.synchronize()
    assert np.array_equal(d.to_array(np.float32, rows.shape), rows)
    turned = out.to_array(np.float32, (T, 10, dim))
    assert (turned[:, 8:] == 0).all()
    keys, values = cache.read(0), cache.read(1)
    for s in (0, 1):
        for i, pos in enumerate(b.positions(s)):
            t = int(b.starts[s]) + i
            x = rows[t].reshape(10, dim)
            assert np.max(np.abs(turned[t, :8] - A.rope64(x[:8], pos, f, False))) <= _rope_bound(x)
            for h in range(kv_heads):
                assert np.array_equal(keys[cache.at(s, pos, h)], turned[t, heads + h])
                assert np.array_equal(values[cache.at(s, pos, h)], x[8 + h])


# ---- scores at the ends of the range -----------------------------------------------------


def test_scores_far_below_zero(qmv, hip):  # noqa: F811
    """Rows whose scores all lie near the lowest fp32 number (here -2.3e38, in
    powers of two -3.3e38) are averages like any others. Keys alike, so that the
    weights are: the result is the mean of the values, each held to 2^-22 of
    itself (their sizes are alike), the weights too, and the sums of n terms
    rounded by at most n 2^-23 of them."""
    rng = np.random.default_rng(41)
    for n, dim in ((1, 64), (70, 64), (70, 128)):
        q, k = np.zeros((n, 2, dim), np.float32), np.zeros((n, 1, dim), np.float32)
        q[..., 3], k[..., 3] = 1.5e19, -1.533e19
        v = _rand(rng, n, 1, dim)
        o = _prompt(qmv, hip, [n], 2, 1, dim, q, k, v, 1.0)
        for i in range(n):
            ref, size = v[:i + 1, 0].astype(np.float64).mean(0), np.abs(v[:i + 1, 0]).astype(np.float64).mean(0)
            assert (np.abs(o[i] - ref) <= (2 * 2.0 ** -22 + 2 * (i + 1) * 2.0 ** -23 + 2.0 ** -22) * size).all(), (n, dim, i)


@pytest.mark.parametrize("t", A.TYPES, ids=lambda t: A.NAMES[t])
@pytest.mark.parametrize("new,length", [([1, 20, 1], [40, 60, 33]), ([1, 2], [2000, 1500]), ([45], [2200])])
def test_infinite_keys(qmv, hip, t, new, length):  # noqa: F811
    """Rows whose every score is minus infinity are NaN, like 0 / 0, not zeros;
    one infinite key gives NaN, or has no weight; other rows see none of it. The
    queries' element that meets the infinities is above zero."""
    heads, kv_heads, dim = 7, 1, 128
    b, q, keys, values, _ = _paged_case(qmv, hip, new, length, heads, kv_heads, dim, t, 16, seed=35)
    q[..., 2] = 1 + 0.137 * np.arange(heads)  # whose limbs are of one sign for some heads, and not for others
    odd = [k.copy() for k in keys]
    odd[0][:, 0, 2] = -np.inf
    last = len(new) - 1
    if last:
        odd[last][3, 0, 2] = -np.inf
    o, ok = _paged(qmv, hip, b, q, A.Cache(qmv, hip, b, odd, values, t), dim ** -0.5)
    assert ok == 1
    assert np.isnan(o[:new[0]]).all()
    for s in range(1, len(new)):
        a, n = int(b.starts[s]), new[s]
        keep = np.arange(length[s]) != (3 if s == last else -1)
        ref, bound = A.attention64(q[a:a + n], keys[s][keep], values[s][keep], dim ** -0.5, [p - (s == last) for p in b.positions(s)])
        for i in range(n):
            for h in range(heads):
                dropped = (np.abs(o[a + i, h] - ref[i, h]) <= bound[i, h]).all()
                assert dropped or (s == last and np.isnan(o[a + i, h]).all()), (s, i, h)


def test_prompt_scores_of_minus_infinity(qmv, hip):  # noqa: F811
    """As above for finite keys whose scores are below the lowest number."""
    for n in (5, 700, 1100):
        q, k = np.zeros((n, 4, 128), np.float32), np.zeros((n, 2, 128), np.float32)
        q[..., 3], k[..., 3] = 3e19, -3e19
        v = _rand(np.random.default_rng(42), n, 2, 128)
        assert np.isnan(_prompt(qmv, hip, [n], 4, 2, 128, q, k, v, 1.0)).all()


# ---- workspaces ---------------------------------------------------------------------------

PER_THREAD = 2  # hipStreamPerThread


def test_threads_on_per_thread_streams(qmv, hip):  # noqa: F811
    """Threads that name their own stream by the one handle for it do not share
    a workspace: attention in pieces and a product split along K, in two threads
    at once, then in short-lived threads one after the other (whose variables
    take each other's places). Every result has the bits of a call by itself."""
    cases = [_paged_case(qmv, hip, [1, 2], [1900, 900 + 300 * i], 14, 2, 64, A.F16, 16, seed=50 + i) for i in range(2)]
    rows, cols = 64, 18944
    raws = [qmv.synth_tensor(B.Q4_K, rows, cols, seed=60 + i) for i in range(2)]
    weights = [qmv.DeviceTensor(qmv.make_view(raw, B.Q4_K, rows, cols)) for raw in raws]
    work, expected, failures = [], [], []
    for i, (b, q, keys, values, cache) in enumerate(cases):
        x = hip.DeviceBuffer.from_array(np.random.default_rng(i).standard_normal(4 * cols).astype(np.float32))
        work.append((hip.DeviceBuffer.from_array(q), hip.DeviceBuffer(q.nbytes), b.upload(qmv, hip), cache, x, hip.DeviceBuffer(16 * rows)))

    def once(i, stream):
        dq, do, seq, cache, x, y = work[i]
        qmv.device_attention_paged(dq.ptr, 3, 14, 0.125, seq, cache.c, do.ptr, stream)
        qmv.device_matvec_group([weights[i]], x.ptr, 4, [y.ptr], stream)
        hip.check(hip.rt().hipStreamSynchronize(stream))
        return do.to_array(np.uint32, do.nbytes // 4), y.to_array(np.uint32, 4 * rows)

    def run(i, times):
        try:
            for _ in range(times):
                if not all(np.array_equal(a, e) for a, e in zip(once(i, PER_THREAD), expected[i])):
                    failures.append(i)
        except Exception as e:  # noqa: BLE001
            failures.append(repr(e))

    for i in range(2):
        expected.append(once(i, 0))
    for groups, times in (([[0, 1]], 30), ([[k % 2] for k in range(8)], 2)):
        for group in groups:
            threads = [threading.Thread(target=run, args=(i, times)) for i in group]
            [t.start() for t in threads]
            [t.join() for t in threads]
    assert failures == []
    for w in weights:
        w.close()


def test_a_refused_allocation_leaves_no_error(qmv, hip):  # noqa: F811
    """A call whose workspace the card cannot hold (the images of 2^22 - 64 tokens of
    255 heads, 1.1 TB) is refused before any launch, so that its addresses are
    never read; the next call of the thread is not told of it."""
    tokens, heads = (1 << 22) - 64, 255
    assert plan(tokens, heads, heads, 128, 1).images * (64 * 128 * 8 + 256) > 10 ** 12
    starts = hip.DeviceBuffer.from_array(np.array([0, tokens], np.int32))
    with pytest.raises(qmv.QmvError, match="memory"):
        qmv.device_attention_prompt(1 << 44, 2 << 44, 3 << 44, tokens, heads, heads, 128, 0.1, qmv.make_sequences(starts.ptr, 1), 4 << 44)
    rng = np.random.default_rng(44)
    q, k, v = _rand(rng, 9, 2, 64), _rand(rng, 9, 1, 64), _rand(rng, 9, 1, 64)
    ref, bound = A.attention64(q, k, v, 0.125, range(9))
    assert (np.abs(_prompt(qmv, hip, [9], 2, 1, 64, q, k, v, 0.125) - ref) <= bound).all()
