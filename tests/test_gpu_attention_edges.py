"""Calls of the operators between the projections that the documentation allows
at its edges, against 64 bits."""
import numpy as np
import pytest

import _attention as A
from test_gpu_attention import _prompt, _rand, _rope_bound, hip  # noqa: F401

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
