"""Plain attention and rotary embedding in 64 bits, bounds for what fp32 sums
may differ by, and calls of the library on numpy arrays, for the tests of the
operators between the projections."""
import importlib

import numpy as np

F32, F16, BF16 = 0, 1, 30
TYPES = [F32, F16, BF16]
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
# Half a step of each type, relative to the value.
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8 / 2}


def to_bf16(x):
    """float32 -> bfloat16 bits, nearest, ties to even"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + (0x7FFF + ((u >> 16) & 1))) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), ((u >> 16) | 0x40).astype(np.uint16), r)


def encode(x, t):
    """Values as a cache of type t stores them"""
    with np.errstate(over="ignore"):
        return to_bf16(x) if t == BF16 else np.ascontiguousarray(x, np.float32).astype(np.float16 if t == F16 else np.float32)


def decode(a, t):
    return (a.astype(np.uint32) << 16).view(np.float32) if t == BF16 else a.astype(np.float32)


def dtype_of(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


def attention64(q, k, v, scale, positions):
    """q [n, H, D], k and v [L, Hk, D], the position of each of the n rows ->
    (o [n, H, D] in 64 bits, the bound of each element's error).

    The bound. A score is a sum of D products of values held to 2^-22 each side
    (two f16 limbs), summed in fp32, scaled once: off by at most
        ds = (2 * 2^-22 + (D + 4) * 2^-23) * |scale| * sum |q||k|
    (2^-23, a whole step, per addition: the matrix core's rounding is not said
    to be to nearest). Weights exp(s - max) are then off by a factor within
    exp(2 ds) and by the exponential's own error, 2^-22 with the subtraction
    of numbers up to 2 max|s| before it, 2^-23 of those; the sums over L keys
    by (L + 64) 2^-23, the limbs of weight and value by 2^-21; numerator and
    denominator alike. An element's error is at most the factor times
    sum p |v|, twice where both sums count."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    o = np.zeros((n, heads, dim))
    bound = np.zeros((n, heads, dim))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for i in range(n):
        last = positions[i]
        if last < 0:
            continue
        for h in range(heads):
            kk, vv = k[:last + 1, h // group], v[:last + 1, h // group]
            s = scale * (kk @ q[i, h])
            big = np.max(abs(scale) * (np.abs(kk) @ np.abs(q[i, h])))
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h] = p @ vv
            ds = (2.0 ** -21 + (dim + 4) * 2.0 ** -23) * big + 2.0 ** -23 * 2 * np.max(np.abs(s))
            factor = np.expm1(2 * ds) + 2.0 ** -21 + (last + 65) * 2.0 ** -23 + 2.0 ** -21
            bound[i, h] = 2 * factor * (p @ np.abs(vv)) + 2.0 ** -126
    return o, bound


def rope64(x, position, frequencies, interleaved):
    """x [heads, D] of one token in 64 bits"""
    x = x.astype(np.float64).copy()
    half = len(frequencies)
    a = position * np.asarray(frequencies, np.float64)
    c, s = np.cos(a), np.sin(a)
    i0 = np.arange(half) * 2 if interleaved else np.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    u, w = x[:, i0].copy(), x[:, i1].copy()
    x[:, i0], x[:, i1] = u * c - w * s, u * s + w * c
    return x


def frequencies(rotary, theta=1e6):
    return theta ** (-2 * np.arange(rotary // 2, dtype=np.float64) / max(1, rotary))


class Batch:
    """Sequences of new tokens on the device. `order` shuffles the pages."""

    def __init__(self, new, length=None, page=16, seed=0, spare=3):
        self.new, self.length, self.page = list(new), list(length if length is not None else new), page
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.starts[-1])
        per = [-(-max(0, n) // page) for n in self.length]
        self.columns = max(1, max(per)) + 1
        self.pages = sum(per) + spare
        order = np.random.default_rng(seed).permutation(self.pages)
        self.table = np.full((len(self.new), self.columns), -7, np.int32)  # past the length: never looked at
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n

    def positions(self, s):
        return [self.length[s] - self.new[s] + i for i in range(self.new[s])]

    def upload(self, qmv, hip):
        self.d = [hip.DeviceBuffer.from_array(a) for a in
                  (self.starts, np.array(self.length, np.int32), self.table)]
        return qmv.make_sequences(self.d[0].ptr, len(self.new), self.d[1].ptr, self.d[2].ptr, self.columns)


class Cache:
    """A paged cache filled from per-sequence arrays [L, Hk, D]; everything
    that no sequence has is NaN. layout: "heads" [page][head][token][D],
    "tokens" [page][token][head][D], "shared" keys and values of a page side by
    side, "wide" rows with 8 unused elements."""

    def __init__(self, qmv, hip, batch, keys, values, t, layout="heads"):
        self.t, self.batch = t, batch
        hk, dim = keys[0].shape[1:]
        pages, page = batch.pages, batch.page
        row = dim + 8 if layout == "wide" else dim
        if layout == "tokens":
            strides = (page * hk * row, row, hk * row)
        else:
            strides = (hk * page * row, page * row, row)
        if layout == "shared":
            strides = (2 * hk * page * row,) + strides[1:]
        self.strides, self.shape = strides, (hk, dim)
        total = pages * strides[0]
        self.offset = hk * page * row if layout == "shared" else 0
        stores = []
        for arrays in (keys, values):
            full = np.full(total, np.nan, np.float32)
            if arrays is not None:
                for s, a in enumerate(arrays):
                    for j in range(a.shape[0]):
                        for h in range(hk):
                            full[self.at(s, j, h)] = a[j, h]
            stores.append(encode(full, t))
        size = stores[0].itemsize
        if layout == "shared":
            both = stores[0].copy()
            where = self._owned(batch, keys)
            both[where + self.offset] = stores[1][where]
            # past the end of the last value page there is room by construction
            self.buffers = [hip.DeviceBuffer.from_array(both)]
            pk, pv = self.buffers[0].ptr, self.buffers[0].ptr + self.offset * size
        else:
            self.buffers = [hip.DeviceBuffer.from_array(a) for a in stores]
            pk, pv = self.buffers[0].ptr, self.buffers[1].ptr
        self.total = total
        self.c = qmv.make_paged_cache(pk, pv, t, hk, dim, page, pages, strides[0], strides[1], strides[2])

    def at(self, s, j, h):
        b, (ps, hs, ts) = self.batch, self.strides
        first = int(b.table[s, j // b.page]) * ps + h * hs + (j % b.page) * ts
        return slice(first, first + self.shape[1])

    def _owned(self, batch, arrays):
        return np.concatenate([np.arange(self.at(s, j, h).start, self.at(s, j, h).stop)
                               for s, a in enumerate(arrays) for j in range(a.shape[0]) for h in range(self.shape[0])])

    def read(self, which):
        """The stored codes as one flat array (not for "shared")"""
        return self.buffers[which].to_array(dtype_of(self.t), (self.total,))


def pack(rows, stride, width):
    """rows [T, width] with `stride` floats from row to row, NaN between"""
    out = np.full((rows.shape[0], stride), np.nan, np.float32)
    out[:, :width] = rows.reshape(rows.shape[0], width)
    return out


def hip_module():
    return importlib.import_module("my-inference-engine_amd.hip_runtime")
