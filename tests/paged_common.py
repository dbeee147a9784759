"""A ragged batch over a paged cache in plain numpy, in 64 bits, and the same batch on the device (used by the paged cache's
tests)."""
import numpy as np

import lq8

F32, BF16 = lq8.DTYPE_F32, lq8.DTYPE_BF16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}  # a rounding's largest relative error


def to_bf16(x):
    """float32 -> bf16 bits, to nearest, ties to even, NaN kept."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def rounded(x, dtype):
    x = np.asarray(x, np.float32)
    return x if dtype == F32 else from_bf16(to_bf16(x))


def upload(ctx, x, dtype):
    return lq8.DeviceBuffer.from_array(ctx, np.ascontiguousarray(x, np.float32) if dtype == F32 else to_bf16(x))


def download(buf, n, dtype):
    return buf.download(np.float32, n) if dtype == F32 else from_bf16(buf.download(np.uint16, n))


class At:
    """A place inside a device buffer."""

    def __init__(self, buf, nbytes):
        import ctypes

        self.buf, self.ptr = buf, ctypes.c_void_p(buf.ptr.value + nbytes)


class Cache:
    """Host copy of the pages: what no sequence holds is NaN."""

    def __init__(self, rng, pages, page, kv, dim, dtype, stride=0):
        self.pages, self.page, self.kv, self.dim, self.dtype = pages, page, kv, dim, dtype
        self.dense = kv * page * dim
        self.stride = stride or self.dense
        self.k = np.full((pages, self.stride), np.nan, np.float32)
        self.v = np.full((pages, self.stride), np.nan, np.float32)
        self.free = list(rng.permutation(pages))

    def table(self, positions):
        return [int(self.free.pop()) for _ in range(-(-positions // self.page))]

    def at(self, which, page):
        return (self.k if which == "k" else self.v)[page, :self.dense].reshape(self.kv, self.page, self.dim)

    def put(self, table, k, v):
        """k, v [positions][kv][dim] (values the cache's type has) into a table's pages."""
        for t in range(k.shape[0]):
            self.at("k", table[t // self.page])[:, t % self.page] = k[t]
            self.at("v", table[t // self.page])[:, t % self.page] = v[t]

    def device(self, ctx):
        k, v = upload(ctx, self.k, self.dtype), upload(ctx, self.v, self.dtype)
        return k, v, lq8.KVPages(k, v, self.pages, self.page, self.kv, self.dim, dtype=self.dtype,
                                 page_stride=0 if self.stride == self.dense else self.stride)


def ints(ctx, x):
    return lq8.DeviceBuffer.from_array(ctx, np.ascontiguousarray(x, np.int32))


def tables(rows, width, rng):
    """Page tables side by side; past a sequence's pages stands anything."""
    out = rng.integers(-(2 ** 31), 2 ** 31, (max(1, len(rows)), width)).astype(np.int32)
    for i, r in enumerate(rows):
        out[i, :len(r)] = r
    return out


def attend(q, k, v, scale):
    """q [heads][dim], k and v [n][kv][dim] in 64 bits -> (out [heads][dim], sum p |v|, largest score magnitude)."""
    heads, dim = q.shape
    n, kv = k.shape[:2]
    if n == 0:
        return np.zeros((heads, dim)), np.zeros((heads, dim)), 0.0
    out, mag, top = np.empty((heads, dim)), np.empty((heads, dim)), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(heads):
            g = h // (heads // kv)
            s = k[:, g] @ q[h] * scale
            e = np.exp(s - np.max(s))
            p = e / e.sum()
            out[h], mag[h] = p @ v[:, g], p @ np.abs(v[:, g])
            top = max(top, float(np.max(np.abs(k[:, g]) @ np.abs(q[h]))) * scale)
    return out, mag, top


def tolerance(out, mag, top, dim, n, types):
    """What rounding explains.  A score of largest magnitude `top` is off by at most 2^-24 top for each of its roundings,
    which go either way: 4 sqrt(dim) of them, and 8 more for its products' parts and the exponent's; so are p, the sum and
    the output's sum over n positions (2 sqrt(n)).  bf16 rows: every probability and the output are rounded to bf16."""
    rel = 2.0 ** -24 * ((4 * np.sqrt(dim) + 8) * (top + 1) * 2 + 2 * np.sqrt(n) + 16)
    tol = rel * mag
    if types[0] == BF16:
        tol = tol + 2.0 ** -8 * (mag + np.abs(out))
    return tol + 1e-30
