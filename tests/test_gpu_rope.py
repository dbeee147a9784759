"""GPU: rotary positions with several axes and the append to a paged cache, against the formulas in 64 bits.

Tolerances.  A sine or cosine is off by at most 1.5e-7: its angle's fraction (2.3e-8 of a radian from the cast to float32,
and 5e-16 of the position in turns), the Taylor sums' next terms (3e-8) and their roundings (6e-8).  A rotated value adds
two products and a sum of float32: 4e-7 (|a| + |b|) in all.  bf16 results add half a step."""
import numpy as np
import pytest

import lq8
from paged_common import BF16, F32, HALF, At, Cache, download, from_bf16, ints, rounded, tables, to_bf16, upload

pytestmark = pytest.mark.gpu
THETA = 1e6


def angles(cfg, positions):
    """[rows][pairs] angles in 64 bits; positions [axes][rows]."""
    p = np.arange(cfg.rotary_dim // 2)
    e = (p & ~1) if cfg.repeated else p
    return positions[lq8.rope_axes(cfg)].astype(np.float64).T * cfg.theta ** (-2.0 * e / cfg.rotary_dim)


def turned(x, cfg, positions, inverse=False):
    """(rotated x, tolerance in float32); x [rows][heads][dim] in 64 bits."""
    half, a = cfg.rotary_dim // 2, angles(cfg, positions)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None] * (-1 if inverse else 1)
    u, v = x[..., :half], x[..., half:2 * half]
    y = np.concatenate([u * c - v * s, v * c + u * s, x[..., 2 * half:]], -1)
    # the reference's own angle is off by 2^-52 of itself, too
    far = 2.0 ** -50 * np.abs(a).max() if a.size else 0.0
    t = (4e-7 + far) * (np.abs(u) + np.abs(v))
    return y, np.concatenate([t, t, np.zeros_like(x[..., 2 * half:])], -1)


def check(got, want, tol, dtype):
    tol = tol + np.abs(want) * HALF[dtype] + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.max(np.abs(got - want) / tol):.2f} tolerances"


# (rows, heads, dim, rotary, sections, interleaved, repeated)
ROPES = [
    (1, 1, 16, 16, (), False, False), (1, 24, 128, 128, (24, 20, 20), True, False), (7, 3, 80, 80, (20, 20), False, False),
    (33, 5, 128, 32, (8, 4, 4), True, False), (5, 16, 64, 64, (16, 8, 4, 4), False, False), (129, 2, 256, 256, (), False, True),
    (3, 40, 240, 112, (56, 0), False, False), (600, 9, 48, 16, (), False, True), (2, 7, 128, 128, (64, 0, 0), True, False),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", ROPES)
def test_rope_rows(ctx, case, dtype):
    rows, heads, dim, rotary, sections, inter, rep = case
    rng = np.random.default_rng(rows * 7 + dim)
    rope = lq8.Rope(ctx, dim, THETA, rotary_dim=rotary, sections=sections, interleaved=inter, repeated=rep)
    x = rounded(rng.standard_normal((rows, heads, dim)), dtype)
    pos = rng.integers(0, 70000, (max(1, len(sections)), rows)).astype(np.int32)
    pos[:, 0] = [0, 2 ** 31 - 1, -5, 1][:pos.shape[0]]
    dx, dy, dp = upload(ctx, x, dtype), upload(ctx, np.zeros_like(x), dtype), ints(ctx, pos)
    lq8.rope_device(ctx, rope, lq8.RopeRows(dx, dy, rows, heads, dim, dp, dtype=dtype))
    want, tol = turned(x.astype(np.float64), rope.cfg, pos)
    check(download(dy, x.size, dtype).reshape(x.shape), want, tol, dtype)
    # back again, in place: the transpose, which is also the gradient
    lq8.rope_device(ctx, rope, lq8.RopeRows(dx, dx, rows, heads, dim, dp, dtype=dtype, inverse=True))
    want, tol = turned(x.astype(np.float64), rope.cfg, pos, inverse=True)
    check(download(dx, x.size, dtype).reshape(x.shape), want, tol, dtype)
    for b in (dx, dy, dp, rope):
        b.free()


def test_rope_inverse_is_the_gradient(ctx):
    """y = R x is linear: the gradient of sum(g * R x) is R^T g, and (R^T g) . d = g . (R (x + d) - R x) for any d."""
    rng = np.random.default_rng(5)
    rope = lq8.Rope(ctx, 64, 1e4, sections=(12, 10, 10))
    x, d, g = (rng.standard_normal((9, 4, 64)).astype(np.float32) for _ in range(3))
    dp = ints(ctx, rng.integers(0, 5000, (3, 9)))

    def run(v, inverse):
        dv = upload(ctx, v, F32)
        lq8.rope_device(ctx, rope, lq8.RopeRows(dv, dv, 9, 4, 64, dp, inverse=inverse))
        y = dv.download(np.float32, v.size).reshape(v.shape).astype(np.float64)
        dv.free()
        return y

    left = (run(g, True) * d).sum(-1)
    right = (g * (run(x + d, False) - run(x, False))).sum(-1)
    # both sides: 64 products of values up to about 4 with 4e-7 (|a| + |b|) each
    assert np.max(np.abs(left - right)) < 64 * 4e-7 * 40
    dp.free()
    rope.free()


def test_rope_strides_leave_the_rest(ctx):
    """Rows inside wider rows, positions of a longer array: what lies between is not touched."""
    rng = np.random.default_rng(6)
    rope = lq8.Rope(ctx, 32, 1e4, sections=(8, 8))
    x = rng.standard_normal((5, 200)).astype(np.float32)
    y = np.full((5, 136), 7.0, np.float32)
    pos = rng.integers(0, 900, (2, 11)).astype(np.int32)
    dx, dy, dp = upload(ctx, x, F32), upload(ctx, y, F32), ints(ctx, pos)
    lq8.rope_device(ctx, rope, lq8.RopeRows(At(dx, 16), At(dy, 32), 5, 3, 32, dp, x_stride=200, y_stride=136, positions_stride=11))
    got = dy.download(np.float32, y.size).reshape(y.shape)
    want, tol = turned(x[:, 4:100].reshape(5, 3, 32).astype(np.float64), rope.cfg, pos[:, :5])
    check(got[:, 8:104].reshape(5, 3, 32), want, tol, F32)
    assert np.all(got[:, :8] == 7.0) and np.all(got[:, 104:] == 7.0)
    for rows, heads in ((0, 3), (5, 0)):  # nothing to do
        lq8.rope_device(ctx, rope, lq8.RopeRows(dx, dy, rows, heads, 32, dp))
    assert np.array_equal(dy.download(np.float32, y.size).reshape(y.shape), got)
    for b in (dx, dy, dp, rope):
        b.free()


def normed(x, w, eps):
    """RmsNorm with bf16 input, weight and result; the result's one rounding goes through float32."""
    x, w = from_bf16(to_bf16(x)).astype(np.float64), from_bf16(to_bf16(w)).astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return from_bf16(to_bf16(y.astype(np.float32))).astype(np.float64)


TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


# (rows per sequence, lengths, heads, kv, dim, page, norm, sections; None: no rotation)
APPENDS = [
    ((1,), (1,), 1, 1, 64, 16, False, None),
    ((1, 1, 1, 1), (17, 16, 0, 300), 16, 8, 128, 16, True, ()),
    ((3, 0, 40, 1, 64), (3, 5, 57, 1, 1000), 6, 2, 128, 32, True, (24, 20, 20)),
    ((130, 2), (129, 2), 4, 4, 64, 64, False, (16, 16)),  # the first row of sequence 0 is before its start
    ((70, 33), (70, 33), 5, 1, 128, 128, False, None),
    ((5,) * 300, tuple(range(5, 305)), 2, 1, 64, 16, True, ()),  # more sequences than a workgroup has threads
]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(ctx, case, types):
    counts, lengths, heads, kv, dim, page, norm, sections = APPENDS[case]
    act, ct = types
    rng = np.random.default_rng(100 + case)
    rows, n, spare = sum(counts), len(counts), 3
    cache = Cache(rng, sum(-(-max(1, t) // page) for t in lengths) + 2, page, kv, dim, ct, stride=kv * page * dim + 32)
    tab = [cache.table(t) for t in lengths]
    width = max(len(t) for t in tab) + 1
    begin = np.concatenate([[0], np.cumsum(counts)])
    qkv = rounded(rng.standard_normal((rows + spare, heads + 2 * kv, dim)) * 2, act)
    qw, kw = (1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    slots = np.concatenate([t - c + np.arange(c) for c, t in zip(counts, lengths)]).astype(np.int64)
    axes = max(1, len(sections or ()))
    pos = None if not sections else rng.integers(0, 40000, (axes, rows + spare)).astype(np.int32)
    rope = None if sections is None else lq8.Rope(ctx, dim, THETA, sections=sections)
    single = all(c == 1 for c in counts)
    table = tables(tab, width, rng)
    if case == 1:
        table[0, 1] = cache.pages  # a page that does not exist: position 16 of sequence 0 is dropped
    dk, dv, pages = cache.device(ctx)
    dq, dout = upload(ctx, qkv, act), upload(ctx, np.full((rows + spare, heads * dim), 7.0), act)
    dl, dt, db = ints(ctx, lengths), ints(ctx, table), ints(ctx, begin)
    dqw, dkw = upload(ctx, qw, F32), upload(ctx, kw, F32)
    dp = None if pos is None else ints(ctx, pos)
    es = 4 if act == F32 else 2
    batch = lq8.PagedBatch(dl, dt, n, width, rows=rows if single else rows + spare, row_begin=None if single else db, max_rows=max(counts))
    lq8.paged_append_device(ctx, rope, pages, batch, lq8.QkvRows(
        dq, At(dq, heads * dim * es), At(dq, (heads + kv) * dim * es), heads, dim, q_out=dout, stride=(heads + 2 * kv) * dim,
        q_norm=dqw if norm else None, k_norm=dkw if norm else None, eps=1e-6, positions=dp, positions_stride=rows + spare, dtype=act))
    x = qkv[:rows].astype(np.float64)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], qkv[:rows, heads + kv:]
    if norm:
        q, k = normed(qkv[:rows, :heads], qw, np.float32(1e-6)), normed(qkv[:rows, heads:heads + kv], kw, np.float32(1e-6))
    at = np.repeat(slots[None], axes, 0) if pos is None else pos[:, :rows]
    zero = np.zeros(1)
    (q, qt), (k, kt) = ((turned(y, rope.cfg, at) if rope is not None else (y, zero)) for y in (q, k))
    got = download(dout, (rows + spare) * heads * dim, act).reshape(rows + spare, heads, dim)
    check(got[:rows], q, qt, act)
    assert np.all(got[rows:] == 7.0)  # rows behind the last sequence
    gk, gv = (download(b, cache.k.size, ct).reshape(cache.k.shape) for b in (dk, dv))
    touched = np.zeros(cache.k.shape, bool)
    row = 0
    for s, c in enumerate(counts):
        for i in range(c):
            t = int(slots[row])
            if t >= 0 and not (case == 1 and s == 0):
                cell = np.s_[tab[s][t // page]]
                inner = lambda a: a[cell][:cache.dense].reshape(kv, page, dim)[:, t % page]  # noqa: E731
                check(inner(gk), k[row], kt[row] if kt.size > 1 else kt, ct)
                assert np.array_equal(inner(gv), rounded(v[row], ct))
                inner(touched)[...] = True
            row += 1
    assert np.isnan(gk[~touched]).all() and np.isnan(gv[~touched]).all()
    for b in (dk, dv, dq, dout, dl, dt, db, dqw, dkw, dp, rope):
        if b is not None:
            b.free()


def test_append_keys_and_values_alone_and_nan(ctx):
    """No queries; a NaN and infinities go into bf16 pages as they are."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, 2, 16, 1, 64, BF16)
    tab = cache.table(3)
    dk, dv, pages = cache.device(ctx)
    k, v = rng.standard_normal((2, 64)).astype(np.float32), rng.standard_normal((2, 64)).astype(np.float32)
    k[0, 3], k[1, 5], v[0, 0], v[1, 63] = np.inf, -np.inf, np.inf, np.nan
    k.view(np.uint32)[0, 7] = 0x7F800001  # NaNs whose upper half alone would be an infinity, or turn over
    v.view(np.uint32)[1, 2] = 0x7FFFFFFF
    dkr, dvr, dl, dt, db = upload(ctx, k, F32), upload(ctx, v, F32), ints(ctx, [3]), ints(ctx, [tab]), ints(ctx, [0, 2])
    lq8.paged_append_device(ctx, None, pages, lq8.PagedBatch(dl, dt, 1, 1, rows=2, row_begin=db, max_rows=2),
                            lq8.QkvRows(None, dkr, dvr, 0, 64))
    for buf, x in ((dk, k), (dv, v)):
        got = download(buf, cache.k.size, BF16).reshape(2, 16, 64)[tab[0], 1:3]
        assert np.array_equal(got, rounded(x, BF16), equal_nan=True)
    for b in (dk, dv, dkr, dvr, dl, dt, db):
        b.free()


def test_append_row_begin_out_of_range_stays_inside(ctx):
    """A row_begin that is not ascending, or reaches past the rows, writes no more than the slots its tables name."""
    rng = np.random.default_rng(10)
    cache = Cache(rng, 4, 16, 2, 64, F32)
    tab = [cache.table(16), cache.table(16)]
    dk, dv, pages = cache.device(ctx)
    x = rng.standard_normal((6, 2 * 64)).astype(np.float32)
    dx, dl, dt = upload(ctx, x, F32), ints(ctx, [2 ** 31 - 1, 6]), ints(ctx, tab)
    for begin in ([0, 2 ** 31 - 1, 3], [-(2 ** 31), 4, 2 ** 31 - 1], [5, 2, 0]):
        db = ints(ctx, begin)
        lq8.paged_append_device(ctx, None, pages, lq8.PagedBatch(dl, dt, 2, 1, rows=6, row_begin=db, max_rows=6),
                                lq8.QkvRows(None, dx, dx, 0, 64))
        ctx.synchronize()
        db.free()
    got = download(dk, cache.k.size, F32).reshape(cache.k.shape)
    for page in cache.free:  # of no table
        assert np.isnan(got[page]).all()
    for b in (dk, dv, dx, dl, dt):
        b.free()


def test_rope_other_dim_is_refused(ctx):
    rope = lq8.Rope(ctx, 64, 1e4)
    cache = Cache(np.random.default_rng(1), 1, 16, 1, 128, F32)
    dk, dv, pages = cache.device(ctx)
    dl, dt = ints(ctx, [1]), ints(ctx, [[0]])
    with pytest.raises(lq8.ShapeMismatch):
        lq8.paged_append_device(ctx, rope, pages, lq8.PagedBatch(dl, dt, 1, 1), lq8.QkvRows(None, dk, dv, 0, 128))
    rope.free()
    with pytest.raises(lq8.InvalidArgument):  # a released handle
        lq8._check(lq8.lib().lq8_paged_append_device(ctx.handle, dl.ptr, pages.c, lq8.PagedBatch(dl, dt, 1, 1).c,
                                                     lq8.QkvRows(None, dk, dv, 0, 128).c))
    for b in (dk, dv, dl, dt):
        b.free()
