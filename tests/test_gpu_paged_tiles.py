"""GPU: attention over pages where both row tiles (16 and 128 packed rows) take part: what is masked, not finite, far apart,
tiny or huge reaches each of them.  Which one a call takes is asserted by lq8.paged_plan."""
import numpy as np
import pytest

import lq8
from paged_common import BF16, F32, attend, rounded, tables, tolerance
from test_gpu_paged_attention import TYPES, Batch, compare

pytestmark = pytest.mark.gpu

TALL = (420, 420)  # enough rows for the large tile in every part that holds it


class P:
    ptr = __import__("ctypes").c_void_p(0x10000)


def plan(ctx, b):
    """How the call of a Batch runs on this device."""
    n = len(b.seqs)
    single = all(r == 1 for r, _ in b.seqs)
    page = b.cache.page
    kv = lq8.KVPages(P, P, b.cache.pages, page, b.kv, b.dim, dtype=b.types[1])
    width = max(1, max(len(t) for t in b.tab[:n]))
    batch = lq8.PagedBatch(P, P, n, width, rows=b.rows if single else b.rows + b.spare, row_begin=None if single else P,
                           max_rows=max(1, max(r for r, _ in b.seqs)))
    prefix = lq8.SharedPrefix(P, P, P, len(b.plens), max(1, max(len(t) for t in b.tab[n:])) + 1) if b.plens else None
    p = lq8.paged_plan(kv, batch, lq8.AttnRows(P, P, b.heads, b.dim, dtype=b.types[0]), prefix)
    return p["own_rows"], p["prefix_rows"]


def checked(ctx, b, tiles, **want):
    assert plan(ctx, b) == tiles
    out, tol = b.want(**want)
    compare(b.run()[:b.rows], out, tol)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 128, 16), (8, 2, 64, 32), (14, 2, 64, 16), (10, 2, 128, 128)])
def test_large_tiles(ctx, types, heads, kv, dim, page):
    checked(ctx, Batch(ctx, types, [TALL, (0, 3), (1, 500), (33, 40), (7, 0), (129, 131)], heads, kv, dim, page, seed=1), (128, 0))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_large_tiles_behind_a_prefix(ctx, types, dim):
    checked(ctx, Batch(ctx, types, [TALL, (1, 1), (0, 0), (60, 70), (1, 0)], 8, 2, dim, 16, groups=([0, 3, 5], [290, 411]), seed=2), (128, 128))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens_behind_a_long_prefix(ctx, types, dim):
    """A large tile for the prefix beside small ones, in one launch; values there that are not finite."""
    b = Batch(ctx, types, [(1, 1 + 7 * i % 150) for i in range(90)], 8, 2, dim, 16, groups=([0, 80], [2011]), seed=3)
    b.v[90][2010, 0, 5], b.v[90][100, 1, 7], b.v[90][101, 1, 7], b.v[4][0, 0, 1] = np.inf, np.inf, -np.inf, np.nan
    checked(ctx, b, (16, 128))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [17, 24, 32, 48, 64, 100])
def test_row_counts_between_the_tiles(ctx, types, rows):
    """Up to 100 packed rows, few blocks (small tiles) and many (by the type's rule)."""
    Batch(ctx, types, [(rows, 150), (rows - 5, 700)], 2, 2, 128, 16, seed=rows).check()
    Batch(ctx, types, [(rows, 150)] + [(rows - i, 260 + i) for i in range(12)], 8, 8, 64, 16, seed=rows + 1).check()


@pytest.mark.parametrize("types", TYPES)
def test_a_prefix_in_small_tiles_before_large_own_ones(ctx, types):
    checked(ctx, Batch(ctx, types, [TALL, (50, 900), (3, 1)], 8, 2, 64, 16, groups=([0, 1, 3], [20, 100]), seed=4), (128, 16))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_large_tiles_not_finite(ctx, types, dim):
    """Infinite and NaN values, keys and queries reach the rows that see them, and no others."""
    b = Batch(ctx, types, [TALL, (90, 90), (40, 70)], 8, 2, dim, 16, seed=5)
    for s, t in ((0, 400), (1, 60), (2, 32)):
        b.v[s][t, 0, 5], b.v[s][t, 1, 63], b.v[s][t - 20, 0, 9] = np.inf, np.nan, -np.inf
    b.v[0][410, 0, 5] = -np.inf
    b.k[0][300, 1, 3] = np.nan
    b.k[0][200, 0, 2] = np.inf
    b.k[1][10, 0, 1] = -np.inf
    b.q[3, 70] = np.nan
    b.q[100, 0] = np.inf
    b.q[:, 2] = np.where(np.arange(len(b.q)) % 3 == 0, 0, b.q[:, 2])  # infinity times zero
    checked(ctx, b, (128, 0))


@pytest.mark.parametrize("types", TYPES)
def test_large_tiles_scores_of_minus_infinity(ctx, types):
    b = Batch(ctx, types, [TALL, (70, 70), (1, 130)], 8, 2, 64, 16, seed=6)
    b.q[:, :512] = rounded(np.abs(b.q[:, :512]) + 0.5, types[0])
    b.k[0][:200, :, 7] = -np.inf
    b.k[1][:20, :, 7] = -np.inf
    out, _ = b.want()
    assert np.isnan(out[:200]).all() and np.isfinite(out[200:420]).all()
    checked(ctx, b, (128, 0))


@pytest.mark.parametrize("types", TYPES)
def test_large_tiles_missing_pages(ctx, types):
    b = Batch(ctx, types, [TALL, (70, 100), (16, 16)], 8, 2, 128, 16, seed=7)
    table = tables(b.tab[:3], 30, b.rng)
    table[0, 2], table[0, 20], table[1, 0], table[2, 0] = -1, b.cache.pages, 2 ** 31 - 1, -(2 ** 31)
    gone = {0: np.r_[32:48, 320:336], 1: np.r_[0:16], 2: np.r_[0:16]}
    out, tol = b.want(drop=lambda s: gone[s])
    assert plan(ctx, b)[0] == 128
    # (the tables of Batch.run are as wide as the longest sequence's)
    got = b.run(table=table[:, :27])
    compare(got[:b.rows], out, tol)
    assert np.all(got[b.begin[2]:b.begin[3]] == 0.0)


@pytest.mark.parametrize("types", TYPES)
def test_large_tiles_scores_far_apart(ctx, types):
    b = Batch(ctx, types, [TALL, (80, 300), (30, 257)], 8, 2, 128, 16, seed=8, qstd=40.0)
    b.k[2] = rounded(-np.abs(b.k[2]) * 1e30, types[1])
    b.k[2][256] = rounded(np.abs(b.k[2][256]) * 1e-33, types[1])
    b.q[500:530] = rounded(np.abs(b.q[500:530]) + 1, types[0])
    assert plan(ctx, b)[0] == 128
    b.check()
    b.check(scale=1e-6)
    b.check(scale=3e4)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", [[TALL, (40, 60)], [(1, 300), (1, 77)]])
@pytest.mark.parametrize("power", [-96, 120])
def test_small_and_large_values(ctx, types, seqs, power):
    """Values scaled by a power of two scale the results, far from one too: 2^120 and 2^-96, whose smallest parts (24 bits
    down) are still normal numbers."""
    b = Batch(ctx, types, seqs, 8, 2, 64, 16, seed=9)
    b.v = [np.clip(v, -8, 8) for v in b.v]
    out, tol = b.want()
    b.v = [np.ldexp(v, power) for v in b.v]
    got = b.run()[:b.rows].astype(np.float64)
    compare(np.ldexp(got, -power), out, tol)


@pytest.mark.parametrize("types", TYPES)
def test_more_sequences_than_a_workgroup_has_threads(ctx, types):
    b = Batch(ctx, types, [(i % 4, max(i % 4, (i * 37) % 60)) for i in range(700)], 8, 2, 64, 16, groups=([0, 300, 700], [33, 150]), seed=10)
    b.check()
    Batch(ctx, types, [(60 if i in (3, 299, 300, 599) else 1, 61 + i % 9) for i in range(600)], 8, 2, 64, 16, seed=11).check()


def test_the_same_pages_in_several_sequences(ctx):
    """Sequences may read one another's pages, a page twice in one of them too."""
    b = Batch(ctx, (BF16, BF16), [(1, 100), (1, 64), (1, 90)], 8, 2, 128, 16, seed=12)
    table = tables(b.tab[:3], 7, b.rng)
    table[2, :6] = [table[0, 0], table[1, 2], table[0, 0], table[0, 5], table[1, 0], table[0, 3]]
    k0, k1, v0, v1 = b.k[0], b.k[1], b.v[0], b.v[1]
    got = b.run(table=table)
    b.k[2], b.v[2] = (np.concatenate([x[:16], y[32:48], x[:16], x[80:96], y[:16], x[48:58]]) for x, y in ((k0, k1), (v0, v1)))
    out, tol = b.want()
    compare(got[:b.rows], out, tol)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_rows_result_does_not_depend_on_its_group(ctx, types, dim):
    """Bit for bit, with the other rows of its tiles far larger, and not finite."""
    def batch():
        return Batch(ctx, types, [(1, 1 + 7 * i % 90) for i in range(90)], 8, 2, dim, 16, groups=([0, 90], [2011]), seed=13)

    a, b = batch(), batch()
    assert plan(ctx, a) == (16, 128)
    b.q[1:40] = rounded(b.q[1:40] * 30, types[0])
    b.q[40:60] = rounded(b.q[40:60] * 1e7, types[0])
    b.q[70:75] = np.inf
    x, y = a.run(), b.run()
    same = np.r_[0, 60:70, 75:90]
    assert np.isfinite(x[same]).all() and np.array_equal(x[same], y[same])
