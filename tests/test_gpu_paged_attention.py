"""GPU: attention over a paged cache, with and without shared prefixes, against the formula in 64 bits (tolerances:
paged_common.tolerance).  What no sequence holds is NaN in the pages, and page tables name anything past a sequence's
positions."""
import numpy as np
import pytest

import lq8
from paged_common import BF16, F32, At, Cache, attend, download, ints, rounded, tables, tolerance, upload

pytestmark = pytest.mark.gpu
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


class Batch:
    """Sequences (rows, length) over a cache, optionally in groups (first sequences, prefix lengths)."""

    def __init__(self, ctx, types, seqs, heads, kv, dim, page, groups=None, seed=0, spare=2, pad=0, stride=0, qstd=1.5):
        self.ctx, self.types, self.seqs, self.heads, self.kv, self.dim = ctx, types, seqs, heads, kv, dim
        rng = self.rng = np.random.default_rng(seed)
        self.first, self.plens = groups or ([0], [])
        total = sum(-(-t // page) for _, t in seqs) + sum(-(-t // page) for t in self.plens) + 2
        self.cache = Cache(rng, total, page, kv, dim, types[1], stride=stride)
        self.k, self.v, self.tab = [], [], []
        for t in [t for _, t in seqs] + list(self.plens):
            self.tab.append(self.cache.table(t))
            self.k.append(rounded(rng.standard_normal((t, kv, dim)), types[1]))
            self.v.append(rounded(rng.standard_normal((t, kv, dim)) + 0.25, types[1]))
        self.begin = np.concatenate([[0], np.cumsum([r for r, _ in seqs])]).astype(int)
        self.rows, self.spare = int(self.begin[-1]), spare
        self.wide = heads * dim + pad
        self.q = rounded(rng.standard_normal((self.rows + spare, self.wide)) * qstd, types[0])

    def run(self, in_place=False, max_rows=None, table=None, scale=None):
        ctx, n = self.ctx, len(self.seqs)
        for tab, k, v in zip(self.tab, self.k, self.v):
            self.cache.put(tab, k, v)
        dk, dv, pages = self.cache.device(ctx)
        single = all(r == 1 for r, _ in self.seqs)
        width = max(1, max(len(t) for t in self.tab[:n]))
        table = tables(self.tab[:n], width, self.rng) if table is None else table
        dq = upload(ctx, self.q, self.types[0])
        dout = dq if in_place else upload(ctx, np.full(self.q.shape, 7.0), self.types[0])
        bufs = [dk, dv, dq, ints(ctx, [t for _, t in self.seqs]), ints(ctx, table), ints(ctx, self.begin)] + ([] if in_place else [dout])
        batch = lq8.PagedBatch(bufs[3], bufs[4], n, width, rows=self.rows if single else self.rows + self.spare,
                               row_begin=None if single else bufs[5], max_rows=max_rows or max(1, max(r for r, _ in self.seqs)))
        rows = lq8.AttnRows(dq, dout, self.heads, self.dim, dtype=self.types[0], q_stride=self.wide, out_stride=self.wide, scale=scale)
        if self.plens:
            pw = max(1, max(len(t) for t in self.tab[n:])) + 1
            pt = tables(self.tab[n:], pw, self.rng)
            bufs += [ints(ctx, self.first), ints(ctx, self.plens), ints(ctx, pt)]
            prefix = lq8.SharedPrefix(bufs[-3], bufs[-2], bufs[-1], len(self.plens), pw)
            lq8.prefix_attention_device(ctx, pages, batch, prefix, rows)
        else:
            lq8.paged_attention_device(ctx, pages, batch, rows)
        got = download(dout, self.q.size, self.types[0]).reshape(self.q.shape)
        for b in bufs:
            b.free()
        if not in_place:
            assert np.all(got[self.rows:] == 7.0), "rows behind the last sequence"
            assert np.all(got[:, self.heads * self.dim:] == 7.0), "between the rows"
        return got[:, :self.heads * self.dim].reshape(-1, self.heads, self.dim)

    def want(self, drop=None, scale=None):
        """(out, tolerance); drop(s): positions of sequence s that no page holds."""
        out = np.zeros((self.rows, self.heads, self.dim))
        tol = np.zeros_like(out)
        scale = self.dim ** -0.5 if scale is None else scale
        for s, (r, t) in enumerate(self.seqs):
            g = [i for i in range(len(self.plens)) if self.first[i] <= s < self.first[i + 1]]
            keep = np.ones(t, bool)
            if drop is not None:
                keep[drop(s)] = False
            for i in range(r):
                see = max(0, t - r + i + 1)
                k, v = self.k[s][:see][keep[:see]], self.v[s][:see][keep[:see]]
                for i_g in g:
                    k = np.concatenate([self.k[len(self.seqs) + i_g], k])
                    v = np.concatenate([self.v[len(self.seqs) + i_g], v])
                q = self.q[self.begin[s] + i, :self.heads * self.dim].reshape(self.heads, self.dim).astype(np.float64)
                o, mag, top = attend(q, k.astype(np.float64), v.astype(np.float64), scale)
                at = self.begin[s] + i
                out[at], tol[at] = o, tolerance(o, mag, top, self.dim, len(k), self.types)
        return out, tol

    def check(self, **run):
        got = self.run(**run)[:self.rows]
        out, tol = self.want(scale=run.get("scale"))
        compare(got, out, tol)


def compare(got, out, tol):
    assert np.array_equal(np.isnan(got), np.isnan(out)), "NaN in other places"
    inf = np.isinf(out)
    assert np.array_equal(got[inf], out[inf]), "infinities in other places"
    fine = np.isfinite(out)
    bad = ~(np.abs(got[fine] - out[fine]) <= tol[fine])
    assert not bad.any(), f"{bad.sum()} of {bad.size}, worst {np.max(np.abs(got[fine] - out[fine]) / tol[fine]):.2f} tolerances"


SINGLE = [(1, t) for t in (0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 1025)]
RAGGED = [(0, 0), (1, 5), (3, 1), (17, 17), (0, 9), (64, 100), (65, 65), (2, 700), (130, 131), (4, 0)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 128, 16), (16, 8, 128, 32), (32, 4, 128, 64), (14, 2, 64, 16), (6, 1, 64, 1024),
                                               (20, 1, 128, 16), (34, 2, 64, 128), (65, 1, 128, 256), (1, 1, 64, 16)])
def test_single_tokens(ctx, types, heads, kv, dim, page):
    Batch(ctx, types, SINGLE, heads, kv, dim, page, seed=heads).check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 128, 16), (8, 4, 128, 128), (8, 1, 128, 32), (14, 2, 64, 16), (6, 2, 64, 64),
                                               (40, 2, 128, 16)])
def test_ragged_chunks(ctx, types, heads, kv, dim, page):
    Batch(ctx, types, RAGGED, heads, kv, dim, page, seed=heads + 1, pad=32).check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [2, 3, 5, 8, 9, 16, 20, 33])
def test_few_rows(ctx, types, rows):
    """Drafted tokens: a few rows behind a context, up to and over the row tiles' sizes."""
    Batch(ctx, types, [(rows, 300), (rows, rows), (1, 70), (rows - 1, 1000)], 8, 2, 128, 16, seed=rows).check()


@pytest.mark.parametrize("types", TYPES)
def test_long_sequences_are_split(ctx, types):
    Batch(ctx, types, [(1, 9000), (1, 64), (1, 4097)], 4, 2, 128, 64, seed=3).check()
    Batch(ctx, types, [(37, 3000), (1, 5000)], 4, 1, 64, 32, seed=4).check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("groups", [
    ([0, 5], [1000]),            # one prefix for all
    ([0, 2, 5], [64, 333]),      # two
    ([1, 1, 3], [70, 200]),      # an empty group, a sequence before the first group, two behind the last
    ([0, 3, 5], [0, 17]),        # a prefix of no positions
])
@pytest.mark.parametrize("seqs", [[(1, 1), (1, 0), (1, 100), (1, 17), (1, 513)], [(3, 3), (0, 0), (40, 90), (1, 65), (2, 1)],
                                  [(70, 70), (1, 1), (150, 150), (0, 3), (8, 300)]])
def test_shared_prefixes(ctx, types, groups, seqs):
    Batch(ctx, types, seqs, 8, 2, 128, 16, groups=groups, seed=5).check()


@pytest.mark.parametrize("types", TYPES)
def test_prefix_many_rows(ctx, types):
    Batch(ctx, types, [(1, 1 + i % 40) for i in range(70)], 14, 2, 64, 32, groups=([0, 33, 70], [700, 1500]), seed=6).check()


@pytest.mark.parametrize("types", TYPES)
def test_prefix_equals_its_positions_in_front(ctx, types):
    """The same sequences with the prefix in their own pages: the two calls agree within both tolerances."""
    b = Batch(ctx, types, [(1, 30), (5, 77), (1, 1)], 6, 3, 64, 16, groups=([0, 3], [129]), seed=7)
    got = b.run()[:b.rows]
    c = Batch(ctx, types, [(r, t + 129) for r, t in b.seqs], 6, 3, 64, 16, seed=7)
    c.q = b.q
    for s in range(3):
        c.k[s], c.v[s] = np.concatenate([b.k[3], b.k[s]]), np.concatenate([b.v[3], b.v[s]])
    out, tol = c.want()
    compare(c.run()[:c.rows], out, tol)
    compare(got, out, tol)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", [[(1, 100), (1, 65)], [(70, 100), (3, 40)]])
def test_in_place_and_strides(ctx, types, seqs):
    b = Batch(ctx, types, seqs, 8, 2, 128, 16, seed=8, pad=64, stride=2 * 16 * 128 + 512)
    out, tol = b.want()
    compare(b.run()[:b.rows], out, tol)
    compare(b.run(in_place=True)[:b.rows], out, tol)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", [[(1, 100), (1, 65), (1, 16)], [(70, 100), (3, 65), (16, 16)]])
def test_pages_that_do_not_exist_are_masked(ctx, types, seqs):
    b = Batch(ctx, types, seqs, 4, 2, 128, 16, seed=9)
    table = tables(b.tab[:3], 7, b.rng)
    table[0, 2], table[0, 5], table[1, 0] = -1, b.cache.pages, 2 ** 31 - 1
    table[2, 0] = -(2 ** 31)  # the third sequence has nothing left
    gone = {0: np.r_[32:48, 80:96], 1: np.r_[0:16], 2: np.r_[0:16]}
    out, tol = b.want(drop=lambda s: gone[s][gone[s] < seqs[s][1]])
    compare(b.run(table=table)[:b.rows], out, tol)
    assert np.all(b.run(table=table)[b.begin[2]:b.begin[3]] == 0.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", [[(1, 90), (1, 33)], [(90, 90), (40, 70)]])
def test_values_that_are_not_finite(ctx, types, seqs):
    """Infinite and NaN values reach the rows that see them, and no others; so do NaN keys and queries."""
    b = Batch(ctx, types, seqs, 4, 2, 64, 16, seed=10)
    for s, t in ((0, 60), (1, 32)):
        b.v[s][t, 0, 5], b.v[s][t, 1, 63], b.v[s][t - 20, 0, 9] = np.inf, np.nan, -np.inf
    b.v[0][63, 0, 5] = -np.inf  # inf and -inf: NaN from row 63 on
    b.k[0][80, 1, 3] = np.nan
    b.q[1, 70] = np.nan
    b.q[0, 0] = np.inf
    out, tol = b.want()
    compare(b.run()[:b.rows], out, tol)


@pytest.mark.parametrize("types", TYPES)
def test_scores_of_minus_infinity(ctx, types):
    """Keys whose scores are -inf weigh nothing; a row with no other keys has no answer (0 / 0), unlike one that sees
    nothing."""
    b = Batch(ctx, types, [(70, 70), (1, 130), (1, 0), (1, 64)], 2, 2, 64, 16, seed=11)
    b.q[:, :128] = np.abs(b.q[:, :128]) + rounded(np.float32(0.5), types[0])
    b.q[:] = rounded(b.q, types[0])
    b.k[0][:20, :, 7] = -np.inf
    b.k[1][:100, :, 7] = -np.inf
    b.k[3][:, :, 7] = -np.inf
    out, tol = b.want()
    assert np.isnan(out[:20]).all() and np.isfinite(out[20:72]).all() and np.isnan(out[72]).all()
    compare(b.run()[:b.rows], out, tol)


@pytest.mark.parametrize("types", TYPES)
def test_scores_far_apart(ctx, types):
    """Scores hundreds apart, with the largest first, last and in between; the most negative finite ones."""
    b = Batch(ctx, types, [(80, 300), (1, 257), (1, 400)], 4, 2, 128, 16, seed=12, qstd=40.0)
    b.k[2][:, :, :] = rounded(-np.abs(b.k[2]) * 1e30, types[1])
    b.k[2][399] = rounded(np.abs(b.k[2][399]) * 1e-3 / 1e30, types[1])
    b.q[81] = rounded(np.abs(b.q[81]) + 1, types[0])
    b.check()
    b.check(scale=1e-6)


def test_a_rows_result_does_not_depend_on_other_sequences(ctx):
    a = Batch(ctx, (BF16, BF16), [(1, 2000), (1, 900), (1, 3000)], 8, 2, 128, 16, seed=13)
    x = a.run()
    b = Batch(ctx, (BF16, BF16), [(1, 2000), (1, 3000), (1, 5)], 8, 2, 128, 16, seed=14)
    b.q[0], b.k[0], b.v[0] = a.q[0], a.k[0], a.v[0]
    assert np.array_equal(x[0], b.run()[0])


def test_max_rows_bounds_the_rows(ctx):
    """Rows of a sequence past max_rows are left as they were."""
    b = Batch(ctx, (F32, F32), [(40, 40), (3, 3)], 2, 1, 64, 16, seed=15)
    got = b.run(max_rows=30)
    assert np.all(got[30:40] == 7.0)


def test_far_pages(ctx):
    """Pages whose bytes lie past 2^32: two pages 2^31 elements apart."""
    stride, kv, page, dim = 1 << 31, 1, 16, 64
    rng = np.random.default_rng(16)
    k, v = (rounded(rng.standard_normal((32, dim)), BF16) for _ in range(2))
    q = rounded(rng.standard_normal((1, 2, dim)) * 1.5, BF16)
    big = lq8.DeviceBuffer(ctx, 2 * (stride + 2 * kv * page * dim))  # K pages, V right behind each
    dl, dt = ints(ctx, [32]), ints(ctx, [[1, 0]])
    vbuf = At(big, 2 * kv * page * dim)
    pages = lq8.KVPages(big, vbuf, 2, page, kv, dim, dtype=BF16, page_stride=stride)
    dq, dout = upload(ctx, q, BF16), upload(ctx, q, BF16)
    drows = [upload(ctx, x, BF16) for x in (k, v)]
    # written through the append, too: 32 rows in order
    db = ints(ctx, [0, 32])
    lq8.paged_append_device(ctx, None, pages, lq8.PagedBatch(dl, dt, 1, 2, rows=32, row_begin=db, max_rows=32),
                            lq8.QkvRows(None, drows[0], drows[1], 0, dim, dtype=BF16))
    lq8.paged_attention_device(ctx, pages, lq8.PagedBatch(dl, dt, 1, 2), lq8.AttnRows(dq, dout, 2, dim, dtype=BF16))
    out, mag, top = attend(q[0].astype(np.float64), k[:, None].astype(np.float64), v[:, None].astype(np.float64), dim ** -0.5)
    compare(download(dout, 2 * dim, BF16).reshape(2, dim), out, tolerance(out, mag, top, dim, 32, (BF16, BF16)))
    for b in [big, dl, dt, dq, dout, db] + drows:
        b.free()
