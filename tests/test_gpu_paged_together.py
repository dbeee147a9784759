"""GPU: the operators of the paged cache as a serving loop calls them: prompts, then tokens, behind a prefix that is
prefilled once, by the rotation, the append and both attentions, each step against the formulas in 64 bits; calls from two
contexts at once; buffers of one call grown by the next."""
import threading

import numpy as np
import pytest

import lq8
from paged_common import BF16, F32, HALF, attend, download, from_bf16, ints, rounded, tables, to_bf16, tolerance, upload
from test_gpu_paged_attention import TYPES, Batch, compare
from test_gpu_rope import turned

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e6


def rms(x, w):
    """RmsNorm with input, weight and result rounded to bf16."""
    x, w = (rounded(y, BF16).astype(np.float64) for y in (x, w))
    return rounded((x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w).astype(np.float32), BF16).astype(np.float64)


class Server:
    """Sequences behind one shared prefix; K and V are read back from the pages, so that each step's attention is checked
    with what the append stored, and the append with the formulas."""

    def __init__(self, ctx, types, seed, heads=8, kv=2, dim=64, page=16, n=3, sections=()):
        self.ctx, self.types, self.heads, self.kvh, self.dim, self.page, self.n = ctx, types, heads, kv, dim, page, n
        self.rng = np.random.default_rng(seed)
        self.width, self.pwidth = 12, 9
        pages = n * self.width + self.pwidth + 1
        order = self.rng.permutation(pages)
        self.table = order[:n * self.width].reshape(n, self.width)
        self.ptable = order[n * self.width:n * self.width + self.pwidth].reshape(1, -1)
        self.pages = lq8.KVPages.alloc(ctx, pages, page, kv, dim, dtype=types[1])
        self.pages_n, self.lengths, self.plen = pages, np.zeros(n, int), 0
        self.rope = lq8.Rope(ctx, dim, THETA, sections=sections, interleaved=len(sections) == 3)
        self.norms = [np.float32(1 + 0.1 * self.rng.standard_normal(dim)) for _ in range(2)]
        self.dnorms = [lq8.DeviceBuffer.from_array(ctx, x) for x in self.norms]

    def held(self, which, table, length):
        buf = self.pages.owned[which]
        x = download(buf, self.pages_n * self.kvh * self.page * self.dim, self.types[1]).reshape(self.pages_n, self.kvh, self.page, self.dim)
        return x[table].transpose(0, 2, 1, 3).reshape(-1, self.kvh, self.dim)[:length].astype(np.float64)

    def step(self, counts, prefix=False, positions=None):
        """counts[s] new rows of each sequence (prefix: of the prefix itself), with random projections."""
        ctx, (act, cache), h, g, d = self.ctx, self.types, self.heads, self.kvh, self.dim
        counts = np.asarray(counts)
        n, rows = len(counts), int(sum(counts))
        if prefix:
            self.plen += rows
            lengths, table = np.array([self.plen]), self.ptable
        else:
            self.lengths = self.lengths + counts
            lengths, table = self.lengths, self.table
        begin = np.concatenate([[0], np.cumsum(counts)])
        x = rounded(self.rng.standard_normal((rows, h + 2 * g, d)) * 2, act)
        dx = upload(ctx, x, act)
        es = 4 if act == F32 else 2
        bufs = [dx, ints(ctx, lengths), ints(ctx, table), ints(ctx, begin), upload(ctx, np.zeros((rows, h, d)), act)]
        batch = lq8.PagedBatch(bufs[1], bufs[2], n, table.shape[1], rows=rows, row_begin=bufs[3], max_rows=int(max(counts)))

        class Part:
            def __init__(self, at):
                self.ptr = lq8.C.c_void_p(dx.ptr.value + at * d * es)

        axes = self.rope.cfg.axes
        at = np.concatenate([np.arange(l - c, l) for l, c in zip(lengths, counts)])
        if positions is None:
            pos = np.tile(at + (0 if prefix else self.plen), (axes, 1))
        else:
            pos = positions(at)
        bufs.append(ints(ctx, pos))
        wide = (h + 2 * g) * d
        lq8.paged_append_device(ctx, self.rope, self.pages, batch, lq8.QkvRows(
            Part(0), Part(h), Part(h + g), h, d, q_out=bufs[4], stride=wide, q_norm=self.dnorms[0], k_norm=self.dnorms[1],
            eps=EPS, positions=bufs[5], positions_stride=rows, dtype=act))
        q_dev = bufs[4]
        arows = lq8.AttnRows(q_dev, q_dev, h, d, dtype=act)  # in place
        q = download(q_dev, rows * h * d, act).reshape(rows, h, d).astype(np.float64)
        if prefix or not self.plen:
            lq8.paged_attention_device(ctx, self.pages, batch, arows)
        else:
            bufs += [ints(ctx, [0, n]), ints(ctx, [self.plen]), ints(ctx, self.ptable)]
            lq8.prefix_attention_device(ctx, self.pages, batch, lq8.SharedPrefix(bufs[-3], bufs[-2], bufs[-1], 1, self.pwidth), arows)
        got = download(q_dev, rows * h * d, act).reshape(rows, h, d)
        # the append: a norm rounds to bf16 (half a step more where 32-bit sums fall the other way), then the rotation
        x64 = x.astype(np.float64)
        for what, have, norm in ((x64[:, :h], q, self.norms[0]), (x64[:, h:h + g], None, self.norms[1])):
            want, tol = turned(rms(what, norm), self.rope.cfg, pos)
            tol = tol + 2 * HALF[BF16] * np.hypot(want, 0) + 2 * HALF[BF16] * np.abs(rms(what, norm)).max()
            if have is None:
                have = np.concatenate([self.held(0, table[s], lengths[s])[lengths[s] - counts[s]:] for s in range(n)])
            assert np.all(np.abs(have - want) <= tol)
        v = np.concatenate([self.held(1, table[s], lengths[s])[lengths[s] - counts[s]:] for s in range(n)])
        assert np.array_equal(v, rounded(x[:, h + g:], cache))
        # the attention, with what is stored
        pk, pv = ([], []) if prefix or not self.plen else (self.held(0, self.ptable[0], self.plen), self.held(1, self.ptable[0], self.plen))
        for s in range(n):
            k, v = self.held(0, table[s], lengths[s]), self.held(1, table[s], lengths[s])
            for i in range(counts[s]):
                see = lengths[s] - counts[s] + i + 1
                kk, vv = (np.concatenate([p, y[:see]]) if len(p) else y[:see] for p, y in ((pk, k), (pv, v)))
                out, mag, top = attend(q[begin[s] + i], kk, vv, d ** -0.5)
                compare(got[begin[s] + i], out, tolerance(out, mag, top, d, len(kk), self.types))
        for b in bufs:
            b.free()

    def close(self):
        self.pages.free()
        for b in self.dnorms:
            b.free()
        self.rope.free()


@pytest.mark.parametrize("types", TYPES)
def test_prompts_then_tokens_behind_a_prefix(ctx, types):
    s = Server(ctx, types, 1)
    s.step([100], prefix=True)
    s.step([33], prefix=True)  # the prefix in two pieces
    s.step([40, 1, 17])
    for _ in range(3):
        s.step([1, 1, 1])
    s.step([3, 0, 5])  # drafted tokens
    s.step([0, 60, 1])
    s.close()


@pytest.mark.parametrize("types", TYPES)
def test_prompts_with_images(ctx, types):
    """Positions with three axes: a patch's time, row and column."""
    s = Server(ctx, types, 2, heads=4, kv=4, dim=128, page=32, sections=(24, 20, 20))
    s.step([70, 9, 30], positions=lambda at: np.stack([at // 12, at % 12 // 4, at % 4]))
    s.step([1, 1, 1], positions=lambda at: np.stack([at, at, at]))
    s.close()


def test_two_contexts_at_once(ctx):
    """Threads with a context each, over pages that they share; every result is the one of a single thread."""
    b = Batch(ctx, (BF16, BF16), [(1, 3000), (1, 500), (1, 4100)], 8, 2, 128, 16, seed=3)
    c = Batch(ctx, (F32, F32), [(90, 400), (33, 700)], 8, 2, 128, 16, seed=4)
    want = [b.run(), c.run()]
    bad = []

    def work(which):
        try:
            with lq8.Context(0) as own:
                x = Batch(own, (BF16, BF16), [(1, 3000), (1, 500), (1, 4100)], 8, 2, 128, 16, seed=3) if which == 0 else \
                    Batch(own, (F32, F32), [(90, 400), (33, 700)], 8, 2, 128, 16, seed=4)
                for _ in range(8):
                    x.cache.k[:], x.cache.v[:] = np.nan, np.nan
                    if not np.array_equal(x.run(), want[which]):
                        bad.append(which)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i % 2,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_scratch_grows_between_calls(ctx):
    """A fresh context's first calls, each with more to keep than the last, and a small one again."""
    with lq8.Context(0) as own:
        for seqs in ([(1, 20)], [(1, 700)], [(1, 9000), (1, 5)], [(1, 3000)] * 9, [(1, 20)]):
            Batch(own, (F32, BF16), seqs, 4, 2, 64, 16, seed=len(seqs)).check()


def test_append_of_fewer_rows_than_a_sequence_has(ctx):
    """Rows past max_rows are not written, the others at their own positions."""
    rng = np.random.default_rng(5)
    kv, dim, page = 2, 64, 16
    x = rounded(rng.standard_normal((40, kv, dim)), F32)
    pages = [lq8.DeviceBuffer.from_array(ctx, np.full((4, kv, page, dim), 7.0, np.float32)) for _ in range(2)]
    bufs = [upload(ctx, x, F32), ints(ctx, [45]), ints(ctx, [[2, 0, 3]]), ints(ctx, [0, 40])]
    lq8.paged_append_device(ctx, None, lq8.KVPages(pages[0], pages[1], 4, page, kv, dim), lq8.PagedBatch(
        bufs[1], bufs[2], 1, 3, rows=40, row_begin=bufs[3], max_rows=30), lq8.QkvRows(None, bufs[0], bufs[0], 0, dim))
    got = pages[0].download(np.float32, 4 * kv * page * dim).reshape(4, kv, page, dim)[[2, 0, 3]].transpose(0, 2, 1, 3).reshape(48, kv, dim)
    assert np.array_equal(got[5:35], x[:30]) and np.all(got[:5] == 7.0) and np.all(got[35:] == 7.0)
    for b in bufs + pages:
        b.free()
