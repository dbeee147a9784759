"""CPU: lq8.paged_plan over batches of all shapes: what the attention calls launch and keep stays within their limits."""
import numpy as np
import pytest

import lq8
from test_paged_cpu import BF16, F32, P, batch, kv, prefix, rows

TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


def draw(rng):
    kvh = int(rng.choice([1, 2, 4, 8, 12, 64]))
    heads = kvh * int(rng.choice([1, 2, 4, 7, 16, 40]))
    dim, page = int(rng.choice([64, 128])), int(rng.choice([16, 64, 256, 1024]))
    act, cache = TYPES[rng.integers(3)]
    n = int(2 ** rng.uniform(0, 12))
    width = max(1, int(2 ** rng.uniform(0, 20)) // page)
    if rng.random() < 0.5:
        b = dict(batch=n, max_pages=width)
        count = most = 1
        total = n
    else:
        most = int(2 ** rng.uniform(0, 11))
        total = max(most, int(n * most * rng.uniform(0.1, 1)))
        b = dict(batch=n, max_pages=width, rows=total, row_begin=P(), max_rows=most)
    if total * heads > 1 << 23:
        return None
    pre = dict(groups=int(rng.integers(1, n + 1)), max_pages=max(1, int(2 ** rng.uniform(0, 17)) // page)) if rng.random() < 0.5 else None
    return dict(kvh=kvh, heads=heads, dim=dim, page=page, act=act, cache=cache, n=n, width=width, most=most, total=total, batch=b, pre=pre)


@pytest.mark.parametrize("seed", range(40))
def test_plans(seed):
    rng = np.random.default_rng(seed)
    done = 0
    while done < 50:
        c = draw(rng)
        if c is None:
            continue
        done += 1
        pages = kv(num_kv_heads=c["kvh"], head_dim=c["dim"], page_size=c["page"], dtype=c["cache"])
        pre = prefix(**c["pre"]) if c["pre"] else None
        p = lq8.paged_plan(pages, batch(**c["batch"]), rows(num_heads=c["heads"], head_dim=c["dim"], dtype=c["act"]), pre)
        G = c["heads"] // c["kvh"]
        parts = [("own", c["width"] * c["page"], c["n"], c["most"])]
        if pre:
            parts.append(("prefix", c["pre"]["max_pages"] * c["page"], c["pre"]["groups"], c["total"]))
        slots, blocks = 0, 0
        for name, positions, spans, most in parts:
            tile, splits, chunk = p[name + "_rows"], p[name + "_splits"], p[name + "_chunk"]
            assert tile in (16, 128)
            assert chunk & (chunk - 1) == 0 and 64 <= chunk <= 512
            assert 1 <= splits <= -(-positions // chunk)
            # row tiles for every way of sharing the rows out
            full = min(spans * -(-most * G // tile), (c["total"] * G + (tile - 1) * min(spans, c["total"])) // tile)
            tiles = spans if tile == 16 and most * G <= 16 else full
            blocks += tiles * c["kvh"] * splits
            slots += splits
        assert p["workgroups"] == blocks < 2 ** 31 / 256
        assert p["scratch_bytes"] == (slots * c["total"] * c["heads"] * (c["dim"] * 4 + 8) if slots > 1 else 0)


def test_single_rows_take_small_tiles_and_chunks_large_ones():
    one = lq8.paged_plan(kv(), batch(batch=64, max_pages=500), rows())
    assert one["own_rows"] == 16 and one["prefix_rows"] == 0
    many = lq8.paged_plan(kv(), batch(batch=3, rows=6000, row_begin=P(), max_rows=2000, max_pages=500), rows())
    assert many["own_rows"] == 128
    both = lq8.paged_plan(kv(dtype=BF16), batch(batch=64, max_pages=50), rows(num_heads=32, dtype=BF16), prefix(groups=1, max_pages=512))
    assert both["own_rows"] == 16 and both["prefix_rows"] == 128


def test_shared_prefixes_of_many_groups_stay_small():
    """A thousand groups of a few rows: about a row tile each, not one for every row of the batch in each."""
    p = lq8.paged_plan(kv(), batch(batch=3000, max_pages=4), rows(), prefix(groups=1000, max_pages=20))
    assert p["workgroups"] < 8 * (3000 + 2 * 1000) * 10
