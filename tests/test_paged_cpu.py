"""CPU: what the operators of the paged cache refuse (their checks need no device), the axes of the rotation's pairs, and
the plan of the attention calls over a range of batches."""
import ctypes as C

import numpy as np
import pytest

import lq8

F32, BF16 = lq8.DTYPE_F32, lq8.DTYPE_BF16


class P:
    """An address nobody follows: these checks touch no memory."""

    def __init__(self, at=0x10000):
        self.ptr = C.c_void_p(at)


def kv(**o):
    a = dict(k=P(), v=P(), num_pages=100, page_size=16, num_kv_heads=8, head_dim=128, dtype=F32, page_stride=0)
    a.update(o)
    return lq8.KVPages(**a)


def batch(**o):
    a = dict(lengths=P(), pages=P(), batch=4, max_pages=10)
    a.update(o)
    return lq8.PagedBatch(**a)


def rows(**o):
    a = dict(q=P(), out=P(), num_heads=16, head_dim=128)
    a.update(o)
    return lq8.AttnRows(**a)


def prefix(**o):
    a = dict(seq_begin=P(), lengths=P(), pages=P(), groups=2, max_pages=3)
    a.update(o)
    return lq8.SharedPrefix(**a)


REFUSED = [
    (kv(k=None), batch(), rows(), None, lq8.InvalidArgument),
    (kv(v=P(0x10008)), batch(), rows(), None, lq8.InvalidArgument),
    (kv(dtype=0), batch(), rows(), None, lq8.DTypeMismatch),
    (kv(page_size=24), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(page_size=8), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(page_size=2048), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(page_size=0), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(num_kv_heads=0), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(num_kv_heads=1025), batch(), rows(num_heads=1025), None, lq8.ShapeMismatch),
    (kv(num_pages=0), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(num_pages=2 ** 31), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(head_dim=96), batch(), rows(head_dim=96), None, lq8.ShapeMismatch),
    (kv(page_stride=8 * 16 * 128 - 4), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(page_stride=8 * 16 * 128 + 2), batch(), rows(), None, lq8.InvalidArgument),
    (kv(page_stride=2 ** 58), batch(), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(lengths=None), rows(), None, lq8.InvalidArgument),
    (kv(), batch(pages=None), rows(), None, lq8.InvalidArgument),
    (kv(), batch(rows=5), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(rows=9, row_begin=P(), max_rows=0), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(rows=9, row_begin=P(), max_rows=10), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(max_pages=0), rows(), None, lq8.ShapeMismatch),
    (kv(page_size=1024), batch(max_pages=2 ** 21), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(batch=65537, rows=65537), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(rows=2 ** 23 + 1, row_begin=P()), rows(), None, lq8.ShapeMismatch),
    (kv(), batch(), rows(q=None), None, lq8.InvalidArgument),
    (kv(), batch(), rows(out=P(0x10004)), None, lq8.InvalidArgument),
    (kv(), batch(), rows(num_heads=12), None, lq8.ShapeMismatch),
    (kv(), batch(), rows(num_heads=0), None, lq8.ShapeMismatch),
    (kv(), batch(), rows(q_stride=16 * 128 - 4), None, lq8.ShapeMismatch),
    (kv(), batch(), rows(q_stride=16 * 128 + 1), None, lq8.InvalidArgument),
    (kv(), batch(), rows(out=P(), q_stride=16 * 128 + 4), None, lq8.ShapeMismatch),  # in place with two strides
    (kv(), batch(), rows(scale=0.0), None, lq8.InvalidArgument),
    (kv(), batch(), rows(scale=-1.0), None, lq8.InvalidArgument),
    (kv(), batch(), rows(scale=float("nan")), None, lq8.InvalidArgument),
    (kv(), batch(), rows(scale=float("inf")), None, lq8.InvalidArgument),
    (kv(), batch(), rows(scale=3e38), None, lq8.InvalidArgument),
    (kv(), batch(), rows(dtype=BF16), None, lq8.DTypeMismatch),  # bf16 rows over f32 pages
    (kv(), batch(), rows(dtype=0), None, lq8.DTypeMismatch),
    (kv(), batch(batch=1, rows=2 ** 19 + 1, row_begin=P(), max_rows=5), rows(), None, lq8.ShapeMismatch),  # 2^23 rows of heads
    (kv(num_kv_heads=1024), batch(batch=65536, rows=8000, row_begin=P()), rows(num_heads=1024), None, lq8.ShapeMismatch),  # 2^24 workgroups
    (kv(), batch(), rows(), prefix(groups=5), lq8.ShapeMismatch),
    (kv(), batch(), rows(), prefix(seq_begin=None), lq8.InvalidArgument),
    (kv(), batch(), rows(), prefix(max_pages=0), lq8.ShapeMismatch),
    (kv(page_size=1024), batch(), rows(), prefix(max_pages=2 ** 21), lq8.ShapeMismatch),
    (kv(head_dim=64), batch(), rows(), None, lq8.ShapeMismatch),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_attention_refuses(case):
    pages, b, r, p, error = REFUSED[case]
    with pytest.raises(error):
        lq8.paged_plan(pages, b, r, p)
    # the calls themselves make the same checks, before they look at their context
    class NoContext:
        handle = None

    with pytest.raises(error):
        if p is None:
            lq8.paged_attention_device(NoContext, pages, b, r)
        else:
            lq8.prefix_attention_device(NoContext, pages, b, p, r)


def test_null_descriptions_and_contexts():
    L, bad = lq8.lib(), lq8.InvalidArgument.status
    assert L.lq8_paged_attention_device(None, None, None, None) == bad
    assert L.lq8_paged_attention_device(None, kv().c, batch().c, None) == bad
    assert L.lq8_prefix_attention_device(None, kv().c, batch().c, None, rows().c) == bad
    assert L.lq8_paged_attention_device(C.c_void_p(0x1234), kv().c, batch().c, rows().c) == bad
    assert L.lq8_paged_append_device(None, None, None, None, None) == bad
    assert L.lq8_paged_append_device(None, None, kv().c, batch().c, None) == bad
    assert L.lq8_paged_plan(kv().c, batch().c, None, rows().c, 256, None) == bad
    assert L.lq8_rope_free(C.c_void_p(0x1234)) == bad
    assert L.lq8_rope_device(C.c_void_p(0x1234), None, None) == bad
    assert L.lq8_rope_create(None, None, None) == bad
    assert L.lq8_rope_axes(None, None) == bad


def qkv(**o):
    a = dict(q=P(), k=P(0x20000), v=P(0x30000), num_heads=16, head_dim=128, q_out=P(0x40000))
    a.update(o)
    return lq8.QkvRows(**a)


@pytest.mark.parametrize("pages,b,r,error", [
    (kv(), batch(), qkv(q_out=None), lq8.InvalidArgument),
    (kv(), batch(), qkv(q=None), lq8.InvalidArgument),
    (kv(), batch(), qkv(k=None), lq8.InvalidArgument),
    (kv(), batch(), qkv(v=P(0x30004)), lq8.InvalidArgument),
    (kv(), batch(), qkv(num_heads=0), lq8.ShapeMismatch),
    (kv(), batch(), qkv(stride=1024), lq8.ShapeMismatch),  # below the query row
    (kv(), batch(), qkv(stride=2050), lq8.InvalidArgument),
    (kv(), batch(), qkv(q_out=P(), stride=4096), lq8.ShapeMismatch),  # in place with two strides
    (kv(), batch(), qkv(dtype=BF16), lq8.DTypeMismatch),
    (kv(), batch(), qkv(q_norm=P(), eps=-1.0), lq8.InvalidArgument),
    (kv(), batch(), qkv(q_norm=P(), eps=float("nan")), lq8.InvalidArgument),
    (kv(), batch(), qkv(positions=P(), positions_stride=3), lq8.ShapeMismatch),
    (kv(page_size=40), batch(), qkv(), lq8.ShapeMismatch),
    (kv(), batch(max_pages=0), qkv(), lq8.ShapeMismatch),
    (kv(), batch(), qkv(), lq8.InvalidArgument),  # no context
])
def test_append_refuses(pages, b, r, error):
    class NoContext:
        handle = None

    with pytest.raises(error):
        lq8.paged_append_device(NoContext, None, pages, b, r)


def test_rope_axes_of_pairs():
    # sections side by side
    a = lq8.rope_axes(lq8.rope_config(128, 1e6, sections=(16, 24, 24)))
    assert a.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    # interleaved: t h w t h w ... while the h and w sections last, then t
    a = lq8.rope_axes(lq8.rope_config(128, 1e6, sections=(24, 20, 20), interleaved=True))
    assert a.tolist() == [0, 1, 2] * 20 + [0] * 4
    a = lq8.rope_axes(lq8.rope_config(64, 1e4, rotary_dim=32, sections=(10, 4, 2), interleaved=True))
    assert a.tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 0, 0, 1, 0, 0, 0, 0, 0]
    assert lq8.rope_axes(lq8.rope_config(128, 1e6)).tolist() == [0] * 64
    a = lq8.rope_axes(lq8.rope_config(80, 1e4, sections=(20, 20)))
    assert a.tolist() == [0] * 20 + [1] * 20
    a = lq8.rope_axes(lq8.rope_config(64, 1e4, sections=(0, 32, 0, 0)))
    assert a.tolist() == [1] * 32


@pytest.mark.parametrize("args,error", [
    (dict(head_dim=120), lq8.ShapeMismatch), (dict(head_dim=0), lq8.ShapeMismatch), (dict(head_dim=272), lq8.ShapeMismatch),
    (dict(head_dim=128, rotary_dim=144), lq8.ShapeMismatch), (dict(head_dim=128, rotary_dim=24), lq8.ShapeMismatch),
    (dict(head_dim=128, rotary_dim=0), lq8.ShapeMismatch), (dict(head_dim=128, sections=(16, 24, 25)), lq8.ShapeMismatch),
    (dict(head_dim=128, sections=(63,)), lq8.ShapeMismatch), (dict(head_dim=128, sections=(0, 0)), lq8.ShapeMismatch),
    (dict(head_dim=128, sections=(2 ** 31, 2 ** 31, 64)), lq8.ShapeMismatch),
    (dict(head_dim=128, sections=(20, 22, 22), interleaved=True), lq8.ShapeMismatch),
    (dict(head_dim=128, sections=(1, 1, 1, 1, 60)), lq8.InvalidArgument),
    (dict(head_dim=128, theta=0.0), lq8.InvalidArgument), (dict(head_dim=128, theta=float("inf")), lq8.InvalidArgument),
    (dict(head_dim=128, theta=float("nan")), lq8.InvalidArgument),
])
def test_rope_refuses(args, error):
    with pytest.raises(error):
        lq8.rope_axes(lq8.rope_config(**dict(dict(theta=1e6), **args)))


def test_rope_layout_refused():
    c = lq8.rope_config(128, 1e6)
    c.layout = 2
    with pytest.raises(lq8.InvalidArgument):
        lq8.rope_axes(c)
    c = lq8.rope_config(128, 1e6)
    c.axes = 5
    with pytest.raises(lq8.InvalidArgument):
        lq8.rope_axes(c)
    c.axes = 0
    with pytest.raises(lq8.InvalidArgument):
        lq8.rope_axes(c)


def test_empty_batches_have_a_plan():
    for b in (batch(batch=0, rows=0), batch(batch=3, rows=0, row_begin=P())):
        assert lq8.paged_plan(kv(), b, rows())["workgroups"] == 0
