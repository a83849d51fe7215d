"""The operators in few bits on the device, bit for bit against the oracle (oracle/narrow.py: the definitions in whole
numbers), at the sizes, levels and places where a tile, a chunk, a shift or a mask can go wrong."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import narrow as orc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def space(n):
    return torch.empty(max(16, n), dtype=torch.uint8, device="cuda")


@pytest.fixture(scope="module")
def tabs(sm):
    return sm.tables()


@pytest.fixture(scope="module")
def dtabs(sm, tabs):
    return sm.Tables(tabs)


def plate(rng, nin, nout, small=False):
    w = rng.integers(-128, 128, (nin, nout)).astype(np.int8)
    e = rng.integers(-40, 12, nout).astype(np.int32) if not small else rng.integers(-12, -6, nout).astype(np.int32)
    return w, e, rng.integers(-(1 << 20), 1 << 20, nout)


def rows_of(rng, shape, lo=0, hi=40):
    """rows of very different sizes"""
    x = rng.standard_normal(shape) * 2.0 ** rng.integers(lo, hi, shape[:-1] + (1,))
    return np.round(x).astype(np.int64)


# ---- the product
@pytest.mark.parametrize("rows,nin,nout", [(1, 768, 2304), (1, 1, 1), (2, 63, 17), (16, 64, 16), (17, 65, 15), (31, 129, 48),
                                           (33, 1000, 33), (64, 320, 100), (65, 2051, 31), (129, 200, 70), (300, 72, 130),
                                           (1, 9001, 5), (3, 20000, 20), (700, 130, 1000),
                                           (1025, 64, 2100), (130, 100, 16500), (400, 200, 300)])
def test_product(sm, rows, nin, nout):
    rng = np.random.default_rng(rows * 7 + nin)
    w, e, b = plate(rng, nin, nout)
    X = rows_of(rng, (rows, nin))
    p = sm.Plate8(w, e, b)
    x, out = dev(X), torch.full((rows, nout), -7, dtype=torch.int64, device="cuda")
    n = p.work_bytes(rows)
    wk = space(n)
    p.product(x.data_ptr(), rows, out.data_ptr(), wk.data_ptr(), n, stream=stream())
    assert np.array_equal(out.cpu().numpy(), orc.product(X, w, e, b))


@pytest.mark.parametrize("rows,nin,nout", [(193, 64, 46797), (260, 70, 46848), (1040, 40, 8192), (1100, 200, 16000), (8, 143, 20000)])
def test_product_of_many_tiles(sm, rows, nin, nout):
    """results too many for the row by row oracle: its formula over the whole array (piles below 2^53, so exact in float64)"""
    rng = np.random.default_rng(rows)
    w, e, b = plate(rng, nin, nout, True)
    X = rows_of(rng, (rows, nin), 8, 24)
    p = sm.Plate8(w, e, b)
    x, n = dev(X), p.work_bytes(rows)
    out, wk = torch.full((rows, nout), -7, dtype=torch.int64, device="cuda"), space(n)
    p.product(x.data_ptr(), rows, out.data_ptr(), wk.data_ptr(), n, stream=stream())
    x8, sh = zip(*(orc.digits(r, 8) for r in X))
    pile = np.rint(np.array(x8, np.float64) @ w.astype(np.float64)).astype(np.int64)
    s = -(e.astype(np.int64)[None, :] + np.array(sh, np.int64)[:, None])
    up = np.maximum(s, 0)
    want = np.where(s > 0, (pile + (np.int64(1) << np.maximum(s - 1, 0))) >> up, pile << np.maximum(-s, 0)) + b
    assert np.array_equal(out.cpu().numpy(), want)


def test_product_edges(sm):
    """rows of zeros, of the largest and smallest values, a pile at the edge of 32 bits, powers that shift everything out or
    past 64 bits, biases that wrap"""
    nin, nout = 131071, 16
    w = np.full((nin, nout), -128, np.int8)
    w[:, 1] = 127
    e = np.array([0, 0, -100, -1024, 20, 40, 100, 1024, -17, -16, -15, -1, -31, -63, -64, -65], np.int32)
    b = np.array([0, (1 << 63) - 1, -1, 5] * 4, np.int64)
    X = np.zeros((5, nin), np.int64)
    X[1] = -(1 << 63)
    X[2] = (1 << 63) - 1
    X[3] = -128
    X[4, ::2] = 127
    p = sm.Plate8(w, e, b)
    n = p.work_bytes(5)
    x, out, wk = dev(X), torch.empty((5, nout), dtype=torch.int64, device="cuda"), space(n)
    p.product(x.data_ptr(), 5, out.data_ptr(), wk.data_ptr(), n, stream=stream())
    assert np.array_equal(out.cpu().numpy(), orc.product(X, w, e, b))


def test_product_strides(sm):
    """rows inside wider ones: what is beside them is neither read nor written"""
    rng = np.random.default_rng(11)
    rows, nin, nout = 37, 100, 50
    w, e, b = plate(rng, nin, nout, True)
    X = rows_of(rng, (rows, 131), 3, 20)
    X[:, :5] = X[:, 105:] = 1 << 60
    p = sm.Plate8(w, e, b)
    n = p.work_bytes(rows)
    x, out, wk = dev(X), torch.full((rows, 61), 9, dtype=torch.int64, device="cuda"), space(n)
    p.product(x.data_ptr() + 40, rows, out.data_ptr() + 24, wk.data_ptr(), n, x_stride=131, out_stride=61, stream=stream())
    got = out.cpu().numpy()
    assert np.array_equal(got[:, 3:53], orc.product(X[:, 5:105], w, e, b))
    assert np.all(got[:, :3] == 9) and np.all(got[:, 53:] == 9)


def test_product_refusals(sm):
    p = sm.Plate8(np.ones((8, 4), np.int8), np.zeros(4, np.int32), np.zeros(4, np.int64))
    x, out, wk = dev(np.zeros((2, 8), np.int64)), dev(np.zeros((2, 4), np.int64)), space(p.work_bytes(2))
    ok = dict(x=x.data_ptr(), rows=2, out=out.data_ptr(), work=wk.data_ptr(), work_bytes=p.work_bytes(2))
    for bad in (dict(x=0), dict(out=0), dict(work=0), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(x_stride=7), dict(out_stride=3),
                dict(work_bytes=10), dict(x=x.data_ptr() + 4), dict(work=wk.data_ptr() + 8)):
        with pytest.raises(sm.SmError) as e:
            p.product(**{**ok, **bad})
        assert e.value.code == -1
    p.product(**{**ok, "rows": 0})


# ---- the cache
SHAPES = [(1, 1, 64, 1, 4), (2, 3, 64, 200, 4), (3, 2, 80, 130, 8), (2, 1, 128, 300, 4), (1, 2, 256, 70, 4), (2, 2, 1, 65, 8),
          (1, 1, 256, 129, 8), (2, 5, 40, 64, 4), (2, 2, 128, 100, 8), (1, 2, 64, 150, 8), (1, 1, 100, 190, 4)]


def filled(sm, rng, shape, lo=0, hi=40):
    """a cache with every position written, by calls of uneven numbers of rows, and the oracle's"""
    streams, heads, dim, ctx, bits = shape
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    buf = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda")
    p, i = 0, 0
    while p < ctx:
        n = min([1, 37, 1, 64, 100][i % 5], ctx - p)
        k, v = (rows_of(rng, (streams, n, heads, dim), lo, hi) for _ in range(2))
        start = np.full(streams, p, np.int32)
        dk, dv, ds = dev(k), dev(v), dev(start)
        c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), n, ds.data_ptr(), stream=stream())
        o.write(k, v, start)
        p, i = p + n, i + 1
    return c, o, buf


def read_all(c, shape, rows, start, count=None):
    streams, heads, dim, ctx, bits = shape
    k, v = (torch.full((streams, rows, heads, dim), 77, dtype=torch.int64, device="cuda") for _ in range(2))
    ds, dc = dev(start), None if count is None else dev(count)
    return k, v, ds, dc


def check_read(c, o, buf, shape, rows, start, count=None):
    k, v, ds, dc = read_all(c, shape, rows, start, count)
    c.read(buf.data_ptr(), k.data_ptr(), v.data_ptr(), rows, ds.data_ptr(), dc.data_ptr() if dc is not None else 0, stream=stream())
    wk, wv = (np.full(tuple(k.shape), 77, np.int64) for _ in range(2))
    o.read(rows, start, count, wk, wv)
    assert np.array_equal(k.cpu().numpy(), wk) and np.array_equal(v.cpu().numpy(), wv)


@pytest.mark.parametrize("shape", SHAPES)
def test_write_and_read_back(sm, shape):
    rng = np.random.default_rng(sum(shape))
    c, o, buf = filled(sm, rng, shape)
    check_read(c, o, buf, shape, shape[3], np.zeros(shape[0], np.int32))


@pytest.mark.parametrize("bits", [4, 8])
def test_rewritten_rows_leave_their_neighbours(sm, bits):
    """single positions and short runs written again anywhere in a tile, ragged over the streams, with rows that are not
    there: their neighbours' digits, the ones that share their bytes too, stay"""
    shape = (3, 2, 72, 150, bits)
    rng = np.random.default_rng(bits)
    c, o, buf = filled(sm, rng, shape)
    for start, count, n in (([0, 31, 149], [1, 1, 1], 1), ([32, 33, 64], [1, 0, 1], 1), ([60, -3, 145], [9, 9, 9], 9),
                            ([-70, 140, 0], [70, 70, 70], 70), ([10, 200, -9], [5, 5, 5], 5), ([63, 1, 95], [-4, 1000, 2], 66),
                            ([2147483647, -2147483648, 5], [66, 66, 66], 66)):
        k, v = (rows_of(rng, (3, n, 2, 72), 0, 62) for _ in range(2))
        start, count = np.array(start, np.int32), np.array(count, np.int32)
        dk, dv, ds, dc = dev(k), dev(v), dev(start), dev(count)
        c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), n, ds.data_ptr(), dc.data_ptr(), stream=stream())
        o.write(k, v, start, count)
        check_read(c, o, buf, shape, 150, np.zeros(3, np.int32))
        check_read(c, o, buf, shape, n, start, count)


def test_edge_rows(sm):
    """zeros, single units, the largest and smallest int64"""
    for bits in (4, 8):
        shape = (1, 1, 64, 6, bits)
        x = np.zeros((1, 6, 1, 64), np.int64)
        x[0, 1, 0, 5] = -1
        x[0, 2] = (1 << 63) - 1
        x[0, 3] = -(1 << 63)
        x[0, 4, 0, :2] = [-(1 << (bits - 1)), (1 << (bits - 1)) - 1]
        x[0, 5, 0, ::3] = 1 << (bits - 1)
        c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
        buf, dx, ds = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda"), dev(x), dev(np.zeros(1, np.int32))
        c.write(buf.data_ptr(), dx.data_ptr(), dx.data_ptr(), 6, ds.data_ptr(), stream=stream())
        o.write(x, x, [0])
        check_read(c, o, buf, shape, 6, np.zeros(1, np.int32))


def test_parts_of_wider_rows(sm):
    """k and v as parts of a qkv row, streams further apart than their rows"""
    rng = np.random.default_rng(8)
    shape = (2, 3, 64, 40, 4)
    qkv = rows_of(rng, (2, 50, 576), 10, 20)
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    buf, d, ds = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda"), dev(qkv), dev(np.array([2, 0], np.int32))
    c.write(buf.data_ptr(), d.data_ptr() + 192 * 8, d.data_ptr() + 384 * 8, 30, ds.data_ptr(), row_stride=576,
            stream_stride=50 * 576, stream=stream())
    o.write(qkv[:, :30, 192:384].reshape(2, 30, 3, 64), qkv[:, :30, 384:].reshape(2, 30, 3, 64), [2, 0])
    check_read(c, o, buf, shape, 40, np.zeros(2, np.int32))


# ---- the attention
def attend(c, o, buf, dtabs, tabs, shape, rng, group, rows, start, count, span, scale=None, lo=10, hi=20):
    streams, heads, dim, ctx, bits = shape
    q = rows_of(rng, (streams, rows, heads * group, dim), lo, hi)
    out = torch.full(q.shape, 55, dtype=torch.int64, device="cuda")
    n = c.work_bytes(heads * group, rows, span)
    dq, ds, wk = dev(q), dev(np.asarray(start, np.int32)), space(n)
    dc = None if count is None else dev(np.asarray(count, np.int32))
    c.attend(dtabs, buf.data_ptr(), dq.data_ptr(), heads * group, rows, span, ds.data_ptr(), 0 if dc is None else dc.data_ptr(),
             out.data_ptr(), wk.data_ptr(), n, scale=scale, stream=stream())
    want = np.full(q.shape, 55, np.int64)
    o.attend(tabs, q, start, count, span, c.scale if scale is None else scale, want)
    assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("group", [1, 3, 8, 13, 20])
@pytest.mark.parametrize("shape", [(2, 2, 64, 600, 4), (2, 1, 128, 520, 4), (1, 1, 256, 300, 4), (2, 2, 64, 300, 8),
                                   (1, 2, 96, 530, 8), (1, 1, 200, 260, 8), (2, 1, 7, 130, 4)])
def test_one_row(sm, dtabs, tabs, shape, group):
    """one new row a stream, one stream at the context's end, the other nearer its beginning"""
    rng = np.random.default_rng(group)
    c, o, buf = filled(sm, rng, shape, 12, 20)
    start = [shape[3] - 1, 70][:shape[0]]
    attend(c, o, buf, dtabs, tabs, shape, rng, group, 1, start, None, shape[3])


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 255, 256, 257, 511, 512, 513])
def test_lengths(sm, dtabs, tabs, n):
    """every edge of a tile and of a chunk; a span wider than the row needs changes nothing"""
    for shape in ((1, 1, 64, 513, 4), (1, 1, 128, 513, 8)):
        rng = np.random.default_rng(n)
        c, o, buf = filled(sm, rng, shape, 12, 20)
        attend(c, o, buf, dtabs, tabs, shape, rng, 2, 1, [n - 1], None, n)
        attend(c, o, buf, dtabs, tabs, shape, rng, 2, 1, [n - 1], None, 513)


@pytest.mark.parametrize("bits,dim,group,ctx", [(4, 64, 1, 1025), (8, 64, 4, 1300), (4, 128, 1, 2048), (8, 128, 3, 1537), (4, 256, 2, 1100),
                                                (8, 256, 1, 1281), (4, 64, 6, 1100), (8, 128, 16, 1030), (4, 64, 1, 2049), (4, 128, 2, 2300)])
def test_longer_contexts(sm, dtabs, tabs, bits, dim, group, ctx):
    """five chunks and more: in one block's waves, and split and joined"""
    shape = (2, 1, dim, ctx, bits)
    rng = np.random.default_rng(ctx)
    c, o, buf = filled_by_columns(sm, rng, shape)
    attend(c, o, buf, dtabs, tabs, shape, rng, group, 1, [ctx - 1, 900], None, ctx)


def test_long_context(sm, dtabs, tabs):
    """more chunks than the join's block has threads: 70,000 positions, the other stream's row near its start"""
    shape = (2, 1, 64, 70000, 4)
    rng = np.random.default_rng(70)
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    k, v = (rows_of(rng, (2, 500, 1, 64), 12, 20) for _ in range(2))
    o.write(k, v, [0, 0])
    for name in ("k", "v", "kl", "vl"):                  # the same 500 rows over and over
        a = getattr(o, name)
        for p in range(500, 70000, 500):
            a[:, :, p:p + 500] = a[:, :, :500]
    buf = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda")
    dk, dv = dev(np.tile(k, (1, 140, 1, 1))), dev(np.tile(v, (1, 140, 1, 1)))
    ds = dev(np.zeros(2, np.int32))
    c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), 70000, ds.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    attend(c, o, buf, dtabs, tabs, shape, rng, 1, 1, [69999, 3], None, 70000)


@pytest.mark.parametrize("bits,dim,group,rows", [(4, 64, 1, 5), (8, 64, 2, 3), (4, 128, 4, 7), (8, 96, 3, 33), (4, 64, 1, 100),
                                                 (4, 256, 1, 20), (8, 128, 1, 40)])
def test_many_rows(sm, dtabs, tabs, bits, dim, group, rows):
    """rows at consecutive positions, each seeing the ones before it; uneven counts, rows that are not there"""
    shape = (4, 2, dim, 330, bits)
    rng = np.random.default_rng(rows)
    c, o, buf = filled(sm, rng, shape, 12, 20)
    attend(c, o, buf, dtabs, tabs, shape, rng, group, rows, [330 - rows, 0, 250, -2], [rows, rows // 2, 0, 4], 330)
    attend(c, o, buf, dtabs, tabs, shape, rng, group, rows, [400, 200, 250, -200], None, 260)


@pytest.mark.parametrize("bits,dim,group,rows,ctx", [(4, 64, 2, 17, 700), (8, 128, 1, 40, 600), (4, 64, 2, 50, 700), (8, 128, 1, 100, 600),
                                                     (4, 256, 3, 40, 300), (8, 64, 1, 113, 1100), (4, 100, 1, 97, 530), (8, 200, 2, 60, 270),
                                                     (4, 40, 5, 21, 1030), (4, 128, 2, 49, 520)])
def test_prompt_rows(sm, dtabs, tabs, bits, dim, group, rows, ctx):
    """several and many row tiles (split over chunks, and swept): prompts of uneven lengths at uneven places, some not there
    at all"""
    shape = (8, 12, dim, ctx, bits)
    rng = np.random.default_rng(rows)
    c, o, buf = filled_by_columns(sm, rng, shape)
    start = [ctx - rows, 0, 250, -2, 5, ctx - 3, ctx + 5, 255]
    attend(c, o, buf, dtabs, tabs, shape, rng, group, rows, start, [min(rows, 19), 2, 0, 4, -1, rows, rows, 1], ctx)


def filled_by_columns(sm, rng, shape):
    """a cache written by one call, the heads of stream s > 0 sharing the values of two (the oracle's digits made once)"""
    streams, heads, dim, ctx, bits = shape
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    some = [orc.Cache(1, 1, dim, ctx, bits) for _ in range(4)]
    rows = [[rows_of(rng, (1, ctx, 1, dim), 12, 20) for _ in range(2)] for _ in some]
    for x, (k, v) in zip(some, rows):
        x.write(k, v, [0])
    k, v = (np.zeros((streams, ctx, heads, dim), np.int64) for _ in range(2))
    for s in range(streams):
        for h in range(heads):
            i = int(rng.integers(0, len(some)))
            k[s, :, h], v[s, :, h] = rows[i][0][0, :, 0], rows[i][1][0, :, 0]
            for name in ("k", "v", "kl", "vl"):
                getattr(o, name)[s, h] = getattr(some[i], name)[0, 0]
    buf, dk, dv, ds = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda"), dev(k), dev(v), dev(np.zeros(streams, np.int32))
    c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), ctx, ds.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    return c, o, buf


def test_sweep_levels_far_apart(sm, dtabs, tabs):
    """test_levels_far_apart's keys, values and queries through the sweep"""
    for shape in ((8, 12, 64, 300, 4), (8, 12, 128, 280, 8)):
        rng = np.random.default_rng(shape[4])
        c, o, buf = filled(sm, rng, (1, 1) + shape[2:], 0, 61)
        one = buf.view(1, -1)
        big, wide = sm.NarrowCache(*shape), orc.Cache(*shape)
        for name in ("k", "v", "kl", "vl"):
            getattr(wide, name)[:] = getattr(o, name)
        for scale in (None, 0, -(64 << 16), 64 << 16, 77777):
            attend(big, wide, one.expand(96, -1).contiguous(), dtabs, tabs, shape, rng, 1, 100, [170] * 8, [2, 0, 1, 0, 0, 0, 3, 0], shape[3],
                   scale, 0, 61)


def test_levels_far_apart(sm, dtabs, tabs):
    """keys, values and queries of any size: scores past every clamp, ties there, weights shifted out by the values' levels;
    scales from 2^-64 to 2^64"""
    for shape in ((1, 2, 64, 530, 4), (1, 1, 128, 300, 8)):
        rng = np.random.default_rng(shape[4])
        c, o, buf = filled(sm, rng, shape, 0, 61)
        for scale in (None, 0, -(64 << 16), 64 << 16, -123456, 77777):
            attend(c, o, buf, dtabs, tabs, shape, rng, 2, 2, [shape[3] - 2], None, shape[3], scale, 0, 61)


def test_empty_cache_and_equal_scores(sm, dtabs, tabs):
    """zeroed memory: every score is 0 and every value 0; zero queries over values give their mean"""
    shape = (1, 1, 64, 400, 4)
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    rng = np.random.default_rng(1)
    buf = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda")
    attend(c, o, buf, dtabs, tabs, shape, rng, 1, 1, [399], None, 400)
    c, o, buf = filled(sm, rng, shape, 14, 18)
    q, out = torch.zeros((1, 1, 1, 64), dtype=torch.int64, device="cuda"), torch.zeros((1, 1, 1, 64), dtype=torch.int64, device="cuda")
    n = c.work_bytes(1, 1, 400)
    wk, ds = space(n), dev(np.array([399], np.int32))
    c.attend(dtabs, buf.data_ptr(), q.data_ptr(), 1, 1, 400, ds.data_ptr(), 0, out.data_ptr(), wk.data_ptr(), n, stream=stream())
    want = np.zeros((1, 1, 1, 64), np.int64)
    o.attend(tabs, np.zeros((1, 1, 1, 64), np.int64), [399], None, 400, c.scale, want)
    assert np.array_equal(out.cpu().numpy(), want)


def test_past_four_gigabytes(sm, dtabs, tabs):
    """the last stream's last head of a cache of 10.8 GB, at its context's end"""
    streams, heads, dim, ctx, bits = shape = (40, 8, 256, 65536, 8)
    rng = np.random.default_rng(4)
    c, o = sm.NarrowCache(*shape), orc.Cache(1, 1, dim, 70, bits)
    assert c.bytes > 2 * 2 ** 32
    buf = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda")
    k, v = (rows_of(rng, (1, 70, 1, dim), 12, 20) for _ in range(2))
    o.write(k, v, [0])
    wide = torch.zeros((streams, 70, heads, dim), dtype=torch.int64, device="cuda")
    dk, dv = wide.clone(), wide.clone()
    dk[-1, :, -1], dv[-1, :, -1] = dev(k[0, :, 0]), dev(v[0, :, 0])
    start, count = np.full(streams, ctx - 70, np.int32), np.zeros(streams, np.int32)
    count[-1] = 70
    ds, dc = dev(start), dev(count)
    c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), 70, ds.data_ptr(), dc.data_ptr(), stream=stream())
    k2, v2 = wide.clone(), wide.clone()
    c.read(buf.data_ptr(), k2.data_ptr(), v2.data_ptr(), 70, ds.data_ptr(), dc.data_ptr(), stream=stream())
    wk, wv = np.zeros((1, 70, 1, dim), np.int64), np.zeros((1, 70, 1, dim), np.int64)
    o.read(70, [0], None, wk, wv)
    assert np.array_equal(k2[-1, :, -1].cpu().numpy(), wk[0, :, 0]) and np.array_equal(v2[-1, :, -1].cpu().numpy(), wv[0, :, 0])
    assert int(k2[:-1].abs().sum()) == 0
    # the same 70 rows at the front of the last stream: what a row sees there
    start[-1] = 0
    ds = dev(start)
    c.write(buf.data_ptr(), dk.data_ptr(), dv.data_ptr(), 70, ds.data_ptr(), dc.data_ptr(), stream=stream())
    q = rows_of(rng, (1, 1, 1, dim), 14, 18)
    dq, out = torch.zeros((streams, 1, heads, dim), dtype=torch.int64, device="cuda"), torch.zeros((streams, 1, heads, dim), dtype=torch.int64, device="cuda")
    dq[-1, 0, -1] = dev(q[0, 0, 0])
    start[-1], count[-1] = 69, 1
    ds, dc = dev(start), dev(count)
    n = c.work_bytes(heads, 1, 100)
    wk = space(n)
    c.attend(dtabs, buf.data_ptr(), dq.data_ptr(), heads, 1, 100, ds.data_ptr(), dc.data_ptr(), out.data_ptr(), wk.data_ptr(), n, stream=stream())
    want = np.zeros((1, 1, 1, dim), np.int64)
    o.attend(tabs, q, [69], None, 100, c.scale, want)
    assert np.array_equal(out[-1, 0, -1].cpu().numpy(), want[0, 0, 0])


def test_two_streams_at_once(sm, dtabs, tabs):
    """calls on two streams over one cache and one plate, each with its own workspace and outputs, 20 times over"""
    rng = np.random.default_rng(2)
    shape = (3, 2, 64, 1400, 4)
    c, o, buf = filled_by_columns(sm, rng, shape)
    w, e, b = plate(rng, 512, 700, True)
    p = sm.Plate8(w, e, b)
    X, q = rows_of(rng, (40, 512), 10, 20), rows_of(rng, (3, 2, 4, 64), 12, 18)
    want, att = orc.product(X, w, e, b), np.zeros(q.shape, np.int64)
    o.attend(tabs, q, [1398, 700, 3], None, 1400, c.scale, att)
    x, dq, ds = dev(X), dev(q), dev(np.array([1398, 700, 3], np.int32))
    pn, an = p.work_bytes(40), c.work_bytes(4, 2, 1400)
    torch.cuda.synchronize()
    sides = []
    for _ in range(2):
        st = torch.cuda.Stream()
        sides.append((st, torch.zeros((40, 700), dtype=torch.int64, device="cuda"), torch.zeros(q.shape, dtype=torch.int64, device="cuda"),
                      space(pn), space(an)))
    torch.cuda.synchronize()
    for _ in range(20):
        for st, out, ao, pw, aw in sides:
            p.product(x.data_ptr(), 40, out.data_ptr(), pw.data_ptr(), pn, stream=st.cuda_stream)
            c.attend(dtabs, buf.data_ptr(), dq.data_ptr(), 4, 2, 1400, ds.data_ptr(), 0, ao.data_ptr(), aw.data_ptr(), an, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for _, out, ao, _, _ in sides:
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(ao.cpu().numpy(), att)


def test_graph_of_a_prompt(sm, dtabs, tabs):
    """write and swept attention captured once, replayed on new rows with eager calls and waits between"""
    rng = np.random.default_rng(9)
    shape = (8, 12, 64, 300, 4)
    c, o = sm.NarrowCache(*shape), orc.Cache(*shape)
    buf = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda")
    rows = 100
    k, v, q, out = (torch.zeros((8, rows, 12, 64), dtype=torch.int64, device="cuda") for _ in range(4))
    ds, dc = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    n = c.work_bytes(12, rows, 300)
    wk = space(n)

    def calls():
        c.write(buf.data_ptr(), k.data_ptr(), v.data_ptr(), rows, ds.data_ptr(), dc.data_ptr(), stream=stream())
        c.attend(dtabs, buf.data_ptr(), q.data_ptr(), 12, rows, 300, ds.data_ptr(), dc.data_ptr(), out.data_ptr(), wk.data_ptr(), n, stream=stream())

    calls()                                         # (nothing there: count 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for i in range(3):
        new = [rows_of(rng, (1, rows, 1, 64), 12, 18).repeat(8, 0).repeat(12, 2) for _ in range(3)]
        start, count = np.full(8, 100 * i, np.int32), np.array([3, 0, 1, 0, 0, 2, 0, 0], np.int32) if i else np.full(8, rows, np.int32)
        for t, a in zip((k, v, q), new):
            t.copy_(dev(a))
        ds.copy_(dev(start))
        if i == 0:                                  # fill every stream eagerly, then replay over it with few rows
            dc.copy_(dev(count))
            calls()
            one = orc.Cache(1, 1, 64, 300, 4)
            one.write(new[0][:1, :, :1], new[1][:1, :, :1], [0])
            for name in ("k", "v", "kl", "vl"):
                getattr(o, name)[:, :, :rows] = getattr(one, name)[:, :, :rows]
            count = np.array([0, 2, 0, 0, 1, 0, 0, 0], np.int32)
        dc.copy_(dev(count))
        out.fill_(55)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        o.write(new[0], new[1], start, count)
        want = np.full(tuple(out.shape), 55, np.int64)
        o.attend(tabs, new[2], start, count, 300, c.scale, want)
        assert np.array_equal(out.cpu().numpy(), want), i
        calls()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want), i


def test_other_tables_are_refused(sm, tabs):
    """an arrival that is not base2_convert.py's (its products would not be it)"""
    t = sm.Tables({**tabs, "arrival": tabs["arrival"][:-5]})
    c = sm.NarrowCache(1, 1, 64, 64, 4)
    buf, x = torch.zeros(c.bytes, dtype=torch.uint8, device="cuda"), torch.zeros(64, dtype=torch.int64, device="cuda")
    wk, ds = space(c.work_bytes(1, 1, 64)), dev(np.zeros(1, np.int32))
    with pytest.raises(sm.SmError) as e:
        c.attend(t, buf.data_ptr(), x.data_ptr(), 1, 1, 64, ds.data_ptr(), 0, x.data_ptr(), wk.data_ptr(), wk.numel())
    assert e.value.code == -1


def test_host_memory_is_refused(sm, dtabs):
    c = sm.NarrowCache(1, 1, 64, 64, 4)
    a = np.zeros(c.bytes + 64, np.uint8)
    at = (a.ctypes.data + 15) // 16 * 16
    with pytest.raises(sm.SmError) as e:
        c.write(at, at, at, 1, at)
    assert e.value.code == -1


# ---- together: a step's product, its k and v into the cache, the attention over it, the next product
@pytest.mark.parametrize("graph", [False, True])
def test_a_step(sm, dtabs, tabs, graph):
    """three decode steps of a narrow layer, from a captured graph too (replayed, with the eager steps' own work between)"""
    rng = np.random.default_rng(21)
    streams, heads, dim, ctx, group = 3, 2, 64, 300, 2
    width, kv = heads * group * dim, heads * dim
    shape = (streams, heads, dim, ctx, 4)
    qkv_p, proj_p = plate(rng, width, width + 2 * kv, True), plate(rng, width, width, True)
    pq, pp = sm.Plate8(*qkv_p), sm.Plate8(*proj_p)
    c, o, buf = filled(sm, rng, shape, 12, 18)
    x = torch.zeros((streams, width), dtype=torch.int64, device="cuda")
    start = torch.zeros(streams, dtype=torch.int32, device="cuda")
    qkv = torch.zeros((streams, width + 2 * kv), dtype=torch.int64, device="cuda")
    att, out = torch.zeros((streams, width), dtype=torch.int64, device="cuda"), torch.zeros((streams, width), dtype=torch.int64, device="cuda")
    wn = max(pq.work_bytes(streams), pp.work_bytes(streams))
    an = c.work_bytes(heads * group, 1, ctx)
    ws, aws = space(wn), space(an)

    def step():
        s = stream()
        pq.product(x.data_ptr(), streams, qkv.data_ptr(), ws.data_ptr(), wn, stream=s)
        c.write(buf.data_ptr(), qkv.data_ptr() + 8 * width, qkv.data_ptr() + 8 * (width + kv), 1, start.data_ptr(),
                row_stride=width + 2 * kv, stream_stride=width + 2 * kv, stream=s)
        c.attend(dtabs, buf.data_ptr(), qkv.data_ptr(), heads * group, 1, ctx, start.data_ptr(), 0, att.data_ptr(), aws.data_ptr(), an,
                 q_row=width + 2 * kv, q_stream=width + 2 * kv, out_row=width, out_stream=width, stream=s)
        pp.product(att.data_ptr(), streams, out.data_ptr(), ws.data_ptr(), wn, stream=s)

    run = step
    if graph:
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                step()
        torch.cuda.current_stream().wait_stream(side)
        run = g.replay
    for at in ([10, 255, 298], [256, 11, 299], [12, 100, 0]):
        X = rows_of(rng, (streams, width), 14, 18)
        x.copy_(dev(X))
        start.copy_(dev(np.array(at, np.int32)))
        run()
        want = orc.product(X, *qkv_p)
        row = want.reshape(streams, 1, -1)
        o.write(row[..., width:width + kv].reshape(streams, 1, heads, dim), row[..., width + kv:].reshape(streams, 1, heads, dim), at)
        a = np.zeros((streams, 1, heads * group, dim), np.int64)
        o.attend(tabs, row[..., :width].reshape(a.shape), at, None, ctx, c.scale, a)
        assert np.array_equal(qkv.cpu().numpy(), want)
        assert np.array_equal(att.cpu().numpy(), a.reshape(streams, width))
        assert np.array_equal(out.cpu().numpy(), orc.product(a.reshape(streams, width), *proj_p))
