"""The operators in few bits without a GPU: the oracle's own properties, the 8-bit converter, and every refusal that the
entry points make before a device is asked for anything."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import narrow as orc

DEV = 1 << 20          # an aligned address that no refused call gets to use


@pytest.fixture(scope="module")
def tabs(sm):
    return sm.tables()


@pytest.mark.parametrize("bits", [4, 8])
def test_digits_hold_a_row_to_half_a_step(bits):
    """every digit is in range and off by half a step at most, a step past the top digit (a value that rounds to 2^(b-1))"""
    rng = np.random.default_rng(bits)
    for x in [np.zeros(5, np.int64), np.array([1, -1, 0]), np.array([-(1 << 63), (1 << 63) - 1, 5]), np.array([7, -8, 3]),
              *(np.round(rng.standard_normal(64) * 2.0 ** s).astype(np.int64) for s in (1, 5, 16, 40, 60))]:
        d, sh = orc.digits(x, bits)
        assert d.min() >= -(1 << (bits - 1)) and d.max() < 1 << (bits - 1)
        for a, v in zip(d, x):
            off = abs((int(a) << sh) - int(v))
            assert off <= (1 << sh if a == (1 << (bits - 1)) - 1 else (1 << sh) // 2)


def test_cols8_is_the_narrowest_power(sm):
    rng = np.random.default_rng(3)
    W = rng.standard_normal((40, 7)) * 2.0 ** rng.integers(-9, 3, 7)
    W[:, 2] = 0
    q, e = sm.cols8(W)
    assert q.dtype == np.int8 and np.abs(q.astype(int)).max() <= 127
    assert np.all(np.abs(q * np.exp2(e.astype(float)) - W) <= np.exp2(e.astype(float)) / 2)
    live = np.arange(7) != 2
    assert np.all(np.abs(W).max(0)[live] > 127 * np.exp2(e[live].astype(float) - 1))


def test_one_position_is_its_value(tabs):
    """a row that sees one position gets that position's value back, to the divisor's 2^-16 or so"""
    rng = np.random.default_rng(5)
    k, v = (np.round(rng.standard_normal(64) * 65536).astype(np.int64) for _ in range(2))
    (kd, kl), (vd, vl) = orc.digits(k, 8), orc.digits(v, 8)
    out = orc.attend_row(tabs, k, -3 << 16, kd[None], np.array([kl]), vd[None], np.array([vl]))
    assert np.all(np.abs(out - orc.values(vd, vl)) <= np.abs(orc.values(vd, vl)) * 2.0 ** -14 + 1)


def test_attention_is_near_the_float_one(tabs):
    """8-bit digits of random rows: within the digits' own error of softmax(q k / sqrt(d)) v in float64.  A digit of a row of
    normal values is off by half a step, a step at most 2^-6 of the row's largest value (4 sigma): 2^-5 sigma a step,
    uniform, so 2^-5 / sqrt(12) = 0.009 sigma; v's error averages out to that, q's and k's give a score (a sum of 64 products
    over 8) an error of sqrt(2) 0.009 and a weight that relative one: together under 0.03 sigma for all but far outliers"""
    rng = np.random.default_rng(6)
    n, d = 700, 64
    q, k, v = rng.standard_normal(d), rng.standard_normal((n, d)), rng.standard_normal((n, d))
    s = k @ q / 8
    p = np.exp(s - s.max())
    want = p @ v / p.sum()
    whole = lambda a: np.round(a * 65536).astype(np.int64)           # noqa: E731
    ks, vs = [orc.digits(r, 8) for r in whole(k)], [orc.digits(r, 8) for r in whole(v)]
    got = orc.attend_row(tabs, whole(q), -3 << 16, np.array([a for a, _ in ks]), np.array([b for _, b in ks]),
                         np.array([a for a, _ in vs]), np.array([b for _, b in vs]))
    assert np.abs(got / 65536 - want).max() < 0.03


def test_bytes(sm):
    """64 positions of a head: keys, values and 128 levels; head dimensions go up to 64, 128 or 256 digits"""
    for dim, wide in ((1, 64), (64, 64), (65, 128), (128, 128), (129, 256), (256, 256)):
        for bits in (4, 8):
            assert sm.NarrowCache(3, 5, dim, 65, bits).bytes == 3 * 5 * 2 * (2 * 64 * wide * bits // 8 + 128)


@pytest.mark.parametrize("shape", [(0, 1, 64, 8, 4), (1, 0, 64, 8, 4), (1, 1, 0, 8, 4), (1, 1, 257, 8, 4), (1, 1, 64, 0, 4),
                                   (1, 1, 64, (1 << 24) + 1, 4), (1, 1, 64, 8, 5), (1, 1, 64, 8, 16), (70000, 1, 64, 8, 4)])
def test_shapes_refused(sm, shape):
    with pytest.raises(sm.SmError) as e:
        sm.NarrowCache(*shape)
    assert e.value.code == -1


def refused(sm, call):
    with pytest.raises(sm.SmError) as e:
        call()
    assert e.value.code == -1, str(e.value)


def test_rows_refused(sm):
    c = sm.NarrowCache(2, 3, 64, 100, 4)
    for f in (c.write, c.read):
        refused(sm, lambda: f(DEV, DEV, DEV, -1, DEV))
        refused(sm, lambda: f(DEV, DEV, DEV, 101, DEV))
        refused(sm, lambda: f(0, DEV, DEV, 1, DEV))
        refused(sm, lambda: f(DEV, 0, DEV, 1, DEV))
        refused(sm, lambda: f(DEV, DEV, 0, 1, DEV))
        refused(sm, lambda: f(DEV, DEV, DEV, 1, 0))
        refused(sm, lambda: f(DEV + 8, DEV, DEV, 1, DEV))
        refused(sm, lambda: f(DEV, DEV + 4, DEV, 1, DEV))
        refused(sm, lambda: f(DEV, DEV, DEV, 1, DEV + 2))
        refused(sm, lambda: f(DEV, DEV, DEV, 1, DEV, row_stride=191))
        refused(sm, lambda: f(DEV, DEV, DEV, 1, DEV, stream_stride=-1))
        f(0, 0, 0, 0, 0)                        # no rows: nothing to do


def test_attend_refused(sm):
    c = sm.NarrowCache(2, 3, 64, 100, 4)
    t = type("T", (), {"h": ctypes.c_void_p(DEV)})()
    ok = dict(t=t, cache=DEV, q=DEV, q_heads=6, rows=1, span=100, start=DEV, count=0, out=DEV, work=DEV, work_bytes=1 << 40)
    for bad in (dict(t=type("T", (), {"h": None})()), dict(cache=0), dict(q=0), dict(start=0), dict(out=0), dict(work=0),
                dict(q_heads=4), dict(q_heads=0), dict(rows=-1), dict(rows=101), dict(span=0), dict(span=101),
                dict(scale=(64 << 16) + 1), dict(work_bytes=100), dict(q_row=383), dict(out_row=383), dict(q_stream=-1),
                dict(cache=DEV + 8), dict(work=DEV + 8), dict(q=DEV + 4), dict(out=DEV + 4), dict(start=DEV + 1)):
        refused(sm, lambda: c.attend(**{**ok, **bad}))
    refused(sm, lambda: c.work_bytes(4, 1, 100))
    refused(sm, lambda: c.work_bytes(6, 1, 101))
    assert c.work_bytes(6, 1, 100) > 0
    c.attend(**{**ok, "rows": 0})


def test_plates_refused(sm):
    w, e, b = np.zeros((4, 3), np.int8), np.zeros(3, np.int32), np.zeros(3, np.int64)
    with pytest.raises(ValueError):
        sm.Plate8(w, e[:2], b)
    refused(sm, lambda: sm.Plate8(np.zeros((131072, 1), np.int8), e[:1], b[:1]))
    refused(sm, lambda: sm.Plate8(np.zeros((0, 3), np.int8), e, b))
    refused(sm, lambda: sm.Plate8(w, e + 1025, b))
    L = sm.lib()
    assert L.sm_plate8_product(None, DEV, 4, 1, DEV, 3, DEV, 1 << 20, None) == -1
    assert L.sm_plate8_work(None, 1) == -1
    assert L.sm_plate8_create(None, None, None, 4, 3, None) == -1
    assert L.sm_plate8_destroy(None) == 0 and L.sm_plate8_bytes(None) == 0


def test_sizes_that_no_launch_holds_are_refused(sm):
    for shape in ((65535, 17, 64, 8, 4), (1, 70000, 64, 8, 4)):
        with pytest.raises(sm.SmError) as e:
            sm.NarrowCache(*shape)
        assert e.value.code == -1
    c = sm.NarrowCache(64, 64, 128, 1 << 20, 4)
    assert c.bytes == 64 * 64 * (1 << 14) * (16 * 128 * 4 + 128)
    refused(sm, lambda: c.work_bytes(64, (1 << 16) + 1, 1 << 20))
    refused(sm, lambda: c.work_bytes(64, (1 << 14) + 1, 1 << 20))
    assert 0 < c.work_bytes(64, 1, 1 << 20) < 1 << 40


def test_results_over_one_another_are_refused(sm):
    """outputs whose strides lay streams' rows over one another; streams between the rows of others are fine to ask for"""
    c = sm.NarrowCache(3, 2, 64, 100, 4)
    t = type("T", (), {"h": ctypes.c_void_p(DEV)})()
    L = sm.lib()
    for rows, row, stream in ((1, 128, 127), (2, 128, 128), (2, 128, 255), (4, 300, 128), (2, 383, 128)):
        refused(sm, lambda: c.read(DEV, DEV, DEV, rows, DEV, row_stride=row, stream_stride=stream))
        refused(sm, lambda: c.attend(t, DEV, DEV, 2, rows, 100, DEV, 0, DEV, DEV, 1 << 30, out_row=row, out_stream=stream))
    assert L.sm_narrow_read(c._ref, DEV, DEV, DEV, 128, 0, 1, DEV, None, None) == -1
    # dense, streams apart, and rows of all streams in turn: refused later, since the address is no device's
    for rows, row, stream in ((2, 128, 256), (1, 128, 128), (2, 384, 128)):
        with pytest.raises(sm.SmError) as e:
            c.read(DEV, DEV, DEV, rows, DEV, row_stride=row, stream_stride=stream)
        assert "device's memory" in str(e.value)
