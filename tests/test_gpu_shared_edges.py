"""Attention over shared rows at the edges of what the call accepts: windows that
leave a gap between a group's sequences, soft-caps and queries near the ends of the
floats, empty places beside values that are not finite, bad group starts, pools past
32 bits. Needs a gfx950 device."""
import ctypes as C

import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import bits, f32, ok
from test_gpu_paged import TYPES, U, attention, i32
from test_gpu_shared import Batch, dev, device, own_rows  # noqa: F401

pytestmark = pytest.mark.gpu


def gap(b, window):
    """rows of a group's shared ones that no sequence of it attends: True [groups][shared rows]"""
    out = []
    for g, rows in enumerate(b.shared):
        free = np.ones(rows, bool)
        for n in b.lens[b.start[g]:b.start[g + 1]]:
            free[max(0, n - window):n] = False
        out.append(free)
    return out


GAPS = [
    # one gap, in the first column tile (narrow groups) or in each of several
    (8, 4, 128, 32, 2500, [(60, 2800)], {0: -2670, 7: -2795, 30: -2700}),
    # the short ones at the end: the tile of the others has no gap
    (16, 4, 64, 64, 2500, [(80, 3000)], {77: -2990, 78: -2900, 79: -2680}),
    # three runs of rows with gaps between them, which begin and end within tiles and pages, and a group without one
    (16, 8, 128, 16, 600, [(70, 3100), (30, 480)], {0: -3000, 1: -1717, 2: -1700, 40: -3093, 41: -1690}),
    (8, 4, 256, 16, 1800, [(60, 4000)], {0: -3900, 11: -1990, 12: -2000}),
]


@pytest.fixture(autouse=True)
def no_error():
    yield
    K.hip.krh_clear_error()


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page,window,groups,short", GAPS)
def test_gaps_between_windows(dev, kv_type, nh, nkv, hd, page, window, groups, short, paged):  # noqa: F811
    """rows that no sequence's window reaches may hold anything, and pages of such rows alone need not be in a table"""
    rng = np.random.default_rng(hd + page)
    n = sum(g[0] for g in groups)
    own = [100 + v for v in own_rows(rng, n, 90)]
    for i, v in short.items():
        own[i] = v
    b = Batch(dev, rng, kv_type, nh, nkv, hd, page, groups, own)
    p = b.p
    whole = {name: x.copy() for name, x in p.a.items()}
    free = gap(b, window)
    assert free[0].sum() > 60
    table = p.table.copy()
    for g, rows in enumerate(free):
        a, e = b.start[g], b.start[g + 1]
        for r in np.flatnonzero(rows):
            for name in "kv":
                x = p.a[name + "d"] if kv_type == K.ML_Q8_0 else p.a[name]
                x[p.table[a, r // page], :, r % page] = np.nan if name == "v" or r % 2 else np.inf
        for j in range(len(rows) // page):
            if rows[j * page:(j + 1) * page].all():
                table[a:e, j] = -1
    b.put(window=window)
    assert b.form(window) == 1
    if not paged:
        p.tab = dev.put(table)
    p.a = whole   # (the 64-bit form reads all rows before it leaves out those behind the window)
    b.run(window)
    ok()
    b.check(b.out(), window)


def run(b, scale, cap=0.0, window=0):
    """b's call with a scale of its own"""
    K.hip.krh_paged_attention_shared(b.ob.ptr, b.p.ref, b.p.tab.ptr, b.p.ld, b.lb.ptr, len(b.lens), b.gb.ptr, b.sb.ptr,
                                     len(b.shared), b.max_shared, b.qb.ptr, b.nh, b.max_len, window, scale, cap, b.ws.ptr)
    ok()
    return b.out()


def compare(b, o, scale, score=0.0):
    """against the softmax in 64 bits of scores that no cap changes; `score`: how far a score may be off beside that"""
    for i, n in enumerate(b.lens):
        if n == 0:
            assert (o[i] == 0).all(), i
            continue
        k, v = b.p.rows("k", i, n), b.p.rows("v", i, n)
        for h in range(b.nh):
            g = h * b.nkv // b.nh
            w, _, bound, _ = attention(b.q[i, h].astype(np.float64), k[:, g], v[:, g], scale, 0, 0)
            # a score off by e makes the weights wrong by a factor of e^2e at most
            assert (np.abs(o[i, h] - w) <= bound + 2 * score * np.abs(v[:, g]).max()).all(), (i, h)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("hd,peak,cap", [(64, 0.1, 1e36), (64, 0.01, 1e37), (128, 1.0, 2.0 ** 126), (128, 0.005, 2.0 ** 126),
                                         (48, 0.005, 2.0 ** 126), (256, 0.01, 1e35), (80, 1.0, 2.0 ** 100)])
def test_large_soft_caps(dev, kv_type, hd, peak, cap):  # noqa: F811
    """caps far above the scores leave them, however small the queries are: tanh(x) is x, and what is left is the division's
    rounding, a step of 2^-149 where the quotient is that small, and two roundings of the float"""
    rng = np.random.default_rng(hd)
    b = Batch(dev, rng, kv_type, 4, 2, hd, 16, [(19, 200), (40, 330)], own_rows(rng, 59, 60))
    b.q = f32(b.q * (peak / np.abs(b.q).max()))
    # keys that make the scores differ by a few whatever the queries are
    name = "kd" if kv_type == K.ML_Q8_0 else "k"
    b.p.a[name] = (b.p.a[name] * min(1 / peak, 100)).astype(b.p.a[name].dtype)
    b.put()
    assert b.form() == 1
    o = run(b, hd ** -0.5, cap)
    compare(b, o, hd ** -0.5, 2 * 2.0 ** -149 * cap)


@pytest.mark.parametrize("kv_type", TYPES)
def test_small_soft_caps(dev, kv_type):  # noqa: F811
    """a cap far below the scores gives every row the same weight"""
    rng = np.random.default_rng(5)
    b = Batch(dev, rng, kv_type, 4, 2, 128, 16, [(9, 200), (20, 330)], own_rows(rng, 29, 60)).put()
    assert b.form() == 1
    o = run(b, 128 ** -0.5, 2.0 ** -126)
    b.q = np.zeros_like(b.q)
    compare(b, o, 1.0, 8 * U)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("hd,power,scale", [(128, -140, None), (64, -148, None), (48, -133, None), (64, -10, 2.0 ** -140),
                                            (128, 0, 2.0 ** -149), (256, -100, 1e-20), (64, -126, -2.0 ** -60)])
def test_scores_near_nothing(dev, kv_type, hd, power, scale):  # noqa: F811
    """queries or a scale so small that their product is under the floats: every row has the same weight, and those that
    are cut off none"""
    rng = np.random.default_rng(hd)
    own = own_rows(rng, 40, 60)
    own[2], own[9], own[39] = -190, -5, -330
    b = Batch(dev, rng, kv_type, 4, 2, hd, 16, [(19, 200), (21, 330)], own)
    b.spoil()
    b.q = f32(b.q * 2.0 ** power)
    b.put()
    assert b.form() == 1
    s = hd ** -0.5 if scale is None else scale
    for cap in (0.0, 2.0):
        o = run(b, s, cap)
        assert np.isfinite(o).all()
        compare(b, o, s, 2.0 ** -80)   # no score is larger (2^-100, at most 256 dims, and products below 2^6)


@pytest.mark.parametrize("power,keys", [(0, 95), (-100, 100), (-132, 119), (-140, 124), (124, -119), (110, -112)])
@pytest.mark.parametrize("hd", [64, 128])
def test_8_bit_scales_against_the_queries(dev, hd, power, keys):  # noqa: F811
    """queries and keys' scales at opposite ends of the floats, whose scores are ordinary numbers (or, in the first case,
    large ones: the largest has all the weight)"""
    rng = np.random.default_rng(hd + abs(keys))
    b = Batch(dev, rng, K.ML_Q8_0, 4, 2, hd, 16, [(19, 200), (21, 330)], own_rows(rng, 40, 60))
    b.q = f32(b.q * 2.0 ** power)
    b.p.a["kd"] = f32(b.p.a["kd"] * 2.0 ** keys)
    b.put()
    assert b.form() == 1 and np.abs(b.q).max() > 0
    scale = 2.0 ** -(power + keys) * hd ** -0.5 if power else hd ** -0.5
    o = run(b, scale)
    assert np.isfinite(o).all()
    if power:
        compare(b, o, scale)
        # each sequence reading its own rows as well
        ws = dev.zeros(K.hip.krh_paged_attention_ws(b.p.ref, len(b.lens), 4, b.max_len, 0))
        K.hip.krh_paged_attention(b.ob.ptr, b.p.ref, b.p.tab.ptr, b.p.ld, b.lb.ptr, len(b.lens), b.qb.ptr, 4, b.max_len, 0, scale,
                                  0.0, None, 0, ws.ptr)
        ok()
        compare(b, b.out(), scale)
        return
    for i, n in enumerate(b.lens):
        k, v = b.p.rows("k", i, n), b.p.rows("v", i, n)
        for h in range(4):
            z = k[:, h // 2] @ b.q[i, h].astype(np.float64)
            if np.diff(np.sort(z)[-2:])[0] > 2.0 ** -18 * (np.abs(k[:, h // 2]) @ np.abs(b.q[i, h])).max():
                assert (np.abs(o[i, h] - v[z.argmax(), h // 2]) <= 8 * U * np.abs(v[:, h // 2]).max()).all(), (i, h)


@pytest.mark.parametrize("kv_type", TYPES)
def test_empty_places_beside_values_not_finite(dev, kv_type):  # noqa: F811
    """a place without a sequence gets zeros, whatever the rows hold that its group shares"""
    rng = np.random.default_rng(3)
    own = own_rows(rng, 30, 60)
    own[0], own[7], own[29] = -320, -320, -320
    b = Batch(dev, rng, kv_type, 8, 2, 64, 16, [(30, 320)], own)
    name = "vd" if kv_type == K.ML_Q8_0 else "v"
    b.p.a[name][b.p.table[0, 3], :, 5] = np.nan
    b.p.a[name][b.p.table[0, 4], 0, 6] = np.inf
    b.put()
    assert b.form() == 1
    b.run()
    ok()
    o = b.out()
    for i, n in enumerate(b.lens):
        assert (o[i] == 0).all() if n == 0 else np.isnan(o[i]).all(), i


@pytest.mark.parametrize("what,at,value", [("start", 0, -5), ("end", 2, 61), ("order", 1, 2 ** 30), ("order", 0, 31)])
def test_bad_group_starts(dev, what, at, value):  # noqa: F811
    """are reported, and leave no group: each sequence reads all of its own rows"""
    rng = np.random.default_rng(9)
    b = Batch(dev, rng, K.ML_F16, 8, 2, 64, 16, [(30, 320), (30, 160)], own_rows(rng, 60, 40)).put()
    assert b.form() == 1
    start = i32(b.start)
    start[at] = value
    b.gb = dev.put(start)
    b.run()
    assert K.hip.krh_sync() == K.ML_E_SHAPE
    K.hip.krh_clear_error()
    b.check(b.out())


@pytest.mark.parametrize("kv_type,n", [(K.ML_F16, 270000), (K.ML_Q8_0, 530000)])
def test_offsets_past_32_bits(dev, kv_type, n):  # noqa: F811
    """shared and own rows of halves and 8 bits in pages beyond 2^32 bytes"""
    nkv, hd, page, S, shared = 2, 256, 16, 40, 96
    size = 2 if kv_type == K.ML_F16 else 1
    assert n * nkv * hd * page * size > 2 ** 32
    pool = [K.DevBuf(size * n * nkv * hd * page) for _ in range(2)]
    scales = [K.DevBuf(4 * n * nkv * page) for _ in range(2)] if size == 1 else []
    dev.bufs += pool + scales
    kv = K.KrhPages(*[x.ptr for x in pool], *([x.ptr for x in scales] or [None, None]), kv_type, n, page, nkv, hd)
    ref, rng = C.byref(kv), np.random.default_rng(12)
    table = np.full((S, 7), -1, np.int32)
    table[:, :6] = [n - 1, 7, n - 2, n // 2 + 1, n - 70, 3]
    table[:, 6] = n - 10 - np.arange(S)
    lens = i32(shared + rng.integers(0, 16, S))
    seq = i32([0] * shared + [i for i in range(S) for _ in range(lens[i] - shared)])
    row = i32(list(range(shared)) + [r for i in range(S) for r in range(shared, lens[i])])
    T, nh = len(seq), 4
    q = f32(rng.standard_normal((S, nh, hd)))
    kr, vr = (dev.put(f32(rng.standard_normal((T, nkv * hd)))) for _ in range(2))
    tb, ob, sb, rb = dev.put(table), dev.zeros(q.nbytes), dev.put(seq), dev.put(row)
    K.hip.krh_paged_qkv(None, 0, ref, tb.ptr, 7, S, None, 0, kr.ptr, nkv * hd, vr.ptr, nkv * hd, T, 0, sb.ptr, rb.ptr, None, None,
                        None, 0.0, None, None, 0)
    K.hip.krh_paged_load(kr.ptr, nkv * hd, vr.ptr, nkv * hd, ref, tb.ptr, 7, S, T, sb.ptr, rb.ptr)   # what the pages hold
    most = 128
    while K.hip.krh_paged_attention_shared_form(ref, S, nh, most, 1, most - 1, 0) != 1:
        most *= 2
    ws = dev.zeros(K.hip.krh_paged_attention_shared_ws(ref, S, nh, most, 1, most - 1))
    K.hip.krh_paged_attention_shared(ob.ptr, ref, tb.ptr, 7, dev.put(lens).ptr, S, dev.put(i32([0, S])).ptr,
                                     dev.put(i32([shared])).ptr, 1, most - 1, dev.put(q).ptr, nh, most, 0, 0.0625, 0.0, ws.ptr)
    ok()
    o = ob.get(np.float32, q.size).reshape(q.shape)
    k64, v64 = (x.get(np.float32, T * nkv * hd).reshape(T, nkv, hd).astype(np.float64) for x in (kr, vr))
    assert np.abs(k64).max() > 2
    for i in range(S):
        at = np.concatenate([np.arange(shared), np.flatnonzero((seq == i) & (row >= shared))])
        for h in range(nh):
            w, _, bound, _ = attention(q[i, h].astype(np.float64), k64[at, h // 2], v64[at, h // 2], 0.0625, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all(), (i, h)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,window", [(14, 2, 64, 0), (8, 8, 128, 0), (8, 4, 256, 0), (8, 8, 128, 2500)])
def test_own_rows_as_their_part_is(dev, kv_type, nh, nkv, hd, window):  # noqa: F811
    """lengths from nothing to far more own rows than shared ones, under bounds that allow own rows to be most of the work"""
    rng = np.random.default_rng(hd + window)
    for n, shared, own in ((70, 2000, own_rows(rng, 70, 40)), (70, 320, own_rows(rng, 70, 3000)), (70, 96, [2500] * 3 + [0] * 67)):
        own[4], own[69] = -shared, -shared // 2
        b = Batch(dev, rng, kv_type, nh, nkv, hd, 32, [(n - 20, shared), (20, shared // 2)], own).spoil()
        b.put(max_len=50000, max_shared=4000)
        assert b.form(window) == 1
        b.run(window)
        ok()
        o = b.out()
        b.check(o, window)
        b.run(window)
        ok()
        assert np.array_equal(bits(b.out()), bits(o))
        # no groups at all: every row is a sequence's own
        b.gb = dev.put(i32([n, n, n]))
        b.run(window)
        ok()
        b.check(b.out(), window)
