"""Several sequences over a paged cache on the device: rows into pages, the
attention of one token of each, eviction by weight and the rules on logit rows,
against plain implementations in 64 bits (and, where an operator of one
sequence gives the same bits, against that operator). Needs a gfx950 device."""
import ctypes as C

import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import Dev, bits, f32, ok

pytestmark = pytest.mark.gpu
U = 2.0 ** -24   # half a step of a float, relative
NP = {K.ML_F32: np.float32, K.ML_F16: np.float16, K.ML_Q8_0: np.int8}
TYPES = [K.ML_F32, K.ML_F16, K.ML_Q8_0]


@pytest.fixture(scope="module", autouse=True)
def device():
    K.init_device()
    yield
    K.hip.krh_sync()


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.free()


def i32(a):
    return np.ascontiguousarray(a, np.int32)


class Pool:
    """pages of one layer on the host and the device, and their sequences"""

    def __init__(self, dev, rng, kv_type, lens, page, nkv, hd, spare=2, fill=True):
        used = [-(-n // page) for n in lens]
        n = sum(used) + spare
        self.page, self.nkv, self.hd, self.kv_type, self.n = page, nkv, hd, kv_type, n
        shape = (n, nkv, page, hd)
        self.a, self.b, self.dev = {}, {}, dev
        for name in "kv":
            x = rng.standard_normal(shape) if fill else np.zeros(shape)
            if kv_type == K.ML_Q8_0:
                self.a[name] = np.clip(np.rint(x * 40), -127, 127).astype(np.int8)
                self.a[name + "d"] = f32((0.02 + 0.01 * rng.random(shape[:3])) * (1 if fill else 0))
            else:
                self.a[name] = x.astype(NP[kv_type])
        self.ld = max(used + [1]) + 1
        self.table = np.full((len(lens), self.ld), -1, np.int32)
        ids = rng.permutation(n)
        for i, u in enumerate(used):
            self.table[i, :u] = ids[:u]
            ids = ids[u:]
        self.free = ids

    def put(self):
        for name, x in self.a.items():
            self.b[name] = self.dev.put(x)
        self.d = K.KrhPages(self.b["k"].ptr, self.b["v"].ptr, self.b["kd"].ptr if "kd" in self.b else None,
                            self.b["vd"].ptr if "vd" in self.b else None, self.kv_type, self.n, self.page, self.nkv,
                            self.hd)
        self.ref = C.byref(self.d)
        self.tab = self.dev.put(self.table)
        return self

    def get(self, name):
        x = self.a[name]
        return self.b[name].get(x.dtype, x.size).reshape(x.shape)

    def rows(self, name, seq, n, a=None, table=None):
        """[row][kv head][dim] of a sequence's first n rows in 64 bits"""
        a = a or self.a
        r = np.arange(n)
        t = (self.table if table is None else table)[seq, r // self.page]
        x = a[name][t, :, r % self.page].astype(np.float64)
        return x * a[name + "d"][t, :, r % self.page].astype(np.float64)[..., None] if name + "d" in a else x


def attention(q, k, v, scale, cap, window):
    """one head: q [hd], k, v [n][hd]; the output, the weights and a bound on its error in 32 bits.

    A score's products and sum err by (hd + 8) U of the sum of their magnitudes (its scaling, cap and exponent's
    rounding among the 8); a weight by twice that, relative; the sums over n rows by n U of theirs."""
    n = len(k)
    z = (k @ q) * scale
    dz = (len(q) + 8) * U * (np.abs(k) @ np.abs(q)) * scale
    if cap > 0:
        z, dz = cap * np.tanh(z / cap), dz + 8 * U * cap
    first = max(0, n - window) if window else 0
    z, dz, v = z[first:], dz[first:], v[first:]
    a = np.exp(z - z.max())
    a /= a.sum()
    rel = 2 * (dz.max() + 8 * U * (1 + np.abs(z - z.max()).max())) + 2 * (n + 64) * U
    return a @ v, np.concatenate([np.zeros(first), a]), rel * (a @ np.abs(v)), rel


def check_attention(dev, kv_type, nh, nkv, hd, page, lens, window=0, cap=0.0, mass=False, max_len=None, seed=0, spoil=True,
                    peak=1.5, kscale=1.0, vscale=1.0):
    rng = np.random.default_rng(seed + hd + 7 * nh)
    p = Pool(dev, rng, kv_type, lens, page, nkv, hd)
    for n, f in (("k", kscale), ("v", vscale)):
        n += "d" if kv_type == K.ML_Q8_0 else ""
        p.a[n] = (p.a[n] * f).astype(p.a[n].dtype)
    if spoil:   # what lies behind the rows is never attended, whatever it is
        for name in "kv":
            for i, n in enumerate(lens):
                if n % page:
                    x = p.a[name + "d"] if kv_type == K.ML_Q8_0 else p.a[name]
                    x[p.table[i, n // page], :, n % page:] = np.nan if name == "v" else np.inf
    p.put()
    S, ml = len(lens), max_len or max(max(lens), 1)
    q = f32(rng.standard_normal((S, nh, hd)) * peak)
    m0 = f32(rng.random((S, nkv, ml + 3)))
    # an aligned buffer with room around the outputs, to see that nothing else is written
    ob = dev.put(np.full(S * nh * hd + 64, 777.0, np.float32))
    mb = dev.put(m0)
    nb = K.hip.krh_paged_attention_ws(p.ref, S, nh, ml, int(mass))
    ws = dev.put(np.full(nb + 256, 0xEE, np.uint8))
    qb, lb = dev.put(q), dev.put(i32(lens))
    outs = []
    for _ in range(2):
        K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, lb.ptr, S, qb.ptr, nh, ml, window, hd ** -0.5, cap,
                                  mb.ptr if mass else None, ml + 3, ws.ptr)
        ok()
        outs.append(ob.get(np.float32, S * nh * hd + 64))
    assert np.array_equal(bits(outs[0]), bits(outs[1]))     # the same from call to call
    assert (outs[0][S * nh * hd:] == 777.0).all()
    assert (ws.get(np.uint8, nb + 256)[nb:] == 0xEE).all()
    o = outs[0][:S * nh * hd].reshape(S, nh, hd)
    m = mb.get(np.float32, m0.size).reshape(m0.shape).astype(np.float64)
    sq = su = 0.0
    for i, n in enumerate(lens):
        if n == 0:
            assert (o[i] == 0).all() and np.array_equal(m[i], m0[i])
            continue
        k, v = p.rows("k", i, n), p.rows("v", i, n)
        want, tol = m0[i].astype(np.float64).copy(), np.zeros(m0[i].shape)
        for h in range(nh):
            g = h * nkv // nh
            w, a, bound, rel = attention(q[i, h].astype(np.float64), k[:, g], v[:, g], hd ** -0.5, cap, window)
            err = np.abs(o[i, h] - w)
            assert (err <= bound + 1e-30).all(), (i, h, (err / bound).max())
            sq, su = sq + (err ** 2).sum(), su + (w ** 2).sum()
            want[g, :n] += 2 * a if mass else 0            # two calls
            tol[g, :n] += 2 * rel * a
        assert (np.abs(m[i] - want) <= tol + 8 * nh * U * want).all()
    # over all outputs the roundings are as good as independent
    assert su == 0 or np.sqrt(sq / su) <= 4 * U * np.sqrt(hd + max(lens))
    return o


HEADS = [(6, 6, 48), (14, 2, 64), (8, 2, 128), (3, 1, 80), (4, 1, 96), (8, 4, 256), (16, 1, 64), (9, 1, 128), (5, 5, 8),
         (10, 1, 200), (32, 2, 256)]


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_heads(dev, kv_type, nh, nkv, hd):
    check_attention(dev, kv_type, nh, nkv, hd, 16, [1, 37, 0, 16, 130])


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024])
def test_attention_lengths(dev, kv_type, page):
    check_attention(dev, kv_type, 8, 2, 64, page, [2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 700])


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("window,cap,mass", [(1, 0, False), (16, 0, True), (33, 50.0, False), (1000, 0, True),
                                             (0, 30.0, True), (0, 2.0, False), (5000, 0, False)])
def test_attention_window_cap_mass(dev, kv_type, window, cap, mass):
    check_attention(dev, kv_type, 8, 4, 128, 16, [1, 40, 0, 333, 1025, 1500], window=window, cap=cap, mass=mass)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_long(dev, kv_type):
    """a long axis, split over the chip and joined; and a batch whose longest is far under max_len"""
    check_attention(dev, kv_type, 8, 2, 64, 64, [9001], mass=True)
    check_attention(dev, kv_type, 7, 1, 128, 32, [2500, 3], mass=True, max_len=20000)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_peaked(dev, kv_type):
    """one weight near 1 with many rows far below it, and all weights alike"""
    check_attention(dev, kv_type, 4, 2, 64, 16, [700, 31], mass=True, peak=12.0)
    check_attention(dev, kv_type, 4, 2, 64, 16, [700, 31], mass=True, peak=0.0)
    check_attention(dev, kv_type, 4, 2, 64, 16, [700, 31], mass=True, peak=1e-20)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("kscale,vscale,peak", [(2.0 ** -17, 1.0, 1e5), (1.0, 2.0 ** -18, 1.0), (2.0 ** 12, 2.0 ** 12, 2e-4),
                                                (1.0, 2.0 ** 13, 1e-30), (2.0 ** -15, 2.0 ** -20, 1e30)])
def test_attention_scales(dev, kv_type, kscale, vscale, peak):
    """small and large values, subnormal halves among them"""
    if peak == 1e30:
        kscale, peak = 2.0 ** -15, 3e4
    check_attention(dev, kv_type, 12, 2, 128, 16, [300, 20], mass=True, kscale=kscale, vscale=vscale, peak=peak)
    check_attention(dev, kv_type, 10, 1, 64, 16, [300, 20], kscale=kscale, vscale=vscale, peak=peak)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("ml", [100, 3000])
def test_attention_rows_of_zeros(dev, kv_type, ml):
    """values of zeros, whose 8-bit scale is 0, in all rows of a sequence, in its first ones or in some; and scales far
    apart"""
    rng = np.random.default_rng(31)
    lens = [100, 90, 64, 77, 3000 if ml == 3000 else 50]
    p = Pool(dev, rng, kv_type, lens, 16, 2, 64)
    for i, rows in enumerate([range(100), range(40), range(0, 64, 3), [], []]):
        for r in rows:
            at = (p.table[i, r // 16], slice(None), r % 16)
            p.a["v"][at] = 0
            if kv_type == K.ML_Q8_0:
                p.a["vd"][at] = 0
    if kv_type == K.ML_Q8_0:
        p.a["vd"][p.table[3, :3]] *= np.float32(2.0 ** -60)
        p.a["vd"][p.table[4, :2]] *= np.float32(2.0 ** 40)
    p.put()
    S, nh = len(lens), 6
    q = f32(rng.standard_normal((S, nh, 64)))
    ob, ws = dev.zeros(q.nbytes), dev.zeros(K.hip.krh_paged_attention_ws(p.ref, S, nh, ml, 0))
    K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, dev.put(i32(lens)).ptr, S, dev.put(q).ptr, nh, ml, 0, 0.125,
                              0.0, None, 0, ws.ptr)
    ok()
    o = ob.get(np.float32, q.size).reshape(q.shape)
    assert (o[0] == 0).all()
    for i, n in enumerate(lens):
        k, v = p.rows("k", i, n), p.rows("v", i, n)
        for h in range(nh):
            w, _, bound, _ = attention(q[i, h].astype(np.float64), k[:, h // 3], v[:, h // 3], 0.125, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all(), (i, h)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_many_sequences(dev, kv_type):
    rng = np.random.default_rng(5)
    check_attention(dev, kv_type, 4, 2, 64, 16, list(rng.integers(0, 400, 70)), mass=True)


@pytest.mark.parametrize("n,most", [(65, 40), (128, 90), (333, 60), (1000, 33)])
def test_attention_more_sequences_than_lanes(dev, n, most):
    """past 64 sequences the shares are found over several rounds; runs of empty ones among them"""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, most, n)
    lens[40:n // 2] = 0
    lens[[0, -1]] = 0, most
    check_attention(dev, K.ML_F16, 2, 1, 64, 16, [int(v) for v in lens], mass=True)
    check_attention(dev, K.ML_Q8_0, 2, 1, 64, 16, [int(v) for v in lens])


@pytest.mark.parametrize("kv_type,hd,most", [(K.ML_F16, 128, 256), (K.ML_Q8_0, 64, 256), (K.ML_F16, 256, 128), (K.ML_F32, 64, 128),
                                             (K.ML_F32, 128, 64), (K.ML_F32, 256, 32)])
@pytest.mark.parametrize("many", [False, True])
def test_attention_whole_sequences(dev, kv_type, hd, most, many):
    """each side of the length up to which a sequence is one wave's, for few sequences and for many"""
    rng = np.random.default_rng(hd)
    n, top = (70, 2 * most) if many else (3, most)
    lens = [int(v) for v in rng.integers(0, top, n)]
    lens[1] = 0
    for extra in (0, 1):
        lens[0] = top + extra
        check_attention(dev, kv_type, 4, 2, hd, 16, lens)
        check_attention(dev, kv_type, 4, 2, hd, 16, lens, mass=True)
    check_attention(dev, kv_type, 4, 2, hd, 16, [300, 7, 0, 900], window=most - 31)


def test_attention_many_kv_heads(dev):
    """more KV heads than waves are wanted: a share holds every sequence"""
    check_attention(dev, K.ML_F16, 2100, 2100, 8, 16, [40, 3, 0, 70], mass=True)


@pytest.mark.parametrize("kv_type,hd", [(K.ML_F32, 256), (K.ML_F16, 256), (K.ML_Q8_0, 256), (K.ML_F32, 208), (K.ML_F16, 136),
                                        (K.ML_Q8_0, 144)])
def test_attention_wide_heads(dev, kv_type, hd):
    """heads past 128 dims: tiles of 16 rows"""
    check_attention(dev, kv_type, 8, 2, hd, 16, [1, 15, 16, 17, 33, 700, 0, 48], mass=True)
    check_attention(dev, kv_type, 8, 2, hd, 32, [300, 45], window=37, cap=20.0)


def test_offsets_past_32_bits(dev):
    """pages beyond 2^31 values: rows into them, back, and attended"""
    n, nkv, hd, page = 270000, 2, 256, 16
    k, v = (K.DevBuf(4 * n * nkv * hd * page) for _ in range(2))
    dev.bufs += [k, v]
    kv = K.KrhPages(k.ptr, v.ptr, None, None, K.ML_F32, n, page, nkv, hd)
    rng = np.random.default_rng(9)
    T = 40
    table = i32([[n - 1, 7, n - 2]])
    kr, vr, q = f32(rng.standard_normal((T, nkv * hd))), f32(rng.standard_normal((T, nkv * hd))), f32(
        rng.standard_normal((1, 4, hd)))
    tb, sb, rb = dev.put(table), dev.zeros(4 * T), dev.put(np.arange(T, dtype=np.int32))
    kb, vb, ob = dev.put(kr), dev.put(vr), dev.zeros(q.nbytes)
    ref = C.byref(kv)
    K.hip.krh_paged_qkv(None, 0, ref, tb.ptr, 3, 1, None, 0, kb.ptr, nkv * hd, vb.ptr, nkv * hd, T, 0, sb.ptr, rb.ptr, None,
                        None, None, 0.0, None, None, 0)
    lk, lv = dev.zeros(kr.nbytes), dev.zeros(vr.nbytes)
    K.hip.krh_paged_load(lk.ptr, nkv * hd, lv.ptr, nkv * hd, ref, tb.ptr, 3, 1, T, sb.ptr, rb.ptr)
    ws = dev.zeros(K.hip.krh_paged_attention_ws(ref, 1, 4, T, 0))
    K.hip.krh_paged_attention(ob.ptr, ref, tb.ptr, 3, dev.put(i32([T])).ptr, 1, dev.put(q).ptr, 4, T, 0, 0.0625, 0.0, None, 0,
                              ws.ptr)
    ok()
    assert np.array_equal(lk.get(np.float32, kr.size), kr.reshape(-1)) and np.array_equal(lv.get(np.float32, vr.size), vr.reshape(-1))
    o = ob.get(np.float32, q.size).reshape(4, hd)
    k64, v64 = (x.reshape(T, nkv, hd).astype(np.float64) for x in (kr, vr))
    for h in range(4):
        w, _, bound, _ = attention(q[0, h].astype(np.float64), k64[:, h // 2], v64[:, h // 2], 0.0625, 0, 0)
        assert (np.abs(o[h] - w) <= bound).all()


def test_attention_shared_pages(dev):
    """two sequences over one prompt's pages, their weights apart"""
    rng = np.random.default_rng(3)
    p = Pool(dev, rng, K.ML_F16, [48, 50], 16, 2, 64)
    p.table[1, :3] = p.table[0, :3]
    p.put()
    q = f32(rng.standard_normal((2, 4, 64)))
    ob, mb = dev.zeros(q.nbytes), dev.zeros(2 * 2 * 50 * 4)
    ws = dev.zeros(K.hip.krh_paged_attention_ws(p.ref, 2, 4, 50, 1))
    K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, dev.put(i32([48, 50])).ptr, 2, dev.put(q).ptr, 4, 50, 0, 0.125,
                              0.0, mb.ptr, 50, ws.ptr)
    ok()
    o, m = ob.get(np.float32, q.size).reshape(q.shape), mb.get(np.float32, 200).reshape(2, 2, 50)
    for i, n in enumerate((48, 50)):
        k, v = p.rows("k", i, n), p.rows("v", i, n)
        for h in range(4):
            w, a, bound, _ = attention(q[i, h].astype(np.float64), k[:, h // 2], v[:, h // 2], 0.125, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all()
    assert (m[0, :, 48:] == 0).all() and np.allclose(m.sum(2), 2, rtol=1e-5)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_not_finite(dev, kv_type):
    """a NaN among the rows of one KV head reaches that head's outputs alone; rows outside the window reach none"""
    rng = np.random.default_rng(8)
    p = Pool(dev, rng, kv_type, [100, 90], 16, 2, 64)
    x = p.a["kd"] if kv_type == K.ML_Q8_0 else p.a["k"]
    x[p.table[0, 3], 1, 5] = np.nan          # row 53
    x[p.table[0, 0], 0, 2] = np.nan          # row 2: outside the window
    y = p.a["vd"] if kv_type == K.ML_Q8_0 else p.a["v"]
    y[p.table[0, 1], 0, 9] = np.inf          # row 25: outside
    p.put()
    q = f32(rng.standard_normal((2, 4, 64)))
    ob, ws = dev.zeros(q.nbytes), dev.zeros(K.hip.krh_paged_attention_ws(p.ref, 2, 4, 100, 0))
    K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, dev.put(i32([100, 90])).ptr, 2, dev.put(q).ptr, 4, 100, 60,
                              0.125, 0.0, None, 0, ws.ptr)
    ok()
    o = ob.get(np.float32, q.size).reshape(q.shape)
    assert np.isnan(o[0, 2:]).all() and np.isfinite(o[0, :2]).all() and np.isfinite(o[1]).all()


@pytest.mark.parametrize("bad", ["page", "negative", "length", "short"])
def test_attention_bad_tables(dev, bad):
    """ids and lengths out of range are reported, and nothing else is harmed"""
    rng = np.random.default_rng(4)
    p = Pool(dev, rng, K.ML_F16, [40, 300, 40], 16, 2, 64)
    lens = [40, 300, 40]
    if bad == "page":
        p.table[1, 1] = p.n
    if bad == "negative":
        p.table[1, 0] = -5
    if bad == "length":
        lens[1] = 301
    if bad == "short":   # more rows than the table has pages
        p.ld, p.table = 19, np.ascontiguousarray(p.table[:, :19])
        lens[1] = 19 * 16 + 1
    p.put()
    q = f32(rng.standard_normal((3, 4, 64)))
    ml = 300 if bad != "short" else 19 * 16 + 1
    ob, ws = dev.zeros(q.nbytes), dev.zeros(K.hip.krh_paged_attention_ws(p.ref, 3, 4, ml, 0))
    K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, dev.put(i32(lens)).ptr, 3, dev.put(q).ptr, 4, ml, 0, 0.125, 0.0,
                              None, 0, ws.ptr)
    assert K.hip.krh_sync() == K.ML_E_SHAPE
    assert (b"length" if bad == "length" else b"page") in K.hip.krh_last_error()
    K.hip.krh_clear_error()
    ok()
    o = ob.get(np.float32, q.size).reshape(q.shape)
    for i in (0, 2):
        k, v = p.rows("k", i, 40), p.rows("v", i, 40)
        for h in range(4):
            w, _, bound, _ = attention(q[i, h].astype(np.float64), k[:, h // 2], v[:, h // 2], 0.125, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all()


def tables(rng, n, hd):
    ang = rng.uniform(-3, 3, (n, hd // 2))
    return f32(np.cos(ang)), f32(np.sin(ang))


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,normed", [(6, 6, 48, False), (14, 2, 64, True), (8, 2, 128, True), (3, 1, 80, False),
                                              (4, 4, 256, True), (5, 3, 8, False), (2, 1, 200, True), (0, 2, 96, True)])
def test_qkv(dev, kv_type, nh, nkv, hd, normed):
    """without a norm, the bits of krh_rope and krh_store_kv row by row; with one, the formula's within its roundings.
    Rows at their own positions, strides wider than the rows, and what is not written is left as it was."""
    rng = np.random.default_rng(nh + hd)
    T, page = 9, 16
    p = Pool(dev, rng, kv_type, [20, 5, 40], page, nkv, hd).put()
    seq, row = i32([0, 2, 1, 2, 0, 1, 2, 2, 2]), i32([19, 0, 4, 39, 3, 0, 15, 16, 31])
    pos = i32(rng.integers(0, 50, T))
    cs, sn = tables(rng, 50, hd)
    qd, kd = nh * hd, nkv * hd
    q, k, v = f32(rng.standard_normal((T, qd + 8)) * 3), f32(rng.standard_normal((T, kd + 4))), f32(
        rng.standard_normal((T, kd + 12)))
    v[3] = 0.0
    qw, kw = (f32(1 + 0.1 * rng.standard_normal(hd)) for _ in range(2))
    qb, kb, vb, cb, sb = (dev.put(x) for x in (q, k, v, cs, sn))
    ob = dev.put(np.full((T, qd + 4), 777.0, np.float32))
    wq, wk = (dev.put(qw), dev.put(kw)) if normed else (None, None)
    before = {n: x.copy() for n, x in p.a.items()}
    K.hip.krh_paged_qkv(ob.ptr if nh else None, qd + 4, p.ref, p.tab.ptr, p.ld, 3, qb.ptr if nh else None, qd + 8, kb.ptr,
                        kd + 4, vb.ptr, kd + 12, T, nh, dev.put(seq).ptr, dev.put(row).ptr, dev.put(pos).ptr,
                        wq.ptr if normed and nh else None, wk.ptr if normed else None, 1e-6, cb.ptr, sb.ptr, 50)
    ok()
    got = {n: p.get(n) for n in p.a}
    oq = ob.get(np.float32, T * (qd + 4)).reshape(T, qd + 4)
    assert (oq[:, qd:] == 777.0).all()

    def turned(x, w, t):
        x = x.reshape(-1, hd)
        if w is not None:
            ss = (x.astype(np.float64) ** 2).mean(1, keepdims=True)
            x = x * (1 / np.sqrt(ss + np.float64(np.float32(1e-6)))).astype(np.float32) * w
        a, b, c, s = x[:, 0::2], x[:, 1::2], cs[pos[t]], sn[pos[t]]
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = a * c - b * s, a * s + b * c
        return y.astype(np.float32)

    def same(a, b):
        # the norm's factor, formed in 64 bits on both sides, may round apart at a tie: 2 U of each product
        return np.array_equal(bits(a), bits(b)) if not normed else (np.abs(a - b) <= 8 * U * np.abs(b).max()).all()

    for t in range(T):
        if nh:
            assert same(oq[t, :qd].reshape(nh, hd), turned(q[t, :qd], qw if normed else None, t)), t
        at = (p.table[seq[t], row[t] // page], slice(None), row[t] % page)
        for name, x in (("k", turned(k[t, :kd], kw if normed else None, t)), ("v", v[t, :kd].reshape(nkv, hd))):
            y = got[name][at]
            if kv_type == K.ML_Q8_0:
                m = np.abs(x).max(1, keepdims=True)
                with np.errstate(divide="ignore", invalid="ignore"):
                    n = np.trunc(x * (np.float32(127) * (np.float32(1) / m)) + np.copysign(np.float32(0.5), x))
                n = np.where(m < 1e-30, 0, n)
                assert np.array_equal(bits(got[name + "d"][at]), bits(m[:, 0] / np.float32(127))) or normed
                assert np.array_equal(y, n.astype(np.int8)) if not normed else (np.abs(y - n) <= 1).all()
            elif kv_type == K.ML_F16:
                assert np.array_equal(y, x.astype(np.float16)) if not normed else (
                    np.abs(y.astype(np.float64) - x) <= 2.0 ** -11 * np.abs(x) + 8 * U * np.abs(x).max() + 2.0 ** -25).all()
            else:
                assert same(y, x)
            before[name][at] = y
            if name + "d" in before:
                before[name + "d"][at] = got[name + "d"][at]
    for n, x in before.items():
        assert np.array_equal(x, got[n]), n


@pytest.mark.parametrize("kv_type", [K.ML_F16, K.ML_Q8_0])
def test_qkv_is_store_kv(dev, kv_type):
    """one sequence in order: the pages hold krh_store_kv's rows, and krh_paged_load gives them back"""
    rng = np.random.default_rng(6)
    T, nkv, hd, page = 50, 2, 64, 16
    p = Pool(dev, rng, kv_type, [T], page, nkv, hd, fill=False).put()
    k, v = f32(rng.standard_normal((T, nkv * hd))), f32(rng.standard_normal((T, nkv * hd)))
    kb, vb, seq, row = dev.put(k), dev.put(v), dev.put(np.zeros(T, np.int32)), dev.put(np.arange(T, dtype=np.int32))
    K.hip.krh_paged_qkv(None, 0, p.ref, p.tab.ptr, p.ld, 1, None, 0, kb.ptr, nkv * hd, vb.ptr, nkv * hd, T, 0, seq.ptr, row.ptr,
                        None, None, None, 0.0, None, None, 0)
    w = 2 if kv_type == K.ML_F16 else 1
    ck, cv, ckd, cvd = (dev.zeros(n) for n in (T * nkv * hd * w, T * nkv * hd * w, T * nkv * 4, T * nkv * 4))
    K.hip.krh_store_kv(kv_type, ck.ptr, cv.ptr, ckd.ptr, cvd.ptr, kb.ptr, vb.ptr, nkv, hd, dev.put(i32([0])).ptr, T)
    ok()
    r = np.arange(T)
    for name, c, d in (("k", ck, ckd), ("v", cv, cvd)):
        want = c.get(NP[kv_type], T * nkv * hd).reshape(T, nkv, hd)
        got = p.get(name)[p.table[0, r // page], :, r % page]
        if kv_type == K.ML_F16:
            assert np.array_equal(got, want)
        else:   # the factors may be a step apart: an element next to a border, one in about 2^24 / 127
            off = np.abs(got.astype(int) - want)
            assert off.max() <= 1 and off.sum() <= 2
            assert np.array_equal(bits(p.get(name + "d")[p.table[0, r // page], :, r % page]),
                                  bits(d.get(np.float32, T * nkv)).reshape(T, nkv))
    lk, lv = dev.put(np.full((T, nkv * hd + 4), 777.0, np.float32)), dev.zeros(v.nbytes)
    K.hip.krh_paged_load(lk.ptr, nkv * hd + 4, lv.ptr, nkv * hd, p.ref, p.tab.ptr, p.ld, 1, T, seq.ptr, row.ptr)
    ok()
    got = {n: p.get(n) for n in p.a}
    assert np.array_equal(lv.get(np.float32, v.size).reshape(T, nkv, hd), f32(p.rows("v", 0, T, got)))
    lk = lk.get(np.float32, T * (nkv * hd + 4)).reshape(T, -1)
    assert np.array_equal(lk[:, :-4].reshape(T, nkv, hd), f32(p.rows("k", 0, T, got))) and (lk[:, -4:] == 777.0).all()


@pytest.mark.parametrize("what", ["seq", "row", "negative", "page", "pos"])
def test_qkv_and_load_bad_tokens(dev, what):
    """a token out of range is left out and reported; the others are stored"""
    rng = np.random.default_rng(2)
    p = Pool(dev, rng, K.ML_F32, [20, 20], 16, 1, 64).put()
    seq, row, pos = i32([0, 1, 1]), i32([3, 4, 19]), i32([0, 1, 2])
    if what == "seq":
        seq[1] = 2
    if what == "row":
        row[1] = p.ld * 16
    if what == "negative":
        row[1] = -1
    if what == "page":
        row[1] = 33            # its table entry is -1
    if what == "pos":
        pos[1] = 5
    k = f32(rng.standard_normal((3, 64)))
    kb, cs, sn = dev.put(k), dev.put(np.ones((5, 32), np.float32)), dev.put(np.zeros((5, 32), np.float32))
    sb, rb = dev.put(seq), dev.put(row)
    K.hip.krh_paged_qkv(None, 0, p.ref, p.tab.ptr, p.ld, 2, None, 0, kb.ptr, 64, kb.ptr, 64, 3, 0, sb.ptr, rb.ptr,
                        dev.put(pos).ptr, None, None, 0.0, cs.ptr, sn.ptr, 5)
    assert K.hip.krh_sync() == K.ML_E_SHAPE
    K.hip.krh_clear_error()
    want = {n: x.copy() for n, x in p.a.items()}
    for t in (0, 2):
        for n in "kv":
            want[n][p.table[seq[t], row[t] // 16], 0, row[t] % 16] = k[t]
    for n in "kv":
        got = p.get(n)
        if what == "pos":      # a position out of range turns by row 0
            got[p.table[1, 0], 0, 4] = want[n][p.table[1, 0], 0, 4]
        assert np.array_equal(got, want[n])
    if what != "pos":
        lk = dev.put(np.full((3, 64), 777.0, np.float32))
        K.hip.krh_paged_load(lk.ptr, 64, dev.zeros(768).ptr, 64, p.ref, p.tab.ptr, p.ld, 2, 3, sb.ptr, rb.ptr)
        assert K.hip.krh_sync() == K.ML_E_SHAPE
        K.hip.krh_clear_error()
        lk = lk.get(np.float32, 192).reshape(3, 64)
        assert np.array_equal(lk[[0, 2]], k[[0, 2]]) and (lk[1] == 0).all()


def evicted(w, n, keep, recent):
    """rows kept of n with weights w"""
    if n <= keep:
        return np.arange(n)
    key = np.where(np.isnan(w[:n - recent]), np.inf, w[:n - recent].astype(np.float64))
    key[np.isnan(w[:n - recent])] = np.inf
    order = np.lexsort((np.arange(n - recent), ~np.isnan(w[:n - recent]), -key))   # NaN before +inf
    return np.concatenate([np.sort(order[:keep - recent]), np.arange(n - recent, n)]).astype(int)


def weights(rng, kind, shape):
    if kind == "spread":
        return f32(np.exp(3 * rng.standard_normal(shape)))
    if kind == "ties":
        return f32(rng.integers(0, 4, shape))
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    w = rng.standard_normal(shape)
    w.reshape(-1)[::7] = 0.0
    w.reshape(-1)[3::11] = -0.0
    w.reshape(-1)[5::13] = np.inf
    w.reshape(-1)[6::17] = np.nan
    w.reshape(-1)[4::19] = -np.inf
    w.reshape(-1)[1::23] = 1e-42
    return f32(w)


@pytest.mark.parametrize("kv_type,hd", [(K.ML_F32, 48), (K.ML_F16, 64), (K.ML_Q8_0, 128), (K.ML_Q8_0, 8), (K.ML_F16, 200)])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("keep,recent", [(1, 0), (40, 0), (40, 40), (100, 33), (1100, 100), (5000, 3)])
@pytest.mark.parametrize("inplace", [False, True])
def test_evict(dev, kv_type, hd, kind, keep, recent, inplace):
    rng = np.random.default_rng(keep + hd)
    lens, nkv, page = [1, 40, 0, 41, 2300, 100, 1025], 2, 16
    S, ml = len(lens), 2303
    kept = [min(n, keep) for n in lens]
    p = Pool(dev, rng, kv_type, lens, page, nkv, hd, spare=sum(-(-n // page) for n in kept) + 1)
    out = np.full((S, max(-(-min(keep, ml) // page), 1) + 1), -1, np.int32)
    free = list(p.free)
    for i, n in enumerate(kept):
        for j in range(-(-n // page)):
            out[i, j] = free.pop()
    p.put()
    old = ml + 5
    w = weights(rng, kind, (S, nkv, old))
    wb, lb = dev.put(w), dev.put(i32(lens))
    ld = old if inplace else max(keep, ml) + 2
    ob = wb if inplace and keep <= old else dev.put(np.full((S, nkv, max(ld, keep)), 777.0, np.float32))
    if ob is not wb:
        ld = max(ld, keep)
    nb = lb if inplace else dev.put(np.full(S, -7, np.int32))
    size = K.hip.krh_paged_evict_ws(S, nkv, keep)
    ws = dev.put(np.full(size + 64, 0xEE, np.uint8))
    K.hip.krh_paged_evict(p.ref, p.tab.ptr, p.ld, lb.ptr, wb.ptr, old, S, ml, keep, recent, dev.put(out).ptr, out.shape[1],
                          nb.ptr, ob.ptr, ld, ws.ptr)
    ok()
    assert (ws.get(np.uint8, size + 64)[size:] == 0xEE).all()
    assert nb.get(np.int32, S).tolist() == kept
    om = ob.get(np.float32, S * nkv * ld).reshape(S, nkv, ld)
    got = {n: p.get(n) for n in p.a}
    want = {n: x.copy() for n, x in p.a.items()}
    for i, n in enumerate(lens):
        for g in range(nkv):
            r = evicted(w[i, g], n, keep, recent)
            j = np.arange(len(r))
            assert np.array_equal(bits(om[i, g, :len(r)]), bits(w[i, g, r])), (i, g)
            assert (om[i, g, len(r):max(keep, ml)] == 0).all()
            for name in p.a:
                want[name][out[i, j // page], g, j % page] = p.a[name][p.table[i, r // page], g, r % page]
    for name in p.a:
        assert np.array_equal(got[name].view(np.uint8), want[name].view(np.uint8)), name


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("keep,recent", [(6000, 100), (1, 1), (1, 0), (19999, 5)])
def test_evict_many_rows(dev, kind, keep, recent):
    """more rows of one first digit than a wave holds apart, and fewer"""
    rng = np.random.default_rng(keep)
    lens, nkv, page, hd = [20000, 9001], 2, 64, 8
    kept = [min(n, keep) for n in lens]
    p = Pool(dev, rng, K.ML_F16, lens, page, nkv, hd, spare=sum(-(-n // page) for n in kept))
    out = np.full((2, -(-keep // page)), -1, np.int32)
    free = list(p.free)
    for i, n in enumerate(kept):
        out[i, :-(-n // page)] = [free.pop() for _ in range(-(-n // page))]
    p.put()
    w = weights(rng, kind, (2, nkv, 20000))
    nb, mb = dev.zeros(8), dev.zeros(2 * nkv * keep * 4)
    K.hip.krh_paged_evict(p.ref, p.tab.ptr, p.ld, dev.put(i32(lens)).ptr, dev.put(w).ptr, 20000, 2, 20000, keep, recent,
                          dev.put(out).ptr, out.shape[1], nb.ptr, mb.ptr, keep,
                          dev.zeros(K.hip.krh_paged_evict_ws(2, nkv, keep)).ptr)
    ok()
    assert nb.get(np.int32, 2).tolist() == kept
    om, got = mb.get(np.float32, 2 * nkv * keep).reshape(2, nkv, keep), p.get("k")
    for i, n in enumerate(lens):
        for g in range(nkv):
            r = evicted(w[i, g], n, keep, recent)
            j = np.arange(len(r))
            assert np.array_equal(bits(om[i, g, :len(r)]), bits(w[i, g, r])) and (om[i, g, len(r):] == 0).all()
            assert np.array_equal(got[out[i, j // page], g, j % page], p.a["k"][p.table[i, r // page], g, r % page])


@pytest.mark.parametrize("rows", [65, 256, 257, 4097, 8192, 8193, 28001, 32768, 32769, 40000])
@pytest.mark.parametrize("kind", ["zeros", "negative", "odd", "spread"])
def test_evict_sizes(dev, rows, kind):
    """rows that fill the select's LDS, one more and one less; a few weights among zeros, with as many rows kept as
    are left then; no weight above zero; every row but one"""
    rng = np.random.default_rng(rows)
    nkv, page, hd, recent = 2, 64, 8, rows % 7
    n = rows + recent
    lens = [n, n - 1, n // 3, n // 17 + 2, n]
    for keep in (recent + rows // 2, recent + rows - 1, recent + 1):
        kept = [min(m, keep) for m in lens]
        p = Pool(dev, rng, K.ML_F16, lens, page, nkv, hd, spare=sum(-(-m // page) for m in kept))
        out = np.full((len(lens), -(-keep // page)), -1, np.int32)
        free = list(p.free)
        for i, m in enumerate(kept):
            out[i, :-(-m // page)] = [free.pop() for _ in range(-(-m // page))]
        p.put()
        w = weights(rng, "spread" if kind == "negative" else kind, (len(lens), nkv, n)) if kind != "zeros" else (
            np.where(rng.random((len(lens), nkv, n)) < 0.02, rng.random((len(lens), nkv, n)), 0).astype(np.float32))
        if kind == "negative":
            w = -np.abs(w)
            w[:, :, ::5] = -0.0
        w[4] = 0
        nb, mb = dev.zeros(len(lens) * 4), dev.zeros(len(lens) * nkv * keep * 4)
        K.hip.krh_paged_evict(p.ref, p.tab.ptr, p.ld, dev.put(i32(lens)).ptr, dev.put(w).ptr, n, len(lens), n, keep, recent,
                              dev.put(out).ptr, out.shape[1], nb.ptr, mb.ptr, keep,
                              dev.zeros(K.hip.krh_paged_evict_ws(len(lens), nkv, keep)).ptr)
        ok()
        assert nb.get(np.int32, len(lens)).tolist() == kept
        om, got = mb.get(np.float32, len(lens) * nkv * keep).reshape(len(lens), nkv, keep), p.get("k")
        for i, m in enumerate(lens):
            for g in range(nkv):
                r = evicted(w[i, g], m, keep, recent)
                j = np.arange(len(r))
                assert np.array_equal(bits(om[i, g, :len(r)]), bits(w[i, g, r])), (keep, i, g)
                assert (om[i, g, len(r):] == 0).all()
                assert np.array_equal(got[out[i, j // page], g, j % page], p.a["k"][p.table[i, r // page], g, r % page])


def test_evict_wide_rows(dev):
    """more kept rows than the copy has workgroups for, of the widest rows"""
    rng = np.random.default_rng(5)
    n, keep, page, hd = 18000, 17001, 64, 256
    p = Pool(dev, rng, K.ML_F32, [n], page, 1, hd, spare=-(-keep // page))
    out = np.array([list(p.free)[:-(-keep // page)]], np.int32)
    p.put()
    w = weights(rng, "spread", (1, 1, n))
    nb, mb = dev.zeros(4), dev.zeros(keep * 4)
    K.hip.krh_paged_evict(p.ref, p.tab.ptr, p.ld, dev.put(i32([n])).ptr, dev.put(w).ptr, n, 1, n, keep, 500,
                          dev.put(out).ptr, out.shape[1], nb.ptr, mb.ptr, keep,
                          dev.zeros(K.hip.krh_paged_evict_ws(1, 1, keep)).ptr)
    ok()
    r, j = evicted(w[0, 0], n, keep, 500), np.arange(keep)
    assert nb.get(np.int32, 1).tolist() == [keep]
    assert np.array_equal(bits(mb.get(np.float32, keep)), bits(w[0, 0, r]))
    for name in "kv":
        assert np.array_equal(p.get(name)[out[0, j // page], 0, j % page], p.a[name][p.table[0, r // page], 0, r % page])


def test_evict_bad(dev):
    """a length or a new page out of range is reported; the other sequences are as they should be"""
    rng = np.random.default_rng(1)
    p = Pool(dev, rng, K.ML_F16, [60, 60], 16, 1, 64, spare=6)
    out = np.array([[p.n, -1], [p.free[0], p.free[1]]], np.int32)
    p.put()
    w = weights(rng, "spread", (2, 1, 60))
    nb, mb = dev.zeros(8), dev.zeros(2 * 30 * 4)
    args = lambda lens: (p.ref, p.tab.ptr, p.ld, dev.put(i32(lens)).ptr, dev.put(w).ptr, 60, 2, 60, 30, 5, dev.put(out).ptr, 2,
                         nb.ptr, mb.ptr, 30, dev.zeros(K.hip.krh_paged_evict_ws(2, 1, 30)).ptr)
    for lens, n0 in (([60, 60], 30), ([61, 60], 0), ([-1, 60], 0)):
        K.hip.krh_paged_evict(*args(lens))
        assert K.hip.krh_sync() == K.ML_E_SHAPE
        K.hip.krh_clear_error()
        assert nb.get(np.int32, 2).tolist() == [n0, 30]
        r, j = evicted(w[1, 0], 60, 30, 5), np.arange(30)
        got = p.get("k")
        assert np.array_equal(got[out[1, j // 16], 0, j % 16], p.a["k"][p.table[1, r // 16], 0, r % 16])


def rules(x, n, rep, pre, frq, seen, bias, bits_):
    """one row in 64 bits"""
    x = x.astype(np.float64)
    ids, c = np.unique(np.array([t for t in seen if 0 <= t < n], np.int64), return_counts=True)
    for t, k in zip(ids, c):
        x[t] = (x[t] / rep if x[t] > 0 else x[t] * rep) - frq * k - pre
    for t, b in dict(bias).items():
        if 0 <= t < n:
            x[t] += b
    if bits_ is not None:
        x[~bits_[:n]] = -np.inf
    return x


@pytest.mark.parametrize("n,rows,seen_ld,bias_ld,n_masks", [(1, 1, 1, 1, 1), (31, 2, 5, 3, 1), (33, 1, 0, 0, 0), (4096, 3, 700, 40, 2),
                                                            (4097, 2, 64, 0, 3), (32000, 4, 70, 5, 0), (151936, 5, 9000, 300, 4), (5000, 2, 2049, 1500, 1),
                                                            (50001, 70, 300, 17, 8)])
@pytest.mark.parametrize("inplace", [False, True])
def test_rules(dev, n, rows, seen_ld, bias_ld, n_masks, inplace):
    rng = np.random.default_rng(n + rows)
    ld = n + 3
    x = f32(rng.standard_normal((rows, ld)) * 3)
    x[0, 0] = -np.inf
    x[:, n // 2] = 0.0
    seen = i32(np.minimum(rng.integers(-3, n + 3, (rows, max(seen_ld, 1))), rng.integers(0, n + 3, (rows, max(seen_ld, 1)))))
    b_id = i32(rng.integers(-2, n + 2, (rows, max(bias_ld, 1))))
    bias = f32(rng.standard_normal(b_id.shape) * 5)
    bias[0, 0] = -np.inf
    b_id[:, -1] = b_id[:, 0]
    n_seen, n_bias = i32(rng.integers(0, seen_ld + 1, rows)), i32(rng.integers(0, bias_ld + 1, rows))
    n_seen[-1], n_bias[-1] = seen_ld, bias_ld
    words = (n + 31) // 32
    masks = rng.integers(0, 1 << 32, (max(n_masks, 1), words), dtype=np.uint64).astype(np.uint32)
    masks[0] = 0                                   # a mask that leaves nothing
    rule = (K.LogitRule * rows)()
    par = np.zeros((rows, 3))
    for r in range(rows):
        rule[r] = K.LogitRule(1 + 0.4 * rng.random() if r % 3 else 1.0, rng.random() - 0.3, rng.random() if r % 4 else 0.0,
                              r % (n_masks + 1) - 1)
        par[r] = rule[r].repeat, rule[r].presence, rule[r].frequency
    rb = dev.put(np.frombuffer(bytes(rule), np.uint8))
    xb = dev.put(x)
    ob = xb if inplace else dev.put(np.full((rows, ld + 2), 777.0, np.float32))
    ldo = ld if inplace else ld + 2
    K.hip.krh_logit_rules(ob.ptr, ldo, xb.ptr, ld, n, rows, rb.ptr, dev.put(seen).ptr if seen_ld else None, seen.shape[1],
                          dev.put(n_seen).ptr, dev.put(b_id).ptr if bias_ld else None, dev.put(bias).ptr, b_id.shape[1],
                          dev.put(n_bias).ptr, dev.put(masks).ptr if n_masks else None, n_masks)
    ok()
    o = ob.get(np.float32, rows * ldo).reshape(rows, ldo)
    assert np.array_equal(bits(o[:, n:]), bits(x[:, n:]) if inplace else bits(np.full((rows, ldo - n), 777.0)))
    for r in range(rows):
        m = rule[r].mask
        mb = np.unpackbits(masks[m].view(np.uint8), bitorder="little").astype(bool) if m >= 0 else None
        want = rules(x[r, :n], n, *par[r], seen[r, :n_seen[r]] if seen_ld else [],
                     zip(b_id[r, :n_bias[r]].tolist(), bias[r, :n_bias[r]].tolist()) if bias_ld else [], mb)
        got = o[r, :n].astype(np.float64)
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin])
        # five roundings, each of a value no larger than these together
        big = np.abs(x[r, :n].astype(np.float64)) * 1.5 + np.abs(par[r, 1]) + par[r, 2] * (seen_ld + 1) + 40
        assert (np.abs(got - want)[fin] <= 6 * U * big[fin]).all()
        touched = np.zeros(n, bool)
        touched[[t for t in list(seen[r, :n_seen[r]] if seen_ld else []) + list(b_id[r, :n_bias[r]] if bias_ld else [])
                 if 0 <= t < n]] = True
        keep = ~touched & fin
        assert np.array_equal(bits(o[r, :n][keep]), bits(x[r, :n][keep]))


def test_rules_bad_counts(dev):
    """counts and masks out of range are reported, and taken as none"""
    rng = np.random.default_rng(0)
    x = f32(rng.standard_normal((4, 100)))
    xb, ob = dev.put(x), dev.zeros(x.nbytes)
    rule = (K.LogitRule * 4)(*[K.LogitRule(1.5, 1.0, 1.0, m) for m in (-1, -1, 2, -2)])
    seen = dev.put(i32(np.arange(20).reshape(4, 5)))
    for n_seen, n_bias in (([6, 0, 0, 0], [0, 0, 0, 0]), ([0, -1, 0, 0], [0, 6, 0, 0])):
        K.hip.krh_logit_rules(ob.ptr, 100, xb.ptr, 100, 100, 4, dev.put(np.frombuffer(bytes(rule), np.uint8)).ptr, seen.ptr, 5,
                              dev.put(i32(n_seen)).ptr, seen.ptr, dev.zeros(80).ptr, 5, dev.put(i32(n_bias)).ptr,
                              dev.zeros(4 * 4 * 2).ptr, 2)
        assert K.hip.krh_sync() == K.ML_E_SHAPE
        K.hip.krh_clear_error()
        assert np.array_equal(bits(ob.get(np.float32, 400)), bits(x).reshape(-1))


def test_captured_as_eager(dev):
    """attention with its mass, eviction and the rules in one graph over one workspace, replayed with other inputs and
    with eager calls over the same workspace between: each replay gives what the calls give"""
    rng = np.random.default_rng(21)
    S, nh, nkv, hd, page, ml, n = 3, 8, 2, 64, 16, 700, 4100
    lens = [700, 33, 400]
    p = Pool(dev, rng, K.ML_F16, lens, page, nkv, hd, spare=3 * 4)
    out = np.full((S, 4), -1, np.int32)
    for i, v in enumerate(lens):
        out[i, :-(-min(v, 50) // page)] = p.free[4 * i:4 * i + -(-min(v, 50) // page)]
    p.put()
    lb, ub, qb = dev.put(i32(lens)), dev.put(out), dev.zeros(S * nh * hd * 4)
    rule = (K.LogitRule * S)(*[K.LogitRule(1.3, 0.2, 0.1, -1)] * S)
    rb, seen, ns, xb = dev.put(np.frombuffer(bytes(rule), np.uint8)), dev.put(i32(rng.integers(0, n, (S, 90)))), dev.put(
        i32([90, 0, 40])), dev.zeros(S * n * 4)
    ws = dev.zeros(max(K.hip.krh_paged_attention_ws(p.ref, S, nh, ml, 1), K.hip.krh_paged_evict_ws(S, nkv, 50)))
    m0 = dev.put(f32(rng.random((S, nkv, ml))))

    def outputs():
        return [dev.zeros(v) for v in (S * nh * hd * 4, S * nkv * ml * 4, 4 * S, S * nkv * 50 * 4, S * n * 4)]

    def calls(o, m, ln, om, y):
        K.hip.krh_copy_d2d_async(m.ptr, m0.ptr, m.nbytes)
        K.hip.krh_paged_attention(o.ptr, p.ref, p.tab.ptr, p.ld, lb.ptr, S, qb.ptr, nh, ml, 0, 0.125, 0.0, m.ptr, ml, ws.ptr)
        K.hip.krh_paged_evict(p.ref, p.tab.ptr, p.ld, lb.ptr, m.ptr, ml, S, ml, 50, 10, ub.ptr, 4, ln.ptr, om.ptr, 50, ws.ptr)
        K.hip.krh_logit_rules(y.ptr, n, xb.ptr, n, n, S, rb.ptr, seen.ptr, 90, ns.ptr, None, None, 0, None, None, 0)

    a, b = outputs(), outputs()
    calls(*a)
    ok()
    g = C.c_void_p()
    K.check(K.hip.krh_graph_begin())
    calls(*b)
    K.check(K.hip.krh_graph_end(C.byref(g)))
    for _ in range(4):
        q, x = f32(rng.standard_normal((S, nh, hd))), f32(rng.standard_normal((S, n)))
        for buf, v in ((qb, q), (xb, x)):
            K.check(K.hip.krh_copy_h2d(buf.ptr, v.ctypes.data, v.nbytes))
        K.check(K.hip.krh_graph_launch(g))
        ok()
        pages = [p.get(v).copy() for v in "kv"]
        calls(*a)
        ok()
        for u, v in zip(a, b):
            assert np.array_equal(u.get(np.uint8, u.nbytes), v.get(np.uint8, v.nbytes))
        assert all(np.array_equal(u, p.get(v)) for u, v in zip(pages, "kv"))
    K.hip.krh_graph_free(g)


@pytest.mark.parametrize("kv_type", TYPES)
def test_steps_together(dev, kv_type):
    """Decode steps of three sequences as a server runs them, each step one replay of a captured graph: new rows into
    pages, attention with its weights kept, the rules, the greedy pick; the cache cut on the way. The same steps
    in 64 bits beside them."""
    rng = np.random.default_rng(12)
    S, nh, nkv, hd, page, n_vocab, ml = 3, 4, 2, 64, 16, 500, 80
    lens = np.array([5, 20, 40])
    p = Pool(dev, rng, kv_type, [ml] * S, page, nkv, hd, spare=S * 3)
    out = np.full((S, p.ld), -1, np.int32)
    out[:, :3] = p.free[:S * 3].reshape(S, 3)
    p.put()
    P = 200
    cs, sn = tables(rng, P, hd)
    up = f32(rng.standard_normal((n_vocab, nh * hd)) * 0.2)
    qb, kb, vb, ob = (dev.zeros(S * n * hd * 4) for n in (nh, nkv, nkv, nh))
    posb, rowb, lenb, massb = dev.zeros(4 * S), dev.zeros(4 * S), dev.zeros(4 * S), dev.put(np.zeros((S, nkv, ml), np.float32))
    lgb, rlb, tokb, seenb, nsb = dev.zeros(S * n_vocab * 4), dev.zeros(S * n_vocab * 4), dev.zeros(4 * S), dev.zeros(
        S * 64 * 4), dev.zeros(4 * S)
    rule = (K.LogitRule * S)(*[K.LogitRule(1.2, 0.1, 0.05, -1)] * S)
    csb, snb, seqb, ruleb = dev.put(cs), dev.put(sn), dev.put(np.arange(S, dtype=np.int32)), dev.put(
        np.frombuffer(bytes(rule), np.uint8))
    ws = dev.zeros(max(K.hip.krh_paged_attention_ws(p.ref, S, nh, ml, 1), K.hip.krh_paged_evict_ws(S, nkv, 24)))

    def put(buf, a):
        K.check(K.hip.krh_copy_h2d(buf.ptr, np.ascontiguousarray(a).ctypes.data, a.nbytes))

    graphs = {}

    def step(tab):
        if tab.ptr not in graphs:
            g = C.c_void_p()
            K.check(K.hip.krh_graph_begin())
            K.hip.krh_paged_qkv(qb.ptr, nh * hd, p.ref, tab.ptr, p.ld, S, qb.ptr, nh * hd, kb.ptr, nkv * hd, vb.ptr, nkv * hd, S,
                                nh, seqb.ptr, rowb.ptr, posb.ptr, None, None, 0.0, csb.ptr, snb.ptr, P)
            K.hip.krh_paged_attention(ob.ptr, p.ref, tab.ptr, p.ld, lenb.ptr, S, qb.ptr, nh, ml, 0, 0.125, 0.0, massb.ptr, ml,
                                      ws.ptr)
            K.check(K.hip.krh_graph_end(C.byref(g)))
            graphs[tab.ptr] = g
        K.check(K.hip.krh_graph_launch(graphs[tab.ptr]))
        ok()

    # the same in 64 bits: each sequence's rows a KV head
    cache = [[(p.rows("k", i, n)[:, g], p.rows("v", i, n)[:, g]) for g in range(nkv)] for i, n in enumerate(lens)]
    mass = [[np.zeros(n) for _ in range(nkv)] for n in lens]
    pos, tab, outb, table = lens.copy(), p.tab, dev.put(out), p.table
    seen = [[] for _ in range(S)]
    for it in range(12):
        q, k, v = (f32(rng.standard_normal((S, n, hd))) for n in (nh, nkv, nkv))
        for b, a in ((qb, q), (kb, k), (vb, v), (posb, i32(pos)), (rowb, i32(lens)), (lenb, i32(lens + 1))):
            put(b, a)
        step(tab)
        lens, pos = lens + 1, pos + 1
        got = {n: p.get(n) for n in p.a}
        o = ob.get(np.float32, S * nh * hd).reshape(S, nh, hd)
        m = massb.get(np.float32, S * nkv * ml).reshape(S, nkv, ml)
        for i in range(S):
            kn, vn = p.rows("k", i, lens[i], got, table)[-1], p.rows("v", i, lens[i], got, table)[-1]
            for g in range(nkv):   # the new row as the pages hold it
                cache[i][g] = tuple(np.vstack([c, x[g]]) for c, x in zip(cache[i][g], (kn, vn)))
                mass[i][g] = np.append(mass[i][g], 0.0)
            c, s = cs[pos[i] - 1], sn[pos[i] - 1]
            for h in range(nh):
                x = q[i, h].astype(np.float64)
                y = np.empty(hd)
                y[0::2], y[1::2] = x[0::2] * c - x[1::2] * s, x[0::2] * s + x[1::2] * c
                g = h * nkv // nh
                w, a, bound, _ = attention(y, *cache[i][g], 0.125, 0, 0)
                assert (np.abs(o[i, h] - w) <= 2 * bound).all(), (it, i, h)
                mass[i][g] += a
            for g in range(nkv):
                assert np.allclose(m[i, g, :lens[i]], mass[i][g], rtol=1e-5, atol=1e-6) and (m[i, g, lens[i]:] == 0).all()
        # logits from the outputs, then the rules and the pick
        lg = f32(o.reshape(S, -1) @ up.T)
        for b, a in ((lgb, lg), (seenb, i32([r + [-1] * (64 - len(r)) for r in seen])), (nsb, i32([len(r) for r in seen]))):
            put(b, a)
        K.hip.krh_logit_rules(rlb.ptr, n_vocab, lgb.ptr, n_vocab, n_vocab, S, ruleb.ptr, seenb.ptr, 64, nsb.ptr, None, None, 0,
                              None, None, 0)
        for i in range(S):
            K.hip.krh_argmax(tokb.ptr + 4 * i, rlb.ptr + 4 * n_vocab * i, n_vocab, None, None)
        ok()
        for i, t in enumerate(tokb.get(np.int32, S)):
            want = rules(lg[i], n_vocab, np.float32(1.2), np.float32(0.1), np.float32(0.05), seen[i], [], None)
            assert want[t] >= want.max() - 1e-5
            seen[i].append(int(t))
        if it == 5:   # the cache cut to 24 rows, the last 8 among them
            K.hip.krh_paged_evict(p.ref, tab.ptr, p.ld, lenb.ptr, massb.ptr, ml, S, ml, 24, 8, outb.ptr, p.ld, lenb.ptr,
                                  massb.ptr, ml, ws.ptr)
            ok()
            for i in range(S):
                for g in range(nkv):
                    r = evicted(m[i, g], lens[i], 24, 8)
                    cache[i][g], mass[i][g] = tuple(c[r] for c in cache[i][g]), mass[i][g][r]
            lens = np.minimum(lens, 24)
            assert lenb.get(np.int32, S).tolist() == lens.tolist()
            tab, table = outb, out
    for g in graphs.values():
        K.hip.krh_graph_free(g)
