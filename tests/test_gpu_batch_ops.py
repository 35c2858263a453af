"""8-bit products with a scale a token and an output, and the norms between
blocks, on the device against plain implementations: the products bit for bit,
the norms in 64 bits. Needs a gfx950 device."""
import ctypes as C

import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import Dev, bits, f32, ok

pytestmark = pytest.mark.gpu
U = 2.0 ** -24   # half a step of a float, relative


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


# ---- 8-bit products ----

class Mat:
    """int8 rows with a scale each on the host and the device; what lies behind them is not zero"""

    def __init__(self, dev, rng, rows, cols, pad=0, low=-128):
        self.ld = -(-cols // 16) * 16 + pad
        self.q = rng.integers(low, 128, (rows, self.ld)).astype(np.int8)
        self.s = f32(0.001 + 0.01 * rng.random(rows))
        self.cols = cols
        self.qb, self.sb = dev.put(self.q), dev.put(self.s)
        self.d = K.KrhMat8(self.qb.ptr, self.sb.ptr, self.ld, rows, cols)
        self.ref = C.byref(self.d)

    @property
    def v(self):
        return self.q[:, :self.cols]


def product(w, x):
    """the definition, each rounding to 32 bits as it is stated (sums of whole numbers below 2^31 are exact in 64)"""
    s = (x.v.astype(np.float64) @ w.v.astype(np.float64).T).astype(np.float32)
    return (s * x.s[:, None]) * w.s[None, :]


def check_i8(dev, T, rows, cols, bias=False, add=False, pad=0, ldy=None, seed=0):
    rng = np.random.default_rng(seed + 7 * T + 3 * rows + cols)
    w, x = Mat(dev, rng, rows, cols, pad), Mat(dev, rng, T, cols, 2 * pad)
    ldy = ldy or rows
    b = f32(rng.standard_normal(rows)) if bias else None
    y0 = f32(rng.standard_normal((T + 1, ldy)))
    yb, bb = dev.put(y0), dev.put(b) if bias else None
    K.hip.krh_matmul_i8(yb.ptr, ldy, w.ref, x.qb.ptr, x.ld, x.sb.ptr, bb.ptr if bias else None, T, int(add))
    ok()
    want = product(w, x)
    if bias:
        want = want + b
    full = y0.copy()
    full[:T, :rows] = full[:T, :rows] + want if add else want
    got = yb.get(np.float32, y0.size).reshape(y0.shape)
    assert np.array_equal(bits(got), bits(full)), np.argwhere(got != full)[:5]


TOKENS = [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 100, 129, 200, 257]


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (15, 16), (16, 63), (17, 64), (96, 65), (130, 500), (257, 129), (300, 1040)])
def test_i8(dev, T, rows, cols):
    check_i8(dev, T, rows, cols)


@pytest.mark.parametrize("T,rows,cols", [(1, 768, 288), (3, 896, 4864), (16, 1024, 2048), (40, 600, 4096), (128, 512, 896),
                                         (300, 640, 1000), (512, 1024, 256), (513, 1030, 300)])
def test_i8_bias_add_strides(dev, T, rows, cols):
    for bias in (False, True):
        for add in (False, True):
            check_i8(dev, T, rows, cols, bias, add, pad=16 * bias + 32 * add, ldy=rows + 5 * add + 12 * bias)


@pytest.mark.parametrize("T,rows", [(1, 17), (20, 33), (100, 64), (300, 300)])
def test_i8_largest_sums(dev, T, rows):
    """131071 products of -128 and -128 end one below 2^31 - 2^14 + 1"""
    cols = 131071
    q = np.full((max(T, rows), cols + 1), -128, np.int8)
    q[:, -1] = 127
    d = dev.put(np.ones(max(T, rows), np.float32))
    qb = dev.put(q)
    yb = dev.zeros(4 * T * rows)
    w = K.KrhMat8(qb.ptr, d.ptr, cols + 1, rows, cols)
    K.hip.krh_matmul_i8(yb.ptr, rows, C.byref(w), qb.ptr, cols + 1, d.ptr, None, T, 0)
    ok()
    assert (yb.get(np.float32, T * rows) == np.float32(cols * 2.0 ** 14)).all()


@pytest.mark.parametrize("T", [2, 20, 70, 300])
def test_i8_offsets_past_32_bits(dev, T):
    """a matrix of more than 2^32 bytes, into rows more than 2^32 bytes apart; what the other rows hold does not matter"""
    rng = np.random.default_rng(T)
    rows, cols, ld, some = 530000, 8100, 8192, 300
    ldy = max(rows, 2 ** 31 // T)
    w, d, y = K.DevBuf(rows * ld), K.DevBuf(4 * rows), K.DevBuf(4 * (ldy * (T - 1) + rows))
    dev.bufs += [w, d, y]
    q, s = rng.integers(-128, 128, (some, ld)).astype(np.int8), f32(0.01 * rng.random(some))
    K.check(K.hip.krh_copy_h2d(w.ptr + (rows - some) * ld, q.ctypes.data, q.nbytes))
    K.check(K.hip.krh_copy_h2d(d.ptr + 4 * (rows - some), s.ctypes.data, s.nbytes))
    x = Mat(dev, rng, T, cols, 32)
    m = K.KrhMat8(w.ptr, d.ptr, ld, rows, cols)
    K.hip.krh_matmul_i8(y.ptr, ldy, C.byref(m), x.qb.ptr, x.ld, x.sb.ptr, None, T, 0)
    ok()
    want = ((x.v.astype(np.float64) @ q[:, :cols].astype(np.float64).T).astype(np.float32) * x.s[:, None]) * s[None, :]
    for t in range(T):
        got = np.empty(some, np.float32)
        K.check(K.hip.krh_copy_d2h(got.ctypes.data, y.ptr + 4 * (t * ldy + rows - some), got.nbytes))
        assert np.array_equal(bits(got), bits(want[t])), t


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("rows,cols", [(1, 3), (16, 64), (37, 130), (130, 1000), (300, 272)])
def test_i8_swiglu(dev, T, rows, cols):
    """the definition in 64 bits from the products as krh_matmul_i8 leaves them"""
    check_swiglu(dev, T, rows, cols)


def check_swiglu(dev, T, rows, cols):
    rng = np.random.default_rng(T + rows)
    w1, w3, x = Mat(dev, rng, rows, cols), Mat(dev, rng, rows, cols, 48), Mat(dev, rng, T, cols)
    ldh = rows + 3
    h0 = np.full((T, ldh), 55.0, np.float32)
    hb = dev.put(h0)
    K.hip.krh_matmul_i8_swiglu(hb.ptr, ldh, w1.ref, w3.ref, x.qb.ptr, x.ld, x.sb.ptr, T)
    ok()
    h = hb.get(np.float32, h0.size).reshape(h0.shape)
    assert (h[:, rows:] == 55.0).all()
    g, u = product(w1, x).astype(np.float64), product(w3, x).astype(np.float64)
    want = g / (1 + np.exp(-g)) * u
    # half steps: the power 2 (the instruction's last bit) and 1 (its second part's sum), whose share of 1 + e^-g is less
    # than 1; the sum 1, the reciprocal 2, the two products 1 each
    assert (np.abs(h[:, :rows] - want) <= 8.01 * U * np.abs(want) + 1e-30).all()
    # a token's bits do not depend on the others
    hb2 = dev.zeros(4 * rows)
    t = T // 2
    K.hip.krh_matmul_i8_swiglu(hb2.ptr, rows, w1.ref, w3.ref, x.qb.ptr + t * x.ld, x.ld, x.sb.ptr + 4 * t, 1)
    ok()
    assert np.array_equal(bits(hb2.get(np.float32, rows)), bits(h[t, :rows]))


@pytest.mark.parametrize("scale", [0.02, 0.3, 3.0, 1e4, 1e30])
def test_i8_swiglu_range(dev, scale):
    """from products near zero to those whose power leaves the floats, both signs"""
    rng = np.random.default_rng(3)
    w1, w3, x = Mat(dev, rng, 64, 100), Mat(dev, rng, 64, 100), Mat(dev, rng, 40, 100)
    for m, f in ((w1, scale), (w3, min(scale, 1.0))):
        m.s = f32(m.s * f)
        m.sb = dev.put(m.s)
        m.d.d = m.sb.ptr
    hb = dev.zeros(4 * 40 * 64)
    K.hip.krh_matmul_i8_swiglu(hb.ptr, 64, w1.ref, w3.ref, x.qb.ptr, x.ld, x.sb.ptr, 40)
    ok()
    h = hb.get(np.float32, 40 * 64).reshape(40, 64)
    g, u = product(w1, x).astype(np.float64), product(w3, x).astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g)) * u
    assert (np.abs(h - want) <= 8.01 * U * np.abs(want) + 1e-35 * (1 + np.abs(u))).all()


FORMS = [(0, 5, 40, 100), (0, 40, 200, 1300), (1, 8, 16000, 300), (8, 20, 3000, 1000), (8, 32, 4096, 5000), (2, 33, 4100, 300), (3, 33, 9000, 700), (4, 130, 6000, 1500), (5, 200, 9000, 5000),
         (6, 1030, 3000, 200), (7, 2050, 6000, 2100)]
PAIR_FORMS = [(0, 5, 40, 300), (0, 16, 3000, 130), (6, 16, 9000, 130), (0, 50, 300, 1100), (1, 20, 5000, 600), (2, 33, 4100, 700), (4, 100, 4100, 2100), (5, 100, 9000, 5000), (6, 700, 2100, 130),
              (7, 1500, 4100, 2100)]


@pytest.mark.parametrize("form,T,rows,cols", FORMS)
def test_i8_forms(dev, form, T, rows, cols):
    """each of the forms, by sizes that take it"""
    assert K.hip.krh_matmul_i8_form(rows, cols, T, 0) == form
    check_i8(dev, T, rows, cols, bias=True, add=True, ldy=rows + 3)


@pytest.mark.parametrize("form,T,rows,cols", PAIR_FORMS)
def test_i8_swiglu_forms(dev, form, T, rows, cols):
    assert K.hip.krh_matmul_i8_form(rows, cols, T, 1) == form
    check_swiglu(dev, T, rows, cols)


def test_i8_captured(dev):
    """replays of a captured pair of products see new inputs"""
    rng = np.random.default_rng(2)
    w, xs = Mat(dev, rng, 200, 320), [Mat(dev, rng, 70, 320) for _ in range(3)]
    xb, sb, yb = dev.put(xs[0].q), dev.put(xs[0].s), dev.zeros(4 * 70 * 200)

    def step():
        K.hip.krh_matmul_i8(yb.ptr, 200, w.ref, xb.ptr, xs[0].ld, sb.ptr, None, 70, 0)
        K.hip.krh_matmul_i8(yb.ptr, 200, w.ref, xb.ptr, xs[0].ld, sb.ptr, None, 5, 1)

    K.check(K.hip.krh_graph_begin())
    step()
    g = C.c_void_p()
    K.check(K.hip.krh_graph_end(C.byref(g)))
    for x in xs + xs:
        K.check(K.hip.krh_copy_h2d(xb.ptr, x.q.ctypes.data, x.q.nbytes))
        K.check(K.hip.krh_copy_h2d(sb.ptr, x.s.ctypes.data, x.s.nbytes))
        K.check(K.hip.krh_graph_launch(g))
        ok()
        want = product(w, x)
        want[:5] = want[:5] + want[:5]
        assert np.array_equal(bits(yb.get(np.float32, want.size).reshape(want.shape)), bits(want))
        step()
        ok()
        assert np.array_equal(bits(yb.get(np.float32, want.size).reshape(want.shape)), bits(want))
    K.hip.krh_graph_free(g)


# ---- the norms between blocks ----

def rms(v, eps):
    return 1 / np.sqrt((v * v).mean(1, keepdims=True) + eps)


def check_norm(dev, n, rows, y=True, post=True, gate="channel", alpha=0.7, pre=True, xo=True, z=True, q=True, pad=0, off=0,
               eps=1e-6, place=None, scale=1.0, seed=0):
    """off: floats by which each array starts past an aligned address"""
    rng = np.random.default_rng(seed + n + 13 * rows)
    ld = n + pad

    def rows_of(k, f):
        return f32(rng.standard_normal((k, ld)) * f)

    def put(a):
        return dev.put(np.concatenate([np.zeros(off, a.dtype), a.reshape(-1), np.full(8, 99, a.dtype)]))

    def at(b, size=4):
        return b.ptr + off * size if b is not None else None

    xv, yv = rows_of(rows, 2.0 * scale), rows_of(rows, 0.5 * scale)
    pw, rw = f32(1 + 0.2 * rng.standard_normal(n)), f32(1 + 0.2 * rng.standard_normal(n))
    gv = rows_of(rows, 1.0) if gate == "token" else f32(rng.standard_normal(n))
    xb, yb, gb, pb, rb = put(xv), put(yv), put(gv), put(pw), put(rw)
    fill = np.full((rows, ld), 33.0, np.float32)
    xob = xb if place == "x" else put(fill) if xo else None
    zb = yb if place == "x" else put(fill) if z else None
    qb, db = (put(np.full((rows, ld), 33, np.int8)), put(np.full(rows, 33.0, np.float32))) if q else (None, None)
    K.hip.krh_block_norm(at(xob), ld, at(xb), ld, at(yb) if y else None, ld, at(pb) if post else None,
                         at(gb) if gate else None, ld if gate == "token" else 0, alpha, at(rb) if pre else None, eps,
                         at(zb), ld, at(qb, 1), ld, at(db), n, rows)
    ok()

    def get(b, a, dt=np.float32):
        v = b.get(dt, off + a.size + 8)
        assert (v[:off] == 0).all() and (v[off + a.size:] == 99).all()
        return v[off:off + a.size].reshape(a.shape)

    x64, y64 = xv[:, :n].astype(np.float64), yv[:, :n].astype(np.float64)
    eps, alpha = float(np.float32(eps)), float(np.float32(alpha))
    want, err = x64, 0.0
    if y:
        b = y64 * rms(y64, eps) * pw if post else y64
        if gate:
            b = b * (gv[:, :n] if gate == "token" else gv)
        want = x64 + alpha * b
        # half a step each: the reciprocal root and its two products, the gate's product, alpha's, the sum
        err = (3 * post + bool(gate) + 1.01) * U * np.abs(alpha * b) + 1.01 * U * np.abs(want)
    got = None
    if xo:
        full = get(xob, fill)
        got = full[:, :n]
        assert (np.abs(got - want) <= err + 1e-37).all()
        assert np.array_equal(full[:, n:], (xv if place == "x" else fill)[:, n:])
    if z:
        full = get(zb, fill)
        assert np.array_equal(full[:, n:], (yv if place == "x" else fill)[:, n:])
        if xo:   # of the x' that was stored: the reciprocal root and two products
            x2 = got.astype(np.float64)
            w = x2 * rms(x2, eps) * rw
            assert (np.abs(full[:, :n] - w) <= 3.01 * U * np.abs(w) + 1e-37).all()
    if q and z:   # krh_quantize_row_rows of that z
        q2, d2 = dev.zeros(rows * ld), dev.zeros(4 * rows)
        src = dev.put(full)
        K.hip.krh_quantize_row_rows(q2.ptr, ld, d2.ptr, 1, src.ptr, ld, n, rows)
        ok()
        qv = get(qb, np.empty((rows, ld), np.int8), np.int8)
        assert np.array_equal(qv[:, :n], q2.get(np.int8, rows * ld).reshape(rows, ld)[:, :n])
        assert (qv[:, n:] == 33).all()
        assert np.array_equal(bits(get(db, np.empty(rows, np.float32))), bits(d2.get(np.float32, rows)))
    return got, (full[:, :n] if z else None), (qb, db)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 64, 255, 288, 896, 1023, 1024, 1025, 2048, 4095, 4096, 4097, 4100, 8192, 14336,
                               16383, 16384])
@pytest.mark.parametrize("rows", [1, 5])
def test_block_norm_sizes(dev, n, rows):
    check_norm(dev, n, rows)
    check_norm(dev, n, rows, pad=4, gate="token")
    check_norm(dev, n, rows, pad=3, off=1, gate="token")


@pytest.mark.parametrize("kw", [dict(y=False, post=False, gate=None), dict(y=False, post=False, gate=None, xo=False),
                                dict(post=False), dict(gate=None), dict(post=False, gate=None, alpha=1.0),
                                dict(pre=False, z=False, q=False), dict(z=False), dict(q=False), dict(xo=False),
                                dict(place="x"), dict(place="x", pad=8), dict(alpha=-3.0, eps=0.1), dict(alpha=0.0),
                                dict(scale=1e-12), dict(scale=1e18), dict(scale=1e-25, eps=0.0)], ids=str)
def test_block_norm_forms(dev, kw):
    for n in (100, 1001, 4096):
        check_norm(dev, n, 3, **kw)


def test_block_norm_q_alone(dev):
    """the 8-bit rows do not depend on which other outputs are asked for"""
    for n in (288, 4099):
        a = check_norm(dev, n, 4)
        b = check_norm(dev, n, 4, z=False, xo=False)
        for k, (dt, m) in enumerate(((np.int8, 4 * n), (np.float32, 4))):
            assert np.array_equal(a[2][k].get(dt, m), b[2][k].get(dt, m))


def test_block_norm_many_rows(dev):
    check_norm(dev, 48, 5000)
    check_norm(dev, 4, 65535, gate="token")


def test_block_norm_rows_without_numbers(dev):
    """zeros give zeros; a NaN or infinity anywhere in a row shows in its scale, and other rows do not see it"""
    n, rows = 300, 6
    x = f32(np.random.default_rng(1).standard_normal((rows, n)))
    x[0] = 0
    x[2, 7] = np.nan
    x[3, 299] = np.inf
    w = np.ones(n, np.float32)
    w2 = w.copy()
    w2[5] = np.nan
    xb, wb, zb, qb, db = dev.put(x), dev.put(w), dev.zeros(x.nbytes), dev.zeros(rows * n), dev.zeros(4 * rows)
    K.hip.krh_block_norm(None, n, xb.ptr, n, None, 0, None, None, 0, 1.0, wb.ptr, 1e-6, zb.ptr, n, qb.ptr, n, db.ptr, n, rows)
    ok()
    q, d = qb.get(np.int8, rows * n).reshape(rows, n), db.get(np.float32, rows)
    assert (q[0] == 0).all() and d[0] == 0 and np.isnan(d[2]) and not np.isfinite(d[3]) and np.isfinite(d[[1, 4, 5]]).all()
    K.hip.krh_block_norm(None, n, xb.ptr, n, None, 0, None, None, 0, 1.0, dev.put(w2).ptr, 1e-6, None, 0, qb.ptr, n, db.ptr, n,
                         rows)
    ok()
    assert np.isnan(db.get(np.float32, rows)).all()


@pytest.mark.parametrize("n,off,ld", [(1, 0, 1), (7, 0, 7), (64, 0, 64), (64, 1, 67), (1000, 0, 1004), (5001, 3, 5001)])
def test_dequantize_rows(dev, n, off, ld):
    rng = np.random.default_rng(n)
    q, d = rng.integers(-128, 128, (5, ld)).astype(np.int8), f32(rng.random((5, 2)))
    qb, db = dev.put(np.concatenate([np.zeros(off, np.int8), q.reshape(-1)])), dev.put(d)
    x0 = np.full(off + 5 * ld, 7.0, np.float32)
    xb = dev.put(x0)
    K.hip.krh_dequantize_row_rows(xb.ptr + 4 * off, ld, qb.ptr + off, ld, db.ptr, 2, n, 5)
    ok()
    want = np.full((5, ld), 7.0, np.float32)
    want[:, :n] = q[:, :n].astype(np.float32) * d[:, :1]
    got = xb.get(np.float32, x0.size)
    assert (got[:off] == 7.0).all() and np.array_equal(got[off:].reshape(5, ld), want)
