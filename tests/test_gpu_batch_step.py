"""A decode step of a batch behind a common prompt: the 8-bit products, the norms
between blocks and the attention over shared rows of a paged cache as one layer
calls them, eager and captured, each stage against its definition from what the
stage before left. Needs a gfx950 device."""
import ctypes as C

import numpy as np
import pytest

import krafla as K
from test_gpu_batch_ops import Mat, U, product, rms
from test_gpu_kernels import Dev, bits, f32, ok
from test_gpu_shared import Batch, i32

pytestmark = pytest.mark.gpu


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


NH, NKV, HD, DIM, FFN, STEPS, EPS = 8, 2, 64, 272, 352, 3, 1e-5
QKV = (NH + 2 * NKV) * HD
LIVE = 23   # of 26 places: the last three are padding, of no rows


class Layer:
    """post: the blocks' outputs are normed and gated before the residual adds them; else the products add to it"""

    def __init__(self, dev, kv_type, post, window):
        rng = np.random.default_rng(31 + post)
        self.dev, self.post, self.window = dev, post, window
        own = [int(v) for v in rng.integers(STEPS, 70, 20)] + [40, 17, 5]
        # 20 sequences behind 211 rows, three alone, three places without a sequence
        self.b = b = Batch(dev, rng, kv_type, NH, NKV, HD, 16, [(20, 211)], own + [0, 0, 0], (0, 6)).put(window=window)
        assert b.form(window) == (window == 0)   # so short a window has each sequence read its own rows
        self.final = list(b.lens)
        S = len(b.lens)

        def mat(rows, cols, size):
            m = Mat(dev, rng, rows, cols, 16)
            m.s = f32(m.s * size)
            m.sb = dev.put(m.s)
            m.d.d = m.sb.ptr
            return m

        self.wqkv, self.wo = mat(QKV, DIM, 0.1), mat(DIM, NH * HD, 0.01)
        self.w1, self.w3, self.w2 = mat(FFN, DIM, 0.1), mat(FFN, DIM, 0.1), mat(DIM, FFN, 0.01)
        self.w = {}
        for name, n in dict(bias=QKV, norm1=DIM, post1=DIM, gate=DIM, norm2=DIM, post2=DIM, last=DIM).items():
            self.w[name] = f32((name != "bias") + 0.2 * rng.standard_normal(n))
        self.wb = {k: dev.put(v) for k, v in self.w.items()}
        a = rng.random((512, HD // 2)) * 6.28
        self.cos, self.sin = dev.put(f32(np.cos(a))), dev.put(f32(np.sin(a)))
        self.x0 = f32(rng.standard_normal((STEPS, LIVE, DIM)))
        self.at = dict(seq=i32(np.arange(LIVE)), row=i32(np.zeros(LIVE)))
        self.atb = {k: dev.put(v) for k, v in self.at.items()}
        # rows of the intermediate values: their floats, or their bytes a value for 8-bit rows
        self.f = {k: (LIVE, n, dev.zeros(4 * LIVE * n)) for k, n in
                  dict(x=DIM, x1=DIM, x2=DIM, y1=DIM, y2=DIM, z=DIM, qkv=QKV, qr=NH * HD, h=FFN, d1=1, d2=1, d3=1, d4=1).items()}
        self.f["qr"] = (S, NH * HD, dev.zeros(4 * S * NH * HD))
        self.i = {k: (-(-n // 16) * 16, dev.zeros(LIVE * (-(-n // 16) * 16))) for k, n in
                  dict(q1=DIM, q2=NH * HD, q3=DIM, q4=FFN).items()}
        # the attention reads its queries where the rotation left them
        self.qbuf, b.qb = b.qb, self.f["qr"][2]
        self.pages = {n: b.p.a[n].copy() for n in b.p.a}

    def p(self, name):
        return (self.f[name][2] if name in self.f else self.i[name][1]).ptr

    def floats(self, name):
        n, m, b = self.f[name]
        return b.get(np.float32, n * m).reshape(n, m)

    def bytes(self, name, d, cols):
        """8-bit rows with their scales, as product() takes them"""
        ld, b = self.i[name]
        r = type("Rows", (), {})()
        r.v, r.s = b.get(np.int8, LIVE * ld).reshape(LIVE, ld)[:, :cols], self.floats(d)[:, 0]
        return r

    def start(self, step):
        """what the host sets before a step: its tokens' rows, lengths and positions"""
        b = self.b
        b.lens = [n - (STEPS - 1 - step) if n else 0 for n in self.final]
        self.at["row"] = i32([n - 1 for n in b.lens[:LIVE]])
        for dst, src in ((b.lb, i32(b.lens)), (self.atb["row"], self.at["row"]), (self.f["x"][2], self.x0[step])):
            K.check(K.hip.krh_copy_h2d(dst.ptr, src.ctypes.data, src.nbytes))

    def reset(self):
        for n, x in self.pages.items():
            K.check(K.hip.krh_copy_h2d(self.b.p.b[n].ptr, x.ctypes.data, x.nbytes))

    def norm(self, xo, x, y, post, pre, z, q, d):
        w, h = self.wb, K.hip
        h.krh_block_norm(self.p(xo) if xo else None, DIM, self.p(x), DIM, self.p(y) if y else None, DIM, w[post].ptr if post else None,
                         w["gate"].ptr if y else None, 0, 0.7, w[pre].ptr, EPS, self.p(z) if z else None, DIM,
                         self.p(q) if q else None, self.i[q][0] if q else 0, self.p(d) if d else None, DIM, LIVE)

    def product(self, y, ldy, m, q, d, bias=None, add=0):
        K.hip.krh_matmul_i8(self.p(y), ldy, m.ref, self.p(q), self.i[q][0], self.p(d), bias, LIVE, add)

    def eight(self, q, d, x, ldx, n):
        K.hip.krh_quantize_row_rows(self.p(q), self.i[q][0], self.p(d), 1, x, ldx, n, LIVE)

    def step(self):
        h, b = K.hip, self.b
        self.norm(None, "x", None, None, "norm1", None, "q1", "d1")
        self.product("qkv", QKV, self.wqkv, "q1", "d1", self.wb["bias"].ptr)
        qkv = self.p("qkv")
        h.krh_paged_qkv(self.p("qr"), NH * HD, b.p.ref, b.p.tab.ptr, b.p.ld, len(b.lens), qkv, QKV, qkv + 4 * NH * HD, QKV,
                        qkv + 4 * (NH + NKV) * HD, QKV, LIVE, NH, self.atb["seq"].ptr, self.atb["row"].ptr, self.atb["row"].ptr,
                        None, None, EPS, self.cos.ptr, self.sin.ptr, 512)
        b.run(self.window)
        self.eight("q2", "d2", b.ob.ptr, NH * HD, NH * HD)
        if self.post:
            self.product("y1", DIM, self.wo, "q2", "d2")
            self.norm("x1", "x", "y1", "post1", "norm2", None, "q3", "d3")
        else:
            h.krh_copy_d2d_async(self.p("x1"), self.p("x"), 4 * LIVE * DIM)
            self.product("x1", DIM, self.wo, "q2", "d2", None, 1)
            self.norm(None, "x1", None, None, "norm2", None, "q3", "d3")
        h.krh_matmul_i8_swiglu(self.p("h"), FFN, self.w1.ref, self.w3.ref, self.p("q3"), self.i["q3"][0], self.p("d3"), LIVE)
        self.eight("q4", "d4", self.p("h"), FFN, FFN)
        if self.post:
            self.product("y2", DIM, self.w2, "q4", "d4")
            self.norm("x2", "x1", "y2", "post2", "last", "z", None, None)
        else:
            h.krh_copy_d2d_async(self.p("x2"), self.p("x1"), 4 * LIVE * DIM)
            self.product("x2", DIM, self.w2, "q4", "d4", None, 1)
            self.norm(None, "x2", None, None, "last", "z", None, None)

    def outputs(self):
        return {k: bits(self.floats(k)) for k in self.f} | {"o": bits(self.b.out())} | {n: self.b.p.get(n).view(np.uint8) for n in self.pages}

    # ---- each stage from what lies on the device ----

    def check_rows(self, q, d, z, cols):
        """8-bit rows of z, which is known to 4 half steps: a scale a row, and each value at most half a step (and z's
        own error, and the scale's) off"""
        r = self.bytes(q, d, cols)
        big = np.abs(z).max(1)
        assert (np.abs(r.s - big / 127) <= 6 * U * big / 127 + 1e-37).all()
        assert (np.abs(r.v * r.s[:, None].astype(np.float64) - z) <= 0.5 * r.s[:, None] + 16 * U * big[:, None] + 1e-37).all()
        return r

    def check_norm(self, x, y, post, pre, alpha=float(np.float32(0.7))):
        """x' and z in 64 bits, and what x' may be off: as the operator's own test has it"""
        x, w = x.astype(np.float64), {k: v.astype(np.float64) for k, v in self.w.items()}
        eps = float(np.float32(EPS))
        if y is not None:
            v = y.astype(np.float64)
            v = alpha * v * rms(v, eps) * w[post] * w["gate"]
            x, err = x + v, 5.01 * U * np.abs(v) + 1.01 * U * np.abs(x + v)
        else:
            err = np.zeros_like(x)
        return x, err, lambda x2: x2 * rms(x2, eps) * w[pre]

    def check(self):
        F, b = self.floats, self.b
        x0, x1, x2, z = F("x"), F("x1"), F("x2"), F("z")
        _, _, n1 = self.check_norm(x0, None, None, "norm1")
        r = self.check_rows("q1", "d1", n1(x0.astype(np.float64)), DIM)
        assert np.array_equal(bits(F("qkv")), bits(product(self.wqkv, r) + self.w["bias"]))
        # the attention of the rows that lie in the pages by now
        for n in b.p.a:
            b.p.a[n] = b.p.get(n)
        b.q = F("qr").reshape(b.q.shape)
        o = b.out()
        b.check(o, self.window)
        assert (o[LIVE:] == 0).all()
        r = self.check_rows("q2", "d2", o[:LIVE].reshape(LIVE, -1).astype(np.float64), NH * HD)
        y1 = product(self.wo, r)
        if self.post:
            assert np.array_equal(bits(F("y1")), bits(y1))
            want, err, n2 = self.check_norm(x0, y1, "post1", "norm2")
            assert (np.abs(x1 - want) <= err).all()
        else:
            assert np.array_equal(bits(x1), bits(x0 + y1))
            n2 = self.check_norm(x1, None, None, "norm2")[2]
        r = self.check_rows("q3", "d3", n2(x1.astype(np.float64)), DIM)
        g, u = product(self.w1, r).astype(np.float64), product(self.w3, r).astype(np.float64)
        h = F("h")
        want = g / (1 + np.exp(-g)) * u
        assert (np.abs(h - want) <= 8.01 * U * np.abs(want) + 1e-30).all()
        y2 = product(self.w2, self.check_rows("q4", "d4", h.astype(np.float64), FFN))
        if self.post:
            assert np.array_equal(bits(F("y2")), bits(y2))
            want, err, n3 = self.check_norm(x1, y2, "post2", "last")
            assert (np.abs(x2 - want) <= err).all()
        else:
            assert np.array_equal(bits(x2), bits(x1 + y2))
            n3 = self.check_norm(x2, None, None, "last")[2]
        want = n3(x2.astype(np.float64))
        assert (np.abs(z - want) <= 3.01 * U * np.abs(want) + 1e-37).all()


@pytest.mark.parametrize("kv_type", [K.ML_F32, K.ML_F16, K.ML_Q8_0])
@pytest.mark.parametrize("post,window", [(False, 0), (True, 0), (True, 100)])
def test_steps(dev, kv_type, post, window):
    """steps of a layer, each stage against its definition; the captured step's replays leave the same bits"""
    m = Layer(dev, kv_type, post, window)
    eager = []
    for k in range(STEPS):
        m.start(k)
        m.step()
        ok()
        m.check()
        eager.append(m.outputs())
    K.check(K.hip.krh_graph_begin())
    m.step()
    g = C.c_void_p()
    K.check(K.hip.krh_graph_end(C.byref(g)))
    for turn in range(2):
        m.reset()
        for k in range(STEPS):
            m.start(k)
            K.check(K.hip.krh_graph_launch(g))
            ok()
            got = m.outputs()
            for n, v in eager[k].items():
                assert np.array_equal(got[n], v), (turn, k, n)
            if k == 1:   # eager work between replays
                m.step()
                ok()
                got = m.outputs()
                assert all(np.array_equal(got[n], v) for n, v in eager[k].items())
    K.hip.krh_graph_free(g)
