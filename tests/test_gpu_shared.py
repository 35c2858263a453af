"""Attention of one token of each sequence where groups of sequences begin with
the same rows of a paged cache, on the device against a plain implementation in
64 bits. Needs a gfx950 device."""
import ctypes as C

import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import Dev, bits, f32, ok
from test_gpu_paged import TYPES, Pool, U, attention, i32

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


class Batch:
    """groups: (sequences, shared rows); alone: sequences before and behind them; own: rows of each sequence behind its
    group's shared ones (negative: it ends within them)"""

    def __init__(self, dev, rng, kv_type, nh, nkv, hd, page, groups, own, alone=(0, 0), copies=False):
        self.start = [alone[0]]
        shared = [0] * alone[0]
        for n, rows in groups:
            self.start.append(self.start[-1] + n)
            shared += [rows] * n
        shared += [0] * alone[1]
        self.shared = [rows for _, rows in groups]
        self.lens = [max(0, s + o) for s, o in zip(shared, own)]
        assert len(own) == len(shared)
        # a leader's table reaches as far as any of its group attends
        reach = list(self.lens)
        for g, (n, rows) in enumerate(groups):
            a = self.start[g]
            reach[a] = max([reach[a]] + [min(rows, v) for v in self.lens[a:a + n]])
        self.p = p = Pool(dev, rng, kv_type, reach, page, nkv, hd)
        for g, (n, rows) in enumerate(groups):
            a = self.start[g]
            for i in range(a + 1, a + n):
                k = min(rows, self.lens[i])
                whole = 0 if copies else k // page
                p.table[i, :whole] = p.table[a, :whole]
                for j in range(whole, -(-k // page)):   # pages of the same rows: the last one, or all
                    m = min(page, k - j * page)
                    for x in p.a.values():
                        x[p.table[i, j], :, :m] = x[p.table[a, j], :, :m]
        self.nh, self.nkv, self.hd, self.dev = nh, nkv, hd, dev
        self.q = f32(rng.standard_normal((len(own), nh, hd)) * 1.5)

    def spoil(self):
        """what lies behind all rows of a page is never attended, whatever it is"""
        p, page = self.p, self.p.page
        used = {}
        for i, n in enumerate(self.lens):
            for j in range(-(-n // page)):
                t = int(p.table[i, j])
                used[t] = max(used.get(t, 0), min(page, n - j * page))
        for g, s in enumerate(self.shared):   # a leader's pages that only others reach
            a, b = self.start[g], self.start[g + 1]
            m = max([0] + [min(s, v) for v in self.lens[a:b]])
            for j in range(-(-m // page)):
                t = int(p.table[a, j])
                used[t] = max(used.get(t, 0), min(page, m - j * page))
        for t in range(p.n):
            for name in "kv":
                x = p.a[name + "d"] if p.kv_type == K.ML_Q8_0 else p.a[name]
                x[t, :, used.get(t, 0):] = np.nan if name == "v" else np.inf
        return self

    def put(self, max_len=None, max_shared=None, window=0):
        """the bounds that the host gives as they are, or so large that sharing pays by them, whatever the lengths are"""
        self.p.put()
        S = len(self.lens)
        self.max_len = max_len or max(max(self.lens), 1)
        self.max_shared = min(self.max_len, max(self.shared)) if max_shared is None else max_shared
        while max_len is None and self.max_len < 2 ** 19 and not self.form(window):
            self.max_len *= 2
            self.max_shared = self.max_len - 1
        self.qb, self.lb = self.dev.put(self.q), self.dev.put(i32(self.lens))
        self.gb, self.sb = self.dev.put(i32(self.start)), self.dev.put(i32([min(s, self.max_shared) for s in self.shared]))
        self.ob = self.dev.put(np.full(self.q.size + 64, 777.0, np.float32))
        self.nb = K.hip.krh_paged_attention_shared_ws(self.p.ref, S, self.nh, self.max_len, len(self.shared), self.max_shared)
        self.ws = self.dev.put(np.full(self.nb + 256, 0xEE, np.uint8))
        return self

    def form(self, window=0):
        return K.hip.krh_paged_attention_shared_form(self.p.ref, len(self.lens), self.nh, self.max_len, len(self.shared),
                                                     self.max_shared, window)

    def run(self, window=0, cap=0.0, ws=None):
        K.hip.krh_paged_attention_shared(self.ob.ptr, self.p.ref, self.p.tab.ptr, self.p.ld, self.lb.ptr, len(self.lens),
                                         self.gb.ptr, self.sb.ptr, len(self.shared), self.max_shared, self.qb.ptr, self.nh,
                                         self.max_len, window, self.hd ** -0.5, cap, (ws or self.ws).ptr)

    def out(self):
        o = self.ob.get(np.float32, self.q.size + 64)
        assert (o[self.q.size:] == 777.0).all()
        assert (self.ws.get(np.uint8, self.nb + 256)[self.nb:] == 0xEE).all()
        return o[:self.q.size].reshape(self.q.shape)

    def check(self, o, window=0, cap=0.0, only=None):
        sq = su = 0.0
        for i, n in enumerate(self.lens):
            if only is not None and i not in only:
                continue
            if n == 0:
                assert (o[i] == 0).all(), i
                continue
            k, v = self.p.rows("k", i, n), self.p.rows("v", i, n)
            for h in range(self.nh):
                g = h * self.nkv // self.nh
                w, _, bound, _ = attention(self.q[i, h].astype(np.float64), k[:, g], v[:, g], self.hd ** -0.5, cap, window)
                err = np.abs(o[i, h] - w)
                assert (err <= bound + 1e-30).all(), (i, h, n, (err / bound).max())
                sq, su = sq + (err ** 2).sum(), su + (w ** 2).sum()
        # over all outputs the roundings are as good as independent
        assert su == 0 or np.sqrt(sq / su) <= 4 * U * np.sqrt(self.hd + max(self.lens))


def check(dev, kv_type, nh, nkv, hd, page, groups, own, window=0, cap=0.0, alone=(0, 0), copies=False, max_len=None, seed=0, form=1):
    rng = np.random.default_rng(seed + hd + 7 * nh + len(own))
    b = Batch(dev, rng, kv_type, nh, nkv, hd, page, groups, own, alone, copies).spoil().put(max_len, window=window)
    assert form is None or b.form(window) == form
    outs = []
    for _ in range(2):
        b.run(window, cap)
        ok()
        outs.append(b.out())
    assert np.array_equal(bits(outs[0]), bits(outs[1]))   # the same from call to call
    b.check(outs[0], window, cap)
    return b


def own_rows(rng, n, most):
    return [int(v) for v in np.exp(rng.uniform(0, np.log(most), n))]


HEADS = [(6, 6, 48), (14, 2, 64), (8, 2, 128), (3, 1, 80), (4, 1, 96), (8, 4, 256), (16, 1, 64), (9, 1, 128), (5, 5, 8),
         (10, 1, 200), (32, 2, 256), (4, 2, 200)]


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_heads(dev, kv_type, nh, nkv, hd):
    check(dev, kv_type, nh, nkv, hd, 16, [(5, 144)], [1, 37, 16, 0, 60], form=None)
    # narrow heads and 16 of a KV head pay for many sequences only, wide ones where few share a KV head
    n, form = 20 if hd > 8 and nh < 16 * nkv and hd != 200 else 100, int(hd <= 128 or nh <= 2 * nkv)
    check(dev, kv_type, nh, nkv, hd, 32, [(n, 320)], own_rows(np.random.default_rng(hd), n, 90), form=form)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("page,shared", [(16, 16), (16, 31), (16, 33), (32, 1), (32, 96), (64, 200), (256, 255), (256, 512),
                                         (1024, 1000)])
@pytest.mark.parametrize("n", [2, 9, 33])
def test_shared_rows(dev, kv_type, page, shared, n):
    """shared rows of any number: the page that they end in is each sequence's own"""
    rng = np.random.default_rng(page + n)
    check(dev, kv_type, 8, 2, 64, page, [(n, shared)], own_rows(rng, n, 50), copies=shared == 200, form=int(n > 2))


@pytest.mark.parametrize("kv_type", TYPES)
def test_groups(dev, kv_type):
    """several groups, one of a single sequence, one of nothing shared, sequences outside them, empty ones"""
    rng = np.random.default_rng(1)
    check(dev, kv_type, 8, 2, 64, 16, [(12, 160), (1, 64), (7, 0), (30, 336), (2, 48)], own_rows(rng, 57, 80), alone=(2, 3))
    own = own_rows(rng, 40, 30)
    own[3], own[20], own[39] = -160, -300, -64
    check(dev, kv_type, 4, 4, 128, 16, [(17, 160), (16, 272), (7, 64)], own)


@pytest.mark.parametrize("kv_type", TYPES)
def test_sequences_within_the_shared_rows(dev, kv_type):
    """sequences that end before the shared rows do, the first of the group among them, and empty ones"""
    check(dev, kv_type, 8, 2, 64, 16, [(9, 160)], [-150, 5, -1, 0, -160, -80, 3, 17, -159])
    check(dev, kv_type, 8, 2, 128, 16, [(20, 96), (9, 200)], [-96] * 20 + [-200, -190, -30, -130, -200, -100, -60, -199, -64])
    check(dev, kv_type, 8, 2, 64, 16, [(9, 64)], [-64] * 9)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("window,cap,form", [(1, 0, 0), (33, 50.0, 0), (400, 2.0, 0), (0, 30.0, 1), (5000, 0, 1)])
def test_window_cap(dev, kv_type, window, cap, form):
    """short windows leave nothing to share: each sequence reads its own"""
    rng = np.random.default_rng(window)
    check(dev, kv_type, 8, 4, 128, 16, [(12, 320), (30, 160)], [1, 40, 0, 333, 25, 600, 7, -20, -320, 90, 100, 320] +
          [200, 5, 40, -100, 33] + own_rows(rng, 25, 60), window=window, cap=cap, form=form)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("window,shared,cap", [(2500, 2800, 0), (2500, 2544, 30.0), (4000, 3008, 0)])
def test_long_windows(dev, kv_type, window, shared, cap):
    """windows that begin within the shared rows, of some sequences or of all, or behind them"""
    rng = np.random.default_rng(window + shared)
    own = own_rows(rng, 60, 300)
    own[1], own[7], own[30], own[41] = 2400, -shared, 2600, -1000
    check(dev, kv_type, 8, 4, 128, 32, [(40, shared), (20, shared - 600)], own, window=window, cap=cap)


@pytest.mark.parametrize("kv_type,hd", [(t, h) for t in TYPES for h in (64, 128, 256)])
def test_many_sequences(dev, kv_type, hd):
    """more columns than a workgroup has, more sequences than lanes"""
    rng = np.random.default_rng(hd)
    check(dev, kv_type, 4, 1, hd, 32, [(75, 224)], own_rows(rng, 75, 40))
    check(dev, kv_type, 2, 1, hd, 16, [(70, 64), (70, 160)], own_rows(rng, 170, 20), alone=(30, 0))


@pytest.mark.parametrize("hd", [40, 128, 256])
@pytest.mark.parametrize("n", [31, 60, 70])
def test_heads_of_a_call(dev, n, hd):
    """480 heads, 944 and 1104: joined by fewer threads a head the more there are"""
    rng = np.random.default_rng(hd + n)
    check(dev, K.ML_F16, 16, 4, hd, 16, [(n - 3, 192)], own_rows(rng, n - 1, 50), alone=(1, 1))


@pytest.mark.parametrize("kv_type", TYPES)
def test_long(dev, kv_type):
    """long shared rows, cut into many parts; a batch whose longest is far under max_len"""
    rng = np.random.default_rng(4)
    check(dev, kv_type, 8, 2, 64, 64, [(10, 5120)], own_rows(rng, 10, 300))
    check(dev, kv_type, 7, 1, 128, 32, [(20, 1600)], own_rows(rng, 20, 100), max_len=20000, form=None)
    check(dev, kv_type, 4, 1, 64, 64, [(3, 640), (32, 2560)], own_rows(rng, 35, 900))


def test_offsets_past_32_bits(dev):
    """shared and own rows in pages beyond 2^31 values"""
    n, nkv, hd, page, S, shared = 270000, 2, 256, 16, 40, 96
    k, v = (K.DevBuf(4 * n * nkv * hd * page) for _ in range(2))
    dev.bufs += [k, v]
    kv = K.KrhPages(k.ptr, v.ptr, None, None, K.ML_F32, n, page, nkv, hd)
    ref, rng = C.byref(kv), np.random.default_rng(12)
    table = np.full((S, 7), -1, np.int32)
    table[:, :6] = [n - 1, 7, n - 2, n // 2 + 1, n - 70, 3]
    table[:, 6] = n - 10 - np.arange(S)
    lens = i32(shared + rng.integers(0, 16, S))
    seq = i32([0] * shared + [i for i in range(S) for _ in range(lens[i] - shared)])
    row = i32(list(range(shared)) + [r for i in range(S) for r in range(shared, lens[i])])
    T, nh = len(seq), 4
    kr, vr = (f32(rng.standard_normal((T, nkv * hd))) for _ in range(2))
    q = f32(rng.standard_normal((S, nh, hd)))
    tb, ob = dev.put(table), dev.zeros(q.nbytes)
    K.hip.krh_paged_qkv(None, 0, ref, tb.ptr, 7, S, None, 0, dev.put(kr).ptr, nkv * hd, dev.put(vr).ptr, nkv * hd, T, 0,
                        dev.put(seq).ptr, dev.put(row).ptr, None, None, None, 0.0, None, None, 0)
    most = 128
    while K.hip.krh_paged_attention_shared_form(ref, S, nh, most, 1, most - 1, 0) != 1:
        most *= 2
    ws = dev.zeros(K.hip.krh_paged_attention_shared_ws(ref, S, nh, most, 1, most - 1))
    K.hip.krh_paged_attention_shared(ob.ptr, ref, tb.ptr, 7, dev.put(lens).ptr, S, dev.put(i32([0, S])).ptr,
                                     dev.put(i32([shared])).ptr, 1, most - 1, dev.put(q).ptr, nh, most, 0, 0.0625, 0.0, ws.ptr)
    ok()
    o = ob.get(np.float32, q.size).reshape(q.shape)
    k64, v64 = (x.reshape(T, nkv, hd).astype(np.float64) for x in (kr, vr))
    for i in range(S):
        at = np.concatenate([np.arange(shared), np.flatnonzero((seq == i) & (row >= shared))])
        for h in range(nh):
            w, _, bound, _ = attention(q[i, h].astype(np.float64), k64[at, h // 2], v64[at, h // 2], 0.0625, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all(), (i, h)


def test_64_groups(dev):
    rng = np.random.default_rng(6)
    check(dev, K.ML_F16, 4, 2, 64, 16, [(3, 16 * (g % 5 + 1)) for g in range(64)], own_rows(rng, 200, 30), alone=(0, 8))


def test_bounds_decide(dev):
    """with the bounds as the lengths are, few rows are each sequence's own and many are shared"""
    rng = np.random.default_rng(7)
    for groups, own, form in (([(4, 208)], [90, 3, 17, 40], 0), ([(64, 4096)], own_rows(rng, 64, 100), 1)):
        b = Batch(dev, rng, K.ML_F16, 8, 2, 128, 16, groups, own).spoil()
        b.put(max_len=max(b.lens), max_shared=groups[0][1])
        assert b.form() == form
        b.run()
        ok()
        b.check(b.out())


def test_long_shared_of_many_kv_heads(dev):
    """more KV heads than workgroups are wanted: a share holds everything"""
    check(dev, K.ML_F16, 2100, 2100, 8, 16, [(100, 48)], [v % 5 for v in range(100)])


def test_equals_the_call_without_shares(dev):
    """to rounding; and the call is the other one where nothing is shared"""
    rng = np.random.default_rng(8)
    b = Batch(dev, rng, K.ML_F16, 8, 2, 64, 16, [(30, 640)], own_rows(rng, 30, 100)).put()
    assert b.form() == 1
    b.run()
    ok()
    o = b.out()
    ws = dev.zeros(K.hip.krh_paged_attention_ws(b.p.ref, 30, 8, b.max_len, 0))
    K.hip.krh_paged_attention(b.ob.ptr, b.p.ref, b.p.tab.ptr, b.p.ld, b.lb.ptr, 30, b.qb.ptr, 8, b.max_len, 0, 0.125, 0.0, None,
                              0, ws.ptr)
    ok()
    o2 = b.out()
    b.check(o)
    b.check(o2)
    b.sb = dev.put(i32([0]))
    for ng, ms in ((0, 0), (0, 640), (1, 0)):
        K.hip.krh_paged_attention_shared(b.ob.ptr, b.p.ref, b.p.tab.ptr, b.p.ld, b.lb.ptr, 30, None if ng == 0 else b.gb.ptr,
                                         None if ng == 0 else b.sb.ptr, ng, ms, b.qb.ptr, 8, b.max_len, 0, 0.125, 0.0,
                                         b.ws.ptr)
        ok()
        assert np.array_equal(bits(b.out()), bits(o2))


@pytest.mark.parametrize("what", ["start", "end", "order", "rows", "negative", "len", "page"])
def test_bad_device_data(dev, what):
    """reported, never used as an address: the outputs' and the workspace's surroundings stay, other groups' results too"""
    rng = np.random.default_rng(9)
    b = Batch(dev, rng, K.ML_F16, 8, 2, 64, 16, [(30, 320), (30, 160)], own_rows(rng, 60, 40)).put()
    start, shared, lens, table = i32(b.start), i32(b.shared), i32(b.lens), b.p.table.copy()
    good = []
    if what == "start":
        start[0] = -5
    elif what == "end":
        start[2] = 61
    elif what == "order":
        start[1] = 2 ** 30
    elif what == "rows":
        shared[1], good = b.max_shared + 1, range(30)   # (then the second group shares nothing)
    elif what == "negative":
        shared[0], good = -7, range(30, 60)
    elif what == "len":
        lens[31], good = b.max_len + 1, [i for i in range(60) if i != 31]
    else:
        table[0, 2], good = 10 ** 6, range(30, 60)
    b.gb, b.sb, b.lb, b.p.tab = (dev.put(x) for x in (start, shared, lens, table))
    b.run()
    assert K.hip.krh_sync() == K.ML_E_SHAPE
    K.hip.krh_clear_error()
    b.check(b.out(), only=good)
    b.gb, b.sb, b.lb, b.p.tab = (dev.put(x) for x in (i32(b.start), i32(b.shared), i32(b.lens), b.p.table))
    b.run()
    ok()
    b.check(b.out())


def test_not_finite(dev):
    """a NaN or an infinite key of one sequence's own row reaches that sequence alone; one in a shared row reaches every
    head that attends it, and no other group"""
    rng = np.random.default_rng(10)
    b = Batch(dev, rng, K.ML_F16, 8, 2, 64, 16, [(30, 320), (30, 160)], [20] * 60)
    p = b.p
    p.a["k"][p.table[3, 20], 1, 5, 7] = np.nan        # row 325 of sequence 3
    p.a["v"][p.table[7, 20], 0, 3, 9] = np.inf        # row 323 of sequence 7
    p.a["k"][p.table[30, 4], 0, 2, 1] = np.nan        # shared row 66 of the second group
    b.put()
    b.run()
    ok()
    o = b.out()
    assert np.isnan(o[3, 4:]).all() and np.isfinite(o[3, :4]).all()
    assert not np.isfinite(o[7, :4, 9]).any() and np.isfinite(np.delete(o[7, :4], 9, 1)).all()
    assert np.isnan(o[30:, :4]).all() and np.isfinite(o[30:, 4:]).all()
    b.check(o, only=[i for i in range(30) if i not in (3, 7)])


def test_captured(dev):
    """two captured calls share a workspace; replays see other lengths, groups and tables, between eager calls"""
    rng = np.random.default_rng(11)
    a = Batch(dev, rng, K.ML_F16, 8, 2, 64, 16, [(20, 320), (13, 96)], own_rows(rng, 33, 60))
    b = Batch(dev, rng, K.ML_Q8_0, 8, 2, 128, 16, [(33, 160)], own_rows(rng, 33, 60))
    a.put(max_len=2 ** 17, max_shared=2 ** 16)
    b.put(max_len=2 ** 17, max_shared=2 ** 16)
    assert a.form() == b.form() == 1
    if b.nb > a.nb:
        a.ws, a.nb = b.ws, b.nb
    else:
        b.ws, b.nb = a.ws, a.nb
    graphs = []
    for x in (a, b):
        K.check(K.hip.krh_graph_begin())
        x.run()
        g = C.c_void_p()
        K.check(K.hip.krh_graph_end(C.byref(g)))
        graphs.append(g)
    for turn in range(4):
        a.lens = [max(0, v - 3 * turn) for v in a.lens]
        lens, start = i32(a.lens), i32([0, 20, 20])
        K.check(K.hip.krh_copy_h2d(a.lb.ptr, lens.ctypes.data, lens.nbytes))
        if turn == 2:   # the second group is dissolved: its sequences' rows are all their own
            K.check(K.hip.krh_copy_h2d(a.gb.ptr, start.ctypes.data, start.nbytes))
        for g in graphs:
            K.check(K.hip.krh_graph_launch(g))
        ok()
        oa, ob = a.out(), b.out()
        a.check(oa)
        b.check(ob)
        a.run()
        b.run()
        ok()
        assert np.array_equal(bits(a.out()), bits(oa)) and np.array_equal(bits(b.out()), bits(ob))
    for g in graphs:
        K.hip.krh_graph_free(g)
