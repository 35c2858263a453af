"""The paged cache's operators and the logit rules on the device at the edges
of what their calls allow. Needs a gfx950 device."""
import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import bits, f32, ok
from test_gpu_paged import NP, TYPES, Pool, U, attention, dev, device, i32, rules, tables  # noqa: F401  (dev, device: fixtures)

pytestmark = pytest.mark.gpu


def at_end(d, a):
    """the address of `a` on the device where its last value is its buffer's last (buffers are whole multiples of 2 MiB)"""
    size = 2 << 20
    assert a.nbytes <= size
    x = np.zeros(size, np.uint8)
    x[size - a.nbytes:] = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
    return d.put(x).ptr + size - a.nbytes


@pytest.mark.parametrize("n,seen_ld,bias_ld,n_seen,n_bias", [(300, 3000, 2000, 10, 3), (32000, 5000, 1500, 2049, 1025), (4097, 700, 9, 0, 0),
                                                             (50, 4, 4, 4, 4)])
def test_rules_last_row_to_its_count(dev, n, seen_ld, bias_ld, n_seen, n_bias):  # noqa: F811
    """rows wider than what they count, the last one allocated to its count alone; ids behind the other's count do not"""
    rng = np.random.default_rng(n)
    x = f32(rng.standard_normal((2, n)) * 3)
    seen, b_id = i32(rng.integers(0, n, seen_ld + n_seen)), i32(rng.integers(0, n, bias_ld + n_bias))
    bias = f32(rng.standard_normal(bias_ld + n_bias))
    counts = [(seen_ld // 2, n_seen), (bias_ld // 2, n_bias)]
    rule = (K.LogitRule * 2)(*[K.LogitRule(1.25, 0.5, 0.125, -1)] * 2)
    ob = dev.zeros(x.nbytes)
    K.hip.krh_logit_rules(ob.ptr, n, dev.put(x).ptr, n, n, 2, dev.put(np.frombuffer(bytes(rule), np.uint8)).ptr, at_end(dev, seen),
                          seen_ld, at_end(dev, i32(counts[0])), at_end(dev, b_id), at_end(dev, bias), bias_ld,
                          at_end(dev, i32(counts[1])), None, 0)
    ok()
    o = ob.get(np.float32, 2 * n).reshape(2, n)
    for r in range(2):
        s, b = (slice(r * ld, r * ld + c[r]) for ld, c in ((seen_ld, counts[0]), (bias_ld, counts[1])))
        want = rules(x[r], n, 1.25, 0.5, 0.125, seen[s], zip(b_id[b].tolist(), bias[b].tolist()), None)
        # five roundings, each of a value no larger than these together
        big = np.abs(x[r].astype(np.float64)) * 1.25 + 0.5 + 0.125 * (counts[0][r] + 1) + 8
        assert (np.abs(o[r] - want) <= 6 * U * big).all()
        same = np.setdiff1d(np.arange(n), np.concatenate([seen[s], b_id[b]]))
        assert np.array_equal(bits(o[r][same]), bits(x[r][same]))


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("at", [5, -1, 2**31 - 1])
def test_qkv_bad_position_stores_nothing(dev, kv_type, at):  # noqa: F811
    """a token whose position is outside the tables leaves both its rows as they were, and is reported"""
    rng = np.random.default_rng(3)
    p = Pool(dev, rng, kv_type, [20, 20], 16, 2, 64).put()
    seq, row, pos = i32([0, 1, 1]), i32([3, 4, 19]), i32([0, at, 4])
    k, v = f32(rng.standard_normal((3, 128))), f32(rng.standard_normal((3, 128)))
    q = f32(rng.standard_normal((3, 256)))
    cs, sn = dev.put(np.ones((5, 32), np.float32)), dev.put(np.zeros((5, 32), np.float32))
    K.hip.krh_paged_qkv(dev.zeros(q.nbytes).ptr, 256, p.ref, p.tab.ptr, p.ld, 2, dev.put(q).ptr, 256, dev.put(k).ptr, 128,
                        dev.put(v).ptr, 128, 3, 4, dev.put(seq).ptr, dev.put(row).ptr, dev.put(pos).ptr, None, None, 0.0, cs.ptr,
                        sn.ptr, 5)
    assert K.hip.krh_sync() == K.ML_E_SHAPE and b"position" in K.hip.krh_last_error()
    K.hip.krh_clear_error()
    for name in p.a:
        got, want = p.get(name), p.a[name].copy()
        for t in (0, 2):
            x = (p.table[seq[t], row[t] // 16], slice(None), row[t] % 16)
            assert not np.array_equal(got[x], want[x])
            want[x] = got[x]
        assert np.array_equal(got, want), name


def attend(d, p, lens, q, nh, mass, scale=1.0, cap=0.0, max_len=None):
    """the outputs, and the masses from zero (or None), of one call"""
    S, ml = len(lens), max_len or max(lens)
    ob, mb = d.zeros(q.nbytes), d.zeros(S * p.nkv * ml * 4)
    ws = d.zeros(K.hip.krh_paged_attention_ws(p.ref, S, nh, ml, int(mass)))
    K.hip.krh_paged_attention(ob.ptr, p.ref, p.tab.ptr, p.ld, d.put(i32(lens)).ptr, S, d.put(f32(q)).ptr, nh, ml, 0, scale, cap,
                              mb.ptr if mass else None, ml, ws.ptr)
    ok()
    return (ob.get(np.float32, q.size).reshape(S, nh, p.hd).astype(np.float64),
            mb.get(np.float32, S * p.nkv * ml).reshape(S, p.nkv, ml).astype(np.float64) if mass else None)


def along_first(p, z, rows, seq):
    """K of the sequence's rows: z (for a query of ones times the first unit vector) on the first dim, nothing on the others"""
    at = (p.table[seq, rows // p.page], slice(None), rows % p.page)
    p.a["k"][at] = 0
    if p.kv_type == K.ML_Q8_0:
        p.a["k"][at + (0,)] = np.sign(z).astype(np.int8)[:, None]
        p.a["kd"][at] = np.abs(z)[:, None]
    else:
        p.a["k"][at + (0,)] = np.asarray(z)[:, None]


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("n", [33, 3000])
@pytest.mark.parametrize("mass", [False, True])
def test_attention_of_large_equal_scores(dev, kv_type, n, mass):  # noqa: F811
    """scores past 2^24, whose steps are larger than the weights' scale: rows of one score share their weight, whatever it is"""
    rng = np.random.default_rng(n)
    scores = [c * 2.0 ** e for e in (20, 24, 25, 26, 27, 28, 30) for c in (1.0, 1.125, 1.5, 1.875)]
    lens = [n if i < 2 else 33 for i in range(len(scores))]
    p = Pool(dev, rng, kv_type, lens, 16, 1, 64)
    q = np.zeros((len(scores), 1, 64), np.float32)
    for i, z in enumerate(scores):
        rows = np.arange(lens[i])
        along_first(p, np.where(rows % 3 == 1, -1.0, 1.0), rows, i)   # every third row far below the others
        q[i, 0, 0] = z
    p.put()
    o, m = attend(dev, p, lens, q, 1, mass)
    for i, ln in enumerate(lens):
        high = np.arange(ln) % 3 != 1
        a = high / high.sum()
        v = p.rows("v", i, ln)[:, 0]
        # equal weights are 1 before their sum: what is left are the sums over n rows and the quotient
        rel = 2 * (ln + 64) * U
        assert (np.abs(o[i, 0] - a @ v) <= rel * (a @ np.abs(v))).all(), (i, scores[i])
        if mass:
            assert (np.abs(m[i, 0, :ln] - a) <= rel * a).all() and (m[i, 0, ln:] == 0).all()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("mass", [False, True])
def test_attention_weights_keep_their_bits(dev, kv_type, mass):  # noqa: F811
    """Two rows, whose weights' quotient e^-t, 0 < t < 1, the outputs show.

    In half steps U, at most: the score's factor and product (8 bits: one product more) 2 (3) t, the power 2 (a step of a
    value over 1/2), the operand's two halves 2 (a half step of the lower one), the two outputs' products 2. Spread evenly
    within these, but for the power's which may lie on one side: a root mean square of 2.6 U, with a tenth for the sample."""
    rng = np.random.default_rng(1)
    S = 1000
    p = Pool(dev, rng, kv_type, [2] * S, 16, 1, 64, fill=False)
    t = rng.random(S) * 0.98 + 0.01
    t = (t.astype(np.float16) if kv_type == K.ML_F16 else f32(t)).astype(np.float64)
    for i in range(S):
        along_first(p, np.array([0.0, -t[i]]), np.arange(2), i)
        at = p.table[i, 0]
        p.a["v"][at, 0, [0, 1], [0, 1]] = 64 if kv_type == K.ML_Q8_0 else 1
        if kv_type == K.ML_Q8_0:
            p.a["vd"][at, 0, :2] = 2.0 ** -6
    p.put()
    q = np.zeros((S, 1, 64), np.float32)
    q[:, 0, 0] = 1
    o, m = attend(dev, p, [2] * S, q, 1, mass)
    for x, y in [(o[:, 0, 0], o[:, 0, 1])] + ([(m[:, 0, 0], m[:, 0, 1])] if mass else []):
        err = y / x / np.exp(-t) - 1
        assert np.abs(err).max() <= 9 * U, np.abs(err).max() / U
        assert np.sqrt((err ** 2).mean()) <= 2.9 * U, np.sqrt((err ** 2).mean()) / U


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_small_weights(dev, kv_type):  # noqa: F811
    """Weights down to 2^-36 of the largest, each on a dim of its own: to 2^-22 (two halves) and the score's roundings
    of their value, and below 2^-17 of the largest to 2^-39 of it"""
    rng = np.random.default_rng(2)
    n = 64
    p = Pool(dev, rng, kv_type, [n], 16, 1, 64, fill=False)
    r = np.arange(n)
    t = (r * 0.4).astype(np.float16).astype(np.float64)
    along_first(p, -t, r, 0)
    p.a["v"][p.table[0, r // 16], 0, r % 16, r] = 64 if kv_type == K.ML_Q8_0 else 1
    if kv_type == K.ML_Q8_0:
        p.a["vd"][p.table[0, r // 16], 0, r % 16] = 2.0 ** -6
    p.put()
    q = np.zeros((1, 1, 64), np.float32)
    q[0, 0, 0] = 1
    o, _ = attend(dev, p, [n], q, 1, False)
    a = np.exp(-t)
    a /= a.sum()
    assert (np.abs(o[0, 0] - a) <= (3 * t + 80) * U * a + 2.0 ** -39 * a.max()).all()


@pytest.mark.parametrize("ratio", [2.0 ** 20, 2.0 ** 30, 2.0 ** 60])
@pytest.mark.parametrize("n,far", [(250, 0), (250, 100), (250, 249), (5000, 3), (5000, 2600)])
def test_attention_large_scale_without_weight(dev, ratio, n, far):  # noqa: F811
    """an 8-bit row of a large scale that no head looks at takes no bits of the others, wherever it lies"""
    rng = np.random.default_rng(n + far)
    lens = [n, 40]
    p = Pool(dev, rng, K.ML_Q8_0, lens, 16, 2, 64)
    q = f32(np.abs(rng.standard_normal((2, 4, 64))) + 0.1)
    at = (p.table[0, far // 16], slice(None), far % 16)
    p.a["vd"][at] *= np.float32(ratio)
    p.a["k"][at], p.a["kd"][at] = -127, 8.0     # a score under -100 for every head
    p.put()
    o, _ = attend(dev, p, lens, q, 4, n == 250, scale=0.125)
    for i, ln in enumerate(lens):
        k, v = p.rows("k", i, ln), p.rows("v", i, ln)
        for h in range(4):
            keep = np.ones(ln, bool)
            if i == 0:      # the row has no weight at all, and its own score's error is no other row's
                z = (k[:, h // 2] @ q[0, h]) * 0.125
                assert z[far] - z.max() < -100
                keep[far] = False
            w, _, bound, _ = attention(q[i, h].astype(np.float64), k[keep, h // 2], v[keep, h // 2], 0.125, 0, 0)
            assert (np.abs(o[i, h] - w) <= bound).all(), (i, h, (np.abs(o[i, h] - w) / bound).max())


@pytest.mark.parametrize("mass", [False, True])
def test_attention_scales_behind_a_new_maximum(dev, mass):  # noqa: F811
    """rows of large scales first, then rows of small scales whose scores leave those without weight, and the other way round"""
    rng = np.random.default_rng(11)
    lens = [200, 200, 64, 3000]
    p = Pool(dev, rng, K.ML_Q8_0, lens, 16, 1, 64)
    q = np.zeros((4, 1, 64), np.float32)
    q[:, 0, 0] = 1
    for i, n in enumerate(lens):
        r = np.arange(n)
        late = r >= n // 2 if i != 1 else r < n // 2
        along_first(p, np.where(late, 90.0, 0.5) + rng.random(n), r, i)
        at = (p.table[i, r // 16], 0, r % 16)
        p.a["vd"][at] *= f32(np.where(late, 2.0 ** -20, 2.0 ** 20))
    p.put()
    o, m = attend(dev, p, lens, q, 1, mass)
    for i, n in enumerate(lens):
        k, v = p.rows("k", i, n)[:, 0], p.rows("v", i, n)[:, 0]
        w, a, bound, rel = attention(q[i, 0].astype(np.float64), k, v, 1.0, 0, 0)
        assert (np.abs(o[i, 0] - w) <= bound).all(), (i, (np.abs(o[i, 0] - w) / bound).max())
        if mass:
            assert (np.abs(m[i, 0, :n] - a) <= rel * a + 1e-30).all()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (8, 1, 128), (3, 3, 48), (2, 1, 256)])
def test_qkv_normed_rows(dev, kv_type, nh, nkv, hd):  # noqa: F811
    """Normalized heads: values are stored as without a norm, bit for bit; 8-bit keys' scales are their rows' maxima over
    127, and scale times element is the key within half a step.

    In 32 bits a normalized and rotated value errs by at most 10 U of its row's largest before the rotation (the factor, two
    products, then two products and a sum of two values), its maximum by as much; the element's factor and product by 4 U."""
    rng = np.random.default_rng(hd)
    T, page = 30, 16
    p = Pool(dev, rng, kv_type, [T], page, nkv, hd).put()
    k, v, q = (f32(rng.standard_normal((T, n * hd)) * 3) for n in (nkv, nkv, nh))
    v[4] = 0
    pos = i32(rng.integers(0, 50, T))
    cs, sn = tables(rng, 50, hd)
    kw = f32(1 + 0.1 * rng.standard_normal(hd))
    K.hip.krh_paged_qkv(dev.zeros(q.nbytes).ptr, nh * hd, p.ref, p.tab.ptr, p.ld, 1, dev.put(q).ptr, nh * hd, dev.put(k).ptr,
                        nkv * hd, dev.put(v).ptr, nkv * hd, T, nh, dev.zeros(4 * T).ptr, dev.put(i32(np.arange(T))).ptr,
                        dev.put(pos).ptr, dev.put(kw).ptr, dev.put(kw).ptr, 1e-6, dev.put(cs).ptr, dev.put(sn).ptr, 50)
    ok()
    got = {n: p.get(n) for n in p.a}
    for t in range(T):
        at = (p.table[0, t // page], slice(None), t % page)
        x = v[t].reshape(nkv, hd)
        if kv_type == K.ML_Q8_0:
            m = np.abs(x).max(1, keepdims=True)
            assert np.array_equal(bits(got["vd"][at]), bits(m[:, 0] / np.float32(127)))
            with np.errstate(divide="ignore", invalid="ignore"):
                e = np.trunc(x * (np.float32(127) * (np.float32(1) / m)) + np.copysign(np.float32(0.5), x))
            assert np.array_equal(got["v"][at], np.where(m < 1e-30, 0, e).astype(np.int8))
        else:
            assert np.array_equal(got["v"][at].view(np.uint8), np.ascontiguousarray(x.astype(NP[kv_type])).view(np.uint8))
        x = k[t].reshape(nkv, hd).astype(np.float64)
        x = x / np.sqrt((x ** 2).mean(1, keepdims=True) + 1e-6) * kw
        pre = np.abs(x).max(1)
        a, b, c, s = x[:, 0::2], x[:, 1::2], cs[pos[t]], sn[pos[t]]
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = a * c - b * s, a * s + b * c
        g = got["k"][at].astype(np.float64)
        if kv_type == K.ML_Q8_0:
            d = got["kd"][at].astype(np.float64)
            assert (np.abs(d - np.abs(y).max(1) / 127) <= 11 * U * pre / 127).all()
            assert (np.abs(g * d[:, None] - y) <= d[:, None] * (0.5 + 127 * 4 * U) + 10 * U * pre[:, None]).all()
            assert (np.abs(g).max(1) == 127).all()
        else:
            step = 2.0 ** -11 if kv_type == K.ML_F16 else 0.0
            assert (np.abs(g - y) <= step * np.abs(y) + 12 * U * pre[:, None] + (2.0 ** -25 if step else 0)).all()


def test_rules_on_most_ids(dev):  # noqa: F811
    """as many ids as an int counts, and ids at both ends of the ints, on a row in place"""
    n = 2 ** 31 - 1
    xb = K.DevBuf(4 * n)
    dev.bufs.append(xb)
    at = [0, 1, 5, 4095, 4096, n - 4097, n - 4096, n - 2, n - 1]
    for i in at:
        v = f32([i % 97 + 1])
        K.check(K.hip.krh_copy_h2d(xb.ptr + 4 * i, v.ctypes.data, 4))
    seen = i32([0, n - 1, 5, -1, -2 ** 31, 5, 2 ** 31 - 1, n - 4097, -2 ** 31 + 1])   # n itself is passed over
    b_id, bias = i32([n - 2, -2 ** 31, 4096, -1, n - 2]), f32([9, 100, 2, 100, 4])
    rule = K.LogitRule(2.0, 0.25, 0.5, -1)
    K.hip.krh_logit_rules(xb.ptr, n, xb.ptr, n, n, 1, dev.put(np.frombuffer(bytes(rule), np.uint8)).ptr, dev.put(seen).ptr, 9,
                          dev.put(i32([9])).ptr, dev.put(b_id).ptr, dev.put(bias).ptr, 5, dev.put(i32([5])).ptr, None, 0)
    ok()
    for i in at:
        v = np.empty(1, np.float32)
        K.check(K.hip.krh_copy_d2h(v.ctypes.data, xb.ptr + 4 * i, 4))
        c = int((seen == i).sum())
        want = (i % 97 + 1) / (2 if c else 1) - 0.5 * c - (0.25 if c else 0) + {n - 2: 4, 4096: 2}.get(i, 0)
        assert v[0] == want, i


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("cap", [2.0 ** 126, 2.0 ** -126])
def test_attention_extreme_soft_caps(dev, kv_type, cap):  # noqa: F811
    """a cap far above the scores leaves them (to a step of 2^-149 times the cap), one far below gives every row the same weight"""
    rng = np.random.default_rng(4)
    p = Pool(dev, rng, kv_type, [50, 7], 16, 2, 64).put()
    q = f32(rng.standard_normal((2, 4, 64)))
    o, _ = attend(dev, p, [50, 7], q, 4, False, scale=0.125, cap=cap)
    for i, n in enumerate((50, 7)):
        k, v = p.rows("k", i, n), p.rows("v", i, n)
        for h in range(4):
            w, _, bound, _ = attention(q[i, h].astype(np.float64) * (cap > 1), k[:, h // 2], v[:, h // 2], 0.125, 0, 0)
            more = 2 * 2.0 ** -149 * cap * np.abs(v[:, h // 2]).max() if cap > 1 else 0
            assert (np.abs(o[i, h] - w) <= bound + more + 8 * U * np.abs(v[:, h // 2]).max()).all(), (i, h)
