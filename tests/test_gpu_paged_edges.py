"""The paged cache's operators and the logit rules on the device at the edges
of what their calls allow. Needs a gfx950 device."""
import numpy as np
import pytest

import krafla as K
from test_gpu_kernels import bits, f32, ok
from test_gpu_paged import TYPES, Pool, U, dev, device, i32, rules, tables  # noqa: F401  (dev, device: fixtures)

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
