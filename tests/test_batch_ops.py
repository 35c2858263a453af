"""8-bit products, the norms between blocks and the attention over shared rows
without a device: what the calls refuse."""
import ctypes as C

import pytest

import krafla as K

PTR = 0x100000   # an address that a refused call never reads


def mat(**kw):
    return K.KrhMat8(**dict(dict(q=PTR, d=PTR, ld=64, rows=24, cols=50), **kw))


I8 = dict(Y=PTR, ldy=24, W=mat(), xq=PTR, ldx=64, xd=PTR, bias=PTR, T=3, accumulate=0)
GLU = dict(H=PTR, ldh=24, w1=mat(), w3=mat(), xq=PTR, ldx=64, xd=PTR, T=3)
NORM = dict(xo=PTR, ldxo=64, x=PTR, ldx=64, y=PTR + 4096, ldy=64, post=PTR, gate=PTR, ldg=0, alpha=1.0, pre=PTR, eps=1e-6,
            z=PTR + 8192, ldz=64, q=PTR, ldq=64, d=PTR, n=64, rows=3)
DEQ = dict(x=PTR, ldx=64, q=PTR, ldq=64, d=PTR, ldd=1, n=64, rows=3)

BAD_MATS = [dict(q=None), dict(d=None), dict(q=PTR + 8), dict(ld=48), dict(ld=56), dict(rows=0), dict(rows=-1),
            dict(rows=2**31 - 1), dict(ld=2**23 + 16), dict(cols=0), dict(cols=-5), dict(cols=65), dict(cols=1 << 17, ld=1 << 17)]

CASES = [("krh_matmul_i8", I8, kw) for kw in
         [dict(Y=None), dict(xq=None), dict(xd=None), dict(W=None), dict(T=-1), dict(T=70000), dict(ldy=23), dict(ldx=48),
          dict(ldx=72), dict(ldx=2**23 + 16), dict(xq=PTR + 4)] + [dict(W=mat(**b)) for b in BAD_MATS]]
CASES += [("krh_matmul_i8_swiglu", GLU, kw) for kw in
          [dict(H=None), dict(xq=None), dict(xd=None), dict(w1=None), dict(w3=None), dict(T=-1), dict(T=70000), dict(ldh=23),
           dict(ldx=48), dict(ldx=72), dict(ldx=2**23 + 16), dict(xq=PTR + 8), dict(w3=mat(rows=25)), dict(w1=mat(cols=49))] +
          [dict(w1=mat(**b)) for b in BAD_MATS] + [dict(w3=mat(**b)) for b in BAD_MATS]]
CASES += [("krh_block_norm", NORM, kw) for kw in
          [dict(x=None), dict(xo=None, z=None, q=None, d=None), dict(pre=None), dict(y=None), dict(q=None), dict(d=None),
           dict(n=0), dict(n=16385), dict(rows=-1), dict(rows=70000), dict(ldx=63), dict(ldxo=63, xo=PTR + 64), dict(ldy=60),
           dict(ldg=32), dict(ldz=8), dict(ldq=63), dict(ldxo=68), dict(z=PTR, ldz=68), dict(z=PTR + 4096, ldz=68),
           dict(xo=PTR + 4096, ldxo=72)]]
CASES += [("krh_dequantize_row_rows", DEQ, kw) for kw in
          [dict(x=None), dict(q=None), dict(d=None), dict(n=-1), dict(rows=-1), dict(rows=70000), dict(ldx=63)]]


def call(name, args, **kw):
    a = dict(args, **kw)
    K.hip.krh_clear_error()
    getattr(K.hip, name)(*[C.byref(v) if isinstance(v, C.Structure) else v for v in a.values()])
    st = K.hip.krh_status()
    K.hip.krh_clear_error()
    return st


@pytest.mark.parametrize("name,base,kw", CASES, ids=["%s-%d" % (n[4:], i) for i, (n, _, _) in enumerate(CASES)])
def test_refused(name, base, kw):
    assert call(name, base, **kw) == K.ML_E_SHAPE


def test_nothing_to_do():
    assert call("krh_matmul_i8", I8, T=0) == K.ML_OK
    assert call("krh_matmul_i8_swiglu", GLU, T=0) == K.ML_OK
    assert call("krh_block_norm", NORM, rows=0) == K.ML_OK
    assert call("krh_dequantize_row_rows", DEQ, rows=0) == K.ML_OK
    assert call("krh_dequantize_row_rows", DEQ, n=0) == K.ML_OK


def test_before_init():
    """without a device a good call is refused, not launched"""
    if K.hip.krh_device_cus() > 0:
        pytest.skip("the device is open")
    for name, base, more in (("krh_matmul_i8", I8, [dict(bias=None), dict(accumulate=1)]), ("krh_matmul_i8_swiglu", GLU, []),
                             ("krh_block_norm", NORM, [dict(y=None, post=None, gate=None), dict(q=None, d=None),
                                                       dict(pre=None, z=None, q=None, d=None), dict(xo=None), dict(rows=1, ldxo=68),
                                                       dict(ldg=64)]),
                             ("krh_dequantize_row_rows", DEQ, [dict(rows=1, ldx=0)])):
        for kw in [{}] + more:
            assert call(name, base, **kw) == K.ML_E_ISA, (name, kw)


# ---- attention over shared rows ----

def pages(**kw):
    f = dict(k=PTR, v=PTR, kd=None, vd=None, kv_type=K.ML_F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    return K.KrhPages(**dict(f, **kw))


SHARE = dict(o=PTR, kv=pages(), table=PTR, table_ld=4, len=PTR, n_seq=20, group=PTR, shared=PTR, n_groups=2, max_shared=48, q=PTR,
             n_heads=4, max_len=64, window=0, scale=1.0, softcap=0.0, ws=PTR)


@pytest.mark.parametrize("kw", [dict(o=None), dict(table=None), dict(len=None), dict(group=None), dict(shared=None), dict(q=None),
                                dict(ws=None), dict(o=PTR + 8), dict(q=PTR + 4), dict(ws=PTR + 8), dict(n_seq=-1),
                                dict(n_seq=70000), dict(n_groups=-1), dict(n_groups=65), dict(max_shared=-1),
                                dict(max_shared=65), dict(n_heads=0), dict(n_heads=5), dict(n_heads=34), dict(max_len=0),
                                dict(max_len=2**30), dict(n_seq=60000, max_len=2**29), dict(table_ld=0), dict(window=-1),
                                dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=1e-40),
                                dict(kv=None), dict(kv=pages(k=None)), dict(kv=pages(kv_type=K.ML_Q8_0)),
                                dict(kv=pages(page_size=24)), dict(kv=pages(head_dim=12))],
                         ids=lambda kw: "-".join(kw))
def test_shared_attention_refused(kw):
    assert call("krh_paged_attention_shared", SHARE, **kw) == K.ML_E_SHAPE


def test_shared_attention_nothing_to_do():
    assert call("krh_paged_attention_shared", SHARE, n_seq=0) == K.ML_OK
    if K.hip.krh_device_cus() == 0:
        for kw in ({}, dict(n_groups=0, group=None, shared=None), dict(max_shared=0), dict(n_groups=64), dict(max_shared=64)):
            assert call("krh_paged_attention_shared", SHARE, **kw) == K.ML_E_ISA, kw


def test_shared_attention_workspaces():
    ws = K.hip.krh_paged_attention_shared_ws
    kv = C.byref(pages())
    assert ws(kv, 20, 4, 64, 2, 48) >= K.hip.krh_paged_attention_ws(kv, 20, 4, 64, 0) > 0
    assert ws(kv, 20, 4, 64, 0, 0) == K.hip.krh_paged_attention_ws(kv, 20, 4, 64, 0)
    for bad in ((kv, 0, 4, 64, 2, 48), (kv, 20, 5, 64, 2, 48), (kv, 20, 4, 64, 65, 48), (kv, 20, 4, 64, 2, 65),
                (None, 20, 4, 64, 2, 48)):
        assert ws(*bad) == 0


@pytest.mark.parametrize("kw,nh", [(dict(), 4), (dict(head_dim=128, n_kv_heads=8), 32), (dict(kv_type=K.ML_F32, head_dim=256), 4),
                                   (dict(kv_type=K.ML_Q8_0, kd=PTR, vd=PTR, n_kv_heads=1), 7)])
def test_shared_attention_workspaces_grow(kw, nh):
    """a workspace for larger sizes serves smaller ones, whichever of them pass over shared rows once"""
    kv = C.byref(pages(**kw))
    sizes = [(n, most, g, shared) for n in (1, 2, 7, 16, 31, 32, 33, 64, 65, 200) for most in (64, 4096, 40000) for g in (1, 3, 64)
             for shared in (1, 48, 64, 1000, 4000, 39000) if shared <= most]
    ws = {s: K.hip.krh_paged_attention_shared_ws(kv, s[0], nh, *s[1:]) for s in sizes}
    assert len({K.hip.krh_paged_attention_shared_form(kv, s[0], nh, *s[1:], 0) for s in sizes}) == 2
    for a in sizes:
        assert ws[a] > 0
        for b in sizes:
            if all(x <= y for x, y in zip(a, b)):
                assert ws[a] <= ws[b], (a, b)


def test_forms():
    """which tiles or passes a call takes, and that sizes without one have none"""
    i8 = K.hip.krh_matmul_i8_form
    for size in ((0, 64, 1), (64, 0, 1), (64, 1 << 17, 1), (64, 64, 0), (-1, 64, 1)):
        assert i8(*size, 0) == i8(*size, 1) == -1
    seen = {(glu, i8(rows, cols, T, glu)) for glu in (0, 1) for rows in (16, 300, 4096, 14336) for cols in (64, 4096, 14336)
            for T in (1, 8, 9, 40, 64, 128, 300, 2047, 8192)}
    assert {f for _, f in seen} <= set(range(9)) and len(seen) >= 8
    form = K.hip.krh_paged_attention_shared_form
    kv = C.byref(pages(head_dim=128, n_kv_heads=8))
    for bad in ((kv, 0, 32, 4096, 1, 48, 0), (kv, 20, 31, 4096, 1, 48, 0), (kv, 20, 32, 4096, 65, 48, 0),
                (kv, 20, 32, 4096, 1, 4097, 0), (None, 20, 32, 4096, 1, 48, 0)):
        assert form(*bad) == -1
    assert form(kv, 64, 32, 40000, 1, 32000, 0) == 1
    # nothing shared, few rows, or a window that ends behind them
    for few in ((kv, 64, 32, 40000, 0, 0, 0), (kv, 64, 32, 40000, 1, 0, 0), (kv, 1, 32, 64, 1, 16, 0), (kv, 64, 32, 40000, 1, 32000, 16)):
        assert form(*few) == 0
