"""The paged cache's operators without a device: the page lookups, which keep
every access in bounds whatever the tables hold, and what the calls refuse."""
import ctypes as C
import os
import subprocess

import pytest

import krafla as K

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
PTR = 0x100000   # an address that a refused call never reads


def test_lookups_stay_in_bounds(tmp_path):
    exe = str(tmp_path / "page_bounds")
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "isa-lm_amd", "csrc"),
                    os.path.join(HERE, "csrc", "page_bounds.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe, "300000"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr


def pages(**kw):
    f = dict(k=PTR, v=PTR, kd=None, vd=None, kv_type=K.ML_F16, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
    f.update(kw)
    return K.KrhPages(**f)


BAD_PAGES = [dict(k=None), dict(v=None), dict(k=PTR + 8), dict(v=PTR + 2), dict(kv_type=K.ML_Q4_0), dict(kv_type=9),
             dict(kv_type=K.ML_Q8_0), dict(kv_type=K.ML_Q8_0, kd=PTR), dict(n_pages=0), dict(n_pages=-1),
             dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(page_size=0), dict(n_kv_heads=0),
             dict(n_kv_heads=70000), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264)]

QKV = dict(qo=PTR, ldqo=256, kv=None, table=PTR, table_ld=4, n_seq=2, q=PTR, ldq=256, k=PTR, ldk=128, v=PTR, ldv=128,
           ntok=3, n_heads=4, seq=PTR, row=PTR, pos=PTR, q_norm=PTR, k_norm=PTR, eps=1e-6, cos=PTR, sin=PTR, n_pos=10)
LOAD = dict(k=PTR, ldk=128, v=PTR, ldv=128, kv=None, table=PTR, table_ld=4, n_seq=2, n=3, seq=PTR, row=PTR)
ATT = dict(o=PTR, kv=None, table=PTR, table_ld=4, len=PTR, n_seq=2, q=PTR, n_heads=4, max_len=64, window=0, scale=1.0,
           softcap=0.0, mass=PTR, mass_ld=64, ws=PTR)
EVICT = dict(kv=None, table=PTR, table_ld=4, len=PTR, mass=PTR, mass_ld=64, n_seq=2, max_len=64, keep=32, recent=8,
             out_table=PTR + 64, out_table_ld=2, out_len=PTR, out_mass=PTR + 4096, out_ld=32, ws=PTR)
RULES = dict(out=PTR, ldo=100, logits=PTR, ld=100, n=100, rows=2, rule=PTR, seen=PTR, seen_ld=8, n_seen=PTR,
             bias_id=PTR, bias=PTR, bias_ld=8, n_bias=PTR, masks=PTR, n_masks=1)

CASES = [("krh_paged_qkv", QKV, kw) for kw in
         [dict(qo=None), dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(seq=None), dict(row=None),
          dict(pos=None), dict(cos=None), dict(sin=None), dict(q_norm=None), dict(k_norm=None), dict(ntok=-1),
          dict(n_heads=-1), dict(n_seq=0), dict(table_ld=0), dict(n_pos=0), dict(ldq=252), dict(ldq=258),
          dict(ldqo=255), dict(ldk=124), dict(ldk=130), dict(ldv=64), dict(k=PTR + 4), dict(q=PTR + 8),
          dict(cos=PTR + 8), dict(q_norm=PTR + 4), dict(ntok=2**31 - 1)]]
CASES += [("krh_paged_load", LOAD, kw) for kw in
          [dict(k=None), dict(v=None), dict(table=None), dict(seq=None), dict(row=None), dict(n=-1), dict(n_seq=0),
           dict(table_ld=0), dict(ldk=127), dict(ldv=120), dict(v=PTR + 8)]]
CASES += [("krh_paged_attention", ATT, kw) for kw in
          [dict(o=None), dict(q=None), dict(table=None), dict(len=None), dict(ws=None), dict(q=PTR + 4),
           dict(ws=PTR + 8), dict(n_seq=-1), dict(n_seq=70000), dict(n_heads=0), dict(n_heads=5), dict(n_heads=34),
           dict(max_len=0), dict(window=-1), dict(softcap=-1.0), dict(softcap=float("nan")), dict(mass_ld=63),
           dict(table_ld=0), dict(max_len=2**30), dict(n_seq=60000, max_len=2**29)]]
CASES += [("krh_paged_evict", EVICT, kw) for kw in
          [dict(table=None), dict(len=None), dict(mass=None), dict(out_table=None), dict(out_len=None),
           dict(out_mass=None), dict(ws=None), dict(out_table=PTR), dict(n_seq=-1), dict(n_seq=70000), dict(max_len=0),
           dict(keep=0), dict(recent=-1), dict(recent=33), dict(mass_ld=63), dict(out_ld=31), dict(out_mass=PTR),
           dict(table_ld=0), dict(out_table_ld=1), dict(max_len=2**30, mass_ld=2**30)]]
CASES += [("krh_logit_rules", RULES, kw) for kw in
          [dict(out=None), dict(logits=None), dict(rule=None), dict(n_seen=None), dict(n_bias=None), dict(bias=None),
           dict(masks=None), dict(n=0), dict(rows=-1), dict(rows=70000), dict(n_masks=-1), dict(ldo=99, out=PTR + 4),
           dict(ld=99), dict(ldo=101), dict(seen_ld=2**31)]]


def call(name, args, kv):
    a = dict(args)
    if "kv" in a:
        a["kv"] = C.byref(kv) if kv is not None else None
    K.hip.krh_clear_error()
    getattr(K.hip, name)(*a.values())
    st = K.hip.krh_status()
    K.hip.krh_clear_error()
    return st


@pytest.mark.parametrize("name,base,kw", CASES, ids=["%s-%s" % (n[4:], kw) for n, _, kw in CASES])
def test_refused(name, base, kw):
    assert call(name, dict(base, **kw), pages()) == K.ML_E_SHAPE


@pytest.mark.parametrize("kw", BAD_PAGES, ids=str)
def test_bad_pages_refused(kw):
    for name, base in (("krh_paged_qkv", QKV), ("krh_paged_load", LOAD), ("krh_paged_attention", ATT),
                       ("krh_paged_evict", EVICT)):
        assert call(name, base, pages(**kw)) == K.ML_E_SHAPE, name
        assert call(name, base, None) == K.ML_E_SHAPE, name
    assert K.hip.krh_paged_attention_ws(C.byref(pages(**kw)), 1, 4, 100, 0) == 0


def test_nothing_to_do():
    """no tokens, rows or sequences: no error, no launch"""
    kv = pages()
    assert call("krh_paged_qkv", dict(QKV, ntok=0), kv) == K.ML_OK
    assert call("krh_paged_load", dict(LOAD, n=0), kv) == K.ML_OK
    assert call("krh_paged_attention", dict(ATT, n_seq=0), kv) == K.ML_OK
    assert call("krh_paged_evict", dict(EVICT, n_seq=0), kv) == K.ML_OK
    assert call("krh_logit_rules", dict(RULES, rows=0), kv) == K.ML_OK


def test_workspaces():
    assert K.hip.krh_paged_attention_ws(C.byref(pages()), 3, 4, 100, 1) > 0
    assert K.hip.krh_paged_attention_ws(C.byref(pages()), 3, 5, 100, 1) == 0
    assert K.hip.krh_paged_evict_ws(3, 2, 7) >= 4 * 3 * 2 * 7
    assert K.hip.krh_paged_evict_ws(3, 2, 0) == 0


def test_before_init():
    """without a device a good call is refused, not launched"""
    if K.hip.krh_device_cus() > 0:
        pytest.skip("the device is open")
    kv = pages()
    for name, base in (("krh_paged_qkv", QKV), ("krh_paged_load", LOAD), ("krh_paged_attention", ATT),
                       ("krh_paged_evict", EVICT), ("krh_logit_rules", RULES)):
        assert call(name, base, kv) == K.ML_E_ISA, name
