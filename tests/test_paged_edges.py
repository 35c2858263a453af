"""The paged cache's operators and the logit rules without a device, at the
edges of what their calls allow: the bounds of lists and rows, and refusals."""
import ctypes as C
import os
import subprocess

import pytest

import krafla as K
from test_paged import ATT, EVICT, HERE, PTR, QKV, ROOT, call, pages


def host_check(tmp_path, name, trials):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "isa-lm_amd", "csrc"),
                    os.path.join(HERE, "csrc", name + ".cpp"), "-o", exe], check=True)
    r = subprocess.run([exe, str(trials)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), (r.returncode, r.stdout + r.stderr)


def refused(name, args, kv):
    """what a refused call says"""
    K.hip.krh_clear_error()
    a = dict(args)
    if "kv" in a:
        a["kv"] = C.byref(kv)
    getattr(K.hip, name)(*a.values())
    said = K.hip.krh_last_error()
    K.hip.krh_clear_error()
    return said


def test_lists_are_read_to_their_counts(tmp_path):
    host_check(tmp_path, "list_bounds", 1000)


def test_negative_rows_are_out_of_range(tmp_path):
    host_check(tmp_path, "row_bounds", 100000)


@pytest.mark.parametrize("ldqo", [260, 512])
def test_queries_in_place_have_one_stride(ldqo):
    """tokens pass in no order, so one's output would lie on another's query"""
    assert call("krh_paged_qkv", dict(QKV, qo=PTR, q=PTR, ldq=256, ldqo=ldqo), pages()) == K.ML_E_SHAPE
    assert b"in place" in refused("krh_paged_qkv", dict(QKV, qo=PTR, q=PTR, ldq=256, ldqo=ldqo), pages())
    # apart, or without queries, the strides are the caller's
    if K.hip.krh_device_cus() == 0:
        assert call("krh_paged_qkv", dict(QKV, qo=PTR + 65536, ldqo=ldqo), pages()) == K.ML_E_ISA
        assert call("krh_paged_qkv", dict(QKV, n_heads=0, q_norm=None, ldqo=ldqo), pages()) == K.ML_E_ISA


@pytest.mark.parametrize("cap", [float("inf"), 3e38, 1e-40, 1e-45])
def test_soft_caps_without_a_reciprocal_refused(cap):
    """Infinity times a score's tanh, 0 there, is no number, and the smallest floats' reciprocals are infinite. 3e38 times
    log2 e, by which powers are taken, is infinite too."""
    assert call("krh_paged_attention", dict(ATT, softcap=cap), pages()) == K.ML_E_SHAPE
    if K.hip.krh_device_cus() == 0:
        assert call("krh_paged_attention", dict(ATT, softcap=8e37), pages()) == K.ML_E_ISA
        assert call("krh_paged_attention", dict(ATT, softcap=1.2e-38), pages()) == K.ML_E_ISA


@pytest.mark.parametrize("keep", [2**29 + 1, 2**31 - 1])
def test_more_rows_kept_than_a_sequence_has_refused(keep):
    """the masses' zeros go as far as `keep`, and steps past an int's last value would come out below the row"""
    assert call("krh_paged_evict", dict(EVICT, keep=keep, out_ld=2**31), pages()) == K.ML_E_SHAPE
    assert K.hip.krh_paged_evict_ws(1, 2, keep) == 0
    if K.hip.krh_device_cus() == 0:
        assert call("krh_paged_evict", dict(EVICT, keep=2**29, out_table_ld=4, out_ld=2**31), pages()) == K.ML_E_ISA
    assert K.hip.krh_paged_evict_ws(1, 2, 2**29) == 4 * (4 * 2**29 + 1)
