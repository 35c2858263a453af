"""What a batch's calls decide without a device, at the edges of what they accept."""
import ctypes as C

import pytest

import krafla as K
from test_batch_ops import pages


@pytest.mark.parametrize("glu", [0, 1])
def test_no_tiles_for_refused_sizes(glu):
    form = K.hip.krh_matmul_i8_form
    for size in ((64, 64, 65536), (64, 64, 2 ** 31 - 1), (2 ** 31 - 1, 64, 1), (2 ** 31 - 1024, 64, 1), (64, 131072, 1)):
        assert form(*size, glu) == -1, size
    for size in ((64, 64, 65535), (2 ** 31 - 1025, 64, 1), (64, 131071, 1)):
        assert form(*size, glu) >= 0, size


def test_no_form_for_a_negative_window():
    kv = C.byref(pages(head_dim=128, n_kv_heads=8))
    assert K.hip.krh_paged_attention_shared_form(kv, 64, 32, 40000, 1, 32000, 0) == 1
    assert K.hip.krh_paged_attention_shared_form(kv, 64, 32, 40000, 1, 32000, -1) == -1


B8 = dict(head_dim=128, n_kv_heads=8)   # the 8B shape's, with 32 heads


@pytest.mark.parametrize("kw,nh,n,groups,shared,window,form", [
    # halves: up to 16 groups of 1024 rows, or any that leave none alone where the rows are many
    (B8, 32, 64, 1, 1024, 0, 1), (B8, 32, 64, 8, 1024, 0, 1), (B8, 32, 64, 16, 1024, 0, 1), (B8, 32, 64, 32, 1024, 0, 0),
    (B8, 32, 64, 63, 1024, 0, 0), (B8, 32, 64, 32, 8192, 0, 1), (B8, 32, 64, 63, 8192, 0, 0), (B8, 32, 64, 64, 8192, 0, 0),
    # floats and 8 bits, whose column tiles take longer
    (dict(B8, kv_type=K.ML_F32), 32, 64, 1, 2048, 0, 1), (dict(B8, kv_type=K.ML_F32), 32, 64, 16, 2048, 0, 0),
    (dict(B8, kv_type=K.ML_F32), 32, 64, 32, 8192, 0, 0),
    (dict(n_kv_heads=8, kv_type=K.ML_Q8_0, kd=4096, vd=4096), 32, 64, 8, 2048, 0, 1),
    (dict(n_kv_heads=8, kv_type=K.ML_Q8_0, kd=4096, vd=4096), 32, 64, 32, 8192, 0, 0),
    (dict(n_kv_heads=4, head_dim=256, kv_type=K.ML_F32), 8, 64, 1, 2048, 0, 1),
    (dict(n_kv_heads=4, head_dim=256, kv_type=K.ML_F32), 8, 64, 8, 2048, 0, 0),
    # windows: a group's first rows are looked for one group after another
    (B8, 32, 64, 1, 4096, 2048, 1), (B8, 32, 128, 64, 8192, 256, 0)])
def test_groups_decide_with_the_rows(kw, nh, n, groups, shared, window, form):
    """one answer whatever the own rows may be"""
    for more in (1, 150, 100000):
        assert K.hip.krh_paged_attention_shared_form(C.byref(pages(**kw)), n, nh, shared + more, groups, shared, window) == form
