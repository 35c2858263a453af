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
