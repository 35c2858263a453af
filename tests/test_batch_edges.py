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
