"""Host-side checks of the norms' sizes: what the kernels' indexes do not hold is refused before any launch."""
import ctypes

import pytest

import qwen35_amd
from qwen35_amd._lib import QhipRows

INVALID = 1
X, OUT = 1 << 40, 1 << 41  # never dereferenced: there is nothing to do, or the checks fail first


def norm(dim, heads=1, tokens=0, stride=0):
    rows = [ctypes.byref(QhipRows(at, stride, stride)) for at in (X, OUT)]
    return qwen35_amd.load().qhip_launch_rms_norm(30, rows[0], None, None, None, 1e-6, rows[1], 0, None, tokens, heads, dim, None)


@pytest.mark.parametrize("tokens", [0, 1])
def test_rows_whose_end_an_index_would_step_past(tokens):
    """A row is walked 8192 values at a time: the step behind its last values has to fit an int."""
    most = 2 ** 31 - 1 - 8192
    for dim in (most + 1, most + 4096, 2 ** 31 - 1):
        assert norm(dim, tokens=tokens) == INVALID, dim
    assert norm(most) == 0
    assert norm(512, heads=2 ** 22 - 1) == 0  # heads whose product is as large are no long rows
