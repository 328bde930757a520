"""Counts that the kernels' 32-bit indexes could not pass the end of are refused on the host."""
import ctypes

import pytest

import qwen35_amd
from qwen35_amd._lib import QhipKvBatch, QhipKvCache

INVALID = 1
MOST = 2 ** 31 - 1 - 1024  # a workgroup's tokens, or a block's, may be counted past the last


@pytest.fixture(scope="module")
def lib():
    return qwen35_amd.load()


def cache():
    return ctypes.byref(QhipKvCache(0x1000, 0x1000, 0x1000, 0x1000, 4, 16, 1, 64))


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 257, 2 ** 31 - 1])
def test_tables(lib, n):
    """Addresses 2^40 apart that nothing dereferences."""
    a = [(i + 1) << 40 for i in range(10)]
    assert lib.qhip_launch_kv_tables(a[0], a[1], 2, a[2], 3, a[3], 16, a[4], 4, n, a[5], a[6], a[7], a[8], a[9], None) == INVALID
    assert lib.qhip_launch_kv_tables(a[0], a[1], n, a[2], 3, a[3], 16, a[4], 4, 5, a[5], a[6], a[7], a[8], a[9], None) == INVALID


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 255, 2 ** 31 - 1])
def test_append(lib, n):
    assert lib.qhip_launch_kv_append(cache(), 0, 0x1000, 0, 0, 0x1000, 0, 0, 0x1000, n, None) == INVALID


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 64, 2 ** 31 - 1])
def test_attention(lib, n):
    b = ctypes.byref(QhipKvBatch(0x1000, 0x1000, 0x1000, n, 1, 1, 10, 1))
    assert lib.qhip_launch_kv_attention(cache(), b, 0, 0x1000, 64, 64, 1, 0.125, 1, 0, 0x1000, 64, 64, None, None, 0,
                                        None) == INVALID
    assert lib.qhip_kv_attention_work_bytes(cache(), b, 1) == -1
