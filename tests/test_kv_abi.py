"""Host-side checks of the key/value cache entry points: bad arguments are refused before any launch."""
import ctypes

import pytest

import qwen35_amd
from qwen35_amd._lib import QhipKvBatch, QhipKvCache

INVALID, DECLINE = 1, -1


@pytest.fixture(scope="module")
def lib():
    return qwen35_amd.load()


P = 0x1000  # never dereferenced: the checks fail first


def cache(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, num_blocks=4, block_size=16, kv_heads=2, head_dim=64)
    return ctypes.byref(QhipKvCache(**{**f, **kw}))


def batch(**kw):
    f = dict(offsets=P, kv_lens=P, table=P, nseq=2, tokens=2, max_new=1, max_kv=100, table_width=8)
    return ctypes.byref(QhipKvBatch(**{**f, **kw}))


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4),
              dict(k_scale=P + 2), dict(num_blocks=0), dict(num_blocks=-1), dict(block_size=0), dict(block_size=8),
              dict(block_size=48), dict(block_size=512), dict(kv_heads=0), dict(kv_heads=70000), dict(head_dim=0),
              dict(num_blocks=2 ** 27)]


def test_tables(lib):
    ok = [P, P, 2, P, 3, P, 16, P, 4, 5, P, P, P, P, P, None]
    for at, bad in [(0, None), (1, None), (2, -1), (3, None), (4, -1), (6, 0), (6, 8), (6, 24), (6, 512), (7, None), (8, -1),
                    (9, -1), (10, None), (11, None), (12, None), (14, None)]:
        args = list(ok)
        args[at] = bad
        assert lib.qhip_launch_kv_tables(*args) == INVALID, (at, bad)


def test_tables_in_place_are_refused(lib):
    at = [P + 0x100 * i for i in range(9)]  # cached, new, free, taken, table, offsets, kv_lens, slots, taken_out
    for inp, out in [(0, 5), (0, 6), (1, 6), (2, 8), (3, 8), (3, 5)]:
        x = list(at)
        x[out] = x[inp]
        assert lib.qhip_launch_kv_tables(x[0], x[1], 2, x[2], 3, x[3], 16, x[4], 4, 5, x[5], x[6], x[7], None, x[8],
                                         None) == INVALID, (inp, out)


def test_append(lib):
    def call(c, type=0, k=P, v=P, slots=P, tokens=3):
        return lib.qhip_launch_kv_append(c, type, k, 128, 64, v, 128, 64, slots, tokens, None)

    assert call(None) == INVALID
    for bad in BAD_CACHES:
        assert call(cache(**bad)) == INVALID, bad
    for bad in (dict(type=8), dict(type=2), dict(k=None), dict(v=None), dict(slots=None), dict(tokens=-1), dict(k=P + 2),
                dict(type=30, v=P + 1)):
        assert call(cache(), **bad) == INVALID, bad
    assert call(cache(head_dim=80)) == DECLINE
    assert call(cache(), tokens=0, k=None, v=None, slots=None) == 0


def test_read(lib):
    def call(c, blocks=P, n=1, type=0, k=P, v=P):
        return lib.qhip_launch_kv_read(c, blocks, n, type, k, v, None)

    for bad in BAD_CACHES:
        assert call(cache(**bad)) == INVALID, bad
    for bad in (dict(blocks=None), dict(n=-1), dict(type=12), dict(k=P + 8), dict(v=P + 2)):
        assert call(cache(), **bad) == INVALID, bad
    assert call(cache(head_dim=192)) == DECLINE
    assert call(cache(), n=0) == 0 and call(cache(), k=None, v=None) == 0


def test_attention(lib):
    def call(c, b, type=0, q=P, heads=4, causal=1, window=0, out=P, work=None, nwork=0):
        return lib.qhip_launch_kv_attention(c, b, type, q, 256, 64, heads, 0.125, causal, window, out, 256, 64, None, work,
                                            nwork, None)

    for bad in BAD_CACHES:
        assert call(cache(**bad), batch()) == INVALID, bad
    for bad in (dict(offsets=None), dict(kv_lens=None), dict(table=None), dict(nseq=-1), dict(tokens=-1), dict(max_new=-1),
                dict(max_kv=-1), dict(table_width=-1)):
        assert call(cache(), batch(**bad)) == INVALID, bad
    assert call(cache(), None) == INVALID
    for bad in (dict(type=8), dict(q=None), dict(q=P + 2), dict(out=None), dict(out=P + 1), dict(heads=0), dict(heads=3),
                dict(heads=70000), dict(causal=2), dict(window=-1), dict(causal=0, window=3), dict(work=P + 4, nwork=64),
                dict(nwork=-1)):
        assert call(cache(), batch(), **bad) == INVALID, bad
    assert call(cache(head_dim=96), batch()) == DECLINE
    assert call(cache(), batch(tokens=0)) == 0 and call(cache(), batch(nseq=0)) == 0


def test_attention_workspace(lib):
    assert lib.qhip_kv_attention_work_bytes(cache(block_size=8), batch(), 4) == -1
    assert lib.qhip_kv_attention_work_bytes(cache(), batch(tokens=-1), 4) == -1
    assert lib.qhip_kv_attention_work_bytes(cache(), batch(), 3) == -1
    assert lib.qhip_kv_attention_work_bytes(cache(), batch(), 4) >= 0


def test_attention_workspace_covers_the_types_and_stays_moderate(lib):
    c = cache(kv_heads=4, head_dim=128, block_size=64, num_blocks=100)
    for nseq, tokens, new, kv in [(1, 1, 1, 131072), (64, 64, 1, 8192), (13, 65, 5, 4000), (12, 1032, 1021, 6021)]:
        n = lib.qhip_kv_attention_work_bytes(c, batch(nseq=nseq, tokens=tokens, max_new=new, max_kv=kv), 16)
        assert 32768 < n <= 64 << 20, (nseq, tokens, n)
    # enough row tiles as they are, nothing to cut, no rows
    assert lib.qhip_kv_attention_work_bytes(c, batch(nseq=2000, tokens=2000, max_new=1, max_kv=9000), 16) == 0
    assert lib.qhip_kv_attention_work_bytes(c, batch(nseq=1, tokens=1, max_new=1, max_kv=32), 16) == 0
    assert lib.qhip_kv_attention_work_bytes(c, batch(nseq=1, tokens=1, max_new=0, max_kv=9000), 16) == 0
    assert lib.qhip_kv_attention_work_bytes(cache(kv_heads=1), batch(), 513) == -1
