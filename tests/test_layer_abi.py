"""Host-side checks of norms, rotary positions and linear attention: bad arguments are refused before any launch."""
import ctypes

import pytest

import qwen35_amd
from qwen35_amd._lib import QhipLinearBatch, QhipRows

INVALID, DECLINE = 1, -1
P = 0x100000  # never dereferenced: the checks fail first, or there is nothing to do


@pytest.fixture(scope="module")
def lib():
    return qwen35_amd.load()


def rows(at=P, token=512, head=128):
    return ctypes.byref(QhipRows(at, token, head))


FAR = [P + (i << 24) for i in range(12)]


def test_norm(lib):
    def call(type=0, x=rows(FAR[0]), residual=rows(FAR[1]), gate=rows(FAR[2]), weight=FAR[3], eps=1e-6, out=rows(FAR[4]), ttype=8,
             xq=FAR[5], tokens=3, heads=4, dim=128):
        return lib.qhip_launch_rms_norm(type, x, residual, gate, weight, eps, out, ttype, xq, tokens, heads, dim, None)

    assert call(tokens=0) == 0
    for bad in (dict(type=2), dict(type=8), dict(x=None), dict(x=rows(None)), dict(x=rows(FAR[0] + 2)), dict(x=rows(FAR[0], -512)),
                dict(x=rows(FAR[0], 512, -1)), dict(x=rows(FAR[0], 2 ** 31)), dict(residual=rows(FAR[1] + 1)), dict(gate=rows(FAR[2] + 2)),
                dict(weight=FAR[3] + 2), dict(eps=-1.0), dict(eps=float("nan")), dict(out=None, xq=None), dict(out=rows(FAR[4], 0)),
                dict(out=rows(FAR[4], 512, 64)), dict(residual=rows(FAR[1], 256)), dict(ttype=6), dict(ttype=99), dict(xq=FAR[5] + 1),
                dict(ttype=12, xq=FAR[5] + 2), dict(tokens=-1), dict(heads=0), dict(dim=0), dict(heads=3, dim=8), dict(ttype=12, heads=3),
                dict(tokens=2 ** 30, heads=4), dict(heads=2 ** 20, dim=2 ** 12),
                # overlaps: everything written against everything else
                dict(residual=rows(FAR[0])), dict(residual=rows(FAR[2])), dict(residual=rows(FAR[4])), dict(out=rows(FAR[0] + 4)),
                dict(out=rows(FAR[2] + 4096)), dict(out=rows(FAR[3])), dict(xq=FAR[0] + 8), dict(xq=FAR[3]), dict(xq=FAR[4]), dict(weight=FAR[1])):
        assert call(**bad) == INVALID, bad
    assert call(ttype=12, heads=8, dim=96) == DECLINE


def test_rope_steps(lib):
    steps, gain = (ctypes.c_ulonglong * 64)(), ctypes.c_float()

    def call(rot=64, base=1e4, scaling=0, factor=2.0, original=4096, fast=32.0, slow=1.0, steps=steps, gain=ctypes.byref(gain)):
        return lib.qhip_rope_steps(rot, base, scaling, factor, original, fast, slow, steps, gain)

    for bad in (dict(rot=0), dict(rot=63), dict(rot=-2), dict(base=1.0), dict(base=float("inf")), dict(base=float("nan")), dict(scaling=4),
                dict(scaling=-1), dict(factor=0.0), dict(factor=float("nan")), dict(factor=float("inf")), dict(scaling=2, rot=2),
                dict(scaling=3, original=0), dict(scaling=3, fast=1.0), dict(scaling=3, slow=0.0), dict(scaling=3, factor=0.5),
                dict(steps=None), dict(gain=None)):
        assert call(**bad) == INVALID, bad
    # one radian a position is 2^64 / 2 pi; the next pairs follow to the last bits of 64
    assert call() == 0 and gain.value == 1.0 and abs(steps[0] - 2935890503282001226) <= 1
    from fractions import Fraction
    assert abs(Fraction(steps[16]) - Fraction(steps[0], 100)) <= 2  # 10^4 ^ -(32 / 64)
    assert call(scaling=1, factor=4.0) == 0 and abs(steps[0] - 2935890503282001226 // 4) <= 1
    assert call(scaling=3, factor=8.0) == 0 and abs(gain.value - 1.2079441541679836) < 1e-7 and abs(steps[0] - 2935890503282001226) <= 1


def test_rope(lib):
    def call(type=0, q=rows(FAR[0]), q_out=rows(FAR[1]), q_heads=4, k=rows(FAR[2]), k_out=rows(FAR[3]), k_heads=2, dim=128, rot=64,
             steps=FAR[4], gain=1.0, interleaved=0, positions=FAR[5], tokens=3):
        return lib.qhip_launch_rope(type, q, q_out, q_heads, k, k_out, k_heads, dim, rot, steps, gain, interleaved, positions, tokens, None)

    assert call(tokens=0) == 0
    for bad in (dict(type=8), dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(q=rows(FAR[0] + 1)), dict(q_heads=0),
                dict(k_heads=-1), dict(dim=0), dict(rot=0), dict(rot=63), dict(rot=130), dict(steps=None), dict(steps=FAR[4] + 4),
                dict(positions=None), dict(positions=FAR[5] + 2), dict(interleaved=2), dict(tokens=-1), dict(tokens=2 ** 31 - 1),
                dict(q_out=rows(FAR[1], 512, 64)), dict(k_out=rows(FAR[3], 0)), dict(q_out=rows(FAR[0] + 4)), dict(q_out=rows(FAR[2])),
                dict(k_out=rows(FAR[0])), dict(k_out=rows(FAR[1] + 512)), dict(q_out=rows(FAR[4])), dict(k_out=rows(FAR[5])),
                dict(q_out=rows(FAR[0], 1024))):
        assert call(**bad) == INVALID, bad
    assert call(dim=2050, rot=2050, q=rows(FAR[0], 2 ** 20, 4096), q_out=rows(FAR[1], 2 ** 20, 4096)) == DECLINE
    assert call(dim=2050, rot=2) == DECLINE


def test_linear_attention(lib):
    f = dict(offsets=P, slots=P, source=P, nseq=2, tokens=7, max_new=4, num_states=5, k_heads=2, v_heads=4, key_dim=64, value_dim=64)

    def batch(**kw):
        return ctypes.byref(QhipLinearBatch(**{**f, **kw}))

    def call(b=batch(), type=0, q=rows(FAR[0]), k=rows(FAR[1]), v=rows(FAR[2]), decay=FAR[3], decay_stride=4, beta=FAR[4], beta_stride=4,
             states=FAR[5], out=rows(FAR[6]), work=None, work_bytes=0):
        return lib.qhip_launch_linear_attention(b, type, q, k, v, decay, decay_stride, beta, beta_stride, 1.0, states, out, work,
                                                work_bytes, None)

    assert call(batch(nseq=0)) == 0
    sizes = [dict(nseq=-1), dict(nseq=65536), dict(tokens=-1), dict(tokens=2 ** 31 - 1), dict(max_new=-1), dict(num_states=-1), dict(k_heads=0),
             dict(v_heads=0), dict(v_heads=5), dict(v_heads=65536), dict(key_dim=0), dict(value_dim=-64)]
    for bad in sizes:
        assert call(batch(**bad)) == INVALID, bad
        assert lib.qhip_linear_attention_work_bytes(batch(**bad), 0, 1) == -1, bad
    assert call(None) == INVALID
    for bad in (dict(offsets=None), dict(slots=None), dict(offsets=P + 2), dict(source=P + 1)):
        assert call(batch(**bad)) == INVALID, bad
    for bad in (dict(type=8), dict(q=None), dict(k=rows(FAR[1] + 2)), dict(v=rows(FAR[2], -512)), dict(decay=None), dict(decay=FAR[3] + 2),
                dict(beta=FAR[4] + 1), dict(decay_stride=-1), dict(beta_stride=-4), dict(states=None), dict(states=FAR[5] + 4),
                dict(out=None), dict(out=rows(FAR[6], 512, 32)), dict(out=rows(FAR[6], 0)), dict(out=rows(FAR[0])), dict(out=rows(FAR[2])),
                dict(out=rows(FAR[5])), dict(out=rows(FAR[3])), dict(out=rows(FAR[4])), dict(v=rows(FAR[5])), dict(q=rows(FAR[5] + 256))):
        assert call(**bad) == INVALID, bad
    for bad in (dict(key_dim=32), dict(key_dim=256), dict(value_dim=96), dict(value_dim=512)):
        assert call(batch(**bad)) == DECLINE, bad
    assert lib.qhip_linear_attention_work_bytes(batch(), 0, 1) >= 0


def test_linear_attention_work(lib):
    def need(type=0, delta=1, **kw):
        f = dict(offsets=P, slots=P, source=P, nseq=2, tokens=700, max_new=400, num_states=5, k_heads=2, v_heads=4, key_dim=64, value_dim=64)
        return lib.qhip_linear_attention_work_bytes(ctypes.byref(QhipLinearBatch(**{**f, **kw})), type, delta)

    full = need()
    assert full > 0 and full % 16 == 0 and 0 < need(delta=0) < full and need(type=1) > 0
    assert need(nseq=0) == need(tokens=0) == need(max_new=16) == 0
    assert need(max_new=17) > 0 and need(max_new=17, nseq=64) == need(max_new=32, nseq=64) == 0 < need(max_new=33, nseq=64)
    # grids of 2^32 threads: token by token
    assert need(nseq=65535, v_heads=64, k_heads=64) == 0 == need(tokens=2 ** 30, k_heads=1, v_heads=1)
    batch = QhipLinearBatch(P, P, None, 2, 700, 400, 5, 2, 4, 64, 64)
    for work, size in ((P, full - 1), (P + 8, full), (P, 0)):
        assert lib.qhip_launch_linear_attention(ctypes.byref(batch), 0, rows(FAR[0]), rows(FAR[1]), rows(FAR[2]), FAR[3], 4, FAR[4], 4, 1.0,
                                                FAR[5], rows(FAR[6]), work, size, None) == INVALID
    assert lib.qhip_launch_linear_attention(ctypes.byref(batch), 0, rows(FAR[0], 2 ** 23 + 1), rows(FAR[1]), rows(FAR[2]), FAR[3], 4, FAR[4], 4,
                                            1.0, FAR[5], rows(FAR[6]), None, 0, None) == INVALID
