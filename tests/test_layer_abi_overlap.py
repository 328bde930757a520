"""Host-side checks of linear attention: what a call writes may share memory with nothing else of it."""
import ctypes

import pytest

import qwen35_amd
from qwen35_amd._lib import QhipLinearBatch, QhipRows

INVALID = 1
# never dereferenced: every call here is refused before any launch
Q, K, V, OUT, DECAY, BETA, STATES, WORK, OFFSETS, SLOTS, SOURCE = ((1 << 40) + (i << 28) for i in range(11))


def call(q=Q, k=K, v=V, out=OUT, decay=DECAY, beta=BETA, states=STATES, work=WORK, offsets=OFFSETS, slots=SLOTS, source=SOURCE, tokens=100,
         type=0):
    lib = qwen35_amd.load()
    batch = ctypes.byref(QhipLinearBatch(offsets, slots, source, 2, tokens, 90, 5, 2, 4, 64, 64))
    need = lib.qhip_linear_attention_work_bytes(batch, type, 1)
    rows = [ctypes.byref(QhipRows(at, 256, 64)) for at in (q, k, v, out)]
    return lib.qhip_launch_linear_attention(batch, type, *rows[:3], decay, 4, beta, 4, 1.0, states, rows[3], work, need, None)


STATE_BYTES = 5 * 4 * 64 * 64 * 4


@pytest.mark.parametrize("name", ["q", "k", "v", "out", "decay", "beta", "states", "offsets", "slots", "source"])
def test_the_workspace(name):
    need = qwen35_amd.load().qhip_linear_attention_work_bytes(
        ctypes.byref(QhipLinearBatch(OFFSETS, SLOTS, None, 2, 100, 90, 5, 2, 4, 64, 64)), 0, 1)
    assert need > 0
    for at in (WORK, WORK + need - 16):
        assert call(**{name: at}) == INVALID


@pytest.mark.parametrize("tokens", [100, 0])
@pytest.mark.parametrize("name", ["decay", "beta", "offsets", "slots", "source"])
def test_the_states(name, tokens):
    if tokens == 0 and name in ("decay", "beta"):
        return  # nothing of them is read
    for at in (STATES, STATES + STATE_BYTES - 4):
        assert call(**{name: at}, tokens=tokens) == INVALID


@pytest.mark.parametrize("name", ["offsets", "slots", "source"])
@pytest.mark.parametrize("type", [0, 30])
def test_the_outputs(name, type):
    for at in (OUT, OUT + (99 * 256 + 256) * (4 if type == 0 else 2) - 4):
        assert call(**{name: at}, type=type) == INVALID
