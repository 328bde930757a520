"""Host-side checks of qhip_launch_kv_tables, every array at an address of its own, so that a refusal can only come from
the argument that was changed."""
import pytest
import torch

import qwen35_amd

INVALID = 1
NAMES = ["cached", "new", "nseq", "free", "nfree", "taken", "block", "table", "width", "tokens", "offsets", "kv_lens", "slots",
         "positions", "taken_out", "stream"]
INPUTS, OUTPUTS = ["cached", "new", "free", "taken", "table"], ["offsets", "kv_lens", "slots", "positions", "taken_out"]


@pytest.fixture(scope="module")
def lib():
    return qwen35_amd.load()


def args(**changed):
    """Two sequences, three free blocks, four columns, five tokens; addresses 4 KiB apart that nothing dereferences."""
    x = dict(nseq=2, nfree=3, block=16, width=4, tokens=5, stream=None)
    x.update({n: 0x1000 * (i + 1) for i, n in enumerate(INPUTS + OUTPUTS)})
    assert set(changed) <= set(x)
    return [{**x, **changed}[n] for n in NAMES]


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on addresses that are none")
def test_the_arguments_that_the_others_vary_are_accepted(lib):
    assert lib.qhip_launch_kv_tables(*args()) != INVALID  # the launch itself fails: no GPU


@pytest.mark.parametrize("changed", [
    dict(cached=None), dict(new=None), dict(nseq=-1), dict(free=None), dict(nfree=-1), dict(block=0), dict(block=8),
    dict(block=24), dict(block=512), dict(block=-16), dict(table=None), dict(width=-1), dict(tokens=-1), dict(offsets=None),
    dict(kv_lens=None), dict(slots=None), dict(taken_out=None)], ids=str)
def test_each_bad_argument_is_refused(lib, changed):
    assert lib.qhip_launch_kv_tables(*args(**changed)) == INVALID


LENGTHS = dict(cached=2, new=2, free=3, taken=1, table=8, offsets=3, kv_lens=2, slots=5, positions=5, taken_out=1)


@pytest.mark.parametrize("one,other", [(x, y) for x in ["table"] + OUTPUTS for y in INPUTS + OUTPUTS if x != y])
def test_arrays_over_each_other_are_refused(lib, one, other):
    """At the same address, and where only the last element of one lies on the first of the other."""
    at = 0x1000 * (1 + (INPUTS + OUTPUTS).index(other))
    for place in (at, at + 4 * (LENGTHS[other] - 1), at - 4 * (LENGTHS[one] - 1)):
        assert lib.qhip_launch_kv_tables(*args(**{one: place})) == INVALID


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on addresses that are none")
def test_arrays_side_by_side_and_empty_ones_are_accepted(lib):
    at = 0x1000 * (1 + INPUTS.index("cached"))
    assert lib.qhip_launch_kv_tables(*args(kv_lens=at + 4 * LENGTHS["cached"])) != INVALID
    assert lib.qhip_launch_kv_tables(*args(free=0x1000 * (1 + len(INPUTS)) + 4, nfree=0)) != INVALID  # inside offsets
