"""What a launch of rotary positions is given of its table: the frequencies that the table holds at that call."""
import copy
import pickle

import pytest
import torch

from qwen35_amd import ops


class Launches:
    """The library with launches noted in place of done."""

    def __init__(self, lib):
        self.lib, self.steps = lib, []

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def qhip_launch_rope(self, *args):
        self.steps.append(args[9])
        return 0


@pytest.fixture
def launches(monkeypatch):
    lib = Launches(ops.load())
    monkeypatch.setattr(ops, "load", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda device: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # where get_device() puts tensors of the CPU
    return lib


def call(table):
    ops.rope(torch.zeros((3, 2, 128)), None, torch.zeros(3, dtype=torch.int32), table)


def test_copies_and_other_steps(launches):
    first = ops.RopeTable(64, device="cpu")
    tables = [first, copy.deepcopy(first), copy.copy(first), pickle.loads(pickle.dumps(first))]
    for table in tables:
        assert torch.equal(table.steps, first.steps) and table.rot_dim == 64 and table.gain == first.gain and table.device == -1
        call(table)
    assert launches.steps == [t.steps.data_ptr() for t in tables]
    assert len({t.steps.data_ptr() for t in tables}) == 3  # (a shallow copy shares them)
    first.steps = first.steps * 2
    call(first)
    assert launches.steps[-1] == first.steps.data_ptr() != launches.steps[0]


def test_steps_that_do_not_fit(launches):
    table = ops.RopeTable(64, device="cpu")
    with pytest.raises(AttributeError):
        table.rot_dim = 128
    assert table.rot_dim == 64
    steps = table.steps
    for bad in (steps[:31], steps.int(), torch.stack([steps, steps], 1)[:, 0], steps.view(2, 16)):
        table.steps = bad
        with pytest.raises(ValueError):
            call(table)
    table.steps = steps
    table.__dict__["rot_dim"] = 128
    with pytest.raises(ValueError):
        call(table)
    assert launches.steps == []
