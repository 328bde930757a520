"""Block tables: block ids that no slot can number, and steps of thousands of tokens for more than 1024 sequences.

Whole numbers: equal to the plain form's."""
import random

import pytest

import kv_reference as ref
import test_gpu_kv_cache as t
from qwen35_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [16, 64, 256])
def test_block_ids_that_no_slot_can_number_give_no_slot(gpu, block):
    """A slot is block * block_size + place in 31 bits: a larger block is outside every pool, like a negative one."""
    top = 2 ** 31 // block
    for bad in (top, top + 3, 2 ** 30, 2 ** 31 - 1, -1, -2 ** 31):
        # the held, partly filled block of the first sequence; a fresh one of the second
        step = ops.KvStep(2, 2 + block)
        table = t.ints([[bad, 0], [0, 0]])
        ops.kv_tables(t.ints([3, 0]), t.ints([2, block]), t.ints([bad]), table, block, step)
        assert step.slots.tolist() == [-1] * (2 + block), bad
        assert step.positions.tolist() == [3, 4] + list(range(block))
        assert table.tolist() == [[bad, 0], [bad, 0]]
    step = ops.KvStep(1, 1)
    ops.kv_tables(t.ints([block - 1]), t.ints([1]), t.ints([]), t.ints([[top - 1]]), block, step)
    assert step.slots.tolist() == [2 ** 31 - 1]
