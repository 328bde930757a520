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


@pytest.mark.parametrize("block", [16, 128])
@pytest.mark.parametrize("nseq,nlo,nhi", [(1030, 0, 12), (2047, 1, 7), (3000, 0, 5), (1025, 4, 4)])
def test_thousands_of_tokens_for_more_than_1024_sequences(gpu, nseq, nlo, nhi, block):
    """Four tokens a thread, which may belong to sequences on both sides of 1024; whole, padded and cut short."""
    rng = random.Random(nseq)
    cached, new = [rng.randint(0, 100) for _ in range(nseq)], [rng.randint(nlo, nhi) for _ in range(nseq)]
    total, width = sum(new), (100 + nhi) // block + 2
    assert total > 4096
    free = [rng.randint(0, 2 ** 22) for _ in range(total // block + nseq)]
    t.check_tables(cached, new, free, width, block)
    for tokens in (total + 1, total + 1030, total + 4099):
        t.check_tables(cached, new, free, width, block, tokens=tokens)


@pytest.mark.parametrize("short", [1, 2, 3, 5])
@pytest.mark.parametrize("lens", [[9000], [3, 5000, 2, 4000], [6] * 1500])
def test_thousands_of_slots_of_fewer_than_the_tokens(gpu, lens, short):
    """`tokens` below the sum of the lengths: nothing past it is written, wherever a thread's four tokens are cut."""
    tokens, block = sum(lens) - short, 16
    width = max(lens) // block + 2
    free = list(range(sum(n // block + 1 for n in lens)))
    want = ref.tables([1] * len(lens), lens, free, 0, [[7] * width for _ in lens], block, tokens)
    step = ops.KvStep(len(lens), tokens)
    guard = t.ints([-7] * (2 * tokens + 64))
    step.slots, step.positions = guard[:tokens], guard[tokens + 32:2 * tokens + 32]
    table = t.ints([[7] * width for _ in lens])
    ops.kv_tables(t.ints([1] * len(lens)), t.ints(lens), t.ints(free), table, block, step)
    assert (table.tolist(), step.offsets.tolist(), step.kv_lens.tolist()) == want[:3]
    assert (step.slots.tolist(), step.positions.tolist(), int(step.taken)) == want[3:]
    assert guard[tokens:tokens + 32].tolist() == [-7] * 32 and guard[2 * tokens + 32:].tolist() == [-7] * 32
