"""What the binding of the 8-bit key/value cache refuses before any launch, and what it takes."""
import pytest
import torch

import test_gpu_kv_attention as t
import test_gpu_kv_cache as c
from qwen35_amd import ops

pytestmark = pytest.mark.gpu


def test_work_is_a_byte_tensor_on_the_gpu(gpu):
    cache, table, offsets, kv_lens, q = t.make([(9000, 1)], 2, 4, 64, 128, torch.float32)
    args = (q, cache, t.ints(table), t.ints(offsets), t.ints(kv_lens), 1, 9000)
    work = ops.kv_attention_work(cache, 8, 1, 1, 1, 9000)
    for bad in (work.cpu(), work.view(torch.float32), work[::2], work[:1].expand(len(work)), work.view(2, -1).t()):
        with pytest.raises(ValueError):
            ops.kv_attention(*args, work=bad)
    ops.kv_attention(*args, work=work)
    assert not bool(work[:32768].any())


def test_taken_has_one_entry(gpu):
    """No entry would count as none taken, and read nothing."""
    step = ops.KvStep(2, 4)
    for bad in (c.ints([]), c.ints([1, 2]), c.ints([[1]]), torch.tensor([1], device="cuda"), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError):
            ops.kv_tables(c.ints([0, 0]), c.ints([2, 2]), c.ints([4, 5, 6]), c.ints([[0], [0]]), 16, step, taken=bad)
