"""What the binding of the 8-bit key/value cache refuses before any launch, and what it takes."""
import pytest
import torch

import test_gpu_kv_attention as t
import test_gpu_kv_cache as c
from qwen35_amd import ops

pytestmark = pytest.mark.gpu
FIELDS = ("k", "v", "k_scale", "v_scale")


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


def test_tensors_put_in_a_caches_place_are_the_ones_used(gpu):
    cache, other = c.pool(3, 2, 16, 64), c.pool(3, 2, 16, 64, seed=1)
    old = [getattr(cache, n).clone() for n in FIELDS]
    kept = [getattr(cache, n) for n in FIELDS]
    want = c.pool(3, 2, 16, 64, seed=1)
    for name in FIELDS:
        setattr(cache, name, getattr(other, name))
    kv = torch.randn((2, 3, 2, 64), device="cuda")
    slots = c.ints([16, 17, 18])
    ops.kv_append(want, kv[0], kv[1], slots)
    ops.kv_append(cache, kv[0], kv[1], slots)
    assert all(torch.equal(getattr(other, n), getattr(want, n)) for n in FIELDS)
    assert all(torch.equal(a, b) for a, b in zip(old, kept))


def test_what_does_not_fit_a_cache_is_refused(gpu):
    cache = c.pool(3, 2, 16, 64)
    before = [getattr(cache, n).data_ptr() for n in FIELDS]
    for name, bad in [("k", cache.k.float()), ("k", cache.k[:2]), ("v", cache.v.cpu()), ("v", cache.v.transpose(0, 1)), ("k", None),
                      ("k_scale", cache.k_scale[:2]), ("v_scale", cache.v_scale.double()), ("v_scale", cache.v_scale.t())]:
        with pytest.raises(ValueError):
            setattr(cache, name, bad)
    for name in ("num_blocks", "kv_heads", "block_size", "head_dim"):
        with pytest.raises(AttributeError):
            setattr(cache, name, 1)
    assert before == [getattr(cache, n).data_ptr() for n in FIELDS]
    for bad in ((cache.k[0], cache.v[0]), (cache.k.cpu(), cache.v)):
        with pytest.raises(ValueError):
            ops.KvCache(*bad, cache.k_scale, cache.v_scale)


def test_a_steps_sizes_are_fixed(gpu):
    """The kernel writes as many entries as the step says."""
    step = ops.KvStep(2, 4)
    for name in ("nseq", "tokens"):
        with pytest.raises(AttributeError):
            setattr(step, name, 100)
    step.slots = c.ints([0] * 4)
    for name, bad in (("slots", c.ints([0] * 3)), ("offsets", c.ints([0] * 2)), ("taken", c.ints([])), ("kv_lens", None)):
        with pytest.raises(ValueError):
            setattr(step, name, bad)
    assert (step.nseq, step.tokens) == (2, 4)


def test_tensors_of_another_device_are_refused(gpu, monkeypatch):
    """Launches go to the current device's stream: as if that were another one."""
    cache, table, offsets, kv_lens, q = t.make([(40, 2), (70, 1)], 2, 2, 32, 64, torch.float32)
    step, slots = ops.KvStep(2, 4), c.ints([0, 1, 2])
    table, offsets, kv_lens = t.ints(table), t.ints(offsets), t.ints(kv_lens)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: ops.kv_tables(slots[:2], slots[:2], slots, table, 16, step), lambda: ops.kv_append(cache, q[:, :2], q[:, 2:], slots),
                 lambda: ops.kv_read(cache, slots), lambda: ops.kv_attention(q, cache, table, offsets, kv_lens, 2, 70)):
        with pytest.raises(ValueError):
            call()


def test_launches_go_to_the_current_stream(gpu):
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            assert (ops._stream().value or 0) == torch.cuda.current_stream().cuda_stream == stream.cuda_stream


def test_numbers_past_32_bits_are_refused(gpu):
    """They would be cut to their lowest 32 bits: a bound of 2^32 to none."""
    cache, table, offsets, kv_lens, q = t.make([(40, 2), (70, 1)], 2, 2, 32, 64, torch.float32)
    args = (q, cache, t.ints(table), t.ints(offsets), t.ints(kv_lens))
    for most, longest, window in ((2 ** 32, 70, 0), (2, 2 ** 32 + 70, 0), (2, 70, 2 ** 32 + 3), (2 ** 31, 70, 0),
                                  (-2 ** 32, 70, 0)):
        with pytest.raises(ValueError):
            ops.kv_attention(*args, most, longest, window=window)
    for bad in ((2 ** 32 + 2, 3, 2, 70), (2, 2 ** 32 + 3, 2, 70), (2, 3, 2 ** 32, 70), (2, 3, 2, 2 ** 32 + 70)):
        with pytest.raises(ValueError):
            ops.kv_attention_work(cache, 4, *bad)
    with pytest.raises(ValueError):
        ops.kv_tables(c.ints([0]), c.ints([0]), c.ints([1]), c.ints([[0]]), 2 ** 32 + 16, ops.KvStep(1, 0))
