"""Workspaces of the attention over steps of many kinds: one that is large enough serves them all."""
import gc
import importlib.util
import os
import weakref

import pytest
import torch

import kv_reference as ref
import test_gpu_kv_attention as t
from qwen35_amd import ops

pytestmark = pytest.mark.gpu


def test_the_example_keeps_one_workspace(gpu, monkeypatch):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv_serving.py")
    spec = importlib.util.spec_from_file_location("kv_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    made, make = [], ops.kv_attention_work

    def record(*a, **kw):
        w = make(*a, **kw)
        if w is not None:
            made.append(weakref.ref(w))
        return w

    monkeypatch.setattr(ops, "kv_attention_work", record)
    backend = ops.Backend()
    layer = example.Layer(backend, 256, 8, 2, 64, 80, 64)
    server = example.Server(layer, 2, 2500)
    for new in ([700, 3], [300, 1], [251, 2], [1, 1], [333, 44], [127, 1], [1, 0]):
        y, _ = server.step(torch.randn((sum(new), 256), device="cuda"), new)
        assert bool(torch.isfinite(y).all())
    gc.collect()
    torch.cuda.synchronize()
    assert made and len({id(w()) for w in made if w() is not None}) == 1
    backend.close()


def test_a_workspace_that_is_large_enough_is_kept(gpu):
    cache, table, offsets, kv_lens, q = t.make([(9000, 1), (8000, 1)], 2, 4, 64, 128, torch.float32)
    work = ops.kv_attention_work(cache, 8, 2, 2, 1, 9000)
    assert ops.kv_attention_work(cache, 8, 2, 2, 1, 4000, work=work) is work
    assert ops.kv_attention_work(cache, 8, 2, 2, 1, 10, work=work) is work  # nothing to cut
    larger = ops.kv_attention_work(cache, 8, 2, 100, 60, 9000, work=work)
    assert larger is not work and larger.numel() > work.numel() and not bool(larger.any())
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5)
    own = t.attend(cache, table, offsets, kv_lens, q)
    for _ in range(3):
        got = ops.kv_attention(q, cache, t.ints(table), t.ints(offsets), t.ints(kv_lens), 1, 9000, work=larger)
        t.compare(*got, *want, torch.float32)
        assert torch.equal(got[0], own[0]) and torch.equal(got[1], own[1])
    for bad in (work.cpu(), work.view(torch.float32)):
        with pytest.raises(ValueError):
            ops.kv_attention_work(cache, 8, 2, 2, 1, 4000, work=bad)


def test_a_batch_past_its_bounds_leaves_the_workspace_usable(gpu):
    """More new tokens than max_new says: rows may stay unwritten, but no counter is left for the next call."""
    lens = [(9000, 508)] + [(0, 0)] * 12
    cache, table, offsets, kv_lens, q = t.make(lens, 2, 4, 64, 128, torch.float32)
    args = (q, cache, t.ints(table), t.ints(offsets), t.ints(kv_lens))
    work = ops.kv_attention_work(cache, 8, 13, 508, 508, 9000)
    work = ops.kv_attention_work(cache, 8, 13, 508, 4, 9000, work=work)
    ops.kv_attention(*args, 4, 9000, work=work)
    assert not bool(work[:32768].any())
    want = t.attend(cache, table, offsets, kv_lens, q)
    got = ops.kv_attention(*args, 508, 9000, work=work)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
