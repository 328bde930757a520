"""Sequences that fall back: draft tokens are appended, verified, and some of them rejected.

The next step's `cached` is what was kept.  Blocks behind it go back to the free list (into entries that are spent)
before the next tables, which give the sequence fresh ones; a block that is kept keeps its scale."""
import random

import pytest
import torch

import kv_reference as ref
import test_gpu_kv_attention as t
from qwen35_amd import ops

pytestmark = pytest.mark.gpu


def give_back(table, free, taken, had, keep, block):
    """Blocks of each sequence behind keep[i] of had[i] tokens, into the free list's last taken entries."""
    j = torch.arange(table.shape[1], device="cuda")
    gone = (j >= ((keep + block - 1) // block)[:, None]) & (j < ((had + block - 1) // block)[:, None])
    ids = table[gone]
    free[int(taken) - len(ids):int(taken)] = ids
    return taken - len(ids)


@pytest.mark.parametrize("block,dim", [(16, 64), (32, 128)])
def test_rejected_drafts(gpu, block, dim):
    rng, gen = random.Random(block), torch.Generator(device="cuda").manual_seed(block)
    nseq, heads, group, pool = 7, 2, 3, 60
    cache, mirror = ops.KvCache.empty(pool, heads, block, dim), ops.KvCache.empty(pool, heads, block, dim)
    order = list(range(pool))
    rng.shuffle(order)
    free, taken = t.ints(order), t.ints([0])
    table = torch.full((nseq, 12), -1, dtype=torch.int32, device="cuda")
    kept = [rng.randint(0, 3 * block) for _ in range(nseq)]
    cached, new = [0] * nseq, kept  # the prompts first
    for _ in range(12):
        step = ops.KvStep(nseq, sum(new))
        ops.kv_tables(t.ints(cached), t.ints(new), free, table, block, step, taken=taken)
        taken = step.taken
        kv = torch.randn((2, sum(new), heads, dim), device="cuda", generator=gen) * rng.choice([0.5, 1.0, 3.0])
        ops.kv_append(cache, kv[0], kv[1], step.slots)
        slots = step.slots.tolist()
        assert min(slots) >= 0 and len(set(slots)) == len(slots)
        for name, x in (("k", kv[0]), ("v", kv[1])):
            codes, scales = ref.append(getattr(mirror, name), getattr(mirror, name + "_scale"), x, slots)
            assert torch.equal(getattr(cache, name), codes) and torch.equal(getattr(cache, name + "_scale"), scales)
            getattr(mirror, name).copy_(codes)
            getattr(mirror, name + "_scale").copy_(scales)
        had = [c + n for c, n in zip(cached, new)]
        q = torch.randn((sum(new), heads * group, dim), device="cuda", generator=gen)
        offsets = step.offsets.tolist()
        got = ops.kv_attention(q, cache, table, step.offsets, step.kv_lens, max(new), max(had))
        want = ref.attention(q, mirror.k, mirror.v, mirror.k_scale, mirror.v_scale, table.tolist(), offsets, had, dim ** -0.5)
        t.compare(*got, *want, torch.float32)
        # from none to all of the step's tokens are given up
        cached = [c + rng.randint(0, n) for c, n in zip(cached, new)]
        taken = give_back(table, free, taken, t.ints(had), t.ints(cached), block)
        own = [e for row, c in zip(table.tolist(), cached) for e in row[:-(-c // block)]]
        assert sorted(own + free[int(taken):].tolist()) == list(range(pool))  # no block lost, none twice
        new = [rng.randint(0, 9) for _ in range(nseq)]
        new[0] += 1
