"""Block tables, append and read-back of the 8-bit key/value cache against a plain 64-bit form.

Whole numbers (tables, slots, codes) and scales are equal: the codes and scales
are defined by single f32 operations."""
import ctypes
import math
import random

import pytest
import torch

import kv_reference as ref
from qwen35_amd import QhipError, ops

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_tables(cached, new, free, width, block, tokens=None, taken=0, table=None):
    tokens = sum(max(n, 0) for n in new) if tokens is None else tokens
    table = [[random.Random(i).randint(0, 10 ** 6) for _ in range(width)] for i in range(len(new))] if table is None else table
    want = ref.tables(cached, new, free, taken, table, block, tokens)
    step = ops.KvStep(len(new), tokens)
    for t in (step.slots, step.positions, step.offsets, step.kv_lens):
        t.fill_(-77)
    dev = ints(table).reshape(len(new), width)
    ops.kv_tables(ints(cached), ints(new), ints(free), dev, block, step, taken=ints([taken]))
    got = (dev.tolist(), step.offsets.tolist(), step.kv_lens.tolist(), step.slots.tolist(), step.positions.tolist(),
           int(step.taken))
    assert got == want


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("nseq,lo,hi,nlo,nhi", [(1, 0, 0, 1, 1), (1, 5, 5, 2111, 2111), (3, 0, 40, 0, 3), (64, 0, 700, 1, 1),
                                               (130, 0, 300, 0, 200), (1025, 0, 90, 0, 7), (2500, 0, 33, 0, 2)])
def test_tables(gpu, block, nseq, lo, hi, nlo, nhi):
    rng = random.Random(nseq + block)
    cached = [rng.randint(lo, hi) for _ in range(nseq)]
    new = [rng.randint(nlo, nhi) for _ in range(nseq)]
    width = (hi + nhi) // block + 2
    free = [rng.randint(0, 2 ** 22) for _ in range(sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(cached, new)) + 3)]
    check_tables(cached, new, free, width, block)


def test_tables_of_idle_rows_and_padding(gpu):
    check_tables([0, 17, 0, 5, 0], [0, 0, 0, 1, 0], [9, 8], 3, 16, tokens=6)
    check_tables([0], [0], [], 2, 16, tokens=0)
    check_tables([0] * 5, [0] * 5, [3], 2, 16, tokens=2100)
    check_tables([-4, 3], [2, -1], [7, 6], 2, 16, tokens=3)  # negative counts are none


def test_tables_when_blocks_or_columns_run_out(gpu):
    check_tables([0, 16, 30], [40, 20, 40], [5, 6, 7, 8], 6, 16)
    check_tables([0, 16, 30], [40, 20, 40], list(range(50, 80)), 3, 16)
    check_tables([3, 3], [20, 20], [1, 2, 3], 4, 16, taken=2)
    check_tables([3, 3], [20, 20], [1, 2, 3], 4, 16, taken=9)
    check_tables([20], [5], [1, 2], 2, 16, table=[[-1, -1]])  # a held block that is missing


def test_tables_of_fewer_slots_than_tokens(gpu):
    """`tokens` below the sum of the lengths: nothing past it is written, the table still is."""
    table = ints([[4, 0, 0, 0]])
    step = ops.KvStep(1, 20)
    guard = torch.full((64,), -7, dtype=torch.int32, device="cuda")
    step.slots, step.positions = guard[:20], guard[32:52]
    ops.kv_tables(ints([10]), ints([40]), ints([1, 2, 3]), table, 16, step)
    assert table.tolist() == [[4, 1, 2, 3]] and int(step.taken) == 3
    assert guard[20:32].tolist() == [-7] * 12 and guard[52:].tolist() == [-7] * 12
    assert step.slots.tolist() == [4 * 16 + 10 + i if i < 6 else 16 + i - 6 for i in range(20)]


def test_tables_steps_follow_each_other(gpu):
    """Decode steps that pass lengths and the free list's place on, all on the GPU."""
    nseq, block, width = 5, 16, 6
    cached, taken = ints([0, 15, 16, 31, 3]), ints([0])
    table = torch.full((nseq, width), -1, dtype=torch.int32, device="cuda")
    table[1, 0], table[2, 0], table[3, :2], table[4, 0] = 90, 91, ints([92, 93]), 94
    want, c, k = table.tolist(), cached.tolist(), 0
    free = list(range(40))
    for _ in range(20):
        step = ops.KvStep(nseq, nseq)
        ops.kv_tables(cached, ints([1] * nseq), ints(free), table, block, step, taken=taken)
        want, _, c, slots, _, k = ref.tables(c, [1] * nseq, free, k, want, block, nseq)
        cached, taken = step.kv_lens, step.taken
        assert step.slots.tolist() == slots
    assert table.tolist() == want and cached.tolist() == c and int(taken) == k


# ---- append ------------------------------------------------------------------------------

def pool(blocks, heads, block, dim, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (blocks, heads, block, dim)
    k = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
    v = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
    ks = torch.rand(shape[:2], device="cuda", generator=gen) * 0.03 + 1e-3
    vs = torch.rand(shape[:2], device="cuda", generator=gen) * 0.03 + 1e-3
    return ops.KvCache(k, v, ks, vs)


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


def check_append(cache, k, v, slots):
    wk = ref.append(cache.k, cache.k_scale, k, slots)
    wv = ref.append(cache.v, cache.v_scale, v, slots)
    ops.kv_append(cache, k, v, ints(slots))
    assert same(cache.k_scale, wk[1]) and same(cache.v_scale, wv[1])
    assert torch.equal(cache.k, wk[0]) and torch.equal(cache.v, wv[0])


RUNS = {
    "one": [(3, 0, 1)], "one_inside": [(2, 9, 1)], "last_place": [(1, -1, 1)],
    "runs": [(0, 0, 5), (4, 3, 2), (2, -2, 2), (5, 0, -1)], "whole_blocks": [(5, 0, -1), (1, 0, -1), (3, 7, -1)],
}


def slots_of(runs, block):
    """(block, first place, count) with negative places and counts from the block's end."""
    out = []
    for b, first, n in runs:
        first = first % block
        n = n if n > 0 else block - first
        out += [b * block + first + i for i in range(n)]
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block,dim,heads", [(16, 64, 3), (32, 128, 2), (64, 256, 2), (128, 128, 1), (256, 256, 1), (256, 64, 2)])
@pytest.mark.parametrize("runs", sorted(RUNS))
def test_append(gpu, dtype, block, dim, heads, runs):
    gen = torch.Generator(device="cuda").manual_seed(block + dim)
    slots = slots_of(RUNS[runs], block)
    for loud in (0.01, 1.0, 40.0):  # scales that stay, and that grow
        cache = pool(6, heads, block, dim, seed=int(loud))
        kv = (torch.randn((2, len(slots), heads, dim), device="cuda", generator=gen) * loud).to(dtype)
        check_append(cache, kv[0], kv[1], slots)


def test_append_again_keeps_the_codes(gpu):
    cache = pool(3, 2, 16, 64)
    kv = torch.randn((2, 4, 2, 64), device="cuda") * 30
    slots = slots_of([(1, 5, 4)], 16)
    check_append(cache, kv[0], kv[1], slots)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    ops.kv_append(cache, kv[0], kv[1], ints(slots))
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)))


def test_append_skips_slots_outside_the_pool(gpu):
    cache = pool(3, 2, 16, 64)
    kv = torch.randn((2, 7, 2, 64), device="cuda")
    kv[:, [0, 3, 6]] = math.nan
    check_append(cache, kv[0], kv[1], [-1, 16, 17, 48, 36, 37, 2 ** 31 - 1])
    cache2 = pool(3, 2, 16, 64)
    before = cache2.k.clone()
    ops.kv_append(cache2, kv[0], kv[1], ints([-1] * 7))
    ops.kv_append(cache2, kv[0, :0], kv[1, :0], ints([]))
    assert torch.equal(before, cache2.k)


@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf, 0.0, 1e-44, 3e38])
@pytest.mark.parametrize("first", [0, 4])
def test_append_of_extreme_values(gpu, odd, first):
    cache = pool(3, 2, 16, 64)
    kv = torch.randn((2, 3, 2, 64), device="cuda") * (0.0 if abs(odd) < 1 else 1.0)
    kv[0, 1, 0, 7] = odd
    kv[1, 2, 1, 0] = odd
    check_append(cache, kv[0], kv[1], slots_of([(1, first, 3)], 16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_of_strided_and_unaligned_rows(gpu, dtype):
    """Keys and values inside a projection's output, and rows that 16-byte loads cannot read."""
    tokens, heads, dim = 20, 3, 128
    slots = slots_of([(2, 0, 16), (0, 1, 4)], 16)
    wide = torch.randn((tokens, 2 * heads * dim + 4 * dim), device="cuda").to(dtype)
    kv = wide[:, :2 * heads * dim].reshape(tokens, heads, 2, dim)
    check_append(pool(4, heads, 16, dim), kv[:, :, 0], kv[:, :, 1], slots)
    flat = torch.randn(1 + tokens * heads * (dim + 1) * 2, device="cuda").to(dtype)[1:]
    kv = flat.reshape(tokens, heads, 2, dim + 1)[..., :dim]
    check_append(pool(4, heads, 16, dim), kv[:, :, 0], kv[:, :, 1], slots)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block,dim", [(16, 64), (64, 128), (256, 256)])
def test_read(gpu, dtype, block, dim):
    cache = pool(7, 3, block, dim)
    ids = [4, 0, 0, 6, -1, 7]
    k, v = ops.kv_read(cache, ints(ids), dtype)
    for got, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        want = (codes[ids[:4]].float() * scales[ids[:4]][..., None, None]).to(dtype)
        assert torch.equal(got[:4], want) and bool(got[4:].isnan().all())


def test_pool_past_32_bit_offsets(gpu):
    """A pool of more than 2^32 codes: the last block's bytes lie behind 4 GiB."""
    blocks, heads, block, dim = 16500, 4, 256, 256
    shape = (blocks, heads, block, dim)
    k, v = torch.zeros(shape, dtype=torch.int8, device="cuda"), torch.zeros(shape, dtype=torch.int8, device="cuda")
    cache = ops.KvCache(k, v, torch.zeros(shape[:2], device="cuda"), torch.zeros(shape[:2], device="cuda"))
    kv = torch.randn((2, 9, heads, dim), device="cuda")
    last = blocks - 1
    slots = [last * block + 3 + i for i in range(9)]
    ops.kv_append(cache, kv[0], kv[1], ints(slots))
    wk = ref.append(torch.zeros((1, *shape[1:]), dtype=torch.int8, device="cuda"), torch.zeros((1, heads), device="cuda"), kv[0],
                    [3 + i for i in range(9)])
    assert torch.equal(cache.k[last], wk[0][0]) and torch.equal(cache.k_scale[last], wk[1][0])
    assert not bool(cache.k[:last].any())
    got, _ = ops.kv_read(cache, ints([last]))
    assert torch.equal(got[0], cache.k[last].float() * cache.k_scale[last][:, None, None])


def test_refusals(gpu):
    cache = pool(3, 2, 16, 64)
    k = torch.randn((4, 2, 64), device="cuda")
    slots = ints([0, 1, 2, 3])
    for bad in (k.double(), k[:, :1], k[:, :, :32], k.transpose(1, 2), k[:3], k.cpu()):
        with pytest.raises(ValueError):
            ops.kv_append(cache, bad, k, slots)
    with pytest.raises(ValueError):
        ops.kv_append(cache, k, k.half(), slots)
    with pytest.raises(ValueError):
        ops.kv_append(cache, k, k, slots.long())
    with pytest.raises(ValueError):
        ops.KvCache(cache.k, cache.v, cache.k_scale.double(), cache.v_scale)
    with pytest.raises(ValueError):
        ops.KvCache(cache.k.float(), cache.v, cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        ops.KvCache(cache.k, cache.v[:2], cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        ops.kv_read(cache, slots, torch.float64)
    step = ops.KvStep(2, 4)
    with pytest.raises(ValueError):
        ops.kv_tables(slots[:2], slots[:3], slots, ints([[0], [0]]), 16, step)
    with pytest.raises(QhipError):
        ops.kv_tables(slots[:2], slots[:2], slots, ints([[0], [0]]), 24, step)
    odd = ops.KvCache.empty(2, 2, 16, 80)
    with pytest.raises(QhipError) as e:
        ops.kv_append(odd, torch.randn((1, 2, 80), device="cuda"), torch.randn((1, 2, 80), device="cuda"), slots[:1])
    assert e.value.code == -1  # declined: no kernel for this head width
    assert ctypes.sizeof(cache._c) == 48
