"""Attention over the 8-bit cache for batches of much work, which f16 and bf16 rows have staged through LDS.

Tolerances as in test_gpu_kv_attention.py: relative L2 1e-5, 1e-3 and 4e-3."""
import math

import pytest
import torch

import kv_reference as ref
import test_gpu_kv_attention as t
from qwen35_amd import QhipError, ops


pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]
#: (kv_len, rows): whole prompts, a chunk beside decodes and short prompts, rows that see nothing
PROMPTS = [(3001, 3001)]
MIXED = [(6000, 1000), (700, 1), (0, 0), (90, 7), (3000, 260), (5, 40), (1, 1), (0, 3)]


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 8), (128, 2, 8), (256, 3, 8), (128, 16, 1), (64, 3, 5)])
@pytest.mark.parametrize("lens", [PROMPTS, MIXED])
def test_batches(gpu, lens, dim, heads, group, dtype):
    t.check(lens, heads, group, 64, dim, dtype, seed=dim)


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 8), (128, 2, 8), (256, 3, 8), (64, 12, 1)])
def test_a_short_sequence_among_long_ones(gpu, dim, heads, group, dtype):
    lens = [(3001, 3001), (2500, 1), (2900, 2500), (0, 0)]
    t.check(lens, heads, group, 64, dim, dtype, seed=dim)
    t.check(lens, heads, group, 64, dim, dtype, seed=dim, window=700)


@pytest.mark.parametrize("block", [16, 32, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_block_sizes(gpu, dim, block):
    t.check(MIXED, 4, 8, block, dim, torch.bfloat16, seed=block)


@pytest.mark.parametrize("window", [1, 40, 700, 2900])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_windows(gpu, dim, window):
    t.check([(9000, 6000)], 4, 8, 32, dim, torch.float16, window=window, seed=window)
    t.check(MIXED, 4, 8, 16, dim, torch.bfloat16, window=window, seed=window)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_without_causality(gpu, dim):
    t.check(MIXED, 4, 8, 64, dim, torch.float16, causal=False)


@pytest.mark.parametrize("dtype", HALVES)
def test_scales_of_queries_values_and_softmax(gpu, dtype):
    t.check(MIXED, 2, 8, 32, 128, dtype, scale=0.0)
    t.check(MIXED, 2, 8, 32, 128, dtype, scale=-0.1)
    cache, table, offsets, kv_lens, q = t.make(MIXED, 2, 8, 16, 128, dtype, seed=3)
    n = cache.num_blocks
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache.v_scale.mul_(torch.logspace(-6, 6, n, device="cuda")[torch.randperm(n, device="cuda", generator=gen)][:, None])
    cache.v_scale.clamp_(max=200)
    cache.k_scale[::3] = 0
    cache.v_scale[1::5] = 0
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5)
    out, lse = t.attend(cache, table, offsets, kv_lens, q)
    rows = want[0].norm(dim=-1)
    # every row on its own: rounding to the type, and the weights' 11 bits
    assert bool(((out.double() - want[0]).norm(dim=-1) <= 2 * t.REL[dtype] * rows + 1e-30).all())
    assert torch.equal(torch.isfinite(lse), torch.isfinite(want[1]))


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("dim,lens", [(64, [(90000, 40)]), (128, [(90000, 40), (70, 9)]), (256, [(150000, 60)])])
def test_few_tiles_on_many_keys(gpu, dim, lens, dtype):
    """As many chunks of a row tile as a join takes."""
    t.check(lens, 2, 8, 64, dim, dtype, seed=dim)


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_poisoned_blocks_reach_their_rows_only(gpu, odd):
    lens = [(4000, 1500), (3000, 700)]
    cache, table, offsets, kv_lens, q = t.make(lens, 2, 8, 64, 128, torch.float16)
    plain = t.attend(cache, table, offsets, kv_lens, q)
    block = 50  # places 3200.. of the first sequence, whose new tokens begin at 2500
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    hit[3200 - 2500:1500, 8:] = True
    cache.v_scale[table[0][block], 1] = odd
    out, lse = t.attend(cache, table, offsets, kv_lens, q)
    assert torch.equal(out.isnan().all(-1), hit) and torch.equal(out.isnan().any(-1), hit)
    assert torch.equal(out[~hit], plain[0][~hit]) and torch.equal(lse, plain[1])
    cache.v_scale[table[0][block], 1] = 0.01
    cache.k_scale[table[0][block], 1] = odd
    out, lse = t.attend(cache, table, offsets, kv_lens, q)
    assert torch.equal(out.isnan().all(-1), hit) and torch.equal(lse.isnan(), hit)
    bad = [list(r) for r in table]
    bad[0][block] = -1
    cache.k_scale[table[0][block], 1] = 0.01
    out, _ = t.attend(cache, bad, offsets, kv_lens, q)
    assert torch.equal(out.isnan().all((1, 2)), hit.any(1))


def test_the_same_results_on_every_run_and_at_odd_addresses(gpu):
    for lens in (PROMPTS, MIXED):
        cache, table, offsets, kv_lens, q = t.make(lens, 2, 8, 64, 128, torch.bfloat16)
        first = t.attend(cache, table, offsets, kv_lens, q)
        for _ in range(3):
            again = t.attend(cache, table, offsets, kv_lens, q)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        flat = torch.empty(1 + len(q) * 16 * 131, dtype=torch.bfloat16, device="cuda")
        odd = flat[1:].reshape(len(q), 16, 131)[..., :128]
        odd.copy_(q)
        to = torch.full_like(flat, 7.0)[1:].reshape(len(q), 16, 131)
        got = t.attend(cache, table, offsets, kv_lens, odd, out=to[..., :128])
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
        assert bool((to[..., 128:] == 7.0).all())


@pytest.mark.parametrize("dtype", t.DTYPES)
def test_many_query_heads_of_a_key_head(gpu, dtype):
    """More than 64 rows a token, in every kernel, and the most that is served."""
    for group in (65, 130, 512):
        t.check([(300, 1), (40, 3), (0, 1)], 1, group, 32, 64, dtype, seed=group)
    t.check([(700, 200)], 1, 100, 32, 64, dtype)
    cache = ops.KvCache.empty(4, 1, 16, 64)
    with pytest.raises(QhipError) as e:
        ops.kv_attention(torch.zeros((1, 513, 64), dtype=dtype, device="cuda"), cache, t.ints([[0]]), t.ints([0, 1]), t.ints([1]),
                         1, 1)
    assert e.value.code == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_lengths_that_the_table_cannot_hold(gpu, dtype):
    """Rows behind the table's end are NaN, rows before it are not touched, and the kernels end."""
    cache, table, offsets, kv_lens, q = t.make([(200, 40), (90, 1)], 2, 4, 32, 64, dtype)
    plain = t.attend(cache, table, offsets, kv_lens, q)
    short = [r[:5] for r in table]  # 160 places: the first sequence's new tokens are places 160..199
    for window in (0, 30):
        want = t.attend(cache, table, offsets, kv_lens, q, window=window)
        out, lse = t.attend(cache, short, offsets, kv_lens, q, window=window)
        assert bool(out[:40].isnan().all()) and torch.equal(out[40], want[0][40]) and torch.equal(lse[40], want[1][40])
        big = ops.kv_attention(q, cache, t.ints(short), t.ints(offsets), t.ints([2 ** 31 - 1, 90]), 40, 200, window=window)
        assert bool(big[0][:40].isnan().all()) and torch.equal(big[0][40], want[0][40])
    assert not bool(plain[0].isnan().any())


def test_more_tokens_than_rows(gpu):
    """Offsets that go past the packed rows (a batch that was cut short): the rows that are there, and nothing else."""
    cache, table, offsets, kv_lens, q = t.make([(300, 100), (500, 120)], 2, 4, 32, 64, torch.float16)
    want = t.attend(cache, table, offsets, kv_lens, q)
    guard = torch.full((400, 8, 64), 9.0, dtype=torch.float16, device="cuda")
    lse = torch.full((400, 8), 9.0, device="cuda")
    b = 150
    ops.kv_attention(q[:b], cache, t.ints(table), t.ints(offsets), t.ints(kv_lens), 120, 500, out=guard[:b], lse=lse[:b])
    assert bool((guard[b:] == 9.0).all()) and bool((lse[b:] == 9.0).all())
    assert float((guard[:b].double() - want[0][:b].double()).norm()) <= 1e-3 * float(want[0][:b].double().norm())
