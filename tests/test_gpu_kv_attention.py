"""Attention over the 8-bit key/value cache against a 64-bit form.

Tolerances.  The codes and block scales are exact in both, so what differs is
the kernel's own arithmetic.  f32 rows are computed with f32-like products and
sums throughout: relative L2 1e-5, the tolerance of this library's products.
f16 and bf16 rows: the output is rounded to the type (at most 2^-11 and 2^-8 of
a value, a rms of about a third of that), and the softmax weights may be
rounded to 11 bits before they are summed: relative L2 1e-3 and 4e-3.  One
value may be off by 40 times that of the larger of itself and the rms.  lse is
f32 in any case: its error is the scores', sums of 256 products of order one:
absolute 2e-5 (1 + |lse| / 16)."""
import math
import random

import pytest
import torch

import kv_reference as ref
from qwen35_amd import QhipError, ops

pytestmark = pytest.mark.gpu

REL = {torch.float32: 1e-5, torch.float16: 1e-3, torch.bfloat16: 4e-3}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(lens, heads, group, block, dim, dtype, seed=0, slack=2, loud=1.0):
    """A pool, a table whose unused entries are garbage, packed queries, for (kv_len, rows) of each sequence."""
    rng, gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-max(n, 0) // block) for n, _ in lens]
    blocks = sum(need) + 3
    ids = list(range(blocks))
    rng.shuffle(ids)
    width = max(need + [1]) + slack
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [rng.choice([-1, 2 ** 30, -2 ** 31, 7]) for _ in range(width - n)])
        at += n
    shape = (blocks, heads, block, dim)
    x = torch.randn((2, *shape), device="cuda", generator=gen)
    x *= torch.exp(0.5 * torch.randn((2, *shape[:2], 1, 1), device="cuda", generator=gen))
    x[0] *= loud
    scale = x.abs().amax((3, 4)) / 127
    codes = (x / scale[..., None, None]).round().to(torch.int8)
    cache = ops.KvCache(codes[0], codes[1], scale[0].contiguous(), scale[1].contiguous())
    offsets = [0]
    for _, n in lens:
        offsets.append(offsets[-1] + n)
    q = torch.randn((offsets[-1], heads * group, dim), device="cuda", generator=gen).to(dtype)
    return cache, table, offsets, [n for n, _ in lens], q


def compare(out, lse, want, want_lse, dtype):
    rel = REL[dtype]
    assert bool((out.isnan() == want.isnan()).all())
    seen = ~want.isnan()
    o, w = out.double()[seen], want[seen]
    off, norm = float((o - w).norm()), float(w.norm())
    assert off <= rel * norm, f"relative L2 {off / max(norm, 1e-300):.3g}"
    rms = norm / math.sqrt(max(w.numel(), 1))
    assert bool(((o - w).abs() <= 40 * rel * torch.clamp(w.abs(), min=rms)).all())
    assert bool((lse.isnan() == want_lse.isnan()).all()) and torch.equal(lse == -math.inf, want_lse == -math.inf)
    fine = torch.isfinite(want_lse)
    assert bool(((lse.double() - want_lse)[fine].abs() <= 2e-5 * (1 + want_lse[fine].abs() / 16)).all())


def attend(cache, table, offsets, kv_lens, q, scale=None, causal=True, window=0, work=True, **more):
    most = max([b - a for a, b in zip(offsets, offsets[1:])] + [0])
    longest = max([0] + kv_lens)
    w = ops.kv_attention_work(cache, q.shape[1], len(kv_lens), len(q), most, longest) if work else None
    got = ops.kv_attention(q, cache, ints(table), ints(offsets), ints(kv_lens), most, longest, scale, causal, window, work=w,
                           **more)
    if w is not None:
        assert not bool(w[:32768].any())  # as it was before the launch
    return got


def check(lens, heads, group, block, dim, dtype, causal=True, window=0, seed=0, scale=None, loud=1.0):
    cache, table, offsets, kv_lens, q = make(lens, heads, group, block, dim, dtype, seed, loud=loud)
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens,
                         dim ** -0.5 if scale is None else scale, causal, window)
    for work in (True, False):
        out, lse = attend(cache, table, offsets, kv_lens, q, scale, causal, window, work)
        compare(out, lse, *want, dtype)
    return cache, table, offsets, kv_lens, q, out, lse


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
#: (kv_len, rows) of each sequence: single tokens, several, prompts, prompts on a past, empty and idle rows
BATCHES = {
    "one": [(1, 1)],
    "decode": [(1, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (333, 1), (1000, 1)],
    "decode_long": [(5000, 1), (12, 1), (0, 0), (3071, 1)],
    "verify": [(5, 5), (70, 5), (131, 4), (1029, 3), (33, 2)],
    "prompt": [(1, 1), (2, 2), (31, 31), (130, 130), (257, 257)],
    "prompt_past": [(300, 77), (1031, 200), (129, 64)],
    "mixed": [(700, 1), (400, 150), (0, 0), (90, 7), (1, 1), (513, 33)],
    "empty": [(0, 1), (0, 0), (3, 5), (0, 20), (40, 1), (10, 40)],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch", sorted(BATCHES))
def test_batches(gpu, batch, dim, dtype):
    group = {64: 1, 128: 4, 256: 6}[dim]
    check(BATCHES[batch], 2, group, 64, dim, dtype, seed=dim)


@pytest.mark.parametrize("block", [16, 32, 128, 256])
@pytest.mark.parametrize("batch", ["decode", "verify", "prompt_past", "mixed", "empty"])
def test_block_sizes(gpu, batch, block):
    check(BATCHES[batch], 3, 2, block, 128, torch.float32, seed=block)
    check(BATCHES[batch], 1, 4, block, 256, torch.bfloat16, seed=block)


@pytest.mark.parametrize("heads,group", [(1, 1), (1, 3), (5, 5), (2, 8), (1, 16), (2, 17), (1, 40)])
@pytest.mark.parametrize("batch", ["decode", "verify", "mixed"])
def test_head_layouts(gpu, batch, heads, group):
    check(BATCHES[batch], heads, group, 32, 64, torch.float32, seed=group)
    check(BATCHES[batch], heads, group, 64, 128, torch.float16, seed=group)


@pytest.mark.parametrize("window", [1, 2, 16, 33, 100, 4096])
@pytest.mark.parametrize("batch", ["decode", "verify", "prompt_past", "mixed", "empty", "decode_long"])
def test_windows(gpu, batch, window):
    check(BATCHES[batch], 2, 4, 32, 128, torch.float32, window=window, seed=window)
    check(BATCHES[batch], 2, 2, 64, 64, torch.bfloat16, window=window, seed=window)


@pytest.mark.parametrize("batch", sorted(BATCHES))
def test_without_causality(gpu, batch):
    check(BATCHES[batch], 2, 4, 64, 128, torch.float32, causal=False)
    check(BATCHES[batch], 2, 3, 16, 256, torch.float16, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[(33000, 1)], [(20001, 6)], [(9000, 260)], [(2500, 2500)]])
def test_long(gpu, lens, dtype):
    check(lens, 2, 4, 64, 128, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", ["decode", "verify", "prompt_past"])
def test_sharp_and_flat_softmax(gpu, batch, dtype):
    """Scores of a few hundred (one key takes all), of zero, and of either sign of scale."""
    check(BATCHES[batch], 2, 2, 32, 128, dtype, scale=0.0)
    check(BATCHES[batch], 2, 2, 32, 128, dtype, scale=-0.1)
    cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 2, 32, 128, dtype, loud=8.0)
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 1.0)
    out, lse = attend(cache, table, offsets, kv_lens, q, 1.0)
    # scores of up to about 400, so f32 rounds them to 2^-15: e^s is that much off, twice
    assert float((out.double() - want[0]).norm()) <= (REL[dtype] + 2.0 ** -12) * float(want[0].norm())
    assert bool(torch.isfinite(lse[want[1] != -math.inf]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_query_magnitudes(gpu, dtype):
    """Queries far above and below one: the products keep their precision."""
    for size, batch in ((2.0 ** 12, "decode"), (2.0 ** -12, "decode"), (2.0 ** 12, "prompt_past"), (2.0 ** -12, "prompt_past")):
        cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 4, 64, 128, dtype)
        q = (q.float() * size).to(dtype)
        want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5 / size)
        compare(*attend(cache, table, offsets, kv_lens, q, 128 ** -0.5 / size), *want, dtype)


def test_block_scales_of_any_size(gpu):
    """Scales that differ from block to block by many orders, and blocks of zeros."""
    for batch in ("decode", "prompt_past", "mixed"):
        cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 2, 16, 128, torch.float32)
        n = cache.num_blocks
        cache.v_scale.mul_(torch.logspace(-12, 9, n, device="cuda")[torch.randperm(n, device="cuda")][:, None])
        cache.k_scale[::3] = 0
        cache.v_scale[1::5] = 0
        want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5)
        out, lse = attend(cache, table, offsets, kv_lens, q)
        assert float((out.double() - want[0]).norm()) <= 1e-5 * float(want[0].norm())
        rows = want[0].norm(dim=-1)
        assert bool(((out.double() - want[0]).norm(dim=-1) <= 4e-5 * rows + 1e-30).all())
        assert torch.equal(torch.isfinite(lse), torch.isfinite(want[1]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_within_other_tensors(gpu, dtype):
    """Queries inside a projection (a gate beside each head), outputs inside a wider row, rows at odd addresses."""
    for batch in ("decode", "mixed"):
        cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 4, 64, 128, dtype)
        plain = attend(cache, table, offsets, kv_lens, q)
        wide = torch.full((len(q), 8, 256), math.nan, dtype=dtype, device="cuda")
        wide[..., :128] = q
        out = torch.full((len(q), 2000), 5.0, dtype=dtype, device="cuda")
        rows = out[:, 100:100 + 8 * 200].reshape(len(q), 8, 200)[..., :128]
        rows = out.as_strided((len(q), 8, 128), (2000, 200, 1), 100)
        got = attend(cache, table, offsets, kv_lens, wide[..., :128], out=rows)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
        rows.fill_(5.0)
        assert bool((out == 5.0).all())
        flat = torch.empty(1 + len(q) * 8 * 129, dtype=dtype, device="cuda")
        odd = flat[1:].reshape(len(q), 8, 129)[..., :128]
        odd.copy_(q)
        to = torch.empty_like(flat)[1:].reshape(len(q), 8, 129)[..., :128]
        got = attend(cache, table, offsets, kv_lens, odd, out=to)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


def test_hidden_places_hold_anything(gpu):
    """Codes behind a sequence's end, blocks it does not own, and scales of unread blocks change nothing."""
    for batch in ("decode", "verify", "mixed", "empty"):
        cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 4, 64, 128, torch.float32)
        plain = attend(cache, table, offsets, kv_lens, q)
        used = {t for row, n in zip(table, kv_lens) for t in row[:-(-n // 64)]}
        for b in set(range(cache.num_blocks)) - used:
            cache.k[b], cache.v[b], cache.k_scale[b], cache.v_scale[b] = 127, -128, math.nan, math.inf
        for row, n in zip(table, kv_lens):
            if n % 64:
                cache.k[row[n // 64], :, n % 64:] = -128
                cache.v[row[n // 64], :, n % 64:] = 127
        got = attend(cache, table, offsets, kv_lens, q)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


@pytest.mark.parametrize("odd", [math.nan, math.inf])
@pytest.mark.parametrize("lens", [[(200, 1), (150, 1)], [(200, 5), (150, 3)], [(200, 140), (150, 150)], [(900, 300), (700, 1)]])
def test_poisoned_blocks_reach_their_rows_only(gpu, lens, odd):
    """A value scale that is no number, in the second block of the first sequence, second head."""
    cache, table, offsets, kv_lens, q = make(lens, 2, 2, 64, 128, torch.float32)
    plain = attend(cache, table, offsets, kv_lens, q)
    cache.v_scale[table[0][1], 1] = odd
    out, lse = attend(cache, table, offsets, kv_lens, q)
    first = lens[0][0] - lens[0][1]
    hit = torch.zeros((len(q), 4), dtype=torch.bool, device="cuda")
    hit[max(0, 64 - first):lens[0][1], 2:] = True
    assert torch.equal(out.isnan().all(-1), hit) and torch.equal(out.isnan().any(-1), hit)
    assert torch.equal(out[~hit], plain[0][~hit]) and torch.equal(lse, plain[1])
    cache.v_scale[table[0][1], 1] = 0.01
    cache.k_scale[table[0][1], 1] = math.nan
    out, lse = attend(cache, table, offsets, kv_lens, q)
    assert torch.equal(out.isnan().all(-1), hit) and torch.equal(lse.isnan(), hit)


def test_entries_outside_the_pool_make_their_rows_nan(gpu):
    lens = [(100, 1), (300, 130), (64, 1)]
    cache, table, offsets, kv_lens, q = make(lens, 2, 2, 64, 128, torch.float32)
    plain = attend(cache, table, offsets, kv_lens, q)
    for bad in (-1, cache.num_blocks, 2 ** 31 - 1, -2 ** 31):
        t = [list(r) for r in table]
        t[0][0] = bad       # the first sequence's only row needs it
        t[1][4] = bad       # places 256.. of the second: rows that see them
        out, lse = attend(cache, t, offsets, kv_lens, q)
        hit = torch.zeros(len(q), dtype=torch.bool, device="cuda")
        hit[0] = True
        hit[1 + 256 - 170:131] = True
        assert torch.equal(out.isnan().all((1, 2)), hit) and torch.equal(out.isnan().any((1, 2)), hit)
        assert torch.equal(out[~hit], plain[0][~hit]) and torch.equal(lse[~hit], plain[1][~hit])
    # a table with too few columns for the lengths
    out, _ = attend(cache, [r[:1] for r in table], offsets, kv_lens, q)
    assert bool(out[0].isnan().all()) and bool(out[1:131].isnan().all()) and torch.equal(out[131], plain[0][131])


def test_nan_queries_stay_in_their_rows(gpu):
    for batch in ("decode", "verify", "prompt_past"):
        cache, table, offsets, kv_lens, q = make(BATCHES[batch], 2, 2, 64, 128, torch.float32)
        plain = attend(cache, table, offsets, kv_lens, q)
        q[::3, 1, 5] = math.nan
        q[1::3, 2, 9] = math.inf
        out, lse = attend(cache, table, offsets, kv_lens, q)
        hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
        hit[::3, 1], hit[1::3, 2] = True, True
        assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], plain[0][~hit]) and torch.equal(lse[~hit], plain[1][~hit])


def test_the_same_results_on_every_run(gpu):
    for lens in ([(9000, 1)], [(3000, 1), (8000, 1), (17, 1)], [(4000, 4)], [(2100, 300)]):
        cache, table, offsets, kv_lens, q = make(lens, 2, 4, 64, 128, torch.float32)
        first = attend(cache, table, offsets, kv_lens, q)
        for _ in range(5):
            again = attend(cache, table, offsets, kv_lens, q)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_bounds_above_the_lengths(gpu):
    """max_new and max_kv are bounds: larger ones, and padding behind the packed rows, change only what is cut where."""
    cache, table, offsets, kv_lens, q = make(BATCHES["mixed"], 2, 4, 64, 128, torch.float32)
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5)
    padded = torch.cat([q, torch.full((37, 8, 128), math.nan, device="cuda")])
    work = ops.kv_attention_work(cache, 8, len(kv_lens), len(padded), 500, 40000)
    out, lse = torch.full_like(padded, 3.0), torch.full((len(padded), 8), 3.0, device="cuda")
    ops.kv_attention(padded, cache, ints(table), ints(offsets), ints(kv_lens), 500, 40000, work=work, out=out, lse=lse)
    compare(out[:len(q)], lse[:len(q)], *want, torch.float32)
    assert bool((out[len(q):] == 3.0).all()) and bool((lse[len(q):] == 3.0).all())


def test_small_workspace_is_no_error(gpu):
    cache, table, offsets, kv_lens, q = make([(9000, 1)], 2, 4, 64, 128, torch.float32)
    plain = attend(cache, table, offsets, kv_lens, q, work=False)
    work = torch.zeros(64, dtype=torch.uint8, device="cuda")
    got = ops.kv_attention(q, cache, ints(table), ints(offsets), ints(kv_lens), 1, 9000, work=work)
    assert torch.equal(got[0], plain[0]) and not bool(work.any())


def test_on_another_stream_and_in_a_graph(gpu):
    """A decode step -- tables, append, attention -- captured once and replayed as the sequences grow."""
    nseq, heads, group, block, dim, steps = 3, 2, 4, 16, 128, 40
    cache = ops.KvCache.empty(64, heads, block, dim)
    mirror = ops.KvCache.empty(64, heads, block, dim)
    table = torch.full((nseq, 20), -1, dtype=torch.int32, device="cuda")
    free = ints(list(range(63, -1, -1)))
    cached, taken, new = ints([0, 0, 0]), ints([0]), ints([1] * nseq)
    step = ops.KvStep(nseq, nseq)
    qkv = torch.zeros((nseq, heads * (group + 2), dim), device="cuda")
    work = ops.kv_attention_work(cache, heads * group, nseq, nseq, 1, 300)
    out, lse = torch.empty((nseq, heads * group, dim), device="cuda"), torch.empty((nseq, heads * group), device="cuda")

    def once():
        ops.kv_tables(cached, new, free, table, block, step, taken=taken)
        ops.kv_append(cache, qkv[:, heads * group:heads * (group + 1)], qkv[:, heads * (group + 1):], step.slots)
        ops.kv_attention(qkv[:, :heads * group], cache, table, step.offsets, step.kv_lens, 1, 300, work=work, out=out, lse=lse)
        cached.copy_(step.kv_lens)
        taken.copy_(step.taken)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        once()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    for t in (cached, taken, cache.k, cache.v, cache.k_scale, cache.v_scale):
        t.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once()
    torch.cuda.synchronize()
    table.fill_(-1)
    gen = torch.Generator(device="cuda").manual_seed(4)
    for i in range(steps):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        slots = step.slots.tolist()
        for name, x in (("k", qkv[:, heads * group:heads * (group + 1)]), ("v", qkv[:, heads * (group + 1):])):
            codes, scales = ref.append(getattr(mirror, name), getattr(mirror, name + "_scale"), x, slots)
            getattr(mirror, name).copy_(codes)
            getattr(mirror, name + "_scale").copy_(scales)
        assert torch.equal(cache.k, mirror.k) and torch.equal(cache.v_scale, mirror.v_scale)
        want = ref.attention(qkv[:, :heads * group], mirror.k, mirror.v, mirror.k_scale, mirror.v_scale, table.tolist(),
                             [0, 1, 2, 3], [i + 1] * nseq, dim ** -0.5)
        compare(out, lse, *want, torch.float32)
    assert int(taken) == nseq * -(-steps // block)


def test_pool_past_32_bit_offsets(gpu):
    """Blocks that lie behind 4 GiB of codes."""
    heads, group, block, dim = 4, 2, 256, 256
    lens = [(700, 1), (600, 40)]
    cache, table, offsets, kv_lens, q = make(lens, heads, group, block, dim, torch.float32)
    n, far = cache.num_blocks, 16500
    big = ops.KvCache(*(torch.zeros((far + n, *t.shape[1:]), dtype=t.dtype, device="cuda")
                        for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    for a, b in ((big.k, cache.k), (big.v, cache.v), (big.k_scale, cache.k_scale), (big.v_scale, cache.v_scale)):
        a[far:] = b
    want = attend(cache, table, offsets, kv_lens, q)
    moved = [[t + far if 0 <= t < n else t for t in row] for row in table]
    got = attend(big, moved, offsets, kv_lens, q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(gpu):
    cache, table, offsets, kv_lens, q = make([(40, 2), (70, 1)], 2, 2, 32, 64, torch.float32)
    args = (cache, ints(table), ints(offsets), ints(kv_lens), 2, 70)
    for bad in (q.double(), q[..., :32], q.transpose(0, 2), q[0]):
        with pytest.raises(ValueError):
            ops.kv_attention(bad, *args)
    with pytest.raises(ValueError):
        ops.kv_attention(q, cache, ints(table)[:1], ints(offsets), ints(kv_lens), 2, 70)
    with pytest.raises(ValueError):
        ops.kv_attention(q, cache, ints(table), ints(offsets).long(), ints(kv_lens), 2, 70)
    with pytest.raises(ValueError):
        ops.kv_attention(q, *args, out=torch.empty_like(q).half())
    with pytest.raises(ValueError):
        ops.kv_attention(q, *args, lse=torch.empty((3, 3), device="cuda"))
    with pytest.raises(ValueError):
        ops.kv_attention_work(cache, 3, 2, 3, 2, 70)
    for kw in ({"causal": False, "window": 5}, {"window": -1}):
        with pytest.raises(QhipError) as e:
            ops.kv_attention(q, *args, **kw)
        assert e.value.code == 1
    with pytest.raises(QhipError) as e:
        ops.kv_attention(torch.randn((3, 3, 64), device="cuda"), *args)  # three query heads over two key heads
    assert e.value.code == 1
    odd = ops.KvCache.empty(6, 2, 32, 96)
    with pytest.raises(QhipError) as e:
        ops.kv_attention(torch.randn((3, 4, 96), device="cuda"), odd, *args[1:])
    assert e.value.code == -1  # declined: no kernel for this head width
