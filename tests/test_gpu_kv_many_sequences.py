"""Attention of batches of more than 64 sequences, whose plan goes by groups of 64.

Tolerances as in test_gpu_kv_attention.py: relative L2 1e-5, 1e-3 and 4e-3."""
import random

import pytest
import torch

import kv_reference as ref
import test_gpu_kv_attention as t

pytestmark = pytest.mark.gpu


def lengths(n, lo, hi, new, seed):
    """(kv_len, rows) of n sequences; some idle, a few much longer than the others."""
    rng = random.Random(seed)
    out = []
    for i in range(n):
        length = rng.randint(lo, hi) * (9 if i % 41 == 7 else 1)
        out.append((0, 0) if i % 23 == 5 else (length, min(length, rng.choice(new))))
    return out


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("nseq", [65, 128, 129, 300, 1000])
def test_decodes(gpu, nseq, dtype):
    t.check(lengths(nseq, 1, 200, [1], nseq), 2, 4, 32, 128, dtype, seed=nseq)


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_cut_among_many(gpu, dim, dtype):
    """Long sequences in the second and third group of 64, cut into chunks beside short ones that are not."""
    lens = lengths(150, 1, 60, [1], dim)
    lens[100], lens[149], lens[64] = (9000, 1), (20000, 1), (5000, 3)
    t.check(lens, 1, 4, 64, dim, dtype, seed=dim)
    t.check(lens, 1, 4, 64, dim, dtype, seed=dim, window=3000)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 8), (128, 2, 8), (256, 3, 8)])
def test_prompts_beside_decodes(gpu, dim, heads, group, dtype):
    """Both kernels in one batch, the prompts in different groups of 64."""
    lens = lengths(140, 1, 300, [1, 1, 2], dim)
    lens[3], lens[70], lens[139] = (6000, 1100), (3000, 700), (2500, 900)
    t.check(lens, heads, group, 64, dim, dtype, seed=dim)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_drafts(gpu, dtype):
    t.check(lengths(200, 5, 400, [2, 5, 5, 9], 3), 2, 6, 32, 256, dtype)


def test_the_same_bits_without_the_others(gpu):
    """A sequence's rows do not depend on what stands beside it where nothing is cut."""
    lens = lengths(180, 1, 200, [1, 3], 11)
    cache, table, offsets, kv_lens, q = t.make(lens, 2, 4, 32, 128, torch.float32, seed=1)
    out, lse = t.attend(cache, table, offsets, kv_lens, q, work=False)
    want = ref.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, offsets, kv_lens, 128 ** -0.5)
    t.compare(out, lse, *want, torch.float32)
    for i in (0, 63, 64, 100, 127, 128, 179):
        a, b = offsets[i], offsets[i + 1]
        if a == b:
            continue
        one, one_lse = t.attend(cache, [table[i]], [0, b - a], [kv_lens[i]], q[a:b], work=False)
        assert torch.equal(one, out[a:b]) and torch.equal(one_lse, lse[a:b])
