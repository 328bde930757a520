"""The append of more than 128 tokens: 16 tokens a workgroup, the tiles of eight blocks side by side, for every block size.

Codes and scales are equal to the plain form's, as in test_gpu_kv_cache.py."""
import random

import pytest
import torch

import test_gpu_kv_cache as t

pytestmark = pytest.mark.gpu
SIZES = [(16, 64), (32, 128), (64, 256), (128, 64), (256, 128)]


def rows(n, heads, dim, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((2, n, heads, dim), device="cuda", generator=gen) * 2).to(dtype)


def run_of(blocks, block, first, n):
    """n tokens from place `first` of the first of `blocks` (any order of ids) on."""
    return [blocks[p // block] * block + p % block for p in range(first, first + n)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [1, 3])
@pytest.mark.parametrize("block,dim", SIZES)
def test_prompts_of_several_rounds(gpu, block, dim, heads, dtype):
    """Eight blocks are a round: one and a bit, two whole ones, three and a half, begun inside a block and outside one."""
    for tokens, first in ((8 * block + 121, 0), (16 * block, block - 5), (28 * block + 7, 3), (128 + 1, block // 2)):
        n = (first + tokens - 1) // block + 1
        ids = random.Random(tokens).sample(range(n + 4), n)
        cache = t.pool(n + 4, heads, block, dim, seed=tokens)
        kv = rows(tokens, heads, dim, dtype, first)
        t.check_append(cache, kv[0], kv[1], run_of(ids, block, first, tokens))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("block,dim", SIZES)
def test_single_tokens(gpu, block, dim, dtype):
    """As many sequences, a token each in a block of its own: sixteen runs to a workgroup."""
    for tokens in (129, 256, 401):
        rng = random.Random(tokens)
        cache = t.pool(tokens, 2, block, dim, seed=tokens)
        slots = [b * block + rng.randrange(block) for b in rng.sample(range(tokens), tokens)]
        kv = rows(tokens, 2, dim, dtype, tokens)
        t.check_append(cache, kv[0], kv[1], slots)


@pytest.mark.parametrize("block,dim", SIZES)
def test_prompts_single_tokens_and_padding_in_one(gpu, block, dim):
    """Runs that begin and end anywhere in a 16-token tile, idle tokens between and behind them."""
    rng = random.Random(block)
    ids = rng.sample(range(120), 120)
    slots, at = [], 0

    def take(n):
        nonlocal at
        at += n
        return ids[at - n:at]

    for part in range(6):
        for _ in range(rng.randint(1, 9)):
            slots.append(take(1)[0] * block + rng.randrange(block))
        slots += [-1] * rng.randint(0, 5)
        first, tokens = rng.randrange(block), rng.randint(1, 5 * block)
        slots += run_of(take((first + tokens - 1) // block + 1), block, first, tokens)
        slots += [-1, 120 * block][:rng.randint(0, 2)]
    slots += [-1] * (130 if len(slots) < 129 else 7)
    cache = t.pool(120, 2, block, dim, seed=block)
    kv = rows(len(slots), 2, dim, torch.float32, block)
    t.check_append(cache, kv[0], kv[1], slots)
