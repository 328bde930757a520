"""Attention over the 8-bit cache where a row sees very many keys alike.

One key scores higher than all others, which are alike, so that each adds the same weight: a running f32 sum of them
rounds the same way each time, and its error grows with the number of additions instead of its square root.  Values that
are alike too do the same to the outputs.

Tolerances as in test_gpu_kv_attention.py, of each row by itself: relative L2 1e-5, 1e-3 and 4e-3, lse 2e-5 (1 + |lse| /
16).  Of f32 rows that leaves (the products being good to 22 bits) some 150 additions each off by at most 2^-24 of a sum
that is half grown on average, for the weights and the outputs alike."""
import math

import pytest
import torch

import test_gpu_kv_attention as t
from qwen35_amd import ops

pytestmark = pytest.mark.gpu


def attend_alike(dim, tokens, group, keys, dtype, values, work):
    """(out, lse) and the same in 64 bits, of `tokens` causal rows at the end of one sequence."""
    block, gen = 256, torch.Generator(device="cuda").manual_seed(dim + tokens)
    blocks = -(-keys // block)
    sign = torch.where(torch.rand(dim, device="cuda", generator=gen) < 0.5, -1, 1)
    k = (64 * sign).to(torch.int8).expand(blocks, 1, block, dim).contiguous()
    k[0, 0, 0] = (127 * sign).to(torch.int8)
    if values == "alike":
        v = torch.randint(40, 128, (dim,), device="cuda", generator=gen).to(torch.int8).expand(k.shape).contiguous()
    else:
        v = torch.randint(-127, 128, k.shape, device="cuda", generator=gen).to(torch.int8)
    scale = torch.full((blocks, 1), 1 / 64, device="cuda")
    cache = ops.KvCache(k, v, scale, scale.clone())
    # a row's weights of the others: from 1 down to e^-8
    q = (8 * torch.rand((tokens, group, 1), device="cuda", generator=gen) * sign / math.sqrt(dim)).to(dtype)
    other = q.double() @ sign.double() / math.sqrt(dim)
    top = other * (127 / 64)
    seen = keys - tokens + torch.arange(tokens, device="cuda")  # keys of the others
    x = v.double().reshape(-1, dim)[:keys] / 64
    rest = (x.cumsum(0) - x[0])[seen][:, None]
    w = torch.exp(other - top)
    total = 1 + w * seen[:, None]
    want = (x[0] + w[..., None] * rest) / total[..., None], top + total.log()
    work = ops.kv_attention_work(cache, group, 1, tokens, tokens, keys) if work else None
    got = ops.kv_attention(q, cache, t.ints([list(range(blocks))]), t.ints([0, tokens]), t.ints([keys]), tokens, keys, work=work)
    return got, want


#: rows of a workgroup: 16 (cut, and uncut), 32 (pairs, and 256 dimensions), 64; all uncut from the second on
ROWS = [(64, 4, 4, True), (128, 4, 4, False), (256, 4, 4, False), (64, 520, 16, False), (128, 520, 16, True), (256, 520, 16, True),
        (64, 2520, 16, True), (128, 2520, 16, True)]


@pytest.mark.parametrize("dtype", t.DTYPES)
@pytest.mark.parametrize("values", ["alike", "any"])
@pytest.mark.parametrize("dim,tokens,group,work", ROWS)
def test_many_keys_alike(gpu, dim, tokens, group, work, values, dtype):
    (out, lse), (want, want_lse) = attend_alike(dim, tokens, group, 131072, dtype, values, work)
    far = (out.double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(far.max()) <= t.REL[dtype]
    assert bool(((lse.double() - want_lse).abs() <= 2e-5 * (1 + want_lse.abs() / 16)).all())
