"""Linear attention whose inputs are finite and whose updates are not: the tokens before the first update past f32 are as
they are token by token, in chunks too."""
import pytest
import torch

import layer_reference as ref
from qwen35_amd import ops
from test_gpu_linear_attention import TYPES, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("token", [0, 3, 20, 37, 63, 64, 99])
def test_an_update_past_f32(gpu, token, dk, dtype):
    """beta (v - k S) = 1e38 * 100 at one token of one head: R = v - k S and the token's row of T = beta are finite."""
    def batch():
        return Batch([100, 30], 2, 2, dk, 64, dtype, seed=token)

    clean, b, alone = batch(), batch(), batch()
    for x in (b, alone):
        x.beta[token, 1], x.v[token, 1] = 1e38, 100.0
    want, got, steps = clean.run(), b.run(), alone.run(work=None)
    lost = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    lost[token:100, 1] = True
    assert not bool(torch.isfinite(steps[lost]).any()) and bool(torch.isfinite(steps[~lost]).all())
    assert torch.equal(torch.isfinite(got), ~lost)
    assert torch.equal(got[~lost], want[~lost])  # (the same sums, whatever comes behind)
    bad = torch.zeros(b.states.shape, dtype=torch.bool, device="cuda")
    bad[b.slots[0], 1] = True
    assert torch.equal(torch.isfinite(b.states), ~bad) and torch.equal(b.states[~bad], clean.states[~bad])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("grows,first_lost", [
    # each update 1e9 times the one before: the block of the inverse on the diagonal overflows, in its fifth row
    ({16 + i: 1e9 for i in range(16)}, 20),
    # up to 1e36 at the end of a block of 16, then next to nothing, then past f32 in the middle of the next block: the sum
    # of L_ik X_kj overflows there
    ({**{12 + i: 1e9 for i in range(4)}, **{16 + i: 2.0 ** -40 for i in range(8)}, 24: 1e15}, 24),
    ({**{28 + i: 1e9 for i in range(4)}, **{32 + i: 2.0 ** -40 for i in range(21)}, 53: 1e15}, 53),
])
def test_updates_that_grow_past_f32(gpu, grows, first_lost, dk, dtype):
    """All keys alike, no decay, beta k^2 as given (0 elsewhere): k S is multiplied by 1 - beta k^2 each token.

    Tolerance: one term outweighs the others by 1e9, and it goes through at most 64 roundings of 2^-24; the output's
    type adds half its step."""
    n = 90
    k = torch.ones((n, 1, dk), device="cuda", dtype=dtype)
    q, v = k / dk, (1 + torch.rand((n, 1, 64), device="cuda")).to(dtype)
    beta, decay = torch.zeros((n, 1), device="cuda"), torch.zeros((n, 1), device="cuda")
    for t, x in grows.items():
        beta[t] = x / dk
    slots, offsets = torch.tensor([0], device="cuda", dtype=torch.int32), torch.tensor([0, n], device="cuda", dtype=torch.int32)
    source = torch.tensor([-1], device="cuda", dtype=torch.int32)
    states = torch.zeros((1, 1, dk, 64), device="cuda")
    want, _ = ref.linear_attention(q, k, v, decay, beta, states, [0], [0, n], [-1], 1.0)
    own = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    bound = want.abs() * (64 * 2.0 ** -24 + own * (1 + 2.0 ** -10))
    for work in (None, ops.linear_attention_work(states, q, 1, n)):
        states.zero_()
        got = ops.linear_attention(q, k, v, decay, states, slots, offsets, n, beta=beta, source=source, scale=1.0, work=work)
        good = torch.isfinite(got).all(-1)[:, 0]
        assert bool(good[:first_lost].all()) and not bool(torch.isfinite(got[first_lost:]).any())
        assert bool(((got.double() - want).abs() <= bound)[:first_lost].all())
        assert not bool(torch.isfinite(states).any())
