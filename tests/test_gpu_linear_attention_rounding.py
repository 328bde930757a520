"""Linear attention in chunks: outputs of 16-bit rows are rounded once, from sums that are good to f32.

Tolerance: an output may be off by half a step of its type, and before that rounding by what test_gpu_linear_attention
allows f32 sums, 4 * sqrt(n + key_dim) * 2^-24, here of the largest output of its head, value by value."""
import math

import pytest
import torch

from test_gpu_linear_attention import Batch

pytestmark = pytest.mark.gpu


def half_step(x, dtype):
    _, exponent = torch.frexp(x.abs().clamp(min=torch.finfo(dtype).smallest_normal))
    return torch.ldexp(torch.full_like(x, torch.finfo(dtype).eps / 2), exponent - 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("k_heads,v_heads,dk,dv", [(2, 2, 64, 128), (1, 2, 128, 128)])
@pytest.mark.parametrize("lengths", [[40], [64, 65], [900, 1, 130]])
def test_one_rounding(gpu, dtype, delta, k_heads, v_heads, dk, dv, lengths):
    b = Batch(lengths, k_heads, v_heads, dk, dv, dtype, delta, seed=dk)
    want, _ = b.want()
    got = b.run().double()
    far = (got - want).abs() - half_step(torch.maximum(got.abs(), want.abs()), dtype)
    bound = 4 * math.sqrt(max(lengths) + dk) * 2.0 ** -24 * want.abs().amax((0, 2))
    assert bool((far.amax((0, 2)) <= bound).all()), (far.amax((0, 2)) / bound).tolist()
