"""The serving example: ragged prompts, a late prompt beside single tokens, single tokens.

Tolerance: codes of 8 bits relative to a block's largest value (about 4 to 5 deviations of its 64 x 256 values) have an
error of 5 / 127 / sqrt(12) = 1.1% of a deviation.  A block that grows token by token is rounded anew at each new
maximum, a few times more: 3% of a deviation at most.  Scores are of deviation one, so keys and values each move an
output by at most that: 6% together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kv_heads", [(256, 4), (128, 2), (64, 16)])
def test_outputs_stay_near_those_of_f32_keys_and_values(gpu, dim, kv_heads):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv_serving.py")
    spec = importlib.util.spec_from_file_location("kv_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    far, _ = example.run(dim=dim, kv_heads=kv_heads, decode=4)
    assert len(far) == 6 and all(0 < d < 0.06 for d in far), far
