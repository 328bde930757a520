"""Linear attention of padded batches: which form a sequence takes goes by its own tokens, not by the rows of the batch."""
import pytest
import torch

from test_gpu_linear_attention import TYPES, Batch

pytestmark = pytest.mark.gpu


def padded(lengths, each, extra, dtype, delta):
    """Rows for `each` tokens of every sequence, and `extra` more."""
    b = Batch(lengths, 2, 4, 128, 64, dtype, delta, pad=each * len(lengths) + extra - sum(lengths))
    b.max_new = each
    return b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lengths", [[1], [16], [1] * 9, [3, 0, 16, 1]])
def test_short_sequences_go_token_by_token(gpu, dtype, delta, lengths):
    """Steps captured with rows for prompts of 64 tokens run short sequences: the bits of the form without a workspace."""
    one = padded(lengths, 64, 0, dtype, delta)
    want, states = one.run(work=None, out=torch.zeros_like(one.v)), one.states
    for extra in (0, 1):
        b = padded(lengths, 64, extra, dtype, delta)
        for name in ("q", "k", "v", "log_decay", "beta"):  # (other rows in all give other random numbers)
            x, y = getattr(b, name), getattr(one, name)
            if x is not None:
                x[:len(y)] = y
        b.states = padded(lengths, 64, 0, dtype, delta).states
        b.slots = one.slots
        assert b.work() is not None
        got = b.run(out=torch.zeros_like(b.v))
        assert torch.equal(got[:len(want)], want) and torch.equal(b.states, states)
        assert bool((got[sum(lengths):] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_short_and_long_ones(gpu, dtype):
    """Both forms in one padded batch, against 64 bits."""
    padded([1, 64, 0, 40, 16, 17, 2], 64, 0, dtype, True).check()
