"""Linear attention token by token: one NaN or infinity among the inputs stays in its head (in v its column) and behind its
token, as in chunks."""
import pytest
import torch

from test_gpu_linear_attention import TYPES, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lengths", [[1, 1], [12, 3]])
@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "beta"])
def test_what_is_not_finite_stays_behind_its_token(gpu, name, lengths, delta, dtype):
    if name == "beta" and not delta:
        return
    n = lengths[0]
    for token in {0, n // 2, n - 1}:
        for value in (torch.nan, torch.inf):
            clean, b = (Batch(lengths, 2, 2, 64, 64, dtype, delta, seed=token) for _ in range(2))
            x = getattr(b, name)
            if x.dim() == 3:
                x[token, 1, 5] = value
            else:
                x[token, 1] = value
            want, got = clean.run(work=None), b.run(work=None)
            lost = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
            lost[token:token + 1 if name == "q" else n, 1, 5 if name == "v" else slice(None)] = True
            assert torch.equal(torch.isfinite(got), ~lost) and torch.equal(got[~lost], want[~lost])
            bad = torch.zeros(b.states.shape, dtype=torch.bool, device="cuda")
            if name == "v":
                bad[b.slots[0], 1, :, 5] = True
            elif name == "k" and not delta:
                bad[b.slots[0], 1, 5] = True
            elif name != "q":
                bad[b.slots[0], 1] = True
            assert torch.equal(torch.isfinite(b.states), ~bad) and torch.equal(b.states[~bad], clean.states[~bad])
