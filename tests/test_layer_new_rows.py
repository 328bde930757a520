"""Outputs that the operators on rows make themselves, of inputs whose rows overlap."""
import pytest
import torch

from qwen35_amd import ops


def windows(tokens, heads, dim, device="cpu"):
    """Every head begins one value behind the one before it, every token `heads` behind."""
    x = torch.randn(tokens * heads + dim, device=device, generator=torch.Generator(device=device).manual_seed(1))
    return x.as_strided((tokens, heads, dim), (heads, 1, 1))


@pytest.mark.parametrize("shape", [(3, 31, 64), (4, 1, 64), (1, 5, 8), (2, 3, 1)])
def test_a_new_output_has_its_rows_side_by_side(shape):
    for x in (windows(*shape), windows(*shape).transpose(0, 1), torch.zeros(shape[2]).expand(shape), torch.zeros(shape)):
        out, rows = ops._new_rows(x.shape, x)
        assert out.shape == x.shape and (out.stride(2) == 1 or out.shape[2] == 1) and out.dtype == x.dtype
        assert (rows.at, rows.token_stride, rows.head_stride) == (out.data_ptr(), *out.stride()[:2])
        places = (torch.arange(x.shape[0])[:, None, None] * rows.token_stride + torch.arange(x.shape[1])[:, None] * rows.head_stride
                  + torch.arange(x.shape[2]))
        assert len(places.unique()) == places.numel()


@pytest.mark.gpu
def test_windows(gpu):
    """Inputs that are only read may overlap, with an output given or not."""
    x = windows(3, 31, 64, "cuda")
    want = ops.rms_norm(x.contiguous(), None, 1e-6)
    assert torch.equal(ops.rms_norm(x, None, 1e-6), want)
    flat = torch.randn(300, device="cuda").unfold(0, 64, 1)
    assert torch.equal(ops.rms_norm(flat, None, 1e-6), ops.rms_norm(flat.contiguous(), None, 1e-6))
    at, table = torch.arange(3, dtype=torch.int32, device="cuda"), ops.RopeTable(64)
    q, k = ops.rope(x, x, at, table)
    assert torch.equal(q, ops.rope(x.contiguous(), None, at, table)[0]) and torch.equal(k, q)
    n = torch.full((3, 31), -0.1, device="cuda")
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    outs = [ops.linear_attention(y, y, y, n, torch.zeros((1, 31, 64, 64), device="cuda"), ints(0), ints(0, 3), 3) for y in (x, x.contiguous())]
    assert torch.equal(*outs)
