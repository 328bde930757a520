"""Root-mean-square norms against 64 bits.

Tolerance: h is one f32 sum (the same here), r = 1 / sqrt(..) is rounded once and two products follow: 3 roundings of
2^-24, relative.  A gate adds expf (at most 2 units in the last place, 2^-22), the sum 1 + e, the quotient and a product:
in all below 11 * 2^-24.  The output's type adds half its step."""
import pytest
import torch

import layer_reference as ref
from qwen35_amd import ops

pytestmark = pytest.mark.gpu
EPS = 1e-6
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rows(gen, dtype, *shape, loud=4.0):
    x = torch.randn(shape, device="cuda", generator=gen)
    x[..., ::7] *= loud
    return x.to(dtype)


def near(got, want, roundings):
    far = (got.double() - want).abs()
    bound = want.abs() * (roundings * U + (torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0)) * (1 + 2 ** -10)
    assert bool((far <= bound + (1e-30 if got.dtype == torch.float32 else torch.finfo(got.dtype).smallest_normal * 2 ** -7)).all()), float((far - bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 1), (3, 1, 7), (2, 3, 8), (5, 2, 31), (1, 1, 2560), (33, 16, 128), (7, 3, 96),
                                              (4, 5, 512), (3, 1, 513), (9, 1, 1000), (2, 2, 2049), (3, 1, 4100), (2, 1, 8192),
                                              (2, 1, 9001), (3, 1, 16384), (2, 1, 16385), (1, 1, 40001), (300, 1, 1024)])
@pytest.mark.parametrize("residual,gate", [(False, False), (True, False), (True, True)])
def test_rows(gpu, dtype, tokens, heads, dim, residual, gate):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    shape = (tokens, heads, dim) if heads > 1 else (tokens, dim)
    x, w = rows(gen, dtype, *shape), 1 + rows(gen, torch.float32, dim, loud=1.0) / 5
    r = rows(gen, dtype, *shape) if residual else None
    g = rows(gen, dtype, *shape) if gate else None
    want, h = ref.rms_norm(x, w, EPS, r, g)
    out = ops.rms_norm(x, w, EPS, residual=r, gate=g)
    near(out, want, 11 if gate else 3)
    if residual:
        assert torch.equal(r, h.float().to(dtype))
    assert torch.equal(ops.rms_norm(x, None, EPS), ops.rms_norm(x, torch.ones_like(w), EPS))


@pytest.mark.parametrize("ttype", [8, 12])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 256), (3, 1, 512), (5, 1, 2560), (4, 1, 5120), (2, 1, 9728), (2, 1, 16640),
                                              (7, 16, 128), (3, 4, 64), (5, 2, 256), (2, 32, 8), (3, 3, 512), (2, 2, 1024)])
def test_codes_are_those_of_the_quantizers(gpu, ttype, dtype, tokens, heads, dim):
    gen = torch.Generator(device="cuda").manual_seed(dim + ttype)
    shape = (tokens, heads, dim) if heads > 1 else (tokens, dim)
    x, r, w = rows(gen, dtype, *shape), rows(gen, dtype, *shape), 1 + rows(gen, torch.float32, dim, loud=1.0) / 5
    g = rows(gen, dtype, *shape)
    # the f32 y, which rows of f32 give as they are
    y = ops.rms_norm(x.float(), w, EPS, residual=r.float().clone(), gate=g.float())
    out = torch.empty_like(x)
    xq = ops.rms_norm_quantize(ttype, x, w, EPS, residual=r.clone(), gate=g, out=out)
    assert torch.equal(xq, ops.quantize_act(ttype, y.reshape(tokens, -1)))
    assert torch.equal(out, y.to(dtype))
    again = ops.rms_norm_quantize(ttype, x, w, EPS, residual=r, gate=g, xq=torch.empty_like(xq))
    assert torch.equal(again, xq)


def test_codes_of_32_values_of_rows_that_leave_lanes_idle(gpu):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = rows(gen, torch.float32, 5, 3, 96)
    assert torch.equal(ops.rms_norm_quantize(8, x, None, EPS), ops.quantize_act(8, ops.rms_norm(x, None, EPS).reshape(5, -1)))


def test_zeros_infinities_and_nan(gpu):
    x = torch.randn((6, 640), device="cuda")
    x[1], x[2, 5], x[3, 7], x[4] = 0, torch.nan, torch.inf, 1e30
    out = ops.rms_norm(x, None, EPS)
    assert bool((out[1] == 0).all()) and bool(out[2].isnan().all())
    assert bool(out[3, 7].isnan()) and bool((out[3].nan_to_num() == 0).all())  # 1 / sqrt(inf) = 0, inf * 0
    near(out[[0, 4, 5]], ref.rms_norm(x[[0, 4, 5]], None, EPS)[0], 3)  # squares beyond f32 among them
    q = ops.rms_norm_quantize(8, x, None, EPS)
    assert torch.equal(q, ops.quantize_act(8, out))


@pytest.mark.parametrize("dtype", TYPES)
def test_columns_of_wider_rows_in_place(gpu, dtype):
    """x, the gate and the output inside one projection's rows, at odd elements; heads behind tokens."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = rows(gen, dtype, 9, 1003)
    keep = wide.clone()
    x, g = wide[:, 1:1 + 384].view(9, 3, 128), wide[:, 501:501 + 384].view(9, 3, 128)
    want, _ = ref.rms_norm(x.clone(), None, EPS, gate=g.clone())
    assert ops.rms_norm(x, None, EPS, gate=g, out=x) is x
    near(x, want, 11)
    keep[:, 1:385] = wide[:, 1:385]
    assert torch.equal(keep, wide)
    y = rows(gen, dtype, 5, 9, 64).transpose(0, 1)  # [tokens 9, heads 5, 64], a head's tokens side by side
    out = torch.empty((5, 9, 64), dtype=dtype, device="cuda").transpose(0, 1)
    near(ops.rms_norm(y, None, EPS, out=out), ref.rms_norm(y, None, EPS)[0], 3)


def test_the_length_of_a_head(gpu):
    """x / sqrt(sum x^2 + eps) by weight and eps."""
    x = torch.randn((11, 4, 128), device="cuda")
    w = torch.full((128,), 128 ** -0.5, device="cuda")
    want = x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + EPS)
    got = ops.rms_norm(x, w, EPS / 128)
    assert float(((got.double() - want) / want).abs().max()) <= 5 * U * (1 + 2 ** -10)  # 3 roundings, the weight's and eps'


def test_no_tokens(gpu):
    x = torch.empty((0, 512), device="cuda")
    assert ops.rms_norm(x, None, EPS).shape == (0, 512) and ops.rms_norm_quantize(8, x, None, EPS).shape == (0, 544)


def test_refusals(gpu):
    x, w = torch.randn((4, 512), device="cuda"), torch.ones(512, device="cuda")
    for kw in (dict(weight=w.half()), dict(weight=w[:-1]), dict(weight=w.cpu()), dict(residual=x.half()), dict(residual=x[:3]),
               dict(gate=x[:, :-1]), dict(out=x.t().contiguous().t()), dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]),
               dict(out=torch.empty((4, 512), dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            ops.rms_norm(**{**dict(x=x, weight=w, eps=EPS), **kw})
    wide = torch.randn((4, 1024), device="cuda")
    for kw in (dict(residual=x), dict(out=wide[:, 256:768], x=wide[:, :512]), dict(residual=wide[:, 256:768], x=wide[:, :512]),
               dict(eps=-1.0), dict(eps=float("nan")), dict(out=w.expand(4, 512)), dict(residual=torch.zeros((1, 512), device="cuda").expand(4, 512))):
        with pytest.raises(RuntimeError):
            ops.rms_norm(**{**dict(x=x, weight=w, eps=EPS), **kw})
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(12, x[:, :500], None, EPS)
    with pytest.raises(RuntimeError):  # blocks of 256 over heads of 96
        ops.rms_norm_quantize(12, torch.randn((2, 8, 96), device="cuda"), None, EPS)
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(8, x, None, EPS, xq=torch.empty((4, 512), dtype=torch.uint8, device="cuda"))


def test_in_a_graph_on_another_stream(gpu):
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, r, w = rows(gen, torch.float32, 64, 2560), rows(gen, torch.float32, 64, 2560), torch.ones(2560, device="cuda")
    xq, r0 = torch.empty((64, 2720), dtype=torch.uint8, device="cuda"), r.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.rms_norm_quantize(8, x, w, EPS, residual=r, xq=xq)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.rms_norm_quantize(8, x, w, EPS, residual=r, xq=xq)
    torch.cuda.synchronize()
    for _ in range(3):
        r.copy_(r0)
        x.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.rms_norm_quantize(8, x, w, EPS, residual=r0.clone())
        assert torch.equal(xq, want) and torch.equal(r, r0 + x)


@pytest.mark.parametrize("dim", [257, 513])
def test_more_rows_than_a_launch_takes(gpu, dim):
    """A grid holds fewer than 2^32 threads: rows before, at and behind the place where the next launch begins."""
    tokens = 2 ** 21 * (4 if dim <= 512 else 1) + 7  # (four rows a workgroup of 256, and one)
    gen = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.zeros((tokens, dim), device="cuda", dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 5000, tokens - 12, tokens - 8, tokens - 7, tokens - 6, tokens - 1], device="cuda")
    x[some] = rows(gen, torch.bfloat16, len(some), dim)
    w = 1 + rows(gen, torch.float32, dim, loud=1.0) / 5
    out = ops.rms_norm(x, w, EPS, out=torch.full_like(x, 7.0))
    near(out[some], ref.rms_norm(x[some], w, EPS)[0], 3)
    assert int((out == 0).all(-1).sum()) == tokens - len(some)


@pytest.mark.parametrize("tokens", [1, 5])
def test_parts_of_one_array_s_heads(gpu, tokens):
    """Values and gates side by side in each head: the norm in the values' place."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    both = rows(gen, torch.float32, tokens, 4, 2, 64)
    w, x, g = torch.ones(64, device="cuda"), both[:, :, 0], both[:, :, 1]
    want, gates = ref.rms_norm(x, w, EPS, None, g)[0], g.clone()
    near(ops.rms_norm(x, w, EPS, gate=g, out=x), want, 11)
    assert torch.equal(g, gates)
    with pytest.raises(RuntimeError):  # one value into the gates
        ops.rms_norm(x, w, EPS, gate=g, out=both.view(tokens, 4, 128)[:, :, 1:65])
    k = rows(gen, torch.float32, tokens + 3, 4, 64)[:tokens]
    with pytest.raises(ValueError):
        ops.rms_norm(k[:1, :1, :1].expand(2 ** 31, 1, 1), None, EPS, out=k)
