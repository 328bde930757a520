"""Rotary positions against 64 bits.

Tolerance, relative to gain (|a| + |b|) of a pair: the turn is rounded to 2^-33 turns (7e-10 rad), turned into at most
pi / 4 rad with two roundings, the Taylor sums leave out 2e-9 and round twice: cosine and sine are off by at most 4 * 2^-24,
the gain and the two products add 3 * 2^-24; 8 * 2^-24 in all.  The output's type adds half its step."""
import pytest
import torch

import layer_reference as ref
from qwen35_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def near(got, x, positions, freq, gain, interleaved):
    want, size = ref.rope(x, positions, freq, gain, interleaved)
    own = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    bound = size * 8 * 2.0 ** -24 + want.abs() * own * (1 + 2 ** -10) + (1e-30 if own == 0 else torch.finfo(got.dtype).smallest_normal * 2 ** -7)
    far = (got.double() - want).abs()
    assert bool((far <= bound).all()), float((far - bound).max())
    rot = 2 * len(freq)
    assert torch.equal(got[..., rot:], x[..., rot:])


def places(tokens, far, gen):
    return torch.randint(0, far, (tokens,), device="cuda", generator=gen, dtype=torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rot", [(1, 1, 0, 2, 2), (1, 8, 2, 256, 64), (5, 3, 1, 64, 64), (64, 16, 4, 256, 64),
                                                            (33, 2, 2, 128, 126), (7, 5, 1, 130, 22), (3, 4, 4, 96, 96), (9, 2, 1, 67, 34),
                                                            (300, 32, 8, 128, 128), (2, 1, 1, 1030, 1022), (4, 1, 1, 1026, 6),
                                                            (2000, 3, 1, 64, 18)])
def test_layouts_and_sizes(gpu, dtype, interleaved, tokens, q_heads, k_heads, dim, rot):
    gen = torch.Generator(device="cuda").manual_seed(dim + rot)
    qkv = torch.randn((tokens, q_heads + 2 * k_heads, dim), device="cuda", generator=gen).to(dtype)
    q, k = qkv[:, :q_heads], qkv[:, q_heads:q_heads + k_heads]
    at = places(tokens, 40000, gen)
    table = ops.RopeTable(rot, 10000.0)
    freq, gain = ref.frequencies(rot, 10000.0)
    qo, ko = ops.rope(q, k if k_heads else None, at, table, interleaved=interleaved)
    near(qo, q, at, freq, gain, interleaved)
    if k_heads:
        near(ko, k, at, freq, gain, interleaved)
    else:
        assert ko is None
    # in place: the same bits, and nothing beside them touched
    keep = qkv.clone()
    ops.rope(q, k if k_heads else None, at, table, interleaved=interleaved, q_out=q, k_out=k if k_heads else None)
    assert torch.equal(q, qo) and (not k_heads or torch.equal(k, ko))
    assert torch.equal(qkv[:, q_heads + k_heads:], keep[:, q_heads + k_heads:])


@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 8.0), ("yarn", 1.0), ("yarn", 40.0)])
@pytest.mark.parametrize("base,rot", [(10000.0, 64), (1e6, 128), (5e5, 20)])
def test_long_contexts(gpu, scaling, factor, base, rot):
    gen = torch.Generator(device="cuda").manual_seed(rot)
    q = torch.randn((257, 2, 128), device="cuda", generator=gen)
    at = places(257, 2 ** 31 - 1, gen)
    at[:6] = torch.tensor([0, 1, 2 ** 31 - 1, -1, -(2 ** 31), -12345], dtype=torch.int32)
    more = dict(scaling=scaling, factor=factor, original=32768)
    freq, gain = ref.frequencies(rot, base, **more)
    table = ops.RopeTable(rot, base, **more)
    # frequencies: exact to 2^-64 turns and gain to f32
    want = torch.tensor(freq, dtype=torch.float64) / (2 * torch.pi)
    got = (table.steps.cpu().double() % 2.0 ** 64) / 2.0 ** 64
    assert float((got - want % 1.0).abs().max()) < 2e-16 and abs(table.gain - gain) <= gain * 2 ** -24
    # an f64 angle of position 2^31 is off by 2^31 * f * 2^-53 itself: 2.4e-7 rad at f = 1, so near places count here
    near_by = at.clamp(-2 ** 24, 2 ** 24)
    near(ops.rope(q, None, near_by, table)[0], q, near_by, freq, gain, False)
    # far ones by a property: turning by p and then by -p gives the head back, times gain^2
    there, _ = ops.rope(q, None, at[6:].repeat(2)[:257].contiguous(), table)
    back, _ = ops.rope(there, None, (-at[6:].repeat(2)[:257]).contiguous(), table)
    back[..., :rot] /= table.gain ** 2
    assert float((back - q).abs().max()) < 40 * 2 ** -24 * float(q.abs().max())


def test_turns_add_up_at_far_places(gpu):
    """Position p and p + 2^20 * 1000 differ by the turn of 2^20 * 1000, at any p (angles are integers mod 2^64)."""
    table = ops.RopeTable(64, 1e6)
    q = torch.randn((128, 1, 64), device="cuda")
    p = torch.arange(128, dtype=torch.int32, device="cuda") * 7
    step = torch.full_like(p, 2 ** 20 * 1000)
    a, _ = ops.rope(ops.rope(q, None, p, table)[0], None, step, table)
    b, _ = ops.rope(q, None, p + step, table)
    assert float((a - b).abs().max()) < 40 * 2 ** -24 * float(q.abs().max())


def test_infinities_and_nan_stay_in_their_pair(gpu):
    q = torch.randn((3, 2, 64), device="cuda")
    q[1, 0, 3], q[1, 1, 40], q[2, 0, 63] = torch.nan, torch.inf, torch.nan
    table = ops.RopeTable(40)
    at = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    out, _ = ops.rope(q, None, at, table)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 23] = want[1, 1, 40] = want[2, 0, 63] = True
    assert torch.equal(bad, want)


def test_no_tokens(gpu):
    q = torch.empty((0, 2, 64), device="cuda")
    out, _ = ops.rope(q, None, torch.empty(0, dtype=torch.int32, device="cuda"), ops.RopeTable(64))
    assert out.shape == q.shape


def test_refusals(gpu):
    q, k = torch.randn((4, 4, 64), device="cuda"), torch.randn((4, 2, 64), device="cuda")
    at, table = torch.arange(4, dtype=torch.int32, device="cuda"), ops.RopeTable(64)
    ok = dict(q=q, k=k, positions=at, table=table)
    ops.rope(**ok)
    for kw in (dict(q=q.double()), dict(q=q[0]), dict(q=q.cpu()), dict(q=q.transpose(1, 2)), dict(k=k.half()), dict(k=k[:3]), dict(k=k[..., :32]),
               dict(positions=at.long()), dict(positions=at[:3]), dict(positions=at.cpu()), dict(q_out=k), dict(k_out=k.half()),
               dict(table=ops.RopeTable(64, device="cpu"))):
        with pytest.raises(ValueError):
            ops.rope(**{**ok, **kw})
    wide = torch.randn((4, 8, 64), device="cuda")
    for kw in (dict(table=ops.RopeTable(66)), dict(q_out=q[:1].expand(4, 4, 64)), dict(q_out=wide[:, :4], k_out=wide[:, 3:5]),
               dict(q=wide[:, :4], q_out=wide[:, 2:6]), dict(k=wide[:, :2], q_out=wide[:, 1:5]),
               dict(q=torch.randn((4, 1, 2100), device="cuda"), k=None, table=ops.RopeTable(2100))):
        with pytest.raises(RuntimeError):
            ops.rope(**{**ok, **kw})


def test_in_a_graph_on_another_stream(gpu):
    q, k = torch.randn((17, 8, 128), device="cuda").half(), torch.randn((17, 2, 128), device="cuda").half()
    at, table = torch.arange(17, dtype=torch.int32, device="cuda"), ops.RopeTable(64)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.rope(q, k, at, table, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    for i in range(3):
        at += 1000 * i
        graph.replay()
        torch.cuda.synchronize()
        a, b = ops.rope(q, k, at, table)
        assert torch.equal(a, qo) and torch.equal(b, ko)


def test_more_tokens_than_a_launch_takes(gpu):
    """A grid holds fewer than 2^32 threads: one head of 2048 values a workgroup of 256, all tokens of one row."""
    tokens = 2 ** 23 + 5
    x = torch.randn((1, 1, 2048), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16().expand(tokens, 1, 2048)
    at = torch.arange(tokens, device="cuda", dtype=torch.int32)
    out, _ = ops.rope(x, None, at, ops.RopeTable(1024), interleaved=True)
    some = torch.tensor([0, 1, 70000, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 4], device="cuda")
    freq, gain = ref.frequencies(1024, 10000.0)
    near(out[some], x[some], at[some], freq, gain, True)
