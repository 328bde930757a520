"""Linear attention with decay against its recurrence in 64 bits.

Tolerance, relative L2 of all outputs and of all states: a result is made of sums over key_dim products and over at most n
tokens' updates, each rounded to 2^-24 of a state whose updates do not grow (keys of length one, 0 < beta < 1, decays <=
1), with independent signs: 4 * sqrt(n + key_dim) * 2^-24.  An output's type adds half its step."""
import math

import pytest
import torch

import layer_reference as ref
from qwen35_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


class Batch:
    def __init__(self, lengths, k_heads, v_heads, dk, dv, dtype, delta=True, seed=0, pool=None, pad=0, alike=0.5, rate=(-3, 0.5)):
        gen = torch.Generator(device="cuda").manual_seed(seed + 7)
        n, tokens = len(lengths), sum(lengths) + pad
        self.lengths, self.offsets = lengths, [0]
        for length in lengths:
            self.offsets.append(self.offsets[-1] + length)
        normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
        qk = normal(tokens, 2 * k_heads, dk) + alike * normal(1, 2 * k_heads, dk)
        qk = (qk / qk.norm(dim=-1, keepdim=True)).to(dtype)
        self.q, self.k = qk.split([k_heads, k_heads], 1)
        self.v = normal(tokens, v_heads, dv).to(dtype)
        self.log_decay = -torch.logspace(*rate, v_heads, device="cuda") * torch.nn.functional.softplus(normal(tokens, v_heads))
        self.beta = torch.sigmoid(normal(tokens, v_heads)) if delta else None
        pool = n + 2 if pool is None else pool
        self.states = normal(pool, v_heads, dk, dv)
        self.slots = torch.randperm(pool, device="cuda", generator=gen)[:n].tolist()
        self.source, self.max_new = None, max(lengths, default=0)
        self.scale = None

    def args(self):
        ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        return (self.q, self.k, self.v, self.log_decay, self.states, ints(self.slots), ints(self.offsets), self.max_new), \
            dict(beta=self.beta, source=ints(self.source), scale=self.scale)

    def work(self):
        return ops.linear_attention_work(self.states, self.q, len(self.lengths), self.max_new, delta=self.beta is not None)

    def want(self):
        scale = self.q.shape[-1] ** -0.5 if self.scale is None else self.scale
        return ref.linear_attention(self.q, self.k, self.v, self.log_decay, self.beta, self.states, self.slots, self.offsets,
                                    self.source, scale, self.max_new)

    def run(self, **kw):
        a, k = self.args()
        return ops.linear_attention(*a, **{**k, "work": self.work(), **kw})

    def check(self, far=4.0):
        out, after = self.want()
        before = self.states.clone()
        mark = torch.full_like(self.v, 77.0)
        got = self.run(out=mark)
        some = ~out[..., 0].isnan()  # rows of some sequence
        n, dk = max(self.lengths, default=0), self.q.shape[-1]
        bound = far * math.sqrt(n + dk) * 2.0 ** -24
        if bool(some.any()):
            own = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
            assert float((got[some].double() - out[some]).norm() / out[some].norm()) <= bound + own
        assert bool((got[~some] == 77).all())
        written = torch.tensor([s for s in self.slots if 0 <= s < len(before)], dtype=torch.long, device="cuda")
        if len(written):
            assert float((self.states[written].double() - after[written]).norm() / after[written].norm()) <= bound
        rest = torch.ones(len(before), dtype=torch.bool, device="cuda")
        rest[written] = False
        assert torch.equal(self.states[rest], before[rest])
        return got


SIZES = [(1, 1, 64, 64), (2, 2, 128, 128), (1, 3, 64, 256), (2, 4, 128, 64), (3, 3, 64, 128), (1, 2, 128, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("k_heads,v_heads,dk,dv", SIZES)
@pytest.mark.parametrize("lengths", [[1], [1, 1, 1], [2, 0, 5, 1], [31, 9, 17], [32, 1], [33, 64, 65, 127], [300], [1, 200, 1, 96]])
def test_ragged_batches(gpu, dtype, delta, k_heads, v_heads, dk, dv, lengths):
    Batch(lengths, k_heads, v_heads, dk, dv, dtype, delta, seed=dk + dv, pad=3).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("length", [8, 16, 95, 1025])
def test_sequences_that_start_from_nothing_from_another_state_and_leave_none(gpu, dtype, delta, length):
    b = Batch([length, 3, length + 1, 0, 40], 2, 2, 128, 128, dtype, delta, pool=9)
    b.slots, b.source = [4, 0, -1, 7, 2], [-1, 5, 5, 8, 2]  # two start from state 5; the one without tokens copies 8 to 7
    b.check()


def test_sources_and_slots_outside_the_pool(gpu):
    b = Batch([3, 50, 2, 70], 2, 2, 64, 64, torch.float32, pool=4)
    before = b.states.clone()
    b.slots, b.source = [0, 1, 4, -2 ** 31], [4, -2, 2, 2 ** 31 - 1]
    out = b.run()
    bad = torch.tensor([True] * 53 + [False] * 2 + [True] * 70, device="cuda")
    assert bool(out[bad].isnan().all()) and bool(torch.isfinite(out[~bad]).all())
    assert bool(b.states[:2].isnan().all()) and torch.equal(b.states[2:], before[2:])


@pytest.mark.parametrize("length", [1, 5, 33, 200])
def test_strides(gpu, length):
    """Columns of one projection's rows at odd elements, heads in front of tokens, numbers inside wider rows."""
    b = Batch([length, 2, 7], 2, 4, 64, 64, torch.bfloat16)
    tokens = len(b.v)
    wide = torch.full((tokens, 3 + 128 + 128 + 256 + 2), torch.nan, device="cuda", dtype=torch.bfloat16)
    cut = [wide[:, 3:131].view(tokens, 2, 64), wide[:, 131:259].view(tokens, 2, 64), wide[:, 259:515].view(tokens, 4, 64)]
    for to, x in zip(cut, (b.q, b.k, b.v)):
        to.copy_(x)
    b.q, b.k, b.v = cut
    numbers = torch.full((tokens, 11), torch.nan, device="cuda")
    numbers[:, 1:5], numbers[:, 6:10] = b.log_decay, b.beta
    b.log_decay, b.beta = numbers[:, 1:5], numbers[:, 6:10]
    got = b.check()
    again = Batch([length, 2, 7], 2, 4, 64, 64, torch.bfloat16)
    out = torch.empty((4, tokens, 64), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    q, k = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (again.q, again.k))
    again.q, again.k = q, k
    assert torch.equal(again.run(out=out), got) and torch.equal(again.states, b.states)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [3, 70])
@pytest.mark.parametrize("delta", [True, False])
def test_decays_that_forget_and_that_keep(gpu, dtype, length, delta):
    """log_decay of -infinity, -1000, 0 and -1e-30, in the middle of a chunk too."""
    b = Batch([length, 2], 1, 4, 64, 64, dtype, delta)
    b.log_decay[length // 2, 0] = -math.inf
    b.log_decay[length // 3:, 1] = -1000.0
    b.log_decay[:, 2] = 0.0
    b.log_decay[:, 3] = -1e-30
    b.log_decay[0, 3] = -math.inf
    b.check()


@pytest.mark.parametrize("length", [9, 64, 200])
def test_keys_all_alike(gpu, length):
    """The triangular system of a chunk at its worst: equal keys, beta 1, no decay; a token then replaces the one before."""
    b = Batch([length], 1, 2, 128, 64, torch.float32, alike=0)
    b.k[:] = b.k[0]
    b.beta[:], b.log_decay[:] = 1.0, 0.0
    # no contraction: an error stays, and outputs are as large as one token's value
    b.check(far=8.0)


@pytest.mark.parametrize("scale", [1.0, -0.25, 0.0])
def test_scales(gpu, scale):
    b = Batch([40, 1], 1, 2, 64, 64, torch.float32)
    b.scale = scale
    out, _ = b.want()
    got = b.run()
    assert float((got.double() - out).abs().max()) <= 4 * math.sqrt(40 + 64) * 2.0 ** -24 * (abs(scale) * float(b.v.abs().max()) * 8)


def test_nan_and_infinity_stay_in_their_head_and_behind_their_token(gpu):
    clean, b = (Batch([100, 30], 2, 4, 64, 64, torch.float32) for _ in range(2))
    b.v[50, 1, 7], b.k[10, 1, 3], b.v[100 + 3, 0, 0] = torch.nan, torch.inf, torch.inf
    a, got = clean.run(), b.run()
    same = torch.ones_like(a, dtype=torch.bool)
    same[50:100, 1, 7] = False         # its own column from its token on
    same[10:100, 2:] = False           # both heads of the key
    same[103:, 0, 0] = False
    assert bool(torch.isfinite(got[same]).all())
    assert float((got - a)[same].abs().max()) < 1e-5


def test_lengths_past_max_new_and_offsets_out_of_range(gpu):
    b = Batch([40, 90, 3], 1, 1, 64, 64, torch.float32)
    b.max_new = 35
    b.check()
    b = Batch([40, 90, 3], 1, 1, 64, 64, torch.float32)
    b.offsets = [-5, 40, 30, 2 ** 31 - 1]  # before the rows, running back, past the rows
    b.max_new = 200
    before = b.states.clone()
    got = b.run(out=torch.full_like(b.v, 77.0))
    assert bool((got[:30] == 77).all()) and bool((got[30:] != 77).all())
    for i in (0, 1):
        assert torch.equal(b.states[b.slots[i]], before[b.slots[i]])


def test_one_call_or_many_the_same_values(gpu):
    """A prompt in one call, in pieces, and token by token; decays of 1 keep every rounding."""
    def pieces(cuts):
        b = Batch([150], 2, 2, 128, 128, torch.float32, rate=(-6, -1))
        outs, at = [], 0
        for n in cuts:
            part = Batch([n], 2, 2, 128, 128, torch.float32)
            for name in ("q", "k", "v", "log_decay", "beta"):
                setattr(part, name, getattr(b, name)[at:at + n])
            part.states, part.slots = b.states, b.slots
            outs.append(part.run())
            at += n
        return torch.cat(outs), b.states
    whole, states = pieces([150])
    for cuts in ([70, 1, 79], [1] * 150, [33, 117]):
        out, after = pieces(cuts)
        bound = 8 * math.sqrt(150 + 128) * 2.0 ** -24
        assert float((out - whole).norm() / whole.norm()) <= bound and float((after - states).norm() / states.norm()) <= bound


def test_the_same_bits_every_time(gpu):
    for lengths in ([1] * 20, [500, 3, 64]):
        a, b = (Batch(lengths, 2, 4, 128, 128, torch.bfloat16) for _ in range(2))
        assert torch.equal(a.run(), b.run()) and torch.equal(a.states, b.states)


def test_nothing_to_do(gpu):
    b = Batch([], 2, 2, 64, 64, torch.float32)
    assert b.run().shape == (0, 2, 64)
    b = Batch([0, 0], 2, 2, 64, 64, torch.float32)
    before = b.states.clone()
    b.slots, b.source = [3, 1], [2, -1]
    b.run()
    assert torch.equal(b.states[3], before[2]) and bool((b.states[1] == 0).all())


def test_refusals(gpu):
    b = Batch([4, 3], 2, 4, 64, 64, torch.float32)
    names = ("q", "k", "v", "log_decay", "states", "slots", "offsets", "max_new")
    a, kw = b.args()
    ok = {**dict(zip(names, a)), **kw}
    ops.linear_attention(**ok)
    s = ok["states"]
    for bad in (dict(q=ok["q"].half()), dict(k=ok["k"][:5]), dict(k=ok["k"].half()), dict(v=ok["v"][:, :3]), dict(v=ok["v"].half()),
                dict(q=ok["q"].cpu()), dict(log_decay=ok["log_decay"].half()), dict(log_decay=ok["log_decay"][:5]),
                dict(beta=ok["beta"].t().contiguous().t()), dict(beta=ok["beta"][:, :1]), dict(states=s.half()), dict(states=s[0]),
                dict(states=s.transpose(2, 3)), dict(states=s.cpu()), dict(slots=ok["slots"].long()), dict(slots=ok["slots"][:1]),
                dict(offsets=ok["offsets"][:2]), dict(source=ok["slots"][:1]), dict(source=ok["slots"].cpu()), dict(out=ok["v"].half()),
                dict(out=ok["v"][:, :2]), dict(work=torch.empty(9, device="cuda")), dict(max_new=2 ** 31)):
        with pytest.raises(ValueError):
            ops.linear_attention(**{**ok, **bad})
    wide = torch.randn((7, 9, 64), device="cuda")
    for bad in (dict(q=torch.randn((7, 3, 64), device="cuda"), k=torch.randn((7, 3, 64), device="cuda")),  # heads do not divide
                dict(out=ok["v"]), dict(out=wide[:, 2:6], v=wide[:, 4:8]), dict(out=torch.zeros((1, 4, 64), device="cuda").expand(7, 4, 64)),
                dict(max_new=-1), dict(out=s.view(-1)[:7 * 256].view(7, 4, 64)), dict(v=s.view(-1)[:7 * 256].view(7, 4, 64)),
                dict(states=torch.zeros((4, 4, 64, 96), device="cuda"), v=torch.zeros((7, 4, 96), device="cuda")),
                dict(states=torch.zeros((4, 4, 64, 64), device="cuda").view(-1)[1:-4 * 64 * 64 + 1 or None].view(-1)[:3 * 4 * 64 * 64].view(3, 4, 64, 64))):
        with pytest.raises(RuntimeError):
            ops.linear_attention(**{**ok, **bad})
    with pytest.raises(ValueError):
        ops.linear_attention_work(s, ok["q"][:, :1].expand(7, 3, 64).contiguous(), 2, 4)


def test_in_a_graph_on_another_stream(gpu):
    for lengths in ([1] * 5, [130, 1, 40]):
        b, want = (Batch(lengths, 2, 4, 128, 128, torch.float32) for _ in range(2))
        (args, kw), work = b.args(), b.work()
        out, first = torch.empty_like(b.v), b.states.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                ops.linear_attention(*args, **kw, work=work, out=out)
        torch.cuda.synchronize()
        assert torch.equal(b.states, first)
        for _ in range(3):  # the states go on from replay to replay
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want.run()) and torch.equal(b.states, want.states)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lengths", [[70, 3, 0, 40], [64, 0, 64, 0], [0, 0, 5, 90], [33, 1, 16, 17]])
def test_rows_of_a_padded_batch(gpu, dtype, delta, lengths):
    """As many rows as sequences of the longest length would have; short sequences and those without tokens, which copy."""
    longest = max(lengths)
    b = Batch(lengths, 2, 2, 128, 128, dtype, delta, pool=9, pad=longest * len(lengths) - sum(lengths))
    b.slots, b.source = [4, 0, 7, 2], [-1, 5, 8, 2]
    b.check()
    b = Batch(lengths, 1, 2, 64, 256, dtype, delta, pool=9, pad=longest * len(lengths) - sum(lengths))
    b.slots, b.source = [4, 0, 7, -1], [4, 0, 8, 2]
    b.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_sequences_of_all_lengths(gpu, dtype):
    """More sequences than a wave has lanes, those without tokens between, in chunks and token by token."""
    lengths = [(0, 1, 70, 3, 0, 0, 129, 16, 17, 64, 65, 2)[i % 12] for i in range(150)]
    Batch(lengths, 1, 2, 64, 128, dtype, pad=1).check()
    Batch([0] * 130 + [90] + [0] * 67 + [1, 200], 1, 2, 64, 64, dtype).check()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_workspace_used_again_and_none(gpu, dtype):
    """What a workspace holds is not read; without one every token goes by itself."""
    got, bound = [], 8 * math.sqrt(300 + 128) * 2.0 ** -24
    for work in ("nan", "larger", None):
        b = Batch([300, 20, 1], 2, 4, 128, 128, dtype)
        w = b.work()
        if work == "nan":
            w.view(torch.float32).fill_(torch.nan)
        elif work == "larger":
            w = torch.full((2 * w.numel(),), 255, dtype=torch.uint8, device="cuda")
            assert ops.linear_attention_work(b.states, b.q, 3, 300, work=w) is w
        got.append((b.run(work=None if work is None else w), b.states[b.slots]))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    own = torch.finfo(dtype).eps if dtype != torch.float32 else 0.0  # two roundings
    for x, y, more in ((got[0][0], got[2][0], own), (got[0][1], got[2][1], 0.0)):
        assert float((x.double() - y.double()).norm() / y.double().norm()) <= bound + more


def test_workspaces_that_do_not_fit(gpu):
    b = Batch([300, 20], 1, 2, 64, 64, torch.float32)
    w = b.work()
    for bad in (w[:-1], torch.zeros(w.numel() + 4, dtype=torch.uint8, device="cuda")[4:], w[:0]):
        with pytest.raises((RuntimeError, ValueError)):
            b.run(work=bad)
    assert Batch([16] * 3, 1, 2, 64, 64, torch.float32).work() is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_states_past_32_bits(gpu, dtype):
    """A pool of more than 2^32 values, tokens further apart than 2^32 bytes in all."""
    pool = torch.empty((2 ** 32 // (4 * 128 * 128) + 3, 4, 128, 128), device="cuda")
    b = Batch([2, 90, 1], 2, 4, 128, 128, dtype, pool=3)
    small, n = b.states, len(pool)
    far = [n - 1, 0, n - 3]
    want, after = b.want()
    for i, s in enumerate(b.slots):
        pool[far[i]] = small[s]
    rows = torch.empty((len(b.v), 1 << 23), device="cuda", dtype=dtype)
    for name, heads in (("q", 2), ("k", 2), ("v", 4)):
        x = getattr(b, name)
        at = {"q": 0, "k": 1000, "v": 2 ** 23 - 512}[name]
        wide = rows[:, at:at + heads * 128].view(-1, heads, 128)
        wide.copy_(x)
        setattr(b, name, wide)
    old, b.slots, b.states = b.slots, far, pool
    got = b.run()
    bound = 4 * math.sqrt(90 + 128) * 2.0 ** -24
    own = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    assert float((got.double() - want).norm() / want.norm()) <= bound + own
    assert float((pool[far].double() - after[old]).norm() / after[old].norm()) <= bound
    further = torch.empty((3, (1 << 23) + 8), device="cuda", dtype=dtype)[:, :256].view(3, 2, 128)
    c = Batch([3], 2, 4, 128, 128, dtype)
    c.q = further
    with pytest.raises(RuntimeError):
        c.run()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("token", [0, 1, 16, 37, 63, 64, 101, 149])
@pytest.mark.parametrize("name", ["q", "k", "v", "log_decay", "beta"])
def test_what_is_not_finite_stays_behind_its_token(gpu, name, token, dk, delta, dtype):
    """One NaN or infinity in the middle of a chunk, of a block of the triangular system and of neither: the tokens before
    are as without it, those after it and the state are lost, other heads and sequences are not."""
    if name == "beta" and not delta:
        pytest.skip("no beta")
    for value in (torch.nan, torch.inf):
        clean, b = (Batch([150, 30], 2, 2, dk, 64, dtype, delta, seed=token) for _ in range(2))
        x = getattr(b, name)
        if x.dim() == 3:
            x[token, 1, 5] = value
        else:
            x[token, 1] = value
        want, got = clean.run(), b.run()
        same = torch.ones(got.shape, dtype=torch.bool, device="cuda")
        if name == "q":
            same[token, 1] = False
        elif name == "v":
            same[token:150, 1, 5] = False
        else:
            same[token:150, 1] = False
        assert bool(torch.isfinite(got[same]).all())
        bound = 4 * math.sqrt(150 + dk) * 2.0 ** -24 + torch.finfo(dtype).eps
        assert float((got - want)[same].float().norm() / want[same].float().norm()) <= bound
        assert not bool(torch.isfinite(got[~same]).any())
        states, state = clean.states, b.states[b.slots[0], 1]
        assert torch.equal(b.states[b.slots[1]], states[b.slots[1]]) and torch.equal(b.states[b.slots[0], 0], states[b.slots[0], 0])
        if name == "q":
            assert torch.equal(b.states, states)
        elif name == "v":
            assert not bool(torch.isfinite(state[:, 5]).any()) and torch.equal(state[:, :5], states[b.slots[0], 1][:, :5])
        elif name == "k" and not delta:
            assert not bool(torch.isfinite(state[5]).any())  # the key's row
        else:
            assert not bool(torch.isfinite(state).any())
