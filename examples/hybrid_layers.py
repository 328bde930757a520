"""Serves a ragged batch through layers of linear attention with one of attention over the 8-bit cache between them: prompts,
a prompt that arrives beside running sequences, then single tokens.

Between two quantized products a layer calls one operator for each thing it does: the residual's sum, the norm and the
activation rows of the next product in one; norms of heads; rotary positions; the states or the cache; the gated norm of
the outputs with the rows of the output projection.  Run: python examples/hybrid_layers.py
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from qwen35_amd import ops, synth  # noqa: E402

Q8_0 = 8
EPS = 1e-6


class Product:
    """A Q8_0 weight [rows, cols] that takes activation rows."""

    def __init__(self, rows, cols, seed, tag):
        self.rows, self.cols = rows, cols
        self.w = torch.from_numpy(synth.make_weight(Q8_0, rows, cols, seed, tag)).cuda()

    def __call__(self, xq):
        return ops.mul_mat(Q8_0, self.w, xq, self.rows, self.cols, len(xq))


class LinearLayer:
    """Linear attention with the delta rule: k_heads keys and queries of length one, v_heads values, a gate on the outputs."""

    def __init__(self, hidden, k_heads, v_heads, key_dim, value_dim, nseq, seed, gen):
        self.k_heads, self.v_heads, self.dk, self.dv = k_heads, v_heads, key_dim, value_dim
        self.widths = [2 * k_heads * key_dim, v_heads * value_dim, v_heads * value_dim, v_heads, v_heads]
        self.inner = Product(sum(self.widths), hidden, seed, 1)
        self.outer = Product(hidden, v_heads * value_dim, seed, 2)
        ones = dict(device="cuda")
        self.norm, self.out_norm = torch.ones(hidden, **ones), torch.ones(value_dim, **ones)
        self.length = torch.full((key_dim,), key_dim ** -0.5, **ones)  # the norm of weight 1 / sqrt(dim) is the L2 norm
        self.rate = torch.rand(v_heads, device="cuda", generator=gen) * 0.3
        self.states = torch.empty((nseq, v_heads, key_dim, value_dim), **ones)
        self.slots = torch.arange(nseq, dtype=torch.int32, device="cuda")
        self.work = None

    def step(self, hidden, x, batch):
        """What this layer adds to `hidden` (which takes up x, the layer before's)."""
        y = self.inner(ops.rms_norm_quantize(Q8_0, x, self.norm, EPS, residual=hidden))
        qk, v, gate, slow, learn = y.split(self.widths, 1)
        heads = lambda t, dim: t.view(len(t), -1, dim)  # noqa: E731
        q, k = ops.rms_norm(heads(qk, self.dk), self.length, EPS / self.dk).split(self.k_heads, 1)
        log_decay, beta = -self.rate * torch.nn.functional.softplus(slow), torch.sigmoid(learn)
        # one workspace serves every kind of step; it grows with what they need
        work = ops.linear_attention_work(self.states, q, len(batch.new), max(batch.new), work=self.work)
        self.work = work if work is not None else self.work
        source = torch.where(batch.cached == 0, -1, self.slots)  # sequences that begin do so from nothing
        o = ops.linear_attention(q, k, heads(v, self.dv), log_decay, self.states, self.slots, batch.step.offsets, max(batch.new),
                                 beta=beta, source=source, work=work)
        return self.outer(ops.rms_norm_quantize(Q8_0, o, self.out_norm, EPS, gate=heads(gate, self.dv)))


class AttentionLayer:
    """Attention of q_heads over kv_heads in the 8-bit cache; a quarter of each head turns with the position."""

    def __init__(self, hidden, q_heads, kv_heads, dim, blocks, block_size, seed):
        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.inner = Product((q_heads + 2 * kv_heads) * dim, hidden, seed, 3)
        self.outer = Product(hidden, q_heads * dim, seed, 4)
        self.norm, self.head_norm = torch.ones(hidden, device="cuda"), torch.ones(dim, device="cuda")
        self.table = ops.RopeTable(dim // 4, 1e6)
        self.cache = ops.KvCache.empty(blocks, kv_heads, block_size, dim)
        self.work = None

    def step(self, hidden, x, batch):
        y = self.inner(ops.rms_norm_quantize(Q8_0, x, self.norm, EPS, residual=hidden))
        y = y.view(len(x), -1, self.dim)
        both, v = y.split([self.q_heads + self.kv_heads, self.kv_heads], 1)
        q, k = ops.rms_norm(both, self.head_norm, EPS, out=both).split([self.q_heads, self.kv_heads], 1)
        ops.rope(q, k, batch.step.positions, self.table, q_out=q, k_out=k)
        ops.kv_append(self.cache, k, v, batch.step.slots)
        most = max(batch.new)
        self.work = ops.kv_attention_work(self.cache, self.q_heads, len(batch.new), len(x), most, batch.max_kv, work=self.work)
        o, _ = ops.kv_attention(q, self.cache, batch.table, batch.step.offsets, batch.step.kv_lens, most, batch.max_kv,
                                work=self.work)
        return self.outer(ops.quantize_act(Q8_0, o.view(len(x), -1)))


class Batch:
    """One step's new tokens of each sequence: block tables, offsets and positions."""

    def __init__(self, server, new):
        self.new, self.cached, self.table = new, server.cached, server.table
        self.step = ops.KvStep(len(new), sum(new))
        ops.kv_tables(server.cached, torch.tensor(new, dtype=torch.int32, device="cuda"), server.free, server.table,
                      server.block_size, self.step, taken=server.taken)
        server.lens = [a + b for a, b in zip(server.lens, new)]
        self.max_kv = 1 << (max(server.lens) - 1).bit_length()
        server.cached, server.taken = self.step.kv_lens, self.step.taken


class Server:
    def __init__(self, nseq, max_kv, hidden, k_heads, v_heads, key_dim, value_dim, q_heads, kv_heads, dim, block_size, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        blocks, self.block_size, self.lens = nseq * -(-max_kv // block_size), block_size, [0] * nseq
        linear = lambda i: LinearLayer(hidden, k_heads, v_heads, key_dim, value_dim, nseq, seed + i, gen)  # noqa: E731
        self.layers = [linear(0), AttentionLayer(hidden, q_heads, kv_heads, dim, blocks, block_size, seed), linear(1)]
        self.norm = torch.ones(hidden, device="cuda")
        ints = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((nseq, -(-max_kv // block_size)), -1, **ints)
        self.free = torch.arange(blocks, **ints)
        self.cached, self.taken = torch.zeros(nseq, **ints), torch.zeros(1, **ints)

    def step(self, x, new):
        """x [sum(new), hidden]: `new` tokens of each sequence.  The last layer's normed rows."""
        batch, hidden = Batch(self, new), torch.zeros_like(x)
        for layer in self.layers:
            x = layer.step(hidden, x, batch)
        return ops.rms_norm(x, self.norm, EPS, residual=hidden)


def run(prompts=(700, 33, 1, 0, 300), late=(3, 150), decode=8, hidden=2560, k_heads=16, v_heads=16, key_dim=128, value_dim=128,
        q_heads=16, kv_heads=4, dim=256, block_size=64, seed=0):
    """Each step's rows, and its milliseconds."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nseq = len(prompts)
    steps = [list(prompts), [1 if n else 0 for n in prompts]]
    steps[1][late[0]] = late[1]  # a prompt beside the others' single tokens
    steps += [[1] * nseq for _ in range(decode)]
    server = Server(nseq, max(sum(s[i] for s in steps) for i in range(nseq)), hidden, k_heads, v_heads, key_dim, value_dim, q_heads,
                    kv_heads, dim, block_size, seed)
    rows, ms = [], []
    for new in steps:
        x = torch.randn((sum(new), hidden), device="cuda", generator=gen)
        torch.cuda.synchronize()
        t = time.perf_counter()
        rows.append(server.step(x, new))
        torch.cuda.synchronize()
        ms.append((time.perf_counter() - t) * 1e3)
    return rows, ms


if __name__ == "__main__":
    run()  # (the first steps load kernels)
    rows, ms = run()
    print("tokens of a step:", " ".join(str(len(r)) for r in rows))
    print("milliseconds:    ", " ".join(f"{m:.3f}" for m in ms))
