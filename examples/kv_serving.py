"""Serves a ragged batch through one attention layer: prompts, a prompt that arrives beside running sequences, then
single tokens.

The query/key/value and output projections are Q8_0 weights of the backend (qhip_backend_matvec_batch_k); the keys and
values lie in the 8-bit cache.  A step is kv_tables once, then for each layer the projection, kv_append, kv_attention
and the output projection.  Run: python examples/kv_serving.py
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from qwen35_amd import ops, synth  # noqa: E402

Q8_0 = 8


class Layer:
    """Attention of `hidden` values a token with q_heads query and kv_heads key/value heads of head_dim, f32 rows."""

    def __init__(self, backend, hidden, q_heads, kv_heads, head_dim, blocks, block_size, seed=0):
        self.backend, self.hidden, self.q_heads, self.kv_heads, self.dim = backend, hidden, q_heads, kv_heads, head_dim
        self.rows = (q_heads + 2 * kv_heads) * head_dim
        self.qkv = backend.load_linear(Q8_0, self.rows, hidden, synth.make_weight(Q8_0, self.rows, hidden, seed, 1))
        self.out = backend.load_linear(Q8_0, hidden, q_heads * head_dim,
                                       synth.make_weight(Q8_0, hidden, q_heads * head_dim, seed, 2))
        self.cache = ops.KvCache.empty(blocks, kv_heads, block_size, head_dim)

    def project(self, x):
        """Queries, keys and values [tokens, heads, dim] of x [tokens, hidden]: three views of one product."""
        y = torch.empty((len(x), self.rows), device=x.device)
        self.backend.matvec_batch_k(y, self.qkv, x, len(x))
        y = y.view(len(x), -1, self.dim)
        y[:, :self.q_heads + self.kv_heads] *= torch.rsqrt(y[:, :self.q_heads + self.kv_heads].square().mean(-1, keepdim=True))
        return y.split([self.q_heads, self.kv_heads, self.kv_heads], 1)

    def step(self, x, step, table, max_new, max_kv, work):
        """Output projection and attention of the packed tokens x."""
        q, k, v = self.project(x)
        ops.kv_append(self.cache, k, v, step.slots)
        o, _ = ops.kv_attention(q, self.cache, table, step.offsets, step.kv_lens, max_new, max_kv, work=work)
        y = torch.empty_like(x)
        self.backend.matvec_batch_k(y, self.out, o.view(len(x), -1), len(x))
        return y, o


class Server:
    """Block tables of `nseq` sequences over a pool of blocks, and one layer."""

    def __init__(self, layer, nseq, max_kv):
        c = layer.cache
        self.layer, self.nseq, self.lens = layer, nseq, [0] * nseq
        ints = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((nseq, -(-max_kv // c.block_size)), -1, **ints)
        self.free = torch.randperm(c.num_blocks, device="cuda").to(torch.int32)  # any order
        self.cached, self.taken = torch.zeros(nseq, **ints), torch.zeros(1, **ints)
        self.work = None

    def step(self, x, new):
        """x [sum(new), hidden]: `new` tokens of each sequence."""
        tokens, most = len(x), max(new)
        self.lens = [a + b for a, b in zip(self.lens, new)]
        step = ops.KvStep(self.nseq, tokens)
        ops.kv_tables(self.cached, torch.tensor(new, dtype=torch.int32, device="cuda"), self.free, self.table,
                      self.layer.cache.block_size, step, taken=self.taken)
        self.cached, self.taken = step.kv_lens, step.taken
        # one workspace serves every kind of step; it grows with what they need
        max_kv = 1 << (max(self.lens) - 1).bit_length()
        self.work = ops.kv_attention_work(self.layer.cache, self.layer.q_heads, self.nseq, tokens, most, max_kv, work=self.work)
        return self.layer.step(x, step, self.table, most, max_kv, self.work)


def exact(layer, history, new):
    """The attention of the last new[i] tokens of each sequence with its keys and values in f32."""
    outs = []
    for x, n in zip(history, new):
        if n == 0:
            continue
        q, k, v = (t.transpose(0, 1) for t in layer.project(x))
        group = layer.q_heads // layer.kv_heads
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        s = (q[:, -n:] @ k.transpose(1, 2).contiguous()) * layer.dim ** -0.5
        place = torch.arange(len(x), device="cuda")
        s.masked_fill_(place > place[-n:, None], -torch.inf)
        outs.append((s.softmax(-1) @ v.contiguous()).transpose(0, 1))
    return torch.cat(outs)


def run(prompts=(700, 33, 1, 0, 300), late=(3, 150), decode=8, hidden=2560, q_heads=16, kv_heads=4, dim=256, block_size=64,
        seed=0):
    """Relative L2 distances of each step's attention from f32 keys and values, and the last step's milliseconds."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    torch.manual_seed(seed)
    nseq = len(prompts)
    steps = [list(prompts), [1 if n else 0 for n in prompts]]
    steps[1][late[0]] = late[1]  # a prompt beside the others' single tokens
    steps += [[1] * nseq for _ in range(decode)]
    most = max(sum(s[i] for s in steps) for i in range(nseq))
    backend = ops.Backend()
    layer = Layer(backend, hidden, q_heads, kv_heads, dim, nseq * -(-most // block_size), block_size, seed)
    server = Server(layer, nseq, most)
    history = [torch.empty((0, hidden), device="cuda") for _ in range(nseq)]
    far = []
    for new in steps:
        x = torch.randn((sum(new), hidden), device="cuda", generator=gen)
        history = [torch.cat([h, y]) for h, y in zip(history, x.split(new))]
        torch.cuda.synchronize()
        t = time.perf_counter()
        y, o = server.step(x, new)
        torch.cuda.synchronize()
        ms = (time.perf_counter() - t) * 1e3
        want = exact(layer, history, new)
        far.append(float((o - want).norm() / want.norm()))
        assert bool(torch.isfinite(y).all())
    backend.close()
    return far, ms


if __name__ == "__main__":
    distances, ms = run()
    print("relative distance from f32 keys and values, step by step:", " ".join(f"{d:.4f}" for d in distances))
    print(f"last step (one token a sequence): {ms:.3f} ms")
