"""The operators between a layer's products and its caches, run together as examples/hybrid_layers.py runs them: every
call of a served batch against its 64-bit form on the same inputs, with the operators' own tolerances."""
import importlib.util
import math
import os

import pytest
import torch

import layer_reference as ref
import test_gpu_norm
import test_gpu_rope
from qwen35_amd import ops as real

pytestmark = pytest.mark.gpu


class Watched:
    """The ops module, with the calls of this file's operators looked at."""

    def __init__(self):
        self.seen = {}

    def __getattr__(self, name):
        return getattr(real, name)

    def count(self, name):
        self.seen[name] = self.seen.get(name, 0) + 1

    def rms_norm(self, x, weight, eps, residual=None, out=None):
        want, h = ref.rms_norm(x, weight, eps, residual)
        got = real.rms_norm(x, weight, eps, residual=residual, out=out)
        test_gpu_norm.near(got, want, 3)
        assert residual is None or torch.equal(residual, h.float())
        self.count("rms_norm")
        return got

    def rms_norm_quantize(self, ttype, x, weight, eps, residual=None, gate=None):
        want, h = ref.rms_norm(x, weight, eps, residual, gate)
        y = real.rms_norm(x, weight, eps, residual=None if residual is None else residual.clone(), gate=gate)
        test_gpu_norm.near(y, want, 11)
        got = real.rms_norm_quantize(ttype, x, weight, eps, residual=residual, gate=gate)
        assert torch.equal(got, real.quantize_act(ttype, y.reshape(len(y), -1)))
        assert residual is None or torch.equal(residual, h.float())
        self.count("rms_norm_quantize")
        return got

    def rope(self, q, k, positions, table, q_out, k_out):
        before = q.clone(), k.clone()
        got = real.rope(q, k, positions, table, q_out=q_out, k_out=k_out)
        freq, gain = ref.frequencies(table.rot_dim, 1e6)
        for x, y in zip(before, got):
            test_gpu_rope.near(y, x, positions, freq, gain, False)
        self.count("rope")
        return got

    def linear_attention(self, q, k, v, log_decay, states, slots, offsets, max_new, beta, source, work):
        want, after = ref.linear_attention(q, k, v, log_decay, beta, states, slots.tolist(), offsets.tolist(), source.tolist(),
                                           q.shape[-1] ** -0.5, max_new)
        got = real.linear_attention(q, k, v, log_decay, states, slots, offsets, max_new, beta=beta, source=source, work=work)
        bound = 4 * math.sqrt(max_new + q.shape[-1]) * 2.0 ** -24
        assert float((got - want).norm() / want.norm()) <= bound and float((states - after).norm() / after.norm()) <= bound
        self.count("linear_attention")
        return got


@pytest.mark.parametrize("sizes", [{}, dict(hidden=512, k_heads=2, v_heads=6, key_dim=64, value_dim=128, q_heads=4, kv_heads=1, dim=64),
                                   dict(hidden=1024, k_heads=4, v_heads=4, value_dim=256, q_heads=8, kv_heads=8, dim=128, seed=3)])
def test_a_served_batch(gpu, monkeypatch, sizes):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_layers.py")
    spec = importlib.util.spec_from_file_location("hybrid_layers", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    plain, _ = example.run(decode=3, **sizes)
    watch = Watched()
    monkeypatch.setattr(example, "ops", watch)
    rows, _ = example.run(decode=3, **sizes)
    assert watch.seen == dict(rms_norm=5 * 4, rms_norm_quantize=5 * 5, rope=5, linear_attention=5 * 2)
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(plain, rows))
