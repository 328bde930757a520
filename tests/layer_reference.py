"""Norms, rotary positions and linear attention in plain 64-bit form, for the GPU tests."""
import math

import torch


def f32(x):
    """x (a number) as f32 holds it."""
    return float(torch.tensor(x, dtype=torch.float32))


def rms_norm(x, weight, eps, residual=None, gate=None):
    """f64 (y, h) over the last dimension; h = x + residual, one f32 sum."""
    h = x.double() if residual is None else (x.float() + residual.float()).double()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + f32(eps))
    if weight is not None:
        y = y * weight.double()
    if gate is not None:
        g = gate.double()
        y = y * g / (1 + torch.exp(-g))
    return y, h


def frequencies(rot, base, scaling=None, factor=1.0, original=0, fast=32.0, slow=1.0):
    """Radians a position of each pair, and the factor on the turned values."""
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    freq = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    if scaling != "yarn":
        return freq, 1.0
    def pair(turns):
        return rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
    out = []
    for i, f in enumerate(freq):
        r = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(f * (1 - r) + f / factor * r)
    return out, 1 + 0.1 * math.log(factor)


def rope(x, positions, freq, gain, interleaved):
    """f64 of x [tokens, heads, dim], and for each value the sum of its pair's absolute values (0 where it is copied)."""
    y, half = x.double(), len(freq)
    z, size = y.clone(), torch.zeros_like(y)
    for i, f in enumerate(freq):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = (positions.double() * f)[:, None]
        c, s = torch.cos(angle) * gain, torch.sin(angle) * gain
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = (y[..., a].abs() + y[..., b].abs()) * gain
    return z, size


def linear_attention(q, k, v, log_decay, beta, states, slots, offsets, source, scale, max_new=1 << 30):
    """f64 (out, states): token by token.  Rows of no sequence are NaN."""
    group = v.shape[1] // q.shape[1]
    q, k = (t.double().repeat_interleave(group, 1) for t in (q, k))
    v, keep, before = v.double(), log_decay.double().exp(), states.double()
    out, after = torch.full_like(v, math.nan), before.clone()
    for i, slot in enumerate(slots):
        src = slot if source is None else source[i]
        s = before[src].clone() if 0 <= src < len(before) else torch.full_like(before[0], 0.0 if src == -1 else math.nan)
        for t in range(offsets[i], min(offsets[i + 1], len(v), offsets[i] + max_new)):
            s = s * keep[t, :, None, None]
            u = v[t] if beta is None else beta[t].double()[:, None] * (v[t] - torch.matmul(k[t, :, None], s)[:, 0])
            s = s + k[t, :, :, None] * u[:, None]
            out[t] = scale * torch.matmul(q[t, :, None], s)[:, 0]
        if 0 <= slot < len(before):
            after[slot] = s
    return out, after
