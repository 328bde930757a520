"""The 8-bit key/value cache in plain 64-bit form, for the GPU tests: block tables, append and attention."""
import math

import torch


def tables(cached, new, free, taken, table, block, tokens):
    """Lists in; (table, offsets, kv_lens, slots, positions, taken) as lists out."""
    table, offsets, kv_lens, slots, positions = [list(r) for r in table], [0], [], [], []
    width = len(table[0]) if table else 0
    for row, c, n in zip(table, cached, new):
        c, n = max(c, 0), max(n, 0)
        for j in range(-(-c // block), -(-(c + n) // block)):
            entry = free[taken] if 0 <= taken < len(free) else -1
            if j < width:
                row[j] = entry
            taken += 1
        for p in range(c, c + n):
            entry = row[p // block] if p // block < width else -1
            slots.append(entry * block + p % block if entry >= 0 else -1)
            positions.append(p)
        offsets.append(offsets[-1] + n)
        kv_lens.append(c + n)
    pad = tokens - len(slots)
    return table, offsets, kv_lens, (slots + [-1] * pad)[:tokens], (positions + [0] * pad)[:tokens], taken


#: a code step's share of the largest value: the f32 nearest 1/127
PART = float(torch.tensor(1.0) / torch.tensor(127.0))


def _f32(x):
    return x.float().double()


def append(codes, scales, x, slots):
    """int8 codes [blocks, heads, block, dim] and f32 scales after the append of x [tokens, heads, dim].

    Scales and codes are defined by single f32 operations, so each is rounded to f32 where it is one."""
    codes, scales, x, block = codes.clone(), scales.clone(), x.double(), codes.shape[2]
    runs = {}
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * block:
            runs.setdefault(s // block, []).append((s % block, t))
    for b, run in runs.items():
        first, at, rows = run[0][0], [p for p, _ in run], [t for _, t in run]
        for h in range(codes.shape[1]):
            old = scales[b, h].double() if first else torch.zeros((), dtype=torch.float64, device=x.device)
            top = x[rows, h].abs().max()
            scale = torch.maximum(old, _f32(top * PART))
            c = codes[b, h].double()
            usable = bool(torch.isfinite(scale) and scale > 0)
            ratio = _f32(old / scale) if usable else torch.zeros_like(old)
            inv = _f32(1 / scale) if usable else torch.zeros_like(old)
            c[:first] = _f32(c[:first] * ratio).round()
            c[at] = _f32(x[rows, h] * inv).round().clamp(-127, 127) if usable else 0
            codes[b, h], scales[b, h] = c.to(torch.int8), scale.float()
    return codes, scales


def attention(q, k, v, k_scale, v_scale, table, offsets, kv_lens, scale, causal=True, window=0):
    """f64 (out, lse) of q [tokens, q_heads, dim]; rows that see nothing are 0 and -inf."""
    q, block, dim = q.double(), k.shape[2], k.shape[3]
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for i, length in enumerate(kv_lens):
        a, b = offsets[i], offsets[i + 1]
        if a == b or length <= 0:
            continue
        ids = torch.tensor(table[i][:-(-length // block)], device=q.device)
        kk = (k[ids].double() * k_scale[ids].double()[..., None, None]).transpose(0, 1).reshape(k.shape[1], -1, dim)[:, :length]
        vv = (v[ids].double() * v_scale[ids].double()[..., None, None]).transpose(0, 1).reshape(k.shape[1], -1, dim)[:, :length]
        at = (length - (b - a) + torch.arange(b - a, device=q.device))[:, None]
        j = torch.arange(length, device=q.device)
        seen = torch.ones((b - a, length), dtype=torch.bool, device=q.device)
        if causal:
            seen = j <= at
            if window:
                seen &= j > at - window
        some = seen.any(1)
        for h in range(q.shape[1]):
            s = q[a:b, h] @ kk[h // group].T.contiguous() * scale
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s[some], -1)
            # a hidden place may hold anything: its value is left out, not weighed with 0
            vals = torch.where(seen.any(0)[:, None], vv[h // group], 0)
            out[a:b, h][some] = p @ vals
            lse[a:b, h] = torch.logsumexp(s, -1)
    return out, lse
