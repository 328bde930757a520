"""What a hybrid decoder layer does between its quantized products and its caches, as it is measured: inputs, plain forms
and 64-bit results.

    norm    root-mean-square norm of rows or of heads, with the residual's addition in front, a gate behind, and an output
            in 8 bits with scales (the rows that the quantized products read)
    rope    rotary positions of queries and keys: half and interleaved layouts, part of the head, scaled for long contexts
    linear  linear attention with a decay for each head, as a plain sum or with the delta rule: the chunked form for
            prompts, the recurrent one for single tokens, over a pool of states

The formulas, for a head's q, k of dk values and v of dv, with a = exp(log_decay) and S the head's state [dk, dv]:

    S <- a S;  u = beta (v - k S) with the delta rule, else v;  S <- S + k^T u;  out = scale q S

Sizes are generic: the widths of small and middle models, head layouts of 64 to 256, lengths from one token to a long
prompt; 16 heads of 128 are those of the [6144, 1024] product (queries, keys and values) and the eight prompts of 16 to
256 tokens those of the ragged prompt, both of the benchmark.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
Q8_0 = 8
EPS = 1e-6
#: the most operations and bytes that a drawn case may have
MOST_FLOPS, MOST_BYTES = 2.5e10, 4.5e8


def _norm_case(tokens, heads, dim, dtype, residual=False, gate=False, quant=False):
    return {"kind": "norm", "tokens": tokens, "heads": heads, "dim": dim, "type": dtype, "residual": residual, "gate": gate,
            "quant": quant}


def _rope_case(tokens, q_heads, k_heads, dim, rot, dtype, interleaved=False, scaling="", factor=1.0, far=0):
    """`far` 0: prompts' consecutive places; else single tokens at places below it."""
    return {"kind": "rope", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "rot": rot, "type": dtype,
            "interleaved": interleaved, "scaling": scaling, "factor": factor, "far": far}


def _linear_case(k_heads, v_heads, dk, dv, dtype, delta=True, fresh=False, decodes=0, step=1, prompts=0, lo=1, hi=1, lengths=0):
    """`decodes` sequences that bring `step` tokens and `prompts` of lo..hi; `fresh` ones begin from a state of zeros."""
    return {"kind": "linear", "k_heads": k_heads, "v_heads": v_heads, "dk": dk, "dv": dv, "type": dtype, "delta": delta,
            "fresh": fresh, "decodes": decodes, "step": step, "prompts": prompts, "lo": lo, "hi": hi, "lengths": lengths}


def listed():
    return [
        # one token's hidden state in front of a layer's products: the smallest call
        {"name": "norm_decode", **_norm_case(1, 1, 2560, "f32", residual=True, quant=True)},
        # a ragged prompt in front of the products
        {"name": "norm_prompt_q8", **_norm_case(1673, 1, 5120, "f32", residual=True, quant=True)},
        # a long prompt of 16-bit rows, for a reader that takes them
        {"name": "norm_prompt", **_norm_case(4096, 1, 5120, "bf16", residual=True)},
        # the heads of a linear attention's output and their gates
        {"name": "norm_heads_gate", **_norm_case(8191, 16, 128, "f32", gate=True)},
        # the queries and keys of 64 decoding sequences, far into a long context; a quarter of each head turns
        {"name": "rope_decode", **_rope_case(64, 16, 4, 256, 64, "f32", scaling="yarn", factor=8.0, far=262144)},
        # a prompt's, from one projection's output
        {"name": "rope_prompt", **_rope_case(4097, 8, 2, 256, 64, "f32")},
        # whole heads, pairs side by side, 16-bit rows
        {"name": "rope_prompt_pairs", **_rope_case(8192, 32, 8, 128, 128, "bf16", interleaved=True, scaling="linear", factor=4.0)},
        # one token of one sequence through a layer of 16 heads
        {"name": "linear_decode_one", **_linear_case(16, 16, 128, 128, "f32", decodes=1)},
        # a token for each of 64 sequences, two value heads a key head
        {"name": "linear_decode_batch", **_linear_case(16, 32, 128, 128, "bf16", decodes=64)},
        # eight fresh prompts of 16 to 256 tokens
        {"name": "linear_prompt_ragged", **_linear_case(16, 16, 128, 128, "f32", fresh=True, prompts=8, lo=16, hi=256)},
        # plain decayed sums: a chunk of a prompt beside eleven decoding sequences
        {"name": "linear_mixed_plain", **_linear_case(8, 8, 64, 128, "f16", delta=False, decodes=11, prompts=2, lo=700, hi=2100)},
        # a whole prompt of 8192 tokens: the largest call
        {"name": "linear_prompt_8k", **_linear_case(16, 32, 128, 128, "bf16", fresh=True, prompts=1, lo=8192, hi=8192)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind, dtype = rng.choice(["norm", "heads", "rope", "rope", "linear", "linear", "linear"]), rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        quant = rng.random() < 0.5
        dim = 32 * _log(rng, 4, 512) if quant else _log(rng, 65, 16384)
        return _norm_case(_log(rng, 1, 8192), 1, dim, dtype, rng.random() < 0.7, False, quant)
    if kind == "heads":
        return _norm_case(_log(rng, 1, 16384), rng.randint(1, 48), rng.choice([64, 96, 128, 256]), dtype, False,
                          rng.random() < 0.6, False)
    if kind == "rope":
        dim, k_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 4, 8])
        rot = 2 * rng.choice([dim // 2, dim // 4, dim // 8, rng.randint(1, dim // 2)])
        scaling = rng.choice(["", "linear", "ntk", "yarn"]) if rot > 2 else ""
        return _rope_case(_log(rng, 1, 12000), k_heads * rng.choice([1, 2, 4, 6]), k_heads, dim, rot, dtype,
                          rng.random() < 0.5, scaling, rng.choice([2.0, 4.0, 32.0]) if scaling else 1.0,
                          rng.choice([0, _log(rng, 100, 2 ** 20)]))
    k_heads, dk, dv = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 128]), rng.choice([64, 128, 256])
    v_heads = min(k_heads * rng.choice([1, 1, 2, 3]), 48)
    shape = dict(k_heads=k_heads, v_heads=v_heads, dk=dk, dv=dv, dtype=dtype, delta=rng.random() < 0.75,
                 fresh=rng.random() < 0.4, lengths=rng.randint(0, 9999))
    what = rng.choice(["decode", "prompt", "prompt", "mixed"])
    if what == "decode":
        return _linear_case(decodes=_log(rng, 1, 256), step=rng.choice([1, 1, 1, rng.randint(2, 9)]), **shape)
    hi = _log(rng, 16, 8192)
    if what == "prompt":
        return _linear_case(prompts=_log(rng, 1, 16), lo=max(1, hi // rng.choice([1, 3, 16])), hi=hi, **shape)
    return _linear_case(decodes=_log(rng, 1, 64), prompts=rng.randint(1, 3), lo=max(1, hi // 3), hi=hi, **shape)


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
            continue
        if case["kind"] == "linear":  # the padded plain form
            n = _lengths(case)
            if len(n) * max(max(n), 64) * case["v_heads"] * (case["dk"] + case["dv"]) > 1.2e8:
                continue
        return case


def _lengths(case):
    rng = random.Random(case["lengths"])
    return [case["step"]] * case["decodes"] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["prompts"])]


def work(case):
    """Bytes: each input once and each result once; flops of the linear attention: the recurrence's products."""
    size = SIZES[case["type"]]
    if case["kind"] == "norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        passes = 1 + 2 * case["residual"] + case["gate"] + (not case["quant"])
        return {"bytes": n * size * passes + (n * 34 // 32 if case["quant"] else 0) + 4 * case["dim"], "flops": 0}
    if case["kind"] == "rope":
        return {"bytes": 2 * size * case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"] + 4 * case["tokens"],
                "flops": 0}
    lengths, dk, dv, heads = _lengths(case), case["dk"], case["dv"], case["v_heads"]
    tokens = sum(lengths)
    rows = tokens * size * (2 * case["k_heads"] * dk + 2 * heads * dv) + 4 * tokens * heads * (1 + case["delta"])
    states = 4 * len(lengths) * heads * dk * dv * (1 if case["fresh"] else 2)
    return {"bytes": rows + states, "flops": (6 if case["delta"] else 4) * tokens * heads * dk * dv}


# ---- inputs ---------------------------------------------------------------------------

def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 31)
    rng, dtype = random.Random(seed), DTYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    state = {"case": case}
    if case["kind"] == "norm":
        rows = (case["tokens"], case["heads"], case["dim"])
        # hidden states: some channels are much louder
        x = normal(*rows)
        x[..., ::61] *= 8.0
        state["x"], state["weight"] = x.to(dtype), 1 + 0.2 * normal(case["dim"])
        if case["residual"]:
            state["residual"] = (3 * normal(*rows)).to(dtype)
        if case["gate"]:
            state["gate"] = normal(*rows).to(dtype)
        if case["heads"] == 1:
            for name in ("x", "residual", "gate"):
                if name in state:
                    state[name] = state[name][:, 0]
        return state
    if case["kind"] == "rope":
        # one projection's output: a token's queries, keys and values
        qkv = normal(case["tokens"], case["q_heads"] + 2 * case["k_heads"], case["dim"]).to(dtype)
        state["q"], state["k"], _ = qkv.split([case["q_heads"], case["k_heads"], case["k_heads"]], 1)
        if case["far"]:
            at = [rng.randrange(case["far"]) for _ in range(case["tokens"])]
        else:
            at = list(range(rng.randint(0, 999), 10 ** 6))[:case["tokens"]]
        state["positions"] = _int(at)
        return state
    lengths = _lengths(case)
    rng.shuffle(lengths)
    tokens, n, k_heads, heads, dk, dv = sum(lengths), len(lengths), case["k_heads"], case["v_heads"], case["dk"], case["dv"]
    offsets = [0]
    for length in lengths:
        offsets.append(offsets[-1] + length)
    # queries and keys of length one; neighbouring keys are alike to a degree, as a text's are
    qk = normal(tokens, 2 * k_heads, dk) + 0.5 * normal(1, 2 * k_heads, dk)
    qk = (qk / qk.norm(dim=-1, keepdim=True)).to(dtype)
    state["q"], state["k"] = qk.split([k_heads, k_heads], 1)
    state["v"] = normal(tokens, heads, dv).to(dtype)
    # from heads that keep thousands of tokens to heads that keep a few
    rate = torch.logspace(-3, 0.5, heads, device="cuda")
    state["log_decay"] = -rate * torch.nn.functional.softplus(normal(tokens, heads))
    if case["delta"]:
        state["beta"] = torch.sigmoid(normal(tokens, heads))
    slots = list(range(n + 2))
    rng.shuffle(slots)
    state["states"] = 0.3 * normal(n + 2, heads, dk, dv)
    state["slots"], state["offsets"] = _int(slots[:n]), _int(offsets)
    state["source"] = _int([-1] * n) if case["fresh"] else state["slots"]
    state["max_new"], state["nseq"] = max(lengths), n
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _norm_own, "rope": _rope_own, "linear": _linear_own}[kind](state)
    return {"norm": _norm, "rope": _rope, "linear": _linear}[kind](state)


def _norm_own(state):
    from qwen35_amd import ops
    more = {"residual": state.get("residual"), "gate": state.get("gate")}
    if not state["case"]["quant"]:
        found = {"out": ops.rms_norm(state["x"], state["weight"], EPS, **more)}
    else:
        xq = ops.rms_norm_quantize(Q8_0, state["x"], state["weight"], EPS, **more)
        found = {"values": ops.dequantize(Q8_0, xq, state["x"].numel() // 32)}
    if "residual" in state:
        found["residual"] = state["residual"]
    return found


def _rope_own(state):
    from qwen35_amd import ops
    case = state["case"]
    if "table" not in state:
        state["table"] = ops.RopeTable(case["rot"], BASE, case["scaling"] or None, case["factor"], original=ORIGINAL)
    q, k = ops.rope(state["q"], state["k"], state["positions"], state["table"], interleaved=case["interleaved"])
    return {"q": q, "k": k}


def _linear_own(state):
    from qwen35_amd import ops
    if "work" not in state:
        state["work"] = ops.linear_attention_work(state["states"], state["q"], state["nseq"], state["max_new"],
                                                  delta="beta" in state)
    out = ops.linear_attention(state["q"], state["k"], state["v"], state["log_decay"], state["states"], state["slots"],
                               state["offsets"], state["max_new"], beta=state.get("beta"), source=state["source"],
                               work=state["work"])
    return {"out": out, "states": state["states"]}


def _norm(state):
    case, h = state["case"], state["x"].float()
    found = {}
    if "residual" in state:
        h = h + state["residual"].float()
        found["residual"] = state["residual"].copy_(h)
    # the mean square in 64 bits: codes next to a border depend on its last bits
    mean = h.double().square().sum(-1, keepdim=True) / case["dim"]
    y = h * (1 / torch.sqrt(mean + _f32_of(EPS))).float() * state["weight"]
    if "gate" in state:
        g = state["gate"].float()
        y = y * (g / (1 + torch.exp(-g)))
    if not case["quant"]:
        return {"out": y.to(state["x"].dtype), **found}
    y = y.reshape(-1, 32)
    top = y.abs().amax(-1, keepdim=True)
    scale = top / torch.full_like(top, 127)  # (a division by a number is a product with its inverse)
    inverse = torch.where(scale > 0, 1 / scale, 0)
    codes = (y * inverse + torch.where(y >= 0, 0.5, -0.5)).trunc().clamp(-128, 127)
    return {"values": (codes * scale.half().float()).reshape(-1), **found}


BASE, ORIGINAL, BETA_FAST, BETA_SLOW = 1e6, 32768, 32.0, 1.0


def _frequencies(case):
    """Radians a position of each pair, and the factor on the turned values."""
    rot, factor, base = case["rot"], case["factor"], BASE
    if case["scaling"] == "ntk":
        base *= factor ** (rot / (rot - 2))
    freq = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if case["scaling"] == "linear":
        freq = [f / factor for f in freq]
    if case["scaling"] != "yarn":
        return freq, 1.0
    # pairs that turn often over the original context stay, those that turn less than once are stretched
    low, high = (rot * math.log(ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (BETA_FAST, BETA_SLOW))
    low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
    ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
    return [f * (1 - r) + f / factor * r for f, r in zip(freq, ramp)], 1 + 0.1 * math.log(factor)


def _turned(x, cos, sin, case):
    rot = case["rot"]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    cos, sin = cos[:, None], sin[:, None]
    pair = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rope(state):
    case = state["case"]
    freq, gain = _frequencies(case)
    angle = state["positions"].double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    cos, sin = (torch.cos(angle) * gain).float(), (torch.sin(angle) * gain).float()
    return {name: _turned(state[name].float(), cos, sin, case).to(state[name].dtype) for name in ("q", "k")}


def _inverse(low):
    """(1 + low)^-1 of strictly lower triangular [.., n, n]: inverses of blocks of 1, 2, 4, .. rows, joined two by two."""
    n = low.shape[-1]
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
    x, s = torch.eye(n, device="cuda", dtype=low.dtype).expand_as(low), 1
    while s < n:
        corner = (i // (2 * s) == j // (2 * s)) & (i // s != j // s)
        x = x - x @ (low * corner) @ x
        s *= 2
    return x


def _linear(state):
    case, offsets, states = state["case"], state["offsets"].long(), state["states"]
    group, dk = case["v_heads"] // case["k_heads"], case["dk"]
    size = min(64, state["max_new"])
    chunks = -(-state["max_new"] // size)
    place = torch.arange(chunks * size, device="cuda")
    seen = place < (offsets[1:] - offsets[:-1])[:, None]
    rows = torch.where(seen, offsets[:-1, None] + place, 0)

    def packed(x, times=1):  # [tokens, heads, ..] -> [sequence, head, chunk, place, ..], 0 behind a sequence's end
        x = torch.where(seen.reshape(seen.shape + (1,) * (x.dim() - 1)), x[rows], 0)
        return x.movedim(2, 1).unflatten(2, (chunks, size)).repeat_interleave(times, 1)

    q, k, v = packed(state["q"].float(), group), packed(state["k"].float(), group), packed(state["v"].float())
    # decays between places that lie far behind the chunk's start are differences of long sums: in 64 bits
    total = packed(state["log_decay"].double()).cumsum(-1)
    i = torch.arange(size, device="cuda")
    between = (total[..., :, None] - total[..., None, :]).masked_fill(i[:, None] < i, -math.inf).exp().float()
    since, left = total.exp().float()[..., None], (total[..., -1:] - total).exp().float()[..., None]
    inside = (q @ k.transpose(-1, -2)) * between * dk ** -0.5
    if case["delta"]:
        beta = packed(state["beta"])[..., None]
        solve = _inverse(torch.tril(k @ k.transpose(-1, -2) * between * beta, -1)) * beta.transpose(-1, -2)
    source = state["source"].long()
    s = torch.where((source >= 0)[:, None, None, None], states[source.clamp(min=0)], 0)
    out = torch.empty_like(v)
    for c in range(chunks):
        u = v[:, :, c]
        if case["delta"]:
            u = solve[:, :, c] @ (u - since[:, :, c] * (k[:, :, c] @ s))
        out[:, :, c] = inside[:, :, c] @ u + since[:, :, c] * (q[:, :, c] @ s) * dk ** -0.5
        s = s * since[:, :, c, -1:] + (k[:, :, c] * left[:, :, c]).transpose(-1, -2) @ u
    states[state["slots"].long()] = s
    out = out.flatten(2, 3).movedim(1, 2)[seen]
    return {"out": out.to(state["v"].dtype), "states": states}


# ---- exact results ------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _norm_exact, "rope": _rope_exact, "linear": _linear_exact}[case["kind"]](state)


def _f32(x):
    """Rounded to f32 where the definition rounds: sums, factors and codes are made of single f32 operations."""
    return x.float().double()


def _f32_of(x):
    return float(torch.tensor(x))


def _norm_exact(state):
    case, h, found = state["case"], state["x"].double(), {}
    if "residual" in state:
        h = _f32(h + state["residual"].double())
        found["residual"] = h
    root = torch.sqrt((h * h).mean(-1, keepdim=True) + _f32_of(EPS))
    w = state["weight"].double()
    if not case["quant"]:
        y = h / root * w
        if "gate" in state:
            y = y * state["gate"].double() * torch.sigmoid(state["gate"].double())
        return {"out": y, **found}
    y = _f32(_f32(h * _f32(1 / root)) * w).reshape(-1, 32)
    scale = _f32(y.abs().amax(-1, keepdim=True) / 127)
    steps = _f32(y * _f32(1 / scale))
    # halves go away from zero
    codes = torch.sign(steps) * torch.floor(_f32(steps.abs() + 0.5))
    return {"values": (codes.clamp(-128, 127) * scale.half().double()).reshape(-1), **found}


def _rope_exact(state):
    case, found = state["case"], {}
    freq, gain = _frequencies(case)
    half = case["rot"] // 2
    for name in ("q", "k"):
        y = state[name].double()
        z = y.clone()
        for i, f in enumerate(freq):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            turn = torch.polar(torch.full((case["tokens"], 1), gain, dtype=torch.float64, device="cuda"),
                               state["positions"].double()[:, None] * f)
            turned = torch.complex(y[..., a], y[..., b]) * turn
            z[..., a], z[..., b] = turned.real, turned.imag
        found[name] = z
    return found


def _linear_exact(state):
    """Token by token."""
    case, states = state["case"], state["states"].double()
    group, dk = case["v_heads"] // case["k_heads"], case["dk"]
    q, k = (state[name].double().repeat_interleave(group, 1) for name in "qk")
    v, keep = state["v"].double(), state["log_decay"].double().exp()
    beta = state["beta"].double() if case["delta"] else None
    out, offsets = torch.empty_like(v), state["offsets"].tolist()
    after = states.clone()
    for n, (source, slot) in enumerate(zip(state["source"].tolist(), state["slots"].tolist())):
        s = states[source].clone() if source >= 0 else torch.zeros_like(states[0])
        for t in range(offsets[n], offsets[n + 1]):
            s *= keep[t, :, None, None]
            u = v[t]
            if case["delta"]:
                u = (u - torch.matmul(k[t, :, None], s)[:, 0]) * beta[t, :, None]
            s.baddbmm_(k[t, :, :, None], u[:, None])
            out[t] = torch.matmul(q[t, :, None], s)[:, 0]
        after[slot] = s
    return {"out": out * dk ** -0.5, "states": after}
