"""The operators of a key/value cache held in 8 bits, as they are measured: inputs, plain forms and 64-bit results.

A model's attention layers keep the keys and values of every token.  Here they
are held as int8 in blocks of `block` tokens, with one f32 scale for each block
and head, in a pool that all sequences share:

    k, v              int8 [blocks, kv_heads, block, head_dim]
    k_scale, v_scale  f32  [blocks, kv_heads]            value = code * scale

A serving step takes, for sequence i, `cached[i]` tokens that are in the cache
and `new[i]` that arrive (packed one after the other), and does three things:

    tables     gives every sequence the blocks that its new tokens need and every
               new token its slot (block * block size + place in it)
    append     writes the new tokens' keys and values into their slots, after
               bringing the tokens that a block already holds to its new scale
    attention  lets each new token's query heads read the cached keys and values
               of its own sequence, causally, through the block table

Sizes are generic: the head layouts of small and middle models, block sizes that
pools use, lengths from one token to a long context.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: the most operations, bytes and scores (of the padded plain form) a drawn case may have
MOST_FLOPS, MOST_BYTES, MOST_SCORES = 5.4e11, 6.0e8, 2.1e9


def _batch(decodes=0, lo=1, hi=1, step=1, prompts=0, past_lo=0, past_hi=0, new_lo=1, new_hi=1, idle=0, lengths=0):
    """`decodes` sequences of lo..hi cached tokens that bring `step`, `prompts` of past_lo..past_hi that bring
    new_lo..new_hi, and `idle` rows of the batch that hold no sequence."""
    return {"decodes": decodes, "lo": lo, "hi": hi, "step": step, "prompts": prompts, "past_lo": past_lo,
            "past_hi": past_hi, "new_lo": new_lo, "new_hi": new_hi, "idle": idle, "lengths": lengths}


def listed():
    return [
        # the tables of a decode step: one token for each of 64 sequences
        {"name": "tables_decode", "kind": "tables", "block": 64, "width": 160, **_batch(64, 1, 8192)},
        # a step of a full server: decodes, arriving prompts, empty rows; small blocks
        {"name": "tables_mixed", "kind": "tables", "block": 16, "width": 1024,
         **_batch(700, 1, 12000, 1, 203, 0, 12000, 1, 4096, 97)},
        # the keys and values of a decode step
        {"name": "append_decode", "kind": "append", "block": 16, "heads": 8, "dim": 128, "type": "bf16", "pad": 0,
         **_batch(64, 1, 8192)},
        # three prompts that go on in the middle of a block, from f32 activations;
        # the last rows of the batch are padding
        {"name": "append_prompt", "kind": "append", "block": 64, "heads": 4, "dim": 256, "type": "f32", "pad": 7,
         **_batch(prompts=3, past_hi=300, new_lo=900, new_hi=2500)},
        # one token of a small model on a short context: the smallest call
        {"name": "attn_decode_one", "kind": "attention", "block": 64, "q_heads": 8, "heads": 2, "dim": 256, "type": "f32",
         "window": 0, **_batch(1, 333, 333)},
        # one token on a long context
        {"name": "attn_decode_long", "kind": "attention", "block": 128, "q_heads": 16, "heads": 4, "dim": 256,
         "type": "f32", "window": 0, **_batch(1, 131071, 131071)},
        # one token for each of 64 sequences of very different lengths
        {"name": "attn_decode_batch", "kind": "attention", "block": 64, "q_heads": 32, "heads": 8, "dim": 128,
         "type": "bf16", "window": 0, **_batch(64, 1, 8192)},
        # five draft tokens to be verified for each of 13 sequences; six query heads share a key head
        {"name": "attn_verify", "kind": "attention", "block": 32, "q_heads": 24, "heads": 4, "dim": 256, "type": "f16",
         "window": 0, **_batch(13, 500, 4000, 5)},
        # eight prompts of 16..256 tokens packed into one call, f32 activations
        {"name": "attn_prompt_ragged", "kind": "attention", "block": 64, "q_heads": 8, "heads": 2, "dim": 256,
         "type": "f32", "window": 0, **_batch(prompts=8, new_lo=16, new_hi=256)},
        # a chunk of a long prompt beside eleven decoding sequences
        {"name": "attn_mixed", "kind": "attention", "block": 64, "q_heads": 16, "heads": 2, "dim": 128, "type": "bf16",
         "window": 0, **_batch(11, 100, 6000, 1, 1, 5000, 5000, 1021, 1021)},
        # prompts under a sliding window, every query head with a key head of its own
        {"name": "attn_prompt_window", "kind": "attention", "block": 16, "q_heads": 12, "heads": 12, "dim": 64,
         "type": "f16", "window": 1024, **_batch(prompts=2, past_hi=700, new_lo=2500, new_hi=3500)},
        # a whole prompt of 8192 tokens: the largest call
        {"name": "attn_prompt_8k", "kind": "attention", "block": 64, "q_heads": 32, "heads": 8, "dim": 128, "type": "bf16",
         "window": 0, **_batch(prompts=1, new_lo=8192, new_hi=8192)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["tables", "append", "append", "decode", "decode", "verify", "prompt", "prompt", "mixed"])
    lengths, block = rng.randint(0, 9999), rng.choice([16, 32, 64, 128])
    if kind == "tables":
        hi = _log(rng, 64, 12000)
        b = _batch(_log(rng, 1, 1000), 1, hi, 1, rng.choice([0, _log(rng, 1, 200)]), 0, hi, 1, _log(rng, 2, 4096),
                   rng.choice([0, _log(rng, 1, 100)]), lengths)
        return {"kind": "tables", "block": block, "width": 17000 // block + rng.randint(0, 99), **b}
    dim, heads, dtype = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 4, 8, 12]), rng.choice(["f32", "f16", "bf16"])
    if kind == "append":
        if rng.random() < 0.5:
            b = _batch(_log(rng, 1, 512), 1, _log(rng, 2, 4096), rng.choice([1, 1, rng.randint(2, 9)]), lengths=lengths)
        else:
            b = _batch(_log(rng, 1, 32), 1, 4096, 1, _log(rng, 1, 8), 0, _log(rng, 1, 500), _log(rng, 1, 100),
                       _log(rng, 100, 3000), lengths=lengths)
        return {"kind": "append", "block": block, "heads": heads, "dim": dim, "type": dtype,
                "pad": rng.choice([0, rng.randint(1, 40)]), **b}
    group = rng.choice([1, 2, 3, 4, 4, 6, 8])
    if heads * group > 40:
        heads = max(1, 40 // group)
    window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
    if kind == "decode":
        n = _log(rng, 1, 256)
        hi = _log(rng, 16, min(131072, 2 ** 20 // n))
        b = _batch(n, rng.choice([1, hi // 2, hi]), hi, lengths=lengths)
    elif kind == "verify":
        b = _batch(_log(rng, 1, 64), 1, _log(rng, 64, 8192), rng.randint(2, 12), lengths=lengths)
    elif kind == "prompt":
        b = _batch(prompts=_log(rng, 1, 12), past_hi=rng.choice([0, _log(rng, 16, 4096)]), new_lo=_log(rng, 1, 64),
                   new_hi=_log(rng, 64, 8192), lengths=lengths)
    else:
        b = _batch(_log(rng, 1, 24), 1, _log(rng, 64, 8192), 1, rng.randint(1, 2), 0, _log(rng, 16, 4096), 64,
                   _log(rng, 64, 2048), lengths=lengths)
    return {"kind": "attention", "block": block, "q_heads": heads * group, "heads": heads, "dim": dim, "type": dtype,
            "window": window, **b}


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
            continue
        if case["kind"] == "attention":
            n = _lengths(case)
            if len(n) * case["q_heads"] * max(q for _, q in n) * max(c + q for c, q in n) > MOST_SCORES:
                continue
            if len(n) * case["heads"] * case["dim"] * max(c + q for c, q in n) > MOST_SCORES:
                continue
        return case


def _lengths(case):
    """(cached, new) tokens of each sequence."""
    rng = random.Random(case["lengths"])
    rows = [(_log(rng, case["lo"], case["hi"]), case["step"]) for _ in range(case["decodes"])]
    rows += [(rng.randint(case["past_lo"], case["past_hi"]), _log(rng, case["new_lo"], max(case["new_lo"], case["new_hi"])))
             for _ in range(case["prompts"])]
    return rows + [(0, 0)] * case["idle"]


def _ceil(a, b):
    return -(-a // b)


def work(case):
    """Bytes: each length, key, value and query once, each result once; flops: two products over the visible keys."""
    rows, block = _lengths(case), case["block"]
    total = sum(n for _, n in rows)
    if case["kind"] == "tables":
        blocks = sum(_ceil(c + n, block) - _ceil(c, block) for c, n in rows)
        # lengths in; offsets and lengths out; the new entries (read from the free
        # list, written into the table); a slot and a position for each new token
        return {"bytes": 4 * (4 * len(rows) + 2 * blocks + 2 * total), "flops": 0}
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["kind"] == "append":
        touched = sum(_ceil(c + n, block) - c // block for c, n in rows if n)
        token = case["heads"] * case["dim"]
        # new tokens in, codes out; then the touched blocks read back whole, as f32
        return {"bytes": 2 * (total * token * (size + 1) + touched * block * token * 5), "flops": 0}
    seen = pairs = 0
    window = case["window"] or 1 << 60
    for c, n in rows:
        seen += c + n - max(0, c + 1 - window)
        full = min(n, max(0, window - c))          # queries whose window reaches the sequence's start
        pairs += full * c + full * (full + 1) // 2 + (n - full) * min(window, c + n)
    kv = 2 * case["heads"] * case["dim"] * seen + 8 * case["heads"] * _ceil(seen, block)
    io = total * case["q_heads"] * (2 * size * case["dim"] + 4)
    return {"bytes": kv + io, "flops": 4 * case["q_heads"] * case["dim"] * pairs}


# ---- inputs ---------------------------------------------------------------------------

def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(shape, gen, loud):
    """int8 codes and block scales of normal values, some of whose channels are louder (as keys' are)."""
    x = torch.randn(shape, device="cuda", generator=gen)
    if loud:
        x[..., ::37] *= 3.0
    scale = x.abs().amax((2, 3)) / 127
    return (x / scale[..., None, None]).round_().to(torch.int8), scale


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)
    rows, block = _lengths(case), case["block"]
    rng.shuffle(rows)
    cached, new = [c for c, _ in rows], [n for _, n in rows]
    before, need = [_ceil(c, block) for c in cached], [_ceil(c + n, block) for c, n in rows]
    total = sum(new)
    width = case.get("width", max(max(need), 1))
    if width < max(need):
        raise ValueError("a sequence is longer than its row of the table")
    blocks = sum(need) + 5
    ids = torch.randperm(blocks, device="cuda", generator=gen).int().cpu()
    table, at = torch.full((len(rows), width), -1, dtype=torch.int32), 0
    held = before if case["kind"] == "tables" else need
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    state = {"case": case, "block": block, "tokens": total, "cached": _int(cached), "new": _int(new), "table": table.cuda()}
    if case["kind"] == "tables":
        # the free list lies behind what earlier steps have taken of it
        state["free"] = torch.cat([torch.full((3,), -1, dtype=torch.int32), ids[at:]]).cuda()
        state["taken"] = _int([3])
        return state
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    shape = (blocks, case["heads"], block, case["dim"])
    state["k"], state["k_scale"] = _codes(shape, gen, True)
    state["v"], state["v_scale"] = _codes(shape, gen, False)
    dtype = DTYPES[case["type"]]
    if case["kind"] == "append":
        slots, touched = [], []
        for i, (c, n) in enumerate(rows):
            entries = table[i].tolist()
            slots += [entries[p // block] * block + p % block for p in range(c, c + n)]
            touched += entries[c // block:need[i]] if n else []
        slots += [-1] * case["pad"]
        tokens = len(slots)
        state["slots"], state["touched"] = _int(slots), _int(sorted(touched))
        # one projection's output: each token's keys, then its values
        kv = torch.randn((tokens, 2, case["heads"], case["dim"]), device="cuda", generator=gen)
        kv[:, 0, :, ::37] *= 3.0
        kv[tokens - case["pad"]:] = math.nan          # rows of padding hold anything
        state["kv"] = kv.to(dtype)
        return state
    state["offsets"], state["kv_lens"] = _int(offsets), _int([c + n for c, n in rows])
    state["max_new"], state["max_kv"] = max(new), max(c + n for c, n in rows)
    state["q"] = torch.randn((total, case["q_heads"], case["dim"]), device="cuda", generator=gen).to(dtype)
    return state


# ---- one pass ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tables": _tables_own, "append": _append_own, "attention": _attention_own}[kind](state)
    return {"tables": _tables, "append": _append, "attention": _attention}[kind](state)


def _tables_own(state):
    from qwen35_amd import ops
    if "step" not in state:
        state["step"] = ops.KvStep(len(state["cached"]), state["tokens"], "cuda")
    s = state["step"]
    ops.kv_tables(state["cached"], state["new"], state["free"], state["table"], state["block"], s, taken=state["taken"])
    return {"table": state["table"], "offsets": s.offsets, "kv_lens": s.kv_lens, "slots": s.slots,
            "positions": s.positions, "taken": s.taken}


def _cache(state):
    from qwen35_amd import ops
    if "cache" not in state:
        state["cache"] = ops.KvCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state["cache"]


def _append_own(state):
    from qwen35_amd import ops
    cache, kv = _cache(state), state["kv"]
    ops.kv_append(cache, kv[:, 0], kv[:, 1], state["slots"])
    k, v = ops.kv_read(cache, state["touched"])
    return {"k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}


def _attention_own(state):
    from qwen35_amd import ops
    cache, case = _cache(state), state["case"]
    if "work" not in state:
        state["work"] = ops.kv_attention_work(cache, case["q_heads"], len(state["kv_lens"]), state["tokens"],
                                              state["max_new"], state["max_kv"])
    out, lse = ops.kv_attention(state["q"], cache, state["table"], state["offsets"], state["kv_lens"], state["max_new"],
                                state["max_kv"], window=case["window"], work=state["work"])
    return {"out": out, "lse": lse}


def _tables(state):
    block, table, cached, new, free = state["block"], state["table"], state["cached"], state["new"], state["free"]
    before, kv_lens = (cached + block - 1) // block, cached + new
    need = (kv_lens + block - 1) // block
    fresh = need - before
    first = state["taken"] + torch.cumsum(fresh, 0) - fresh
    j = torch.arange(table.shape[1], device="cuda")
    at = first[:, None] + j - before[:, None]
    entry = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], -1)
    table = torch.where((j >= before[:, None]) & (j < need[:, None]), entry, table)
    offsets = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)]).int()
    t = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(offsets.long(), t, right=True) - 1
    positions = cached[seq] + t - offsets[seq]
    entry = table[seq, positions // block]
    slots = torch.where(entry >= 0, entry * block + positions % block, -1)
    return {"table": table.int(), "offsets": offsets, "kv_lens": kv_lens, "slots": slots.int(), "positions": positions.int(),
            "taken": (state["taken"] + fresh.sum()).int()}


def _append_one(codes, scales, x, state):
    """New codes and scales of the touched blocks (the pool's are brought up to date), and the values they stand for."""
    block, touched, slots = state["block"], state["touched"].long(), state["slots"].long()
    n, places = len(touched), torch.arange(state["block"], device="cuda")
    x = x.float()
    # padding goes to a row of its own behind the touched blocks
    row = torch.where(slots >= 0, torch.searchsorted(touched, slots.clamp(min=0) // block), n)
    place = slots.clamp(min=0) % block
    first = torch.full((n + 1,), block, device="cuda").scatter_reduce(0, row, place, "amin")[:n]
    top = torch.zeros((n + 1, x.shape[1]), device="cuda")
    top = top.scatter_reduce(0, row[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")[:n]
    old = torch.where((first > 0)[:, None], scales[touched], 0)
    scale = torch.maximum(old, top / 127)
    held = codes[touched]
    ratio = torch.where(scale > 0, old / scale, 0)[..., None, None]
    keep = (places >= first[:, None])[:, None, :, None]
    held = torch.where(keep, held, (held.float() * ratio).round().to(torch.int8))
    inverse = torch.cat([torch.where(scale > 0, 1 / scale, 0), torch.zeros_like(top[:1])])
    new = (x * inverse[row][..., None]).round().clamp(-127, 127)
    grown = torch.cat([held, held[:1]])
    grown[row, :, place] = new.nan_to_num().to(torch.int8)
    codes[touched], scales[touched] = grown[:n], scale
    return grown[:n].float() * scale[..., None, None]


def _append(state):
    kv = state["kv"]
    k = _append_one(state["k"], state["k_scale"], kv[:, 0], state)
    v = _append_one(state["v"], state["v_scale"], kv[:, 1], state)
    return {"k": k, "v": v, "k_scale": state["k_scale"], "v_scale": state["v_scale"]}


def _attention(state):
    case, q, offsets, kv_lens = state["case"], state["q"], state["offsets"].long(), state["kv_lens"].long()
    heads, dim, longest, most = case["heads"], case["dim"], state["max_kv"], state["max_new"]
    group, n = case["q_heads"] // heads, len(kv_lens)
    ids = state["table"][:, :_ceil(longest, case["block"])].long().clamp(min=0)

    def gather(codes, scales):
        x = codes[ids].float() * scales[ids][..., None, None]
        return x.transpose(1, 2).reshape(n, heads, -1, dim)

    k, v = gather(state["k"], state["k_scale"]), gather(state["v"], state["v_scale"])
    counts = offsets[1:] - offsets[:-1]
    i, j = torch.arange(most, device="cuda"), torch.arange(k.shape[2], device="cuda")
    rows = (offsets[:-1, None] + i).clamp(max=state["tokens"] - 1)
    qs = q[rows].float().reshape(n, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, -1, dim)
    s = torch.matmul(qs, k.transpose(2, 3)).mul_(1 / math.sqrt(dim)).reshape(n, heads, group, most, -1)
    at = (kv_lens - counts)[:, None] + i                                 # the query's own place
    seen = (j <= at[..., None]) & (j < kv_lens[:, None, None])
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, heads, group * most, -1), v).reshape(n, heads, group, most, dim) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    # packed rows: [sequence, head, group, query] -> [token, query head]
    t = torch.arange(state["tokens"], device="cuda")
    seq = torch.searchsorted(offsets, t, right=True) - 1
    at = t - offsets[seq]
    out = out.permute(0, 3, 1, 2, 4)[seq, at].reshape(-1, case["q_heads"], dim)
    return {"out": out.to(q.dtype), "lse": lse.permute(0, 3, 1, 2)[seq, at].reshape(-1, case["q_heads"])}


# ---- exact results ------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"tables": _tables_exact, "append": _append_exact, "attention": _attention_exact}[case["kind"]](state)


def _tables_exact(state):
    """Block by block and token by token, as the step is defined."""
    block, table, free = state["block"], state["table"].tolist(), state["free"].tolist()
    taken, offsets, kv_lens, slots, positions = int(state["taken"]), [0], [], [], []
    for row, c, n in zip(table, state["cached"].tolist(), state["new"].tolist()):
        for j in range(_ceil(c, block), _ceil(c + n, block)):
            row[j] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(c, c + n):
            entry = row[p // block]
            slots.append(entry * block + p % block if entry >= 0 else -1)
            positions.append(p)
        offsets.append(offsets[-1] + n)
        kv_lens.append(c + n)
    return {"table": _int(table), "offsets": _int(offsets), "kv_lens": _int(kv_lens), "slots": _int(slots),
            "positions": _int(positions), "taken": _int([taken])}


def _f32(x):
    """Rounded to f32 where the definition rounds: scales and codes are made of single f32 operations."""
    return x.float().double()


def _append_exact(state):
    block, dtype = state["block"], torch.float64
    places = {}
    for t, slot in enumerate(state["slots"].tolist()):
        if slot >= 0:
            places.setdefault(slot // block, []).append((slot % block, t))
    found = {}
    for part, name in enumerate("kv"):
        codes, scales, x = state[name].clone(), state[name + "_scale"].to(dtype), state["kv"][:, part].to(dtype)
        values = []
        for b in state["touched"].tolist():
            at, t = (list(c) for c in zip(*places[b]))
            old = scales[b] if min(at) > 0 else torch.zeros_like(scales[b])
            scale = torch.maximum(old, _f32(x[t].abs().amax((0, 2)) / 127))
            safe = torch.where(scale > 0, scale, 1)[:, None, None]
            now = codes[b].to(dtype)
            kept = min(at)
            now[:, :kept] = _f32(now[:, :kept] * _f32(old[:, None, None] / safe)).round()
            now[:, at] = _f32(x[t].transpose(0, 1) * _f32(1 / safe)).round().clamp(-127, 127)
            scales[b] = scale
            values.append(now * scale[:, None, None])
        found[name], found[name + "_scale"] = torch.stack(values), scales
    return found


def _attention_exact(state):
    case, block, dim = state["case"], state["block"], state["case"]["dim"]
    group = case["q_heads"] // case["heads"]
    q, offsets = state["q"].double(), state["offsets"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for i, length in enumerate(state["kv_lens"].tolist()):
        a, b = offsets[i], offsets[i + 1]
        if a == b:
            continue
        ids = state["table"][i, :_ceil(length, block)].long()
        for h in range(case["heads"]):
            k = (state["k"][ids, h].double() * state["k_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
            v = (state["v"][ids, h].double() * state["v_scale"][ids, h].double()[:, None, None]).reshape(-1, dim)[:length]
            for c in range(a, b, 2048):  # a piece of the queries at a time
                e = min(b, c + 2048)
                at = torch.arange(length - b + c, length - b + e, device="cuda")[:, None]
                j = torch.arange(length, device="cuda")
                hidden = (j > at) | ((j <= at - case["window"]) if case["window"] else torch.zeros_like(j > at))
                for g in range(h * group, (h + 1) * group):
                    s = (q[c:e, g] @ k.T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
                    lse[c:e, g] = torch.logsumexp(s, -1)
                    out[c:e, g] = torch.softmax(s, -1) @ v
    return {"out": out, "lse": lse}
