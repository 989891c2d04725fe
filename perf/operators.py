"""Performance cases of the 8-bit key/value cache and what goes with it: rotary positions, writing tokens and reading them
back, and attention over the cache.

The cache of one attention layer keeps, for every sequence and key/value head, blocks of 32 tokens.  A block that is full is
held as 8-bit codes with one FP32 scale for its keys and one for its values:

    scale = max |x| / 127 over the block's 32 x head_dim numbers,  code = round_half_even(127 x / max |x|),  value = code * scale

and a block that is not full yet is held as it came.  So what the cache holds depends on the tokens alone, not on how many came
at a time.  Head counts and head sizes are those of TinyLlama-1.1B (32 query and 4 key/value heads of 64) and Llama-70B (64 and 8 of
128), which the benchmark uses, and generic ones around them.

A case is one of
  rotary     rotary positions of queries and keys, ``apply_rotary``
  append     tokens written into the cache and what was written read back, ``QuantizedKVCache.append`` and ``.read``
  read       a whole cache read back, ``QuantizedKVCache.read``
  attention  attention of the newest tokens over the cache, ``QuantizedKVCache.attention``
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rotary(name, tokens, heads, head_dim, rotary_dim, interleaved, scale, furthest, dtype):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "scale": scale, "furthest": furthest, "dtype": dtype}


def _append(name, batch, tokens, kv_heads, head_dim, start, ragged, dtype):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "start": start, "ragged": ragged, "dtype": dtype}


def _read(name, batch, length, kv_heads, head_dim, ragged, dtype):
    return {"name": name, "op": "read", "batch": batch, "length": length, "kv_heads": kv_heads, "head_dim": head_dim,
            "ragged": ragged, "dtype": dtype}


def _attention(name, batch, tokens, length, q_heads, kv_heads, head_dim, ragged, dtype):
    return {"name": name, "op": "attention", "batch": batch, "tokens": tokens, "length": length, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged, "dtype": dtype}


def listed():
    return [
        # Queries and keys of one decoded token of a small model.
        _rotary("rotary_tl_token", 1, 36, 64, 64, False, 1.0, 1500, "fp16"),
        # Queries and keys of a long prompt's chunk far into a context; adjacent pairs, three quarters of the head turned,
        # cosines and sines scaled as for a stretched context.
        _rotary("rotary_70b_prompt_partial", 4096, 72, 128, 96, True, 1.2079441541679836, 131071, "bf16"),
        # One token into the cache of a small model: the write of every decode step.
        _append("append_tl_token", 1, 1, 4, 64, 1503, False, "fp16"),
        # Drafted tokens of a serving batch, one to five for each sequence, at any place within a block.
        _append("append_70b_drafts_b32", 32, 5, 8, 128, 2500, True, "bf16"),
        # Two prompts of 8191 tokens.
        _append("append_70b_prompt", 2, 8191, 8, 128, 0, False, "fp16"),
        # The cache of a short conversation read back, as for handing it to another process.
        _read("read_tl_777", 1, 777, 4, 64, False, "fp16"),
        # A long context read back.
        _read("read_70b_32k", 1, 32768, 8, 128, False, "fp16"),
        # One token of a small model, short context: latency is all.
        _attention("attn_tl_token_500", 1, 1, 500, 32, 4, 64, False, "fp16"),
        # One token of a large model over a long context of odd length.
        _attention("attn_70b_token_64k", 1, 1, 65501, 64, 8, 128, False, "fp16"),
        # One token for each of 48 sequences with contexts of every length.
        _attention("attn_70b_batch48", 48, 1, 8192, 64, 8, 128, True, "fp16"),
        # Five drafted tokens for each of eight sequences of a small model.
        _attention("attn_tl_drafts_b8", 8, 5, 2900, 32, 4, 64, True, "bf16"),
        # The last chunk of a prompt.
        _attention("attn_70b_prompt_chunk", 1, 2048, 8192, 64, 8, 128, False, "fp16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))) - 0.5))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "read", "attention", "attention", "attention"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "rotary":
        head_dim = rng.choice((64, 128))
        heads = _log_int(rng, 1, 80)
        return _without_name(_rotary("", _log_int(rng, 1, min(16384, 4096 * 72 * 128 // (heads * head_dim))), heads, head_dim,
                                     2 * rng.randint(head_dim // 8, head_dim // 2), rng.random() < 0.5, rng.choice((1.0, 1.1)),
                                     _log_int(rng, 64, 1 << 20), dtype))
    q_heads, kv_heads = rng.choice(((32, 4), (64, 8), (8, 8), (12, 2), (40, 8), (16, 1)))
    head_dim = rng.choice((64, 128))
    wide = kv_heads * head_dim
    if kind == "append":
        batch = _log_int(rng, 1, 64)
        tokens = _log_int(rng, 1, 2 * 8191 * 1024 // (wide * batch))
        # (prompts come in chunks of whole blocks, a few tokens at any place)
        start = rng.randint(0, 4000) if tokens <= BLOCK else BLOCK * rng.randint(0, 100)
        return _without_name(_append("", batch, tokens, kv_heads, head_dim, start, rng.random() < 0.5, dtype))
    if kind == "read":
        batch = _log_int(rng, 1, 16)
        return _without_name(_read("", batch, _log_int(rng, 1, 32768 * 1024 // (wide * batch)), kv_heads, head_dim,
                                   rng.random() < 0.5, dtype))
    form = rng.choice(("token", "token", "drafts", "chunk"))
    if form == "chunk":
        tokens = _log_int(rng, 33, 2048)
        length = tokens + rng.randint(0, 6144)
        return _without_name(_attention("", 1, tokens, length, q_heads, kv_heads, head_dim, False, dtype))
    batch = _log_int(rng, 1, 64)
    tokens = 1 if form == "token" else rng.randint(2, 12)
    length = _log_int(rng, tokens, max(tokens, min(65536, 48 * 4096 * 1024 // (wide * batch))))
    return _without_name(_attention("", batch, tokens, length, q_heads, kv_heads, head_dim, batch > 1 and rng.random() < 0.7,
                                    dtype))


def _without_name(case):
    return {key: value for key, value in case.items() if key != "name"}


# ------------------------------------------------------------------ what a case implies


def _lengths(case):
    """Tokens in the cache of each sequence, the newest included; for a write, before it."""
    rng = random.Random(f"{case['op']} {case['batch']} {case['ragged']}")
    if case["op"] == "append":
        top, low = case["start"], 0
        if case["tokens"] > BLOCK:
            return [case["start"]] * case["batch"]
    else:
        top, low = case["length"], case.get("tokens", 1)
    if not case["ragged"]:
        return [top] * case["batch"]
    return [top] + [rng.randint(low, top) for _ in range(case["batch"] - 1)]


def _counts(case):
    """New tokens of each sequence."""
    rng = random.Random(f"{case['op']} {case['batch']} {case['ragged']} counts")
    if not case["ragged"]:
        return [case["tokens"]] * case["batch"]
    return [case["tokens"]] + [rng.randint(1, case["tokens"]) for _ in range(case["batch"] - 1)]


def _held_bytes(length, kv_heads, head_dim):
    """What the cache holds of one sequence: full blocks in 8 bits with two scales, the rest in 16 bits."""
    full = length // BLOCK
    return kv_heads * (full * (2 * BLOCK * head_dim + 8) + (length - full * BLOCK) * head_dim * 4)


def work(case):
    if case["op"] == "rotary":
        numbers = case["tokens"] * case["heads"] * case["head_dim"]
        turned = case["tokens"] * case["heads"] * case["rotary_dim"]
        return {"bytes": 4 * numbers + 8 * case["tokens"] + 2 * case["rotary_dim"], "flops": 3 * turned}
    kv_heads, head_dim = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        total = flops = 0
        for start, count in zip(_lengths(case), _counts(case)):
            row = kv_heads * head_dim
            older = start % BLOCK if start // BLOCK != (start + count) // BLOCK else 0     # of a block that becomes full
            total += 4 * row * (count + older)                                           # read
            total += _held_bytes(start + count, kv_heads, head_dim) - _held_bytes(start - start % BLOCK, kv_heads, head_dim)
            total += 4 * row * case["tokens"]                                            # what was written, read back
            flops += 4 * row * count
        return {"bytes": total, "flops": flops}
    lengths = _lengths(case)
    held = sum(_held_bytes(length, kv_heads, head_dim) for length in lengths)
    if case["op"] == "read":
        return {"bytes": held + 4 * case["batch"] * case["length"] * kv_heads * head_dim,
                "flops": 2 * sum(lengths) * kv_heads * head_dim}
    pairs = 0
    for length, count in zip(lengths, _counts(case)):
        pairs += count * length - count * (count - 1) // 2
    rows = case["batch"] * case["tokens"] * case["q_heads"]
    return {"bytes": held + 4 * rows * head_dim, "flops": 4 * pairs * case["q_heads"] * head_dim}


# ------------------------------------------------------------------ inputs


def _keys(shape, g, dtype):
    """Keys as models have them: a spread and an offset of their own for every channel, a few channels far out."""
    spread = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device=DEVICE))
    offset = torch.randn(shape[-2:], generator=g, device=DEVICE)
    offset = torch.where(torch.rand(shape[-2:], generator=g, device=DEVICE) < 0.03, 6.0 * offset, 0.3 * offset)
    return torch.randn(shape, generator=g, device=DEVICE).mul_(spread).add_(offset).to(dtype)


def _values(shape, g, dtype):
    spread = torch.exp(0.3 * torch.randn(shape[-2:], generator=g, device=DEVICE))
    return torch.randn(shape, generator=g, device=DEVICE).mul_(spread).to(dtype)


def _int64(values):
    return torch.tensor(values, dtype=torch.long, device=DEVICE)


def _inputs(case, seed):
    """Everything random, the same for every form."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        tokens = case["tokens"]
        inverse = 10000.0 ** (-torch.arange(0, case["rotary_dim"], 2, dtype=torch.float64) / case["rotary_dim"])
        last = case["furthest"] - int(torch.randint(0, 64, (1,), generator=g, device=DEVICE))
        return {"x": torch.randn((tokens, case["heads"], case["head_dim"]), generator=g, device=DEVICE).to(dtype),
                "positions": (torch.arange(tokens, device=DEVICE) + (last - tokens + 1)).clamp_(min=0),
                "inv_freq": inverse.float().to(DEVICE)}
    batch, kv_heads, head_dim = case["batch"], case["kv_heads"], case["head_dim"]
    lengths = _lengths(case)
    if case["op"] == "append":
        shape = (batch, case["tokens"], kv_heads, head_dim)
        held = (batch, BLOCK, kv_heads, head_dim)         # of the block that is being filled: the first start % 32 tokens
        return {"k": _keys(shape, g, dtype), "v": _values(shape, g, dtype), "older_k": _keys(held, g, dtype),
                "older_v": _values(held, g, dtype), "start": _int64(lengths), "counts": _int64(_counts(case))}
    shape = (batch, case["length"], kv_heads, head_dim)
    made = {"k": _keys(shape, g, dtype), "v": _values(shape, g, dtype), "lengths": _int64(lengths)}
    if case["op"] == "attention":
        made["q"] = torch.randn((batch, case["tokens"], case["q_heads"], head_dim), generator=g, device=DEVICE).to(dtype)
        made["counts"] = _int64(_counts(case))
    return made


def _to_blocks(x, lengths):
    """[batch, length, heads, d] -> codes [batch, heads, blocks, 32, d], scales [batch, heads, blocks] and the newest, unfilled
    block of every sequence [batch, heads, 32, d] as it came."""
    batch, length, heads, d = x.shape
    padded = torch.zeros((batch, (length // BLOCK + 1) * BLOCK, heads, d), dtype=x.dtype, device=x.device)
    padded[:, :length] = x
    padded = padded.view(batch, -1, BLOCK, heads, d).permute(0, 3, 1, 2, 4)
    newest = lengths // BLOCK
    tail = padded[torch.arange(batch, device=x.device), :, newest].contiguous()
    codes = torch.empty(padded.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(padded.shape[:3], dtype=torch.float32, device=x.device)
    for b in range(batch):
        wide = padded[b].float()
        top = wide.abs().amax((-1, -2))
        scales[b] = top / 127.0
        codes[b] = (wide * 127.0 / torch.where(top > 0, top, 1.0)[..., None, None]).round().to(torch.int8)
    return codes, scales, tail


def prepare(case, seed):
    made = _inputs(case, seed)
    if case["op"] == "rotary":
        return {"case": case, **made}
    if own:
        from nibble_b200 import QuantizedKVCache

        if case["op"] == "append":
            ends = made["start"] + made["counts"]
            cache = QuantizedKVCache(case["batch"], case["kv_heads"], case["start"] + case["tokens"], case["head_dim"],
                                     dtype=made["k"].dtype, device=DEVICE)
            inside = made["start"] % BLOCK
            cache.append(made["older_k"], made["older_v"], made["start"] - inside, inside)
            return {"case": case, "cache": cache, "k": made["k"], "v": made["v"], "start": made["start"],
                    "counts": made["counts"], "ends": ends}
        cache = QuantizedKVCache(case["batch"], case["kv_heads"], case["length"], case["head_dim"], dtype=made["k"].dtype,
                                 device=DEVICE)
        cache.append(made["k"], made["v"], torch.zeros_like(made["lengths"]), made["lengths"])
        return {"case": case, "cache": cache, "lengths": made["lengths"], "q": made.get("q"), "counts": made.get("counts")}
    if case["op"] == "append":
        return {"case": case, **made}
    state = {"case": case, "lengths": made["lengths"], "q": made.get("q"), "counts": made.get("counts")}
    for name in ("k", "v"):
        state[name + "_codes"], state[name + "_scales"], state[name + "_tail"] = _to_blocks(made[name], made["lengths"])
    return state


# ------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if own:
        if case["op"] == "rotary":
            from nibble_b200 import apply_rotary

            return apply_rotary(state["x"], state["positions"], state["inv_freq"], scale=case["scale"],
                                interleaved=case["interleaved"])
        cache = state["cache"]
        if case["op"] == "append":
            cache.append(state["k"], state["v"], state["start"], state["counts"])
            return cache.read(state["ends"], first=state["start"], tokens=case["tokens"])
        if case["op"] == "read":
            return cache.read(state["lengths"])
        return cache.attention(state["q"], state["lengths"], state["counts"])
    return {"rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}[case["op"]](state)


def _plain_rotary(state):
    case, x = state["case"], state["x"]
    turned = case["rotary_dim"]
    angles = state["positions"].double()[:, None] * state["inv_freq"].double()
    cos = (angles.cos() * case["scale"]).float()[:, None]
    sin = (angles.sin() * case["scale"]).float()[:, None]
    wide = x.float()
    if case["interleaved"]:
        a, b = wide[..., 0:turned:2], wide[..., 1:turned:2]
    else:
        a, b = wide[..., :turned // 2], wide[..., turned // 2:turned]
    first, second = a * cos - b * sin, b * cos + a * sin
    front = torch.stack((first, second), -1).flatten(-2) if case["interleaved"] else torch.cat((first, second), -1)
    return torch.cat((front, wide[..., turned:]), -1).to(x.dtype)


def _plain_append(state):
    """The tokens from `start` on as the cache holds them afterwards; zeros behind a sequence's last."""
    k, start, counts = state["k"], state["start"], state["counts"]
    batch, tokens, heads, d = k.shape
    inside = start % BLOCK
    slots = (tokens + BLOCK - 1 + BLOCK - 1) // BLOCK * BLOCK          # from the beginning of the first block on
    place = torch.arange(slots, device=k.device) - inside[:, None]       # of a slot among the new tokens
    is_new = (place >= 0) & (place < counts[:, None])
    at = place.clamp(0, tokens - 1)[..., None, None].expand(-1, -1, heads, d)
    back = (inside[:, None] + torch.arange(tokens, device=k.device))[..., None, None].expand(-1, -1, heads, d)
    asked = (torch.arange(tokens, device=k.device) < counts[:, None])[..., None, None]
    full = torch.arange(slots // BLOCK, device=k.device) < ((inside + counts) // BLOCK)[:, None]
    outputs = []
    for name in ("k", "v"):
        held = torch.zeros((batch, slots, heads, d), dtype=torch.float32, device=k.device)
        held[:, :BLOCK] = torch.where((place[:, :BLOCK] < 0)[..., None, None], state["older_" + name].float(), 0.0)
        held = torch.where(is_new[..., None, None], state[name].float().gather(1, at), held)
        blocks = held.view(batch, -1, BLOCK, heads, d)
        top = blocks.abs().amax((2, 4), keepdim=True)
        codes = (blocks * 127.0 / torch.where(top > 0, top, 1.0)).round()
        blocks = torch.where(full[..., None, None, None], codes * (top / 127.0), blocks)
        outputs.append(torch.where(asked, blocks.reshape(batch, slots, heads, d).gather(1, back), 0.0).to(k.dtype))
    return tuple(outputs)


def _plain_held(state, name, b=None):
    """What the cache holds, FP32 [batch, heads, blocks * 32, d]; of one sequence [heads, blocks * 32, d]."""
    codes, scales, tail = (state[name + part] for part in ("_codes", "_scales", "_tail"))
    lengths = state["lengths"]
    if b is not None:
        codes, scales, tail, lengths = codes[b:b + 1], scales[b:b + 1], tail[b:b + 1], lengths[b:b + 1]
    held = codes.float() * scales[..., None, None]
    held[torch.arange(lengths.numel(), device=held.device), :, lengths // BLOCK] = tail.float()
    held = held.flatten(2, 3)
    return held if b is None else held[0]


def _plain_read(state):
    case = state["case"]
    asked = (torch.arange(case["length"], device=DEVICE) < state["lengths"][:, None])[..., None, None]
    return tuple(torch.where(asked, _plain_held(state, name)[:, :, :case["length"]].transpose(1, 2), 0.0).to(_DTYPES[case["dtype"]])
                 for name in ("k", "v"))


def _plain_attention(state):
    """Query i of a sequence stands at position length - count + i and sees the positions up to its own."""
    case, q = state["case"], state["q"]
    batch, tokens, q_heads, d = q.shape
    kv_heads = case["kv_heads"]
    group = q_heads // kv_heads
    out = torch.empty((batch, tokens, q_heads, d), dtype=torch.float32, device=q.device)
    for b in range(batch):
        k, v = _plain_held(state, "k", b), _plain_held(state, "v", b)
        rows = q[b].float().view(tokens, kv_heads, group, d).permute(1, 2, 0, 3).reshape(kv_heads, group * tokens, d)
        scores = torch.matmul(rows, k.transpose(1, 2)).mul_(d ** -0.5).view(kv_heads, group, tokens, -1)
        last = (state["lengths"][b] - state["counts"][b]) + torch.arange(tokens, device=q.device)
        scores.masked_fill_(torch.arange(k.shape[1], device=q.device) > last[:, None], -math.inf)
        scores = scores.view(kv_heads, group * tokens, -1)
        scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        total = scores.sum(-1, keepdim=True)
        seen = torch.arange(k.shape[1], device=q.device) < state["lengths"][b]
        rows = torch.matmul(scores, torch.where(seen[:, None], v, 0.0)) / total
        out[b] = rows.view(kv_heads, group, tokens, d).permute(2, 0, 1, 3).reshape(tokens, q_heads, d)
    asked = (torch.arange(tokens, device=q.device) < state["counts"][:, None])[..., None, None]
    return torch.where(asked, out, 0.0).to(q.dtype)


# ------------------------------------------------------------------ the same from the definitions, in 64 bits


def _held_exactly(numbers, length):
    """[tokens, heads, d] in 64 bits -> what a cache of `length` tokens holds of them (the first stands at a block's begin)."""
    held = numbers.clone()
    for begin in range(0, length - BLOCK + 1, BLOCK):
        block = held[begin:begin + BLOCK]                     # (a view: written in place)
        top = block.abs().amax(dim=(0, 2), keepdim=True)
        steps = torch.round(block / torch.where(top == 0, torch.ones_like(top), top) * 127.0)
        exact_tie = (block * 254.0) / torch.where(top == 0, torch.ones_like(top), top)
        # a quotient that lies on a tie goes to the even code: 254 x / top is an odd integer there
        tie = (exact_tie == torch.round(exact_tie)) & (torch.remainder(exact_tie, 2.0) == 1.0)
        even = 2.0 * torch.round((exact_tie / 2.0) / 2.0)
        block.copy_(torch.where(tie, even, steps) * top / 127.0)
    return held


def exact(case, seed):
    made = _inputs(case, seed)
    if case["op"] == "rotary":
        x = made["x"].double()
        half = case["rotary_dim"] // 2
        out = x.clone()
        for j in range(half):
            angle = made["positions"].double() * made["inv_freq"][j].double()
            c, s = (torch.cos(angle) * case["scale"])[:, None], (torch.sin(angle) * case["scale"])[:, None]
            one, two = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
            out[..., one] = x[..., one] * c - x[..., two] * s
            out[..., two] = x[..., two] * c + x[..., one] * s
        return out
    if case["op"] == "append":
        outputs = []
        for name in ("k", "v"):
            out = torch.zeros(made[name].shape, dtype=torch.float64, device=DEVICE)
            for b, (start, count) in enumerate(zip(_lengths(case), _counts(case))):
                inside = start % BLOCK
                numbers = torch.cat((made["older_" + name][b, :inside], made[name][b, :count])).double()
                out[b, :count] = _held_exactly(numbers, inside + count)[inside:]
            outputs.append(out)
        return tuple(outputs)
    if case["op"] == "read":
        outputs = []
        for name in ("k", "v"):
            out = torch.zeros(made[name].shape, dtype=torch.float64, device=DEVICE)
            for b, length in enumerate(_lengths(case)):
                out[b, :length] = _held_exactly(made[name][b, :length].double(), length)
            outputs.append(out)
        return tuple(outputs)
    q = made["q"].double()
    batch, tokens, q_heads, d = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
    for b, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
        k = _held_exactly(made["k"][b, :length].double(), length)
        v = _held_exactly(made["v"][b, :length].double(), length)
        places = torch.arange(length, device=DEVICE)
        hidden = places[None, :] > (length - count + torch.arange(count, device=DEVICE))[:, None]
        for head in range(q_heads):
            kv = head // (q_heads // case["kv_heads"])
            scores = (q[b, :count, head] @ k[:, kv].T) / math.sqrt(d)
            out[b, :count, head] = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1) @ v[:, kv]
    return out
