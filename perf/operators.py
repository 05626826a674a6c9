"""Cases of the serving operators: prompt attention over packed sequences with grouped heads, and a key/value
cache held in 8 bits (written, read back, attended to).

The cache is four tensors: K codes ``[blocks, heads, tokens, dim]`` and V codes ``[blocks, heads, dim, tokens]`` in int8,
and a scale in f32 for each block and head of either. A sequence's position ``p`` lies in block
``block_table[sequence, p // tokens]``. A value ``x`` is held as ``rint(x / scale)``, where the scale is the largest
magnitude of the block's tokens (of that head) over 127, and at least 2^-100; when a token makes the scale of a block
grow, the codes of the older tokens become ``rint(code * old / new)``.
"""

import functools
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SMALLEST_SCALE = 2.0 ** -100


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # Prompts. Three short requests of a small model that arrived together: latency is all.
        {"name": "prompt_small", "op": "prompt", "dtype": "bf16", "batch": 3, "tokens": 170, "prefix": 0, "heads": 8,
         "kv_heads": 2, "dim": 64, "causal": True},
        # A batch of requests of uneven lengths, some with a part of their keys computed before (a later chunk of a prompt).
        {"name": "prompt_packed", "op": "prompt", "dtype": "bf16", "batch": 9, "tokens": 4099, "prefix": 300, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True},
        # One long document.
        {"name": "prompt_long", "op": "prompt", "dtype": "bf16", "batch": 1, "tokens": 8192, "prefix": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True},
        # f32, a head size that is no power of two, no mask (an encoder).
        {"name": "prompt_f32", "op": "prompt", "dtype": "f32", "batch": 5, "tokens": 1501, "prefix": 0, "heads": 6,
         "kv_heads": 6, "dim": 80, "causal": False},
        # One new token for each of many sequences, then what their last blocks hold.
        {"name": "append_tokens", "op": "append", "dtype": "bf16", "batch": 64, "length": 1000, "new": 1, "kv_heads": 8,
         "dim": 128, "block": 16},
        # Whole prompts into the cache.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "batch": 6, "length": 0, "new": 2731, "kv_heads": 8,
         "dim": 128, "block": 64},
        # A cached prefix read back: a short one in f32, and many long ones in bf16 before a further chunk of each.
        {"name": "read_small", "op": "read", "dtype": "f32", "batch": 3, "length": 333, "kv_heads": 2, "dim": 64, "block": 32},
        {"name": "read_prefixes", "op": "read", "dtype": "bf16", "batch": 12, "length": 4096, "kv_heads": 8, "dim": 128,
         "block": 64},
        # Single tokens. One conversation with a small model.
        {"name": "cached_small", "op": "cached", "dtype": "bf16", "batch": 1, "length": 777, "tokens": 1, "heads": 8,
         "kv_heads": 2, "dim": 64, "block": 16},
        # A serving batch with contexts of every length.
        {"name": "cached_batch", "op": "cached", "dtype": "bf16", "batch": 64, "length": 4096, "tokens": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 64},
        # A few very long contexts.
        {"name": "cached_long", "op": "cached", "dtype": "bf16", "batch": 4, "length": 131072, "tokens": 1, "heads": 64,
         "kv_heads": 8, "dim": 128, "block": 64},
        # Four proposed tokens a sequence, f32.
        {"name": "cached_proposed", "op": "cached", "dtype": "f32", "batch": 16, "length": 2048, "tokens": 4, "heads": 16,
         "kv_heads": 4, "dim": 128, "block": 32},
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "append", "read", "cached", "cached"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    block = rng.choice([16, 32, 64])
    if op == "prompt":
        if rng.random() < 0.3:
            dim = rng.choice([16, 40, 72, 80, 96, 112, 256])
        tokens = _spread(rng, 1, 6000 if dtype == "bf16" else 1500)
        return {"op": op, "dtype": dtype, "batch": min(tokens, _spread(rng, 1, 24)), "tokens": tokens,
                "prefix": rng.choice([0, 0, _spread(rng, 1, 700)]), "heads": kv_heads * rng.choice([1, 2, 3, 4]),
                "kv_heads": kv_heads, "dim": dim, "causal": rng.random() < 0.8}
    if op == "append":
        new = rng.choice([1, 1, _spread(rng, 2, 2700)])
        batch = _spread(rng, 1, 128) if new == 1 else _spread(rng, 1, 6)
        return {"op": op, "dtype": dtype, "batch": batch, "length": rng.choice([0, _spread(rng, 1, 900)]), "new": new,
                "kv_heads": kv_heads, "dim": dim, "block": block}
    if op == "read":
        return {"op": op, "dtype": dtype, "batch": _spread(rng, 1, 12), "length": _spread(rng, 1, 4000), "kv_heads": kv_heads,
                "dim": dim, "block": block}
    batch = _spread(rng, 1, 64)
    return {"op": op, "dtype": dtype, "batch": batch, "length": _spread(rng, 1, min(100000, 260000 // batch)),
            "tokens": rng.choice([1, 1, 1, 2, 4, 5]), "heads": kv_heads * rng.choice([1, 2, 4, 6, 8]), "kv_heads": kv_heads,
            "dim": dim, "block": block}


def _sizes(case):
    """Whole numbers that follow from the case alone, the same for every seed: lengths of the sequences."""
    op, batch = case["op"], case["batch"]
    if op == "prompt":
        # uneven parts of the tokens, one at least each
        weights = [1 + (7 * i + 3) % 5 for i in range(batch)]
        new = [1 + (case["tokens"] - batch) * w // sum(weights) for w in weights]
        new[0] += case["tokens"] - sum(new)
        return {"new": new, "keys": [n + (case["prefix"] * (i % 3) // 2) for i, n in enumerate(new)]}
    if op == "append":
        before = [max(0, case["length"] - (case["length"] * ((5 * i) % 8)) // 9) for i in range(batch)]
        new = [max(1, case["new"] - (case["new"] * ((3 * i) % 7)) // 9) for i in range(batch)]
        return {"before": before, "new": new, "after": [b + n for b, n in zip(before, new)]}
    # some sequences are whole, the others shorter, none empty
    return {"after": [max(1, case["length"] - (case["length"] * ((5 * i) % 8)) // 9) for i in range(batch)]}


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    s, h, d = _sizes(case), case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        pairs = sum(n * k - (n * (n - 1) // 2 if case["causal"] else 0) for n, k in zip(s["new"], s["keys"]))
        return {"bytes": size * d * (2 * sum(s["new"]) * case["heads"] + 2 * sum(s["keys"]) * h),
                "flops": 4 * d * case["heads"] * pairs}
    if case["op"] == "append":
        # new tokens in, their codes out; older tokens of the blocks and the new ones come back as f32
        held = sum(a - b // case["block"] * case["block"] for a, b in zip(s["after"], s["before"]))
        blocks = sum(-(-a // case["block"]) - b // case["block"] for a, b in zip(s["after"], s["before"]))
        return {"bytes": 2 * h * (d * sum(s["new"]) * (size + 1) + 4 * blocks + held * d * (1 + 4)), "flops": 0}
    blocks = sum(-(-a // case["block"]) for a in s["after"])
    held = 2 * h * (d * sum(s["after"]) + 4 * blocks)
    if case["op"] == "read":
        return {"bytes": held + 2 * h * d * sum(s["after"]) * size, "flops": 0}
    pairs = sum(max(0, a - i) for a in s["after"] for i in range(case["tokens"]))
    return {"bytes": held + 2 * size * case["batch"] * case["tokens"] * case["heads"] * d,
            "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, h, d, batch = _TYPES[case["dtype"]], case["kv_heads"], case["dim"], case["batch"]
    s = _sizes(case)
    state = {"case": case}

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dtype)

    def keys(n):
        # keys of a model: some channels are several times as large as the others
        return (torch.randn(n, h, d, generator=gen, device=dev) * (1 + 3 * (torch.arange(d, device=dev) % 16 == 5))).to(dtype)

    if case["op"] == "prompt":
        state.update(q=normal(case["tokens"], case["heads"], d), k=keys(sum(s["keys"])), v=normal(sum(s["keys"]), h, d),
                     offsets=ints(_offsets(s["new"])), k_offsets=ints(_offsets(s["keys"])))
        return state
    block = case["block"]
    each = [-(-a // block) for a in s["after"]]
    total = sum(each) + 1  # one block of the cache belongs to nobody
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)  # a sequence's blocks lie anywhere
    where = torch.zeros(batch, max(each), dtype=torch.int32)
    first = _offsets(each)
    for i, n in enumerate(each):
        where[i, :n] = torch.arange(first[i], first[i] + n)
    table = order[where.to(dev).long()]
    k_codes = torch.randint(-127, 128, (total, h, block, d), generator=gen, device=dev, dtype=torch.int8)
    v_codes = torch.randint(-127, 128, (total, h, d, block), generator=gen, device=dev, dtype=torch.int8)
    # codes of normal values are denser near zero than even ones are; the scales give the size of keys and values
    k_scales = 0.02 * (1 + torch.rand(total, h, generator=gen, device=dev))
    v_scales = 0.02 * (1 + torch.rand(total, h, generator=gen, device=dev))
    state.update(cache=(k_codes, v_codes, k_scales, v_scales), table=table.contiguous())
    if case["op"] == "append":
        starts = [b // block * block for b in s["before"]]
        state.update(k=keys(sum(s["new"])), v=normal(sum(s["new"]), h, d), offsets=ints(_offsets(s["new"])),
                     before=ints(s["before"]), after=ints(s["after"]), starts=ints(starts),
                     read_offsets=ints(_offsets([a - b for a, b in zip(s["after"], starts)])),
                     read_total=sum(s["after"]) - sum(starts))
    elif case["op"] == "read":
        state.update(starts=ints([0] * batch), after=ints(s["after"]), read_offsets=ints(_offsets(s["after"])),
                     read_total=sum(s["after"]))
    else:
        state.update(q=normal(batch, case["tokens"], case["heads"], d), after=ints(s["after"]))
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def _rows(offsets, count):
    """Of each of ``count`` packed rows: its sequence, and its place within that."""
    row = torch.arange(count, device=offsets.device)
    sequence = torch.searchsorted(offsets[1:].contiguous(), row.to(torch.int32), right=True)
    return sequence, row - offsets[sequence]


def _plain_prompt(q, k, v, offsets, k_offsets, causal):
    heads, h, d = q.shape[1], k.shape[1], q.shape[2]
    (qs, qi), (ks, ki) = _rows(offsets, q.shape[0]), _rows(k_offsets, k.shape[0])
    seen = qs[:, None] == ks[None, :]
    if causal:
        longer = (k_offsets[1:] - k_offsets[:-1]) - (offsets[1:] - offsets[:-1])
        seen &= ki[None, :] <= (qi + longer[qs])[:, None]
    grouped = q.float().reshape(q.shape[0], h, heads // h, d).permute(1, 2, 0, 3).reshape(h, -1, d)
    scores = (grouped @ k.float().permute(1, 2, 0)).reshape(h, heads // h, q.shape[0], -1)
    scores.mul_(d ** -0.5).masked_fill_(~seen, -torch.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.reshape(h, -1, k.shape[0]) @ v.float().permute(1, 0, 2)).reshape(h, heads // h, q.shape[0], d) / total
    return out.permute(2, 0, 1, 3).reshape(q.shape).to(q.dtype)


def _plain_append_one(codes, scales, x, tokens_last, table, before, offsets):
    """New tokens ``x`` into codes (``[blocks, heads, tokens, dim]``; seen so through a view) and scales."""
    held = codes.transpose(2, 3) if tokens_last else codes
    tokens = held.shape[2]
    sequence, place = _rows(offsets, x.shape[0])
    position = before[sequence] + place
    block, slot = table[sequence, position // tokens].long(), position % tokens
    largest = torch.zeros_like(scales).index_reduce_(0, block, x.float().abs().amax(-1), "amax")
    # blocks that hold older tokens of the sequence: their scale is a lower bound, their codes follow it
    last = table.gather(1, (before // tokens).clamp(max=table.shape[1] - 1).long()[:, None])[:, 0].long()
    older = before % tokens != 0
    floor = torch.zeros_like(scales)
    floor[last] = torch.where(older[:, None], scales[last], 0.0)
    new = torch.maximum(floor, (largest.double() / 127).float().clamp(min=_SMALLEST_SCALE))
    again = (held[last].double() * scales[last].double()[:, :, None, None] / new[last].double()[:, :, None, None]).round()
    held[last] = torch.where(older[:, None, None, None], again, held[last].double()).to(torch.int8)
    scales[block] = new[block]
    held[block, :, slot] = (x.double() / new[block].double()[:, :, None]).round().to(torch.int8)


def _plain_read_one(codes, scales, tokens_last, table, starts, offsets, total, dtype):
    held = codes.transpose(2, 3) if tokens_last else codes
    sequence, place = _rows(offsets, total)
    position = starts[sequence] + place
    block, slot = table[sequence, position // held.shape[2]].long(), position % held.shape[2]
    return (held[block, :, slot].float() * scales[block][:, :, None]).to(dtype)


def _plain_cached(q, cache, table, after):
    k_codes, v_codes, k_scales, v_scales = cache
    batch, n, heads, d = q.shape
    h, tokens = k_codes.shape[1:3]
    at = table.long()
    k = (k_codes[at].float() * k_scales[at][..., None, None]).transpose(1, 2).reshape(batch, h, -1, d)
    grouped = q.float().reshape(batch, n, h, heads // h, d).permute(0, 2, 3, 1, 4).reshape(batch, h, -1, d)
    scores = (grouped @ k.transpose(2, 3)).reshape(batch, h, heads // h, n, -1) * d ** -0.5
    del k
    position = torch.arange(table.shape[1] * tokens, device=q.device)
    limit = after[:, None] - n + 1 + torch.arange(n, device=q.device)
    seen = position[None, None, :] < limit[:, :, None]
    some = limit > 0
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = (v_codes[at].float() * v_scales[at][..., None, None]).permute(0, 2, 1, 4, 3).reshape(batch, h, -1, d)
    out = (p.reshape(batch, h, -1, p.shape[-1]) @ v).reshape(batch, h, heads // h, n, d) / torch.where(total > 0, total, 1.0)
    out = torch.where(some[:, None, None, :, None], out, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)


@functools.lru_cache(maxsize=1)
def _operators():
    """The framework's operator set (its folder's name is no name of a package)."""
    sys.path.insert(0, os.path.join(os.getcwd(), "helion-mlir-xsmm_b200"))
    import helion_mlir_utils

    return helion_mlir_utils


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        ops = _operators()
        if op == "prompt":
            return ops.attention_packed(s["q"], s["k"], s["v"], s["offsets"], s["k_offsets"], causal=case["causal"])
        if op == "cached":
            return ops.attention_cached(s["q"], s["cache"], s["table"], s["after"])
        if op == "append":
            ops.cache_append(s["cache"], s["k"], s["v"], s["table"], s["before"], s["offsets"])
            dtype = torch.float32
        else:
            dtype = _TYPES[case["dtype"]]
        return ops.cache_read(s["cache"], s["table"], s["starts"], s["after"], s["read_offsets"], s["read_total"], dtype)
    if op == "prompt":
        return _plain_prompt(s["q"], s["k"], s["v"], s["offsets"], s["k_offsets"], case["causal"])
    if op == "cached":
        return _plain_cached(s["q"], s["cache"], s["table"], s["after"])
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    if op == "append":
        _plain_append_one(k_codes, k_scales, s["k"], False, s["table"], s["before"], s["offsets"])
        _plain_append_one(v_codes, v_scales, s["v"], True, s["table"], s["before"], s["offsets"])
        dtype = torch.float32
    else:
        dtype = _TYPES[case["dtype"]]
    where = (s["table"], s["starts"], s["read_offsets"], s["read_total"], dtype)
    return _plain_read_one(k_codes, k_scales, False, *where), _plain_read_one(v_codes, v_scales, True, *where)


# ------------------------------------------------------------------------------------------------ definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        return _exact_prompt(s)
    if case["op"] == "cached":
        return _exact_cached(s)
    after, starts = s["after"].tolist(), s["starts"].tolist()
    if case["op"] == "append":
        return _exact_append(s, after, starts)
    found = [[], []]
    for b, (start, end) in enumerate(zip(starts, after)):
        for which, x in enumerate(_exact_sequence(s["cache"], s["table"][b], end)):
            found[which].append(x[start:])
    return tuple(torch.cat(x) for x in found)


def _exact_sequence(cache, row, length):
    """K and V of one sequence, ``[length, heads, dim]`` each."""
    k_codes, v_codes, k_scales, v_scales = cache
    blocks = row[: -(-length // k_codes.shape[2])].long()
    k = torch.einsum("nhtd,nh->nthd", k_codes[blocks].double(), k_scales[blocks].double())
    v = torch.einsum("nhdt,nh->nthd", v_codes[blocks].double(), v_scales[blocks].double())
    return k.flatten(0, 1)[:length], v.flatten(0, 1)[:length]


def _exact_attention(q, k, v, causal):
    """One sequence: ``q [n, heads, dim]``, ``k, v [m, kv_heads, dim]``; the queries are its last positions."""
    q, k, v = q.double(), k.double(), v.double()
    n, m, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
    out = torch.zeros_like(q)
    for head in range(q.shape[1]):
        p = torch.softmax((q[:, head] @ k[:, head // group].T / q.shape[2] ** 0.5).masked_fill(hidden, -torch.inf), -1)
        out[:, head] = p.nan_to_num(0.0) @ v[:, head // group]  # a row that sees nothing is zeros
    return out


def _exact_prompt(s):
    at, k_at = s["offsets"].tolist(), s["k_offsets"].tolist()
    return torch.cat([_exact_attention(s["q"][at[b]:at[b + 1]], s["k"][k_at[b]:k_at[b + 1]], s["v"][k_at[b]:k_at[b + 1]],
                                       s["case"]["causal"]) for b in range(len(at) - 1)])


def _exact_cached(s):
    out = [_exact_attention(s["q"][b], *_exact_sequence(s["cache"], s["table"][b], length), True)
           for b, length in enumerate(s["after"].tolist())]
    return torch.stack(out)


def _exact_append(s, after, starts):
    k_codes, v_codes, k_scales, v_scales = s["cache"]
    tokens = k_codes.shape[2]
    before, at = s["before"].tolist(), s["offsets"].tolist()
    found = [[], []]
    for which, (codes, scales, x) in enumerate(((k_codes, k_scales, s["k"]), (v_codes.transpose(2, 3), v_scales, s["v"]))):
        for b, (old, end) in enumerate(zip(before, after)):
            for start in range(starts[b], end, tokens):
                block, stop = int(s["table"][b, start // tokens]), min(start + tokens, end)
                first = max(old, start)  # the first new position of this block
                new = x[at[b] + first - old:at[b] + stop - old].double().transpose(0, 1)  # [heads, new, dim]
                scale = (new.abs().amax((1, 2)) / 127).clamp(min=_SMALLEST_SCALE).float().double()
                if first > start:
                    scale = torch.maximum(scale, scales[block].double())
                whole = torch.round(new / scale[:, None, None])
                if first > start:
                    kept = codes[block][:, :first - start].double() * scales[block].double()[:, None, None]
                    whole = torch.cat([torch.round(kept / scale[:, None, None]), whole], 1)
                found[which].append((whole * scale[:, None, None]).transpose(0, 1))
    return tuple(torch.cat(x) for x in found)
