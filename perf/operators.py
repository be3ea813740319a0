"""Performance cases of the operators of a 4-bit key/value cache and of 4-bit products.

A reader model that answers over retrieved passages keeps their keys and values
in the framework's int4 row format: one scale per token and head, s = max|x| / 7
in single precision (1 for a row of zeros), codes clip(rint(x / s), -7, 7),
two's complement nibbles with the even dim low.  Rows live in pages of a pool;
a sequence is a row of a page table and a length.

Operators:
  store    new key and value rows quantised into the cache, and read back
  read     rows of sequences read back from the cache
  attend   attention of new tokens over the cache, shared key/value heads
  linear   x W^T with W in 4 bits and a scale per group of a row

``own`` chooses between the framework's entry points and the plain form of the
same formulas in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decoding step of a batch: a token per sequence enters the cache.
        {"name": "store_step", "op": "store", "batch": 32, "lo": 100, "hi": 4000, "new": 1, "kv_heads": 8, "dim": 128,
         "page": 64, "type": "bf16"},
        # Prompts of ragged lengths enter the cache, some behind a prefix that is there.
        {"name": "store_prompts", "op": "store", "batch": 12, "lo": 300, "hi": 6000, "new": 0, "kv_heads": 8,
         "dim": 128, "page": 16, "type": "f16"},
        # The cache of a few passages read back, to be moved or recomputed.
        {"name": "read_passages", "op": "read", "batch": 9, "lo": 64, "hi": 700, "kv_heads": 4, "dim": 96, "page": 32,
         "type": "f32"},
        # Long sequences read back whole.
        {"name": "read_long", "op": "read", "batch": 4, "lo": 8000, "hi": 33000, "kv_heads": 8, "dim": 128,
         "page": 64, "type": "bf16"},
        # One user, one token, a short context: latency.
        {"name": "attend_first", "op": "attend", "batch": 1, "lo": 391, "hi": 391, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "window": 0, "mask": False},
        # A decoding batch over ragged contexts.
        {"name": "attend_step", "op": "attend", "batch": 32, "lo": 100, "hi": 8000, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "window": 0, "mask": False},
        # Few sequences, very long contexts.
        {"name": "attend_long", "op": "attend", "batch": 3, "lo": 100001, "hi": 131072, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "f16", "window": 0, "mask": False},
        # Five drafted tokens per sequence under a mask of their own, one key/value
        # head per query head, single precision.
        {"name": "attend_drafts", "op": "attend", "batch": 7, "lo": 33, "hi": 3001, "new": 5, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "type": "f32", "window": 0, "mask": True},
        # A piece of a long prompt behind the pieces before it.
        {"name": "attend_prompt", "op": "attend", "batch": 2, "lo": 9000, "hi": 17000, "new": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "window": 0, "mask": False},
        # One token through a square projection.
        {"name": "linear_token", "op": "linear", "rows": 1, "out": 4096, "in": 4096, "group": 128, "type": "bf16"},
        # A decoding batch through a wide one.
        {"name": "linear_batch", "op": "linear", "rows": 16, "out": 28672, "in": 8192, "group": 64, "type": "bf16"},
        # Odd sizes, small groups, single precision.
        {"name": "linear_odd", "op": "linear", "rows": 5, "out": 1001, "in": 2080, "group": 32, "type": "f32"},
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    costs = [work(case) for case in listed()]
    most = {key: max(cost[key] for cost in costs) for key in ("bytes", "flops")}
    while True:
        op = rng.choice(["store", "read", "attend", "attend", "attend", "linear", "linear"])
        kind = rng.choice(["bf16", "bf16", "f16", "f32"])
        if op == "linear":
            group = rng.choice([32, 64, 128])
            # Row lengths are a power of two or an odd number of groups.
            width = rng.choice([2 ** rng.randint(8, 14), group * (2 * log_int(1, 8192 // group) + 1)])
            case = {"op": op, "rows": log_int(1, 48), "out": log_int(200, 28672), "in": width, "group": group,
                    "type": kind}
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 8, 10])
            hi = log_int(40, 131072 if op == "attend" else 33000)
            case = {"op": op, "batch": log_int(1, 64), "lo": max(1, int(hi * rng.choice([0.02, 0.3, 0.9]))), "hi": hi,
                    "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128, 128, 128, 256]),
                    "page": rng.choice([16, 32, 64, 128]), "type": kind}
            if op == "store":
                case["new"] = rng.choice([0, 1, 1, log_int(2, 500)])
            if op == "attend":
                case["heads"] = kv_heads * rng.choice([1, 2, 4, 4, 6, 8])
                case["new"] = rng.choice([1, 1, 1, log_int(2, 16), log_int(17, 2048)])
                case["window"] = rng.choice([0, 0, 0, log_int(16, 4096)])
                case["mask"] = 1 < case["new"] <= 16 and rng.random() < 0.5
        # Small enough in tokens for its plain form too, and no dearer than the dearest listed case.
        cost = work(case)
        if cost["bytes"] > most["bytes"] or cost["flops"] > most["flops"]:
            continue
        if op != "linear" and case["batch"] * case["hi"] * case["kv_heads"] * case["dim"] > 3 * 131072 * 8 * 128:
            continue
        return case


# ------------------------------------------------------------------- inputs


def _generator(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + stream)
    return g


def _lengths(case):
    """(length of every sequence, new or read rows of it): spread between lo and
    hi, the first one of length hi."""
    g = torch.Generator()
    g.manual_seed(1000003 * case["hi"] + 1009 * case["lo"] + case["batch"])
    span = case["hi"] - case["lo"]
    lengths = [case["hi"]] + [case["lo"] + int(x) for x in torch.randint(0, span + 1, (case["batch"] - 1,), generator=g)]
    if case["op"] == "read":
        return lengths, list(lengths)
    if case["new"] == 0:  # whole prompts; every third behind a prefix
        return lengths, [n if b % 3 else n - n // 3 for b, n in enumerate(lengths)]
    return lengths, [min(case["new"], n) for n in lengths]


def _rows(tokens, heads, dim, g, keys):
    """Key or value rows as a model makes them: keys share a mean per channel, a
    few channels are large; values differ in size from token to token."""
    x = torch.randn((tokens, heads, dim), generator=g, device=DEV)
    if keys:
        x += 0.7 * torch.randn((1, heads, dim), generator=g, device=DEV)
        x[..., :: max(1, dim // 3)] *= 3.0
    else:
        x *= torch.exp(0.4 * torch.randn((tokens, heads, 1), generator=g, device=DEV))
    return x


def _cache_inputs(case, seed):
    dtype = DTYPES[case["type"]]
    lengths, new = _lengths(case)
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    used = [-(-n // page) for n in lengths]
    num_pages = sum(used) + 3
    order = torch.randperm(num_pages, generator=_generator(seed, 2), device=DEV).to(torch.int32)
    table = torch.zeros((case["batch"], max(used)), dtype=torch.int32, device=DEV)
    first = 0
    for b, n in enumerate(used):
        table[b, :n] = order[first:first + n]
        first += n
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    data = {
        "lengths_host": lengths, "new_host": new, "num_pages": num_pages, "table": table, "rows": offsets[-1],
        "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV),
        "offsets": None if offsets[-1] == case["batch"] and max(new) == 1
        else torch.tensor(offsets, dtype=torch.int32, device=DEV),
        "dtype": dtype,
    }
    # What the pool holds: rows of every slot, those of no sequence included.
    g = _generator(seed, 3)
    if case["op"] == "store":
        data["k"] = _rows(offsets[-1], heads, dim, g, True).to(dtype)
        data["v"] = _rows(offsets[-1], heads, dim, g, False).to(dtype)
    else:
        for name in ("k", "v"):
            codes = torch.empty((num_pages, heads, page, dim // 2), dtype=torch.uint8, device=DEV)
            scales = torch.empty((num_pages, heads, page), dtype=torch.float32, device=DEV)
            step = max(1, (1 << 26) // (heads * page * dim))
            for i in range(0, num_pages, step):
                n = min(step, num_pages - i)
                x = _rows(n * page, heads, dim, g, name == "k").view(n, page, heads, dim).transpose(1, 2)
                scales[i:i + n] = x.abs().amax(-1) / 7.0
                c = torch.round(x / scales[i:i + n, ..., None]).clamp(-7, 7).to(torch.int8).view(torch.uint8)
                codes[i:i + n] = (c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)
            data[name + "_codes"], data[name + "_scales"] = codes, scales
    if case["op"] == "attend":
        g = _generator(seed, 4)
        data["q"] = (1.3 * torch.randn((offsets[-1], case["heads"], dim), generator=g, device=DEV)).to(dtype)
        data["mask"] = None
        if case["mask"]:
            # Drafted tokens see the context and some of the drafts before them;
            # a tenth of the rows belong to drafts already given up and see nothing.
            mask = torch.ones((offsets[-1], max(lengths)), dtype=torch.bool, device=DEV)
            for b, (n, m) in enumerate(zip(lengths, new)):
                mask[offsets[b]:offsets[b + 1], n - m:n] = torch.rand((m, m), generator=g, device=DEV) < 0.6
            mask &= torch.rand((offsets[-1], 1), generator=g, device=DEV) < 0.9
            data["mask"] = mask
    return data


def _linear_inputs(case, seed):
    g = _generator(seed, 5)
    rows, n, k, group = case["rows"], case["out"], case["in"], case["group"]
    w = torch.randn((n, k), generator=g, device=DEV) / math.sqrt(k)
    scales = (w.view(n, k // group, group).abs().amax(-1) / 7.0).to(torch.bfloat16)
    c = torch.round(w.view(n, k // group, group) / scales.float()[..., None]).clamp(-7, 7)
    c = c.to(torch.int8).view(n, k).view(torch.uint8)
    x = torch.randn((rows, k), generator=g, device=DEV)
    x[:, :: max(1, k // 5)] *= 8.0  # a few large channels
    return {"codes": (c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4), "scales": scales, "group": group,
            "x": x.to(DTYPES[case["type"]])}


def prepare(case, seed):
    if case["op"] == "linear":
        state = _linear_inputs(case, seed)
        if own:
            from maxsim_amd import Int4Linear

            state["linear"] = Int4Linear(state["codes"], state["scales"])
    else:
        state = _cache_inputs(case, seed)
        shape = (state["num_pages"], case["kv_heads"], case["page"])
        if own:
            from maxsim_amd import Int4KVCache

            cache = Int4KVCache(shape[0], case["kv_heads"], case["dim"], page_size=case["page"])
            if case["op"] != "store":
                for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
                    getattr(cache, name).copy_(state.pop(name))
            state["cache"] = cache
        elif case["op"] == "store":
            for name in ("k", "v"):
                state[name + "_codes"] = torch.zeros((*shape, case["dim"] // 2), dtype=torch.uint8, device=DEV)
                state[name + "_scales"] = torch.zeros(shape, dtype=torch.float32, device=DEV)
    state["case"] = dict(case)
    return state


# --------------------------------------------------------------- plain forms


def _slots(state):
    """Page and slot of every new (or read) row."""
    page = state["case"]["page"]
    rows = torch.arange(state["rows"], device=DEV)
    if state["offsets"] is None:
        b = rows
        pos = (state["lengths"] - 1).long()
    else:
        offsets = state["offsets"].long()
        b = torch.searchsorted(offsets, rows, right=True) - 1
        pos = state["lengths"].long()[b] - offsets[b + 1] + rows
    return state["table"][b, pos // page].long(), pos % page


def _unpack(codes):
    low = (codes & 15).to(torch.int8)
    high = (codes >> 4).to(torch.int8)
    both = torch.stack((low, high), -1).flatten(-2)
    return torch.where(both > 7, both - 16, both).float()


def _plain_store(state):
    pages, slots = _slots(state)
    for name in ("k", "v"):
        x = state[name].float()
        s = x.abs().amax(-1)
        s = s / torch.full_like(s, 7.0)  # a quotient; by a plain number it is a product with 1 / 7
        s = torch.where(s == 0, torch.ones_like(s), s)
        c = torch.round(x / s[..., None]).clamp(-7, 7).to(torch.int8).view(torch.uint8)
        state[name + "_codes"][pages, :, slots] = (c[..., 0::2] & 15) | ((c[..., 1::2] & 15) << 4)
        state[name + "_scales"][pages, :, slots] = s
    return _plain_read(state)


def _plain_read(state):
    pages, slots = _slots(state)
    out = []
    for name in ("k", "v"):
        s = state[name + "_scales"][pages, :, slots]
        out.append((_unpack(state[name + "_codes"][pages, :, slots]) * s[..., None]).to(state["dtype"]))
    return out


def _sequence_rows(state, b, name):
    """Keys or values [kv_heads, length, dim] of a sequence, in single precision."""
    n, page = state["lengths_host"][b], state["case"]["page"]
    ids = state["table"][b, :-(-n // page)].long()
    x = _unpack(state[name + "_codes"][ids]) * state[name + "_scales"][ids][..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_attend(state):
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    share = heads // kv_heads
    out = torch.empty((state["rows"], heads, dim), dtype=state["dtype"], device=DEV)
    first = 0
    for b, (n, m) in enumerate(zip(state["lengths_host"], state["new_host"])):
        k, v = _sequence_rows(state, b, "k"), _sequence_rows(state, b, "v")
        keys = torch.arange(n, device=DEV)
        for i in range(0, m, 512):
            rows = slice(first + i, first + min(m, i + 512))
            count = rows.stop - rows.start
            q = state["q"][rows].float().view(count, kv_heads, share, dim).permute(1, 2, 0, 3)
            s = torch.matmul(q.reshape(kv_heads, share * count, dim), k.transpose(1, 2)) * (dim ** -0.5)
            s = s.view(kv_heads, share, count, n)
            pos = torch.arange(n - m + i, n - m + i + count, device=DEV)[:, None]
            see = keys <= pos
            if case["window"]:
                see = see & (keys > pos - case["window"])
            if state["mask"] is not None:
                see = see & state["mask"][rows, :n]
            top = torch.where(see, s, -torch.inf).amax(-1, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            p = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(kv_heads, share * count, n), v).view(kv_heads, share, count, dim)
            o = torch.where(total > 0, o / total, torch.zeros_like(o))
            out[rows] = o.permute(2, 0, 1, 3).reshape(count, heads, dim).to(out.dtype)
        first += m
    return out


def _plain_linear(state):
    w = _unpack(state["codes"]).view(state["codes"].shape[0], -1, state["group"]) * state["scales"].float()[..., None]
    return torch.matmul(state["x"].float(), w.flatten(1).t()).to(state["x"].dtype)


# --------------------------------------------------------------------- passes


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend, "linear": _plain_linear}[op](state)
    if op == "linear":
        return state["linear"](state["x"])
    cache, table, lengths, offsets = state["cache"], state["table"], state["lengths"], state["offsets"]
    if op == "attend":
        return cache.attend(state["q"], table, lengths, offsets, window=case["window"] or None, mask=state["mask"])
    if op == "store":
        cache.append(state["k"], state["v"], table, lengths, offsets)
    return list(cache.read(table, lengths, offsets, rows=state["rows"], dtype=state["dtype"]))


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "linear":
        m, n, k = case["rows"], case["out"], case["in"]
        return {"bytes": n * k // 2 + 2 * n * (k // case["group"]) + size * m * (k + n), "flops": 2 * m * n * k}
    lengths, new = _lengths(case)
    heads, dim = case["kv_heads"], case["dim"]
    row = 2 * heads * (dim // 2 + 4)  # a token's key and value in the cache
    tokens = sum(new)
    if case["op"] == "store":  # read the rows, write them in 4 bits, read those, write the values
        return {"bytes": tokens * (2 * row + 4 * heads * dim * size), "flops": 6 * tokens * heads * dim}
    if case["op"] == "read":
        return {"bytes": tokens * (row + 2 * heads * dim * size), "flops": 2 * tokens * heads * dim}
    seen = pairs = mask = 0
    window = case["window"]
    for n, m in zip(lengths, new):
        seen += min(n, window + m - 1) if window else n
        if window:
            pairs += sum(min(p + 1, window) for p in range(n - m, n))
        else:
            pairs += m * (n - m) + m * (m + 1) // 2
        mask += m * n if case["mask"] else 0
    return {"bytes": seen * row + 2 * tokens * case["heads"] * dim * size + mask,
            "flops": 4 * pairs * case["heads"] * dim}


# ------------------------------------------------------------ the definitions


def exact(case, seed):
    """The operators from their definitions, in float64."""
    if case["op"] == "linear":
        data = _linear_inputs(case, seed)
        codes = data["codes"].to(torch.int64)
        n, k, group = case["out"], case["in"], case["group"]
        w = torch.empty((n, k), dtype=torch.float64, device=DEV)
        w[:, 0::2] = ((codes % 16 + 8) % 16 - 8).double()
        w[:, 1::2] = ((codes // 16 + 8) % 16 - 8).double()
        w *= data["scales"].double().repeat_interleave(group, dim=1)
        return (data["x"].double() @ w.T.contiguous()).cpu()
    data = _cache_inputs(case, seed)
    if case["op"] == "store":
        # The scale and the quotient are single-precision numbers of the format:
        # a float64 quotient of two of them rounds to the same one.
        out = []
        for name in ("k", "v"):
            x = data[name].double()
            s = (x.abs().max(dim=-1, keepdim=True).values / 7).float().double()
            s[s == 0] = 1.0
            out.append((torch.clamp(torch.round((x / s).float().double()), -7, 7) * s).cpu())
        return out

    def values(name, b):
        """[length, kv_heads, dim] of a sequence."""
        n = data["lengths_host"][b]
        pos = torch.arange(n, device=DEV)
        page, slot = data["table"][b].long()[pos // case["page"]], pos % case["page"]
        codes = data[name + "_codes"][page, :, slot].to(torch.int16)
        x = torch.empty((n, case["kv_heads"], case["dim"]), dtype=torch.float64, device=DEV)
        x[..., 0::2] = ((codes % 16 + 8) % 16 - 8).double()
        x[..., 1::2] = ((codes // 16 + 8) % 16 - 8).double()
        return x.mul_(data[name + "_scales"][page, :, slot].double().unsqueeze(-1))

    if case["op"] == "read":
        return [torch.cat([values(name, b).cpu() for b in range(case["batch"])]) for name in ("k", "v")]
    share = case["heads"] // case["kv_heads"]
    parts = []
    first = 0
    for b, (n, m) in enumerate(zip(data["lengths_host"], data["new_host"])):
        k, v = values("k", b), values("v", b)
        q = data["q"][first:first + m].double()
        at = torch.arange(m, device=DEV).unsqueeze(1) + (n - m)
        key = torch.arange(n, device=DEV).unsqueeze(0)
        hidden = key > at
        if case["window"]:
            hidden |= key <= at - case["window"]
        if data["mask"] is not None:
            hidden |= ~data["mask"][first:first + m, :n]
        o = torch.zeros((m, case["heads"], case["dim"]), dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            logits = (q[:, h] @ k[:, h // share].T.contiguous()) / math.sqrt(case["dim"])
            logits.masked_fill_(hidden, -math.inf)
            logits -= logits.max(dim=1, keepdim=True).values.clamp(min=-1e300)
            weights = logits.exp_()
            total = weights.sum(dim=1, keepdim=True)
            o[:, h] = (weights @ v[:, h // share].contiguous()) / total.clamp(min=1e-300)
        parts.append(o.cpu())
        first += m
    return torch.cat(parts)
