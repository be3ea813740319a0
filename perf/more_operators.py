"""Performance cases of a reader's decoding step over the 4-bit key/value cache.

What a reader model that streams long contexts, drafts several tokens a step and
looks at page images does between its products, none of it on the host:

  pages   which pages of the pool a sequence holds, and where new rows go: the
          sequences are cut to given lengths, their pages past those go back to
          the stack of free pages, new rows get pages from it
  rotary  queries and keys turned by their positions, on one axis or several
  sinks   attention over a sliding window and the first tokens of a sequence
  tree    attention of a tree of drafted tokens: a row sees the context, its
          ancestors and itself
  keep    drafted rows enter the cache, the accepted ones move up to the end of
          the context, and are read back

A cache row is in the framework's int4 format: one scale per token and head, s =
max|x| / 7 in single precision (1 for a row of zeros), codes clip(rint(x / s), -7,
7), two's complement nibbles with the even dim low.  Rows live in pages of a pool;
a sequence is a row of a page table and a length.

``own`` chooses between the framework's entry points and the plain form of the
same formulas in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # Between two drafting steps of a batch: three of eight drafts stayed, the
        # next eight need rows.
        {"name": "pages_step", "op": "pages", "batch": 64, "lo": 100, "hi": 8000, "back": 5, "new": 8, "page": 64,
         "pool": 100},
        # Prompts are taken in where others ended, and the pool does not hold the last.
        {"name": "pages_prompts", "op": "pages", "batch": 48, "lo": 1000, "hi": 20000, "back": 1000, "new": 0,
         "page": 16, "pool": 95},
        # A decoding step's queries and keys.
        {"name": "rotary_step", "op": "rotary", "rows": 16, "heads": 32, "kv_heads": 8, "dim": 128, "part": 128,
         "axes": 1, "adjacent": False, "type": "bf16"},
        # The patches of page images: page, line and column.
        {"name": "rotary_images", "op": "rotary", "rows": 9216, "heads": 32, "kv_heads": 8, "dim": 128, "part": 128,
         "axes": 3, "adjacent": False, "type": "bf16"},
        # A decoding batch that streams: a window and four first tokens.
        {"name": "sinks_step", "op": "sinks", "batch": 32, "lo": 100, "hi": 30000, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "window": 1024, "sinks": 4},
        # Few sequences far past a wide window, with a system prompt that stays.
        {"name": "sinks_long", "op": "sinks", "batch": 3, "lo": 60001, "hi": 131072, "new": 3, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "f16", "window": 16384, "sinks": 300},
        # A piece of a long prompt, streamed.
        {"name": "sinks_prompt", "op": "sinks", "batch": 2, "lo": 9000, "hi": 17000, "new": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "window": 4096, "sinks": 64},
        # One user's drafts behind a short context: latency.
        {"name": "tree_first", "op": "tree", "batch": 1, "lo": 700, "hi": 700, "new": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "type": "bf16"},
        # A batch's trees, one key/value head per query head, single precision.
        {"name": "tree_batch", "op": "tree", "batch": 7, "lo": 133, "hi": 3001, "new": 27, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "type": "f32"},
        # Wide trees behind long contexts.
        {"name": "tree_long", "op": "tree", "batch": 4, "lo": 20000, "hi": 65000, "new": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16"},
        # After a drafting step of a batch.
        {"name": "keep_step", "op": "keep", "batch": 32, "lo": 100, "hi": 4000, "new": 16, "width": 5, "kv_heads": 8,
         "dim": 128, "page": 64, "type": "bf16"},
        # After large trees with long accepted branches.
        {"name": "keep_wide", "op": "keep", "batch": 64, "lo": 300, "hi": 2500, "new": 250, "width": 61,
         "kv_heads": 10, "dim": 96, "page": 16, "type": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    most = {}
    for case in listed():
        for key, value in work(case).items():
            most[key] = max(most.get(key, 0), value)
    while True:
        op = rng.choice(["pages", "rotary", "sinks", "sinks", "tree", "tree", "keep"])
        if op == "pages":
            hi = _log_int(rng, 40, 40000)
            case = {"op": op, "batch": _log_int(rng, 1, 3000), "lo": max(1, int(hi * rng.choice([0.02, 0.4]))),
                    "hi": hi, "back": rng.choice([0, _log_int(rng, 1, hi)]),
                    "new": rng.choice([0, 1, _log_int(rng, 2, 64)]), "page": rng.choice([16, 32, 64, 128]),
                    "pool": rng.choice([100, 100, 90])}
            if case["batch"] * hi > 1500000:
                continue
        elif op == "rotary":
            kv_heads = rng.choice([1, 2, 4, 8, 10])
            dim = rng.choice([64, 96, 128, 128, 256])
            case = {"op": op, "rows": _log_int(rng, 1, 30000), "heads": kv_heads * rng.choice([1, 2, 4, 8]),
                    "kv_heads": kv_heads, "dim": dim, "part": rng.choice([dim, dim, dim // 2]),
                    "axes": rng.choice([1, 2, 3]), "adjacent": rng.random() < 0.3,
                    "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 8, 10])
            hi = _log_int(rng, 40, 4000 if op == "keep" else 131072)
            case = {"op": op, "batch": _log_int(rng, 1, 64), "lo": max(1, int(hi * rng.choice([0.05, 0.3, 0.9]))),
                    "hi": hi, "new": 1, "kv_heads": kv_heads, "dim": rng.choice([64, 96, 128, 128, 128, 256]),
                    "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
            if op == "keep":
                case["new"] = _log_int(rng, 1, 300)
                case["width"] = _log_int(rng, 1, 64)
            else:
                case["heads"] = kv_heads * rng.choice([1, 2, 4, 4, 6, 8])
            if op == "sinks":
                case["new"] = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 2048)])
                case["window"] = _log_int(rng, 64, 16384)
                case["sinks"] = _log_int(rng, 1, 500)
            if op == "tree":
                case["new"] = _log_int(rng, 2, 200)
            # Small enough in tokens for its plain form too.
            if case["batch"] * hi * kv_heads * case["dim"] > 3 * 131072 * 8 * 128:
                continue
        cost = work(case)
        if all(cost[key] <= most[key] for key in most):
            return case


# ------------------------------------------------------------------- inputs


def _generator(seed, stream, device=DEV):
    g = torch.Generator(device=device)
    g.manual_seed(1000003 * int(seed) + stream)
    return g


def _lengths(case):
    """Lengths of the sequences, of the sizes alone: the first is the longest."""
    g = _generator(case["hi"] + 7 * case["lo"], case["batch"], "cpu")
    rest = torch.randint(case["lo"], case["hi"] + 1, (case["batch"] - 1,), generator=g)
    return [case["hi"], *rest.tolist()]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages_inputs(case, seed):
    """A server's pages in mid-course: sequence b is to be cut to cut[b] tokens and
    to get new[b] more."""
    page, batch = case["page"], case["batch"]
    lengths = _lengths(case)
    g = _generator(batch, 1, "cpu")  # rows and lengths go by the sizes alone, the pages' order by the seed
    back = torch.randint(0, case["back"] + 1, (batch,), generator=g).tolist()
    if case["new"] == 0:
        # A third of the sequences ended; longer prompts come in their place.
        ended = torch.rand(batch, generator=g) < 0.34
        cut = [0 if ended[b] else max(0, n - back[b]) for b, n in enumerate(lengths)]
        fresh = torch.randint((case["lo"] + case["hi"]) // 2, case["hi"] + 1, (batch,), generator=g).tolist()
        new = [fresh[b] if ended[b] else 1 for b in range(batch)]
    else:
        cut = [max(0, n - back[b]) for b, n in enumerate(lengths)]
        new = [case["new"]] * batch
    held = [-(-n // page) for n in lengths]
    after = [-(-(c + n) // page) for c, n in zip(cut, new)]
    max_pages = max(held + after) + 1
    num_pages = max(sum(held), sum(after) * case["pool"] // 100)
    order = torch.randperm(num_pages, generator=_generator(seed, 2, "cpu")).to(torch.int32)
    table = torch.full((batch, max_pages), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(held):
        table[b, :n] = order[first:first + n]
        first += n
    free = torch.full((num_pages,), -1, dtype=torch.int32)
    free[:num_pages - first] = order[first:]
    return {"table": table.to(DEV), "lengths": _int32(lengths), "free": free.to(DEV),
            "free_count": _int32([num_pages - first]), "cut": _int32(cut), "new": _int32(new), "rows": sum(new)}


def _rotary_axes(case):
    """The axis of each pair of dims: a quarter of them time, the rest in halves; or
    all alike."""
    pairs = case["part"] // 2
    if case["axes"] == 1:
        return [0] * pairs
    if case["axes"] == 2:
        return [i % 2 for i in range(pairs)]
    time = pairs // 4
    line = (pairs - time) // 2
    return [0] * time + [1] * line + [2] * (pairs - time - line)


def _rotary_inputs(case, seed):
    g = _generator(seed, 2)
    rows, axes = case["rows"], case["axes"]
    kind = DTYPES[case["type"]]
    q = 1.3 * torch.randn((rows, case["heads"], case["dim"]), generator=g, device=DEV)
    k = torch.randn((rows, case["kv_heads"], case["dim"]), generator=g, device=DEV)
    k[..., :: max(1, case["dim"] // 3)] *= 3.0  # a few large channels
    if axes == 1:  # tokens of sequences somewhere in long contexts
        positions = torch.randint(0, 131072, (rows,), generator=g, device=DEV)
    else:  # pages behind a text, in rows of 32 patches
        at = torch.arange(rows, device=DEV)
        start = torch.randint(0, 4000, (1,), generator=g, device=DEV)
        axis = (start + at // 1024, start + at % 1024 // 32, start + at % 32)
        positions = torch.stack(axis[3 - axes:])
    return {"q": q.to(kind), "k": k.to(kind), "positions": positions.to(torch.int32).contiguous()}


def _model_rows(tokens, heads, dim, g, keys):
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
    kind = DTYPES[case["type"]]
    lengths = _lengths(case)
    new = [min(case["new"], n) for n in lengths]
    page, heads, dim, batch = case["page"], case["kv_heads"], case["dim"], case["batch"]
    held = [-(-n // page) for n in lengths]
    num_pages = sum(held) + 2
    order = torch.randperm(num_pages, generator=_generator(seed, 3, "cpu")).to(torch.int32)
    table = torch.full((batch, max(held)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(held):
        table[b, :n] = order[first:first + n]
        first += n
    offsets = np.cumsum([0, *new]).tolist()
    rows = offsets[-1]
    data = {"lengths_host": lengths, "new_host": new, "num_pages": num_pages, "rows": rows, "type": kind,
            "table": table.to(DEV), "lengths": _int32(lengths),
            "offsets": None if case["new"] == 1 else _int32(offsets)}
    g = _generator(seed, 4)
    if case["op"] == "keep":
        data["k"] = _model_rows(rows, heads, dim, g, True).to(kind)
        data["v"] = _model_rows(rows, heads, dim, g, False).to(kind)
        # Accepted branches: ascending rows of the tree, none to width of them (one at
        # least of the first).
        host, sizes = _generator(seed, 5, "cpu"), _generator(batch, 5, "cpu")
        kept = torch.full((batch, case["width"]), -1, dtype=torch.int32)
        counts = []
        for b, n in enumerate(new):
            count = int(torch.randint(0 if b else 1, min(n, case["width"]) + 1, (1,), generator=sizes))
            kept[b, :count] = torch.randperm(n, generator=host)[:count].sort().values.to(torch.int32)
            counts.append(count)
        data["kept"] = kept.to(DEV)
        data["kept_rows"] = sum(counts)
        data["kept_offsets"] = _int32(np.cumsum([0, *counts]).tolist())
        return data
    for name in ("k", "v"):  # every slot of the pool, those of no sequence included
        codes = torch.empty((num_pages, heads, page, dim // 2), dtype=torch.uint8, device=DEV)
        scales = torch.empty((num_pages, heads, page), dtype=torch.float32, device=DEV)
        step = max(1, (1 << 26) // (heads * page * dim))
        for i in range(0, num_pages, step):
            n = min(step, num_pages - i)
            x = _model_rows(n * page, heads, dim, g, name == "k").view(n, page, heads, dim).transpose(1, 2)
            codes[i:i + n], scales[i:i + n] = _quantise(x)
        data[name + "_codes"], data[name + "_scales"] = codes, scales
    data["q"] = (1.3 * torch.randn((rows, case["heads"], dim), generator=g, device=DEV)).to(kind)
    if case["op"] == "tree":
        # Likely continuations get more children: parents lean towards the first rows.
        host = _generator(seed, 6, "cpu")
        data["parents_host"] = [(torch.arange(n) * torch.rand(n, generator=host) ** 1.5).long() - 1 for n in new]
        data["parents"] = torch.cat(data["parents_host"]).to(torch.int32).to(DEV)
    return data


def prepare(case, seed):
    op = case["op"]
    state = _pages_inputs(case, seed) if op == "pages" else \
        _rotary_inputs(case, seed) if op == "rotary" else _cache_inputs(case, seed)
    if op == "pages" and own:
        from maxsim_amd import CachePages

        pages = CachePages(state["free"].shape[0], case["batch"], state["table"].shape[1], page_size=case["page"])
        for name in ("table", "lengths", "free", "free_count"):
            getattr(pages, name).copy_(state.pop(name))
        state["pages"] = pages
    elif op == "rotary" and own:
        from maxsim_amd import Rotary

        state["rotary"] = Rotary(case["dim"], rotary_dim=case["part"], axes=_rotary_axes(case),
                                 adjacent=case["adjacent"])
    elif op == "rotary":
        pairs = case["part"] // 2
        state["axes"] = torch.tensor(_rotary_axes(case), device=DEV)
        state["frequencies"] = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=DEV) / pairs)
    elif op != "pages" and own:
        from maxsim_amd import Int4KVCache

        cache = Int4KVCache(state["num_pages"], case["kv_heads"], case["dim"], page_size=case["page"])
        if op != "keep":
            for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
                getattr(cache, name).copy_(state.pop(name))
        state["cache"] = cache
    elif op == "keep":
        shape = (state["num_pages"], case["kv_heads"], case["page"])
        for name in ("k", "v"):
            state[name + "_codes"] = torch.zeros((*shape, case["dim"] // 2), dtype=torch.uint8, device=DEV)
            state[name + "_scales"] = torch.zeros(shape, dtype=torch.float32, device=DEV)
    state["case"] = dict(case)
    return state


# --------------------------------------------------------------- plain forms


def _plain_pages(state):
    table, lengths, free, count = (state[name] for name in ("table", "lengths", "free", "free_count"))
    page, rows, new = state["case"]["page"], state["rows"], state["new"].long()
    max_pages, num_pages = table.shape[1], free.shape[0]

    def pages_of(n):
        return (n + page - 1) // page

    kept = torch.minimum(lengths, state["cut"]).long()
    held, stay = pages_of(lengths.long())[:, None], pages_of(kept)[:, None]
    column = torch.arange(max_pages, device=DEV)
    back = (column >= stay) & (column < held)
    order = torch.cumsum(back.flatten(), 0).view_as(back)  # from 1 on
    total = count.long() + order[-1, -1]
    stack = torch.cat((free, free.new_zeros(1)))  # the last entry takes what stays
    stack[torch.where(back, total - order, num_pages)] = table
    table.masked_fill_(back, -1)
    new = torch.where(kept + new > max_pages * page, 0, new)
    need = pages_of(kept + new) - stay[:, 0]
    given = (need == 0) | (torch.cumsum(need, 0) <= total)
    new, need = new * given, need * given
    before = (torch.cumsum(need, 0) - need)[:, None]
    take = (column >= stay) & (column < stay + need[:, None])
    table.copy_(torch.where(take, stack[(total - 1 - before - column + stay).clamp(0, num_pages)], table))
    left = total - need.sum()
    free.copy_(torch.where(torch.arange(num_pages, device=DEV) < left, stack[:-1], -1))
    count.copy_(left)
    lengths.copy_(kept + new)
    ends = torch.cumsum(new, 0)
    offsets = torch.cat((ends.new_zeros(1), ends)).to(torch.int32)
    row = torch.arange(rows, device=DEV)
    b = torch.searchsorted(ends, row, right=True).clamp(max=lengths.shape[0] - 1)
    position = kept[b] + row - (ends - new)[b]
    there = row < ends[-1]
    slot = table[b, torch.where(there, position // page, 0)].long() * page + position % page
    return [offsets, torch.where(there, position, -1).to(torch.int32), torch.where(there, slot, -1), table, lengths,
            free, count]


def _plain_rotary(state):
    case, positions = state["case"], state["positions"]
    positions = positions[None] if positions.ndim == 1 else positions
    angle = positions.double()[state["axes"]] * state["frequencies"][:, None]  # [pairs, rows]
    cos, sin = torch.cos(angle).float().t()[:, None], torch.sin(angle).float().t()[:, None]
    part = case["part"]
    out = []
    for x in (state["q"], state["k"]):
        y = x.float()
        if case["adjacent"]:
            a, b = y[..., 0:part:2], y[..., 1:part:2]
            turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = y[..., :part // 2], y[..., part // 2:part]
            turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        out.append(torch.cat((turned, y[..., part:]), -1).to(x.dtype))
    return out


def _quantise(x):
    """Codes [..., dim / 2] and scales of rows in single precision."""
    top = x.abs().amax(-1)
    scale = top / torch.full_like(top, 7.0)  # a quotient; by a plain number it is a product with 1 / 7
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    code = torch.round(x / scale[..., None]).clamp(-7, 7).to(torch.int8).view(torch.uint8) & 15
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales):
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int8)
    return torch.where(nibbles > 7, nibbles - 16, nibbles).float() * scales[..., None]


def _sequence(state, b, name):
    """Keys or values [kv_heads, length, dim] of a sequence, in single precision."""
    n, page = state["lengths_host"][b], state["case"]["page"]
    ids = state["table"][b, :-(-n // page)].long()
    x = _values(state[name + "_codes"][ids], state[name + "_scales"][ids])
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _plain_attend(state):
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    share = heads // kv_heads
    out = torch.empty_like(state["q"])
    first = 0
    for b, (n, m) in enumerate(zip(state["lengths_host"], state["new_host"])):
        k, v = _sequence(state, b, "k"), _sequence(state, b, "v")
        key = torch.arange(n, device=DEV)
        if case["op"] == "tree":
            parents = state["parents"][first:first + m].long()
            line = torch.eye(m, device=DEV)
            line[torch.arange(m, device=DEV), parents.clamp(min=0)] += (parents >= 0).float()
            step = 1
            while step < m:  # lines of twice the length
                line = (torch.matmul(line, line) > 0).float()
                step *= 2
        for i in range(0, m, 512):
            count = min(512, m - i)
            rows = slice(first + i, first + i + count)
            q = state["q"][rows].float().view(count, kv_heads, share, dim).permute(1, 2, 0, 3)
            s = torch.matmul(q.reshape(kv_heads, share * count, dim), k.transpose(1, 2)) * dim ** -0.5
            s = s.view(kv_heads, share, count, n)
            if case["op"] == "tree":
                see = torch.cat((torch.ones((count, n - m), device=DEV), line[i:i + count]), 1) > 0
            else:
                at = torch.arange(n - m + i, n - m + i + count, device=DEV)[:, None]
                see = (key <= at) & ((key > at - case["window"]) | (key < case["sinks"]))
            p = torch.softmax(s.masked_fill_(~see, -torch.inf), -1)
            o = torch.matmul(p.view(kv_heads, share * count, n), v).view(kv_heads, share, count, dim)
            out[rows] = o.permute(2, 0, 1, 3).reshape(count, heads, dim).to(out.dtype)
        first += m
    return out


def _plain_keep(state):
    case, table, lengths = state["case"], state["table"], state["lengths"].long()
    page, rows, kept = case["page"], state["rows"], state["kept"].long()

    def places(b, position):
        return table[b, position // page].long(), position % page

    row = torch.arange(rows, device=DEV)
    if state["offsets"] is None:
        new, b, position = torch.ones_like(lengths), row, lengths - 1
    else:
        offsets = state["offsets"].long()
        new = offsets[1:] - offsets[:-1]
        b = torch.searchsorted(offsets, row, right=True) - 1
        position = lengths[b] - offsets[b + 1] + row
    at = places(b, position)
    start = lengths - new
    there = kept >= 0
    sequence = torch.arange(len(new), device=DEV)[:, None].expand_as(kept)
    place = torch.arange(kept.shape[1], device=DEV).expand_as(kept)
    source = places(sequence, start[:, None] + kept.clamp(min=0))
    target = places(sequence, (start[:, None] + torch.where(there, place, 0)).clamp(max=lengths[:, None] - 1))
    row = torch.arange(state["kept_rows"], device=DEV)
    ends = state["kept_offsets"].long()
    b = torch.searchsorted(ends, row, right=True) - 1
    read = places(b, start[b] + row - ends[b])
    out = [(start + there.sum(1)).to(torch.int32)]
    for name in ("k", "v"):
        codes, scales = state[name + "_codes"], state[name + "_scales"]
        codes[at[0], :, at[1]], scales[at[0], :, at[1]] = _quantise(state[name].float())
        for x in (codes, scales):
            moved = x[source[0], :, source[1]][there]
            x[target[0][there], :, target[1][there]] = moved
        out.append(_values(codes[read[0], :, read[1]], scales[read[0], :, read[1]]).to(state["type"]))
    return out


# --------------------------------------------------------------------- passes


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"pages": _plain_pages, "rotary": _plain_rotary, "sinks": _plain_attend, "tree": _plain_attend,
                "keep": _plain_keep}[op](state)
    if op == "pages":
        pages = state["pages"]
        offsets, positions, slots = pages.update(state["new"], lengths=state["cut"], rows=state["rows"])
        return [offsets, positions, slots, pages.table, pages.lengths, pages.free, pages.free_count]
    if op == "rotary":
        return list(state["rotary"](state["q"], state["k"], state["positions"]))
    cache, table, lengths, offsets = state["cache"], state["table"], state["lengths"], state["offsets"]
    if op == "sinks":
        return cache.attend(state["q"], table, lengths, offsets, window=case["window"], sinks=case["sinks"])
    if op == "tree":
        return cache.attend(state["q"], table, lengths, offsets, parents=state["parents"])
    cache.append(state["k"], state["v"], table, lengths, offsets)
    after = cache.keep(table, lengths, offsets, state["kept"])
    return [after, *cache.read(table, after, state["kept_offsets"], rows=state["kept_rows"], dtype=state["type"])]


def work(case):
    op = case["op"]
    if op == "pages":
        rows = case["batch"] * (case["new"] or (case["lo"] + 3 * case["hi"]) // 12)
        # Lengths, cuts and new rows come in, lengths and offsets go out; a page that
        # changes hands is read and written; a row has a position and a slot.
        changed = 2 * case["batch"] + rows // case["page"]
        return {"bytes": 20 * case["batch"] + 8 * changed + 12 * rows, "flops": 4 * rows + 20 * case["batch"]}
    if op == "rotary":
        values = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * values * case["dim"] * SIZE[case["type"]] + 4 * case["rows"] * case["axes"],
                "flops": 3 * values * case["part"]}
    size, heads, dim = SIZE[case["type"]], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    new = [min(case["new"], n) for n in lengths]
    tokens = sum(new)
    row = 2 * heads * (dim // 2 + 4)  # a token's key and value in the cache
    if op == "keep":
        # The rows come in and are kept in 4 bits; half the width of them is moved and
        # read back.
        kept = sum(min(n, case["width"]) for n in new) // 2
        return {"bytes": tokens * (row + 2 * heads * dim * size) + kept * (3 * row + 2 * heads * dim * size),
                "flops": 6 * tokens * heads * dim}
    seen = pairs = 0
    for n, m in zip(lengths, new):
        if op == "tree":
            seen += n
            pairs += m * (n - m + 1)  # the context and itself at least
        else:
            window, sinks = case["window"], case["sinks"]
            seen += min(n, window + m - 1 + sinks)
            for p in range(n - m, n):
                low = max(0, p + 1 - window)
                pairs += p + 1 - low + min(sinks, low)
    return {"bytes": seen * row + 2 * tokens * case["heads"] * dim * size + (4 * tokens if op == "tree" else 0),
            "flops": 4 * pairs * case["heads"] * dim}


# ------------------------------------------------------------ the definitions


def _exact_pages(case, seed):
    """One sequence after the other, with a list for the stack."""
    data = {name: x.cpu().numpy() if torch.is_tensor(x) else x for name, x in _pages_inputs(case, seed).items()}
    page, table, lengths = case["page"], data["table"], data["lengths"].tolist()
    stack = data["free"][:int(data["free_count"][0])].tolist()
    batch, max_pages = table.shape
    owned = [table[b, :math.ceil(lengths[b] / page)].tolist() for b in range(batch)]
    given_back = []
    for b in range(batch):
        lengths[b] = min(lengths[b], int(data["cut"][b]))
        stay = math.ceil(lengths[b] / page)
        given_back += owned[b][stay:]
        del owned[b][stay:]
    stack += given_back[::-1]
    offsets, positions, slots = [0], [], []
    asked, most = 0, len(stack)
    for b in range(batch):
        n = int(data["new"][b])
        need = math.ceil((lengths[b] + n) / page) - len(owned[b])
        if lengths[b] + n > max_pages * page:
            n = 0
        elif need > 0:
            asked += need
            if asked <= most:
                owned[b] += [stack.pop() for _ in range(need)]
            else:
                n = 0
        at = np.arange(lengths[b], lengths[b] + n)
        positions.append(at)
        slots.append(np.asarray(owned[b] + [0], dtype=np.int64)[at // page] * page + at % page)
        lengths[b] += n
        offsets.append(offsets[-1] + n)

    def filled(values, size, kind):
        x = np.full(size, -1, dtype=kind)
        x[:len(values)] = values
        return torch.from_numpy(x)

    return [torch.tensor(offsets, dtype=torch.int32), filled(np.concatenate(positions), data["rows"], np.int32),
            filled(np.concatenate(slots), data["rows"], np.int64),
            torch.stack([filled(row, max_pages, np.int32) for row in owned]),
            torch.tensor(lengths, dtype=torch.int32), filled(stack, len(data["free"]), np.int32),
            torch.tensor([len(stack)], dtype=torch.int32)]


def _exact_rotary(case, seed):
    """Every pair as a complex number times a unit one."""
    data = _rotary_inputs(case, seed)
    positions = data["positions"].view(case["axes"], -1).double()
    pairs = case["part"] // 2
    out = []
    for x in (data["q"], data["k"]):
        y = x.double()
        for i, axis in enumerate(_rotary_axes(case)):
            j, l = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + pairs)
            unit = torch.polar(torch.ones_like(positions[axis]), positions[axis] / 10000.0 ** (2 * i / case["part"]))
            z = torch.complex(y[:, :, j], y[:, :, l]) * unit[:, None]
            y[:, :, j], y[:, :, l] = z.real, z.imag
        out.append(y.cpu())
    return out


def _exact_keep(case, seed):
    """The format's scale and quotient are single-precision numbers: a float64
    quotient of two of them rounds to the same one."""
    data = _cache_inputs(case, seed)
    index, after = [], []
    first = 0
    for n, m, kept in zip(data["lengths_host"], data["new_host"], data["kept"].tolist()):
        accepted = [i for i in kept if i >= 0]
        index += [first + i for i in accepted]
        after.append(n - m + len(accepted))
        first += m
    out = [torch.tensor(after, dtype=torch.int32)]
    for name in ("k", "v"):
        x = data[name][torch.tensor(index, dtype=torch.int64, device=DEV)].double()
        s = (x.abs().amax(dim=-1, keepdim=True) / 7).float().double()
        s[s == 0] = 1.0
        out.append((torch.clamp(torch.round((x / s).float().double()), -7, 7) * s).cpu())
    return out


def exact(case, seed):
    """The operators from their definitions, in float64."""
    special = {"pages": _exact_pages, "rotary": _exact_rotary, "keep": _exact_keep}.get(case["op"])
    if special is not None:
        return special(case, seed)
    data = _cache_inputs(case, seed)

    def values(name, b):
        """[length, kv_heads, dim] of a sequence."""
        pos = torch.arange(data["lengths_host"][b], device=DEV)
        page, slot = data["table"][b].long()[pos // case["page"]], pos % case["page"]
        codes = data[name + "_codes"][page, :, slot].to(torch.int16)
        x = torch.empty((*codes.shape[:2], case["dim"]), dtype=torch.float64, device=DEV)
        x[..., 0::2] = ((codes % 16 + 8) % 16 - 8).double()
        x[..., 1::2] = ((codes // 16 + 8) % 16 - 8).double()
        return x.mul_(data[name + "_scales"][page, :, slot].double().unsqueeze(-1))

    share = case["heads"] // case["kv_heads"]
    parts = []
    first = 0
    for b, (n, m) in enumerate(zip(data["lengths_host"], data["new_host"])):
        k, v = values("k", b), values("v", b)
        q = data["q"][first:first + m].double()
        seen = torch.zeros((m, n), dtype=torch.bool)
        if case["op"] == "tree":
            seen[:, :n - m] = True
            for i in range(m):
                j = i
                while j >= 0:
                    seen[i, n - m + j] = True
                    j = int(data["parents_host"][b][j])
        else:
            for i in range(m):
                p = n - m + i
                seen[i, max(0, p + 1 - case["window"]):p + 1] = True
                seen[i, :min(case["sinks"], p + 1)] = True
        hidden = ~seen.to(DEV)
        o = torch.empty((m, case["heads"], case["dim"]), dtype=torch.float64, device=DEV)
        for h in range(case["heads"]):
            logits = (q[:, h] @ k[:, h // share].T.contiguous()) / math.sqrt(case["dim"])
            logits.masked_fill_(hidden, -math.inf)
            weights = (logits - logits.max(dim=1, keepdim=True).values).exp_()
            o[:, h] = (weights @ v[:, h // share].contiguous()) / weights.sum(dim=1, keepdim=True)
        parts.append(o.cpu())
        first += m
    return torch.cat(parts)
