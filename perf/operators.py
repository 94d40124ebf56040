"""The paged key/value cache's operators as they are measured: writing new rows (quantised where the cache holds
8 bits), reading rows back, and the attention of new rows over the pages.

Every case is a batch of sequences at their own lengths. A sequence has `held` rows in its pages and brings `new`
ones; row i of its n new rows stands at position length - n + i, where length counts the new rows too. The cache is
two pools [pages, heads, page_rows, width] and, for 8-bit storage, two arrays of scale bytes [pages, heads,
page_rows]: byte b stands for 2^(b - 127), 0 for zero and 255 for NaN, and a held value for its 8 bits times that.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# 8-bit storage: the type, the largest finite value L, and L's mantissa and exponent as frexp gives them.
EIGHT = {"e4m3": (torch.float8_e4m3fn, 448.0, 0.875, 9), "int8": (torch.int8, 127.0, 127.0 / 128.0, 7)}


# ------------------------------------------------------------------------------------------------------- the cases

def _attend(name, sequences, heads, group, width, page_rows, storage, dtype, held, new, chunks, causal=True):
    return {"name": name, "kind": "attend", "sequences": sequences, "heads": heads, "group": group, "width": width,
            "page_rows": page_rows, "storage": storage, "dtype": dtype, "held_min": held[0], "held_max": held[1],
            "new_min": new[0], "new_max": new[1], "chunks": chunks, "causal": causal}


def _rows(name, kind, sequences, heads, width, page_rows, storage, dtype, held, new):
    return {"name": name, "kind": kind, "sequences": sequences, "heads": heads, "group": 1, "width": width,
            "page_rows": page_rows, "storage": storage, "dtype": dtype, "held_min": held[0], "held_max": held[1],
            "new_min": new[0], "new_max": new[1], "chunks": sequences, "causal": True}


def listed():
    return [
        # One window of the smallest decoder at token 226: the latency of a single call.
        _attend("token_1_window", 1, 6, 1, 64, 16, "float16", "float16", (225, 225), (1, 1), 0),
        # The self attention of 64 windows that stand at their own tokens (lockstep ends where pages begin).
        _attend("tokens_64_windows", 64, 16, 1, 64, 16, "bfloat16", "bfloat16", (3, 447), (1, 1), 0),
        # The cross attention of one step over 1500 encoder rows held in 8 bits: the largest stream of a step.
        _attend("cross_int8_64_windows", 64, 20, 1, 64, 64, "int8", "bfloat16", (1499, 1499), (1, 1), 0, False),
        # Single tokens over long ragged contexts with shared heads and 128-wide heads.
        _attend("tokens_long_shared_heads", 12, 8, 4, 128, 64, "bfloat16", "bfloat16", (900, 32767), (1, 1), 0),
        # Prompts with up to 224 tokens of previous text, ragged, over what the windows already hold.
        _attend("prompts_32_windows", 32, 12, 1, 64, 16, "float16", "float16", (0, 223), (3, 224), 32),
        # Long chunks over long contexts: the products bound it.
        _attend("chunks_long", 2, 8, 4, 128, 128, "bfloat16", "bfloat16", (9001, 14001), (777, 1500), 2),
        # One batch of both: two windows bring prompts, the others single tokens, over an e4m3 cache.
        _attend("mixed_e4m3", 48, 20, 1, 64, 32, "e4m3", "float16", (40, 1450), (150, 448), 2),
        # One step's new rows of 64 windows into a 16-bit cache.
        _rows("append_64_windows", "append", 64, 16, 64, 16, "bfloat16", "bfloat16", (0, 447), (1, 1)),
        # One step's new rows quantised as they are written, and read back.
        _rows("store_int8_64_windows", "store", 64, 16, 64, 16, "int8", "bfloat16", (0, 447), (1, 1)),
        # A sequence start: every encoder row of 48 windows quantised into the cross cache, and read back.
        _rows("store_e4m3_encoder_rows", "store", 48, 20, 64, 64, "e4m3", "float16", (0, 0), (1500, 1500)),
        # Reading a whole ragged cache back for a caller that wants plain rows.
        _rows("read_int8_ragged", "read", 32, 12, 64, 32, "int8", "float16", (0, 0), (1, 1500)),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "append", "store", "store", "read"])
    storage = rng.choice(["float16", "bfloat16", "int8", "e4m3"])
    dtype = storage if storage in DTYPES else rng.choice(["float16", "bfloat16"])
    width, page_rows = rng.choice([64, 64, 128]), rng.choice([16, 32, 64, 128])
    heads = rng.choice([1, 2, 4, 5, 6, 8, 12, 16, 20])
    if kind != "attend":
        if kind == "append":
            storage, dtype = rng.choice([("float16", "float16"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
        elif kind == "store" and storage in DTYPES:
            storage = "int8"
        sequences = _log(rng, 1, 64)
        most = max(1, min(1500, 90_000_000 // (sequences * heads * width)))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, most)
        return {k: v for k, v in _rows("", kind, sequences, heads, width, page_rows, storage, dtype, (0, rng.randint(0, 448)),
                                       (rng.randint(1, new), new)).items() if k != "name"}
    group = rng.choice([1, 1, 2, 3, 4, 7, 8]) if heads <= 8 else 1
    sequences = _log(rng, 1, 64)
    chunks = rng.choice([0, 0, sequences, rng.randint(0, sequences)])
    new = _log(rng, 2, 1200) if chunks else 1
    # The products and the plain form's padded scores stay below the largest listed case's.
    pairs = int(2.5e9 / (sequences * heads * group * new * max(1, width // 64)))
    context = min(pairs, int(3e8 / (sequences * heads * width)), 32768)
    new = max(1, min(new, context))
    held = max(0, _log(rng, 1, max(1, context)) - new)
    return {k: v for k, v in _attend("", sequences, heads, group, width, page_rows, storage, dtype,
                                     (rng.randint(0, held), held), (rng.randint(1, new), new), chunks,
                                     rng.random() < 0.8).items() if k != "name"}


def _lengths(case):
    """The sequences' held and new rows: the case's own, the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    held = [rng.randint(case["held_min"], case["held_max"]) for _ in range(case["sequences"])]
    new = [rng.randint(case["new_min"], case["new_max"]) if s < case["chunks"] else 1 for s in range(case["sequences"])]
    held[-1] = case["held_max"]
    if case["chunks"]:
        new[0] = case["new_max"]
    return held, new


def work(case):
    held, new = _lengths(case)
    heads, width, size = case["heads"], case["width"], {"float32": 4}.get(case["dtype"], 2)
    row = heads * width * (2 if case["storage"] in DTYPES else 1) + (0 if case["storage"] in DTYPES else heads)
    rows, plain = sum(new), heads * width * size
    if case["kind"] == "attend":
        queries = heads * case["group"]
        pairs = sum(n * h + n * (n + 1) // 2 if case["causal"] else n * (h + n) for h, n in zip(held, new))
        return {"bytes": 2 * row * sum(h + n for h, n in zip(held, new)) + rows * queries * (2 * width * size + 4),
                "flops": 4.0 * pairs * queries * width}
    # 8 bits: the written rows are read back, from the pages into plain rows.
    return {"bytes": rows * 2 * (plain + row) * (2 if case["kind"] == "store" else 1), "flops": 2.0 * rows * heads * width}


# ------------------------------------------------------------------------------------------------ what a caller holds

def _quantise(x, storage):
    """Rows [..., width] as their 8 bits and scale bytes: the smallest power of two that keeps the row within L."""
    kind, largest, mantissa, exponent = EIGHT[storage]
    x = x.float()
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = torch.where(m <= mantissa, e - exponent, e - exponent + 1)
    byte = torch.where(top == 0, torch.ones_like(e), (e + 127).clamp(1, 254))
    scaled = torch.ldexp(x, (127 - byte).unsqueeze(-1))
    fine = torch.isfinite(top)
    scaled = torch.where(fine.unsqueeze(-1), scaled, torch.zeros_like(scaled))
    scaled = scaled.round().clamp(-largest, largest) if kind is torch.int8 else scaled
    return scaled.to(kind), torch.where(fine, byte, torch.full_like(byte, 255)).to(torch.uint8)


def _scale(byte):
    """2^(byte - 127); 0 for byte 0 and NaN for 255."""
    b = byte.to(torch.int32)
    s = torch.ldexp(torch.ones_like(b, dtype=torch.float32), b - 127)
    return torch.where(b == 0, torch.zeros_like(s), torch.where(b == 255, torch.full_like(s, math.nan), s))


def prepare(case, seed):
    held, new = _lengths(case)
    sequences, heads, width, page_rows = case["sequences"], case["heads"], case["width"], case["page_rows"]
    dtype, storage, rows = DTYPES[case["dtype"]], case["storage"], sum(new)
    device, g = "cuda", torch.Generator("cuda").manual_seed(seed)
    columns = -(-max(h + n for h, n in zip(held, new)) // page_rows)
    need = [-(-(h + n) // page_rows) for h, n in zip(held, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=device, dtype=torch.int32)
    # Entries behind a sequence's last page name some page too, as a table that was used before does.
    table = torch.randint(0, pages, (sequences, columns), generator=g, device=device, dtype=torch.int32)
    column = torch.arange(columns, device=device)
    needed = torch.tensor(need, device=device)
    first = torch.cumsum(needed, 0) - needed
    inside = column[None, :] < needed[:, None]
    table = torch.where(inside, order[(first[:, None] + column[None, :]).clamp(max=pages - 1)], table)
    pools, scales = [], []
    for spread in (1.0, 1.0):
        pool = torch.randn(pages, heads, page_rows, width, generator=g, device=device, dtype=torch.float32)
        if storage in DTYPES:
            pools.append((pool * spread).to(DTYPES[storage]))
            scales.append(None)
        else:
            # Rows' magnitudes differ, as tokens' do.
            pool *= torch.exp(0.7 * torch.randn(pages, heads, page_rows, 1, generator=g, device=device))
            q, b = _quantise(pool, storage)
            pools.append(q)
            scales.append(b)
        del pool
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=device)
    state = {"case": case, "table": table, "starts": starts, "rows": rows, "most": max(new),
             "lengths": torch.tensor([h + n for h, n in zip(held, new)], dtype=torch.int32, device=device),
             "keys": pools[0], "values": pools[1], "key_scales": scales[0], "value_scales": scales[1]}
    # What the projections leave: queries, keys and values of a row beside one another.
    queries = heads * case["group"]
    projected = torch.randn(rows, queries + 2 * heads, width, generator=g, device=device)
    projected = (projected * torch.exp(0.3 * torch.randn(rows, 1, 1, generator=g, device=device))).to(dtype)
    state |= {"q": projected[:, :queries], "k": projected[:, queries:queries + heads], "v": projected[:, queries + heads:]}
    if own:
        from whispereacp_b200 import CacheBatch, PagedCache
        state["cache"] = PagedCache(state["keys"], state["values"], state["key_scales"], state["value_scales"])
        state["batch"] = CacheBatch(table, state["lengths"], starts, max_rows=max(new))
    return state


# ------------------------------------------------------------------------------------------------------- the operators

def _places(state):
    """(sequence, position, page, row of the page) of every new row."""
    counts = state["starts"][1:] - state["starts"][:-1]
    sequence = torch.repeat_interleave(counts, output_size=state["rows"])
    index = torch.arange(state["rows"], device=counts.device) - state["starts"][sequence]
    position = state["lengths"][sequence] - counts[sequence] + index
    page_rows = state["case"]["page_rows"]
    return sequence, position, state["table"][sequence, position // page_rows].long(), (position % page_rows).long()


def _plain_write(state):
    case = state["case"]
    _, _, page, row = _places(state)
    for_pool = ((state["k"], state["keys"], state["key_scales"]), (state["v"], state["values"], state["value_scales"]))
    (x, pool, scale), (y, other, other_scale) = for_pool
    if case["storage"] in DTYPES:
        pool[page, :, row] = x.to(pool.dtype)
        other[page, :, row] = y.to(other.dtype)
        return
    (q, b), (p, c) = _quantise(x, case["storage"]), _quantise(y, case["storage"])
    pool.view(torch.uint8)[page, :, row] = q.view(torch.uint8)
    other.view(torch.uint8)[page, :, row] = p.view(torch.uint8)
    scale[page, :, row] = b
    other_scale[page, :, row] = c


def _widened(pool, scale):
    return pool.float() if scale is None else pool.float() * _scale(scale).unsqueeze(-1)


def _rows_of(pool, scale, page, row):
    """Rows (page, row) of a pool as fp32 values [..., heads, width]."""
    held = pool.view(torch.uint8)[page, :, row].view(pool.dtype) if scale is not None else pool[page, :, row]
    return _widened(held, None if scale is None else scale[page, :, row])


def _plain_read(state):
    _, _, page, row = _places(state)
    dtype = DTYPES[state["case"]["dtype"]]
    return (_rows_of(state["keys"], state["key_scales"], page, row).to(dtype),
            _rows_of(state["values"], state["value_scales"], page, row).to(dtype))


def _plain_attend(state):
    case = state["case"]
    heads, group, width, page_rows = case["heads"], case["group"], case["width"], case["page_rows"]
    table, lengths, starts, most = state["table"], state["lengths"], state["starts"], state["most"]
    sequences, columns = table.shape
    counts = starts[1:] - starts[:-1]
    index = torch.arange(most, device=table.device)
    row = (starts[:-1, None] + index[None, :]).clamp(max=state["rows"] - 1).long()           # [S, most]

    def gathered(pool, scale):
        flat = pool.view(torch.uint8)[table.long()].view(pool.dtype) if scale is not None else pool[table.long()]
        x = _widened(flat, None if scale is None else scale[table.long()])                     # [S, columns, heads, page_rows, width]
        return x.permute(0, 2, 1, 3, 4).reshape(sequences, heads, columns * page_rows, width)

    q = state["q"][row].float().reshape(sequences, most, heads, group, width)
    q = q.permute(0, 2, 3, 1, 4).reshape(sequences, heads, group * most, width)
    s = torch.matmul(q, gathered(state["keys"], state["key_scales"]).transpose(-1, -2)) * (1.0 / math.sqrt(width))
    s = s.reshape(sequences, heads, group, most, columns * page_rows)
    key = torch.arange(columns * page_rows, device=table.device)
    last = (lengths[:, None] - counts[:, None] + index[None, :]) if case["causal"] else (lengths[:, None] - 1).expand(-1, most)
    seen = key[None, None, :] <= last[:, :, None]                                             # [S, most, keys]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = gathered(state["values"], state["value_scales"])
    o = torch.matmul(p.reshape(sequences, heads, group * most, -1), v).reshape(sequences, heads, group, most, width)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    # [S, heads, group, most] back to the rows of the batch
    sequence = torch.repeat_interleave(counts, output_size=state["rows"])
    at = torch.arange(state["rows"], device=table.device) - starts[sequence]
    o = o.permute(0, 3, 1, 2, 4)[sequence, at].reshape(state["rows"], heads * group, width)
    lse = lse.permute(0, 3, 1, 2)[sequence, at].reshape(state["rows"], heads * group)
    return o.to(state["q"].dtype), lse


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        cache, batch = state["cache"], state["batch"]
        if kind == "attend":
            out, lse = cache.attend(batch, state["q"], causal=case["causal"], return_lse=True)
            return {"out": out, "lse": lse}
        if kind == "append":
            cache.append(batch, state["k"], state["v"])
            return {"keys": state["keys"], "values": state["values"]}
        if kind == "store":
            cache.append(batch, state["k"], state["v"])
        # How many rows there are the program knows; asking the batch for them waits for the device.
        keys, values = cache.read(batch, dtype=DTYPES[case["dtype"]], rows=state["rows"])
    else:
        if kind == "attend":
            out, lse = _plain_attend(state)
            return {"out": out, "lse": lse}
        if kind in ("append", "store"):
            _plain_write(state)
        if kind == "append":
            return {"keys": state["keys"], "values": state["values"]}
        keys, values = _plain_read(state)
    if kind == "read":
        return {"keys": keys, "values": values}
    return {"keys": keys, "values": values, "key_scales": state["key_scales"], "value_scales": state["value_scales"]}


# ------------------------------------------------------------------------------------------------- from the definition

def _exact_scale(byte):
    b = byte.double()
    return torch.where(b == 255, torch.full_like(b, math.nan), torch.where(b == 0, torch.zeros_like(b), torch.exp2(b - 127)))


def _exact_held(state, which, s):
    """Sequence s's rows in order, [length, heads, width] in 64 bits."""
    pool, scale = state[which], state[which[:-1] + "_scales"]
    n = int(state["lengths"][s])
    page_rows = state["case"]["page_rows"]
    pages = state["table"][s, : -(-n // page_rows)].long()
    parts = pool.view(torch.uint8)[pages].view(pool.dtype) if scale is not None else pool[pages]
    x = parts.double()
    if scale is not None:
        x = x * _exact_scale(scale[pages])[..., None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]


def _exact_eight(x, storage):
    """8-bit values and scale bytes of rows [n, heads, width], from the definition: the smallest power of two 2^E with
    |x| <= L 2^E, then the nearest representable value, ties to even."""
    largest = EIGHT[storage][1]
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / largest))
    e = torch.where(top > largest * torch.exp2(e), e + 1, e)
    e = torch.where(top <= largest * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(-126, 127)
    y = x * torch.exp2(-e)
    if storage == "e4m3":
        # three bits behind the leading one, and steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        y = torch.round(y / step) * step
    else:
        y = torch.round(y)
    return y * torch.exp2(e), (e + 127).squeeze(-1).to(torch.uint8)


def exact(case, seed):
    state = prepare({k: v for k, v in case.items()}, seed)
    starts, lengths = state["starts"].tolist(), state["lengths"].tolist()
    if case["kind"] == "attend":
        out, lse = [], []
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            n, length = b - a, lengths[s]
            k, v = _exact_held(state, "keys", s), _exact_held(state, "values", s)
            q = state["q"][a:b].double().reshape(n, case["heads"], case["group"], case["width"])
            o = torch.empty_like(q)
            m = torch.empty(q.shape[:3], dtype=torch.float64, device=q.device)
            reach = torch.arange(length, device=q.device)[None, :] > torch.arange(length - n, length, device=q.device)[:, None]
            for h in range(case["heads"]):
                x = torch.einsum("igd,jd->igj", q[:, h], k[:, h]) / math.sqrt(case["width"])
                if case["causal"]:
                    x = x.masked_fill(reach[:, None, :], -math.inf)
                m[:, h] = torch.logsumexp(x, -1)
                o[:, h] = torch.einsum("igj,jd->igd", torch.exp(x - m[:, h, :, None]), v[:, h])
            out.append(o.reshape(n, -1, case["width"]))
            lse.append(m.reshape(n, -1))
        return {"out": torch.cat(out), "lse": torch.cat(lse)}
    if case["kind"] == "read":
        rows = [[_exact_held(state, w, s)[lengths[s] - (b - a):] for s, (a, b) in enumerate(zip(starts, starts[1:]))] for w in ("keys", "values")]
        return {"keys": torch.cat(rows[0]), "values": torch.cat(rows[1])}
    eight = case["kind"] == "store"
    answer = {}
    for x, which in ((state["k"], "keys"), (state["v"], "values")):
        held, byte = _exact_eight(x, case["storage"]) if eight else (x.double(), None)
        pool = None if eight else state[which].double()
        scale = state[which[:-1] + "_scales"]
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            at = torch.arange(lengths[s] - (b - a), lengths[s], device=x.device)
            page, row = state["table"][s][at // case["page_rows"]].long(), at % case["page_rows"]
            if eight:
                scale[page, :, row] = byte[a:b]
            else:
                pool[page, :, row] = held[a:b]
        answer[which] = held if eight else pool
        if eight:
            answer[which[:-1] + "_scales"] = scale
    return answer
