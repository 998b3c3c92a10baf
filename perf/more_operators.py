"""Cases for the operators of a reader's serving step around its 4-bit key/value cache: attention with a window and
first tokens that stay visible, attention of a tree of drafted tokens, page tables and slot maps from the requests'
lengths, rotary positions with several axes, and moving cached tokens.

The cache's format.  A cached vector (one token, one key/value head) is ``head_dim`` symmetric codes in [-7, 7], two
to a byte with the even dimension in the low nibble, and one fp32 scale; pages of ``page_size`` tokens hold ``codes
[pages, kv_heads, page_size, head_dim / 2]`` and ``scales [pages, kv_heads, page_size]``.

``run`` computes in elementary torch operations in 32 bits (angles in 64); with ``own`` it calls the framework.
"""

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # One long answer of a windowed model: a token over the last 1,024 and the first 4 tokens. The smallest call.
        _sinks("one sequence, window and sinks", batch=1, low=30001, high=30001, heads=32, kv_heads=8, head_dim=128,
               dtype="bf16", page_size=64, window=1024, sinks=4),
        # A serving batch: 64 sequences of very different lengths (two not begun) generate a token each; the system
        # prompt's first 64 tokens stay visible.
        _sinks("serving batch, window and sinks", batch=64, low=1, high=16384, empty=2, heads=32, kv_heads=8,
               head_dim=128, dtype="bf16", page_size=64, window=4096, sinks=64),
        # Chunks of long prompts under a window, a first page of 100 tokens visible to all rows: bound by the products.
        _sinks("prompt chunks, window and sinks", batch=4, low=1500, high=16000, q_low=512, q_high=512, heads=32,
               kv_heads=8, head_dim=128, dtype="bf16", page_size=64, window=2048, sinks=100),
        # Trees of 25 to 64 drafted tokens for each of 16 sequences are checked in one call.
        _tree("serving batch, trees", batch=16, low=100, high=8192, q_low=25, q_high=64, heads=32, kv_heads=8,
              head_dim=128, dtype="bf16", page_size=64),
        # A small model without shared heads, small trees of odd sizes, a window with sinks.
        _tree("small trees, window and sinks", batch=7, low=30, high=2000, q_low=1, q_high=13, heads=12, kv_heads=12,
              head_dim=64, dtype="f16", page_size=32, window=255, sinks=3),
        # A step's bookkeeping: each of 64 sequences gets one token's place (and gives it back).
        _pages("a token for each sequence", sequences=64, max_pages=512, page_size=64, low=0, high=20000, new_low=1,
               new_high=1),
        # Chunks of many requests' prompts in small pages; the pool has too few for the last ones.
        _pages("chunks for many requests", sequences=500, max_pages=2048, page_size=16, low=0, high=32000, new_low=0,
               new_high=512),
        # Queries and keys of one token each of 64 sequences, views of the projection's rows.
        _rotate("rotate a token of each sequence", tokens=64, heads=32, kv_heads=8, head_dim=128, dtype="bf16",
                sections="16,24,24"),
        # The patches of a prompt's page images: time, height and width, interleaved over the pairs.
        _rotate("rotate a prompt of page images", tokens=16384, heads=32, kv_heads=8, head_dim=128, dtype="bf16",
                sections="24,20,20", interleaved=True),
        # Odd sizes in fp32: neighbours are pairs, a part of the head rotates, backwards.
        _rotate("rotate odd sizes back", tokens=777, heads=5, kv_heads=1, head_dim=96, dtype="f32", sections="7,17",
                rotary_dim=48, pairs="neighbours", inverse=True),
        # The accepted paths of 64 trees take the first places of their drafts, and are read back: latency counts.
        _move("accepted paths", sequences=64, each=4, kv_heads=8, head_dim=128, page_size=64),
        # A cached document of 16,411 tokens is copied for a second answer, and read back.
        _move("copy a document", sequences=1, each=16411, kv_heads=8, head_dim=128, page_size=64),
    ]


def draw(rng):
    kind = rng.choice(["sinks", "sinks", "sinks", "tree", "tree", "tree", "pages", "rotate", "rotate", "move"])
    if kind == "pages":
        page_size = rng.choice([16, 32, 64, 128])
        high = _log(rng, 1, 32000)
        return {"kind": kind, "sequences": _log(rng, 1, 500), "max_pages": -(-high // page_size) + rng.randint(0, 500),
                "page_size": page_size, "low": rng.randint(0, high), "high": high, "new_low": rng.choice([0, 1]),
                "new_high": _log(rng, 1, 512)}
    if kind == "rotate":
        head_dim = rng.choice([64, 96, 128, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
        interleaved = rng.random() < 0.4
        half = rotary_dim // 2
        if interleaved:
            sections = [half - 2 * (half // 3), half // 3, half // 3]
        else:
            first = rng.randint(1, half - 2)
            second = rng.randint(1, half - first - 1)
            sections = rng.choice([[half], [first, half - first], [first, second, half - first - second]])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        heads, kv_heads = rng.randint(1, 32), rng.randint(0, 8)
        most = 16384 * 40 * 128 * 2 // ((heads + kv_heads) * head_dim * _BYTES[dtype])
        return _case(None, kind=kind, tokens=_log(rng, 1, min(16384, most)), heads=heads, kv_heads=kv_heads,
                     head_dim=head_dim, dtype=dtype, sections=",".join(map(str, sections)), rotary_dim=rotary_dim,
                     interleaved=interleaved, pairs=rng.choice(["halves", "neighbours"]), inverse=rng.random() < 0.2)
    if kind == "move":
        sequences = _log(rng, 1, 100)
        return {"kind": kind, "sequences": sequences, "each": _log(rng, 1, 16411 // sequences),
                "kv_heads": rng.randint(1, 8), "head_dim": rng.choice([64, 128]), "page_size": rng.choice([16, 32, 64, 128])}
    # Attention: no case costs more than the listed ones (bounds on rows, cached tokens and (row, token) pairs).
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    shared = rng.choice([1, 2, 4, 7, 8])
    batch = _log(rng, 1, 64)
    if kind == "tree":
        q_high = min(_log(rng, 1, 100), max(1, 500_000 // (batch * kv_heads * shared)))
    else:
        q_high = min(rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 512)]),
                     max(1, 60_000 // (batch * kv_heads * shared)))
    high = max(q_high, min(_log(rng, 16, 30001), min(500_000, 4_000_000 // kv_heads) // batch))
    window = _log(rng, 16, 4096) if kind == "sinks" or rng.random() < 0.3 else 0
    seen = min(high, window + q_high) if window else high
    while batch > 1 and batch * q_high * kv_heads * shared * seen > 140_000_000:
        batch = (batch + 1) // 2
    while q_high * kv_heads * shared * seen > 140_000_000:
        q_high = (q_high + 1) // 2
    q_low = q_high if q_high == 1 or rng.random() < 0.3 else rng.randint(1, q_high)
    return {"kind": kind, "batch": batch, "low": rng.randint(q_high, high), "high": high,
            "empty": rng.choice([0, 0, 1]) if batch > 1 else 0, "q_low": q_low, "q_high": q_high,
            "heads": kv_heads * shared, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128]),
            "dtype": rng.choice(["bf16", "f16"]), "page_size": rng.choice([16, 32, 64, 128]), "window": window,
            "sinks": rng.choice([1, 4, _log(rng, 2, 256)]) if window else 0}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _case(name, **kw):
    return kw if name is None else dict(name=name, **kw)


def _sinks(name, empty=0, q_low=1, q_high=1, **kw):
    return _case(name, kind="sinks", empty=empty, q_low=q_low, q_high=q_high, **kw)


def _tree(name, empty=0, window=0, sinks=0, **kw):
    return _case(name, kind="tree", empty=empty, window=window, sinks=sinks, **kw)


def _pages(name, **kw):
    return _case(name, kind="pages", **kw)


def _rotate(name, rotary_dim=None, interleaved=False, pairs="halves", inverse=False, **kw):
    return _case(name, kind="rotate", rotary_dim=rotary_dim or kw["head_dim"], interleaved=interleaved, pairs=pairs,
                 inverse=inverse, **kw)


def _move(name, **kw):
    return _case(name, kind="move", **kw)


def _spread(low, high, n):
    """n whole numbers from high down to low."""
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """The lengths and numbers of query tokens of an attention case's sequences; a seed only changes their order."""
    b = case["batch"]
    lengths = _spread(case["low"], case["high"], b)
    for i in range(case["empty"]):
        lengths[b - 1 - i] = 0
    span = case["q_high"] - case["q_low"] + 1
    return lengths, [case["q_high"] - (i * 7919) % span for i in range(b)]


def _requests(case):
    """The lengths of a page table's sequences and what each gets."""
    n = case["sequences"]
    span = case["new_high"] - case["new_low"] + 1
    return _spread(case["low"], case["high"], n), [case["new_high"] - (i * 7919) % span for i in range(n)]


def _axes(case):
    """How many pairs each axis of a rotary case has."""
    return [int(n) for n in case["sections"].split(",")]


def work(case):
    kind = case["kind"]
    if kind == "pages":
        lengths, new = _requests(case)
        size = case["page_size"]
        pages = sum(-(-(n + m) // size) - -(-n // size) for n, m in zip(lengths, new))
        # Lengths and new tokens are read, lengths and offsets written, twice over; new pages read, entered, returned.
        return {"bytes": 12 * sum(new) + 28 * len(lengths) + 16 * pages, "flops": 0}
    if kind == "rotate":
        vectors = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * vectors * case["head_dim"] * _BYTES[case["dtype"]] + 8 * case["tokens"] * len(_axes(case)),
                "flops": 3 * vectors * case["rotary_dim"]}
    if kind == "move":
        tokens = case["sequences"] * case["each"]
        vectors = 2 * tokens * case["kv_heads"]
        # read and written, then read back in fp32
        return {"bytes": vectors * (3 * (case["head_dim"] // 2 + 4) + 4 * case["head_dim"]) + 24 * tokens,
                "flops": vectors * case["head_dim"]}
    lengths, rows = _lengths(case)
    window, sinks = case["window"], case["sinks"]
    seen = pairs = 0
    for length, r in zip(lengths, rows):
        if kind == "tree":  # a row sees itself and, at the least, what is before the drafts
            before = max(0, length - r)
            context = min(before, window - 1 + min(sinks, max(0, before - window + 1))) if window else before
            seen += context + min(length, r)
            pairs += r * (context + 1)
        else:
            first = max(0, length - r)
            some = 0
            for i in range(r):
                p = length - r + i
                if p >= 0:
                    inside = min(p + 1, window)
                    some = inside + min(sinks, p + 1 - inside)
                    pairs += some
            if length > 0:
                inside = min(first + 1, window)
                seen += inside + min(sinks, first + 1 - inside) + (length - 1 - first)
    d = case["head_dim"]
    return {"bytes": seen * case["kv_heads"] * (d + 8) + 2 * sum(rows) * case["heads"] * d * _BYTES[case["dtype"]],
            "flops": 4 * pairs * case["heads"] * d}


def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + salt)
    return g


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _pack(codes):
    codes = codes.to(torch.int16)
    return ((codes[..., 0::2] & 15) | ((codes[..., 1::2] & 15) << 4)).to(torch.uint8)


def _unpack(data):
    """Codes of packed bytes, fp32 [..., 2 * bytes]."""
    low, high = data & 15, data >> 4
    codes = torch.stack((low, high), dim=-1).flatten(-2).to(torch.float32)
    return torch.where(codes > 7, codes - 16, codes)


def _filled_cache(case, pages, g):
    """Pages of keys and values as a model makes them: some key channels are several times wider than the rest."""
    h, s, d = case["kv_heads"], case["page_size"], case["head_dim"]
    wide = 1 + 3 * (torch.rand((h, 1, d), generator=g, device="cuda") < 0.05).float()
    out = []
    for which in range(2):
        codes = torch.empty((pages, h, s, d // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((pages, h, s), dtype=torch.float32, device="cuda")
        step = max(1, (1 << 26) // (h * s * d))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            x = _normal((n, h, s, d), g) * (wide if which == 0 else 0.3)
            scale = x.abs().amax(dim=-1) / 7
            codes[at:at + n] = _pack(torch.round(x / scale.unsqueeze(-1)).clamp(-7, 7))
            scales[at:at + n] = scale
        out += [codes, scales]
    return dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), out))


def prepare(case, seed):
    g = _generator(seed, 29)
    state = {"case": case}
    kind = case["kind"]
    if kind == "rotate":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        qkv = _normal((t, h + 2 * kv, d), g, _TYPES[case["dtype"]])
        state["query"], state["keys"] = qkv[:, :h], qkv[:, h:h + kv] if kv else None
        if len(_axes(case)) == 1:
            # Far positions of a running sequence.
            state["positions"] = 100_000 + torch.arange(t, device="cuda").view(1, t) + 7 * seed
        else:
            # Patches of images of 37 x 29, one after the other: image, row, column, as models count them.
            i = torch.arange(t, device="cuda")
            image, place = i // 1073, i % 1073
            start = 500 + image * 38 + seed
            axes = (start, start + place // 29, start + place % 29)
            state["positions"] = torch.stack(axes[:len(_axes(case))])
        if own:
            from maxsim_b200 import Rotary

            state["rotary"] = Rotary(d, sections=_axes(case), theta=1e6, rotary_dim=case["rotary_dim"],
                                     interleaved=case["interleaved"], pairs=case["pairs"])
        else:  # angles a position and pair in 64 bits, the pairs' axes
            half = case["rotary_dim"] // 2
            state["frequencies"] = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
            axis = [a for a, n in enumerate(_axes(case)) for _ in range(n)]
            if case["interleaved"]:
                axis = [i % 3 if i < 3 * _axes(case)[i % 3] else 0 for i in range(half)]
            state["axis"] = torch.tensor(axis, device="cuda")
        return state
    if kind == "pages":
        lengths, new = _requests(case)
        order = list(range(case["sequences"]))
        random.Random(seed).shuffle(order)
        lengths, new = [lengths[i] for i in order], [new[i] for i in order]
        size, columns = case["page_size"], case["max_pages"]
        length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        have = (length + size - 1) // size
        # All that is asked for, but for the last hundredth of it.
        used = int(have.sum())
        wanted = sum(-(-(n + m) // size) - -(-n // size) for n, m in zip(lengths, new))
        spare = wanted - wanted // 100 + 1
        ids = torch.randperm(used + spare, generator=g, device="cuda").to(torch.int32)
        column = torch.arange(columns, device="cuda").unsqueeze(0)
        inside = column < have.unsqueeze(1)
        place = (torch.cumsum(have, 0) - have).unsqueeze(1) + column
        state["page_table"] = torch.where(inside, ids[torch.where(inside, place, 0)], -1).to(torch.int32)
        state["lengths"] = length
        state["free_pages"] = torch.cat((ids[used:], torch.full((used,), -1, dtype=torch.int32, device="cuda")))
        state["free_count"] = torch.tensor([spare], dtype=torch.int32, device="cuda")
        state["before"] = length.clone()
        state["tokens"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        state["rows"] = sum(new) + 3  # a step's rows are padded
        if own:
            from maxsim_b200 import PageTable

            state["pages"] = PageTable.from_tensors(state["page_table"], state["lengths"], state["free_pages"],
                                                    state["free_count"], page_size=size)
        return state
    page = case["page_size"]
    if kind == "move":
        # Sources and targets lie in pages of their own order, targets apart from sources.
        n, each = case["sequences"], case["each"]
        drafted = 4 * each if n > 1 else 2 * each
        per = -(-drafted // page)
        cache = _filled_cache(case, n * per + 1, g)
        ids = torch.randperm(n * per + 1, generator=g, device="cuda")[:n * per].view(n, per)
        target = torch.arange(each, device="cuda").expand(n, each)
        if n > 1:  # nodes of the tree behind its first ones, ascending
            step = torch.randint(1, 4, (n, each), generator=g, device="cuda")
            source = each - 1 + torch.cumsum(step, 1)
        else:
            source = target + each
        row = torch.arange(n, device="cuda").unsqueeze(1)
        state["source"] = (ids[row, source // page] * page + source % page).flatten()
        state["target"] = (ids[row, target // page] * page + target % page).flatten()
    else:
        lengths, rows = _lengths(case)
        rng = random.Random(seed)
        order = list(range(case["batch"]))
        rng.shuffle(order)
        lengths, rows = [lengths[i] for i in order], [rows[i] for i in order]
        per = -(-max(lengths) // page)
        used = [-(-n // page) for n in lengths]
        pages = sum(used) + 1
        cache = _filled_cache(case, pages, g)
        # Pages in any order; table entries past a sequence's end name page 0.
        ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        first = torch.tensor([sum(used[:i]) for i in range(len(used))], device="cuda").unsqueeze(1)
        column = torch.arange(per, device="cuda").unsqueeze(0)
        inside = column * page < length.unsqueeze(1)
        state["page_table"] = torch.where(inside, ids[(first + column).clamp(max=pages - 1)], 0).to(torch.int32)
        state["lengths"] = length
        at = [0]
        for r in rows:
            at.append(at[-1] + r)
        state["query_offsets"] = (None if case["q_high"] == 1 and kind == "sinks" else
                                  torch.tensor(at, dtype=torch.int32, device="cuda"))
        state["query"] = _normal((at[-1], case["heads"], case["head_dim"]), g, _TYPES[case["dtype"]]) * 1.5
        if kind == "tree":  # a node's parent is one of the eight before it, or the context's last token
            parents = [rng.randint(max(-1, i - 8), i - 1) for r in rows for i in range(r)]
            state["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
    state.update(cache)
    if own:
        from maxsim_b200 import Int4KVCache

        state["cache"] = Int4KVCache.from_tensors(cache["k_codes"], cache["k_scales"], cache["v_codes"],
                                                  cache["v_scales"])
    return state


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "rotate":
        if own:
            query, keys = state["rotary"](state["query"], state["keys"], state["positions"], inverse=case["inverse"])
        else:
            query, keys = _plain_rotate(state, state["query"]), _plain_rotate(state, state["keys"])
        return {"query": query} if keys is None else {"query": query, "keys": keys}
    if kind == "pages":
        if own:
            pages = state["pages"]
            offsets, slots, positions = pages.extend(state["tokens"], state["rows"])
            pages.truncate(state["before"])
        else:
            offsets, slots, positions = _plain_extend(state)
            _plain_truncate(state, state["before"])
        return {"offsets": offsets, "slots": slots, "positions": positions, "page_table": state["page_table"],
                "lengths": state["lengths"], "free_pages": state["free_pages"], "free_count": state["free_count"]}
    if kind == "move":
        if own:
            state["cache"].move(state["source"], state["target"])
            keys, values = state["cache"].read(state["target"], dtype=torch.float32)
        else:
            _plain_move(state)
            keys, values = _plain_read(state, "k"), _plain_read(state, "v")
        return {"keys": keys, "values": values}
    if own:
        ancestors, out = None, {}
        if kind == "tree":
            from maxsim_b200 import draft_ancestors

            ancestors, out["depths"] = draft_ancestors(state["parents"], state["query_offsets"],
                                                       max_query_tokens=case["q_high"])
        out["rows"] = state["cache"].attend(state["query"], state["page_table"], state["lengths"],
                                            query_offsets=state["query_offsets"], max_query_tokens=case["q_high"],
                                            window=case["window"] or None, sinks=case["sinks"], ancestors=ancestors)
        return out
    return _plain_attend(state)


def _plain_rotate(state, x):
    case = state["case"]
    if x is None:
        return None
    rotary, half = case["rotary_dim"], case["rotary_dim"] // 2
    angle = state["positions"][state["axis"]].t() * state["frequencies"]
    if case["inverse"]:
        angle = -angle
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    turned = x[..., :rotary].float()
    if case["pairs"] == "halves":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    return torch.cat((turned.to(x.dtype), x[..., rotary:]), dim=-1)


def _plain_extend(state):
    case = state["case"]
    size, rows = case["page_size"], state["rows"]
    table, lengths, free, count = (state[n] for n in ("page_table", "lengths", "free_pages", "free_count"))
    device = table.device
    n, columns = table.shape
    new = state["tokens"].long().clamp(min=0)
    end = torch.cumsum(new, 0)
    length = lengths.long()
    have, want = (length + size - 1) // size, (length + new + size - 1) // size
    fits = (want <= columns) & (end <= rows)
    grow = torch.where(fits, want - have, 0)
    upto = torch.cumsum(grow, 0)
    served = fits & ((grow == 0) | (upto <= count))  # one that lacks no page gets its rows all the same
    column = torch.arange(columns, device=device).unsqueeze(0)
    entered = served.unsqueeze(1) & (column >= have.unsqueeze(1)) & (column < want.unsqueeze(1))
    place = count.long() - 1 - ((upto - grow - have).unsqueeze(1) + column)
    table.copy_(torch.where(entered, free[torch.where(entered, place, 0)], table))
    lengths.copy_(torch.where(served, length + new, length))
    count.sub_(torch.where(served, grow, 0).sum().to(torch.int32))
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64, device=device), end)).clamp(max=rows).to(torch.int32)
    row = torch.arange(rows, device=device)
    seq = torch.searchsorted(end, row, right=True)
    known = seq < n
    seq = seq.clamp(max=n - 1)
    known = known & served[seq]
    position = torch.where(known, length[seq] + row - (end - new)[seq], -1)
    held = position.clamp(min=0)
    slot = table[seq, (held // size).clamp(max=columns - 1)].long() * size + held % size
    return offsets, torch.where(known, slot, -1), position.to(torch.int32)


def _plain_truncate(state, to):
    size = state["case"]["page_size"]
    table, lengths, free, count = (state[n] for n in ("page_table", "lengths", "free_pages", "free_count"))
    length = lengths.long()
    left = torch.minimum(to.long().clamp(min=0), length)
    have, keep = (length + size - 1) // size, (left + size - 1) // size
    back = have - keep
    upto = torch.cumsum(back, 0)
    column = torch.arange(table.shape[1], device=table.device).unsqueeze(0)
    leaves = (column >= keep.unsqueeze(1)) & (column < have.unsqueeze(1))
    # The first sequence's first page comes to lie on top.
    place = count.long() + upto[-1] - 1 - ((upto - back - keep).unsqueeze(1) + column)
    free[place[leaves]] = table[leaves]
    table[leaves] = -1
    count.add_(upto[-1].to(torch.int32))
    lengths.copy_(left)


def _plain_move(state):
    page = state["case"]["page_size"]
    for name in ("k", "v"):
        codes, scales = state[name + "_codes"], state[name + "_scales"]
        s, t = state["source"], state["target"]
        moved, by = codes[s // page, :, s % page], scales[s // page, :, s % page]
        codes[t // page, :, t % page] = moved
        scales[t // page, :, t % page] = by


def _plain_read(state, name):
    page = state["case"]["page_size"]
    codes, scales, t = state[name + "_codes"], state[name + "_scales"], state["target"]
    return _unpack(codes[t // page, :, t % page]) * scales[t // page, :, t % page].unsqueeze(-1)


def _plain_ancestors(state, seq, place, offsets, most):
    """[rows, most] truth values: the row sees this node of its sequence's tree (its ancestors and itself)."""
    rows = place.shape[0]
    parent = state["parents"].long()
    seen = torch.zeros((rows, most), dtype=torch.bool, device=place.device)
    at, alive = place.clone(), torch.ones_like(place, dtype=torch.bool)
    row = torch.arange(rows, device=place.device)
    for _ in range(most):  # no path is longer than the tree
        seen[row, at] = seen[row, at] | alive
        up = parent[offsets[seq] + at]
        alive = alive & (up >= 0)
        at = torch.where(alive, up, at)
    return seen


def _plain_attend(state):
    case = state["case"]
    q, table, lengths = state["query"], state["page_table"].long(), state["lengths"].long()
    b, h, d, page = case["batch"], case["kv_heads"], case["head_dim"], case["page_size"]
    shared, most, span = case["heads"] // h, case["q_high"], table.shape[1] * page
    window, sinks, tree = case["window"], case["sinks"], case["kind"] == "tree"
    device = q.device
    offsets = state["query_offsets"]
    offsets = (torch.arange(b + 1, device=device) if offsets is None else offsets).long()
    row = torch.arange(q.shape[0], device=device)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    place = row - offsets[seq]
    first = lengths - (offsets[1:] - offsets[:-1])  # the position of a sequence's first row
    # The tokens that some row may see: the sinks, then those from the first row's window on.
    near = span if not window else min(span, window + most)
    begin = (first - window).clamp(min=sinks) if window else torch.zeros_like(first)
    j = torch.cat((torch.arange(sinks, device=device).expand(b, sinks),
                   begin.unsqueeze(1) + torch.arange(near, device=device)), dim=1)
    pages = torch.gather(table, 1, (j // page).clamp(max=table.shape[1] - 1))
    k = (_unpack(state["k_codes"][pages, :, j % page]) * state["k_scales"][pages, :, j % page].unsqueeze(-1)).transpose(1, 2)
    v = (_unpack(state["v_codes"][pages, :, j % page]) * state["v_scales"][pages, :, j % page].unsqueeze(-1)).transpose(1, 2)
    padded = torch.zeros((b, most, h * shared, d), dtype=torch.float32, device=device)
    padded[seq, place] = q.float()
    padded = padded.view(b, most, h, shared, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * shared, d)
    score = (padded @ k.transpose(2, 3)).view(b, h, most, shared, -1) / math.sqrt(d)
    at = j.unsqueeze(1)
    out = {}
    if tree:
        nodes = _plain_ancestors(state, seq, place, offsets, most)
        count = nodes.sum(dim=1)
        out["depths"] = (count - 1).to(torch.int32)
        tree_nodes = torch.zeros((b, most, most), dtype=torch.bool, device=device)
        tree_nodes[seq, place] = nodes
        counts = torch.zeros((b, most), dtype=torch.int64, device=device)
        counts[seq, place] = count
        node = at - first.view(b, 1, 1)
        seen = torch.gather(tree_nodes, 2, node.clamp(0, most - 1).expand(b, most, -1)) & (node >= 0) & (node < most)
        context = (at < first.view(b, 1, 1)).expand(b, most, -1)
        if window:
            context = context & ((at >= (first.unsqueeze(1) + counts - window).unsqueeze(2)) | (at < sinks))
        seen = seen | context
    else:
        pos = (first.unsqueeze(1) + torch.arange(most, device=device)).unsqueeze(2)
        seen = (at <= pos) & ((at > pos - window) | (at < sinks))
    seen = (seen & (at < lengths.view(b, 1, 1))).view(b, 1, most, 1, -1)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = (p.view(b, h, most * shared, -1) @ v).view(b, h, most, shared, d).permute(0, 2, 1, 3, 4)
    out["rows"] = o.reshape(b, most, h * shared, d)[seq, place].to(q.dtype)
    return out


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers only
    state = prepare(case, seed)
    f64 = torch.float64

    def value(data, scale):
        """Bytes [..., d / 2] and scales [...] -> values in 64 bits."""
        out = torch.empty(data.shape[:-1] + (2 * data.shape[-1],), dtype=f64, device=data.device)
        out[..., 0::2] = ((data.to(torch.int16) & 15) ^ 8).to(f64) - 8
        out[..., 1::2] = ((data.to(torch.int16) >> 4) ^ 8).to(f64) - 8
        return out.mul_(scale.to(f64).unsqueeze(-1))

    if case["kind"] == "rotate":
        half, n = case["rotary_dim"] // 2, len(_axes(case))
        positions = state["positions"].to(f64)
        first, second = ([2 * i for i in range(half)], [2 * i + 1 for i in range(half)]) if case["pairs"] == "neighbours" \
            else (list(range(half)), list(range(half, 2 * half)))
        out = {}
        for name in ("query", "keys"):
            if state[name] is None:
                continue
            x = state[name].to(f64)
            for i in range(half):
                if case["interleaved"]:
                    axis = i % n if i < n * _axes(case)[i % n] else 0
                else:
                    axis, left = 0, i
                    while left >= _axes(case)[axis]:
                        left -= _axes(case)[axis]
                        axis += 1
                turn = positions[axis] * math.pow(1e6, -i / half) * (-1 if case["inverse"] else 1)
                c, s = torch.cos(turn).unsqueeze(1), torch.sin(turn).unsqueeze(1)
                u, w = x[:, :, first[i]].clone(), x[:, :, second[i]].clone()
                x[:, :, first[i]] = c * u - s * w
                x[:, :, second[i]] = s * u + c * w
            out[name] = x
        return out
    page = case["page_size"]
    if case["kind"] == "move":
        p, i = state["source"] // page, state["source"] % page
        return {"keys": value(state["k_codes"][p, :, i], state["k_scales"][p, :, i]),
                "values": value(state["v_codes"][p, :, i], state["v_scales"][p, :, i])}
    query = state["query"].to(f64)
    shared, window, sinks = case["heads"] // case["kv_heads"], case["window"], case["sinks"]
    out = torch.zeros_like(query)
    lengths = state["lengths"].tolist()
    offsets = list(range(case["batch"] + 1)) if state["query_offsets"] is None else state["query_offsets"].tolist()
    parents = state["parents"].tolist() if case["kind"] == "tree" else None
    for b, length in enumerate(lengths):
        rows = offsets[b + 1] - offsets[b]
        if length == 0:
            continue
        first = length - rows
        seen = torch.zeros((rows, length), dtype=torch.bool)
        for i in range(rows):
            if parents is None:
                p = first + i
                if p >= 0:
                    seen[i, max(0, p - window + 1):p + 1] = True
                    seen[i, :min(sinks, p + 1)] = True
                continue
            path, at = [], i
            while at >= 0:
                path.append(at)
                at = parents[offsets[b] + at]
            if first > 0:
                low = 0 if not window else min(max(0, first + len(path) - window), first)
                seen[i, low:first] = True
                seen[i, :min(sinks, first)] = True
            for node in path:
                if first + node >= 0:
                    seen[i, first + node] = True
        keep = seen.any(dim=0).nonzero().squeeze(1)  # the tokens that some row sees
        seen = seen[:, keep].cuda()
        keep = keep.cuda()
        pages = state["page_table"][b].long()[keep // page]
        for head in range(case["kv_heads"]):
            k = value(state["k_codes"][pages, head, keep % page], state["k_scales"][pages, head, keep % page])
            v = value(state["v_codes"][pages, head, keep % page], state["v_scales"][pages, head, keep % page])
            for at in range(0, rows, 64):
                n = min(64, rows - at)
                here = slice(offsets[b] + at, offsets[b] + at + n), slice(head * shared, (head + 1) * shared)
                off = ~seen[at:at + n].unsqueeze(1)
                s = torch.einsum("nsd,jd->nsj", query[here], k) * case["head_dim"] ** -0.5
                w = torch.softmax(s.masked_fill(off, -torch.inf), dim=-1)
                out[here] = torch.where(off.all(dim=-1, keepdim=True), 0.0, torch.einsum("nsj,jd->nsd", w, v))
    return {"rows": out} if parents is None else {"depths": None, "rows": out}
