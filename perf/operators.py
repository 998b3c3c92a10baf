"""Cases for the operators of a reader model that answers from retrieved passages: a key/value cache held in
4 bits (written, read back, attended over) and products of few rows with 4-bit weights.

Formats.  A cached vector (one token, one key/value head) is ``head_dim`` symmetric codes in [-7, 7], two to a
byte with the even dimension in the low nibble, and one fp32 scale.  Pages of ``page_size`` tokens hold
``codes [pages, kv_heads, page_size, head_dim / 2]`` and ``scales [pages, kv_heads, page_size]``.  A weight
``[out, in]`` is the same codes with one bfloat16 scale per row and group of ``group`` inputs.

``run`` computes in elementary torch operations in 32 bits; with ``own`` it calls the framework.
"""

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # One token of each of 64 running sequences goes into the cache and is read back: latency counts.
        _write("write one token each", tokens=64, kv_heads=8, head_dim=128, dtype="bf16", page_size=16),
        # The passages of a prompt are written at once and read back.
        _write("write a prompt", tokens=32768, kv_heads=8, head_dim=128, dtype="bf16", page_size=64),
        # A short passage of a small model is read back for another consumer, in fp32.
        _read("read a short passage", tokens=777, kv_heads=5, head_dim=64, dtype="f32", page_size=32),
        # A long document's cache is read back in the model's type.
        _read("read a document", tokens=32768, kv_heads=8, head_dim=128, dtype="bf16", page_size=64),
        # One sequence with one page of 1,030 patch tokens generates a token: the smallest call.
        _attend("one sequence, one token", batch=1, low=1030, high=1030, heads=32, kv_heads=8, head_dim=128,
                dtype="bf16", page_size=64),
        # A serving batch: 64 sequences of very different lengths (two not begun) generate a token each.
        _attend("serving batch, one token", batch=64, low=1, high=8192, empty=2, heads=32, kv_heads=8, head_dim=128,
                dtype="bf16", page_size=64),
        # Two sequences over very long contexts, eight query heads to a key/value head.
        _attend("long contexts, one token", batch=2, low=100003, high=131071, heads=64, kv_heads=8, head_dim=128,
                dtype="f16", page_size=128),
        # Chunks of prompts over what is cached already: causal within the chunk, bound by the products.
        _attend("prompt chunks", batch=4, low=1500, high=4096, q_low=512, q_high=512, heads=32, kv_heads=8,
                head_dim=128, dtype="bf16", page_size=64),
        # A small model without shared heads: sliding window, one to five drafted tokens to check per sequence.
        _attend("drafted tokens, window", batch=7, low=3, high=2000, q_low=1, q_high=5, heads=12, kv_heads=12,
                head_dim=64, dtype="f16", page_size=32, window=255),
        # The projection of one token.
        _product("one row", rows=1, n=4096, k=4096, group=128, dtype="bf16"),
        # A wide layer for a serving batch.
        _product("wide layer, 16 rows", rows=16, n=16384, k=8192, group=64, dtype="bf16"),
        # Odd sizes, the finest scales, a bias.
        _product("odd sizes, 5 rows", rows=5, n=1111, k=2080, group=32, dtype="f16", bias=True),
    ]


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "product", "product"])
    dtype = rng.choice(["bf16", "f16"])
    if kind in ("write", "read"):
        return {"kind": kind, "tokens": _log(rng, 1, 32768), "kv_heads": rng.randint(1, 8),
                "head_dim": rng.choice([64, 128]), "dtype": rng.choice(["bf16", "f16", "f32"]) if kind == "read" else dtype,
                "page_size": rng.choice([16, 32, 64, 128])}
    if kind == "product":
        group = rng.choice([32, 64, 128])
        return {"kind": kind, "rows": _log(rng, 1, 32), "n": _log(rng, 100, 16384),
                "k": 8 * _log(rng, 64, 1024), "group": group, "dtype": dtype, "bias": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    shared = rng.choice([1, 2, 4, 7, 8, 16])
    q_high = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 512)])
    batch = _log(rng, 1, 64)
    # No case costs more than the listed ones: bounds on rows, on cached tokens and on (row, token) pairs.
    q_high = min(q_high, max(1, 700_000 // (batch * kv_heads * shared)))
    q_low = q_high if q_high == 1 or rng.random() < 0.3 else rng.randint(1, q_high)
    high = _log(rng, 16, 131072)
    high = max(1, min(high, min(500_000, 3_200_000 // kv_heads) // batch,
                      160_000_000 // (batch * q_high * kv_heads * shared)))
    return {"kind": "attend", "batch": batch, "low": rng.randint(1, high), "high": high,
            "empty": rng.choice([0, 0, 1]) if batch > 1 else 0, "q_low": q_low, "q_high": q_high,
            "heads": kv_heads * shared, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128]), "dtype": dtype,
            "page_size": rng.choice([16, 32, 64, 128]),
            "window": rng.choice([0, 0, _log(rng, 1, 4096)])}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _write(name, **kw):
    return dict(name=name, kind="write", **kw)


def _read(name, **kw):
    return dict(name=name, kind="read", **kw)


def _attend(name, empty=0, q_low=1, q_high=1, window=0, **kw):
    return dict(name=name, kind="attend", empty=empty, q_low=q_low, q_high=q_high, window=window, **kw)


def _product(name, bias=False, **kw):
    return dict(name=name, kind="product", bias=bias, **kw)


def _lengths(case):
    """The lengths and numbers of query tokens of a case's sequences; a seed only changes their order."""
    b, low, high = case["batch"], case["low"], case["high"]
    lengths = [high - (high - low) * i // max(1, b - 1) for i in range(b)]
    for i in range(case["empty"]):
        lengths[b - 1 - i] = 0
    span = case["q_high"] - case["q_low"] + 1
    return lengths, [case["q_high"] - (i * 7919) % span for i in range(b)]


def _visible(case, length, rows):
    """Cached tokens that some row sees, and the number of (row, token) pairs."""
    seen, pairs = 0, 0
    for i in range(rows):
        pos = length - rows + i
        if pos >= 0:
            pairs += min(pos + 1, case["window"] or pos + 1)
    if length > 0:
        first = max(0, length - rows)
        seen = min(length, first + 1 if not case["window"] else case["window"]) + (length - 1 - first)
        seen = min(seen, length)
    return seen, pairs


def work(case):
    kind = case["kind"]
    if kind in ("write", "read"):
        vectors = 2 * case["tokens"] * case["kv_heads"]
        wide, packed = vectors * case["head_dim"], vectors * (case["head_dim"] // 2 + 4)
        if kind == "read":
            return {"bytes": packed + wide * _BYTES[case["dtype"]] + 8 * case["tokens"], "flops": wide}
        # written once, read back once in fp32
        return {"bytes": wide * _BYTES[case["dtype"]] + 2 * packed + 4 * wide + 16 * case["tokens"], "flops": 4 * wide}
    if kind == "product":
        m, n, k = case["rows"], case["n"], case["k"]
        groups = -(-k // case["group"])
        return {"bytes": n * k // 2 + 2 * n * groups + 2 * m * (n + k) + (2 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    lengths, rows = _lengths(case)
    seen = pairs = 0
    for length, r in zip(lengths, rows):
        s, p = _visible(case, length, r)
        seen += s
        pairs += p
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


def _quantise(x):
    """fp32 vectors -> (codes, fp32 scales)."""
    scale = x.abs().amax(dim=-1) / 7
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x / scale.unsqueeze(-1)).clamp(-7, 7), scale


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
            c, sc = _quantise(x)
            codes[at:at + n], scales[at:at + n] = _pack(c), sc
        out += [codes, scales]
    return dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), out))


def prepare(case, seed):
    kind = case["kind"]
    g = _generator(seed, 17)
    state = {"case": case}
    if kind == "product":
        n, k, group = case["n"], case["k"], case["group"]
        groups = -(-k // group)
        w = _normal((n, k), g) / math.sqrt(k)
        w = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
        scale = (w.abs().amax(dim=-1) / 7).to(torch.bfloat16)
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        codes = torch.round(w / scale.float().unsqueeze(-1)).clamp(-7, 7).view(n, -1)[:, :k]
        state["codes"], state["scales"] = _pack(codes), scale
        state["x"] = _normal((case["rows"], k), g, _TYPES[case["dtype"]])
        state["bias"] = _normal((n,), g, _TYPES[case["dtype"]]) if case["bias"] else None
        if own:  # the weights as the framework lays them out, once
            from maxsim_b200 import Int4Linear

            state["linear"] = Int4Linear(state["codes"], state["scales"], group_size=group, bias=state["bias"])
        return state
    page = case["page_size"]
    if kind in ("write", "read"):
        t, h, d = case["tokens"], case["kv_heads"], case["head_dim"]
        pages = -(-t // page) + 3
        cache = _filled_cache(case, pages, g)
        order = torch.randperm(pages, generator=g, device="cuda")
        slot = torch.arange(t, device="cuda")
        state["slots"] = order[slot // page] * page + slot % page
        if kind == "write":
            state["keys"] = _normal((t, h, d), g, _TYPES[case["dtype"]])
            state["values"] = _normal((t, h, d), g, _TYPES[case["dtype"]]) * 0.3
    else:
        lengths, rows = _lengths(case)
        order = list(range(case["batch"]))
        random.Random(seed).shuffle(order)
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
        state["query_offsets"] = None if case["q_high"] == 1 else torch.tensor(at, dtype=torch.int32, device="cuda")
        state["query"] = _normal((at[-1], case["heads"], case["head_dim"]), g, _TYPES[case["dtype"]]) * 1.5
    state.update(cache)
    if own:  # the cache as the framework's object over the same tensors
        from maxsim_b200 import Int4KVCache

        state["cache"] = Int4KVCache.from_tensors(cache["k_codes"], cache["k_scales"], cache["v_codes"],
                                                  cache["v_scales"])
    return state


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        if kind == "product":
            return state["linear"](state["x"])
        cache = state["cache"]
        if kind == "write":
            cache.append(state["keys"], state["values"], state["slots"])
            keys, values = cache.read(state["slots"], dtype=torch.float32)
            return {"keys": keys, "values": values}
        if kind == "read":
            keys, values = cache.read(state["slots"], dtype=_TYPES[case["dtype"]])
            return {"keys": keys, "values": values}
        return cache.attend(state["query"], state["page_table"], state["lengths"],
                            query_offsets=state["query_offsets"], max_query_tokens=case["q_high"],
                            window=case["window"] or None)
    if kind == "product":
        return _plain_product(state)
    if kind == "attend":
        return _plain_attend(state)
    if kind == "write":
        _plain_write(state["keys"], state["k_codes"], state["k_scales"], state["slots"])
        _plain_write(state["values"], state["v_codes"], state["v_scales"], state["slots"])
    out = torch.float32 if kind == "write" else _TYPES[case["dtype"]]
    return {"keys": _plain_read(state["k_codes"], state["k_scales"], state["slots"]).to(out),
            "values": _plain_read(state["v_codes"], state["v_scales"], state["slots"]).to(out)}


def _plain_write(x, codes, scales, slots):
    c, s = _quantise(x.float())
    page = codes.shape[2]
    codes[slots // page, :, slots % page] = _pack(c)
    scales[slots // page, :, slots % page] = s


def _plain_read(codes, scales, slots):
    page = codes.shape[2]
    return _unpack(codes[slots // page, :, slots % page]) * scales[slots // page, :, slots % page].unsqueeze(-1)


def _plain_product(state):
    codes = _unpack(state["codes"])
    n, k = codes.shape
    w = codes * state["scales"].float().repeat_interleave(state["case"]["group"], dim=1)[:, :k]
    y = state["x"].float() @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _plain_attend(state):
    case = state["case"]
    q, table, lengths = state["query"], state["page_table"].long(), state["lengths"].long()
    b, h, d, page = case["batch"], case["kv_heads"], case["head_dim"], case["page_size"]
    shared, most, span = case["heads"] // h, case["q_high"], table.shape[1] * page
    k = (_unpack(state["k_codes"][table]) * state["k_scales"][table].unsqueeze(-1)).transpose(1, 2).reshape(b, h, span, d)
    v = (_unpack(state["v_codes"][table]) * state["v_scales"][table].unsqueeze(-1)).transpose(1, 2).reshape(b, h, span, d)
    offsets = state["query_offsets"]
    if offsets is None:
        offsets = torch.arange(b + 1, device=q.device)
    offsets = offsets.long()
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    place = row - offsets[seq]
    padded = torch.zeros((b, most, h * shared, d), dtype=torch.float32, device=q.device)
    padded[seq, place] = q.float()
    padded = padded.view(b, most, h, shared, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * shared, d)
    score = (padded @ k.transpose(2, 3)).view(b, h, most, shared, span) / math.sqrt(d)
    j = torch.arange(span, device=q.device)
    pos = (lengths - (offsets[1:] - offsets[:-1])).unsqueeze(1) + torch.arange(most, device=q.device)
    seen = (j <= pos.unsqueeze(2)) & (j < lengths.view(b, 1, 1))
    if case["window"]:
        seen = seen & (j > pos.unsqueeze(2) - case["window"])
    seen = seen.view(b, 1, most, 1, span)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = (p.view(b, h, most * shared, span) @ v).view(b, h, most, shared, d).permute(0, 2, 1, 3, 4)
    return o.reshape(b, most, h * shared, d)[seq, place].to(q.dtype)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64

    def value(data, scale):
        """Bytes [..., d / 2] and scales [...] -> values in 64 bits."""
        out = torch.empty(data.shape[:-1] + (2 * data.shape[-1],), dtype=f64, device=data.device)
        out[..., 0::2] = ((data.to(torch.int16) & 15) ^ 8).to(f64) - 8
        out[..., 1::2] = ((data.to(torch.int16) >> 4) ^ 8).to(f64) - 8
        return out.mul_(scale.to(f64).unsqueeze(-1))

    if kind == "product":
        out = []
        for at in range(0, case["n"], 1024):  # in pieces of the rows
            w = value(state["codes"][at:at + 1024], torch.ones((min(1024, case["n"] - at),), device="cuda"))
            for i in range(state["scales"].shape[1]):
                w[:, i * case["group"]:(i + 1) * case["group"]] *= state["scales"][at:at + 1024, i:i + 1].to(f64)
            out.append(state["x"].to(f64) @ w.t())
        y = torch.cat(out, dim=1)
        return y if state["bias"] is None else y + state["bias"].to(f64)
    if kind == "write":
        both = {}
        for name in ("keys", "values"):
            # The format's scale and the quotient that is rounded to a code are fp32 numbers (in 64 bits the
            # many ties of 16-bit inputs, such as half of a vector's maximum, would fall to either side).
            x = state[name].to(torch.float32)
            s = x.abs().max(dim=-1, keepdim=True).values.div(7)
            s[s == 0] = 1
            both[name] = torch.round((x / s).to(f64)).clamp_(-7, 7) * s.to(f64)
        return both
    page = case["page_size"]
    if kind == "read":
        p, i = state["slots"] // page, state["slots"] % page
        return {"keys": value(state["k_codes"][p, :, i], state["k_scales"][p, :, i]),
                "values": value(state["v_codes"][p, :, i], state["v_scales"][p, :, i])}
    query = state["query"].to(f64)
    shared = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(query)
    lengths = state["lengths"].tolist()
    offsets = list(range(case["batch"] + 1)) if state["query_offsets"] is None else state["query_offsets"].tolist()
    for b, length in enumerate(lengths):
        rows = offsets[b + 1] - offsets[b]
        pages = state["page_table"][b, :-(-length // page)].long()
        if length == 0:
            continue
        for head in range(case["kv_heads"]):
            k = value(state["k_codes"][pages, head], state["k_scales"][pages, head]).flatten(0, 1)[:length]
            v = value(state["v_codes"][pages, head], state["v_scales"][pages, head]).flatten(0, 1)[:length]
            for at in range(0, rows, 64):
                n = min(64, rows - at)
                here = slice(offsets[b] + at, offsets[b] + at + n), slice(head * shared, (head + 1) * shared)
                s = torch.einsum("nsd,jd->nsj", query[here], k) * case["head_dim"] ** -0.5
                pos = (length - rows + at + torch.arange(n, device="cuda")).view(n, 1, 1)
                j = torch.arange(length, device="cuda").view(1, 1, length)
                off = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j < 0))
                w = torch.softmax(s.masked_fill(off, -torch.inf), dim=-1)
                out[here] = torch.where(off.all(dim=-1, keepdim=True), 0.0, torch.einsum("nsj,jd->nsd", w, v))
    return out
