"""What the operators of a decoding step over a paged key-value cache are measured on.

A case is a dict of plain values. Its "op" names the operator a pass goes through:

* ``tables``: ``decode.kv_block_tables``: pages for the tokens a step adds, their slots, positions and offsets, from the
  requests' lengths;
* ``append``: ``decode.kv_cache_append``: new key and value rows into their slots, as they are or as the framework's 8-bit rows
  (``store`` "rows8"; the pass then reads the cache back as the values it stands for, with ``ops.dequantize_rowwise``);
* ``attention``: ``decode.paged_attention``: one new token of every request over its pages, 16-bit rows or 8-bit ones;
* ``logits``: ``decode.penalize_logits``: penalties for repeated tokens, biases and a grammar mask on the step's logits.

Lengths are spread evenly between a shortest and a longest and dealt to the requests from the seed; pages are a random
permutation of the cache, which is full of earlier rows.
"""
import math

import torch

own = False

_TORCH = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # One step of a server with 64 requests in flight: a token each, now and then a page.
        {"name": "tables_step", "op": "tables", "requests": 64, "prefills": 0, "chunk": 1, "context": 4096, "block": 16, "bits": 32},
        # A large mixed step: 2 048 requests, an eighth of them with a chunk of their prompt, wide tables, 64-bit lengths.
        {"name": "tables_mixed", "op": "tables", "requests": 2048, "prefills": 256, "chunk": 1023, "context": 8191, "block": 16, "bits": 64},
        # The rows of one decoding step, cut out of the fused projection's output.
        {"name": "append_step", "op": "append", "tokens": 64, "heads": 8, "dim": 128, "block": 16, "type": "bf16", "store": "same", "group": 4},
        # The rows of several prompts at once.
        {"name": "append_prompts", "op": "append", "tokens": 16384, "heads": 8, "dim": 128, "block": 16, "type": "fp16", "store": "same", "group": 4},
        # Prompts into a cache of 8-bit rows, odd numbers of tokens and heads; the rows are read back as prefill attention reads them.
        {"name": "append_rows8", "op": "append", "tokens": 8191, "heads": 5, "dim": 128, "block": 32, "type": "bf16", "store": "rows8", "group": 1},
        # The smallest attention call: one request, a short context.
        {"name": "attention_one", "op": "attention", "requests": 1, "heads": 32, "kv_heads": 8, "dim": 128, "shortest": 500, "longest": 500,
         "block": 16, "type": "bf16", "store": "same", "window": 0, "softcap": 0.0},
        # An ordinary step: 64 requests of 1 to 4 096 tokens, four queries to a key head.
        {"name": "attention_step", "op": "attention", "requests": 64, "heads": 32, "kv_heads": 8, "dim": 128, "shortest": 1, "longest": 4096,
         "block": 16, "type": "bf16", "store": "same", "window": 0, "softcap": 0.0},
        # As many key heads as queries, narrow heads, a window, softcap, an odd page, more requests than a wave has lanes.
        {"name": "attention_heads", "op": "attention", "requests": 131, "heads": 12, "kv_heads": 12, "dim": 64, "shortest": 1, "longest": 2049,
         "block": 24, "type": "fp16", "store": "same", "window": 1023, "softcap": 30.0},
        # One long document in a cache of 8-bit rows: all of the device on a single request's tokens.
        {"name": "attention_long", "op": "attention", "requests": 1, "heads": 64, "kv_heads": 8, "dim": 128, "shortest": 262_143, "longest": 262_143,
         "block": 64, "type": "bf16", "store": "rows8", "window": 0, "softcap": 0.0},
        # The largest: 256 requests of 16 to 8 192 tokens, eight queries to a key head.
        {"name": "attention_large", "op": "attention", "requests": 256, "heads": 64, "kv_heads": 8, "dim": 128, "shortest": 16, "longest": 8192,
         "block": 16, "type": "bf16", "store": "same", "window": 0, "softcap": 0.0},
        # A few rows of a small vocabulary.
        {"name": "logits_few", "op": "logits", "rows": 4, "vocab": 32_000, "history": 500, "biases": 16, "mask": False, "type": "fp32", "bits": 64},
        # A full step over a large, odd vocabulary: long histories, biases and a grammar mask, 16-bit logits.
        {"name": "logits_step", "op": "logits", "rows": 256, "vocab": 131_071, "history": 4096, "biases": 64, "mask": True, "type": "bf16", "bits": 32},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "logits"])
    if op == "tables":
        requests = _spread(rng, 1, 2048)
        return {"op": op, "requests": requests, "prefills": rng.choice([0, requests // 8, requests]) if requests < 256 else requests // 8,
                "chunk": _spread(rng, 1, 1023), "context": _spread(rng, 1, 8191), "block": rng.choice([1, 8, 16, 24, 64]), "bits": rng.choice([32, 64])}
    if op == "append":
        return {"op": op, "tokens": _spread(rng, 1, 16384), "heads": rng.randint(1, 8), "dim": rng.choice([64, 80, 96, 128]),
                "block": rng.choice([1, 8, 16, 24, 32, 64]), "type": rng.choice(["fp16", "bf16"]), "store": rng.choice(["same", "rows8"]),
                "group": rng.choice([1, 4])}
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
        dim = rng.choice([64, 80, 96, 128, 256])
        requests = _spread(rng, 1, 256)
        # no more rows than the largest listed case has: 1 M tokens of 8 heads of 128
        most = max(1, min(262_143, (1 << 30) // (requests * kv_heads * dim)))
        longest = _spread(rng, 1, most)
        return {"op": op, "requests": requests, "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16]), "kv_heads": kv_heads, "dim": dim,
                "shortest": _spread(rng, 1, longest), "longest": longest, "block": rng.choice([8, 16, 24, 32, 64, 128]),
                "type": rng.choice(["fp16", "bf16"]), "store": rng.choice(["same", "same", "rows8"]),
                "window": rng.choice([0, 0, 0, 1023]), "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    return {"op": op, "rows": _spread(rng, 1, 256), "vocab": _spread(rng, 1000, 131_071), "history": _spread(rng, 1, 4096), "biases": rng.choice([0, 16, 64]),
            "mask": rng.random() < 0.5, "type": rng.choice(["fp32", "bf16", "fp16"]), "bits": rng.choice([32, 64])}


def _evenly(count, low, high):
    return [low + (i * (high - low)) // max(1, count - 1) for i in range(count)] if count > 1 else [high]


def _dealt(values, g, dtype):
    """`values`, in an order of the generator's."""
    t = torch.tensor(values, dtype=dtype, device="cuda")
    return t[torch.randperm(len(values), generator=g, device="cuda")]


def _pages_of(lengths, block):
    return (lengths + block - 1) // block


def _rows8(shape, dim, g):
    """Rows of the 8-bit format: fp16 scale and bias, then the bytes; values of a few units either side of zero."""
    rows = torch.randint(0, 256, (*shape, dim + 4), dtype=torch.uint8, device="cuda", generator=g)
    scale = 4.0 / 255 * (0.5 + torch.rand((*shape, 1), device="cuda", generator=g))
    rows[..., :4] = torch.cat((scale, scale * -127.5), -1).half().view(torch.uint8)
    return rows


def _prepare_tables(case, g):
    R, S = case["requests"], case["block"]
    index = torch.int64 if case["bits"] == 64 else torch.int32
    held = _evenly(R, 0, case["context"])
    added = [1] * (R - case["prefills"]) + _evenly(case["prefills"], 1, case["chunk"]) if case["prefills"] else [1] * R
    lengths, new = _dealt(held, g, index), _dealt(added, g, index)
    width = -(-(case["context"] + max(added)) // S)
    old, need = _pages_of(lengths, S), _pages_of(lengths + new, S)
    pages = torch.randperm(int(need.sum()) + 64, generator=g, device="cuda", dtype=torch.int32)
    # the pages that are held, dealt row by row, in front of the free ones, which are given out from `start` on
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda") < old[:, None]
    tables[used] = pages[: int(old.sum())]
    start = old.sum().to(torch.int32).reshape(1)
    return {"lengths": lengths, "new": new, "tables": tables, "free": pages, "start": start, "tokens": sum(added)}


def _prepare_append(case, g):
    N, H, D, S, G = case["tokens"], case["heads"], case["dim"], case["block"], case["group"]
    pages = -(-N // S) + 4
    # the fused projection's output: query heads, key heads, value heads side by side
    fused = torch.randn((N, (G + 2) * H, D), device="cuda", generator=g).to(_TORCH[case["type"]])
    slots = torch.randperm(pages * S, generator=g, device="cuda")[:N]
    if case["store"] == "rows8":
        caches = [_rows8((pages, H, S), D, g) for _ in range(2)]
    else:
        caches = [torch.randn((pages, H, S, D), device="cuda", generator=g).to(_TORCH[case["type"]]) for _ in range(2)]
    return {"key": fused[:, G * H:(G + 1) * H], "value": fused[:, (G + 1) * H:], "key_cache": caches[0], "value_cache": caches[1], "slots": slots}


def _prepare_attention(case, g):
    B, H, D, S = case["requests"], case["kv_heads"], case["dim"], case["block"]
    held = _evenly(B, case["shortest"], case["longest"])
    lengths = _dealt(held, g, torch.int32)
    count, width = sum(-(-n // S) for n in held), -(-case["longest"] // S)
    pages = torch.randperm(count + 16, generator=g, device="cuda", dtype=torch.int32)
    tables = torch.zeros((B, width), dtype=torch.int32, device="cuda")
    tables[torch.arange(width, device="cuda") < _pages_of(lengths, S)[:, None]] = pages[:count]
    if case["store"] == "rows8":
        caches = [_rows8((count + 16, H, S), D, g) for _ in range(2)]
    else:
        caches = [torch.randn((count + 16, H, S, D), dtype=_TORCH[case["type"]], device="cuda", generator=g) for _ in range(2)]
    query = torch.randn((B, case["heads"], D), device="cuda", generator=g).to(_TORCH[case["type"]])
    return {"query": query, "key_cache": caches[0], "value_cache": caches[1], "tables": tables, "lengths": lengths,
            "window": case["window"], "softcap": case["softcap"], "scale": D ** -0.5}


def _prepare_logits(case, g):
    B, V = case["rows"], case["vocab"]
    index = torch.int64 if case["bits"] == 64 else torch.int32
    count = _dealt(_evenly(B, 0, case["history"]), g, torch.int64)
    total = sum(_evenly(B, 0, case["history"]))
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
    tokens = (V * uniform(total) ** 3).to(index).clamp_(max=V - 1)  # a few tokens come again and again
    offsets = torch.zeros(B + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = count.cumsum(0)
    state = {"logits": (4 * torch.randn((B, V), device="cuda", generator=g)).to(_TORCH[case["type"]]),
             "tokens": tokens, "offsets": offsets.to(index), "prompts": (count * uniform(B)).to(index),
             "repetition": 1 + 0.5 * uniform(B), "frequency": uniform(B), "presence": uniform(B),
             "bias_ids": None, "bias_values": None, "bias_offsets": None, "mask": None, "total": total}
    if case["biases"]:
        state["bias_ids"] = torch.randint(0, V, (B * case["biases"],), device="cuda", generator=g, dtype=index)
        state["bias_values"] = 4 * uniform(B * case["biases"]) - 2
        state["bias_offsets"] = torch.arange(B + 1, device="cuda", dtype=index) * case["biases"]
    if case["mask"]:  # a grammar leaves runs of tokens: whole words of the mask are clear, others have every bit set but some
        words = torch.randint(-(1 << 31), 1 << 31, (B, (V + 31) // 32), device="cuda", generator=g)
        state["mask"] = torch.where(uniform(*words.shape) < 0.5, words, torch.zeros_like(words)).to(torch.int32)
    return state


_PREPARE = {"tables": _prepare_tables, "append": _prepare_append, "attention": _prepare_attention, "logits": _prepare_logits}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, g)}


def _tables_plain(s, S):
    lengths, new, tables, free = s["lengths"], s["new"], s["tables"], s["free"]
    old, need = _pages_of(lengths, S), _pages_of(lengths + new, S)
    ends = (need - old).cumsum(0)
    first = s["start"] + ends - (need - old)
    column = torch.arange(tables.shape[1], device="cuda")
    fresh = (column >= old[:, None]) & (column < need[:, None])
    place = (first[:, None] + column - old[:, None]).clamp(0, len(free) - 1)
    tables.copy_(torch.where(fresh, free[place], tables))
    offsets = torch.zeros(len(new) + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = new.cumsum(0)
    token = torch.arange(s["tokens"], device="cuda")
    request = (torch.searchsorted(offsets, token, right=True) - 1)
    positions = lengths[request] + token - offsets[request]
    slots = tables[request, positions // S].long() * S + positions % S
    return {"tables": tables, "slots": slots, "positions": positions.long(), "offsets": offsets.int(), "lengths": lengths + new,
            "start": (s["start"] + ends[-1]).int()}


def _tables_own(s, S):
    from fbgemm_amd import decode
    t = decode.kv_block_tables(s["lengths"], s["new"], s["tables"], s["free"], s["start"], S, s["tokens"])
    return {"tables": s["tables"], "slots": t.slots, "positions": t.positions, "offsets": t.offsets, "lengths": t.lengths, "start": t.free_start}


def _half(x):
    return x.half().float()


def _append_plain(s, D):
    S = s["key_cache"].shape[2]
    page, place = s["slots"] // S, s["slots"] % S
    values = []
    for new, cache in ((s["key"], s["key_cache"]), (s["value"], s["value_cache"])):
        if cache.dtype != torch.uint8:
            cache[page, :, place] = new
            values.append(cache)
            continue
        x = new.float()
        low = _half(x.amin(-1, keepdim=True))
        span = x.amax(-1, keepdim=True) - low
        scale = _half(torch.where(span == 0, 1.0, span / 255))
        scale = torch.where((scale == 0) | torch.isinf(1 / scale), 1.0, scale)
        rows = torch.empty((*new.shape[:2], D + 4), dtype=torch.uint8, device="cuda")
        rows[..., :4] = torch.cat((scale, low), -1).half().view(torch.uint8)
        rows[..., 4:] = ((x - low) * (1 / scale)).round().clamp(0, 255).to(torch.uint8)
        cache[page, :, place] = rows
        pair = cache[..., :4].contiguous().view(torch.float16).float()
        values.append((cache[..., 4:].float() * pair[..., :1] + pair[..., 1:]).reshape(-1, D))
    return values


def _append_own(s, D):
    from fbgemm_amd import decode, ops
    decode.kv_cache_append(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"])
    if s["key_cache"].dtype != torch.uint8:
        return [s["key_cache"], s["value_cache"]]
    return [ops.dequantize_rowwise(c.view(-1, D + 4), D, 8, layout=ops.QLAYOUT_TBE) for c in (s["key_cache"], s["value_cache"])]


def _gathered(cache, tables, D, dtype):
    """A cache's rows in the order of the requests' tokens, [requests, heads, tokens, D]."""
    if cache.dtype == torch.uint8:
        pair = cache[..., :4].contiguous().view(torch.float16).to(dtype)[tables]
        rows = cache[..., 4:][tables].to(dtype) * pair[..., :1] + pair[..., 1:]
    else:
        rows = cache[tables]
    B, width, H, S, _ = rows.shape
    return rows.permute(0, 2, 1, 3, 4).reshape(B, H, width * S, D).to(dtype)


def _attention_in(s, dtype, query, tables, lengths):
    B, Hq, D = query.shape
    k, v = (_gathered(s[c], tables.long(), D, dtype) for c in ("key_cache", "value_cache"))
    H, L = k.shape[1:3]
    scores = torch.matmul(query.reshape(B, H, Hq // H, D).to(dtype), k.transpose(-1, -2)) * s["scale"]
    if s["softcap"]:
        scores = s["softcap"] * torch.tanh(scores / s["softcap"])
    token, length = torch.arange(L, device="cuda"), lengths[:, None, None, None]
    seen = token < length
    if s["window"]:
        seen = seen & (token >= length - s["window"])
    scores = torch.where(seen, scores, -math.inf)
    most = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(dtype).min)
    weights = torch.exp(scores - most)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v) / total.clamp(min=torch.finfo(dtype).tiny)
    return out.reshape(B, Hq, D), (most + torch.log(total)).reshape(B, Hq)


def _attention_plain(s):
    out, lse = _attention_in(s, torch.float32, s["query"], s["tables"], s["lengths"])
    return [out.to(s["query"].dtype), lse]


def _attention_own(s):
    from fbgemm_amd import decode
    out, lse = decode.paged_attention(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lengths"], scale=s["scale"],
                                      window=s["window"], softcap=s["softcap"])
    return [out, lse]


def _logits_in(s, dtype):
    B, V = s["logits"].shape
    x = s["logits"].to(dtype)
    offsets, tokens = s["offsets"].long(), s["tokens"].long()
    row = torch.repeat_interleave(torch.arange(B, device="cuda"), offsets[1:] - offsets[:-1], output_size=s["total"])
    said = (torch.arange(s["total"], device="cuda") - offsets[row] >= s["prompts"][row]).int()
    place = row * V + tokens
    count = torch.zeros(B * V, dtype=torch.int32, device="cuda").scatter_add_(0, place, said).view(B, V)
    seen = torch.zeros(B * V, dtype=torch.int32, device="cuda").scatter_add_(0, place, torch.ones_like(said)).view(B, V) > 0
    r, f, p = (s[k].to(dtype)[:, None] for k in ("repetition", "frequency", "presence"))
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count
    x = x - p * (count > 0)
    if s["bias_ids"] is not None:  # of several biases for one token the last one counts
        each = len(s["bias_ids"]) // B
        entry = torch.arange(B * each, device="cuda")
        last = torch.zeros(B * V, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(0, entry // each * V + s["bias_ids"].long(), entry + 1, "amax")
        x = x + torch.where(last > 0, s["bias_values"].to(dtype)[(last - 1).clamp(min=0)], 0.0).view(B, V)
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bits.reshape(B, -1)[:, :V] != 0, x, -math.inf)
    return x


def _logits_plain(s):
    return _logits_in(s, torch.float32).to(s["logits"].dtype)


def _logits_own(s):
    from fbgemm_amd import decode
    return decode.penalize_logits(s["logits"], s["tokens"], s["offsets"], s["prompts"], repetition=s["repetition"], frequency=s["frequency"],
                                  presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                                  bias_offsets=s["bias_offsets"], mask=s["mask"])


def run(state):
    case = state["case"]
    if case["op"] == "tables":
        return (_tables_own if own else _tables_plain)(state, case["block"])
    if case["op"] == "append":
        return (_append_own if own else _append_plain)(state, case["dim"])
    if case["op"] == "attention":
        return (_attention_own if own else _attention_plain)(state)
    return (_logits_own if own else _logits_plain)(state)


def work(case):
    if case["op"] == "tables":
        R, S, width = case["requests"], case["block"], case["bits"] // 8
        tokens = R - case["prefills"] + sum(_evenly(case["prefills"], 1, case["chunk"]) if case["prefills"] else [])
        # lengths in, lengths out, offsets; the page of each request's first token; pages out of the list into the tables; slots and positions
        return {"bytes": R * (3 * width + 4 + 4) + tokens / S * 8 + tokens * 16, "flops": 0}
    if case["op"] == "append":
        rows, D = case["tokens"] * case["heads"] * 2, case["dim"]
        if case["store"] == "same":
            return {"bytes": rows * D * 4 + case["tokens"] * 8, "flops": 0}
        cache = (-(-case["tokens"] // case["block"]) + 4) * case["block"] * case["heads"] * 2
        return {"bytes": rows * (D * 2 + D + 4) + cache * (D + 4 + D * 4) + case["tokens"] * 8, "flops": 0}
    if case["op"] == "attention":
        tokens = sum(min(n, case["window"] or n) for n in _evenly(case["requests"], case["shortest"], case["longest"]))
        row = case["dim"] + 4 if case["store"] == "rows8" else 2 * case["dim"]
        return {"bytes": tokens * case["kv_heads"] * 2 * row + case["requests"] * case["heads"] * (4 * case["dim"] + 4) + tokens / case["block"] * 4,
                "flops": 4.0 * tokens * case["heads"] * case["dim"]}
    B, V = case["rows"], case["vocab"]
    tokens = sum(_evenly(B, 0, case["history"]))
    return {"bytes": B * V * 2 * _SIZE[case["type"]] + (tokens + B * case["biases"]) * case["bits"] / 8 + B * case["biases"] * 4 + (B * V / 8 if case["mask"] else 0),
            "flops": 4.0 * B * V}


def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers alone
    s = prepare(case, seed)
    if case["op"] == "append":
        return _append_exact(s, case["dim"])
    if case["op"] == "attention":
        return _attention_exact(s)
    return _logits_exact(s)


def _append_exact(s, D):
    slots, S = s["slots"].tolist(), s["key_cache"].shape[2]
    values = []
    for new, cache in ((s["key"], s["key_cache"]), (s["value"], s["value_cache"])):
        x = new.double()
        if cache.dtype == torch.uint8:
            pair = cache[..., :4].contiguous().view(torch.float16).double()
            held = cache[..., 4:].double() * pair[..., :1] + pair[..., 1:]
            # the row's format: scale and bias are fp16 numbers
            low = x.amin(-1, keepdim=True).half().double()
            scale = ((x.amax(-1, keepdim=True) - low) / 255).half().double()
            x = torch.clamp(torch.round((x - low) / scale), 0, 255) * scale + low
        else:
            held = cache.double()
        rows = held.permute(0, 2, 1, 3).reshape(-1, *held.shape[1::2])  # by slot
        rows.index_copy_(0, torch.tensor(slots, device="cuda"), x)
        held = rows.reshape(held.shape[0], S, *held.shape[1::2]).permute(0, 2, 1, 3)
        values.append(held.reshape(-1, D) if cache.dtype == torch.uint8 else held)
    return values


def _attention_exact(s):
    outs, lses = [], []
    S, (_, Hq, D) = s["key_cache"].shape[2], s["query"].shape
    for b, length in enumerate(s["lengths"].tolist()):
        begin = max(0, length - s["window"]) if s["window"] else 0
        pages = s["tables"][b, : -(-length // S)].long()
        heads = []
        for h in range(s["key_cache"].shape[1]):
            rows = []
            for c in ("key_cache", "value_cache"):
                r = s[c][pages, h].reshape(-1, s[c].shape[-1])[begin:length]
                if r.dtype == torch.uint8:
                    pair = r[:, :4].contiguous().view(torch.float16).double()
                    r = r[:, 4:].double() * pair[:, :1] + pair[:, 1:]
                rows.append(r.double())
            group = Hq // s["key_cache"].shape[1]
            x = s["query"][b, h * group:(h + 1) * group].double() @ rows[0].t() * s["scale"]
            if s["softcap"]:
                x = s["softcap"] * torch.tanh(x / s["softcap"])
            heads.append((torch.softmax(x, -1) @ rows[1], torch.logsumexp(x, -1)))
        outs.append(torch.cat([o for o, _ in heads]))
        lses.append(torch.cat([l for _, l in heads]))
    return [torch.stack(outs), torch.stack(lses)]


def _logits_exact(s):
    rows = []
    V = s["logits"].shape[1]
    offsets, prompts = s["offsets"].tolist(), s["prompts"].tolist()
    for b in range(len(prompts)):
        x = s["logits"][b].double()
        tokens = s["tokens"][offsets[b]:offsets[b + 1]].long()
        count = torch.bincount(tokens[prompts[b]:], minlength=V).double()
        seen = torch.bincount(tokens, minlength=V) > 0
        r = s["repetition"][b].double()
        x = torch.where(seen & (x > 0), x / r, torch.where(seen, x * r, x))
        x = x - s["frequency"][b].double() * count - s["presence"][b].double() * (count > 0)
        if s["bias_ids"] is not None:
            lo, hi = s["bias_offsets"][b:b + 2].tolist()
            last = dict(zip(s["bias_ids"][lo:hi].tolist(), s["bias_values"][lo:hi].double().tolist()))
            x[torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if s["mask"] is not None:
            place = torch.arange(V, device="cuda")
            x[(s["mask"][b][place // 32] >> (place % 32)) & 1 == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)
