"""What the operators that complete a decoding step are measured on: rotary positions, a cache in 4 bits, sampling.

A case is a dict of plain values. Its "op" names the operator a pass goes through:

* ``rotary``: ``decode.rotate_positions``: queries and keys of a fused projection's output, turned by their positions;
* ``append``: ``decode.kv_cache_append`` into a cache of 4-bit rows (``row_bits=4``); the pass then reads the cache back as the
  values it stands for, with ``ops.dequantize_rowwise``;
* ``read``: ``decode.kv_cache_read``: the tokens of every request out of its pages into dense rows, as attention over a prompt's
  later part takes them; 4-bit, 8-bit or 16-bit rows;
* ``attention``: ``decode.paged_attention`` over 4-bit rows: one new token of every request over its pages;
* ``sample``: ``decode.sample_tokens``: a token of every row of logits by temperature, top-k, top-p, min-p and a given random
  number, and the logarithm of its probability.

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
        # One step of a server with 64 requests in flight: their new queries and keys.
        {"name": "rotary_step", "op": "rotary", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False,
         "type": "bf16", "farthest": 4096, "factor": 1.0},
        # Prompts, 4 095 tokens of them, of a model that turns part of its heads of 80, neighbours together, in fp32.
        {"name": "rotary_part", "op": "rotary", "tokens": 4095, "heads": 12, "kv_heads": 12, "dim": 80, "turned": 32, "interleaved": True,
         "type": "fp32", "farthest": 8191, "factor": 1.0},
        # Long documents, far positions, frequencies scaled for them.
        {"name": "rotary_prompts", "op": "rotary", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False,
         "type": "bf16", "farthest": 262_143, "factor": 8.0},
        # The rows of one decoding step, cut out of the fused projection's output.
        {"name": "append4_step", "op": "append", "tokens": 64, "heads": 8, "dim": 128, "block": 16, "type": "bf16", "group": 4},
        # Prompts, odd numbers of tokens and heads.
        {"name": "append4_prompts", "op": "append", "tokens": 8191, "heads": 5, "dim": 128, "block": 32, "type": "fp16", "group": 1},
        # A short prefix that a few requests share their beginning with, out of 16-bit rows and pages of an odd size.
        {"name": "read_short", "op": "read", "requests": 4, "kv_heads": 8, "dim": 128, "shortest": 33, "longest": 200, "block": 24, "type": "bf16", "store": "same"},
        # The earlier chunks of 32 prompts, out of 4-bit rows.
        {"name": "read_prefix", "op": "read", "requests": 32, "kv_heads": 8, "dim": 128, "shortest": 1, "longest": 4096, "block": 16, "type": "bf16", "store": "rows4"},
        # The smallest attention call: one request, a short context.
        {"name": "attention4_one", "op": "attention", "requests": 1, "heads": 32, "kv_heads": 8, "dim": 128, "shortest": 500, "longest": 500,
         "block": 16, "type": "bf16", "window": 0, "softcap": 0.0},
        # An ordinary step, fp16 and pages of 64: 64 requests of 1 to 4 096 tokens, eight queries to a key head.
        {"name": "attention4_step", "op": "attention", "requests": 64, "heads": 64, "kv_heads": 8, "dim": 128, "shortest": 1, "longest": 4096,
         "block": 64, "type": "fp16", "window": 0, "softcap": 0.0},
        # The largest: 256 requests of 16 to 8 192 tokens, which 4 bits are there for.
        {"name": "attention4_large", "op": "attention", "requests": 256, "heads": 64, "kv_heads": 8, "dim": 128, "shortest": 16, "longest": 8192,
         "block": 16, "type": "bf16", "window": 0, "softcap": 0.0},
        # A few rows of a small vocabulary, each with a top-k and a top-p.
        {"name": "sample_few", "op": "sample", "rows": 4, "vocab": 32_000, "type": "fp32", "filters": "both", "masked": False},
        # A full step over a large, odd vocabulary behind a grammar's mask: every request has filters of its own, or none.
        {"name": "sample_step", "op": "sample", "rows": 256, "vocab": 131_071, "type": "bf16", "filters": "mixed", "masked": True},
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "read", "attention", "attention", "sample", "sample"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        most = max(1, 16384 * 40 * 128 // ((heads + kv_heads) * dim) // 2)
        return {"op": op, "tokens": _spread(rng, 1, min(16384, most)), "heads": heads, "kv_heads": kv_heads, "dim": dim, "turned": rng.choice([dim, dim // 2, 32]),
                "interleaved": rng.random() < 0.5, "type": rng.choice(["fp32", "fp16", "bf16"]), "farthest": _spread(rng, 1000, 262_143),
                "factor": rng.choice([1.0, 1.0, 8.0])}
    if op == "append":
        return {"op": op, "tokens": _spread(rng, 1, 8191), "heads": rng.randint(1, 8), "dim": rng.choice([64, 80, 96, 128]),
                "block": rng.choice([1, 8, 16, 24, 32, 64]), "type": rng.choice(["fp16", "bf16"]), "group": rng.choice([1, 4])}
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
    dim = rng.choice([64, 80, 96, 128, 256])
    block = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "read":
        requests = _spread(rng, 1, 32)
        longest = _spread(rng, 1, max(1, min(4096, (1 << 26) // (requests * kv_heads * dim))))
        return {"op": op, "requests": requests, "kv_heads": kv_heads, "dim": dim, "shortest": _spread(rng, 1, longest), "longest": longest, "block": block,
                "type": rng.choice(["fp16", "bf16"]), "store": rng.choice(["rows4", "rows8", "same"])}
    if op == "attention":
        requests = _spread(rng, 1, 256)
        # no more rows than the largest listed case has: 1 M tokens of 8 heads of 128
        longest = _spread(rng, 1, max(1, min(262_143, (1 << 30) // (requests * kv_heads * dim))))
        return {"op": op, "requests": requests, "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 16]), "kv_heads": kv_heads, "dim": dim,
                "shortest": _spread(rng, 1, longest), "longest": longest, "block": block, "type": rng.choice(["fp16", "bf16"]),
                "window": rng.choice([0, 0, 0, 1023]), "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    return {"op": op, "rows": _spread(rng, 1, 256), "vocab": _spread(rng, 1000, 131_071), "type": rng.choice(["fp32", "bf16", "fp16"]),
            "filters": rng.choice(["none", "top_k", "top_p", "min_p", "both", "mixed"]), "masked": rng.random() < 0.5}


def _evenly(count, low, high):
    return [low + (i * (high - low)) // max(1, count - 1) for i in range(count)] if count > 1 else [high]


def _dealt(values, g, dtype):
    """`values`, in an order of the generator's."""
    t = torch.tensor(values, dtype=dtype, device="cuda")
    return t[torch.randperm(len(values), generator=g, device="cuda")]


def _rows(shape, dim, bits, g):
    """Rows of the 8-bit or 4-bit format: fp16 scale and bias, then the codes; values of a few units either side of zero."""
    rows = torch.randint(0, 256, (*shape, dim * bits // 8 + 4), dtype=torch.uint8, device="cuda", generator=g)
    scale = 4.0 / (2 ** bits - 1) * (0.5 + torch.rand((*shape, 1), device="cuda", generator=g))
    rows[..., :4] = torch.cat((scale, scale * -(2 ** bits - 1) / 2), -1).half().view(torch.uint8)
    return rows


def _frequencies(dim, factor):
    """Radians a position, fp64: base 10 000; with a factor, waves longer than 8 192 positions are stretched by it, those shorter than
    2 048 are left alone, and what is between is a mixture."""
    f = 10_000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if factor != 1.0:
        kept = ((8192 * f / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
        f = f * (kept + (1 - kept) / factor)
    return f.cuda()


def _prepare_rotary(case, g):
    N, Hq, H, D = (case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
    fused = torch.randn((N, Hq + 2 * H, D), device="cuda", generator=g).to(_TORCH[case["type"]])
    return {"query": fused[:, :Hq], "key": fused[:, Hq:Hq + H], "frequencies": _frequencies(case["turned"], case["factor"]),
            "positions": torch.randint(0, case["farthest"] + 1, (N,), device="cuda", generator=g),
            "magnitude": 1.0 if case["factor"] == 1.0 else 1.0 + 0.1 * math.log(case["factor"])}


def _prepare_append(case, g):
    N, H, D, S, G = (case[k] for k in ("tokens", "heads", "dim", "block", "group"))
    pages = -(-N // S) + 4
    # the fused projection's output: query heads, key heads, value heads side by side
    fused = torch.randn((N, (G + 2) * H, D), device="cuda", generator=g).to(_TORCH[case["type"]])
    slots = torch.randperm(pages * S, generator=g, device="cuda")[:N]
    caches = [_rows((pages, H, S), D, 4, g) for _ in range(2)]
    return {"key": fused[:, G * H:(G + 1) * H], "value": fused[:, (G + 1) * H:], "key_cache": caches[0], "value_cache": caches[1], "slots": slots}


def _prepare_pages(case, g):
    B, H, D, S = (case[k] for k in ("requests", "kv_heads", "dim", "block"))
    held = _evenly(B, case["shortest"], case["longest"])
    lengths = _dealt(held, g, torch.int32)
    count, width = sum(-(-n // S) for n in held), -(-case["longest"] // S)
    pages = torch.randperm(count + 16, generator=g, device="cuda", dtype=torch.int32)
    tables = torch.zeros((B, width), dtype=torch.int32, device="cuda")
    tables[torch.arange(width, device="cuda") < ((lengths + S - 1) // S)[:, None]] = pages[:count]
    shape, store = (count + 16, H, S), case.get("store", "rows4")
    if store == "same":
        caches = [torch.randn((*shape, D), dtype=_TORCH[case["type"]], device="cuda", generator=g) for _ in range(2)]
    else:
        caches = [_rows(shape, D, int(store[4:]), g) for _ in range(2)]
    return {"key_cache": caches[0], "value_cache": caches[1], "tables": tables, "lengths": lengths, "total": sum(held), "store": store}


def _prepare_read(case, g):
    s = _prepare_pages(case, g)
    s["offsets"] = torch.zeros(case["requests"] + 1, dtype=torch.int32, device="cuda")
    s["offsets"][1:] = s["lengths"].cumsum(0)
    return s


def _prepare_attention(case, g):
    s = _prepare_pages(case, g)
    s["query"] = torch.randn((case["requests"], case["heads"], case["dim"]), device="cuda", generator=g).to(_TORCH[case["type"]])
    s["scale"] = case["dim"] ** -0.5
    return s


def _prepare_sample(case, g):
    B, V, filters = case["rows"], case["vocab"], case["filters"]
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
    logits = 3 * torch.randn((B, V), device="cuda", generator=g)
    if case["masked"]:  # a grammar leaves half of every other row's tokens
        gone = uniform(B, V) < 0.5
        gone[::2] = False
        logits.masked_fill_(gone, -math.inf)
    s = {"logits": logits.to(_TORCH[case["type"]]), "uniform": uniform(B), "temperature": 0.5 + uniform(B), "top_k": None, "top_p": None, "min_p": None}
    if filters in ("top_k", "both", "mixed"):
        s["top_k"] = torch.exp(uniform(B) * math.log(200)).int()  # 1 to 200, small ones as often as large ones
    if filters in ("top_p", "both", "mixed"):
        s["top_p"] = 0.5 + 0.5 * uniform(B)
    if filters in ("min_p", "mixed"):
        s["min_p"] = 0.1 * uniform(B)
    if filters == "mixed":  # a third of the requests has each filter, and some want the most likely token
        for name, none in (("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
            s[name][uniform(B) < 0.67] = none
        s["temperature"][uniform(B) < 0.1] = 0.0
    return s


_PREPARE = {"rotary": _prepare_rotary, "append": _prepare_append, "read": _prepare_read, "attention": _prepare_attention, "sample": _prepare_sample}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, g)}


def _rotary_plain(s, interleaved):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    R = 2 * angle.shape[1]
    results = []
    for x in (s["query"], s["key"]):
        y = x.float()
        a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
        pair = (a * cos - b * sin, b * cos + a * sin)
        turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
        results.append(torch.cat((turned.to(x.dtype), x[..., R:]), -1))
    return results


def _rotary_own(s, interleaved):
    from fbgemm_amd import decode
    return list(decode.rotate_positions(s["query"], s["key"], s["positions"], s["frequencies"], interleaved=interleaved, magnitude=s["magnitude"]))


def _values(rows, bits):
    """What rows of the format stand for, in fp32."""
    pair = rows[..., :4].contiguous().view(torch.float16).float()
    codes = rows[..., 4:]
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return codes.float() * pair[..., :1] + pair[..., 1:]


def _half(x):
    return x.half().float()


def _append_plain(s):
    S = s["key_cache"].shape[2]
    page, place = s["slots"] // S, s["slots"] % S
    values = []
    for new, cache in ((s["key"], s["key_cache"]), (s["value"], s["value_cache"])):
        x = new.float()
        low = _half(x.amin(-1, keepdim=True))
        span = x.amax(-1, keepdim=True) - low
        scale = _half(torch.where(span == 0, 1.0, span / 15))
        scale = torch.where((scale == 0) | torch.isinf(1 / scale), 1.0, scale)
        codes = ((x - low) * (1 / scale)).round().clamp(0, 15).to(torch.uint8)
        rows = torch.empty((*new.shape[:2], new.shape[2] // 2 + 4), dtype=torch.uint8, device="cuda")
        rows[..., :4] = torch.cat((scale, low), -1).half().view(torch.uint8)
        rows[..., 4:] = codes[..., ::2] | codes[..., 1::2] << 4
        cache[page, :, place] = rows
        values.append(_values(cache, 4).reshape(-1, new.shape[2]))
    return values


def _append_own(s):
    from fbgemm_amd import decode, ops
    decode.kv_cache_append(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], row_bits=4)
    D = s["key"].shape[2]
    return [ops.dequantize_rowwise(c.view(-1, D // 2 + 4), D, 4, layout=ops.QLAYOUT_TBE) for c in (s["key_cache"], s["value_cache"])]


def _read_plain(s, dtype):
    S, offsets = s["key_cache"].shape[2], s["offsets"].long()
    token = torch.arange(s["total"], device="cuda")
    request = torch.searchsorted(offsets, token, right=True) - 1
    position = token - offsets[request]
    page, place = s["tables"][request, position // S].long(), position % S
    rows = [c[page, :, place] for c in (s["key_cache"], s["value_cache"])]
    return rows if s["store"] == "same" else [_values(r, int(s["store"][4:])).to(dtype) for r in rows]


def _read_own(s, dtype, dim):
    from fbgemm_amd import decode
    return list(decode.kv_cache_read(s["key_cache"], s["value_cache"], s["tables"], s["offsets"], s["total"], dim, dtype,
                                     row_bits=4 if s["store"] == "rows4" else 8))


def _gathered(cache, tables, D):
    """A cache's rows in the order of the requests' tokens, [requests, heads, tokens, D]."""
    rows = cache[tables.long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
    return _values(rows, 4)


def _attention_plain(s):
    case = s["case"]
    B, Hq, H, D, S = (case[k] for k in ("requests", "heads", "kv_heads", "dim", "block"))
    width = s["tables"].shape[1] * S
    group = max(1, (1 << 28) // (H * width * D))  # requests at a time: 1 GiB of fp32 rows
    outs, lses = [], []
    for b in range(0, B, group):
        tables, lengths = s["tables"][b:b + group], s["lengths"][b:b + group]
        q = s["query"][b:b + group].float().view(len(lengths), H, Hq // H, D)
        k, v = (_gathered(s[c], tables, D) for c in ("key_cache", "value_cache"))
        x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        t = torch.arange(width, device="cuda")
        seen = t < lengths[:, None]
        if case["window"]:
            seen &= t >= (lengths - case["window"])[:, None]
        x = x.masked_fill(~seen[:, None, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - m)
        total = p.sum(-1, keepdim=True)
        outs.append((torch.matmul(p, v) / total).view(-1, Hq, D).to(s["query"].dtype))
        lses.append((m + torch.log(total)).view(-1, Hq))
    return [torch.cat(outs), torch.cat(lses)]


def _attention_own(s):
    from fbgemm_amd import decode
    return list(decode.paged_attention(s["query"], s["key_cache"], s["value_cache"], s["tables"], s["lengths"], scale=s["scale"],
                                       window=s["case"]["window"], softcap=s["case"]["softcap"], row_bits=4))


def _sample_plain(s):
    """In 64 bits: the number drawn may lie next to the border of two tokens, of which a large vocabulary has many."""
    B, V = s["logits"].shape
    one = torch.ones(B, device="cuda", dtype=torch.float64)
    t = s["temperature"].double()
    greedy = ~(t > 0)
    t = torch.where(greedy, one, t)[:, None]
    x, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)  # equal ones: the lower token first
    w = torch.exp((x - x[:, :1]) / t)
    rank = torch.arange(V, device="cuda")
    keep = (rank == 0) | ~greedy[:, None]
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], V)
        keep &= rank < k[:, None]
    w = torch.where(keep, w, 0.0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        ends = w.cumsum(-1)
        w = torch.where((ends - w < p * ends[:, -1:]) | (p >= 1) | (rank == 0), w, 0.0)
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # in the tokens' order
    ends = w.cumsum(-1)
    total = ends[:, -1]
    token = (ends <= (s["uniform"].double() * total)[:, None]).sum(-1)
    return [token, torch.log(w.gather(1, token[:, None])[:, 0] / total).float()]


def _sample_own(s):
    from fbgemm_amd import decode
    return list(decode.sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"]))


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return (_rotary_own if own else _rotary_plain)(state, case["interleaved"])
    if case["op"] == "append":
        return (_append_own if own else _append_plain)(state)
    if case["op"] == "read":
        dtype = _TORCH[case["type"]]
        return _read_own(state, dtype, case["dim"]) if own else _read_plain(state, dtype)
    if case["op"] == "attention":
        return (_attention_own if own else _attention_plain)(state)
    return (_sample_own if own else _sample_plain)(state)


def work(case):
    if case["op"] == "rotary":
        heads = case["tokens"] * (case["heads"] + case["kv_heads"])
        # a product pair for each of a turned pair's two numbers; a sine and a cosine for each token's pairs
        return {"bytes": heads * case["dim"] * 2 * _SIZE[case["type"]] + case["tokens"] * 8 + case["turned"] * 4, "flops": 3.0 * heads * case["turned"]}
    if case["op"] == "append":
        D = case["dim"]
        rows = case["tokens"] * case["heads"] * 2
        cache = (-(-case["tokens"] // case["block"]) + 4) * case["block"] * case["heads"] * 2
        return {"bytes": rows * (D * 2 + D / 2 + 4) + cache * (D / 2 + 4 + D * 4) + case["tokens"] * 8, "flops": 0}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * _SIZE[case["type"]] + 5 * 4 + 12), "flops": 4.0 * case["rows"] * case["vocab"]}
    lengths, D = _evenly(case["requests"], case["shortest"], case["longest"]), case["dim"]
    row = {"rows4": D / 2 + 4, "rows8": D + 4, "same": 2 * D}[case.get("store", "rows4")]
    if case["op"] == "read":
        tokens = sum(lengths)
        return {"bytes": tokens * case["kv_heads"] * 2 * (row + 2 * D) + tokens / case["block"] * 4, "flops": 0}
    tokens = sum(min(n, case["window"] or n) for n in lengths)
    return {"bytes": tokens * case["kv_heads"] * 2 * row + case["requests"] * case["heads"] * (4 * D + 4) + tokens / case["block"] * 4,
            "flops": 4.0 * tokens * case["heads"] * D}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _rotary_exact, "append": _append_exact, "read": _read_exact, "attention": _attention_exact, "sample": _sample_exact}[case["op"]](s)


def _rotary_exact(s):
    # a pair as a complex number
    turn = torch.polar(torch.full((len(s["positions"]), len(s["frequencies"])), s["magnitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["frequencies"]))
    half, results = turn.shape[1], []
    for x in (s["query"], s["key"]):
        y = x.double().clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["case"]["interleaved"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        results.append(y)
    return results


def _unpacked(rows, bits):
    dim = (rows.shape[-1] - 4) * 8 // bits
    place = torch.arange(dim, device="cuda") * bits
    codes = (rows[..., 4 + place // 8].int() >> (place % 8)) & (2 ** bits - 1)
    scale, bias = (rows[..., k:k + 2].contiguous().view(torch.float16).double() for k in (0, 2))
    return scale * codes.double() + bias


def _append_exact(s):
    slots, (pages, H, S, _), D = s["slots"], s["key_cache"].shape, s["key"].shape[2]
    values = []
    for new, cache in ((s["key"], s["key_cache"]), (s["value"], s["value_cache"])):
        x = new.double()
        # the row's format: scale and bias are fp16 numbers, and a code is the nearest whole number to an fp32 product with an fp32
        # reciprocal: 16-bit elements often lie halfway between two codes, where nothing else would say which one it is
        low = x.amin(-1, keepdim=True).half().double()
        scale = ((x.amax(-1, keepdim=True) - low) / 15).half().double()
        rows = _unpacked(cache, 4).permute(0, 2, 1, 3).reshape(-1, H, D)  # by slot
        steps = ((x - low).float().double() * (1 / scale).float().double()).float().double()
        rows[slots] = torch.clamp(torch.round(steps), 0, 15) * scale + low
        values.append(rows.view(pages, S, H, D).permute(0, 2, 1, 3).reshape(-1, D))
    return values


def _requests_rows(s, name, b, length):
    """One request's rows in 64 bits, [tokens, heads, dim]."""
    cache = s[name]
    pages = s["tables"][b, : -(-length // cache.shape[2])].long()
    rows = cache[pages].transpose(1, 2).flatten(0, 1)[:length]
    return rows.double() if s["store"] == "same" else _unpacked(rows, int(s["store"][4:]))


def _read_exact(s):
    return [torch.cat([_requests_rows(s, name, b, n) for b, n in enumerate(s["lengths"].tolist())]) for name in ("key_cache", "value_cache")]


def _attention_exact(s):
    case, outs, lses = s["case"], [], []
    for b, length in enumerate(s["lengths"].tolist()):
        begin = max(0, length - case["window"]) if case["window"] else 0
        group, heads = case["heads"] // case["kv_heads"], []
        k, v = (_requests_rows(s, name, b, length)[begin:] for name in ("key_cache", "value_cache"))
        for h in range(case["kv_heads"]):
            x = s["query"][b, h * group:(h + 1) * group].double() @ k[:, h].t() * s["scale"]
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            heads.append((torch.softmax(x, -1) @ v[:, h], torch.logsumexp(x, -1)))
        outs.append(torch.cat([o for o, _ in heads]))
        lses.append(torch.cat([l for _, l in heads]))
    return [torch.stack(outs), torch.stack(lses)]


def _sample_exact(s):
    """Row by row, the kept tokens as a list; tokens are whole numbers and have no value in 64 bits."""
    values = []
    for b in range(len(s["uniform"])):
        t, x = float(s["temperature"][b]), s["logits"][b].double()
        if not t > 0:
            values.append(0.0)
            continue
        x = x / t
        ids = torch.arange(len(x), device="cuda")
        if s["top_k"] is not None and 0 < int(s["top_k"][b]) < len(x):
            k = int(s["top_k"][b])
            border = torch.topk(x, k).values[-1]
            above = ids[x > border]
            ids = torch.cat((above, ids[x == border][: k - len(above)])).sort().values
        log_p = torch.log_softmax(x[ids], 0)
        if s["top_p"] is not None and float(s["top_p"][b]) < 1:
            by = torch.argsort(log_p, descending=True, stable=True)
            before = torch.cat((torch.zeros(1, device="cuda", dtype=torch.float64), log_p[by].exp().cumsum(0)[:-1]))
            left = by[: max(1, int((before < float(s["top_p"][b])).sum()))].sort().values
            ids, log_p = ids[left], log_p[left]
        if s["min_p"] is not None and float(s["min_p"][b]) > 0:
            log_p = log_p.masked_fill(log_p - log_p.max() < math.log(float(s["min_p"][b])), -math.inf)
        log_p = log_p - torch.logsumexp(log_p, 0)
        place = int((log_p.exp().cumsum(0) <= float(s["uniform"][b])).sum())
        values.append(float(log_p[min(place, len(log_p) - 1)]))
    return [None, torch.tensor(values, dtype=torch.float64, device="cuda")]
