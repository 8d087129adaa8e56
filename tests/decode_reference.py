"""The operators of a decoding step written out in numpy, in 64 bits, one request or row at a time."""
import numpy as np


def block_tables(lengths, new_tokens, tables, free, start, block, num_tokens):
    """(tables, slots, positions, offsets, total lengths, next start, status bits)"""
    tables, width, bits = tables.copy(), tables.shape[1], 0
    slots, positions = np.full(num_tokens, -1, np.int64), np.zeros(num_tokens, np.int64)
    offsets, n, place = [], 0, int(start)
    total = np.maximum(lengths, 0) + np.maximum(new_tokens, 0)
    for r, (held, added) in enumerate(zip(lengths.tolist(), new_tokens.tolist())):
        bits |= 8 if held < 0 or added < 0 else 0
        held, added = max(held, 0), max(added, 0)
        bits |= 2 if held + added > width * block else 0
        room = width * block
        old, need = -(-min(held, room) // block), -(-min(held + added, room) // block)
        for j in range(old, need):
            bits |= 16 if not 0 <= place < len(free) else 0
            tables[r, j] = free[place] if 0 <= place < len(free) else -1
            place += 1
        offsets.append(min(n, num_tokens))
        for k in range(added):
            if n < num_tokens:
                p = min(held, room) + k
                positions[n] = p
                if p < room and tables[r, p // block] >= 0:
                    slots[n] = int(tables[r, p // block]) * block + p % block
            n += 1
    offsets.append(min(n, num_tokens))
    bits |= 4 if n != num_tokens else 0
    return tables, slots, positions, np.array(offsets, np.int32), total, place, bits


def rows8_values(rows, dim):
    """What 8-bit rows stand for."""
    pair = np.ascontiguousarray(rows[..., :4]).view(np.float16).astype(np.float64)
    return rows[..., 4:4 + dim].astype(np.float64) * pair[..., :1] + pair[..., 1:]


def attention(query, key_cache, value_cache, tables, lengths, scale, window=0, softcap=0.0):
    """(out, lse, bound of out's error, bound of lse's error) of float64 queries [B, Hq, D] and caches [blocks, H, S, D].

    The bounds are those of fp32 scores and sums and of weights cut to 16 bits (2^-17 each), before the last rounding: a
    score is off by at most (D + 8) 2^-24 of the sum of its terms' sizes, a weight relatively by the errors of its score
    and of the maximum, of exp2 (2^-22) and of the cut; the sums' own roundings are within the same 2^-16."""
    B, Hq, D = query.shape
    blocks, H, S, _ = key_cache.shape
    out, lse = np.zeros((B, Hq, D)), np.full((B, Hq), -np.inf)
    out_off, lse_off = np.zeros((B, Hq, D)), np.zeros((B, Hq))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), tables.shape[1] * S)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = tables[b, t // S]
        t, page = t[(page >= 0) & (page < blocks)], page[(page >= 0) & (page < blocks)]
        if not len(t):
            continue
        for h in range(Hq):
            k, v, q = key_cache[page, h // (Hq // H), t % S], value_cache[page, h // (Hq // H), t % S], query[b, h]
            s = scale * (k @ q)
            wrong = (D + 8) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q)) + 2.0 ** -22 * np.abs(s)
            if softcap:
                s, wrong = softcap * np.tanh(s / softcap), wrong + 2.0 ** -21 * softcap
            m = s.max()
            p = np.exp(s - m)
            total = p.sum()
            out[b, h], lse[b, h] = p @ v / total, m + np.log(total)
            off = 2 * wrong.max() + 2.0 ** -15
            out_off[b, h] = off * (p @ np.abs(v)) / total
            lse_off[b, h] = wrong.max() + 2.0 ** -20 * (1 + abs(lse[b, h]))
    return out, lse, out_off, lse_off


def logits(x, tokens, offsets, prompts, repetition, frequency, presence, bias_ids, bias_values, bias_offsets, mask):
    """(result, bound of an fp32 result's error: 8 roundings of the largest number on the way)"""
    x = x.astype(np.float64)
    size = np.abs(np.where(np.isfinite(x), x, 0))
    rows, vocab = x.shape
    for r in range(rows):
        if tokens is not None:
            begin, end = max(0, offsets[r]), min(len(tokens), offsets[r + 1])
            seen, count = np.zeros(vocab, bool), np.zeros(vocab)
            for i in range(begin, end):
                if 0 <= tokens[i] < vocab:
                    seen[tokens[i]] = True
                    count[tokens[i]] += i - begin >= (0 if prompts is None else prompts[r])
            rep = 1.0 if repetition is None else repetition[r]
            x[r] = np.where(seen, np.where(x[r] > 0, x[r] / rep, x[r] * rep), x[r])
            size[r] = np.maximum(size[r], np.abs(np.where(np.isfinite(x[r]), x[r], 0)))
            lost = (0.0 if frequency is None else frequency[r]) * count + (0.0 if presence is None else presence[r]) * (count > 0)
            x[r] -= lost
            size[r] += np.abs(lost)
        if bias_ids is not None:
            last = {}
            for i in range(bias_offsets[r], bias_offsets[r + 1]):
                if 0 <= bias_ids[i] < vocab:
                    last[int(bias_ids[i])] = bias_values[i]
            for v, b in last.items():
                x[r, v] += b
                size[r, v] += abs(b) if np.isfinite(b) else 0
        if mask is not None:
            for v in range(vocab):
                if not (int(mask[r, v // 32]) >> (v % 32)) & 1:
                    x[r, v] = -np.inf
    return x, 8 * 2.0 ** -24 * size
