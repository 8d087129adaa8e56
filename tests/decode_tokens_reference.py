"""Rotary positions, 4-bit cache rows, their reading back and sampling written out in numpy, in 64 bits."""
import numpy as np


def rows4_values(rows, dim):
    """What 4-bit rows stand for."""
    pair = np.ascontiguousarray(rows[..., :4]).view(np.float16).astype(np.float64)
    return codes4(rows, dim) * pair[..., :1] + pair[..., 1:]


def codes4(rows, dim):
    data = rows[..., 4:4 + dim // 2]
    return np.stack((data & 15, data >> 4), -1).reshape(*data.shape[:-1], dim).astype(np.float64)


def rotate(x, positions, frequencies, interleaved=False, magnitude=1.0, inverse=False):
    """(result, bound of an fp32 result's error before the last rounding) of float64 x [tokens, heads, dim].

    Sines and cosines are off by at most 4 roundings of 2^-24 (the angle's rest, its product with pi / 2, the series, the magnitude), and by
    the angle's own error, some 2^-51 of it; products and their sum add two more."""
    n = len(frequencies)
    angle = positions.astype(np.float64)[:, None, None] * np.asarray(frequencies)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if inverse else 1)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    off = (6 * 2.0 ** -24 + 2.0 ** -51 * np.abs(angle)) * abs(magnitude) * (np.abs(a) + np.abs(b))
    out, wrong = x.copy(), np.zeros_like(x)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    wrong[..., first] = wrong[..., second] = off
    return out, wrong


def read(cache, tables, offsets, starts, num_tokens):
    """(rows [tokens, heads, row], numbers of tokens that have no page) of a cache [blocks, heads, block, row]."""
    blocks, heads, S, row = cache.shape
    out, bad = np.zeros((num_tokens, heads, row), cache.dtype), []
    for r in range(len(offsets) - 1):
        for i in range(int(offsets[r]), int(offsets[r + 1])):
            p = (0 if starts is None else int(starts[r])) + i - int(offsets[r])
            page = int(tables[r, p // S]) if 0 <= p < tables.shape[1] * S else -1
            if i >= num_tokens:
                continue
            if 0 <= page < blocks:
                out[i] = cache[page, :, p % S]
            else:
                bad.append(i)
    return out, bad


class Sampled:
    """What may be drawn of one row: the kept tokens with their running sums, in 64 bits.

    Kernels add whole numbers of 2^-fraction of the largest: a running sum over V tokens is off by V / 2 such units, and as much of the
    exponentials' 2^-52."""

    def __init__(self, x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
        vocab = len(x)
        self.slack = vocab * 2.0 ** -min(50, 62 - vocab.bit_length())
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        self.empty = len(order) == 0
        if self.empty:
            return
        if not temperature > 0 or not top_p > 0:
            order = order[:1]
        w = np.exp((x[order] - x[order[0]]) / (temperature if temperature > 0 else 1.0))
        if 0 < top_k < len(order):
            order, w = order[:top_k], w[:top_k]
        self.sure = len(order)  # tokens that are kept whatever the roundings; those behind may be
        if 0 < top_p < 1:
            before = np.cumsum(w) - w
            goal = np.float64(top_p) * w.sum()
            self.sure = max(1, int((before < goal - self.slack).sum()))
            most = max(1, int((before < goal + self.slack).sum()))
            order, w = order[:most], w[:most]
        kept = w >= min(min_p, 1.0)
        order, w, self.sure = order[kept], w[kept], min(self.sure, int(kept.sum()))
        self.order, self.w = order, w

    def holds(self, token, u, log_probability):
        """Whether `token` is what `u` draws, and `log_probability` its logarithm, for one of the sets that roundings allow."""
        if self.empty:
            return token == -1 and log_probability == -np.inf
        u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
        for n in range(self.sure, len(self.order) + 1):
            by = np.argsort(self.order[:n])
            tokens, w = self.order[:n][by], self.w[:n][by]
            ends, total = np.cumsum(w), w.sum()
            place = np.flatnonzero(tokens == token)
            if not len(place):
                continue
            i = place[0]
            last = np.flatnonzero(w > 0)[-1]
            inside = ends[i] - w[i] - self.slack <= u * total and (u * total < ends[i] + self.slack or i == last)
            if inside and abs(np.log(w[i] / total) - log_probability) <= 2.0 ** -23 * abs(log_probability) + 2 * self.slack / w[i] + 2.0 ** -40:
                return True
        return False
