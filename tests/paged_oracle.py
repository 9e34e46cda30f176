"""Plain 64-bit numpy forms of the paged 8-bit cache's operators and of sampling,
written from their definitions in include/kraken_hip.h, for the tests."""
import math

import numpy as np


class Pages:
    """A paged 8-bit cache: codes as [page][head][token][dim] for keys and values
    alike; device_values() gives the values' runs of eight tokens."""

    def __init__(self, rng, pages, page_tokens, kv_heads, head_dim, spread=35.0):
        self.pages, self.page_tokens = pages, page_tokens
        self.kv_heads, self.head_dim = kv_heads, head_dim
        shape = (pages, kv_heads, page_tokens, head_dim)

        def codes():
            return np.clip(np.rint(spread * rng.standard_normal(shape)), -127, 127).astype(np.int8)

        self.codes = {"key": codes(), "value": codes()}
        self.scales = {n: (0.03 * np.exp(0.4 * rng.standard_normal((pages, kv_heads)))).astype(
            np.float32) for n in ("key", "value")}

    def device_values(self):
        p, h, t, d = self.codes["value"].shape
        return np.ascontiguousarray(
            self.codes["value"].reshape(p, h, t // 8, 8, d).transpose(0, 1, 2, 4, 3))

    def set_device_values(self, flat):
        p, h, t, d = self.codes["value"].shape
        self.codes["value"] = np.ascontiguousarray(
            flat.reshape(p, h, t // 8, d, 8).transpose(0, 1, 2, 4, 3)).reshape(p, h, t, d)

    def values_of(self, name, page):
        """[token][head][dim] in 64 bits."""
        return (self.codes[name][page].astype(np.float64)
                * self.scales[name][page].astype(np.float64)[:, None, None]).transpose(1, 0, 2)


def inside(cache, page):
    return 0 <= page < cache.pages


def live_sequences(cache, table, starts, lengths, tokens, max_query, max_keys):
    """(sequence, first row, rows, length) of those that keep the batch's bounds."""
    for b in range(len(lengths)):
        first, count, length = int(starts[b]), int(starts[b + 1]) - int(starts[b]), int(lengths[b])
        if (count >= 0 and first + count <= tokens and count <= min(max_query, length)
                and length <= max_keys and length <= table.shape[1] * cache.page_tokens):
            yield b, first, count, length


def norm_rope(x, weight, positions, n_dims, sections, theta, eps):
    """x [tokens][heads][dim], positions [4][tokens]."""
    x = x.astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    out, half = x.copy(), n_dims // 2
    ends = np.cumsum(sections)
    for i in range(half):
        row = int(np.searchsorted(ends[:3], i % ends[3], side="right"))
        angle = positions[row].astype(np.float64) * float(theta) ** (-2.0 * i / n_dims)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        out[..., i] = x[..., i] * c - x[..., i + half] * s
        out[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return out


def append(cache, name, rows, batch):
    """Quantises rows [tokens][heads][dim] (64 bits) into the cache, in place.
    Returns {(page, head): (slots, x / scale before rounding)} for the new codes."""
    table, starts, lengths, tokens, max_query, max_keys = batch
    exact = {}
    pt = cache.page_tokens
    for b, first, count, length in live_sequences(cache, *batch):
        begin = length - count
        for p in range(begin // pt, (length + pt - 1) // pt if count else 0):
            page = int(table[b, p])
            if not inside(cache, page):
                continue
            lo, hi = max(begin, p * pt), min(length, (p + 1) * pt)
            new = rows[first + lo - begin:first + hi - begin]
            for h in range(cache.kv_heads):
                largest = np.abs(new[:, h]).max()
                scale = cache.scales[name][page, h]
                codes = cache.codes[name][page, h]
                slots = slice(lo - p * pt, hi - p * pt)
                if not np.isfinite(new[:, h]).all() or np.isnan(scale) and lo != p * pt:
                    cache.scales[name][page, h] = np.nan
                    if np.isfinite(new[:, h]).all():
                        codes[slots] = 0
                    else:
                        codes[slots] = 0
                    continue
                if lo == p * pt or scale == 0:
                    scale = np.float32(np.float32(largest) / np.float32(127))
                    if scale < 2.0 ** -100:
                        scale = np.float32(0)
                    codes[:lo - p * pt] = 0
                else:
                    steps = 0
                    while largest > 127.0 * float(scale) * 2.0 ** steps:
                        steps += 1
                    if steps:
                        old = codes[:lo - p * pt].astype(np.float64)
                        codes[:lo - p * pt] = np.rint(old * 2.0 ** -steps).astype(np.int8)
                        scale = np.float32(float(scale) * 2.0 ** steps)
                cache.scales[name][page, h] = scale
                x = new[:, h] / float(scale) if scale > 0 else np.zeros_like(new[:, h])
                codes[slots] = np.clip(np.rint(x), -127, 127).astype(np.int8)
                exact[page, h] = (slots, x)
    return exact


def attention(cache, query, batch, heads, gate=None):
    """Returns (output, magnitude, score): magnitude [tokens][heads][dim] is the sum of
    the absolute weighted values, score [tokens][heads][2] the largest sum of absolute
    products of a query with a key, and the number of keys times the largest product of
    a weight with its value page's scale.  Rows of no sequence are NaN."""
    table, starts, lengths, tokens, max_query, max_keys = batch
    d, g, pt = cache.head_dim, heads // cache.kv_heads, cache.page_tokens
    out = np.full((tokens, heads, d), np.nan)
    size, score = np.full_like(out, np.nan), np.full((tokens, heads, 2), np.nan)
    for b, first, count, length in live_sequences(cache, *batch):
        if count == 0:
            continue
        ids = [int(table[b, p]) for p in range(-(-length // pt))]
        where = np.array([pos for pos in range(length) if inside(cache, ids[pos // pt])], np.int64)
        empty = np.zeros((pt, cache.kv_heads, d))
        k, v = (np.concatenate([cache.values_of(n, i) if inside(cache, i) else empty
                                for i in ids])[where] for n in ("key", "value"))
        steps = np.array([cache.scales["value"][ids[pos // pt]] for pos in where], np.float64)
        for i in range(count):
            seen = int((where <= length - count + i).sum())
            for h in range(heads):
                q = query[first + i, h].astype(np.float64)
                if seen == 0:
                    out[first + i, h] = size[first + i, h] = 0
                    score[first + i, h] = 0
                    continue
                kk, vv = k[:seen, h // g], v[:seen, h // g]
                s = kk @ q / math.sqrt(d)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[first + i, h] = w @ vv
                size[first + i, h] = w @ np.abs(vv)
                score[first + i, h] = ((np.abs(kk) @ np.abs(q)).max() / math.sqrt(d),
                                       seen * (w * steps[:seen, h // g]).max())
    if gate is not None:
        out *= 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
    return out, size, score


def attention_tolerance(magnitude, out, score, head_dim, f16):
    """Per value.  A score is a sum of head_dim products in f32: its error is about
    sqrt(head_dim) half steps of the absolute products' sum, taken 8 times, and a
    score's error is its weight's relative one; the sums over keys, the exponential
    and the division add at most 64 half steps.  The exponent of a page's value scale is
    at most 128 in size, so that it and what it is added to are off by half a step of 128
    (2^-18) times ln 2 in the weight.  Beside these, a weight times its scale is held in
    f16 parts whose last place is 2^-24 of a unit that is at least 2^-11 of the largest:
    what lies below is lost, 2^-35 of the largest weight times scale, for codes of up to
    127 and each key.  With f16 a weight is off by half a step of f16, and so is the
    output."""
    step = 2.0 ** -24
    tol = magnitude * step * (8.0 * math.sqrt(head_dim) * score[..., :1] + 64.0)
    tol = tol + magnitude * 2.0 ** -18 + 127.0 * 2.0 ** -35 * score[..., 1:]
    if f16:
        tol = tol + magnitude * 2.0 ** -11 + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    return tol + 1e-30


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.0):
    """One row: (token, probability)."""
    x = np.asarray(logits, np.float64)
    n = len(x)
    real = ~np.isnan(x)
    if not real.any():
        return n, 0.0
    top = x[real].max()
    first = int(np.flatnonzero(real & (x == top))[0])
    if top == -math.inf:
        return first, 0.0
    if not temperature > 0 or min_p > 1:
        return first, 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - top) / np.float64(temperature))
    w[x == top] = 1.0
    w[~real | (x == -math.inf)] = 0.0
    order = np.argsort(-np.where(real, x, -math.inf), kind="stable")
    order = order[real[order]]
    if 0 < top_k < n:
        order = order[:top_k]
    count = len(order)
    if top_p < 1:
        sums = np.cumsum(w[order])
        before = np.concatenate([[0.0], sums[:-1]])
        count = max(1, int((before < np.float64(np.float32(top_p)) * sums[-1]).sum()))
    keep = order[:count]
    if min_p > 0:
        keep = keep[w[keep] >= np.float64(np.float32(min_p))]
    keep = np.sort(keep)
    keep = keep[w[keep] > 0]
    sums = np.cumsum(w[keep])
    u = 0.0 if math.isnan(uniform) else min(max(float(np.float32(uniform)), 0.0), 1.0)
    at = min(int((sums <= u * sums[-1]).sum()), len(keep) - 1)
    return int(keep[at]), float(w[keep[at]] / sums[-1])
