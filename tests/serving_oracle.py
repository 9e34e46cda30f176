"""Plain 64-bit numpy forms of the weight that cached keys receive, of eviction by it and
of log probabilities, written from their definitions in include/kraken_hip.h, for the
tests; and batches whose sequences share prefixes."""
import math

import numpy as np

import paged_oracle as po


def share_prefixes(cache_tokens, batch, groups):
    """groups: (first sequence, one past the last, prefix tokens) each; the tables' rows
    begin alike over the prefix's whole pages.  Returns group_starts and prefix_lengths
    of groups that stand one after another, with empty ones for gaps."""
    starts, lengths = [0], []
    for first, end, prefix in groups:
        if starts[-1] != first:
            starts.append(first)
            lengths.append(0)
        live = [b for b in range(first, end) if batch.new[b] > 0]
        for b in range(first, end):
            n = min(prefix, batch.before[b]) // cache_tokens
            if live:
                batch.table[b, :n] = batch.table[live[0], :n]
        starts.append(end)
        lengths.append(prefix)
    return np.array(starts, np.uint32), np.array(lengths, np.uint32)


def key_weights(cache, query, batch, heads, window, decay, old, stride):
    """old [sequences][kv_heads][stride] -> (new, tolerance of each).

    A weight's relative error is its score's error, and that of the row's sum once more:
    each at most 8 sqrt(head_dim) half steps of f32 of the absolute products' sum, and 64
    for the sums, exponentials and their quotient; the sum over rows adds a half step for
    each row, the decayed old weight three."""
    table, starts, lengths, tokens, max_query, max_keys = batch
    d, g, pt = cache.head_dim, heads // cache.kv_heads, cache.page_tokens
    out, tol = old.astype(np.float64).copy(), np.zeros(old.shape)
    half = 2.0 ** -24
    for b, first, count, length in po.live_sequences(cache, *batch):
        if count == 0 or length > stride:
            continue
        before, rows = length - count, min(count, window or count)
        ids = [int(table[b, p]) for p in range(-(-length // pt))]
        inside = np.array([po.inside(cache, ids[j // pt]) for j in range(length)])
        empty = np.zeros((pt, cache.kv_heads, d))
        k = np.concatenate([cache.values_of("key", i) if po.inside(cache, i) else empty
                            for i in ids])[:length]
        for h in range(cache.kv_heads):
            total, error = np.zeros(length), np.zeros(length)
            for i in range(count - rows, count):
                seen = inside & (np.arange(length) <= before + i)
                for head in range(h * g, (h + 1) * g):
                    if not seen.any():
                        continue
                    q = query[first + i, head].astype(np.float64)
                    s = np.where(seen, k[:, h] @ q / math.sqrt(d), -np.inf)
                    p = np.exp(s - s[seen].max())
                    p /= p.sum()
                    size = (np.abs(k[:, h]) @ np.abs(q))[seen].max() / math.sqrt(d)
                    total += p
                    error += p * half * (16.0 * math.sqrt(d) * size + 128.0)
            kept = np.zeros(length)
            if decay:
                kept[:before] = np.float64(np.float32(decay)) * out[b, h, :before]
            out[b, h, :length] = total + kept
            tol[b, h, :length] = error + half * (rows * g * total + 3 * np.abs(kept)) + 1e-36
    return out, tol


def select_keys(weights, lengths, keep, max_keys, first, last, kept_stride, blank=-7):
    """(kept, kept lengths), `blank` where nothing is written."""
    sequences, kv_heads, _ = weights.shape
    kept = np.full((sequences, kv_heads, kept_stride), blank, np.int32)
    out = np.full(sequences, blank, np.int32).view(np.uint32)
    for b in range(sequences):
        n = int(lengths[b])
        k = min(int(keep[b]), n)
        if n > max_keys or k > kept_stride:
            continue
        out[b] = k
        tail = min(last, k)
        head = min(first, k - tail, n - tail)
        for h in range(kv_heads):
            w = weights[b, h, head:n - tail].astype(np.float64)
            falling = np.where(np.isnan(w), np.inf, -np.where(np.isnan(w), 0, w))
            rank = np.lexsort((np.arange(len(w)), falling, np.isnan(w)))[:k - tail - head]
            kept[b, h, :k] = np.concatenate([np.arange(head), np.sort(rank) + head,
                                             np.arange(n - tail, n)])
    return kept, out


def gather(cache, table, kept, kept_lengths, kept_stride, target, weights=None, stride=0):
    """Changes `cache` (po.Pages) as the gather does; returns the weights' output with NaN
    where nothing is written.  f32 arithmetic, as defined."""
    sequences, kv_heads, _ = kept.shape
    pt, width = cache.page_tokens, target.shape[1]
    moved = None if weights is None else np.full(weights.shape, np.nan, np.float32)
    old = {n: (cache.codes[n].copy(), cache.scales[n].copy()) for n in ("key", "value")}
    for b in range(sequences):
        n = int(kept_lengths[b])
        if n > kept_stride or n > width * pt or weights is not None and n > stride:
            continue
        for h in range(kv_heads):
            if weights is not None:
                for i, j in enumerate(kept[b, h, :n]):
                    moved[b, h, i] = weights[b, h, j] if 0 <= j < stride else 0
            for p in range(-(-n // pt)):
                page = int(target[b, p])
                if not po.inside(cache, page):
                    continue
                source = []
                for j in kept[b, h, p * pt:min(n, (p + 1) * pt)]:
                    at = int(table[b, j // pt]) if 0 <= j // pt < table.shape[1] else -1
                    source.append((at, j % pt) if po.inside(cache, at) else None)
                for name, (codes, scales) in old.items():
                    s = np.array([0 if x is None else scales[x[0], h] for x in source],
                                 np.float32)
                    new = np.zeros((pt, cache.head_dim), np.int8)
                    bad = not np.isfinite(s).all()
                    to = np.float32(np.nan) if bad else np.float32(max(s.max(), 0))
                    for i, x in enumerate(source):
                        if x is None:
                            continue
                        ratio = np.float32(1) if bad or s[i] == to else np.float32(s[i] / to)
                        new[i] = np.rint(codes[x[0], h, x[1]].astype(np.float32) * ratio)
                    cache.codes[name][page, h] = new
                    cache.scales[name][page, h] = to
    return moved


def logprobs(logits, temperature, token, top):
    """One row: a dict of values, and of tolerances for the computed ones.

    Half steps of f32: x = (l - M) / T is off by 4 of itself; a weight by 3 |x| and what an
    exponential and 110 roundings of sums and joins of sums add; the logarithm by 4 of
    itself.  What lies below 2^-126 of the largest weight is lost, 2^22 times at most."""
    x = np.asarray(logits, np.float64)
    n, half, lost = len(x), 2.0 ** -24, 2.0 ** -104
    t = float(temperature) if temperature > 0 else 1.0
    real = ~np.isnan(x)
    order = np.lexsort((np.arange(n), np.where(real, -np.where(real, x, 0), 0), ~real))
    place = np.empty(n, np.int64)
    place[order] = np.arange(n)
    best = x[real].max() if real.any() else -math.inf
    found = {"rank": int(place[token]) if 0 <= token < n else n,
             "top_tokens": [int(i) for i in order[:top] if real[i]]}
    found["top_tokens"] += [n] * (top - len(found["top_tokens"]))
    if best == -math.inf:
        return {**found, "logprob": -math.inf, "entropy": 0.0, "top_logprobs": [-math.inf] * top,
                "logprob_off": 0.0, "entropy_off": 0.0, "top_off": [0.0] * top}
    with np.errstate(invalid="ignore", over="ignore"):
        y = (x - best) / t
    y[x == best] = 0.0
    y[~real | (x == -math.inf) | np.isnan(y)] = -math.inf
    w = np.exp(y)
    first = int(order[0])
    rest = np.delete(np.arange(n), first)
    finite = rest[np.isfinite(y[rest])]
    s = w[finite].sum()
    b = (w[finite] * -y[finite]).sum() / (1 + s)
    c = (w[finite] * y[finite] ** 2).sum() / (1 + s)
    total = math.log1p(s)
    off_sum = half * (3 * b + 115 * s / (1 + s) + 4 * total) + lost

    def of(i):
        if not 0 <= i < n or not np.isfinite(y[i]):
            return -math.inf, 0.0
        return y[i] - total, off_sum + half * (4 * abs(y[i]) + 2 * abs(y[i] - total))

    found["logprob"], found["logprob_off"] = of(token)
    tops = [of(i) for i in found["top_tokens"]]
    found["top_logprobs"], found["top_off"] = [v for v, _ in tops], [o for _, o in tops]
    found["entropy"] = total + b
    found["entropy_off"] = off_sum + half * (4 * c + 120 * b + 4 * (total + b)) + 2e2 * lost
    return found
