"""More operators of batched serving over a paged 8-bit cache, as cases.

Beside appending, attending and sampling, a server over pages of 8-bit keys and
values does the following.  Kinds of case (the sizes each takes are in draw()):

  shared    causal attention of a batch whose sequences begin, group by group,
            with the same pages (a system prompt, a document), with the output
            gate in f32 or in f16
  weights   the attention weight that each cached key receives from the batch's
            last rows, added to what it received before
  evict     the tokens that a cache keeps by that weight (the first ones, the
            newest, the heaviest), moved into fresh pages with their weights, and
            those pages read back as F16 rows, as a program that exports them does
  logprobs  log probability and rank of a given token, the entropy, and the
            likeliest tokens of each row of logits

`own` False computes them from elementary torch operations, True through the
library's entry points.
"""
import math
import os
import sys

import torch

own = False

_context = None


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "kraken-infer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kraken_hip

    return kraken_hip


def _ctx():
    """The program's context: on a torch stream that is made current, with an
    open batch (ops enqueue, the program waits where it needs results)."""
    global _context
    if _context is None:
        stream = torch.cuda.Stream()
        torch.cuda.set_stream(stream)
        _context = _library().Context()
        _context.set_stream(stream.cuda_stream)
        _context.begin_graph()
    return _context


def listed():
    model = {"kv_heads": 2, "group": 4, "head_dim": 256, "page_tokens": 64}
    return [
        # Four answers to one prompt: the smallest shared prefix.
        {"name": "shared_4x2048", "kind": "shared", "groups": 1, "members": 4, "query": 1,
         "prefix": 2048, "own_keys": 256, "f16": False, **model},
        # Batched decode of 64 sequences over one long document: the most bytes and flops.
        {"name": "shared_64x32768", "kind": "shared", "groups": 1, "members": 64, "query": 1,
         "prefix": 32768, "own_keys": 4096, "f16": False, **model},
        # Drafted tokens to verify, three prompts of several lengths, small pages and the
        # legacy layer's heads.
        {"name": "shared_verify_3x8", "kind": "shared", "groups": 3, "members": 8, "query": 8,
         "prefix": 8192, "own_keys": 700, "f16": True, "kv_heads": 8, "group": 2,
         "head_dim": 128, "page_tokens": 16},
        # One decode step of one sequence.
        {"name": "weights_one_4096", "kind": "weights", "sequences": 1, "query": 1,
         "ragged": False, "prefix": 4096, "window": 0, "decay": 0.98, "f16": False, **model},
        # A decode step of 64 sequences.
        {"name": "weights_decode_64", "kind": "weights", "sequences": 64, "query": 1,
         "ragged": False, "prefix": 32768, "window": 0, "decay": 0.98, "f16": False, **model},
        # The last 32 tokens of a prompt's last chunk, which judge the prompt.
        {"name": "weights_window_32", "kind": "weights", "sequences": 1, "query": 1024,
         "ragged": False, "prefix": 7168, "window": 32, "decay": 0.0, "f16": True, **model},
        # Every row of a chunk.
        {"name": "weights_chunk_1024", "kind": "weights", "sequences": 1, "query": 1024,
         "ragged": False, "prefix": 7168, "window": 0, "decay": 1.0, "f16": False, **model},
        # One sequence cut to a quarter.
        {"name": "evict_one_4096", "kind": "evict", "sequences": 1, "length": 4096, "keep": 1024,
         "first": 4, "last": 64, **model},
        # A server short of pages.
        {"name": "evict_16x32768", "kind": "evict", "sequences": 16, "length": 32768,
         "keep": 4096, "first": 16, "last": 256, **model},
        # The logprobs that an answer's token comes with.
        {"name": "logprobs_1x248320", "kind": "logprobs", "rows": 1, "size": 248320, "top": 5,
         "temperature": False, "spread": 2.5},
        # A decode step of 64 over a small vocabulary, the most alternatives.
        {"name": "logprobs_64x32000", "kind": "logprobs", "rows": 64, "size": 32000, "top": 20,
         "temperature": True, "spread": 2.5},
        # A prompt's tokens scored.
        {"name": "logprobs_512x248320", "kind": "logprobs", "rows": 512, "size": 248320, "top": 0,
         "temperature": False, "spread": 2.5},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["shared", "weights", "evict", "logprobs"])
    if kind == "logprobs":
        return {"kind": kind, "rows": _log_int(rng, 1, 256), "size": _log_int(rng, 1000, 248320),
                "top": rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([False, True]),
                "spread": rng.choice([0.5, 1.5, 2.5])}
    heads = rng.choice([{"kv_heads": 2, "group": 4, "head_dim": 256},
                        {"kv_heads": 4, "group": 2, "head_dim": 256},
                        {"kv_heads": 8, "group": 2, "head_dim": 128},
                        {"kv_heads": 4, "group": 7, "head_dim": 128},
                        {"kv_heads": 4, "group": 8, "head_dim": 64},
                        {"kv_heads": 3, "group": 3, "head_dim": 64}])
    case = {"kind": kind, **heads, "page_tokens": rng.choice([16, 32, 64, 64, 128])}
    if kind == "shared":
        groups = rng.choice([1, 1, 2, 3])
        case.update(groups=groups, members=_log_int(rng, 1, 64 // groups),
                    query=rng.choice([1, 1, 1, 2, 4, 8]), prefix=_log_int(rng, 16, 16384),
                    own_keys=rng.choice([0, _log_int(rng, 1, 2048)]),
                    f16=rng.choice([False, True]))
    elif kind == "weights":
        shape = rng.choice(["decode", "decode", "chunk", "mixed"])
        if shape == "decode":
            case.update(sequences=_log_int(rng, 1, 64), query=rng.choice([1, 1, 1, 2, 4]),
                        ragged=False, prefix=_log_int(rng, 1, 16384))
        elif shape == "chunk":
            case.update(sequences=1, query=_log_int(rng, 2, 768), ragged=False,
                        prefix=rng.choice([0, _log_int(rng, 1, 7168)]))
        else:
            case.update(sequences=_log_int(rng, 2, 24), query=_log_int(rng, 8, 256), ragged=True,
                        prefix=_log_int(rng, 1, 4096))
        case.update(window=rng.choice([0, 16, 32, 64]), decay=rng.choice([0.0, 0.95, 1.0]),
                    f16=rng.choice([False, True]))
    else:
        length = _log_int(rng, 64, 32768)
        case.update(sequences=_log_int(rng, 1, 16), length=length,
                    keep=_log_int(rng, 16, max(16, length // 2)),
                    first=rng.choice([0, 1, 4, 16]), last=rng.choice([0, 8, 64]))
    return case


# ------------------------------------------------------------------ inputs ---


def _spread(n):
    """0 .. n - 1 in a fixed order that mixes small and large."""
    step = 1
    while step * step < n or math.gcd(step, n) != 1:
        step += 1
    return [(b * step) % n for b in range(n)]


def _prefixes(case):
    """Each group's prefix in tokens, whole pages."""
    pt, n = case["page_tokens"], case["groups"]
    return [max(1, case["prefix"] * (g + 1) // n // pt) * pt for g in range(n)]


def _batch(case):
    """New tokens and tokens before them of each sequence: spread evenly; every
    second sequence of a ragged batch brings one token."""
    if case["kind"] == "shared":
        n = case["groups"] * case["members"]
        at, shared = _spread(n), _prefixes(case)
        return [case["query"]] * n, [shared[b // case["members"]]
                                     + case["own_keys"] * at[b] // max(1, n - 1)
                                     for b in range(n)]
    n, query, prefix = case["sequences"], case["query"], case["prefix"]
    if n == 1:
        return [query], [prefix]
    before = [prefix * a // (n - 1) for a in _spread(n)]
    new = [query] * n
    if case["ragged"]:
        new = [1 if b % 2 else 1 + (query - 1) * (n - 1 - b) // (n - 1) for b in range(n)]
    return new, before


def _lengths(case):
    """Lengths before an eviction, a quarter of the longest to the longest."""
    n, length = case["sequences"], case["length"]
    return [length] if n == 1 else [length // 4 + (length - length // 4) * a // (n - 1)
                                    for a in _spread(n)]


class _Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def codes(self, *shape):
        """8-bit values as a page's quantised normal values are spread."""
        x = torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float16)
        return x.mul_(35.0).clamp_(-127, 127).to(torch.int8)

    def integers(self, high, *shape):
        return torch.randint(0, high, shape, generator=self.gen, device="cuda")


def _u32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _prepare_pages(case, r, s, counts, shared=None, spare=3):
    """A page pool and the sequences' tables: counts[b] pages each, of which the
    first shared[b] = (group, pages) are its group's."""
    kv, d, pt = case["kv_heads"], case["head_dim"], case["page_tokens"]
    groups = {}
    for g, n in shared or []:
        groups[g] = n
    pages = spare + sum(groups.values()) + sum(counts)
    order = torch.randperm(pages, generator=r.gen, device="cuda").int()
    at = 0
    held = {}
    for g, n in groups.items():
        held[g] = order[at:at + n]
        at += n
    table = torch.full((len(counts), max(counts)), -1, device="cuda", dtype=torch.int32)
    for b, n in enumerate(counts):
        g, same = shared[b] if shared else (0, 0)
        if same:
            table[b, :same] = held[g]
        table[b, same:n] = order[at:at + n - same]
        at += n - same
    s.update(keys=r.codes(pages, kv, pt, d), values=r.codes(pages, kv, pt // 8, d, 8),
             key_scales=0.03 * torch.exp(0.3 * r.normal(pages, kv)),
             value_scales=0.03 * torch.exp(0.3 * r.normal(pages, kv)), table=table, pages=pages,
             width=max(counts), free=order[at:])


def prepare(case, seed):
    ctx = _ctx() if own else None
    r = _Inputs(seed)
    s = {"case": case, "ctx": ctx}
    {"shared": _prepare_batch, "weights": _prepare_batch, "evict": _prepare_evict,
     "logprobs": _prepare_logprobs}[case["kind"]](case, r, s)
    if own:
        kh = _library()
        b = s["view"] = {k: kh.as_buffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if case["kind"] != "logprobs":
            s["cache"] = kh.PagedQ8Cache(b["keys"], b["values"], b["key_scales"],
                                         b["value_scales"], s["pages"], case["page_tokens"],
                                         case["kv_heads"], case["head_dim"])
        if case["kind"] == "evict":
            # A sequence is given the pages that its kept tokens reach into: what others held
            # would be read back as it was.
            first = torch.arange(s["target_width"], device="cuda") * case["page_tokens"]
            has = first < torch.minimum(s["keep"], s["lengths"])[:, None]
            s["given"] = torch.where(has, s["target"], -1)
            b["target"] = kh.as_buffer(s["given"])
        if case["kind"] in ("shared", "weights"):
            s["batch"] = kh.PagedBatch(b["table"], b["starts"], b["lengths"], s["sequences"],
                                       s["width"], s["tokens"], s["max_query"], s["max_keys"])
        if case["kind"] == "shared":
            s["prefixes"] = kh.SharedPrefixes(b["group_starts"], b["prefix_lengths"],
                                              case["groups"], case["members"] * case["query"],
                                              s["max_prefix"])
    return s


def _prepare_batch(case, r, s):
    new, before = _batch(case)
    kv, d, pt = case["kv_heads"], case["head_dim"], case["page_tokens"]
    heads = kv * case["group"]
    lengths = [a + b for a, b in zip(new, before)]
    shared = None
    if case["kind"] == "shared":
        shared = [(b // case["members"], _prefixes(case)[b // case["members"]] // pt)
                  for b in range(len(new))]
    _prepare_pages(case, r, s, [-(-l // pt) for l in lengths], shared)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    kind = torch.float16 if case["f16"] else torch.float32
    s.update(sequences=len(new), starts=_u32(starts), lengths=_u32(lengths), tokens=starts[-1],
             max_query=max(new), max_keys=max(lengths),
             query=(2.0 * r.normal(starts[-1], heads, d)).to(kind))
    if case["kind"] == "shared":
        s.update(group_starts=_u32([case["members"] * g for g in range(case["groups"] + 1)]),
                 prefix_lengths=_u32(_prefixes(case)), max_prefix=max(_prefixes(case)),
                 gate=None if case["f16"] else r.normal(starts[-1], heads, d),
                 out=torch.empty(starts[-1], heads, d, device="cuda", dtype=kind))
    else:
        s["key_weights"] = torch.exp(2.0 * r.normal(len(new), kv, max(lengths)) - 4.0)


def _prepare_evict(case, r, s):
    kv, d, pt = case["kv_heads"], case["head_dim"], case["page_tokens"]
    lengths, n = _lengths(case), case["sequences"]
    width = -(-case["keep"] // pt)
    _prepare_pages(case, r, s, [-(-l // pt) for l in lengths], spare=3 + n * width)
    weights = torch.exp(2.0 * r.normal(n, kv, max(lengths)) - 4.0)
    # Some keys received nothing that f32 can hold: they tie.
    weights = torch.where(r.uniform(n, kv, max(lengths)) < 0.2, 0.0, weights)
    size = (n * width, pt, kv, d)
    s.update(lengths=_u32(lengths), max_keys=max(lengths), key_weights=weights,
             keep=_u32([case["keep"]] * n), target_width=width,
             target=s["free"][:n * width].reshape(n, width).contiguous(),
             kept=torch.full((n, kv, case["keep"]), -1, device="cuda", dtype=torch.int32),
             kept_lengths=torch.zeros(n, device="cuda", dtype=torch.int32),
             kept_weights=torch.zeros_like(weights),
             key_rows=torch.empty(size, device="cuda", dtype=torch.float16),
             value_rows=torch.empty(size, device="cuda", dtype=torch.float16))


def _prepare_logprobs(case, r, s):
    rows, size, top = case["rows"], case["size"], case["top"]
    logits = case["spread"] * r.normal(rows, size)
    # A few likely tokens stand out, as a model's do.
    likely = r.integers(size, rows, 24)
    logits.scatter_add_(1, likely, 10.0 * r.uniform(rows, 24))
    given = torch.where(r.uniform(rows) < 0.7, likely[:, 0], r.integers(size, rows))

    def out(kind, *shape):
        return torch.empty(*shape, device="cuda", dtype=kind)

    s.update(logits=logits, tokens=given.int(),
             temperature=(0.5 + r.uniform(rows)) if case["temperature"] else None,
             logprob=out(torch.float32, rows), rank=out(torch.int32, rows),
             entropy=out(torch.float32, rows),
             top_tokens=out(torch.int32, rows, top) if top else None,
             top_logprobs=out(torch.float32, rows, top) if top else None)


# --------------------------------------------------------------------- run ---


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"shared": _own_shared, "weights": _own_weights, "evict": _own_evict,
                "logprobs": _own_logprobs}[kind](s)
    return {"shared": _plain_shared, "weights": _plain_weights, "evict": _plain_evict,
            "logprobs": _plain_logprobs}[kind](s)


def _own_shared(s):
    c, b = s["case"], s["view"]
    heads = c["kv_heads"] * c["group"]
    if c["f16"]:
        s["ctx"].attention_f16q_shared_paged_q8_kv(b["query"], s["cache"], s["batch"],
                                                   s["prefixes"], heads, b["out"])
    else:
        s["ctx"].attention_f32_shared_paged_q8_kv(b["query"], b["gate"], s["cache"], s["batch"],
                                                  s["prefixes"], heads, b["out"])
    return s["out"]


def _own_weights(s):
    c, b = s["case"], s["view"]
    call = (s["ctx"].key_weights_f16q_paged_q8_kv if c["f16"]
            else s["ctx"].key_weights_f32_paged_q8_kv)
    call(b["query"], s["cache"], s["batch"], c["kv_heads"] * c["group"], c["window"], c["decay"],
         b["key_weights"], s["max_keys"])
    return s["key_weights"]


def _own_evict(s):
    c, ctx, b = s["case"], s["ctx"], s["view"]
    ctx.select_keys_f32_i32(b["key_weights"], s["max_keys"], b["lengths"], b["keep"],
                            c["sequences"], c["kv_heads"], s["max_keys"], c["first"], c["last"],
                            b["kept"], c["keep"], b["kept_lengths"])
    ctx.gather_kv_pages_q8(s["cache"], b["table"], s["width"], b["kept"], b["kept_lengths"],
                           c["keep"], c["sequences"], b["target"], s["target_width"],
                           b["key_weights"], s["max_keys"], b["kept_weights"])
    ctx.dequantize_kv_pages_q8_f16(s["cache"], b["target"], s["target"].numel(), b["key_rows"],
                                   b["value_rows"])
    return {k: s[k] for k in ("kept", "kept_lengths", "kept_weights", "key_rows", "value_rows")}


def _own_logprobs(s):
    c, b = s["case"], s["view"]
    s["ctx"].token_logprobs_f32(b["logits"], c["rows"], c["size"], c["size"],
                                b.get("temperature"), b["tokens"], c["top"], b["logprob"],
                                b["rank"], b["entropy"], b.get("top_tokens"),
                                b.get("top_logprobs"))
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top_tokens", "top_logprobs")}


# ------------------------------------------------------------- plain forms ---


def _token_sequence(s):
    """The sequence of each token, and the token's position in it."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), t.int(), right=True)
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1]).long()
    return seq, first[seq] + t - s["starts"].long()[seq]


def _sequence_keys(s):
    """The keys of every sequence, [sequences][kv_heads][keys][dim]."""
    at = s["table"].long().clamp(min=0)
    keys = s["keys"][at].float() * s["key_scales"][at][..., None, None]
    return keys.transpose(1, 2).reshape(len(at), keys.shape[2], -1, keys.shape[4])


def _sequence_values(s):
    at = s["table"].long().clamp(min=0)
    values = s["values"][at].float() * s["value_scales"][at][..., None, None, None]
    n, p, h, o, d, e = values.shape
    return values.permute(0, 2, 1, 3, 5, 4).reshape(n, h, p * o * e, d)


def _softmax_weights(s, window=0):
    """The batch's rows by sequence, each one's last `window` (0: all): (sequence and place
    of each token, the weights of their keys [sequences][kv_heads][rows][keys])."""
    c = s["case"]
    kv, g, d, n = c["kv_heads"], c["group"], c["head_dim"], s["sequences"]
    rows = min(window or s["max_query"], s["max_query"])
    seq, position = _token_sequence(s)
    # Place 0 takes the rows before the window.
    place = (torch.arange(s["tokens"], device="cuda") - s["starts"].long()[seq + 1] + rows
             if window else torch.arange(s["tokens"], device="cuda") - s["starts"].long()[seq])
    place = (place + 1).clamp(min=0)
    padded = torch.zeros(n, rows + 1, kv, g, d, device="cuda")
    padded[seq, place] = s["query"].float().view(-1, kv, g, d)
    padded = padded[:, 1:].transpose(1, 2).reshape(n, kv, -1, d)
    last = torch.full((n, rows + 1), -1, device="cuda", dtype=torch.int64)
    last[seq, place] = position
    scores = torch.matmul(padded, _sequence_keys(s).transpose(2, 3)) / math.sqrt(d)
    number = torch.arange(scores.shape[-1], device="cuda")
    masked = number > last[:, 1:].repeat_interleave(g, 1)[:, None, :, None]
    scores = scores.masked_fill_(masked, -1e30)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    return seq, place - 1, weights * (last[:, 1:] >= 0).repeat_interleave(g, 1)[:, None, :, None]


def _plain_shared(s):
    c = s["case"]
    kv, g, d, n = c["kv_heads"], c["group"], c["head_dim"], s["sequences"]
    seq, within, weights = _softmax_weights(s)
    out = torch.matmul(weights, _sequence_values(s)).view(n, kv, -1, g, d).transpose(1, 2)
    out = out[seq, within].reshape(-1, kv * g, d)
    if s["gate"] is not None:
        out = out * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return out.to(s["out"].dtype)


def _plain_weights(s):
    c = s["case"]
    _, _, weights = _softmax_weights(s, c["window"])
    count = (s["starts"][1:] - s["starts"][:-1]).long()[:, None]
    received = weights.sum(2)[..., :s["max_keys"]]
    key = torch.arange(s["max_keys"], device="cuda")
    length = s["lengths"].long()[:, None]
    before = torch.where((key < length - count)[:, None], c["decay"] * s["key_weights"], 0.0)
    s["key_weights"].copy_(torch.where((key < length)[:, None], before + received,
                                       s["key_weights"]))
    return s["key_weights"]


def _plain_evict(s):
    c = s["case"]
    n, kv, d, pt = c["sequences"], c["kv_heads"], c["head_dim"], c["page_tokens"]
    # What is kept: the newest, the first, then the heaviest.
    length = s["lengths"].long()[:, None]
    keep = torch.minimum(s["keep"].long()[:, None], length)
    last = keep.clamp(max=c["last"])
    first = torch.minimum((keep - last).clamp(max=c["first"]), length - last)
    key = torch.arange(s["max_keys"], device="cuda")
    always = (key < first) | (key >= length - last) & (key < length)
    rank = torch.where(always[:, None], math.inf, s["key_weights"])
    rank = torch.where((key < length)[:, None], rank, -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :c["keep"]]
    place = torch.arange(order.shape[2], device="cuda")
    counted = (place < keep)[:, None]
    index = torch.sort(torch.where(counted, order, s["max_keys"]), 2).values
    index = torch.where(counted, index, 0)
    s["kept"][..., :index.shape[2]] = torch.where(counted, index, s["kept"][..., :index.shape[2]])
    s["kept_lengths"].copy_(keep[:, 0])
    s["kept_weights"][..., :index.shape[2]] = torch.where(
        counted, s["key_weights"].gather(2, index), s["kept_weights"][..., :index.shape[2]])
    # Their codes, by target page.
    slots = s["target_width"] * pt
    at = torch.zeros(n, kv, slots, device="cuda", dtype=torch.int64)
    at[..., :index.shape[2]] = index
    real = torch.zeros(n, kv, slots, device="cuda", dtype=torch.bool)
    real[..., :index.shape[2]] = counted
    page = s["table"].long().gather(1, (at // pt).view(n, -1)).view(n, kv, slots).clamp(min=0)
    head = torch.arange(kv, device="cuda")[None, :, None].expand_as(at)
    ids = s["target"].long()
    found = {}
    for name, codes in (("key", s["keys"][page, head, at % pt]),
                        ("value", s["values"][page, head, at % pt // 8, :, at % 8])):
        scale = s[name + "_scales"][page, head]
        most = torch.where(real, scale, 0.0).view(n, kv, -1, pt).amax(3)
        wide = most.repeat_interleave(pt, 2)
        codes = torch.round(codes.float() * torch.where(scale == wide, 1.0, scale / wide)[..., None])
        codes = torch.where(real[..., None], codes, 0.0).view(n, kv, -1, pt, d)
        codes, most = codes.transpose(1, 2), most.transpose(1, 2)
        s[name + "_scales"][ids] = most
        if name == "key":
            s["keys"][ids] = codes.to(torch.int8)
        else:
            s["values"][ids] = codes.view(n, -1, kv, pt // 8, 8, d).transpose(4, 5).to(torch.int8)
        rows = codes * most[..., None, None]
        found[name + "_rows"] = rows.transpose(2, 3).reshape(-1, pt, kv, d).half()
    return {**{k: s[k] for k in ("kept", "kept_lengths", "kept_weights")}, **found}


def _plain_logprobs(s):
    logits, top = s["logits"], s["case"]["top"]
    x = logits - logits.amax(1, keepdim=True)
    if s["temperature"] is not None:
        x = x / s["temperature"][:, None]
    weight = torch.exp(x)
    # Without the largest, so that what is near one keeps its distance from it.
    rest = torch.where(x == 0, 0.0, weight)
    equal = (x == 0).sum(1, dtype=torch.float32) - 1.0
    others = rest.sum(1) + equal
    total = torch.log1p(others)
    given = s["tokens"].long()[:, None]
    mine, number = logits.gather(1, given), torch.arange(logits.shape[1], device="cuda")
    rank = ((logits > mine) | (logits == mine) & (number < given)).sum(1, dtype=torch.int32)
    found = {"logprob": x.gather(1, given)[:, 0] - total, "rank": rank,
             "entropy": total - (rest * x).sum(1) / (1.0 + others), "top_tokens": None,
             "top_logprobs": None}
    if top:
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        found.update(top_tokens=order.int(), top_logprobs=x.gather(1, order) - total[:, None])
    return found


# -------------------------------------------------------------------- work ---


def work(case):
    if case["kind"] == "logprobs":
        # Every logit once; a subtraction, an exponential and two sums for each.
        n = case["rows"] * case["size"]
        return {"bytes": 4 * n + case["rows"] * (20 + 8 * case["top"]), "flops": 4 * n}
    kv, d, pt = case["kv_heads"], case["head_dim"], case["page_tokens"]
    if case["kind"] == "evict":
        lengths = _lengths(case)
        kept = sum(min(l, case["keep"]) for l in lengths)
        rows = case["sequences"] * -(-case["keep"] // pt) * pt
        # Weights in, indexes and weights out, codes in and out, F16 rows out.
        return {"bytes": kv * (4 * sum(lengths) + 8 * kept + 4 * d * kept + 4 * d * rows),
                "flops": kv * (sum(lengths) + 2 * d * kept)}
    new, before = _batch(case)
    heads = kv * case["group"]
    size = 2 if case["f16"] else 4
    if case["kind"] == "shared":
        prefixes = _prefixes(case)
        keys = sum(prefixes) + sum(a + b - prefixes[i // case["members"]]
                                   for i, (a, b) in enumerate(zip(new, before)))
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, before))
        rows = sum(new) * heads * d * size * (2 if case["f16"] else 3)
        return {"bytes": 2 * keys * kv * d + 8 * kv * (keys // pt) + rows,
                "flops": 4 * heads * d * pairs}
    keys = sum(a + b for a, b in zip(new, before))
    counted = [min(a, case["window"] or a) for a in new]
    pairs = sum(w * (a + b) - w * (w - 1) // 2 for w, a, b in zip(counted, new, before))
    held = 8 if case["decay"] else 4
    return {"bytes": keys * kv * (d + held) + 4 * kv * (keys // pt)
            + sum(counted) * heads * d * size, "flops": 2 * heads * d * pairs}


# ------------------------------------------------------------------- exact ---


def exact(case, seed):
    """From the definitions, sequence by sequence, in 64 bits."""
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"shared": _exact_shared, "weights": _exact_weights, "evict": _exact_evict,
            "logprobs": _exact_logprobs}[case["kind"]](s)


def _exact_keys(s, b, h, length):
    ids = s["table"][b, :-(-length // s["case"]["page_tokens"])].long()
    k = s["keys"][ids, h].double() * s["key_scales"][ids, h].double()[:, None, None]
    return k.flatten(0, 1)[:length]


def _exact_values(s, b, h, length):
    ids = s["table"][b, :-(-length // s["case"]["page_tokens"])].long()
    v = s["values"][ids, h].double() * s["value_scales"][ids, h].double()[:, None, None, None]
    return v.transpose(2, 3).flatten(0, 2)[:length]


def _exact_softmax(s, b, h, rows):
    """Weights of the last `rows` new tokens of a sequence, [group][rows][keys]."""
    c = s["case"]
    g, length, end = c["group"], int(s["lengths"][b]), int(s["starts"][b + 1])
    q = s["query"][end - rows:end, h * g:(h + 1) * g].double().transpose(0, 1).contiguous()
    k = _exact_keys(s, b, h, length)
    w = (q.view(-1, c["head_dim"]) @ k.T.contiguous()).view(g, rows, length)
    w /= math.sqrt(c["head_dim"])
    limit = torch.arange(length - rows, length, device=w.device)[:, None]
    w.masked_fill_(torch.arange(length, device=w.device) > limit, -math.inf)
    return torch.softmax(w, -1)


def _exact_shared(s):
    c = s["case"]
    out, q = [], c["query"]
    for b in range(s["sequences"]):
        length, rows = int(s["lengths"][b]), []
        for h in range(c["kv_heads"]):
            w = _exact_softmax(s, b, h, q)
            v = _exact_values(s, b, h, length)
            rows.append((w.view(-1, length) @ v).view(c["group"], q, -1).transpose(0, 1))
        out.append(torch.cat(rows, 1))
    out = torch.cat(out)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_weights(s):
    c = s["case"]
    new, before = _batch(c)
    out = s["key_weights"].double()
    for b, (n, p) in enumerate(zip(new, before)):
        for h in range(c["kv_heads"]):
            got = _exact_softmax(s, b, h, min(n, c["window"] or n)).sum((0, 1))
            got[:p] += c["decay"] * out[b, h, :p]
            out[b, h, :n + p] = got
    return out


def _exact_evict(s):
    """The whole numbers have no 64-bit value beside them."""
    c = s["case"]
    kv, d, pt = c["kv_heads"], c["head_dim"], c["page_tokens"]
    weights = torch.zeros_like(s["key_weights"], dtype=torch.float64)
    shape = (c["sequences"], s["target_width"] * pt, kv, d)
    rows = {n: torch.zeros(shape, device="cuda", dtype=torch.float64) for n in ("key", "value")}
    for b, length in enumerate(_lengths(c)):
        n = min(c["keep"], length)
        last = min(n, c["last"])
        first = min(n - last, c["first"], length - last)
        for h in range(kv):
            w = s["key_weights"][b, h, first:length - last].double()
            best = torch.argsort(w, descending=True, stable=True)[:n - last - first] + first
            kept = torch.cat([torch.arange(first, device="cuda"), torch.sort(best).values,
                              torch.arange(length - last, length, device="cuda")])
            weights[b, h, :n] = s["key_weights"][b, h, kept].double()
            ids = s["table"][b].long()[kept // pt]
            for name, read in (("key", _exact_keys), ("value", _exact_values)):
                scale = s[name + "_scales"][ids, h].double()
                value = read(s, b, h, length)[kept]
                for at in range(0, n, pt):
                    step = scale[at:at + pt].max()
                    rows[name][b, at:min(n, at + pt), h] = step * torch.round(
                        value[at:at + pt] / step)
    return {"kept": None, "kept_lengths": None, "kept_weights": weights,
            "key_rows": rows["key"].view(-1, pt, kv, d),
            "value_rows": rows["value"].view(-1, pt, kv, d)}


def _exact_logprobs(s):
    top, x = s["case"]["top"], s["logits"]
    found = {"logprob": [], "rank": None, "entropy": [], "top_tokens": None, "top_logprobs": []}
    for r in range(x.shape[0]):
        row = x[r].double()
        if s["temperature"] is not None:
            row = row / s["temperature"][r].double()
        p = torch.log_softmax(row, 0)
        found["logprob"].append(p[int(s["tokens"][r])])
        found["entropy"].append(-(p.exp() * p).sum())
        if top:
            found["top_logprobs"].append(torch.topk(p, top).values)
    return {k: torch.stack(v) if v else None for k, v in found.items()}
