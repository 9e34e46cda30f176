"""The operators of batched serving over a paged 8-bit cache, as cases.

A server holds the keys and values of its sequences in pages of 16 to 128
tokens, each value in 8 bits with one scale for each page and KV head.  A step
takes a ragged batch: some sequences bring a chunk of a prompt, most bring the
one token that they decode.  Kinds of case (the sizes each takes are in
draw()):

  append  the attention prologue of the batch: q and k RMSNorm, rotary
          positions, the split of the joint q/gate projection, and the new
          keys and values quantised into their pages; then the pages that it
          touched read back as F16 rows, as a program that exports a cache does
  attend  causal attention of the batch's tokens over their pages, in f32 with
          the output gate or in f16
  sample  one token a row from logits, with temperature, top-k, top-p and min-p
          and given uniform numbers

`own` False computes them from elementary torch operations, True through the
library's entry points.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
THETA = 1e7
SECTIONS = (11, 11, 10, 0)

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
        # The one token of a decode step: the smallest call.
        {"name": "append_one", "kind": "append", "sequences": 1, "query": 1, "ragged": False,
         "prefix": 4096, **model},
        # A decode step of 64 sequences.
        {"name": "append_decode_64", "kind": "append", "sequences": 64, "query": 1,
         "ragged": False, "prefix": 32768, **model},
        # A whole prompt chunk that begins inside a page.
        {"name": "append_chunk_1024", "kind": "append", "sequences": 1, "query": 1024,
         "ragged": False, "prefix": 7150, **model},
        # One decode token over a 4k context.
        {"name": "attend_one_4096", "kind": "attend", "sequences": 1, "query": 1, "ragged": False,
         "prefix": 4096, "f16": False, **model},
        # Batched decode of 64 sequences of up to 32768 tokens: the most bytes.
        {"name": "attend_decode_64", "kind": "attend", "sequences": 64, "query": 1,
         "ragged": False, "prefix": 32768, "f16": False, **model},
        # The last few tokens of a prompt, or drafted tokens to verify.
        {"name": "attend_tail_37", "kind": "attend", "sequences": 1, "query": 37, "ragged": False,
         "prefix": 6144, "f16": False, **model},
        # A whole prompt chunk late in a prompt, in f32 and in f16: the most flops.
        {"name": "attend_chunk_1024", "kind": "attend", "sequences": 1, "query": 1024,
         "ragged": False, "prefix": 7168, "f16": False, **model},
        {"name": "attend_chunk_1024_f16", "kind": "attend", "sequences": 1, "query": 1024,
         "ragged": False, "prefix": 7168, "f16": True, **model},
        # A mixed batch: prompt chunks beside single tokens, heads of the
        # legacy layer, small pages.
        {"name": "attend_mixed_17", "kind": "attend", "sequences": 17, "query": 200,
         "ragged": True, "prefix": 4001, "f16": True, "kv_heads": 8, "group": 2, "head_dim": 128,
         "page_tokens": 16},
        # A small vocabulary, a few rows.
        {"name": "sample_8x32000", "kind": "sample", "rows": 8, "size": 32000, "filters": "mixed",
         "spread": 2.5},
        # The full vocabulary: one sequence, and a decode step of 64.
        {"name": "sample_1x248320", "kind": "sample", "rows": 1, "size": 248320,
         "filters": "nucleus", "spread": 2.5},
        {"name": "sample_64x248320", "kind": "sample", "rows": 64, "size": 248320,
         "filters": "mixed", "spread": 2.5},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log_int(rng, 1, 64), "size": _log_int(rng, 1000, 248320),
                "filters": rng.choice(["mixed", "mixed", "nucleus", "none"]),
                "spread": rng.choice([0.5, 1.5, 2.5])}
    heads = rng.choice([{"kv_heads": 2, "group": 4, "head_dim": 256},
                        {"kv_heads": 4, "group": 2, "head_dim": 256},
                        {"kv_heads": 8, "group": 2, "head_dim": 128},
                        {"kv_heads": 4, "group": 7, "head_dim": 128},
                        {"kv_heads": 4, "group": 8, "head_dim": 64},
                        {"kv_heads": 3, "group": 3, "head_dim": 64}])
    case = {"kind": kind, **heads, "page_tokens": rng.choice([16, 32, 64, 64, 128])}
    shape = rng.choice(["decode", "decode", "chunk", "mixed"])
    if shape == "decode":
        case.update(sequences=_log_int(rng, 1, 64), query=rng.choice([1, 1, 1, 2, 4]),
                    ragged=False, prefix=_log_int(rng, 1, 16384))
    elif shape == "chunk":
        case.update(sequences=1, query=_log_int(rng, 2, 1024), ragged=False,
                    prefix=rng.choice([0, _log_int(rng, 1, 8192)]))
    else:
        case.update(sequences=_log_int(rng, 2, 24), query=_log_int(rng, 8, 256), ragged=True,
                    prefix=_log_int(rng, 1, 4096))
    if kind == "attend":
        case["f16"] = rng.choice([False, True])
    return case


# ------------------------------------------------------------------ inputs ---


def _batch(case):
    """New tokens and tokens before them of each sequence: spread evenly in a
    fixed order that mixes short and long ones; every second sequence of a
    ragged batch brings one token."""
    n, query, prefix = case["sequences"], case["query"], case["prefix"]
    if n == 1:
        return [query], [prefix]
    step = 1
    while step * step < n or math.gcd(step, n) != 1:
        step += 1
    at = [(b * step) % n for b in range(n)]
    before = [prefix * a // (n - 1) for a in at]
    new = [query] * n
    if case["ragged"]:
        new = [1 if b % 2 else 1 + (query - 1) * (n - 1 - b) // (n - 1) for b in range(n)]
    return new, before


class _Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda")

    def norm_weight(self, size):
        return 1.0 + 0.2 * self.normal(size)

    def codes(self, *shape):
        """8-bit values as a page's quantised normal values are spread."""
        x = torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float16)
        return x.mul_(35.0).clamp_(-127, 127).to(torch.int8)

    def choice(self, values, count, dtype):
        i = torch.randint(0, len(values), (count,), generator=self.gen, device="cuda")
        return torch.tensor(values, device="cuda", dtype=dtype)[i]


def _i32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _prepare_pages(case, r, s):
    """The page pool, the sequences' tables and the batch's bounds."""
    new, before = _batch(case)
    kv, d, pt = case["kv_heads"], case["head_dim"], case["page_tokens"]
    lengths = [a + b for a, b in zip(new, before)]
    counts = [-(-l // pt) for l in lengths]
    pages, width = sum(counts) + 3, max(counts)
    order = torch.randperm(pages, generator=r.gen, device="cuda").int()
    table = torch.full((len(new), width), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    touched = [(b, p) for b in range(len(new))
               for p in range(before[b] // pt, (lengths[b] - 1) // pt + 1)]
    at = torch.tensor(touched, device="cuda")
    s.update(keys=r.codes(pages, kv, pt, d), values=r.codes(pages, kv, pt // 8, d, 8),
             key_scales=0.03 * torch.exp(0.3 * r.normal(pages, kv)),
             value_scales=0.03 * torch.exp(0.3 * r.normal(pages, kv)), table=table,
             starts=_i32(starts), lengths=_i32(lengths), tokens=starts[-1], pages=pages,
             width=width, max_query=max(new), max_keys=max(lengths),
             touched=table[at[:, 0], at[:, 1]].contiguous())


def prepare(case, seed):
    ctx = _ctx() if own else None
    r = _Inputs(seed)
    s = {"case": case, "ctx": ctx}
    if case["kind"] == "sample":
        rows, size = case["rows"], case["size"]
        logits = case["spread"] * r.normal(rows, size)
        # A few likely tokens stand out, as a model's do.
        likely = torch.randint(0, size, (rows, 24), generator=r.gen, device="cuda")
        logits.scatter_add_(1, likely, 10.0 * r.uniform(rows, 24))
        filters = case["filters"]
        if filters == "mixed":
            s.update(temperature=r.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], rows, torch.float32),
                     top_k=r.choice([0, 1, 20, 50, 1000], rows, torch.int32),
                     top_p=r.choice([0.8, 0.95, 1.0], rows, torch.float32),
                     min_p=r.choice([0.0, 0.0, 0.05], rows, torch.float32))
        elif filters == "nucleus":
            s.update(temperature=torch.full((rows,), 0.8, device="cuda"), top_k=None,
                     top_p=torch.full((rows,), 0.95, device="cuda"), min_p=None)
        else:
            s.update(temperature=None, top_k=None, top_p=None, min_p=None)
        s.update(logits=logits, uniforms=r.uniform(rows),
                 token=torch.empty(rows, device="cuda", dtype=torch.int32),
                 probability=torch.empty(rows, device="cuda"))
    else:
        _prepare_pages(case, r, s)
        t, kv, d = s["tokens"], case["kv_heads"], case["head_dim"]
        heads = kv * case["group"]
        if case["kind"] == "append":
            pt, n = case["page_tokens"], s["touched"].numel()
            s.update(q_gate=r.normal(t, heads, 2, d), key=r.normal(t, kv, d),
                     value=r.normal(t, kv, d), q_norm=r.norm_weight(d), k_norm=r.norm_weight(d),
                     query=torch.empty(t, heads, d, device="cuda"),
                     gate=torch.empty(t, heads, d, device="cuda"),
                     key_rows=torch.empty(n, pt, kv, d, device="cuda", dtype=torch.float16),
                     value_rows=torch.empty(n, pt, kv, d, device="cuda", dtype=torch.float16))
        else:
            kind = torch.float16 if case["f16"] else torch.float32
            s.update(query=(2.0 * r.normal(t, heads, d)).to(kind),
                     gate=None if case["f16"] else r.normal(t, heads, d),
                     out=torch.empty(t, heads, d, device="cuda", dtype=kind))
    if own:
        kh = _library()
        s["view"] = {k: kh.as_buffer(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if case["kind"] != "sample":
            b = s["view"]
            s["cache"] = kh.PagedQ8Cache(b["keys"], b["values"], b["key_scales"],
                                         b["value_scales"], s["pages"], case["page_tokens"],
                                         case["kv_heads"], case["head_dim"])
            s["batch"] = kh.PagedBatch(b["table"], b["starts"], b["lengths"], case["sequences"],
                                       s["width"], s["tokens"], s["max_query"], s["max_keys"])
    return s


def _rope_dims(case):
    return min(64, case["head_dim"])


# --------------------------------------------------------------------- run ---


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[kind](s)


def _own_append(s):
    c, ctx, b = s["case"], s["ctx"], s["view"]
    ctx.qwen35_attention_prologue_paged_q8_kv(
        b["q_gate"], b["key"], b["value"], b["q_norm"], b["k_norm"], None, s["cache"], s["batch"],
        c["kv_heads"] * c["group"], _rope_dims(c), *SECTIONS, THETA, EPS, b["query"], b["gate"])
    ctx.dequantize_kv_pages_q8_f16(s["cache"], b["touched"], s["touched"].numel(), b["key_rows"],
                                   b["value_rows"])
    return {k: s[k] for k in ("query", "gate", "key_rows", "value_rows")}


def _own_attend(s):
    c, ctx, b = s["case"], s["ctx"], s["view"]
    heads = c["kv_heads"] * c["group"]
    if c["f16"]:
        ctx.attention_f16q_paged_q8_kv(b["query"], s["cache"], s["batch"], heads, b["out"])
    else:
        ctx.attention_f32_paged_q8_kv(b["query"], b["gate"], s["cache"], s["batch"], heads,
                                      b["out"])
    return s["out"]


def _own_sample(s):
    c, b = s["case"], s["view"]
    s["ctx"].sample_f32_i32(b["logits"], c["rows"], c["size"], c["size"], b.get("temperature"),
                            b.get("top_k"), b.get("top_p"), b.get("min_p"), b["uniforms"],
                            b["token"], b["probability"])
    return {"token": s["token"], "probability": s["probability"]}


# ------------------------------------------------------------- plain forms ---


def _norm_rope(x, weight, positions, n):
    """RMSNorm with a weight, then the rotation of pairs (i, i + n / 2) of the
    first n elements, the angles in 64 bits.  x [tokens][heads][dim]."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    pair = torch.arange(n // 2, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * THETA ** (-2.0 * pair / n)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :n // 2], x[..., n // 2:n]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., n:]], -1)


def _token_sequence(s):
    """The sequence of each token, and the token's position in it."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].contiguous(), t.int(), right=True)
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1]).long()
    return seq, first[seq] + t - s["starts"].long()[seq]


def _quantise(rows, fresh, codes, scales, new, old):
    """New rows into their pages.  rows f32 and codes [pages][tokens][heads][dim],
    new and old [pages][tokens] truth values, fresh [pages], scales
    [pages][heads]: a fresh page's scale is its new rows' largest magnitude /
    127; one that holds older rows keeps its scale, doubled as often as the new
    rows need, and its older rows' codes follow."""
    largest = torch.where(new[..., None, None], rows.abs(), 0.0).amax((1, 3))
    steps = torch.ceil(torch.log2(largest.double() / (127.0 * scales.double()))).clamp(min=0)
    # log2 may miss by a rounding next to a power of two.
    short = largest.double() > 127.0 * scales.double() * torch.exp2(steps)
    over = (steps > 0) & (largest.double() <= 127.0 * scales.double() * torch.exp2(steps - 1))
    steps = steps + short.double() - over.double()
    grown = (scales.double() * torch.exp2(steps)).float()
    scale = torch.where(fresh[:, None], largest / 127.0, grown)
    shifted = torch.round(codes.double() * torch.exp2(-steps)[:, None, :, None])
    quantised = torch.round(rows / scale[:, None, :, None]).clamp(-127, 127)
    keep = torch.where((old & ~fresh[:, None])[..., None, None], shifted, codes.double())
    return torch.where(new[..., None, None], quantised.double(), keep).to(torch.int8), scale


def _plain_append(s):
    c = s["case"]
    pt, kv, d, n = c["page_tokens"], c["kv_heads"], c["head_dim"], _rope_dims(c)
    seq, position = _token_sequence(s)
    query = _norm_rope(s["q_gate"][:, :, 0], s["q_norm"], position, n)
    key = _norm_rope(s["key"], s["k_norm"], position, n)
    # Every page that the batch may touch: [sequences * spans] pages of pt slots.
    spans = (s["max_query"] + pt - 2) // pt + 1
    first = (s["lengths"] - s["starts"][1:] + s["starts"][:-1]).long()
    page = first[:, None] // pt + torch.arange(spans, device="cuda")
    slot = page[..., None] * pt + torch.arange(pt, device="cuda")
    new = (slot >= first[:, None, None]) & (slot < s["lengths"].long()[:, None, None])
    old = slot < first[:, None, None]
    token = (s["starts"].long()[:-1, None, None] + slot - first[:, None, None])
    token = token.clamp(0, s["tokens"] - 1).view(-1, pt)
    ids = s["table"].gather(1, page.clamp(max=s["width"] - 1)).long().clamp(min=0).view(-1)
    # A span past a sequence's last page repeats its first one, which always has a new row.
    used = new.any(-1)
    repeat = torch.where(used, torch.arange(spans, device="cuda"), 0)
    repeat = (repeat + spans * torch.arange(len(first), device="cuda")[:, None]).view(-1)
    ids, token = ids[repeat], token[repeat]
    new, old = new.view(-1, pt)[repeat], old.view(-1, pt)[repeat]
    fresh = ~old.any(-1)
    codes, scale = _quantise(key[token], fresh, s["keys"][ids].transpose(1, 2),
                             s["key_scales"][ids], new, old)
    s["keys"][ids] = codes.transpose(1, 2)
    s["key_scales"][ids] = scale
    held = s["values"][ids].permute(0, 2, 4, 1, 3).reshape(-1, pt, kv, d)
    codes, scale = _quantise(s["value"][token], fresh, held, s["value_scales"][ids], new, old)
    s["values"][ids] = codes.view(-1, pt // 8, 8, kv, d).permute(0, 3, 1, 4, 2)
    s["value_scales"][ids] = scale
    at = s["touched"].long()
    keys, values = _rows(s, at)
    return {"query": query, "gate": s["q_gate"][:, :, 1].contiguous(), "key_rows": keys.half(),
            "value_rows": values.half()}


def _rows(s, at):
    """The values that the pages at[...] stand for, [...][page_tokens][kv_heads][dim]."""
    keys = s["keys"][at].float() * s["key_scales"][at][..., None, None]
    values = s["values"][at].float() * s["value_scales"][at][..., None, None, None]
    return keys.transpose(-3, -2).contiguous(), _unpack(values)


def _unpack(values):
    """[...][kv_heads][octets][dim][8] -> [...][octets * 8][kv_heads][dim]."""
    n = values.dim()
    lead = list(range(n - 4))
    moved = values.permute(*lead, n - 3, n - 1, n - 4, n - 2)
    return moved.reshape(*values.shape[:n - 4], -1, values.shape[n - 4], values.shape[n - 2])


def _plain_attend(s):
    c = s["case"]
    kv, g, d, n = c["kv_heads"], c["group"], c["head_dim"], c["sequences"]
    seq, position = _token_sequence(s)
    within = torch.arange(s["tokens"], device="cuda") - s["starts"].long()[seq]
    padded = torch.zeros(n, s["max_query"], kv, g, d, device="cuda")
    padded[seq, within] = s["query"].float().view(-1, kv, g, d)
    padded = padded.transpose(1, 2).reshape(n, kv, -1, d)
    last = torch.full((n, s["max_query"]), -1, device="cuda", dtype=torch.int64)
    last[seq, within] = position
    keys, values = _rows(s, s["table"].long().clamp(min=0))
    keys = keys.view(n, -1, kv, d).transpose(1, 2).contiguous()
    scores = torch.matmul(padded, keys.transpose(2, 3)) / math.sqrt(d)
    del keys
    number = torch.arange(scores.shape[-1], device="cuda")
    masked = number > last.repeat_interleave(g, 1)[:, None, :, None]
    scores = scores.masked_fill_(masked, -1e30)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    values = values.view(n, -1, kv, d).transpose(1, 2).contiguous()
    out = torch.matmul(weights, values).view(n, kv, -1, g, d).transpose(1, 2)
    out = out[seq, within].reshape(-1, kv * g, d)
    if s["gate"] is not None:
        out = out * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return out.to(s["out"].dtype)


def _plain_sample(s):
    """In 64 bits: a cut or a draw next to a border has to fall on its side."""
    logits = s["logits"]
    rows, size = logits.shape

    def of(name, default):
        return (s[name].double() if s[name] is not None
                else torch.full((rows,), default, device="cuda", dtype=torch.float64))[:, None]

    temperature, top_k, top_p, min_p = (of("temperature", 1.0), of("top_k", 0.0),
                                        of("top_p", 1.0), of("min_p", 0.0))
    greedy = temperature[:, 0] <= 0
    ranked, index = torch.sort(logits, dim=1, descending=True, stable=True)
    z = ranked.double() - ranked[:, :1].double()
    weight = torch.exp(z / torch.where(temperature > 0, temperature, 1.0))
    rank = torch.arange(size, device="cuda")[None]
    weight = torch.where((top_k <= 0) | (rank < top_k), weight, 0.0)
    total = torch.cumsum(weight, 1)
    before = total - weight
    keep = ((top_p >= 1) | (before < top_p * total[:, -1:])) & (weight > 0) & (weight >= min_p)
    keep = keep | (rank == 0)
    kept = torch.zeros_like(weight).scatter_(1, index, torch.where(keep, weight, 0.0))
    sums = torch.cumsum(kept, 1)
    target = s["uniforms"].double()[:, None] * sums[:, -1:]
    token = (sums <= target).sum(1).clamp(max=size - 1)
    token = torch.where(greedy, index[:, 0], token)
    probability = kept.gather(1, token[:, None])[:, 0] / sums[:, -1]
    return {"token": token.int(),
            "probability": torch.where(greedy, 1.0, probability).float()}


# -------------------------------------------------------------------- work ---


def work(case):
    if case["kind"] == "sample":
        # Every logit once; a subtraction, an exponential and a sum for each.
        n = case["rows"] * case["size"]
        return {"bytes": 4 * n + 32 * case["rows"], "flops": 3 * n}
    new, before = _batch(case)
    t, kv, d, pt = sum(new), case["kv_heads"], case["head_dim"], case["page_tokens"]
    heads = kv * case["group"]
    if case["kind"] == "append":
        touched = sum((a + b - 1) // pt - b // pt + 1 for a, b in zip(new, before))
        # Rows in, query and gate out, codes out; the touched pages read back.
        bytes_ = 4 * t * d * (4 * heads + 2 * kv) + 2 * t * kv * d
        bytes_ += touched * 2 * kv * pt * d * 3
        return {"bytes": bytes_, "flops": t * d * (4 * heads + 8 * kv)}
    keys = sum(a + b for a, b in zip(new, before))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, before))
    size = 2 if case["f16"] else 4
    rows = t * heads * d * size * (2 if case["f16"] else 3)
    return {"bytes": 2 * keys * kv * d + 8 * kv * (keys // pt) + rows,
            "flops": 4 * heads * d * pairs}


# ------------------------------------------------------------------- exact ---


def exact(case, seed):
    """From the definitions, sequence by sequence, in 64 bits."""
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["kind"]](s)


def _exact_page(s, name, page):
    """One page's values in 64 bits, [page_tokens][kv_heads][dim]."""
    codes, scale = s[name + "s"][page].double(), s[name + "_scales"][page].double()
    if name == "key":
        return torch.einsum("htd,h->thd", codes, scale)
    return torch.einsum("hodt,h->othd", codes, scale).flatten(0, 1)


def _exact_rotate(x, weight, first, n):
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
    out = x.clone()
    at = torch.arange(first, first + x.shape[0], device=x.device, dtype=torch.float64)
    for i in range(n // 2):
        a = (at * math.pow(THETA, -2.0 * i / n))[:, None]
        u, v = x[..., i], x[..., i + n // 2]
        out[..., i] = u * torch.cos(a) - v * torch.sin(a)
        out[..., i + n // 2] = v * torch.cos(a) + u * torch.sin(a)
    return out


def _exact_append(s):
    c = s["case"]
    pt, n = c["page_tokens"], _rope_dims(c)
    new, before = _batch(c)
    table = s["table"].tolist()
    query, keys, values, at = [], [], [], 0
    for b, (q, p) in enumerate(zip(new, before)):
        span = slice(at, at + q)
        at += q
        query.append(_exact_rotate(s["q_gate"][span, :, 0], s["q_norm"], p, n))
        rows = {"key": _exact_rotate(s["key"][span], s["k_norm"], p, n),
                "value": s["value"][span].double()}
        for page in range(p // pt, (p + q - 1) // pt + 1):
            lo, hi = max(p, page * pt), min(p + q, (page + 1) * pt)
            for name, out in (("key", keys), ("value", values)):
                held = s[name + "s"][table[b][page]].double()
                held = (held.transpose(0, 1) if name == "key"
                        else held.permute(1, 3, 0, 2).flatten(0, 1)).clone()
                fresh = rows[name][lo - p:hi - p]
                scale = s[name + "_scales"][table[b][page]].double()
                for h in range(c["kv_heads"]):
                    largest = float(fresh[:, h].abs().max())
                    if lo == page * pt:
                        step = largest / 127.0
                    else:
                        step = float(scale[h])
                        while largest > 127.0 * step:
                            step *= 2.0
                            held[:lo - page * pt, h] *= 0.5
                        held[:lo - page * pt, h] = torch.round(held[:lo - page * pt, h])
                    held[lo - page * pt:hi - page * pt, h] = torch.round(fresh[:, h] / step)
                    held[:, h] *= step
                out.append(held)
    return {"query": torch.cat(query), "gate": s["q_gate"][:, :, 1].double(),
            "key_rows": torch.stack(keys), "value_rows": torch.stack(values)}


def _exact_attend(s):
    c = s["case"]
    g, d = c["group"], c["head_dim"]
    new, before = _batch(c)
    out, at = [], 0
    for b, (q, p) in enumerate(zip(new, before)):
        ids = s["table"][b, :-(-(p + q) // c["page_tokens"])].long()
        k = torch.einsum("phtd,ph->phtd", s["keys"][ids].double(), s["key_scales"][ids].double())
        v = torch.einsum("phodt,ph->photd", s["values"][ids].double(),
                         s["value_scales"][ids].double())
        rows = []
        for h in range(c["kv_heads"]):
            kh = k[:, h].reshape(-1, d)[:p + q]
            vh = v[:, h].reshape(-1, d)[:p + q]
            x = s["query"][at:at + q, h * g:(h + 1) * g].double().reshape(q * g, d)
            w = x @ kh.T.contiguous() / math.sqrt(d)
            limit = p + torch.arange(q, device=w.device).repeat_interleave(g)
            w = w.masked_fill(torch.arange(p + q, device=w.device) > limit[:, None], -math.inf)
            rows.append((torch.softmax(w, -1) @ vh).view(q, g, d))
        out.append(torch.cat(rows, 1))
        at += q
    out = torch.cat(out)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_sample(s):
    """Row by row; the token is a whole number and has no 64-bit value beside it."""
    found = []
    for r, row in enumerate(s["logits"].double()):
        t, k, p, m = (float(s[n][r]) if s[n] is not None else v for n, v in (
            ("temperature", 1.0), ("top_k", 0.0), ("top_p", 1.0), ("min_p", 0.0)))
        if t <= 0:
            found.append(1.0)
            continue
        w = torch.exp((row - row.max()) / t)
        order = torch.argsort(row, descending=True, stable=True)
        if k > 0:
            order = order[:int(k)]
        sums = torch.cumsum(w[order], 0)
        count = len(order)
        if p < 1:
            count = max(1, int((sums < p * sums[-1]).sum()) + 1)
        if m > 0:
            count = max(1, min(count, int((w[order] >= m).sum())))
        kept = torch.sort(order[:count]).values
        sums = torch.cumsum(w[kept], 0)
        at = min(int((sums <= float(s["uniforms"][r]) * sums[-1]).sum()), count - 1)
        found.append(float(w[kept[at]] / sums[-1]))
    return {"token": None, "probability": torch.tensor(found, dtype=torch.float64)}
