"""More operators around a paged key/value cache: norms of queries and keys with the rotary append, attention through a sliding
window, and a cache held in 4 bits (append, attention, read).

``listed()`` names fixed cases, ``draw(rng)`` samples further ones from the same ranges.  A case is a dict of plain values;
its ``kind`` selects the operator:

* ``append``   ``torch.ops.flashllm.norm_rotary_append``: the output of a QKV projection to normed and turned queries, keys and
               values in an fp16 cache.
* ``window``   ``torch.ops.flashllm.window_attention``: causal attention of a ragged batch, through a window and with the first
               positions (sinks) always in sight.
* ``append4``  ``torch.ops.flashllm.four_bit_append``: the append into a cache of 4 bits, norms optional.  What the codes stand
               for comes back through ``four_bit_read``.
* ``attend4``  ``torch.ops.flashllm.four_bit_attention``: attention over such a cache, window optional.
* ``read4``    ``torch.ops.flashllm.four_bit_read``: rows of a batch from such a cache.

A cache of 4 bits is uint8 ``[pages][kv_heads][page_size][head_dim * 9 / 16]``.  What a head keeps of a page, page_size times
that many bytes in one piece, begins with the codes ``[page_size][head_dim / 2]``, two to a byte, the even element in the low
bits; behind them ``[page_size][head_dim / 64][2]`` fp16: step and lowest value of each 64 elements.  An element is
lowest + step * code, with lowest = fp16(min), step = fp16((max - lowest) / 15), code = (x - lowest) / step to the nearest.

``run`` computes them from elementary operations in 32 bits (angles, norms and turned keys, whose codes may lie next to a
border, in 64), or, with ``own`` set, through the framework.  Lengths follow from the case alone, everything else from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = torch.device("cuda:0")
GROUP = 64  # elements that share a step

DEFAULTS = {
    "append": {"rotary": 128, "interleaved": False, "scaling": "none"},
    "append4": {"rotary": 64, "interleaved": False, "scaling": "none", "norm": False},
    "window": {"cap": 0.0, "slopes": False, "window": 1024, "sinks": 4},
    "attend4": {"cap": 0.0, "slopes": False, "window": 0, "sinks": 0},
    "read4": {},
}


def _case(kind, name, seqs, tokens, context, heads, kv_heads, head_dim, page, **more):
    return {"kind": kind, "name": name, "seqs": seqs, "tokens_min": tokens[0], "tokens_max": tokens[1],
            "context_min": context[0], "context_max": context[1], "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lengths": 1, **DEFAULTS[kind], **more}


def listed():
    return [
        # One decoding step of a small batch: 16 rows, the latency of a launch.
        _case("append", "norm append decode b16", 16, (1, 1), (200, 4000), 32, 8, 128, 64),
        # Prompts, half of each head rotated, for contexts stretched fourfold: bound by bytes.
        _case("append", "norm append prompts", 9, (150, 2000), (0, 300), 40, 8, 128, 128, rotary=64, interleaved=True,
              scaling="by parts"),
        # Decoding of a large ragged batch in a layer with a window: a few tiles of keys for each sequence.
        _case("window", "window decode b64", 64, (1, 1), (100, 9000), 32, 8, 128, 64),
        # One long prompt in such a layer: a band of the scores, bound by the tensor cores.
        _case("window", "window prompt 7000", 1, (7000, 7000), (0, 0), 32, 8, 128, 128, window=2048, sinks=16),
        # One decoding step of a small batch into a cache of 4 bits.
        _case("append4", "four bit append decode b16", 16, (1, 1), (200, 4000), 32, 8, 128, 64, rotary=128, norm=True),
        # Prompts of usual and odd lengths into a cache of 4 bits.
        _case("append4", "four bit append prompts", 12, (20, 3000), (0, 0), 40, 8, 64, 64),
        # One user, a short context: latency.
        _case("attend4", "four bit decode b1", 1, (1, 1), (210, 210), 16, 16, 64, 16),
        # Ordinary decoding of a large ragged batch.
        _case("attend4", "four bit decode b64", 64, (1, 1), (100, 9000), 32, 8, 128, 64),
        # Long ragged contexts, eight queries to a key: what 4 bits are for, bound by the cache's bytes.
        _case("attend4", "four bit decode long b16", 16, (1, 1), (4000, 40000), 64, 8, 128, 128),
        # Long questions behind long contexts through a window, scores capped: bound by the tensor cores.
        _case("attend4", "four bit prompts window cap", 3, (1000, 3000), (500, 5000), 16, 4, 128, 256, cap=50.0, window=4096,
              sinks=4),
        # One short sequence handed to a worker that keeps 16 bits.
        _case("read4", "four bit read b1", 1, (225, 225), (0, 0), 16, 16, 64, 16),
        # Long sequences handed over at once.
        _case("read4", "four bit read long b8", 8, (4000, 40000), (0, 0), 8, 8, 128, 128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(lo, 0.7)), math.log(hi + 0.99))))))


def _lengths(case):
    """(context, tokens) of each sequence, spread over the logarithm."""
    rng = random.Random(case["lengths"])
    return ([_log_int(rng, case["context_min"], case["context_max"]) if case["context_max"] else 0 for _ in range(case["seqs"])],
            [_log_int(rng, case["tokens_min"], case["tokens_max"]) for _ in range(case["seqs"])])


def draw(rng):
    kind = rng.choices(("append", "window", "append4", "attend4", "read4"), (2, 4, 2, 5, 1))[0]
    most = [work(c) for c in listed() if c["kind"] == kind]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        dim, kv_heads = rng.choice((64, 128, 128)), rng.choice((1, 2, 4, 5, 8, 8, 12, 20, 32))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8))
        page = rng.choice((16, 32, 64, 128, 256))
        seqs = _log_int(rng, 1, 64)
        context = sorted(_log_int(rng, 0, 40000) for _ in range(2))
        if kind in ("append", "append4"):
            tokens = sorted(_log_int(rng, 1, 2000) for _ in range(2))
            more = {"rotary": rng.choice((16, 32, 64, dim)), "interleaved": rng.random() < 0.5,
                    "scaling": rng.choice(("none", "linear", "by parts"))}
            if kind == "append4":
                more["norm"] = rng.random() < 0.5
            context = [c % 2000 for c in context]
        elif kind == "read4":
            tokens, more = sorted(_log_int(rng, 1, 40000) for _ in range(2)), {}
        else:
            tokens = sorted(_log_int(rng, 1, 7000) for _ in range(2)) if rng.random() < 0.6 else [1, 1]
            more = {"cap": rng.choice((0.0, 0.0, round(rng.uniform(10, 60), 1))), "slopes": rng.random() < 0.3}
            if kind == "window" or rng.random() < 0.4:
                more.update(window=_log_int(rng, 1, 8000), sinks=rng.choice((0, 1, 4, 4, 16, 100)))
        case = _case(kind, "", seqs, tokens, sorted(context), heads, kv_heads, dim, page, **more)
        del case["name"]
        case["lengths"] = rng.randrange(1 << 20)
        contexts, counts = _lengths(case)
        # What the plain form holds at a time: scores of every head, padded to the longest sequence.
        padded = seqs * max(counts) * heads * (max(contexts) + max(counts)) if kind in ("window", "attend4") else 0
        size = seqs * (max(contexts) + max(counts) + page) * kv_heads * dim
        w = work(case)
        if padded <= 1.7e9 and size <= 8e8 and w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


# --------------------------------------------------------------------------------------------------- inputs

def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(torch.float16)


def _frequencies(case):
    """Angle per position of each pair, and the factor on the rotated values.  "linear": positions squeezed eightfold; "by
    parts": a context stretched fourfold from 2048, fast pairs kept, slow ones squeezed, a ramp between (1 to 32 turns)."""
    rotary = case["rotary"]
    f = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if case["scaling"] == "linear":
        return f / 8, 1.0
    if case["scaling"] == "by parts":
        keep = ((2048 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f * keep + f / 4 * (1 - keep), 0.1 * math.log(4) + 1
    return f, 1.0


def _to_codes(x):
    """x [..][dim] to codes [..][dim / 64][64], steps and lowest values [..][dim / 64] (fp16 values in x's type)."""
    x = x.unflatten(-1, (-1, GROUP))
    low = x.amin(-1).half().to(x.dtype)
    step = ((x.amax(-1) - low) / torch.full_like(low, 15.0)).half().to(x.dtype)
    code = torch.where(step[..., None] > 0, ((x - low[..., None]) / step[..., None]).round().clamp(0, 15), 0.0)
    return code, step, low


def _page_parts(cache, dim):
    """Views of a 4-bit cache: codes [pages][heads][page][dim / 2] and scales [pages][heads][page][dim / 64][2]."""
    pages, heads, page, _ = cache.shape
    flat = cache.view(pages, heads, -1)
    return (flat[..., :page * dim // 2].unflatten(-1, (page, dim // 2)),
            flat[..., page * dim // 2:].unflatten(-1, (page, -1)).view(torch.float16).unflatten(-1, (-1, 2)))


def _put_codes(cache, dim, at, x):
    """Stores x [..][dim] at the places `at` of the cache; what the codes stand for."""
    code, step, low = _to_codes(x)
    flat = code.flatten(-2).to(torch.uint8)
    codes, scales = _page_parts(cache, dim)
    codes[at] = flat[..., 0::2] | flat[..., 1::2] << 4
    scales[at] = torch.stack([step, low], -1).half()
    return (low[..., None] + step[..., None] * code).flatten(-2)


def _values(cache, dim, at, dtype):
    """What lies at the places `at` of the cache: [..][dim]."""
    codes, scales = (part[at] for part in _page_parts(cache, dim))
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dtype).unflatten(-1, (-1, GROUP))
    scales = scales.to(dtype)
    return (scales[..., 1:] + scales[..., :1] * code).flatten(-2)


def _random_codes(gen, pages, heads, page, dim):
    cache = torch.empty((pages, heads, page, dim * 9 // 16), dtype=torch.uint8, device=DEVICE)
    at_once = max(1, (1 << 26) // (heads * page * dim))
    for p in range(0, pages, at_once):
        n = min(at_once, pages - p)
        _put_codes(cache[p:p + n], dim, ..., torch.randn((n, heads, page, dim), generator=gen, device=DEVICE))
    return cache


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, heads, kv_heads, dim, page = (case[k] for k in ("kind", "heads", "kv_heads", "head_dim", "page"))
    contexts, counts = _lengths(case)
    pages = [-(-(c + t) // page) for c, t in zip(contexts, counts)]
    order = torch.randperm(sum(pages), generator=gen, device=DEVICE).to(torch.int32).split(pages)
    first = [sum(counts[:b]) for b in range(len(counts) + 1)]
    rows = first[-1]
    make = _random_codes if kind in ("append4", "attend4", "read4") else _randn
    state = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows,
             "longest": max(c + t for c, t in zip(contexts, counts)), "most": max(counts),
             "cu_tokens": _int(first), "context": _int(contexts), "counts": _int(counts),
             "page_table": torch.nn.utils.rnn.pad_sequence(list(order), batch_first=True),
             "k_cache": make(gen, sum(pages), kv_heads, page, dim), "v_cache": make(gen, sum(pages), kv_heads, page, dim)}
    if kind in ("append", "append4"):
        frequencies, magnitude = _frequencies(case)
        shape = (rows, (heads + 2 * kv_heads) * dim)
        # For 4 bits spread evenly: a step is then small against the values, and with it what a code is off that lies next to a
        # border and falls to the other side.
        qkv = (3.4 * torch.rand(shape, generator=gen, device=DEVICE) - 1.7).half() if kind == "append4" else _randn(gen, *shape)
        weights = (torch.rand((2, dim), generator=gen, device=DEVICE) * 0.2 + 0.9).half() if case.get("norm", True) else (None, None)
        state.update(qkv=qkv, frequencies=frequencies.to(DEVICE), magnitude=magnitude, interleaved=case["interleaved"],
                     q_norm=weights[0], k_norm=weights[1])
    elif kind != "read4":
        # Heads differ in how sharply they look: scores between 0.5 and 3 standard deviations.
        gain = torch.logspace(math.log10(0.5), math.log10(3.0), heads, device=DEVICE).view(1, heads, 1)
        q = (torch.randn((rows, heads, dim), generator=gen, device=DEVICE) * gain).to(torch.float16)
        slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device=DEVICE) / heads)
        state.update(q=q.view(rows, heads * dim), cap=case["cap"], slopes=slopes if case["slopes"] else None,
                     window=case["window"], sinks=case["sinks"])
    return state


# --------------------------------------------------------------------------------------------------- one pass

EPS = 1e-6


def _own(s):
    import flash_llm_b200.torch_op  # noqa: F401  (registers torch.ops.flashllm)
    ops = torch.ops.flashllm
    batch = (s["k_cache"], s["v_cache"], s["cu_tokens"], s["context"], s["page_table"])
    if s["kind"] == "append":
        q = ops.norm_rotary_append(s["qkv"], *batch, s["q_norm"], s["k_norm"], EPS, s["frequencies"], s["interleaved"],
                                   s["magnitude"])
        return q, s["k_cache"], s["v_cache"]
    if s["kind"] == "append4":
        q = ops.four_bit_append(s["qkv"], *batch, s["q_norm"], s["k_norm"], EPS, s["frequencies"], s["interleaved"], s["magnitude"])
        return (q, *ops.four_bit_read(*batch, s["rows"]))
    if s["kind"] == "read4":
        return ops.four_bit_read(*batch, s["rows"])
    if s["kind"] == "window":
        return ops.window_attention(s["q"], *batch, s["window"], s["sinks"], cap=s["cap"], slopes=s["slopes"])
    return ops.four_bit_attention(s["q"], *batch, s["window"], s["sinks"], cap=s["cap"], slopes=s["slopes"])


def _places(s):
    """(position, page, place in the page) of the batch's rows."""
    row = torch.arange(s["rows"], device=DEVICE)
    sequence = torch.searchsorted(s["cu_tokens"].long(), row, right=True) - 1
    position = s["context"][sequence].long() + row - s["cu_tokens"][sequence]
    return position, s["page_table"][sequence, position // s["page"]].long(), position % s["page"]


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _plain_append(s):
    position, page, place = _places(s)
    four = s["kind"] == "append4"
    angle = position.double()[:, None] * s["frequencies"]
    # Keys of 4 bits in 64: a code may lie next to a border.
    x = s["qkv"].to(torch.float64 if four else torch.float32).view(s["rows"], -1, s["dim"])
    c, d = ((f(angle) * s["magnitude"]).to(x.dtype)[:, None, :] for f in (torch.cos, torch.sin))
    q, k, v = x.split([s["heads"], s["kv_heads"], s["kv_heads"]], 1)
    turned = torch.cat([_normed(q, s["q_norm"]), _normed(k, s["k_norm"])], 1)
    pairs = s["frequencies"].numel()
    y = turned.clone()
    if s["interleaved"]:
        u, w = turned[..., 0:2 * pairs:2], turned[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = u * c - w * d, w * c + u * d
    else:
        u, w = turned[..., :pairs], turned[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = u * c - w * d, w * c + u * d
    q, k = y.split([s["heads"], s["kv_heads"]], 1)
    q = q.reshape(s["rows"], -1).half()
    at = (page, slice(None), place)
    if four:
        # The values are exact in 32 bits: so are their codes there.
        kept = [_put_codes(s["k_cache"], s["dim"], at, k), _put_codes(s["v_cache"], s["dim"], at, v.float())]
        return (q, *(t.reshape(s["rows"], -1).half() for t in kept))
    s["k_cache"][at] = k.half()
    s["v_cache"][at] = v.half()
    return q, s["k_cache"], s["v_cache"]


def _plain_read(s):
    _, page, place = _places(s)
    return tuple(_values(s[c], s["dim"], (page, slice(None), place), torch.float32).reshape(s["rows"], -1).half()
                 for c in ("k_cache", "v_cache"))


def _plain_attention(s):
    heads, kv_heads, dim, longest, most = s["heads"], s["kv_heads"], s["dim"], s["longest"], s["most"]
    seqs = s["counts"].numel()
    column, line = torch.arange(longest, device=DEVICE), torch.arange(most, device=DEVICE)
    start, context = s["cu_tokens"][:-1, None], s["context"][:, None]
    there = line < s["counts"][:, None]                                                     # [B][T]
    row = (start + line).clamp(max=s["rows"] - 1)
    length = context + s["counts"][:, None]
    page = s["page_table"][:, (column // s["page"]).clamp(max=s["page_table"].shape[1] - 1)].long()
    at = (page, slice(None), column % s["page"])
    if s["kind"] == "attend4":
        k, v = (_values(s[c], dim, at, torch.float32).transpose(1, 2) for c in ("k_cache", "v_cache"))
    else:
        k, v = (s[c][at].float().transpose(1, 2) for c in ("k_cache", "v_cache"))           # [B][Hkv][L][D]
    v = v * (column < length)[:, None, :, None]
    q = s["q"][row].float().view(seqs, most, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).view(seqs, heads, most, longest)
    score *= 1 / math.sqrt(dim)
    if s["cap"] > 0:
        score /= s["cap"]
        score.tanh_()
        score *= s["cap"]
    away = column - (context + line)[:, :, None]                                            # [B][T][L], 0: itself
    if s["slopes"] is not None:
        score += s["slopes"].view(1, heads, 1, 1) * away[:, None].float()
    seen = away <= 0
    if s["window"] > 0:
        seen &= (away > -s["window"]) | (column < s["sinks"])
    score.masked_fill_(~seen[:, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(seqs, kv_heads, -1, longest), v).view(seqs, heads, most, dim) / total
    return out.transpose(1, 2)[there].reshape(s["rows"], heads * dim).half()


def run(state):
    if own:
        return _own(state)
    if state["kind"] in ("append", "append4"):
        return _plain_append(state)
    if state["kind"] == "read4":
        return _plain_read(state)
    return _plain_attention(state)


# --------------------------------------------------------------------------------------------------- 64 bits

def _exact_rows(cache, used, h, dim, four):
    """One head of the pages `used`, as rows in 64 bits."""
    if not four:
        return cache[used, h].reshape(-1, dim).double()
    page = cache.shape[2]
    raw = cache[used, h].reshape(len(used), -1)
    byte = raw[:, :page * dim // 2].reshape(-1, dim // 2)
    scale = raw[:, page * dim // 2:].contiguous().view(torch.float16).double().view(-1, dim // GROUP, 1, 2)
    code = torch.empty((byte.shape[0], dim), dtype=torch.float64, device=DEVICE)
    code[:, 0::2], code[:, 1::2] = (byte % 16).double(), (byte // 16).double()
    return (code.view(-1, dim // GROUP, GROUP) * scale[..., 0] + scale[..., 1]).view(-1, dim)


def _exact_kept(x):
    """What a head's elements stand for in 4 bits."""
    kept = torch.empty_like(x)
    for g in range(0, x.shape[-1], GROUP):
        part = x[..., g:g + GROUP]
        low = part.min(-1, keepdim=True).values.half().double()
        step = ((part.max(-1, keepdim=True).values - low) / 15).half().double()
        kept[..., g:g + GROUP] = low + step * torch.nan_to_num((part - low) / step).round().clamp(0, 15)
    return kept


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    contexts, counts = _lengths(case)
    heads, kv_heads, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    share = heads // kv_heads
    cut = s["cu_tokens"].tolist()
    four = case["kind"] in ("append4", "attend4", "read4")
    if case["kind"] in ("append", "append4"):
        frequencies, magnitude = _frequencies(case)
        frequencies = frequencies.to(DEVICE)
        pairs = frequencies.numel()
        first = torch.arange(pairs, device=DEVICE) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        out = torch.empty((s["rows"], heads * dim), dtype=torch.float64, device=DEVICE)
        shape = (s["rows"], kv_heads * dim)
        caches = ([torch.empty(shape, dtype=torch.float64, device=DEVICE) for _ in range(2)] if four
                  else [s["k_cache"].double(), s["v_cache"].double()])
        for b, (context, count) in enumerate(zip(contexts, counts)):
            place = torch.arange(context, context + count, device=DEVICE)
            turn = torch.polar(torch.full((count, pairs), magnitude, dtype=torch.float64, device=DEVICE),
                               place.double()[:, None] * frequencies)[:, None]
            x = s["qkv"][cut[b]:cut[b + 1]].double().view(count, heads + 2 * kv_heads, dim)
            for lo, hi, weight in ((0, heads, s["q_norm"]), (heads, heads + kv_heads, s["k_norm"])):
                if weight is not None:
                    part = x[:, lo:hi].clone()
                    x[:, lo:hi] = part * weight.double() / (part.square().mean(-1, keepdim=True) + EPS).sqrt()
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[cut[b]:cut[b + 1]] = y[:, :heads].reshape(count, -1)
            keys, values = y[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
            if four:
                for cache, kept in zip(caches, (keys, values)):
                    cache[cut[b]:cut[b + 1]] = _exact_kept(kept).reshape(count, -1)
                continue
            pages = s["page_table"][b].long()[place // page]
            caches[0][pages, :, place % page] = keys
            caches[1][pages, :, place % page] = values
        return out, caches[0], caches[1]
    if case["kind"] == "read4":
        kept = [torch.empty((s["rows"], kv_heads, dim), dtype=torch.float64, device=DEVICE) for _ in range(2)]
        for b, (context, count) in enumerate(zip(contexts, counts)):
            used = s["page_table"][b].long()[:-(-(context + count) // page)]
            for h in range(kv_heads):
                for out, cache in zip(kept, (s["k_cache"], s["v_cache"])):
                    out[cut[b]:cut[b + 1], h] = _exact_rows(cache, used, h, dim, True)[context:context + count]
        return tuple(out.view(s["rows"], -1) for out in kept)
    out = torch.empty((s["rows"], heads, dim), dtype=torch.float64, device=DEVICE)
    window = case["window"] or 1 << 40
    for b, (context, count) in enumerate(zip(contexts, counts)):
        used = s["page_table"][b].long()[:-(-(context + count) // page)]
        place = torch.arange(context, context + count, device=DEVICE)[:, None]
        key = torch.arange(context + count, device=DEVICE)[None]
        seen = (key <= place) & ((place - key < window) | (key < case["sinks"]))
        for h in range(kv_heads):
            k, v = (_exact_rows(s[c], used, h, dim, four)[:context + count] for c in ("k_cache", "v_cache"))
            for i in range(h * share, (h + 1) * share):
                score = s["q"][cut[b]:cut[b + 1], i * dim:(i + 1) * dim].double() @ k.T / math.sqrt(dim)
                if s["cap"] > 0:
                    score = s["cap"] * torch.tanh(score / s["cap"])
                if s["slopes"] is not None:
                    score = score + s["slopes"][i].double() * (key - place).double()
                out[cut[b]:cut[b + 1], i] = torch.softmax(torch.where(seen, score, -math.inf), -1) @ v
    return out.view(s["rows"], heads * dim)


# --------------------------------------------------------------------------------------------------- accounting

def _sight(case, context, count):
    """(pairs of a token and a key that it sees, keys that any of them sees) of a sequence."""
    def upto(n):  # pairs of the first n positions
        window, sinks = case["window"] or 1 << 40, case["sinks"]
        full = min(n, window)
        pairs = full * (full + 1) // 2
        if n > window:
            beyond = n - window
            pairs += beyond * window + min(beyond, sinks) * (min(beyond, sinks) + 1) // 2 + max(0, beyond - sinks) * sinks
        return pairs
    keys = context + count
    if case["window"]:
        hidden = max(0, context + 1 - case["window"])
        keys -= max(0, hidden - case["sinks"])
    return upto(context + count) - upto(context), keys


def work(case):
    """Bytes read and written once; multiply-adds of the pairs of a query and a key that it sees (4 * head size each)."""
    contexts, counts = _lengths(case)
    heads, kv_heads, dim, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(counts)
    kept = 2 * rows * kv_heads * dim  # elements of keys and values
    if case["kind"] == "append":
        return {"bytes": 4 * rows * heads * dim + 4 * kept, "flops": rows * (heads + kv_heads) * (4 * dim + 3 * case["rotary"])}
    if case["kind"] == "append4":  # in and out, and the codes' values
        return {"bytes": 4 * rows * heads * dim + 4 * kept + kept * 9 // 16,
                "flops": rows * (heads + kv_heads) * 3 * case["rotary"] + 6 * kept}
    if case["kind"] == "read4":
        return {"bytes": 2 * kept + kept * 9 // 16, "flops": 2 * kept}
    sight = [_sight(case, c, t) for c, t in zip(contexts, counts)]
    element = 9 / 16 if case["kind"] == "attend4" else 2
    return {"bytes": 4 * rows * heads * dim + 2 * sum(k for _, k in sight) * kv_heads * dim * element,
            "flops": 4 * dim * heads * sum(p for p, _ in sight)}
