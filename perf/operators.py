"""The operators around a paged key/value cache: rotary positions with the append, attention of drafted token trees and of
prompts, and the acceptance of a drafted path.

``listed()`` names fixed cases, ``draw(rng)`` samples further ones from the same ranges.  A case is a dict of plain values;
its ``kind`` selects the operator:

* ``append``  ``torch.ops.flashllm.rotary_append``: the output of a QKV projection to rotated queries, keys and values in the
              cache.
* ``tree``    ``torch.ops.flashllm.tree_attention``: up to 64 drafted tokens of each sequence over its cache.
* ``prompt``  ``torch.ops.flashllm.prompt_attention``: causal attention of a ragged batch over its cache; one token of each
              sequence is ordinary decoding.
* ``accept``  ``torch.ops.flashllm.cache_accept``: keys and values of an accepted path move behind the context.

``run`` computes them from elementary operations in 32 bits, or, with ``own`` set, through the framework.  Lengths follow from
the case alone, everything else from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = torch.device("cuda:0")

DEFAULTS = {
    "append": {"rotary": 128, "interleaved": False, "scaling": "none"},
    "tree": {"cap": 0.0, "slopes": False},
    "prompt": {"cap": 0.0, "slopes": False, "prefix": False},
    "accept": {"layers": 1},
}


def _case(kind, name, seqs, tokens, context, heads, kv_heads, head_dim, page, **more):
    return {"kind": kind, "name": name, "seqs": seqs, "tokens_min": tokens[0], "tokens_max": tokens[1],
            "context_min": context[0], "context_max": context[1], "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "lengths": 1, **DEFAULTS[kind], **more}


def listed():
    return [
        # One decoding step of a small batch: 16 rows, the latency of a launch.
        _case("append", "append decode b16", 16, (1, 1), (200, 4000), 32, 8, 128, 64),
        # Prompts of a hidden-9216 layer (72 heads of 128), half of each head rotated, for contexts stretched fourfold.
        _case("append", "append prompts 9216", 9, (150, 2000), (0, 300), 72, 72, 128, 128, rotary=64, interleaved=True,
              scaling="by parts"),
        # One user, one small tree behind a short context: latency.
        _case("tree", "tree b1 t15", 1, (15, 15), (210, 210), 16, 16, 64, 16),
        # Trees that fill the SpMM's N = 64 in a hidden-9216 layer, contexts up to 2048.
        _case("tree", "tree 9216 b4 t16", 4, (16, 16), (1500, 2031), 72, 72, 128, 64),
        # Long ragged contexts, eight queries to a key: bound by the cache's bytes.
        _case("tree", "tree long b16", 16, (5, 16), (4000, 40000), 64, 8, 128, 128),
        # The largest trees, scores capped and biased by distance.
        _case("tree", "tree t64 cap", 7, (40, 64), (1000, 9000), 32, 8, 128, 32, cap=30.0, slopes=True),
        # Ordinary decoding of a large ragged batch with a distance bias.
        _case("prompt", "decode b64 slopes", 64, (1, 1), (100, 9000), 32, 8, 128, 64, slopes=True),
        # Prompts of usual and odd lengths at once, every document by itself.
        _case("prompt", "prompts ragged", 12, (20, 1500), (0, 0), 40, 8, 64, 64),
        # A short question behind a long context whose prefix is seen from both sides, scores capped.
        _case("prompt", "prompts prefix cap", 3, (300, 700), (500, 5000), 16, 4, 128, 256, cap=50.0, prefix=True),
        # One long prompt.
        _case("prompt", "prompt 7000", 1, (7000, 7000), (0, 0), 32, 8, 128, 128),
        # A tree accepted for one user, a layer at a time.
        _case("accept", "accept b1", 1, (15, 15), (210, 210), 16, 16, 64, 16),
        # A batch of trees accepted in all layers of a model at once.
        _case("accept", "accept b24 l32", 24, (30, 64), (20, 200), 32, 8, 128, 64, layers=32),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(max(lo, 0.7)), math.log(hi + 0.99))))))


def _lengths(case):
    """(context, tokens) of each sequence, spread over the logarithm."""
    rng = random.Random(case["lengths"])
    return ([_log_int(rng, case["context_min"], case["context_max"]) if case["context_max"] else 0 for _ in range(case["seqs"])],
            [_log_int(rng, case["tokens_min"], case["tokens_max"]) for _ in range(case["seqs"])])


def _prefixes(case):
    rng = random.Random(case["lengths"] + 1)
    return [int(c + t * rng.uniform(0.0, 0.9)) for c, t in zip(*_lengths(case))]


def draw(rng):
    kind = rng.choices(("append", "tree", "prompt", "accept"), (2, 4, 4, 1))[0]
    most = [work(c) for c in listed() if c["kind"] == kind]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        dim, kv_heads = rng.choice((64, 128, 128)), rng.choice((1, 2, 4, 5, 8, 8, 12, 20, 32))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8))
        page = rng.choice((16, 32, 64, 128, 256))
        seqs = _log_int(rng, 1, 64)
        context = sorted(_log_int(rng, 0, 40000) for _ in range(2))
        if kind == "append":
            tokens = sorted(_log_int(rng, 1, 2000) for _ in range(2))
            more = {"rotary": rng.choice((16, 32, 64, dim)), "interleaved": rng.random() < 0.5,
                    "scaling": rng.choice(("none", "linear", "by parts"))}
            context = [c % 2000 for c in context]
        elif kind == "tree":
            tokens = sorted(_log_int(rng, 1, 64) for _ in range(2))
            more = {"cap": rng.choice((0.0, 0.0, round(rng.uniform(10, 60), 1))), "slopes": rng.random() < 0.3}
        elif kind == "prompt":
            tokens = sorted(_log_int(rng, 1, 7000) for _ in range(2)) if rng.random() < 0.6 else [1, 1]
            more = {"cap": rng.choice((0.0, 0.0, round(rng.uniform(10, 60), 1))), "slopes": rng.random() < 0.3,
                    "prefix": rng.random() < 0.3}
        else:
            tokens = sorted(_log_int(rng, 4, 64) for _ in range(2))
            more = {"layers": _log_int(rng, 1, 40)}
            context = [c % 200 for c in context]
        case = _case(kind, "", seqs, tokens, sorted(context), heads, kv_heads, dim, page, **more)
        del case["name"]
        case["lengths"] = rng.randrange(1 << 20)
        contexts, counts = _lengths(case)
        # What the plain form holds at a time: scores of every head, padded to the longest sequence.
        padded = seqs * max(counts) * heads * (max(contexts) + max(counts)) if kind in ("tree", "prompt") else 0
        size = seqs * (max(contexts) + max(counts) + page) * kv_heads * dim * case.get("layers", 1)
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


def _trees(case, rng):
    """Ancestor masks and depths of a random tree per sequence; a token's parent is one of the eight before it, or no drafted
    token at all (several first tokens)."""
    masks, depths = [], []
    for count in _lengths(case)[1]:
        mask, depth = [], []
        for i in range(count):
            parent = rng.randrange(max(-1, i - 8), i) if i else -1
            mask.append((mask[parent] if parent >= 0 else 0) | 1 << i)
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
        masks += [m - (1 << 64) if m >> 63 else m for m in mask]
        depths += depth
    return masks, depths


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    kind, heads, kv_heads, dim, page = (case[k] for k in ("kind", "heads", "kv_heads", "head_dim", "page"))
    contexts, counts = _lengths(case)
    pages = [-(-(c + t) // page) for c, t in zip(contexts, counts)]
    order = torch.randperm(sum(pages), generator=gen, device=DEVICE).to(torch.int32).split(pages)
    first = [sum(counts[:b]) for b in range(len(counts) + 1)]
    rows = first[-1]
    shape = (sum(pages), kv_heads, page, dim)
    if kind == "accept":
        shape = (case["layers"],) + shape
    state = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "rows": rows,
             "longest": max(c + t for c, t in zip(contexts, counts)), "most": max(counts),
             "cu_tokens": _int(first), "context": _int(contexts), "counts": _int(counts),
             "page_table": torch.nn.utils.rnn.pad_sequence(list(order), batch_first=True),
             "k_cache": _randn(gen, *shape), "v_cache": _randn(gen, *shape)}
    if kind == "append":
        frequencies, magnitude = _frequencies(case)
        state.update(qkv=_randn(gen, rows, (heads + 2 * kv_heads) * dim), frequencies=frequencies.to(DEVICE),
                     magnitude=magnitude, interleaved=case["interleaved"])
    elif kind == "accept":
        # Paths whose later nodes lie behind the slots they move to, as in trees drawn level by level.
        paths = []
        for count in counts:
            length = rng.randint(1, max(1, min(8, count // 2)))
            paths.append([0] + sorted(rng.sample(range(length, count), length - 1)))
        state.update(accepted=_int([p + [0] * (8 - len(p)) for p in paths]), accepted_lengths=_int([len(p) for p in paths]))
    else:
        # Heads differ in how sharply they look: scores between 0.5 and 3 standard deviations.
        gain = torch.logspace(math.log10(0.5), math.log10(3.0), heads, device=DEVICE).view(1, heads, 1)
        q = (torch.randn((rows, heads, dim), generator=gen, device=DEVICE) * gain).to(torch.float16)
        slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device=DEVICE) / heads)
        state.update(q=q.view(rows, heads * dim), cap=case["cap"], slopes=slopes if case["slopes"] else None)
        if kind == "tree":
            masks, depths = _trees(case, rng)
            base = [c for c, t in zip(contexts, counts) for _ in range(t)]
            state.update(tree_mask=_int(masks, torch.int64), positions=_int([b + d for b, d in zip(base, depths)]))
        else:
            state["prefix"] = _int(_prefixes(case)) if case["prefix"] else None
    return state


# --------------------------------------------------------------------------------------------------- one pass

def _own(s):
    import flash_llm_b200.torch_op  # noqa: F401  (registers torch.ops.flashllm)
    ops = torch.ops.flashllm
    batch = (s["k_cache"], s["v_cache"], s["cu_tokens"], s["context"], s["page_table"])
    if s["kind"] == "append":
        q = ops.rotary_append(s["qkv"], *batch, s["frequencies"], s["interleaved"], s["magnitude"])
        return q, s["k_cache"], s["v_cache"]
    if s["kind"] == "accept":
        ops.cache_accept(*batch, s["accepted"], s["accepted_lengths"])
        return s["k_cache"], s["v_cache"]
    if s["kind"] == "tree":
        return ops.tree_attention(s["q"], *batch, s["tree_mask"], cap=s["cap"], slopes=s["slopes"], positions=s["positions"])
    return ops.prompt_attention(s["q"], *batch, prefix=s["prefix"], cap=s["cap"], slopes=s["slopes"])


def _slots(s, sequence, position):
    """(page, place in the page) of positions of sequences."""
    return s["page_table"][sequence, position // s["page"]].long(), position % s["page"]


def _plain_append(s):
    row = torch.arange(s["rows"], device=DEVICE)
    sequence = torch.searchsorted(s["cu_tokens"].long(), row, right=True) - 1
    position = s["context"][sequence].long() + row - s["cu_tokens"][sequence]
    angle = position.double()[:, None] * s["frequencies"]
    c, d = ((f(angle) * s["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = s["qkv"].float().view(s["rows"], -1, s["dim"])
    turned, rest = x[:, :s["heads"] + s["kv_heads"]], x[:, s["heads"] + s["kv_heads"]:]
    pairs = s["frequencies"].numel()
    y = turned.clone()
    if s["interleaved"]:
        u, w = turned[..., 0:2 * pairs:2], turned[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = u * c - w * d, w * c + u * d
    else:
        u, w = turned[..., :pairs], turned[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = u * c - w * d, w * c + u * d
    page, place = _slots(s, sequence, position)
    s["k_cache"][page, :, place] = y[:, s["heads"]:].half()
    s["v_cache"][page, :, place] = rest.half()
    return y[:, :s["heads"]].reshape(s["rows"], -1).half(), s["k_cache"], s["v_cache"]


def _plain_accept(s):
    step = torch.arange(s["accepted"].shape[1], device=DEVICE)
    sequence, step = (step < s["accepted_lengths"][:, None]).nonzero(as_tuple=True)
    start = s["context"][sequence].long()
    page, place = _slots(s, sequence, start + s["accepted"][sequence, step])
    k, v = s["k_cache"][:, page, :, place], s["v_cache"][:, page, :, place]
    page, place = _slots(s, sequence, start + step)
    s["k_cache"][:, page, :, place] = k
    s["v_cache"][:, page, :, place] = v
    return s["k_cache"], s["v_cache"]


def _plain_attention(s):
    heads, kv_heads, dim, longest, most = s["heads"], s["kv_heads"], s["dim"], s["longest"], s["most"]
    seqs = s["counts"].numel()
    column, line = torch.arange(longest, device=DEVICE), torch.arange(most, device=DEVICE)
    start, context = s["cu_tokens"][:-1, None], s["context"][:, None]
    there = line < s["counts"][:, None]                                                     # [B][T]
    row = (start + line).clamp(max=s["rows"] - 1)
    length = context + s["counts"][:, None]
    page = s["page_table"][:, (column // s["page"]).clamp(max=s["page_table"].shape[1] - 1)].long()
    k, v = (s[c][page, :, column % s["page"]].float().transpose(1, 2) for c in ("k_cache", "v_cache"))  # [B][Hkv][L][D]
    v = v * (column < length)[:, None, :, None]
    q = s["q"][row].float().view(seqs, most, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)).view(seqs, heads, most, longest)
    score *= 1 / math.sqrt(dim)
    if s["cap"] > 0:
        score /= s["cap"]
        score.tanh_()
        score *= s["cap"]
    drafted = column - context                                                              # [B][L]
    if s["kind"] == "tree":
        bit = s["tree_mask"][row][:, :, None] >> drafted.clamp(0, 63)[:, None, :] & 1
        seen = (drafted < 0)[:, None, :] | (bit == 1) & (drafted < 64)[:, None, :]
        ahead = s["positions"][(start + drafted).clamp(0, s["rows"] - 1)]
        place, key = s["positions"][row], torch.where(drafted < 0, column, ahead)
    else:
        seen = drafted[:, None, :] <= line[:, None]
        if s["prefix"] is not None:
            seen |= (column < s["prefix"][:, None])[:, None, :]
        place, key = context + line, column.expand(seqs, -1)
    if s["slopes"] is not None:
        score += s["slopes"].view(1, heads, 1, 1) * (key[:, None, None, :] - place[:, None, :, None]).float()
    seen &= (column < length)[:, None, :]
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -math.inf, 0.0, top)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(seqs, kv_heads, -1, longest), v).view(seqs, heads, most, dim)
    out = out / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2)[there].reshape(s["rows"], heads * dim).half()


def run(state):
    if own:
        return _own(state)
    if state["kind"] == "append":
        return _plain_append(state)
    if state["kind"] == "accept":
        return _plain_accept(state)
    return _plain_attention(state)


# --------------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and head by head; acceptance copies and computes nothing."""
    if case["kind"] == "accept":
        return None
    s = prepare(case, seed)
    contexts, counts = _lengths(case)
    heads, kv_heads, dim, page = s["heads"], s["kv_heads"], s["dim"], s["page"]
    share = heads // kv_heads
    cut = s["cu_tokens"].tolist()
    if case["kind"] == "append":
        frequencies, magnitude = _frequencies(case)
        frequencies = frequencies.to(DEVICE)
        pairs = frequencies.numel()
        first = torch.arange(pairs, device=DEVICE) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else pairs)
        out = torch.empty((s["rows"], heads * dim), dtype=torch.float64, device=DEVICE)
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        for b, (context, count) in enumerate(zip(contexts, counts)):
            place = torch.arange(context, context + count, device=DEVICE)
            turn = torch.polar(torch.full((count, pairs), magnitude, dtype=torch.float64, device=DEVICE),
                               place.double()[:, None] * frequencies)[:, None]
            x = s["qkv"][cut[b]:cut[b + 1]].double().view(count, heads + 2 * kv_heads, dim)
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[cut[b]:cut[b + 1]] = y[:, :heads].reshape(count, -1)
            pages = s["page_table"][b].long()[place // page]
            caches[0][pages, :, place % page] = y[:, heads:heads + kv_heads]
            caches[1][pages, :, place % page] = x[:, heads + kv_heads:]
        return out, caches[0], caches[1]
    out = torch.empty((s["rows"], heads, dim), dtype=torch.float64, device=DEVICE)
    prefixes = _prefixes(case) if s.get("prefix") is not None else contexts
    for b, (context, count) in enumerate(zip(contexts, counts)):
        used = s["page_table"][b].long()[:-(-(context + count) // page)]
        line = torch.arange(count, device=DEVICE)[:, None]
        column = torch.arange(context + count, device=DEVICE)[None]
        if case["kind"] == "tree":
            mask = s["tree_mask"][cut[b]:cut[b + 1]]
            among = torch.stack([mask >> j & 1 for j in range(min(count, 64))], 1).bool()
            seen = torch.cat([torch.ones((count, context), dtype=torch.bool, device=DEVICE), among], 1)
            place = s["positions"][cut[b]:cut[b + 1]].double()
            key = torch.cat([torch.arange(context, device=DEVICE).double(), place])
        else:
            seen = (column <= context + line) | (column < prefixes[b])
            place = (context + line[:, 0]).double()
            key = column[0].double()
        for h in range(kv_heads):
            k, v = (s[c][used, h].reshape(-1, dim)[:context + count].double() for c in ("k_cache", "v_cache"))
            for i in range(h * share, (h + 1) * share):
                score = s["q"][cut[b]:cut[b + 1], i * dim:(i + 1) * dim].double() @ k.T / math.sqrt(dim)
                if s["cap"] > 0:
                    score = s["cap"] * torch.tanh(score / s["cap"])
                if s["slopes"] is not None:
                    score = score + s["slopes"][i].double() * (key[None] - place[:, None])
                score = torch.where(seen, score, -math.inf)
                out[cut[b]:cut[b + 1], i] = torch.softmax(score, -1) @ v
    return out.view(s["rows"], heads * dim)


# --------------------------------------------------------------------------------------------------- accounting

def work(case):
    """Bytes read and written once; multiply-adds of the pairs of a query and a key that it sees (4 * head size each)."""
    contexts, counts = _lengths(case)
    heads, kv_heads, dim, rows = case["heads"], case["kv_heads"], case["head_dim"], sum(counts)
    if case["kind"] == "append":
        return {"bytes": 4 * rows * (heads + 2 * kv_heads) * dim, "flops": 3 * rows * (heads + kv_heads) * case["rotary"]}
    if case["kind"] == "accept":
        # Half of a tree's tokens, eight at most, lie on the longest path: one to that many are accepted, the first in place.
        moved = sum(max(1, min(8, t // 2)) - 1 for t in counts) / 2
        return {"bytes": 8 * case["layers"] * kv_heads * dim * max(1.0, moved), "flops": 0}
    if case["kind"] == "tree":
        pairs = sum(t * (c + 1) for c, t in zip(contexts, counts))
    else:
        prefixes = _prefixes(case) if case["prefix"] else contexts
        pairs = 0
        for c, t, p in zip(contexts, counts, prefixes):
            ahead = max(0, min(p - c, t))  # tokens of the prefix, each of which sees all of it
            pairs += t * c + ahead * ahead + (t * (t + 1) - ahead * (ahead + 1)) // 2
    return {"bytes": 4 * rows * heads * dim + 4 * sum(c + t for c, t in zip(contexts, counts)) * kv_heads * dim,
            "flops": 4 * dim * heads * pairs}
