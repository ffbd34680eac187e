"""Batches over a paged key/value cache for the tests of its operators, and the operators' definitions in 64 bits."""
from __future__ import annotations

import math

import torch


class Batch:
    """`contexts` and `counts` per sequence; the cache is filled with random values where the sequences have positions and with
    `unused` (NaN: nobody may use it) everywhere else, its pages are dealt out in random order."""

    def __init__(self, contexts, counts, heads, kv_heads, dim, page, seed=0, unused=float("nan"), spare_pages=2, device="cuda",
                 extra_rows=0, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.contexts, self.counts, self.heads, self.kv_heads, self.dim, self.page = list(contexts), list(counts), heads, kv_heads, dim, page
        self.device = torch.device(device)
        pages = [-(-(c + t) // page) for c, t in zip(contexts, counts)]
        total = sum(pages) + spare_pages
        order = torch.randperm(total, generator=g)
        width = max(pages + [1])
        table = torch.zeros((len(pages), width), dtype=torch.int32)
        self.cut = [0]
        k = torch.full((total, kv_heads, page, dim), unused, dtype=torch.float16)
        v = k.clone()
        at = 0
        for b, (c, t) in enumerate(zip(contexts, counts)):
            table[b, :pages[b]] = order[at:at + pages[b]].to(torch.int32)
            at += pages[b]
            self.cut.append(self.cut[-1] + t)
            for cache in (k, v):
                rows = torch.randn((c + t, kv_heads, dim), generator=g).to(torch.float16)
                place = torch.arange(c + t)
                cache[table[b].long()[place // page], :, place % page] = rows
        self.rows = self.cut[-1] + extra_rows
        self.q = (gain * torch.randn((self.rows, heads * dim), generator=g)).to(torch.float16).to(self.device)
        self.k_cache, self.v_cache, self.page_table = k.to(self.device), v.to(self.device), table.to(self.device)
        self.cu_tokens = torch.tensor(self.cut, dtype=torch.int32, device=self.device)
        self.context = torch.tensor(self.contexts, dtype=torch.int32, device=self.device)

    @property
    def arrays(self):
        return self.k_cache, self.v_cache, self.cu_tokens, self.context, self.page_table

    def pages_of(self, b, place):
        return self.page_table[b].long()[place // self.page], place % self.page

    def rows_of(self, cache, b):
        """[positions][kv_heads][dim] of sequence b in 64 bits."""
        place = torch.arange(self.contexts[b] + self.counts[b], device=self.device)
        page, at = self.pages_of(b, place)
        return cache[page, :, at].double()


def random_tree(counts, contexts, seed, device="cuda", reach=6):
    """(masks int64, positions int32) of random trees; a token sees its ancestors and itself."""
    g = torch.Generator().manual_seed(seed)
    masks, positions = [], []
    for count, context in zip(counts, contexts):
        mask, depth = [], []
        for i in range(count):
            parent = int(torch.randint(max(-1, i - reach), i, (1,), generator=g)) if i else -1
            mask.append(((mask[parent] if parent >= 0 else 0) | 1 << i) & (1 << 64) - 1)
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
        masks += [m - (1 << 64) if m >> 63 else m for m in mask]
        positions += [context + d for d in depth]
    return (torch.tensor(masks, dtype=torch.int64, device=device), torch.tensor(positions, dtype=torch.int32, device=device))


def attention(batch: Batch, tree_mask=None, positions=None, prefix=None, scale=None, cap=0.0, slopes=None):
    """(output, bound on the kernels' error) of every row of a sequence, [rows][heads * dim] in 64 bits.

    The bound: a weight p is rounded to fp16 once (2^-11 of it, or 2^-25 where it is subnormal: the largest weight is at least 1,
    and so is their sum, which they are divided by), the output once (2^-11 of it).  A score is a sum of `dim` products
    in 32 bits, truncated rather than rounded at each of dim / 16 additions of the tensor core: below 2^-20 of the sum of the
    products' sizes; cap and distance are a few roundings of 2^-24 of their own sizes each.  An error d of the scores is one of
    2 d of the weights, numerator and denominator together."""
    dim, share = batch.dim, batch.heads // batch.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((batch.rows, batch.heads, dim), dtype=torch.float64, device=batch.device)
    bound = torch.zeros_like(out)
    for b, (context, count) in enumerate(zip(batch.contexts, batch.counts)):
        if count == 0:
            continue
        lo, hi = batch.cut[b], batch.cut[b + 1]
        line, column = torch.arange(count, device=batch.device), torch.arange(context + count, device=batch.device)
        if tree_mask is not None:
            own = torch.zeros((count, count), dtype=torch.bool, device=batch.device)
            for j in range(min(count, 64)):
                own[:, j] = tree_mask[lo:hi] >> j & 1 == 1
            seen = torch.cat([torch.ones((count, context), dtype=torch.bool, device=batch.device), own], 1)
        else:
            seen = column[None] <= context + line[:, None]
            if prefix is not None:
                seen |= column[None] < int(prefix[b])
        place = context + line.double() if tree_mask is None or positions is None else positions[lo:hi].double()
        key = torch.cat([column[:context].double(), place])
        k, v = batch.rows_of(batch.k_cache, b), batch.rows_of(batch.v_cache, b)
        for h in range(batch.heads):
            q = batch.q[lo:hi, h * dim:(h + 1) * dim].double()
            kh, vh = k[:, h // share], v[:, h // share]
            score = scale * q @ kh.T
            size = scale * q.abs() @ kh.abs().T
            off = 2.0 ** -20 * size
            if cap > 0:
                score = cap * torch.tanh(score / cap)
                off = off + 2.0 ** -20 * cap
            if slopes is not None:
                away = float(slopes[h]) * (key[None] - place[:, None])
                score = score + away
                off = off + 2.0 ** -22 * (away.abs() + score.abs())
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            top = score.amax(1, keepdim=True)
            p = torch.where(seen, torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(score))
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            error = torch.where(seen, off, torch.zeros_like(off)).amax(1, keepdim=True)
            if bool(torch.isfinite(vh).all()):
                o, size_v, all_v = p @ vh, p @ vh.abs(), seen.double() @ vh.abs()
            else:  # a masked key contributes nothing, whatever it holds
                o, size_v, all_v = (torch.stack(x) for x in zip(*((p[r, see] @ vh[see], p[r, see] @ vh[see].abs(), vh[see].abs().sum(0))
                                                                   for r, see in enumerate(seen))))
            out[lo:hi, h] = o
            bound[lo:hi, h] = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2 * error + 2.0 ** -20) * size_v + 2.0 ** -25 * (all_v + 1)
    return out.view(batch.rows, -1), bound.view(batch.rows, -1)


def rotate(x, angle, magnitude, interleaved, rotary):
    """(turned, bound) of x [rows][heads][dim] by angle [rows][rotary / 2] in 64 bits.  The bound: one rounding to fp16, and
    cosine, sine and products in 32 bits, some 2^-21 of the pair's sizes."""
    y, size = x.clone(), torch.zeros_like(x)
    first = torch.arange(rotary // 2, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rotary // 2)
    c, s = magnitude * torch.cos(angle)[:, None], magnitude * torch.sin(angle)[:, None]
    u, w = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - w * s, w * c + u * s
    size[..., first] = size[..., second] = abs(magnitude) * (u.abs() + w.abs())
    return y, 2.0 ** -11 * y.abs() + 2.0 ** -21 * size + 2.0 ** -25
