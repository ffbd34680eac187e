"""Batches over a paged cache of 4 bits for the tests of its operators, and definitions in 64 bits: the codes, attention over what
they stand for, and attention through a window."""
from __future__ import annotations

import math

import torch

from paged_cache import Batch

GROUP = 64


def parts(cache, dim):
    """Views of a 4-bit cache: codes [pages][heads][page][dim / 2] and scales [pages][heads][page][dim / 64][2] (step, lowest)."""
    pages, heads, page, _ = cache.shape
    flat = cache.view(pages, heads, -1)
    return (flat[..., :page * dim // 2].unflatten(-1, (page, dim // 2)),
            flat[..., page * dim // 2:].unflatten(-1, (page, -1)).view(torch.float16).unflatten(-1, (-1, 2)))


def to_codes(x):
    """x [..][dim] in 32 bits: bytes [..][dim / 2] and scales fp16 [..][dim / 64][2], by the definition, operation by operation."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1).half()
    step = ((x.amax(-1) - low.float()) / torch.full_like(x[..., 0], 15.0)).half()
    code = ((x - low.float()[..., None]) / step.float()[..., None]).round().clamp(0, 15)
    code = torch.where(step.float()[..., None] > 0, code, torch.zeros_like(code)).flatten(-2).to(torch.uint8)
    bad = ~(x.abs() <= 65504).all(-1)
    step = torch.where(bad, torch.full_like(step, float("nan")), step)
    low = torch.where(bad, torch.zeros_like(low), low)
    code = torch.where(bad.repeat_interleave(GROUP, -1), torch.zeros_like(code), code)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.stack([step, low], -1)


def put(cache, dim, at, x):
    codes, scales = parts(cache, dim)
    codes[at], scales[at] = to_codes(x)


def values(cache, dim, at):
    """(elements, steps, lowest) at the places `at` in 64 bits, [..][dim] each."""
    codes, scales = (part[at] for part in parts(cache, dim))
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    step, low = (scales[..., i].double().repeat_interleave(GROUP, -1) for i in (0, 1))
    return low + step * code, step, low


class FourBitBatch(Batch):
    """A Batch whose caches hold 4 bits, and bytes of 255 (codes of 15, scales that are no numbers) where no sequence has a position."""

    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        caches = self.k_cache, self.v_cache
        pages, heads, page, dim = self.k_cache.shape
        self.k_cache, self.v_cache = (torch.full((pages, heads, page, dim * 9 // 16), 255, dtype=torch.uint8, device=self.device) for _ in range(2))
        for b, (context, count) in enumerate(zip(self.contexts, self.counts)):
            where, place = self.pages_of(b, torch.arange(context + count, device=self.device))
            for mine, cache in zip((self.k_cache, self.v_cache), caches):
                put(mine, dim, (where, slice(None), place), cache[where, :, place])

    def parts_of(self, cache, b):
        """(elements, steps, lowest) of sequence b, [positions][kv_heads][dim] in 64 bits."""
        where, place = self.pages_of(b, torch.arange(self.contexts[b] + self.counts[b], device=self.device))
        return values(cache, self.dim, (where, slice(None), place))

    def rows_of(self, cache, b):
        return self.parts_of(cache, b)[0]


def attention(batch, window=0, sinks=0, scale=None, cap=0.0, slopes=None):
    """(output, bound on the kernels' error) of every row of a sequence, [rows][heads * dim] in 64 bits.

    Over a cache of 16 bits the bound is that of the operators without a window: a weight rounded to fp16 once (2^-11, or 2^-25 where
    it is subnormal; the largest is at least 1 and so is their sum), the output once (2^-11), scores of `dim` products in 32 bits,
    truncated at each addition of the tensor core (2^-20 of the sum of the products' sizes), an error d of the scores is one of 2 d
    of the weights.  Over 4 bits either the elements are rounded to fp16 once more (2^-11 of each: of the values directly, of the
    keys 2^-11 of the products' sizes), or weights times steps are rounded (2^-11 of step |code - 7.5|, at most 8 steps, and 2^-25
    of at most 2^-5 of the largest step, or of the largest element where they are multiplied as they are), and sums are those of
    steps times codes and lowest values apart, sizes of up to 15 steps and the lowest value each."""
    four = isinstance(batch, FourBitBatch)
    dim, share = batch.dim, batch.heads // batch.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((batch.rows, batch.heads, dim), dtype=torch.float64, device=batch.device)
    bound = torch.zeros_like(out)
    for b, (context, count) in enumerate(zip(batch.contexts, batch.counts)):
        if count == 0:
            continue
        lo, hi = batch.cut[b], batch.cut[b + 1]
        line, column = torch.arange(count, device=batch.device), torch.arange(context + count, device=batch.device)
        away = column[None] - (context + line[:, None])
        seen = away <= 0
        if window:
            seen &= (away > -window) | (column[None] < sinks)
        if four:
            (k, k_step, k_low), (v, v_step, v_low) = batch.parts_of(batch.k_cache, b), batch.parts_of(batch.v_cache, b)
            k_size, v_size = 15 * k_step + k_low.abs(), 15 * v_step + v_low.abs()
        else:
            k, v = batch.rows_of(batch.k_cache, b), batch.rows_of(batch.v_cache, b)
            k_size, v_size = k.abs(), v.abs()
        for h in range(batch.heads):
            q = batch.q[lo:hi, h * dim:(h + 1) * dim].double()
            kh, vh, kz, vz = (x[:, h // share] for x in (k, v, k_size, v_size))
            # What nobody sees may hold anything.
            used = seen.any(0)
            kh, vh, kz, vz = (torch.where(used[:, None], x, torch.zeros_like(x)) for x in (kh, vh, kz, vz))
            score = scale * q @ kh.T
            off = 2.0 ** -20 * scale * q.abs() @ kz.T
            if four:
                off = off + 2.0 ** -11 * scale * (q.abs().square() @ kh.square().T).sqrt() * 4  # independent roundings: four deviations
            if cap > 0:
                score = cap * torch.tanh(score / cap)
                off = off + 2.0 ** -20 * cap
            if slopes is not None:
                score = score + float(slopes[h]) * away
                off = off + 2.0 ** -22 * (float(slopes[h]) * away.abs() + score.abs())
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            p = torch.softmax(score, 1)
            error = torch.where(seen, off, torch.zeros_like(off)).amax(1, keepdim=True)
            out[lo:hi, h] = p @ vh
            weights = p @ vh.abs()
            if four:
                weights = torch.maximum(weights, p @ (8 * torch.where(used[:, None], v_step[:, h // share], torch.zeros_like(vh)))) + p @ vh.abs()
            bound[lo:hi, h] = (2.0 ** -11 * out[lo:hi, h].abs() + 2.0 ** -11 * weights + (2 * error + 2.0 ** -20) * (p @ vz)
                               + 2.0 ** -25 * (seen.double() @ vz + 1))
    return out.view(batch.rows, -1), bound.view(batch.rows, -1)
