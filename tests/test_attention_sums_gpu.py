"""What the running maxima and sums of the attention kernels can lose, on the GPU against the definitions in 64 bits: those of the
warps' kernels, over 4 bits and of single tokens through a window, and the joining of parts."""
import math

import pytest
import torch

import four_bit_cache as four
from four_bit_cache import FourBitBatch
from paged_cache import Batch
from test_more_cache_operators_gpu import healthy, near, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def few_rows(batch, window=0, sinks=0, scale=None):
    """(output, bound on the error of the kernel of few rows) of every row, [rows][heads * dim] in 64 bits.

    Scores: codes times queries are exact, sums of `dim` products in 32 bits, truncated at each addition of the tensor core (2^-20 of
    the sizes of steps times codes and lowest values); an error d of them is one of 2 d of the weights, numerator and denominator
    together, and 2^-20 holds exponentials and sums.  A weight times its step is rounded to fp16, 2^-11 of it at most, which is
    multiplied by a code less 7.5: b = 2^-11 x 7.5 p step.  The roundings of n keys are independent, so their sum passes 6 times the
    root of the sum of b^2 once in 3e7 (Hoeffding).  Products below fp16's normal numbers are off by 2^-25 of units in which the
    largest step is at least 2^5, for each key by 2^-27 of the largest step in the output (the weights' sum is 1 at least).  The output
    is rounded to fp16, 2^-11 of it or 2^-25."""
    dim, share = batch.dim, batch.heads // batch.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((batch.rows, batch.heads, dim), dtype=torch.float64, device=batch.device)
    bound = torch.zeros_like(out)
    for b, (context, count) in enumerate(zip(batch.contexts, batch.counts)):
        lo, hi = batch.cut[b], batch.cut[b + 1]
        if count == 0:
            continue
        away = torch.arange(context + count, device=batch.device)[None] - (context + torch.arange(count, device=batch.device)[:, None])
        seen = away <= 0
        if window:
            seen &= (away > -window) | (away + context + torch.arange(count, device=batch.device)[:, None] < sinks)
        (k, k_step, k_low), (v, v_step, v_low) = batch.parts_of(batch.k_cache, b), batch.parts_of(batch.v_cache, b)
        q = batch.q[lo:hi].double().view(count, batch.kv_heads, share, dim)
        score = scale * torch.einsum("tgsd,jgd->gstj", q, k)
        off = 2.0 ** -20 * scale * torch.einsum("tgsd,jgd->gstj", q.abs(), 15 * k_step + k_low.abs())
        p = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), -1)
        error = torch.where(seen, off, torch.zeros_like(off)).amax(-1)
        mix = lambda w, x: torch.einsum("gstj,jgd->tgsd", w, x).reshape(count, batch.heads, dim)  # noqa: E731
        out[lo:hi] = mix(p, v)
        size = (2 * error.permute(2, 0, 1).reshape(count, batch.heads, 1) + 2.0 ** -20) * mix(p, 15 * v_step + v_low.abs())
        bound[lo:hi] = (2.0 ** -11 * out[lo:hi].abs() + 6 * 2.0 ** -11 * mix(p.square(), (7.5 * v_step).square()).sqrt() + size
                        + 2.0 ** -27 * (context + count) * v_step.amax() + 2.0 ** -25)
    return out.view(batch.rows, -1), bound.view(batch.rows, -1)


def many_rows(batch, window=0, sinks=0, scale=None):
    """(output, bound on the error of the kernel of many rows) as few_rows has them.

    Elements are rounded to fp16, 2^-11 of each at most, and multiplied.  A value's rounding adds p 2^-11 |v| to the output, its
    weight's as much, an element of a key's p |v - output| scale |q| 2^-11 |k|: all independent, so 6 times the root of the sum of their
    squares.  An error d of the scores has a second order, 2 d^2 of the weights: d is 6 times the root of the sum of (scale q 2^-11 k)^2
    at most.  Sums are of the elements' sizes, 2^-20 of them as there, and of weights below fp16's normal numbers 2^-25 each."""
    dim, share = batch.dim, batch.heads // batch.kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros((batch.rows, batch.heads, dim), dtype=torch.float64, device=batch.device)
    bound = torch.zeros_like(out)
    for b, (context, count) in enumerate(zip(batch.contexts, batch.counts)):
        lo, hi = batch.cut[b], batch.cut[b + 1]
        if count == 0:
            continue
        place = torch.arange(context + count, device=batch.device)
        away = place[None] - (context + torch.arange(count, device=batch.device)[:, None])
        seen = away <= 0
        if window:
            seen &= (away > -window) | (place < sinks)
        k, v = batch.rows_of(batch.k_cache, b), batch.rows_of(batch.v_cache, b)
        for h in range(batch.heads):
            q, kh, vh = batch.q[lo:hi, h * dim:(h + 1) * dim].double(), k[:, h // share], v[:, h // share]
            score = scale * q @ kh.T
            p = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), 1)
            o = p @ vh
            keys = (scale * 2.0 ** -11) ** 2 * (q.square() @ kh.square().T)  # the square of a score's error, a key's
            p2 = p.square()
            spread = (p2 * keys) @ vh.square() - 2 * o * ((p2 * keys) @ vh) + o.square() * (p2 * keys).sum(1, keepdim=True)
            off = torch.where(seen, 2.0 ** -20 * scale * (q.abs() @ kh.abs().T), torch.zeros_like(p)).amax(1, keepdim=True)
            second = 2 * 36 * torch.where(seen, keys, torch.zeros_like(keys)).amax(1, keepdim=True)
            out[lo:hi, h] = o
            bound[lo:hi, h] = (2.0 ** -11 * o.abs() + 6 * (2.0 ** -21 * (p2 @ vh.square()) + spread).sqrt()
                               + (2 * off + second + 2.0 ** -20) * (p @ vh.abs()) + 2.0 ** -25 * (seen.double() @ vh.abs() * 2.0 ** -7 + 1))
    return out.view(batch.rows, -1), bound.view(batch.rows, -1)


# --------------------------------------------------------------------------------------------------- what each kernel rounds

@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 5)])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,gain", [
    ([0], [1], 1, 1, 64, 16, 1.0), ([210], [1], 16, 16, 64, 16, 1.0), ([5000, 31, 900], [1, 1, 1], 8, 2, 128, 64, 2.0),
    ([3000, 17], [1, 1], 20, 1, 128, 32, 0.3), ([900, 100], [3, 2], 12, 4, 128, 16, 2.0), ([20000], [8], 4, 1, 64, 128, 4.0)])
def test_few_rows_over_four_bits_round_no_more_than_they_say(ops, contexts, counts, heads, kv_heads, dim, page, gain, window, sinks):  # noqa: F811
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, page, gain=gain)
    near(ops.four_bit_attention(b.q, *b.arrays, window, sinks), *few_rows(b, window, sinks))


@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 5)])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,gain", [
    ([0], [200], 2, 2, 64, 16, 1.0), ([130, 0, 77], [300, 40, 129], 8, 2, 128, 128, 2.0), ([3000], [65], 4, 1, 128, 32, 0.3),
    ([2000, 9], [1, 1], 40, 1, 64, 64, 1.0), ([20000], [12], 4, 1, 64, 128, 4.0)])
def test_many_rows_over_four_bits_round_no_more_than_they_say(ops, contexts, counts, heads, kv_heads, dim, page, gain, window, sinks):  # noqa: F811
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, page, gain=gain)
    near(ops.four_bit_attention(b.q, *b.arrays, window, sinks), *many_rows(b, window, sinks))


# --------------------------------------------------------------------------------------------------- steps of zero

def flat_values(b, s, keys, size=1.0):
    """Makes each 64 values of sequence s at the positions `keys` one value: a step of zero, and a lowest value that is not."""
    g = torch.Generator().manual_seed(11)
    x = (size * (1.0 + torch.rand((len(keys), b.kv_heads, b.dim // four.GROUP), generator=g))).half().float().to(b.device)
    where, place = b.pages_of(s, keys)
    four.put(b.v_cache, b.dim, (where, slice(None), place), x.repeat_interleave(four.GROUP, -1))
    assert bool((four.parts(b.v_cache, b.dim)[1][where, :, place, :, 0] == 0).all())


# Pieces of several blocks of 32 keys, or of 16 where a sequence has more than eight rows.
LONG = [([30000], [1], 4, 1, 128, 64), ([30000], [1], 1, 1, 64, 16), ([30000], [1], 12, 1, 64, 32), ([30000, 9000], [3, 1], 4, 1, 128, 64)]


@pytest.mark.parametrize("size,later", [(1.0, 1.0), (512.0, 1.0), (60.0, 2.0 ** -9), (1.0, 2.0 ** 9)])
@pytest.mark.parametrize("period,flat", [(32, 16), (64, 32), (96, 40), (1024, 512), (1024, 1023)])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page", LONG)
def test_values_without_a_step_keep_their_weight(ops, contexts, counts, heads, kv_heads, dim, page, period, flat, size, later):  # noqa: F811
    """The first `flat` of each `period` positions have values without a step, the others steps `later` times as large as usual."""
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, page)
    four.parts(b.v_cache, dim)[1][:] *= later
    for s, (c, t) in enumerate(zip(contexts, counts)):
        place = torch.arange(c + t, device="cuda")
        flat_values(b, s, place[place % period < flat], size)
    near(ops.four_bit_attention(b.q, *b.arrays), *few_rows(b))


@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4), (200, 40)])
@pytest.mark.parametrize("flat", [1, 4, 16, 32, 40, 100, 300, -1, -40])
@pytest.mark.parametrize("kv_heads,dim,page", [(2, 128, 16), (2, 64, 64)])
def test_values_without_a_step_in_many_sequences(ops, kv_heads, dim, page, flat, window, sinks):  # noqa: F811
    """The first `flat` positions of every sequence, the last for a negative number."""
    n = 320
    b = FourBitBatch([300] * n, [1] * n, kv_heads, kv_heads, dim, page)
    place = torch.arange(301, device="cuda")
    for s in range(n):
        flat_values(b, s, place[:flat] if flat > 0 else place[flat:])
    near(ops.four_bit_attention(b.q, *b.arrays, window, sinks), *few_rows(b, window, sinks))


@pytest.mark.parametrize("count,heads", [(1, 4), (3, 4)])
def test_appended_rows_without_a_step_keep_their_weight(ops, count, heads):  # noqa: F811
    """As a program has them: rows of one value each through the append, others behind them, then attention of them all."""
    dim, total = 128, 20000
    b = FourBitBatch([0], [total], heads, 1, dim, 16)
    qkv = torch.randn((total, (heads + 2) * dim), device="cuda").half()
    flat = torch.arange(total, device="cuda") % 256 < 128
    qkv[flat, -dim:] = torch.linspace(0.5, 2.0, int(flat.sum()), device="cuda").half()[:, None]
    q = ops.four_bit_append(qkv, *b.arrays)
    cu = torch.tensor([0, count], dtype=torch.int32, device="cuda")
    context = torch.tensor([total - count], dtype=torch.int32, device="cuda")
    b.contexts, b.counts, b.cut, b.rows, b.q = [total - count], [count], [0, count], count, q[total - count:].contiguous()
    near(ops.four_bit_attention(b.q, b.k_cache, b.v_cache, cu, context, b.page_table), *few_rows(b))


# --------------------------------------------------------------------------------------------------- large scores

def of_exact_scores(batch, score, window=0, sinks=0):
    """(output, bound) of the rows of one sequence, whose scores [keys] in 64 bits are the same for all rows and exact in the kernels.

    A weight is rounded to fp16, or its product with a step (see few_rows): b = 2^-11 p |v| or 2^-11 x 7.5 p step, 6 times the root of the
    sum of b^2.  The scale times log2 e is off by 2^-23 of itself, exponents, which matter down to -30, by 2^-18 then; sums are of
    sizes |v|, or 15 steps and the lowest value."""
    (context,), (count,), share = batch.contexts, batch.counts, batch.heads // batch.kv_heads
    away = torch.arange(context + count, device="cuda")[None] - (context + torch.arange(count, device="cuda")[:, None])
    seen = away <= 0
    if window:
        seen &= (away > -window) | (torch.arange(context + count, device="cuda") < sinks)
    p = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), 1)
    mix = lambda w, x: torch.einsum("tj,jgd->tgd", w, x).repeat_interleave(share, 1).reshape(count, -1)  # noqa: E731
    if isinstance(batch, FourBitBatch):
        v, step, low = batch.parts_of(batch.v_cache, 0)
        each, size = 7.5 * step, 15 * step + low.abs()
    else:
        v = batch.rows_of(batch.v_cache, 0)
        each = size = v.abs()
    out = mix(p, v)
    return out, (2.0 ** -11 * out.abs() + 6 * 2.0 ** -11 * mix(p.square(), each.square()).sqrt() + 2.0 ** -18 * mix(p, size)
                 + 2.0 ** -25 * float(each.amax()))


def large_scores(b, first, second, small):
    """Queries and keys of a Batch of one sequence whose products are first x second + small, exactly."""
    where, at = b.pages_of(0, torch.arange(len(small), device="cuda"))
    b.k_cache[:] = 0
    b.k_cache[where, :, at, 0] = second
    b.k_cache[where, :, at, 1] = small.half()[:, None].expand(-1, b.kv_heads)
    b.q[:] = 0
    b.q.view(b.rows, b.heads, b.dim)[..., 0], b.q.view(b.rows, b.heads, b.dim)[..., 1] = first, 1.0


LARGE = [(0.5, 1024.0, 32768.0, 4), (2.0 ** -5, 32768.0, 16384.0, 64)]  # 2^25 and 2^29, and a step of 32-bit numbers there


@pytest.mark.parametrize("scale,first,second,step", LARGE)
@pytest.mark.parametrize("dim,page,heads,kv_heads", [(64, 16, 4, 1), (128, 64, 12, 2)])
def test_parts_of_large_scores_keep_their_weight_through_a_window(ops, dim, page, heads, kv_heads, scale, first, second, step):  # noqa: F811
    """Some positions' scores are one or two steps of 32-bit numbers above the others', long runs of them, so that an item's parts have
    other maxima: e^2 apart."""
    b = Batch([20000], [1], heads, kv_heads, dim, page)
    small = step * (torch.arange(20001, device="cuda") // 300 % 3).double()
    large_scores(b, first, second, small)
    near(ops.window_attention(b.q, *b.arrays, 15000, 5, scale=scale), *of_exact_scores(b, scale * small, 15000, 5))


@pytest.mark.parametrize("scale,first,second,step", LARGE)
@pytest.mark.parametrize("count,heads,kv_heads,dim,page", [(1, 4, 1, 64, 16), (3, 8, 2, 128, 64), (140, 2, 1, 64, 128)])
@pytest.mark.parametrize("window", [0, 17000])
def test_parts_of_large_scores_of_many_rows_keep_their_weight(ops, count, heads, kv_heads, dim, page, window, scale, first, second, step):  # noqa: F811
    """The same for the tensor core's kernel, whose parts are those of other CTAs."""
    b = Batch([20000], [count + (window > 0)], heads, kv_heads, dim, page)  # (a single token through a window is the warps')
    small = step * (torch.arange(20000 + b.rows, device="cuda") // 600 % 3).double()
    large_scores(b, first, second, small)
    got = ops.window_attention(b.q, *b.arrays, window, 5, scale=scale) if window else ops.prompt_attention(b.q, *b.arrays, scale=scale)
    near(got, *of_exact_scores(b, scale * small, window, 5))


ONE = 0.6931471824645996  # times log2 e, in 32 bits: 1


@pytest.mark.parametrize("dim,page,heads,kv_heads", [(64, 16, 4, 1), (128, 64, 12, 2)])
@pytest.mark.parametrize("scale,first,second,step,slope", [
    (2.0, 1024.0, 32768.0, 4, False),       # 2^25 and one step of 32-bit numbers more: 2^11.5 times the weight
    (0.125, 32768.0, 16384.0, 64, False),   # 2^29
    (ONE, 32768.0, 4096.0, 16, True),       # 2^27, in units of log 2
])
@pytest.mark.parametrize("base", [0, 1])
def test_a_maximum_grows_by_a_step_of_32_bits_through_a_window(ops, scale, first, second, step, slope, base, dim, page, heads, kv_heads):  # noqa: F811
    """One key in 128 has a score that is one step of 32-bit numbers above the others', which are even (base 0) or odd (1)."""
    b = Batch([20000], [1], heads, kv_heads, dim, page)
    small = step * (base + (torch.arange(20001, device="cuda") % 128 == 127).double())
    large_scores(b, first, second, small)
    slopes = torch.zeros(heads, device="cuda") if slope else None
    near(ops.window_attention(b.q, *b.arrays, 15000, 5, scale=scale, slopes=slopes), *of_exact_scores(b, scale * small, 15000, 5))


@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("base", [0, 1])
@pytest.mark.parametrize("heads,page", [(4, 64), (4, 16), (12, 32)])
def test_a_maximum_grows_by_a_step_of_32_bits_over_four_bits(ops, heads, page, base, slope):  # noqa: F811
    """The same over 4 bits: keys' lowest values alone make scores of 2^27 and 16 or 32 more."""
    b = FourBitBatch([20000], [1], heads, 1, 128, page)
    place = torch.arange(20001, device="cuda")
    small = 16.0 * (base + (place % 128 == 127).double())
    where, at = b.pages_of(0, place)
    codes, scales = four.parts(b.k_cache, 128)
    codes[where, :, at], scales[where, :, at] = 0, 0.0
    scales[where, :, at, 0, 1] = 4096.0
    scales[where, :, at, 1, 1] = small.half()[:, None]
    b.q[:] = 0
    b.q.view(heads, 128)[:, 0], b.q.view(heads, 128)[:, 64] = 32768.0, 1.0
    slopes = torch.zeros(heads, device="cuda") if slope else None
    near(ops.four_bit_attention(b.q, *b.arrays, scale=ONE, slopes=slopes), *of_exact_scores(b, ONE * small))


@pytest.mark.parametrize("count,heads,page", [(140, 2, 64), (12, 4, 16), (1, 40, 32)])
def test_large_scores_of_many_rows_over_four_bits_keep_their_weight(ops, count, heads, page):  # noqa: F811
    """Scores of 2^24, 2 or 4 more for long runs of keys; elements are exact in fp16, values' roundings as large as their weights'."""
    b = FourBitBatch([20000], [count], heads, 1, 128, page)
    place = torch.arange(20000 + count, device="cuda")
    small = 16.0 * (place // 600 % 3).double()
    where, at = b.pages_of(0, place)
    codes, scales = four.parts(b.k_cache, 128)
    codes[where, :, at], scales[where, :, at] = 0, 0.0
    scales[where, :, at, 0, 1] = 4096.0
    scales[where, :, at, 1, 1] = small.half()[:, None]
    b.q[:] = 0
    b.q.view(count, heads, 128)[..., 0], b.q.view(count, heads, 128)[..., 64] = 32768.0, 1.0
    values = Batch([20000], [count], heads, 1, 128, page)  # of 16 bits, of which the bound is
    values.rows_of = lambda cache, s: 2.0 ** 0.5 * b.rows_of(b.v_cache, s)
    want, bound = of_exact_scores(values, 0.125 * small)
    near(ops.four_bit_attention(b.q, *b.arrays, scale=0.125), want / 2.0 ** 0.5, bound)
