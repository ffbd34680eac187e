"""Norms with the rotary append, attention through a window and the cache of 4 bits on the GPU, against their definitions in 64
bits."""
import pytest
import torch

import four_bit_cache as four
from four_bit_cache import FourBitBatch
from paged_cache import Batch, rotate

pytestmark = pytest.mark.gpu

BAD_CACHE = 64


@pytest.fixture(scope="module")
def ops(lib):
    import flash_llm_b200.torch_op  # noqa: F401
    return torch.ops.flashllm


@pytest.fixture(autouse=True)
def healthy(lib):
    lib.consume_status()
    yield
    assert lib.consume_status() == 0


def near(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    worst = (off / bound).max() if off.numel() else torch.zeros(())
    assert float(worst) <= 1.0, f"{what}: {float(worst):.2f} times the bound, at {int((off / bound).argmax())}"


def slopes_of(heads):
    return 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# --------------------------------------------------------------------------------------------------- appends

APPENDS = [
    # contexts, counts, heads, kv_heads, dim, page, rotary, interleaved
    ([0], [1], 1, 1, 64, 16, 64, False),
    ([5, 0, 31], [1, 3, 2], 4, 2, 64, 16, 16, True),
    ([100, 7, 0, 64], [17, 0, 33, 1], 6, 3, 128, 32, 128, False),
    ([100, 7, 0, 64], [17, 0, 33, 1], 6, 3, 128, 32, 128, True),
    ([127, 128], [130, 1], 9, 9, 128, 128, 64, False),
    ([3], [70], 5, 1, 64, 64, 48, False),
    ([200, 1], [4, 5], 8, 8, 128, 256, 0, False),
    ([40], [300], 40, 8, 128, 16, 112, True),
    ([12] * 70, [1] * 70, 2, 1, 64, 16, 32, False),
]


def turned(lib, b, qkv, rotary, interleaved, q_norm, k_norm, eps):
    """(queries and keys, bound, values) of the owned rows in 64 bits, and the arguments of the rotation.

    The bound's second part: the squares' sum of `dim` terms, root, quotient and two products in 32 bits are off by less than 2^-20 of
    the result, and so is what turning makes of it, by its pair's sizes; the first is rotate()'s, the rounding to fp16 in it."""
    frequencies, magnitude = lib.rotary_frequencies(rotary, scaling="by parts", factor=4.0, original_length=64) if rotary else (None, 1.0)
    f = torch.from_numpy(frequencies).cuda() if rotary else None
    owned = b.cut[-1]
    x = qkv[:owned].double().reshape(owned, b.heads + 2 * b.kv_heads, b.dim)
    place = torch.cat([torch.arange(c, c + t) for c, t in zip(b.contexts, b.counts)]).cuda()
    y = x[:, :b.heads + b.kv_heads].clone()
    for lo, hi, w in ((0, b.heads, q_norm), (b.heads, b.heads + b.kv_heads, k_norm)):
        if w is not None:
            y[:, lo:hi] = x[:, lo:hi] * w.double() / (x[:, lo:hi].square().mean(-1, keepdim=True) + eps).sqrt()
    size = y.abs()
    if rotary:
        z, bound = rotate(y, place.double()[:, None] * f, magnitude, interleaved, rotary)
        # both members of a pair may carry the norm's error: the largest of the head stands for them
        size = 2 * abs(magnitude) * size.amax(-1, keepdim=True).expand_as(size)
    else:
        z, bound = y, 2.0 ** -11 * y.abs() + 2.0 ** -25
    return z, bound + 2.0 ** -20 * size, x[:, b.heads + b.kv_heads:], (f, interleaved, magnitude)


def norms(dim, which="qk"):
    g = torch.Generator().manual_seed(5)
    w = (torch.randn((2, dim), generator=g)).to(torch.float16).cuda()
    return w[0] if "q" in which else None, w[1] if "k" in which else None


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,rotary,interleaved", APPENDS)
def test_norm_rotary_append(ops, lib, contexts, counts, heads, kv_heads, dim, page, rotary, interleaved):
    b = Batch(contexts, counts, heads, kv_heads, dim, page, extra_rows=3)
    columns = (heads + 2 * kv_heads) * dim
    qkv = torch.randn((b.rows, columns + 24), device="cuda").to(torch.float16)[:, 8:8 + columns]  # rows apart
    qkv[0, :dim] *= 1e-4  # small, and with an eps that matters
    w = norms(dim)
    y, bound, v, rotary_args = turned(lib, b, qkv, rotary, interleaved, *w, 1e-3)
    before = b.k_cache.clone(), b.v_cache.clone()
    q = ops.norm_rotary_append(qkv, *b.arrays, *w, 1e-3, *rotary_args)
    owned = b.cut[-1]
    near(q[:owned].view(owned, heads, dim), y[:, :heads], bound[:, :heads], "queries")
    for s, (c, t) in enumerate(zip(contexts, counts)):
        lo, hi = b.cut[s], b.cut[s + 1]
        where, place = b.pages_of(s, torch.arange(c, c + t, device="cuda"))
        near(b.k_cache[where, :, place], y[lo:hi, heads:], bound[lo:hi, heads:], "keys")
        assert torch.equal(b.v_cache[where, :, place].double(), v[lo:hi])
        for cache, old in zip((b.k_cache, b.v_cache), before):
            cache[where, :, place] = old[where, :, place]
    for cache, old in zip((b.k_cache, b.v_cache), before):  # nothing else was touched
        assert same_bits(cache, old)


@pytest.mark.parametrize("which", ["", "q", "k", "qk"])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,rotary,interleaved", APPENDS)
def test_four_bit_append(ops, lib, contexts, counts, heads, kv_heads, dim, page, rotary, interleaved, which):
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, page, extra_rows=3)
    columns = (heads + 2 * kv_heads) * dim
    qkv = torch.randn((b.rows, columns + 24), device="cuda").to(torch.float16)[:, 8:8 + columns]
    qkv[0, -dim:] = 0.375  # a step of zero
    w = norms(dim, which)
    y, bound, v, rotary_args = turned(lib, b, qkv, rotary, interleaved, *w, 1e-6)
    want_k, want_v = b.k_cache.clone(), b.v_cache.clone()
    q = ops.four_bit_append(qkv, *b.arrays, *w, 1e-6, *rotary_args)
    owned = b.cut[-1]
    near(q[:owned].view(owned, heads, dim), y[:, :heads], bound[:, :heads], "queries")
    for s, (c, t) in enumerate(zip(contexts, counts)):
        lo, hi = b.cut[s], b.cut[s + 1]
        where, place = b.pages_of(s, torch.arange(c, c + t, device="cuda"))
        at = (where, slice(None), place)
        four.put(want_v, dim, at, v[lo:hi])
        # Keys: scales and codes as the definition makes them of keys in 32 bits, which are off by what `bound` has beyond fp16's
        # rounding.  Scales are rounded once; a code then stands for an element half a step away at most, or is the first or last.
        k, off = y[lo:hi, heads:], bound[lo:hi, heads:] - 2.0 ** -11 * y[lo:hi, heads:].abs()
        kept, step, low = four.values(b.k_cache, dim, at)
        least, most, off_all = (k.unflatten(-1, (-1, 64)).amin(-1), k.unflatten(-1, (-1, 64)).amax(-1), off.unflatten(-1, (-1, 64)).amax(-1))
        least, most, off_all = (x.repeat_interleave(64, -1) for x in (least, most, off_all))
        assert bool(((low - least).abs() <= 2.0 ** -11 * least.abs() + off_all + 2.0 ** -25).all())
        assert bool(((15 * step - (most - low)).abs() <= 2.0 ** -11 * 15 * step + 15 * 2.0 ** -25 + off_all + 2.0 ** -22 * (most - low)).all())
        inside = torch.minimum(torch.maximum(k, low), low + 15 * step)
        assert bool(((kept - inside).abs() <= step * (0.5 + 2.0 ** -20) + off_all).all())
        four.parts(want_k, dim)[0][at], four.parts(want_k, dim)[1][at] = (part[at] for part in four.parts(b.k_cache, dim))
    assert same_bits(b.v_cache, want_v) and same_bits(b.k_cache, want_k)  # values exactly, and nothing else was touched


def test_groups_that_are_not_finite_and_extremes(ops, lib):
    b = FourBitBatch([3], [6], 2, 1, 128, 16)
    qkv = torch.randn((6, 4 * 128), device="cuda").to(torch.float16)
    v = qkv[:, 3 * 128:]
    v[0, 5], v[1, 64], v[2, 127] = float("nan"), float("inf"), float("-inf")
    v[3, 0], v[3, 1] = 65504.0, -65504.0
    v[4] = 2.0 ** -24
    v[4, 3] = 0.0
    k = qkv[:, 2 * 128:3 * 128]
    k[5] = 60000.0  # turned, beyond fp16's range
    f = torch.from_numpy(lib.rotary_frequencies(128)[0]).cuda()
    ops.four_bit_append(qkv, *b.arrays, None, None, 1e-6, f)
    keys, vals = ops.four_bit_read(*b.arrays, 6)
    bad = torch.isnan(vals).view(6, 2, 64)
    assert bad.all(-1).tolist() == [[True, False], [False, True], [False, True], [False, False], [False, False], [False, False]]
    assert torch.equal(bad.all(-1), bad.any(-1))
    assert float(vals[3, 0]) == 65504.0 and float(vals[3, 1]) == -65504.0
    assert bool((vals[4].abs() <= 2.0 ** -23).all())
    assert bool(torch.isnan(keys[5]).any()) and bool(torch.isfinite(keys[:5]).all())


READS = [([0], [1], 1, 64, 16), ([5, 0, 31], [1, 3, 2], 2, 64, 16), ([0, 7, 0, 64], [170, 0, 33, 1], 3, 128, 32), ([0], [5000], 2, 128, 128),
         ([3] * 90, [2] * 90, 1, 64, 64)]


@pytest.mark.parametrize("contexts,counts,kv_heads,dim,page", READS)
def test_four_bit_read(ops, contexts, counts, kv_heads, dim, page):
    b = FourBitBatch(contexts, counts, kv_heads, kv_heads, dim, page)
    keys, vals = ops.four_bit_read(*b.arrays, b.rows + 2)
    for s, (c, t) in enumerate(zip(contexts, counts)):
        for got, cache in ((keys, b.k_cache), (vals, b.v_cache)):
            want = b.rows_of(cache, s)[c:]
            near(got[b.cut[s]:b.cut[s + 1]].view(t, kv_heads, dim), want, 2.0 ** -11 * want.abs() + 2.0 ** -25)


# --------------------------------------------------------------------------------------------------- attention

ATTENTIONS = [
    # contexts, counts, heads, kv_heads, dim, page, window, sinks, cap, slopes
    ([0], [1], 1, 1, 64, 16, 0, 0, 0.0, False),
    ([0], [1], 1, 1, 128, 16, 1, 0, 0.0, False),
    ([210], [1], 16, 16, 64, 16, 0, 0, 0.0, False),
    ([15, 16, 17, 31, 32, 33], [1] * 6, 4, 2, 128, 16, 0, 0, 0.0, False),
    ([0, 5, 300, 0, 1000], [1, 1, 1, 0, 1], 8, 2, 128, 32, 100, 4, 0.0, False),
    ([700, 3], [1, 1], 8, 1, 64, 64, 1, 1, 0.0, True),
    ([2000], [1], 64, 8, 128, 64, 0, 0, 30.0, False),
    ([2000], [1], 64, 8, 128, 64, 257, 130, 30.0, True),
    ([900, 100], [3, 2], 12, 4, 128, 16, 0, 0, 0.0, True),
    ([900, 100], [3, 2], 12, 4, 128, 16, 64, 16, 0.0, False),
    ([500], [2], 40, 2, 64, 32, 0, 0, 0.0, False),
    ([0], [200], 2, 2, 64, 16, 0, 0, 0.0, False),
    ([0], [200], 2, 2, 64, 16, 13, 3, 0.0, False),
    ([130, 0, 77], [300, 1, 129], 8, 2, 128, 128, 0, 0, 0.0, False),
    ([130, 0, 77], [300, 1, 129], 8, 2, 128, 128, 128, 0, 0.0, False),
    ([130, 0, 77], [300, 1, 129], 8, 2, 128, 32, 129, 127, 50.0, False),
    ([0, 1000], [700, 40], 5, 1, 128, 256, 255, 128, 0.0, True),
    ([3000], [260], 4, 4, 128, 64, 384, 300, 0.0, False),
    ([3000], [260], 4, 4, 64, 64, 2000, 1500, 20.0, True),
    ([600], [90], 128, 1, 128, 64, 50, 7, 0.0, False),
    ([40] * 40, [1, 2] * 20, 6, 2, 64, 16, 8, 2, 0.0, False),
    ([1000], [33], 8, 8, 128, 64, 5000, 9000, 0.0, False),
]


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,window,sinks,cap,distance", ATTENTIONS)
def test_window_attention(ops, contexts, counts, heads, kv_heads, dim, page, window, sinks, cap, distance):
    b = Batch(contexts, counts, heads, kv_heads, dim, page, gain=2.0)
    slopes = slopes_of(heads) if distance else None
    window = window or 77
    want, bound = four.attention(b, window, sinks, cap=cap, slopes=slopes)
    near(ops.window_attention(b.q, *b.arrays, window, sinks, cap=cap, slopes=slopes), want, bound)


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,window,sinks,cap,distance", ATTENTIONS)
def test_four_bit_attention(ops, contexts, counts, heads, kv_heads, dim, page, window, sinks, cap, distance):
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, page, gain=2.0)
    slopes = slopes_of(heads) if distance else None
    want, bound = four.attention(b, window, sinks, cap=cap, slopes=slopes)
    near(ops.four_bit_attention(b.q, *b.arrays, window, sinks, cap=cap, slopes=slopes), want, bound)


def test_a_window_over_everything_is_none(ops):
    b = Batch([500, 3], [40, 200], 8, 2, 128, 32)
    want = ops.prompt_attention(b.q, *b.arrays)
    assert torch.equal(ops.window_attention(b.q, *b.arrays, 1 << 20), want)
    near(ops.window_attention(b.q, *b.arrays, 540, 0), *four.attention(b))


WINDOWS = [([700], [1], 8, 2, 128), ([700], [40], 2, 2, 64), ([300], [260], 8, 8, 128), ([0], [500], 16, 1, 64), ([900, 5], [3, 1], 4, 4, 128)]


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim", WINDOWS)
def test_what_lies_outside_a_window_does_not_matter(ops, contexts, counts, heads, kv_heads, dim, what):
    """Keys and values that a row does not see are not finite: those behind the window of a sequence's first row for all, the first
    row's for all others."""
    window, sinks = 100, 5
    b = Batch(contexts, counts, heads, kv_heads, dim, 32)
    want = ops.window_attention(b.q, *b.arrays, window, sinks)
    kept = want.clone()
    for s, (c, t) in enumerate(zip(contexts, counts)):
        first = max(sinks, c - window + 1)  # first key, sinks aside, of the sequence's first row
        hidden = torch.arange(sinks, first, device="cuda")
        where, place = b.pages_of(s, hidden)
        b.k_cache[where, :, place] = what
        b.v_cache[where, :, place] = what
    assert torch.equal(ops.window_attention(b.q, *b.arrays, window, sinks), kept)
    for s, (c, t) in enumerate(zip(contexts, counts)):
        key = max(sinks, c - window + 1)  # in sight of the first row alone
        if c < sinks + window or t < 2:
            continue
        where, place = b.pages_of(s, torch.tensor([key], device="cuda"))
        b.v_cache[where, :, place, 1] = what
        got = ops.window_attention(b.q, *b.arrays, window, sinks).view(b.rows, heads, dim)
        rest = kept.view(b.rows, heads, dim)
        assert torch.equal(got[b.cut[s] + 1:b.cut[s + 1]], rest[b.cut[s] + 1:b.cut[s + 1]])
        mine = got[b.cut[s]]
        assert bool((torch.isnan(mine[:, 1]) if what != what else mine[:, 1] == what).all())
        mine, other = mine.clone(), rest[b.cut[s]].clone()
        mine[:, 1] = other[:, 1] = 0
        assert torch.equal(mine, other)


@pytest.mark.parametrize("heads,kv_heads,dim,context,count", [(8, 2, 128, 600, 1), (64, 1, 64, 600, 3), (4, 4, 128, 0, 300), (2, 2, 64, 40, 20)])
def test_infinite_values_within_a_window_reach_those_who_see_them(ops, heads, kv_heads, dim, context, count):
    b = Batch([context], [count], heads, kv_heads, dim, 16)
    window, sinks = 300, 2
    finite = ops.window_attention(b.q, *b.arrays, window, sinks).view(count, heads, dim)
    keys = [0, max(0, context + count - 150), context + count - 1]
    for i, key in enumerate(keys):
        where, place = b.pages_of(0, torch.tensor([key], device="cuda"))
        b.v_cache[where, :, place, 3 + i] = float("inf") if i % 2 else float("-inf")
    got = ops.window_attention(b.q, *b.arrays, window, sinks).view(count, heads, dim)
    row = context + torch.arange(count, device="cuda")
    for i, key in enumerate(keys):
        sees = (key <= row) & ((row - key < window) | (key < sinks))
        assert bool((got[sees][:, :, 3 + i] == (float("inf") if i % 2 else float("-inf"))).all())
        assert torch.equal(got[~sees][:, :, 3 + i], finite[~sees][:, :, 3 + i])
    rest = [c for c in range(dim) if not 3 <= c < 3 + len(keys)]
    assert torch.equal(got[..., rest], finite[..., rest])


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim", WINDOWS)
def test_groups_without_numbers_reach_those_who_see_them_in_four_bits(ops, contexts, counts, heads, kv_heads, dim):
    window, sinks = 100, 5
    b = FourBitBatch(contexts, counts, heads, kv_heads, dim, 32)
    want = ops.four_bit_attention(b.q, *b.arrays, window, sinks).view(b.rows, heads, dim)
    context, count = contexts[0], counts[0]
    key = max(sinks, context - window + 1)  # in sight of the first row, and of those so near
    where, place = b.pages_of(0, torch.tensor([key], device="cuda"))
    scales = four.parts(b.v_cache, dim)[1]
    scales[where, :, place, -1, 0] = float("nan")
    got = ops.four_bit_attention(b.q, *b.arrays, window, sinks).view(b.rows, heads, dim)
    row = torch.arange(context, context + count, device="cuda")
    sees = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
    sees[:count] = (key <= row) & ((row - key < window) | (key < sinks))
    assert bool(torch.isnan(got[sees][..., -64:]).all()) and torch.equal(got[sees][..., :-64], want[sees][..., :-64])
    assert torch.equal(got[~sees], want[~sees])
    four.parts(b.k_cache, dim)[1][where, :, place, 0, 1] = float("inf")  # a key: all of a row
    got = ops.four_bit_attention(b.q, *b.arrays, window, sinks).view(b.rows, heads, dim)
    assert bool(torch.isnan(got[sees]).all()) and torch.equal(got[~sees], want[~sees])


@pytest.mark.parametrize("count,heads", [(1, 1), (3, 4), (40, 2), (300, 1)])
def test_steps_of_very_different_sizes(ops, count, heads):
    """Values 2^16 times as large, of a key with a small weight, and back: what the others add is not lost."""
    b = FourBitBatch([500], [count], heads, 1, 128, 16)
    dim = 128
    scales = four.parts(b.v_cache, dim)[1]
    for key, factor in ((0, 2.0 ** 10), (200, 2.0 ** -10), (333, 2.0 ** 10)):
        where, place = b.pages_of(0, torch.tensor([key], device="cuda"))
        scales[where, :, place] *= factor
    want, bound = four.attention(b)
    near(ops.four_bit_attention(b.q, *b.arrays), want, bound)


@pytest.mark.parametrize("count,heads,dim,cap", [(1, 1, 64, 0.0), (40, 2, 128, 0.0), (300, 1, 64, 0.0), (150, 1, 128, 300.0)])
def test_long_flat_tails_are_not_lost_in_four_bits(ops, count, heads, dim, cap):
    """One key far above 20000 others whose weights together are of some size: 2^-18 of the largest each."""
    b = FourBitBatch([20000], [count], heads, heads, dim, 64)
    codes, scales = four.parts(b.k_cache, dim)
    codes[:], scales[..., 0], scales[..., 1] = 0, 0.0, 0.0
    where, place = b.pages_of(0, torch.tensor([7], device="cuda"))
    scales[where, :, place, 0, 1] = 1.0
    b.q[:] = 0
    b.q.view(count, heads, dim)[:, :, 0] = 12.5
    want, bound = four.attention(b, scale=1.0, cap=cap)
    near(ops.four_bit_attention(b.q, *b.arrays, scale=1.0, cap=cap), want, bound)


@pytest.mark.parametrize("count", [1, 3, 40, 300])
def test_averages_of_the_largest_value_are_that_value_in_four_bits(ops, count):
    b = FourBitBatch([11], [count], 2, 1, 64, 16)
    codes, scales = four.parts(b.v_cache, 64)
    codes[:] = 0x0f  # even elements 15, odd ones 0
    scales[..., 0], scales[..., 1] = 8736.0, -65504.0
    got = ops.four_bit_attention(b.q, *b.arrays).view(count, 2, 64)
    assert bool((got[..., 0::2] >= 65472).all()) and bool((got[..., 1::2] == -65504).all())


@pytest.mark.parametrize("count,gain", [(1, 300.0), (40, 300.0), (1, 3e4), (200, 3e4)])
def test_large_scores_in_four_bits(ops, count, gain):
    b = FourBitBatch([200], [count], 4, 2, 128, 32)
    b.q = (b.q.float() * gain).clamp(-65504, 65504).half()
    got = ops.four_bit_attention(b.q, *b.arrays, scale=1.0)
    v = [b.rows_of(b.v_cache, 0)[..., c] for c in (0, 1)]
    assert bool(torch.isfinite(got).all()) and float(got.abs().max()) <= 1.001 * float(b.rows_of(b.v_cache, 0).abs().max()) and v
    want, bound = four.attention(b, scale=1.0)
    ok = bound < 0.5  # where the scores' own errors leave an answer
    assert bool(((got.double() - want).abs()[ok] <= bound[ok]).all())


# --------------------------------------------------------------------------------------------------- batches

def calls(ops, b, window=50, sinks=3):
    if isinstance(b, FourBitBatch):
        return ops.four_bit_attention(b.q, *b.arrays, window, sinks)
    return ops.window_attention(b.q, *b.arrays, window, sinks)


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_strided_queries_and_rows_of_nobody(ops, lib, kind):
    b = kind([60, 200], [5, 70], 4, 2, 64, 16, extra_rows=4)
    want = calls(ops, b)
    wide = torch.full((b.rows, 4 * 64 + 40), float("nan"), device="cuda", dtype=torch.float16)
    wide[:, 16:16 + 256] = b.q
    wide[b.cut[-1]:] = float("nan")
    q = b.q
    b.q = wide[:, 16:16 + 256]
    assert torch.equal(calls(ops, b)[:b.cut[-1]], want[:b.cut[-1]])
    b.q = q
    out = torch.full((b.rows, 256), 7.0, device="cuda", dtype=torch.float16)
    workspace = torch.empty(lib.attention_workspace_bytes(64), dtype=torch.uint8, device="cuda")
    args = lib.PagedBatch(b.k_cache.data_ptr(), b.v_cache.data_ptr(), b.k_cache.shape[0], 16, 2, 64, b.cu_tokens.data_ptr(),
                          b.context.data_ptr(), b.page_table.data_ptr(), b.page_table.shape[1], 2, b.rows)
    call = lib.four_bit_attention if kind is FourBitBatch else lib.window_attention
    call(torch.cuda.current_stream().cuda_stream, q.data_ptr(), 256, args, 4, out.data_ptr(), workspace.data_ptr(), 50, 3)
    assert torch.equal(out[:b.cut[-1]], want[:b.cut[-1]]) and bool((out[b.cut[-1]:] == 7).all())


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_repeated_calls_give_the_same_bits(ops, kind):
    for contexts, counts in (([5000, 17, 900], [1, 1, 1]), ([300, 0], [500, 130])):
        b = kind(contexts, counts, 8, 2, 128, 64)
        first = calls(ops, b, 2000)
        for _ in range(5):
            assert torch.equal(calls(ops, b, 2000), first)


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 40, 150]])
def test_bad_pages_and_lengths_are_reported(ops, lib, kind, counts):
    b = kind([100, 250, 300], counts, 4, 2, 64, 16)
    want, bound = four.attention(b, 2000)
    zeros = kind([100, 250, 300], counts, 4, 2, 64, 16)
    for cache in (zeros.k_cache, zeros.v_cache):
        cache[zeros.page_table[1, 3].long()] = 0
    by_zeros, zero_bound = four.attention(zeros, 2000)
    for bad in (-1, b.k_cache.shape[0], 1 << 30):
        table = b.page_table.clone()
        table[1, 3] = bad
        arrays = (b.k_cache, b.v_cache, b.cu_tokens, b.context, table)
        got = (ops.four_bit_attention if kind is FourBitBatch else ops.window_attention)(b.q, *arrays, 2000)
        assert lib.consume_status() == BAD_CACHE
        lo, hi = b.cut[1], b.cut[2]
        near(got[:lo], want[:lo], bound[:lo])
        near(got[hi:], want[hi:], bound[hi:])
        near(got[lo:hi], by_zeros[lo:hi], zero_bound[lo:hi])
    for context in (-1, b.page_table.shape[1] * 16, 2 ** 31 - 1):
        lengths = b.context.clone()
        lengths[1] = context
        arrays = (b.k_cache, b.v_cache, b.cu_tokens, lengths, b.page_table)
        got = (ops.four_bit_attention if kind is FourBitBatch else ops.window_attention)(b.q, *arrays, 2000)
        assert lib.consume_status() == BAD_CACHE
        near(got[:b.cut[1]], want[:b.cut[1]], bound[:b.cut[1]])
        near(got[b.cut[2]:], want[b.cut[2]:], bound[b.cut[2]:])
        assert bool((got[b.cut[1]:b.cut[2]] == 0).all())


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_appends_of_sequences_that_do_not_fit(ops, lib, kind):
    b = kind([30, 62, 9], [2, 5, 3], 4, 2, 64, 16)
    b.context[1] = b.page_table.shape[1] * 16 - 4
    qkv = torch.randn((10, 8 * 64), device="cuda").to(torch.float16)
    w = norms(64)
    append = ops.four_bit_append if kind is FourBitBatch else ops.norm_rotary_append
    before = b.k_cache.clone(), b.v_cache.clone()
    q = append(qkv, *b.arrays, *w)
    assert lib.consume_status() == BAD_CACHE
    assert bool((q[2:7] == 0).all()) and bool((q[:2] != 0).any()) and bool((q[7:] != 0).any())
    table = b.page_table.clone()
    table[1] = -1  # nor to a bad page
    b.context[1] = 62
    append(qkv, b.k_cache, b.v_cache, b.cu_tokens, b.context, table, *w)
    assert lib.consume_status() == BAD_CACHE
    where, _ = b.pages_of(1, torch.arange(67, device="cuda"))
    for cache, old in zip((b.k_cache, b.v_cache), before):
        assert same_bits(cache[where], old[where])
    if kind is FourBitBatch:
        keys, vals = ops.four_bit_read(b.k_cache, b.v_cache, b.cu_tokens, b.context, table, 10)
        assert lib.consume_status() == BAD_CACHE
        assert bool((keys[2:7] == 0).all()) and bool((vals[2:7] == 0).all()) and bool((keys[:2] != 0).any())
        b.context[1] = -1
        keys, vals = ops.four_bit_read(*b.arrays, 10)
        assert lib.consume_status() == BAD_CACHE
        assert bool((keys[2:7] == 0).all()) and bool((vals[7:] != 0).any())


@pytest.mark.parametrize("page", [16, 128])
def test_four_bit_caches_longer_than_32_bits(ops, page):
    """Pages whose bytes lie beyond 2^32 from the start of the cache."""
    kv_heads, dim = 4, 128
    pages = (1 << 32) // (kv_heads * page * 72) + 40
    caches = [torch.empty((pages, kv_heads, page, 72), dtype=torch.uint8, device="cuda") for _ in range(2)]
    count = 3 * page + 5
    used = torch.tensor([[pages - 1, 3, pages - 20, pages - 7]], dtype=torch.int32, device="cuda")
    cu, zero = torch.tensor([0, count], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    qkv = torch.randn((count, 12 * dim), device="cuda").to(torch.float16)
    small = [torch.empty((4, kv_heads, page, 72), dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device="cuda")
    answers = []
    for (k, v), at in ((caches, used), (small, table)):
        q = ops.four_bit_append(qkv, k, v, cu, zero, at)
        last = q[-1:].contiguous()
        one, context = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([count - 1], dtype=torch.int32, device="cuda")
        answers.append((q, *ops.four_bit_read(k, v, cu, zero, at, count), ops.four_bit_attention(q, k, v, cu, zero, at),
                        ops.four_bit_attention(last, k, v, one, context, at)))
    for x, y in zip(*answers):
        assert torch.equal(x, y)


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_captured_calls_follow_the_arrays(ops, lib, kind):
    """A step captured once and replayed with other lengths and pages, two graphs on two streams at once."""
    w = norms(128)
    steps = []
    for seed in (1, 2):
        b = kind([300, 40, 0], [1, 1, 1], 8, 2, 128, 16, seed=seed, spare_pages=8)
        b.qkv = torch.randn((3, 12 * 128), device="cuda").to(torch.float16)
        append = ops.four_bit_append if kind is FourBitBatch else ops.norm_rotary_append

        def step(b=b, append=append):
            b.q = append(b.qkv, *b.arrays, *w)
            return b.q, calls(ops, b, 100)

        step()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        steps.append((b, step, graph, stream, out))
    for turn, contexts in enumerate(([300, 40, 0], [17, 333, 5], [0, 0, 319])):
        got = []
        for b, step, graph, stream, out in steps:
            b.context.copy_(torch.tensor(contexts, dtype=torch.int32))
            b.qkv.copy_(torch.randn((3, 12 * 128), generator=torch.Generator().manual_seed(turn)).half())
            # Where the batch had no room for such lengths, all of its pages are dealt out again.
            pages = torch.randperm(b.k_cache.shape[0], generator=torch.Generator().manual_seed(turn)).int()
            b.page_table.copy_(pages[torch.arange(3)[:, None] * 7 % len(pages) + torch.arange(b.page_table.shape[1])[None] % 7])
            if kind is FourBitBatch:
                b.k_cache.fill_(17), b.v_cache.fill_(18)
            else:
                b.k_cache.fill_(0.5), b.v_cache.fill_(0.25)
        torch.cuda.synchronize()
        for b, step, graph, stream, out in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for b, step, graph, stream, out in steps:
            got.append([x.clone() for x in out])
            for x, y in zip(step(), got[-1]):
                assert torch.equal(x, y)
        assert lib.consume_status() == (BAD_CACHE if max(contexts) >= 304 else 0)  # 19 pages of a table's row


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_another_stream(ops, kind):
    b = kind([2000, 5], [1, 30], 8, 2, 64, 32)
    want = calls(ops, b, 700)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls(ops, b, 700)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv_heads,dim,window", [(8, 2, 128, 0), (4, 4, 64, 40), (12, 1, 128, 150)])
def test_prompts_in_pieces_and_single_tokens_in_four_bits(ops, lib, heads, kv_heads, dim, window):
    """A prompt appended and attended at once, in two pieces, and token by token: the cache has the same bytes, the rows are near."""
    count = 190
    f = torch.from_numpy(lib.rotary_frequencies(dim)[0]).cuda()
    w = norms(dim)
    qkv = torch.randn((count, (heads + 2 * kv_heads) * dim), device="cuda").to(torch.float16)
    outs, caches = [], []
    for pieces in ([count], [77, count - 77], [150] + [1] * (count - 150)):
        b = FourBitBatch([0], [count], heads, kv_heads, dim, 16)
        at, rows = 0, []
        for n in pieces:
            cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            context = torch.tensor([at], dtype=torch.int32, device="cuda")
            batch = (b.k_cache, b.v_cache, cu, context, b.page_table)
            b.q = ops.four_bit_append(qkv[at:at + n], *batch, *w, 1e-6, f)
            rows.append(ops.four_bit_attention(b.q, *batch, window, 2))
            at += n
        outs.append(torch.cat(rows))
        caches.append((b.k_cache, b.v_cache))
    b.q = ops.four_bit_append(qkv, b.k_cache, b.v_cache, torch.tensor([0, count], dtype=torch.int32, device="cuda"),
                              torch.zeros(1, dtype=torch.int32, device="cuda"), b.page_table, *w, 1e-6, f)
    b.contexts, b.counts, b.cut, b.rows = [0], [count], [0, count], count
    want, bound = four.attention(b, window, 2)
    for out, cache in zip(outs, caches):
        near(out, want, bound)
        assert same_bits(cache[0], caches[0][0]) and same_bits(cache[1], caches[0][1])


@pytest.mark.parametrize("four_bit", [False, True])
def test_cached_attention_with_norms_a_window_and_four_bits(ops, lib, four_bit):
    """The layer chain's attention: prompts, then single tokens, against the definition over what the cache holds."""
    from flash_llm_b200.tp_chain import CachedAttention
    heads, dim = 6, 64
    kind = FourBitBatch if four_bit else Batch
    b = kind([0, 0], [60, 9], heads, heads, dim, 16, spare_pages=4)
    q_norm, k_norm = norms(dim)
    f = torch.from_numpy(lib.rotary_frequencies(dim)[0]).cuda()
    layer = CachedAttention(b.k_cache, b.v_cache, b.cu_tokens, b.context, b.page_table, frequencies=f, q_norm=q_norm, k_norm=k_norm,
                            window=20, sinks=2)
    for counts in ([50, 5], [1, 1], [3, 2]):
        done = b.context.tolist()
        layer.cu_tokens = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device="cuda")
        y_qkv = torch.randn((sum(counts), 3 * heads * dim), device="cuda").to(torch.float16)
        got = layer(y_qkv)
        b.contexts, b.counts, b.cut, b.rows = done, counts, [0, counts[0], sum(counts)], sum(counts)
        y, bound_q, _, _ = turned(lib, b, y_qkv, 0, False, q_norm, k_norm, 1e-6)
        append = ops.four_bit_append if four_bit else ops.norm_rotary_append
        b.q = append(y_qkv, b.k_cache.clone(), b.v_cache.clone(), layer.cu_tokens, b.context, b.page_table, q_norm, k_norm, 1e-6, f)
        want, bound = four.attention(b, 20, 2)
        near(got, want, bound)
        b.context += torch.tensor(counts, dtype=torch.int32, device="cuda")


def test_refusals_of_the_operators(ops):
    b, c = Batch([9], [3], 4, 2, 64, 16), FourBitBatch([9], [3], 4, 2, 64, 16)
    qkv = torch.randn((3, 8 * 64), device="cuda").to(torch.float16)
    w = norms(64)
    for bad in ((w[0].float(), w[1]), (w[0][:32], w[1]), (w[0], w[1].cpu())):
        with pytest.raises(RuntimeError, match="norm must be"):
            ops.norm_rotary_append(qkv, *b.arrays, *bad)
        with pytest.raises(RuntimeError, match="norm must be"):
            ops.four_bit_append(qkv, *c.arrays, *bad)
    with pytest.raises(RuntimeError, match="eps"):
        ops.norm_rotary_append(qkv, *b.arrays, *w, -1.0)
    for call in (lambda: ops.norm_rotary_append(qkv, *c.arrays, *w), lambda: ops.window_attention(c.q, *c.arrays, 5),
                 lambda: ops.prompt_attention(c.q, *c.arrays)):
        with pytest.raises(RuntimeError, match="fp16 tensor"):
            call()
    for call in (lambda: ops.four_bit_append(qkv, *b.arrays), lambda: ops.four_bit_attention(b.q, *b.arrays),
                 lambda: ops.four_bit_read(*b.arrays, 3)):
        with pytest.raises(RuntimeError, match="uint8 tensor"):
            call()
    with pytest.raises(RuntimeError, match="36 or 72"):
        ops.four_bit_read(c.k_cache[..., :32].contiguous(), c.v_cache[..., :32].contiguous(), *c.arrays[2:], 3)
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(RuntimeError, match="window"):
            ops.window_attention(b.q, *b.arrays, window, sinks)
    with pytest.raises(RuntimeError, match="window"):
        ops.four_bit_attention(c.q, *c.arrays, -1)
    with pytest.raises(RuntimeError, match="tokens"):
        ops.four_bit_read(*c.arrays, -1)
    assert ops.four_bit_read(*c.arrays, 0)[0].shape == (0, 128)


# --------------------------------------------------------------------------------------------------- where single tokens go another way

@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,window,sinks,cap,distance", [
    ([300, 5, 9, 0], [3, 0, 0, 1], 8, 2, 128, 16, 100, 3, 0.0, False),      # no more tokens than sequences, but several of one
    ([300] + [0] * 9, [9] + [0] * 9, 12, 1, 64, 32, 40, 0, 0.0, True),
    ([1000] * 3, [1] * 3, 40, 2, 128, 64, 333, 17, 25.0, False),            # more heads of a group than a tile's eight rows
    ([5000], [1], 128, 1, 64, 128, 4000, 128, 0.0, False),
    ([31, 32, 33, 47, 48, 49], [1] * 6, 3, 3, 128, 16, 16, 16, 0.0, False),
    ([400] * 20, [1] * 20, 64, 2, 128, 64, 150, 4, 0.0, False),             # more than a tile takes of one token, many and few
    ([400, 90], [1, 1], 96, 2, 64, 32, 150, 4, 0.0, True),
    ([300, 20, 77], [2, 1, 2], 8, 2, 128, 16, 64, 0, 0.0, False),           # two tokens of some
    ([300, 20, 77, 5], [40, 1, 2, 1], 2, 2, 64, 16, 64, 0, 0.0, False),     # few rows on average, many of one
    ([300, 20], [17, 33], 4, 4, 64, 16, 0, 0, 0.0, False),
    ([700] * 450, [1] * 450, 2, 1, 64, 16, 30, 2, 0.0, False),
])
@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_no_more_tokens_than_sequences(ops, kind, contexts, counts, heads, kv_heads, dim, page, window, sinks, cap, distance):
    b = kind(contexts, counts, heads, kv_heads, dim, page, gain=2.0)
    slopes = slopes_of(heads) if distance else None
    want, bound = four.attention(b, window, sinks, cap=cap, slopes=slopes)
    call = ops.four_bit_attention if kind is FourBitBatch else ops.window_attention
    near(call(b.q, *b.arrays, window or (0 if kind is FourBitBatch else 1 << 20), sinks, cap=cap, slopes=slopes), want, bound)


@pytest.mark.parametrize("count", [1, 40])
def test_long_flat_tails_through_a_window(ops, count):
    """One key far above 15000 others whose weights together are of some size: 2^-18 of the largest each."""
    b = Batch([20000], [count], 2, 1, 64, 64)
    b.k_cache[:] = 0
    where, place = b.pages_of(0, torch.tensor([19000], device="cuda"))
    b.k_cache[where, :, place, 0] = 1.0
    b.q[:] = 0
    b.q.view(count, 2, 64)[:, :, 0] = 12.5
    want, bound = four.attention(b, 15000, 5, scale=1.0)
    near(ops.window_attention(b.q, *b.arrays, 15000, 5, scale=1.0), want, bound)


@pytest.mark.parametrize("count", [1, 3, 40])
@pytest.mark.parametrize("value", [65504.0, -65504.0])
def test_averages_of_the_largest_value_through_a_window(ops, count, value):
    b = Batch([300], [count], 4, 1, 128, 16)
    b.v_cache[:] = value
    assert bool((ops.window_attention(b.q, *b.arrays, 100, 3) == value).all())


@pytest.mark.parametrize("count", [1, 60])
def test_scores_beyond_what_their_exponents_hold_through_a_window(ops, count):
    """Scores of 2^26 and more that differ by a few: what is left of the weights is theirs alone."""
    b = Batch([200], [count], 2, 2, 64, 16)
    b.k_cache[:] = 0
    b.q[:] = 0
    b.q.view(count, 2, 64)[:, :, 0] = 1024.0
    b.q.view(count, 2, 64)[:, :, 1] = 1.0
    rows = torch.arange(200 + count, device="cuda")
    where, place = b.pages_of(0, rows)
    b.k_cache[where, :, place, 0] = 32768.0
    b.k_cache[where, :, place, 1] = ((rows % 3) * 4.0).half()[:, None].expand(-1, 2)
    # products: 2^25 exactly and 0, 4 or 8, sums of 32 bits in steps of 4; times 2^2
    want, _ = four.attention(b, 90, 2, scale=4.0)
    got = ops.window_attention(b.q, *b.arrays, 90, 2, scale=4.0)
    assert bool(((got.double() - want).abs() <= 2.0 ** -10 * (want.abs() + 4)).all())


@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_infinite_values_with_weights_too_small_through_a_window(ops, what):
    for count, heads in ((1, 4), (1, 20), (30, 4)):
        b = Batch([900], [count], heads, 1, 128, 16)
        b.k_cache[:] = 0
        b.q[:] = 0
        b.q.view(count, heads, 128)[:, :, 0] = 60.0
        where, place = b.pages_of(0, torch.tensor([880], device="cuda"))
        b.k_cache[where, :, place, 0] = 1.0  # all others' weights: e^-60
        finite = ops.window_attention(b.q, *b.arrays, 400, 2, scale=1.0)
        where, place = b.pages_of(0, torch.tensor([700], device="cuda"))
        b.v_cache[where, :, place, 9] = what
        got = ops.window_attention(b.q, *b.arrays, 400, 2, scale=1.0).view(count, heads, 128)
        assert bool((torch.isnan(got[..., 9]) if what != what else got[..., 9] == what).all())
        rest = [c for c in range(128) if c != 9]
        assert torch.equal(got[..., rest], finite.view(count, heads, 128)[..., rest])


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
def test_as_many_sequences_as_a_call_can_have(ops, kind):
    """4096 of them, every third without a token, every thousandth with many."""
    contexts = [(7 * i) % 50 for i in range(4096)]
    for many in (0, 20):
        counts = [0 if i % 3 == 1 else many + 1 if i % 1000 == 5 else 1 for i in range(4096)]
        b = kind(contexts, counts, 2, 1, 64, 16)
        want, bound = four.attention(b, 11, 3)
        qkv = torch.randn((b.rows, 4 * 64), device="cuda").to(torch.float16)
        call = ops.four_bit_attention if kind is FourBitBatch else ops.window_attention
        near(call(b.q, *b.arrays, 11, 3), want, bound)
        w = norms(64)
        y, off, v, _ = turned(None, b, qkv, 0, False, *w, 1e-6)
        q = (ops.four_bit_append if kind is FourBitBatch else ops.norm_rotary_append)(qkv, *b.arrays, *w)
        near(q.view(b.rows, 2, 64), y[:, :2], off[:, :2])
        kept = torch.cat([b.rows_of(b.v_cache, s)[c:] for s, c in enumerate(contexts) if counts[s]])
        if kind is FourBitBatch:
            keys, vals = ops.four_bit_read(*b.arrays, b.rows)
            near(vals.view(b.rows, 1, 64), kept, 2.0 ** -11 * kept.abs() + 2.0 ** -25)
        else:
            assert torch.equal(kept, v)


@pytest.mark.parametrize("kind", [Batch, FourBitBatch])
@pytest.mark.parametrize("counts", [[1, 1, 1, 0], [1, 2, 0, 30]])
@pytest.mark.parametrize("heads", [2, 24, 80, 256])  # one to 128 query heads of a key/value head
def test_bad_pages_and_lengths_within_a_window(ops, lib, kind, counts, heads):
    contexts, window, sinks = [100, 250, 300, 40], 100, 60  # the bad page is one of the first, behind it one that none sees
    b = kind(contexts, counts, heads, 2, 64, 16, extra_rows=3)
    want, bound = four.attention(b, window, sinks)
    zeros = kind(contexts, counts, heads, 2, 64, 16, extra_rows=3)
    for cache in (zeros.k_cache, zeros.v_cache):
        cache[zeros.page_table[1, 3].long()] = 0
    by_zeros, zero_bound = four.attention(zeros, window, sinks)
    call = ops.four_bit_attention if kind is FourBitBatch else ops.window_attention
    lo, hi, last = b.cut[1], b.cut[2], b.cut[-1]
    for bad in (-1, b.k_cache.shape[0], 2 ** 31 - 1):
        table = b.page_table.clone()
        table[1, 3] = bad
        got = call(b.q, b.k_cache, b.v_cache, b.cu_tokens, b.context, table, window, sinks)
        assert lib.consume_status() == BAD_CACHE
        near(got[:lo], want[:lo], bound[:lo])
        near(got[hi:last], want[hi:last], bound[hi:last])
        near(got[lo:hi], by_zeros[lo:hi], zero_bound[lo:hi])
    for context in (-1, b.page_table.shape[1] * 16, 2 ** 31 - 1):
        lengths = b.context.clone()
        lengths[1] = context
        got = call(b.q, b.k_cache, b.v_cache, b.cu_tokens, lengths, b.page_table, window, sinks)
        assert lib.consume_status() == BAD_CACHE
        near(got[:lo], want[:lo], bound[:lo])
        near(got[hi:last], want[hi:last], bound[hi:last])
        assert bool((got[lo:hi] == 0).all())
    near(call(b.q, *b.arrays, window, sinks)[:last], want[:last], bound[:last])
    assert lib.consume_status() == 0
