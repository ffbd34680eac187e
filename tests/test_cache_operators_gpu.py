"""The paged-cache operators on the GPU against their definitions in 64 bits."""
import math

import pytest
import torch

from paged_cache import Batch, attention, random_tree, rotate

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


# --------------------------------------------------------------------------------------------------- rotary positions

APPENDS = [
    # contexts, counts, heads, kv_heads, dim, page, rotary, interleaved
    ([0], [1], 1, 1, 64, 16, 64, False),
    ([5, 0, 31], [1, 3, 2], 4, 2, 64, 16, 16, True),
    ([100, 7, 0, 64], [17, 0, 33, 1], 6, 3, 128, 32, 128, False),
    ([100, 7, 0, 64], [17, 0, 33, 1], 6, 3, 128, 32, 128, True),
    ([127, 128], [130, 1], 9, 9, 128, 128, 64, False),
    ([3], [70], 5, 1, 64, 64, 48, False),
    ([3], [70], 5, 1, 64, 64, 48, True),
    ([200, 1], [4, 5], 8, 8, 128, 256, 0, False),
    ([40], [300], 40, 8, 128, 16, 112, True),
    ([12] * 70, [1] * 70, 2, 1, 64, 16, 32, False),
]


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,rotary,interleaved", APPENDS)
def test_rotary_append(ops, lib, contexts, counts, heads, kv_heads, dim, page, rotary, interleaved):
    b = Batch(contexts, counts, heads, kv_heads, dim, page, extra_rows=3)
    columns = (heads + 2 * kv_heads) * dim
    wide = torch.randn((b.rows, columns + 24), device="cuda").to(torch.float16)
    qkv = wide[:, 8:8 + columns]  # rows apart, as a slice of a wider matrix
    frequencies, magnitude = lib.rotary_frequencies(max(rotary, 16), scaling="by parts", factor=4.0, original_length=64)
    f = torch.from_numpy(frequencies).cuda()[:rotary // 2] if rotary else None
    before = b.k_cache.clone(), b.v_cache.clone()
    q = ops.rotary_append(qkv, *b.arrays, f, interleaved, magnitude)
    x = qkv.double().reshape(b.rows, heads + 2 * kv_heads, dim)
    place = torch.cat([torch.arange(c, c + t) for c, t in zip(contexts, counts)]).cuda()
    owned = b.cut[-1]
    x = x[:owned]
    if rotary:
        y, bound = rotate(x[:, :heads + kv_heads], place.double()[:, None] * f, magnitude, interleaved, rotary)
    else:
        y, bound = x[:, :heads + kv_heads], torch.full_like(x[:, :heads + kv_heads], 1e-30)
    near(q[:owned].view(owned, heads, dim), y[:, :heads], bound[:, :heads], "queries")
    for s, (c, t) in enumerate(zip(contexts, counts)):
        lo, hi = b.cut[s], b.cut[s + 1]
        page_at = b.pages_of(s, torch.arange(c, c + t, device="cuda"))
        near(b.k_cache[page_at[0], :, page_at[1]], y[lo:hi, heads:], bound[lo:hi, heads:], "keys")
        assert torch.equal(b.v_cache[page_at[0], :, page_at[1]].double(), x[lo:hi, heads + kv_heads:])
        for cache, old in zip((b.k_cache, b.v_cache), before):
            cache[page_at[0], :, page_at[1]] = old[page_at[0], :, page_at[1]]
    for cache, old in zip((b.k_cache, b.v_cache), before):  # nothing else was touched
        assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


def test_rotary_angles_of_far_positions(ops, lib):
    b = Batch([0], [6], 2, 1, 128, 16)
    far = torch.tensor([0, 131071, 1000003, 99999989, 2147483647, -7], dtype=torch.int32, device="cuda")
    f = torch.from_numpy(lib.rotary_frequencies(128)[0]).cuda()
    qkv = torch.randn((6, 4 * 128), device="cuda").to(torch.float16)
    q = ops.rotary_append(qkv, *b.arrays, f, False, 1.0, far)
    # position * frequency in 64 bits is off by 2^-53 of up to 2^31 radians here and in the kernel: 5e-7 radians
    y, bound = rotate(qkv.double().view(6, 4, 128)[:, :3], far.double()[:, None] * f, 1.0, False, 128)
    near(q.view(6, 2, 128), y[:, :2], (bound + 2.0 ** -20 * qkv.double().abs().max())[:, :2])


def test_rotary_in_place_through_the_c_abi(ops, lib):
    b = Batch([9, 2], [4, 1], 4, 2, 64, 16)
    f = torch.from_numpy(lib.rotary_frequencies(64)[0]).cuda()
    qkv = torch.randn((5, 8 * 64), device="cuda").to(torch.float16)
    want = ops.rotary_append(qkv, *b.arrays, f)
    caches = b.k_cache.clone(), b.v_cache.clone()
    rest = qkv[:, 4 * 64:].clone()
    args = lib.PagedBatch(b.k_cache.data_ptr(), b.v_cache.data_ptr(), b.k_cache.shape[0], 16, 2, 64, b.cu_tokens.data_ptr(),
                          b.context.data_ptr(), b.page_table.data_ptr(), b.page_table.shape[1], 2, 5)
    lib.rotary_append(torch.cuda.current_stream().cuda_stream, qkv.data_ptr(), 512, qkv.data_ptr(), 512, args, 4, f.data_ptr(), 64)
    assert torch.equal(qkv[:, :256], want) and torch.equal(qkv[:, 256:], rest)
    for cache, old in zip((b.k_cache, b.v_cache), caches):
        assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


# --------------------------------------------------------------------------------------------------- attention

TREES = [
    # contexts, counts, heads, kv_heads, dim, page, cap, slopes
    ([0], [1], 1, 1, 64, 16, 0.0, False),
    ([1], [1], 1, 1, 128, 16, 0.0, False),
    ([127], [2], 2, 1, 64, 128, 0.0, False),
    ([128], [64], 1, 1, 128, 64, 0.0, False),
    ([200, 0, 13], [15, 15, 15], 4, 4, 64, 16, 0.0, False),
    ([300, 64, 0, 1000], [64, 1, 0, 33], 8, 2, 128, 32, 0.0, False),
    ([65, 700], [63, 64], 15, 3, 128, 256, 20.0, False),
    ([65, 700], [63, 64], 15, 3, 64, 16, 0.0, True),
    ([900, 31, 2], [40, 64, 7], 40, 5, 128, 64, 30.0, True),
    ([3000, 10], [5, 64], 32, 1, 128, 128, 0.0, False),
    ([20], [80], 2, 2, 64, 32, 0.0, False),  # the mask has no bit for tokens behind the 64th
]


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,cap,distance", TREES)
def test_tree_attention(ops, contexts, counts, heads, kv_heads, dim, page, cap, distance):
    b = Batch(contexts, counts, heads, kv_heads, dim, page, seed=1, gain=1.5)
    masks, positions = random_tree(counts, contexts, 2)
    slopes = slopes_of(heads) if distance else None
    got = ops.tree_attention(b.q, *b.arrays, masks, cap=cap, slopes=slopes, positions=positions if distance else None)
    want, bound = attention(b, masks, positions, cap=cap, slopes=slopes)
    near(got, want, bound)


PROMPTS = [
    # contexts, counts, heads, kv_heads, dim, page, cap, slopes, prefix
    ([0], [1], 1, 1, 64, 16, 0.0, False, None),
    ([0], [2], 1, 1, 128, 16, 0.0, False, None),
    ([0], [129], 1, 1, 64, 128, 0.0, False, None),
    ([0, 0, 0], [257, 100, 1], 4, 2, 128, 64, 0.0, False, None),
    ([128, 127, 129], [1, 1, 1], 8, 8, 64, 16, 0.0, False, None),
    ([1000, 0, 50, 3], [1, 300, 64, 0], 6, 2, 128, 32, 0.0, True, None),
    ([0, 77], [500, 200], 3, 1, 64, 256, 25.0, False, None),
    ([40, 0, 600], [300, 129, 20], 16, 4, 128, 16, 15.0, True, [100, 60, 620]),
    ([0, 10], [400, 5], 5, 5, 128, 128, 0.0, False, [400, 0]),
    ([0], [700], 8, 1, 64, 64, 0.0, False, [333]),
    ([5000], [3], 32, 8, 128, 512, 0.0, False, None),
    ([100 + 7 * i for i in range(70)], [1] * 70, 8, 2, 128, 64, 0.0, True, None),
    ([(37 * i) % 300 for i in range(600)], [(i % 7) // 3 for i in range(600)], 7, 1, 64, 16, 0.0, False, None),  # some sequences empty
    ([2, 700, 0], [3, 130, 61], 14, 2, 128, 64, 12.0, True, None),  # single tiles and pairs of them in one call
    ([31, 5], [1, 9], 128, 1, 64, 16, 0.0, False, None),  # a token fills a tile of rows
    ([0, 3], [50, 90], 21, 3, 128, 32, 0.0, False, [-5, 1 << 30]),  # prefixes out of range: none, and all
]


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,page,cap,distance,prefix", PROMPTS)
def test_prompt_attention(ops, contexts, counts, heads, kv_heads, dim, page, cap, distance, prefix):
    b = Batch(contexts, counts, heads, kv_heads, dim, page, seed=3, gain=1.5)
    slopes = slopes_of(heads) if distance else None
    ahead = torch.tensor(prefix, dtype=torch.int32, device="cuda") if prefix else None
    got = ops.prompt_attention(b.q, *b.arrays, prefix=ahead, cap=cap, slopes=slopes)
    want, bound = attention(b, prefix=prefix, cap=cap, slopes=slopes)
    near(got, want, bound)


@pytest.mark.parametrize("contexts,counts,kv_heads,dim", [([0], [5], 1, 64), ([0, 0], [64, 3], 2, 128), ([0, 200], [40, 40], 1, 128)])
def test_rows_that_see_nothing_are_zero(ops, contexts, counts, kv_heads, dim):
    b = Batch(contexts, counts, 4 * kv_heads, kv_heads, dim, 32, seed=4)
    masks, _ = random_tree(counts, contexts, 5)
    masks[::2] = 0
    got = ops.tree_attention(b.q, *b.arrays, masks)
    want, bound = attention(b, masks)
    near(got, want, bound)
    if contexts[0] == 0:
        assert bool((got[:counts[0]:2] == 0).all())


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim", [([90], [40], 2, 2, 64), ([0, 300], [64, 64], 8, 2, 128), ([120], [17], 16, 1, 128)])
def test_masked_keys_and_values_that_are_not_finite(ops, contexts, counts, heads, kv_heads, dim, what):
    """Some drafted tokens hold NaN or infinities that only they themselves see; everybody else's output does not change."""
    b = Batch(contexts, counts, heads, kv_heads, dim, 16, seed=6)
    masks, _ = random_tree(counts, contexts, 7)
    spoilt = [(s, i) for s, t in enumerate(counts) for i in (3, t // 2, t - 1)]
    for s, i in spoilt:
        lo, hi = b.cut[s], b.cut[s + 1]
        bit = 1 << i if i < 63 else -(1 << 63)
        masks[lo:hi] &= ~bit
        masks[lo + i] |= bit
        page, at = b.pages_of(s, torch.tensor([contexts[s] + i], device="cuda"))
        b.k_cache[page, :, at, ::3] = what
        b.v_cache[page, :, at, 5::7] = what
    own = torch.tensor([b.cut[s] + i for s, i in spoilt], device="cuda")
    others = torch.ones(b.rows, dtype=torch.bool, device="cuda")
    others[own] = False
    got = ops.tree_attention(b.q, *b.arrays, masks)
    want, bound = attention(b, masks)
    near(got[others], want[others], bound[others])
    assert bool(torch.isnan(got[own]).any(1).all())  # a score that is not a number, or an infinite one, leaves no number


@pytest.mark.parametrize("tree", [False, True])
def test_values_that_are_not_finite_reach_those_who_see_them(ops, tree):
    """Values alone: the tokens that see them get them, in the elements that hold them; the others never do."""
    b = Batch([130], [60], 4, 2, 128, 64, seed=8)
    page, at = b.pages_of(0, torch.tensor([160, 170], device="cuda"))
    b.v_cache[page[0], 0, at[0], 5] = float("inf")
    b.v_cache[page[1], 0, at[1], 9] = float("nan")
    masks = torch.tensor([(1 << i + 1) - 1 for i in range(60)], dtype=torch.int64, device="cuda")
    got = ops.tree_attention(b.q, *b.arrays, masks) if tree else ops.prompt_attention(b.q, *b.arrays)
    got = got.view(60, 4, 128)
    line = torch.arange(60, device="cuda")[:, None]
    assert torch.equal(got[:, :2, 5] == float("inf"), (line >= 30).expand(60, 2))
    assert torch.equal(torch.isnan(got[:, :2, 9]), (line >= 40).expand(60, 2))
    spoilt = torch.zeros((60, 4, 128), dtype=torch.bool, device="cuda")
    spoilt[30:, :2, 5] = True
    spoilt[40:, :2, 9] = True
    b.v_cache[page[0], 0, at[0], 5] = 0.0
    b.v_cache[page[1], 0, at[1], 9] = 0.0
    want, bound = attention(b)
    near(got[~spoilt], want.view(60, 4, 128)[~spoilt], bound.view(60, 4, 128)[~spoilt])


IN_CONTEXTS = [
    # contexts, counts, heads, kv_heads, dim, tree
    ([300], [1], 1, 1, 64, False),             # one row, laid four times in its tile
    ([300, 129], [1, 1], 8, 2, 128, False),
    ([9000], [1], 8, 2, 128, False),           # cut into parts
    ([9000, 200], [3, 2], 16, 2, 64, True),
    ([260], [20], 4, 2, 128, True),            # a tile of rows
    ([6000, 300], [64, 40], 2, 1, 64, True),
    ([200], [300], 2, 2, 128, False),          # pairs of tiles
    ([3000, 0], [700, 200], 6, 2, 64, False),
]


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,tree", IN_CONTEXTS)
def test_infinite_values_of_a_context_reach_all_rows(ops, contexts, counts, heads, kv_heads, dim, tree):
    """A weight is never zero by its definition: infinity times it is infinity, for keys that weigh next to nothing too."""
    b = Batch(contexts, counts, heads, kv_heads, dim, 32, seed=9, gain=1.5)
    page, at = b.pages_of(0, torch.tensor([5, 37, 70, 101, 102], device="cuda"))
    b.k_cache[page[1], :, at[1]] *= 30.0  # takes some rows' whole weight, and next to none of others'
    inf, column = float("inf"), torch.arange(dim, device="cuda")
    spoilt = [(0, 7, inf), (1, 11, -inf), (1, 40, inf), (2, 50, float("nan")), (3, 13, inf), (4, 13, -inf), (4, 14, inf)]
    want_there = torch.zeros(dim, device="cuda")
    for key, c, value in spoilt:
        b.v_cache[page[key], 0, at[key], c] = value
        want_there[c] += value
    masks, _ = random_tree(counts, contexts, 10) if tree else (None, None)
    got = ops.tree_attention(b.q, *b.arrays, masks) if tree else ops.prompt_attention(b.q, *b.arrays)
    for key, c, value in spoilt:
        b.v_cache[page[key], 0, at[key], c] = 0.0
    want, bound = attention(b, masks)
    share = heads // kv_heads
    mine = got[:counts[0]].view(counts[0], heads, dim)[:, :share]  # of the first sequence, and the heads that read the spoilt one
    there = want_there != 0
    assert torch.equal(mine[..., there].float().nan_to_num(nan=7.0), want_there[there].nan_to_num(nan=7.0).expand(counts[0], share, -1))
    clean = torch.ones((b.rows, heads, dim), dtype=torch.bool, device="cuda")
    clean[:counts[0], :share, there] = False
    near(got.view(b.rows, heads, dim)[clean], want.view(b.rows, heads, dim)[clean], bound.view(b.rows, heads, dim)[clean])


@pytest.mark.parametrize("heads,kv_heads,dim,count", [(66, 2, 128, 260), (128, 1, 128, 250), (64, 1, 64, 400), (8, 8, 128, 900)])
def test_infinite_values_in_whole_items(ops, heads, kv_heads, dim, count):
    """Items that no other CTA shares, whose warps write their outputs by the plain way and find out about infinities at different
    times: ten calls, every element."""
    b = Batch([140], [count], heads, kv_heads, dim, 64, seed=9, gain=1.5)
    page, at = b.pages_of(0, torch.tensor([5, 100], device="cuda"))
    for key, c, value in ((0, 1, float("inf")), (0, 90 % dim, -float("inf")), (1, 50, float("nan"))):
        b.v_cache[page[key], :, at[key], c] = value
    got = [ops.prompt_attention(b.q, *b.arrays).view(count, heads, dim) for _ in range(10)]
    b.v_cache[page, :, at, 1] = b.v_cache[page, :, at, 90 % dim] = b.v_cache[page, :, at, 50] = 0.0
    want, bound = attention(b)
    there = torch.ones(dim, dtype=torch.bool, device="cuda")
    there[[1, 90 % dim, 50]] = False
    for x in got:
        assert bool((x[..., 1] == float("inf")).all()) and bool((x[..., 90 % dim] == -float("inf")).all()) and bool(x[..., 50].isnan().all())
        near(x[..., there], want.view(count, heads, dim)[..., there], bound.view(count, heads, dim)[..., there])


@pytest.mark.parametrize("contexts,counts,heads,dim", [([11], [1], 1, 64), ([11], [1], 4, 128), ([11], [40], 2, 64), ([3000], [2], 1, 128),
                                                       ([11], [300], 1, 128)])
@pytest.mark.parametrize("value", [65504.0, -65504.0])
def test_averages_of_the_largest_value_are_that_value(ops, contexts, counts, heads, dim, value):
    """Weights of 0.50026 all round up, by 4.6e-4 of themselves: their products' sum, divided by that of the unrounded ones, passes
    65520, from where on fp16 rounds to infinity."""
    b = Batch(contexts, counts, heads, 1, dim, 16, seed=9)
    b.q.zero_(), b.k_cache.nan_to_num_(nan=0.0).zero_()
    b.q.view(b.rows, heads, dim)[:, :, 0] = 1.0
    b.k_cache[..., 0] = -1.0
    page, at = b.pages_of(0, torch.tensor([0], device="cuda"))
    b.k_cache[page, :, at, 0] = 0.0
    b.v_cache.nan_to_num_(nan=0.0).fill_(value)
    got = ops.prompt_attention(b.q, *b.arrays, scale=-math.log(0.5 + 1.05 * 2.0 ** -12))
    assert bool((got == value).all())


@pytest.mark.parametrize("count,heads,dim,cap", [(1, 1, 64, 0.0), (40, 2, 128, 0.0), (300, 1, 64, 0.0), (150, 1, 128, 300.0)])
def test_long_flat_tails_are_not_lost(ops, count, heads, dim, cap):
    """One key that weighs 2^25.5 times each of 40000 others, whose values alone are not zero; 300 sequences over the same pages, so
    that most rows are one CTA's.  A weight is off by 2^-11 of itself, or by 2^-32 of the largest (half of fp16's least step, 2^-24,
    where the largest is 2^7), the output by 2^-11 besides."""
    one, many = Batch([40000], [count], heads, 1, dim, 64, seed=9), 300
    one.q.zero_(), one.k_cache.nan_to_num_(nan=0.0).zero_()
    one.q.view(count, heads, dim)[:, :, 0] = 1.0
    one.k_cache[..., 0] = -17.671875
    one.v_cache.nan_to_num_(nan=0.0).fill_(1.0)
    page, at = one.pages_of(0, torch.tensor([0], device="cuda"))
    one.k_cache[page, :, at, 0], one.v_cache[page, :, at] = 0.0, 0.0
    got = ops.prompt_attention(one.q.repeat(many, 1), one.k_cache, one.v_cache,
                               torch.arange(0, (many + 1) * count, count, dtype=torch.int32, device="cuda"),
                               one.context.repeat(many), one.page_table.repeat(many, 1), scale=1.0, cap=cap)
    want, _ = attention(one, scale=1.0, cap=cap)
    bound = 2.0 ** -10 * want + 2.0 ** -32 * (40000 + count) + 2.0 ** -25
    near(got, want.repeat(many, 1), bound.repeat(many, 1))


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,dim,tree,scale,cap", [
    ([300], [1], 1, 1, 64, False, 1.0, 0.0), ([9000, 70], [1, 1], 8, 2, 128, False, 0.1, 0.0), ([700], [40], 2, 1, 64, True, 1.0, 0.0),
    ([2000], [64], 8, 2, 128, True, 1e16, 0.0), ([0], [700], 2, 1, 64, False, 1.0, 0.0), ([1000], [900], 1, 1, 128, False, 1e-2, 0.0),
    ([300], [1], 1, 1, 64, False, 1.0, 1e8), ([700], [40], 2, 1, 64, True, 1e16, 1e12), ([0], [700], 2, 1, 64, False, 1e26, 1e30)])
def test_scores_beyond_what_their_exponents_hold(ops, contexts, counts, heads, kv_heads, dim, tree, scale, cap):
    """Scores of 1e7 to 1e30, which 32 bits hold to 1 to 1e23: rounded on its own, the largest one's multiple of log2 e must not decide
    about its weight.  Each row points at one key, next to which all others, 1e7 below at least, weigh nothing."""
    b = Batch(contexts, counts, heads, kv_heads, dim, 32, seed=9)
    g = torch.Generator().manual_seed(10)
    rows, some = counts[0], 16
    place = torch.linspace(0, max(contexts[0] - 1, some - 1), some).long()  # of the keys that are pointed at
    page, at = b.pages_of(0, torch.arange(contexts[0] + rows, device="cuda"))
    b.k_cache[page, :, at] = 0.0
    for i, j in enumerate(place.tolist()):
        b.k_cache[page[j], :, at[j], i] = 30000.0 + 1900.0 * i
    aim = torch.randint(0, some, (rows, heads), generator=g)
    if contexts[0] == 0:
        aim = torch.minimum(aim, torch.arange(rows)[:, None])  # none behind the row
    q = torch.zeros((rows, heads, dim)).scatter_(2, aim[..., None], torch.randint(40000, 60000, (rows, heads, 1), generator=g).float())
    b.q[:rows] = q.view(rows, -1).to(torch.float16).cuda()
    masks, _ = random_tree(counts, contexts, 11) if tree else (None, None)
    got = (ops.tree_attention(b.q, *b.arrays, masks, scale=scale, cap=cap) if tree
           else ops.prompt_attention(b.q, *b.arrays, scale=scale, cap=cap))
    values = b.rows_of(b.v_cache, 0)[place.cuda()]  # [some][kv_heads][dim]
    want = values[aim.cuda(), torch.arange(heads, device="cuda") // (heads // kv_heads)]
    assert torch.equal(got[:rows].view(rows, heads, dim).double(), want)


def test_large_scores(ops):
    """Scores far apart, rising along the cache, so that the running maximum moves at every tile; and scores of -60000 s."""
    b = Batch([700], [3], 4, 1, 64, 32, seed=9)
    place = torch.arange(703, device="cuda")
    page, at = b.pages_of(0, place)
    b.k_cache[page, 0, at] = 0.0
    b.k_cache[page, 0, at, 0] = place.to(torch.float16)
    b.q.view(3, 4, 64)[:, :, 0] = torch.tensor([[0.5, 4.0, -4.0, -90.0]], device="cuda").to(torch.float16)
    got = ops.prompt_attention(b.q, *b.arrays, scale=1.0)
    want, bound = attention(b, scale=1.0)
    near(got, want, bound)


def test_strided_queries_and_rows_of_nobody(ops, lib):
    b = Batch([50, 20], [5, 9], 6, 2, 64, 16, seed=10, extra_rows=4)
    wide = torch.randn((b.rows, 3 * 6 * 64), device="cuda").to(torch.float16)
    wide[:, 64:64 + 6 * 64] = b.q
    want = ops.prompt_attention(b.q, *b.arrays)[:14]
    assert torch.equal(ops.prompt_attention(wide[:, 64:64 + 6 * 64], *b.arrays)[:14], want)
    out = torch.full((b.rows, 384), 7.0, dtype=torch.float16, device="cuda")
    workspace = torch.empty(lib.attention_workspace_bytes(64), dtype=torch.uint8, device="cuda")
    args = lib.PagedBatch(b.k_cache.data_ptr(), b.v_cache.data_ptr(), b.k_cache.shape[0], 16, 2, 64, b.cu_tokens.data_ptr(),
                          b.context.data_ptr(), b.page_table.data_ptr(), b.page_table.shape[1], 2, b.rows)
    lib.prompt_attention(torch.cuda.current_stream().cuda_stream, b.q.data_ptr(), 384, args, 6, out.data_ptr(), workspace.data_ptr())
    assert torch.equal(out[:14], want) and bool((out[14:] == 7.0).all())


def test_repeated_calls_give_the_same_bits(ops):
    b = Batch([3000, 40, 900], [16, 16, 7], 16, 4, 128, 64, seed=11)
    masks, _ = random_tree(b.counts, b.contexts, 12)
    first = ops.tree_attention(b.q, *b.arrays, masks)
    for _ in range(5):
        assert torch.equal(ops.tree_attention(b.q, *b.arrays, masks), first)


def test_bad_pages_and_lengths_are_reported(ops, lib):
    b = Batch([70, 40], [3, 2], 2, 1, 64, 16, seed=13)
    good = ops.prompt_attention(b.q, *b.arrays)
    for page in (-1, b.k_cache.shape[0], 1 << 30):
        table = b.page_table.clone()
        table[0, 2] = page
        got = ops.prompt_attention(b.q, b.k_cache, b.v_cache, b.cu_tokens, b.context, table)
        assert lib.consume_status() == BAD_CACHE
        assert torch.equal(got[3:], good[3:]) and bool(torch.isfinite(got).all())  # the other sequence is as it was
    for context in (-1, 16 * b.page_table.shape[1] - 2, 1 << 30):
        lengths = b.context.clone()
        lengths[0] = context
        got = ops.prompt_attention(b.q, b.k_cache, b.v_cache, b.cu_tokens, lengths, b.page_table)
        assert lib.consume_status() == BAD_CACHE
        assert torch.equal(got[3:], good[3:]) and bool((got[:3] == 0).all())
    caches = b.k_cache.clone(), b.v_cache.clone()
    qkv = torch.randn((5, 4 * 64), device="cuda").to(torch.float16)
    table = b.page_table.clone()
    table[:] = 1 << 20
    ops.rotary_append(qkv, b.k_cache, b.v_cache, b.cu_tokens, b.context, table)
    assert lib.consume_status() == BAD_CACHE
    ops.rotary_append(qkv, b.k_cache, b.v_cache, b.cu_tokens, b.context + 1000, b.page_table)
    assert lib.consume_status() == BAD_CACHE
    accepted, lengths = torch.tensor([[3], [2]], dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    ops.cache_accept(*b.arrays, accepted, lengths)  # tokens the sequences do not have
    assert lib.consume_status() == BAD_CACHE
    ops.cache_accept(*b.arrays, accepted - 2, lengths + 1)  # longer than the row
    assert lib.consume_status() == BAD_CACHE
    for cache, old in zip((b.k_cache, b.v_cache), caches):
        assert torch.equal(cache.view(torch.int16), old.view(torch.int16))


def test_a_sequence_that_does_not_fit_is_not_appended(ops, lib):
    """Not even those of its rows that would have room; its neighbours are."""
    b = Batch([30, 40, 20], [2, 3, 1], 2, 1, 64, 16, seed=14)
    positions = 16 * b.page_table.shape[1]
    qkv = torch.randn((6, 4 * 64), device="cuda").to(torch.float16)
    k_cache, v_cache = b.k_cache.clone(), b.v_cache.clone()
    ops.rotary_append(qkv, k_cache, v_cache, b.cu_tokens, b.context, b.page_table)
    assert lib.consume_status() == 0
    for context in (-1, positions - 2, positions):
        lengths = b.context.clone()
        lengths[1] = context
        k, v = b.k_cache.clone(), b.v_cache.clone()
        ops.rotary_append(qkv, k, v, b.cu_tokens, lengths, b.page_table)
        assert lib.consume_status() == BAD_CACHE
        for got, old, new in ((k, b.k_cache, k_cache), (v, b.v_cache, v_cache)):
            mine = b.page_table[1].long()
            assert torch.equal(got[mine].view(torch.int16), old[mine].view(torch.int16))
            for other in (0, 2):
                pages = b.page_table[other].long()
                assert torch.equal(got[pages].view(torch.int16), new[pages].view(torch.int16))
    lengths = b.context.clone()
    lengths[1] = positions - 3  # the last that fits
    ops.rotary_append(qkv, b.k_cache, b.v_cache, b.cu_tokens, lengths, b.page_table)
    assert lib.consume_status() == 0


@pytest.mark.parametrize("turned,placed", [(False, False), (True, False), (True, True)])
def test_queries_of_a_sequence_that_does_not_fit_are_zero(ops, lib, turned, placed):
    b = Batch([30, 40, 20], [2, 3, 1], 2, 1, 64, 16, seed=14, extra_rows=1)
    qkv = torch.randn((7, 4 * 64), device="cuda").to(torch.float16)
    f = torch.from_numpy(lib.rotary_frequencies(64)[0]).cuda() if turned else None
    positions = torch.arange(7, dtype=torch.int32, device="cuda") if placed else None
    want = ops.rotary_append(qkv, *b.arrays, f, False, 1.0, positions)
    for context in (-1, 16 * b.page_table.shape[1] - 2, 1 << 30):
        lengths = b.context.clone()
        lengths[1] = context
        got = ops.rotary_append(qkv, b.k_cache, b.v_cache, b.cu_tokens, lengths, b.page_table, f, False, 1.0, positions)
        assert lib.consume_status() == BAD_CACHE
        assert bool((got[2:5] == 0).all()) and torch.equal(got[:2], want[:2]) and torch.equal(got[5], want[5])


@pytest.mark.parametrize("page", [16, 128])
def test_caches_longer_than_32_bits(ops, page):
    """Pages behind the 2^31st element of a cache, for every operator."""
    dim, kv_heads = 128, 8
    pages = (1 << 31) // (dim * kv_heads * page) + 40
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of free memory")
    small = Batch([150], [20], 16, kv_heads, dim, page, seed=14)
    k, v = (torch.empty((pages, kv_heads, page, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    shift = pages - small.k_cache.shape[0]
    k[shift:], v[shift:] = small.k_cache, small.v_cache
    table = small.page_table + shift
    want = ops.prompt_attention(small.q, *small.arrays)
    assert torch.equal(ops.prompt_attention(small.q, k, v, small.cu_tokens, small.context, table), want)
    qkv = torch.randn((20, 32 * dim), device="cuda").to(torch.float16)
    ops.rotary_append(qkv, *small.arrays)
    ops.rotary_append(qkv, k, v, small.cu_tokens, small.context, table)
    path = torch.tensor([[4, 9, 17]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    ops.cache_accept(*small.arrays, *path)
    ops.cache_accept(k, v, small.cu_tokens, small.context, table, *path)
    assert torch.equal(k[shift:].view(torch.int16), small.k_cache.view(torch.int16))
    assert torch.equal(v[shift:].view(torch.int16), small.v_cache.view(torch.int16))


# --------------------------------------------------------------------------------------------------- acceptance

@pytest.mark.parametrize("layers,dim,page", [(None, 64, 16), (3, 128, 32), (1, 128, 128)])
def test_accept(ops, layers, dim, page):
    contexts, counts = [30, 0, 17, 5], [64, 10, 0, 3]
    b = Batch(contexts, counts, 2, 2, dim, page, seed=15)
    # any order, repeated tokens, sources that are targets, nothing, everything
    paths = [list(range(63, -1, -1)), [3, 0, 3, 9, 1], [], [2]]
    wide = 64
    accepted = torch.tensor([p + [-7] * (wide - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
    caches = [c.clone() if layers is None else torch.stack([c + i for i in range(layers)]) for c in (b.k_cache, b.v_cache)]
    want = []
    for cache in caches:
        w = cache.clone()
        for s, path in enumerate(paths):
            for i, token in enumerate(path):
                to, to_at = b.pages_of(s, torch.tensor([contexts[s] + i], device="cuda"))
                source, source_at = b.pages_of(s, torch.tensor([contexts[s] + token], device="cuda"))
                w[..., to[0], :, to_at[0], :] = cache[..., source[0], :, source_at[0], :]
        want.append(w)
    ops.cache_accept(*caches, b.cu_tokens, b.context, b.page_table, accepted, lengths)
    for cache, w in zip(caches, want):
        assert torch.equal(cache.view(torch.int16), w.view(torch.int16))


# --------------------------------------------------------------------------------------------------- together

def test_refusals_of_the_operators(ops, lib):
    b = Batch([20], [3], 4, 2, 64, 16, seed=16)
    k, v, cu, context, table = b.arrays
    masks = torch.ones(3, dtype=torch.int64, device="cuda")
    for bad in ((b.q.float(), k, v, cu, context, table), (b.q, k.float(), v, cu, context, table), (b.q, k, v[:1], cu, context, table),
                (b.q, k.transpose(1, 2), v.transpose(1, 2), cu, context, table), (b.q, k[..., :32].contiguous(), v[..., :32].contiguous(), cu, context, table),
                (b.q, k, v, cu.long(), context, table), (b.q, k, v, cu, context.cpu(), table), (b.q, k, v, cu[:1], context, table),
                (b.q, k, v, cu, context, table[0]), (b.q[:, :192], k, v, cu, context, table), (b.q[:, 1:], k, v, cu, context, table),
                (b.q.t(), k, v, cu, context, table), (b.q[:, :0], k, v, cu, context, table)):
        with pytest.raises(RuntimeError):
            ops.prompt_attention(*bad)
        with pytest.raises(RuntimeError):
            ops.tree_attention(*bad, masks)
    for options in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(cap=-1.0), dict(cap=math.inf), dict(slopes=slopes_of(3)),
                    dict(slopes=slopes_of(4).half())):
        with pytest.raises(RuntimeError):
            ops.prompt_attention(b.q, *b.arrays, **options)
    with pytest.raises(RuntimeError, match="positions"):
        ops.tree_attention(b.q, *b.arrays, masks, slopes=slopes_of(4))
    with pytest.raises(RuntimeError):
        ops.tree_attention(b.q, *b.arrays, masks[:2])
    with pytest.raises(RuntimeError):
        ops.prompt_attention(b.q, *b.arrays, prefix=torch.zeros(2, dtype=torch.int32, device="cuda"))
    qkv = torch.zeros((3, 8 * 64), dtype=torch.float16, device="cuda")
    for f in (torch.ones(32, device="cuda"), torch.ones(40, dtype=torch.float64, device="cuda"), torch.ones(4, dtype=torch.float64, device="cuda"),
              torch.ones(32, dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            ops.rotary_append(qkv, *b.arrays, f)
    for rows in (qkv[:, :4 * 64], qkv[:, :65], qkv.float()):
        with pytest.raises(RuntimeError):
            ops.rotary_append(rows, *b.arrays)
    with pytest.raises(lib.FlashLLMError, match="RotaryAppend"):
        ops.rotary_append(qkv, *b.arrays, torch.ones(32, dtype=torch.float64, device="cuda"), False, math.inf)
    with pytest.raises(RuntimeError):
        ops.cache_accept(*b.arrays, torch.zeros((1, 65), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.cache_accept(*b.arrays, torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    empty = b.q[:0]
    assert ops.prompt_attention(empty, *b.arrays).shape == (0, 256)


def test_a_cap_that_32_bits_take_for_none_is_refused(ops):
    b = Batch([20], [3], 4, 2, 64, 16, seed=16)
    for call in (lambda: ops.prompt_attention(b.q, *b.arrays, cap=1e-50),
                 lambda: ops.tree_attention(b.q, *b.arrays, torch.ones(3, dtype=torch.int64, device="cuda"), cap=1e-50)):
        with pytest.raises(RuntimeError, match="cap"):
            call()


def test_captured_calls_follow_the_arrays(ops):
    """One graph of append and attention, replayed with other lengths, pages and masks; and two graphs at once."""
    contexts, counts = [60, 200, 1500], [16, 16, 16]
    batches = [Batch(c, counts, 8, 4, 128, 32, seed=20 + i) for i, c in enumerate((contexts, [1, 900, 33], [700, 0, 1600]))]
    width = max(x.page_table.shape[1] for x in batches)
    pages = max(x.k_cache.shape[0] for x in batches)
    still = Batch([1600] * 3, counts, 8, 4, 128, 32, seed=30)
    k, v = (torch.zeros((pages, 4, 32, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    q, context = still.q.clone(), still.context.clone()
    table = torch.zeros((3, width), dtype=torch.int32, device="cuda")
    masks = torch.zeros(48, dtype=torch.int64, device="cuda")
    arrays = (k, v, still.cu_tokens, context, table)
    ops.tree_attention(q, *arrays, masks)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.tree_attention(q, *arrays, masks))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i, x in enumerate(batches):
        k.zero_(), v.zero_(), table.zero_()
        k[:x.k_cache.shape[0]] = x.k_cache
        v[:x.v_cache.shape[0]] = x.v_cache
        table[:, :x.page_table.shape[1]] = x.page_table
        context.copy_(x.context), q.copy_(x.q)
        m, _ = random_tree(counts, x.contexts, 40 + i)
        masks.copy_(m)
        want = ops.tree_attention(q, *arrays, masks)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        exact, bound = attention(x, m)
        near(want, exact, bound)


def test_another_stream(ops):
    b = Batch([2000, 100], [16, 3], 8, 2, 128, 64, seed=50)
    want = ops.prompt_attention(b.q, *b.arrays)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        for _ in range(4):
            outs.append(ops.prompt_attention(b.q, *b.arrays))
    here = [ops.prompt_attention(b.q, *b.arrays) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in outs + here)


def test_drafting_and_accepting_ends_where_plain_decoding_does(ops, lib):
    """A prompt, then twice a drafted tree of which a path is accepted, against the prompt attention of the final text: the same
    positions and keys, so the same outputs but for the order of the sums."""
    heads, kv_heads, dim, page, prompt = 8, 2, 128, 16, 37
    f = torch.from_numpy(lib.rotary_frequencies(dim)[0]).cuda()
    text = torch.randn((prompt + 6, (heads + 2 * kv_heads) * dim), device="cuda").to(torch.float16)  # QKV rows of the final text
    b = Batch([0], [96], heads, kv_heads, dim, page, seed=60)
    k, v, table = b.k_cache, b.v_cache, b.page_table
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    k.fill_(float("nan")), v.fill_(float("nan"))
    batch = (k, v, ints(0, prompt), ints(0), table)
    rows = [ops.prompt_attention(ops.rotary_append(text[:prompt], *batch, f), *batch)]
    length = prompt
    for path in ([0, 2, 5], [1, 3, 6]):
        draft = torch.randn((8, text.shape[1]), device="cuda").to(torch.float16)
        draft[path] = text[length:length + 3]
        masks = [1 << i for i in range(8)]
        positions = [length] * 8
        for depth, token in enumerate(path):
            masks[token] = sum(1 << t for t in path[:depth + 1])
            positions[token] = length + depth
        batch = (k, v, ints(0, 8), ints(length), table)
        q = ops.rotary_append(draft, *batch, f, False, 1.0, ints(*positions))
        out = ops.tree_attention(q, *batch, torch.tensor(masks, device="cuda"))
        rows.append(out[path])
        ops.cache_accept(*batch, ints(*path).view(1, 3), ints(3))
        length += 3
    got = torch.cat(rows)
    k.fill_(float("nan")), v.fill_(float("nan"))
    batch = (k, v, ints(0, length), ints(0), table)
    q = ops.rotary_append(text, *batch, f)
    want = ops.prompt_attention(q, *batch)
    whole = Batch([0], [length], heads, kv_heads, dim, page)
    whole.q, whole.k_cache, whole.v_cache, whole.page_table = q, k, v, table
    exact, bound = attention(whole)
    near(want, exact, bound)
    near(got, exact, bound)


def test_layer_chain_attends_to_its_cache(ops, lib):
    """DeviceChain with a cache: a prompt of 16 tokens and a tree of 8, against the layer on the host."""
    from flash_llm_b200.tp_chain import CachedAttention, ChainShape, DeviceChain, reference_chain, shard_weights
    hidden, ffn, dim = 512, 1024, 64
    heads = hidden // dim
    g = torch.Generator().manual_seed(70)
    weights = [(torch.randn(s, generator=g) * 0.05 * (torch.rand(s, generator=g) < 0.3)).half()
               for s in ((3 * hidden, hidden), (hidden, hidden), (ffn, hidden), (hidden, ffn))]
    f, _ = lib.rotary_frequencies(32)
    k, v = (torch.full((6, heads, 16, dim), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[4, 1, 3]], dtype=torch.int32, device="cuda")
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    past = {}

    def host(tokens, masks):
        """The same attention in 32 bits over what earlier calls appended."""
        def call(y):
            q, kk, vv = (t.view(tokens, heads, dim).float() for t in y.chunk(3, 1))
            start = past["k"].shape[0] if past else 0
            place = torch.arange(tokens) if masks is None else torch.tensor([bin(m).count("1") - 1 for m in masks])
            angle = (start + place).double()[:, None] * torch.from_numpy(f)
            q, kk = (rotate(t.double(), angle, 1.0, False, 32)[0].half().float() for t in (q, kk))
            vv = vv.half().float()
            if past:
                kk, vv = torch.cat([past["k"], kk]), torch.cat([past["v"], vv])
            past.update(k=kk, v=vv)
            own = torch.ones((tokens, tokens)).tril().bool() if masks is None else torch.tensor([[m >> j & 1 for j in range(tokens)] for m in masks]).bool()
            seen = torch.cat([torch.ones((tokens, start), dtype=torch.bool), own], 1)
            score = torch.einsum("thd,lhd->htl", q, kk) / math.sqrt(dim)
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            return torch.einsum("htl,lhd->thd", p, vv).reshape(tokens, hidden)
        return call

    tree = [1, 3, 5, 11, 19, 32 | 1, 64 | 3, 128 | 5]
    for tokens, masks, context in ((16, None, 0), (8, tree, 16)):
        shape = ChainShape(hidden=hidden, ffn=ffn, tokens=tokens, world=1)
        chain = DeviceChain(lib, shape, shard_weights(shape, 0, *weights), torch.device("cuda:0"), split_k=8)
        x = torch.randn((tokens, hidden), generator=g).half()
        depth = None if masks is None else ints(*(context + bin(m).count("1") - 1 for m in masks))
        attend = CachedAttention(k, v, ints(0, tokens), ints(context), table, positions=depth, frequencies=torch.from_numpy(f).cuda(),
                                 tree_mask=None if masks is None else torch.tensor(masks, device="cuda"))
        got = chain.step(x.cuda(), all_reduce=lambda t: t, attention=attend).cpu().double()
        want = reference_chain(shape, x, *weights, attention=host(tokens, masks)).double()
        # five roundings to fp16 in a row, each of 2^-11 of values about as large as the row's largest
        assert float((got - want).abs().max()) <= 5 * 2.0 ** -10 * float(want.abs().max())
