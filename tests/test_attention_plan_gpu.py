"""How the attention deals a call's work out over its CTAs: every tile of keys of every item once, evenly, whatever the sizes.
The division is run by itself (attention_plan.cu), since no GPU holds the caches of the largest calls."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

CTAS = 148
CTA = np.dtype([("tiles", "<i8"), ("segments", "<i8")]
               + [(n, "<i4") for n in ("b0", "row0", "head0", "begin0", "b1", "row1", "head1", "end1", "tiles1", "rows1")])


@pytest.fixture(scope="module")
def plan():
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "flash-llm_b200", "csrc"), "plan"], check=True)
    library = ctypes.CDLL(os.path.join(ROOT, "build", "libattention_plan.so"))
    library.attention_plan.argtypes = [ctypes.c_int] + [ctypes.c_void_p] * 3 + [ctypes.c_int] * 6 + [ctypes.c_void_p] * 2

    def call(contexts, counts, heads, kv_heads, prefix=None):
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        cu, context = ints(np.cumsum([0] + counts).tolist()), ints(contexts)
        ahead = ints(prefix) if prefix else None
        status, out = ints([0]), torch.zeros(CTAS * CTA.itemsize, dtype=torch.uint8, device="cuda")
        code = library.attention_plan(CTAS, cu.data_ptr(), context.data_ptr(), ahead.data_ptr() if prefix else None, (1 << 24) - 16, 7,
                                      len(counts), sum(counts), heads, kv_heads, status.data_ptr(), out.data_ptr())
        assert code == 0 and status.item() == 0
        return out.cpu().numpy().view(CTA)
    return call


def items(contexts, counts, heads, kv_heads, prefix):
    """(sequence, first row, tiles of keys, units) of every item of the first key/value head."""
    share = heads // kv_heads
    tile_rows = 128 // share * share
    found = []
    for b, (context, count) in enumerate(zip(contexts, counts)):
        row = np.arange(0, count * share, 2 * tile_rows, dtype=np.int64)
        end = np.minimum(row + 2 * tile_rows, count * share)
        keys = context + (end - 1) // share + 1
        if prefix:
            keys = np.maximum(keys, min(prefix[b], context + count))
        tiles = -(-keys // 128)
        found.append(np.stack([np.full_like(row, b), row, tiles, tiles + np.where(end - row > tile_rows, 2, 4)]))
    return np.concatenate(found, 1)


@pytest.mark.parametrize("contexts,counts,heads,kv_heads,prefix", [
    ([0], [1], 1, 1, None),
    ([5000, 0, 77], [3, 0, 900], 32, 8, None),
    ([(37 * i) % 300 for i in range(600)], [(i % 7) // 3 for i in range(600)], 7, 1, None),
    ([0, 10], [4000, 5], 12, 3, [3000, 0]),
    ([0], [1 << 21], 64, 8, None),                                  # 2^32 units and 1.3 million
    ([4 << 20], [1 << 20], 64, 8, None),                            # 2.25 times 2^32
    ([0] * 5 + [100], [1 << 20] * 5 + [1], 64, 64, None),           # five prompts of a quarter of 2^32
    ([0, 17], [1 << 20, 33], 128, 16, [1 << 20, 0]),                # all keys seen from both sides
    ([5, 0, 9], [2, (1 << 24) - 100, 40], 128, 1, None),            # one sequence's first head alone has 2^40
    ([(1 << 31) - 3000], [3], 128, 1, None),                        # the longest cache
], ids=str)
def test_every_tile_is_somebodys(plan, contexts, counts, heads, kv_heads, prefix):
    got = plan(contexts, counts, heads, kv_heads, prefix)
    _, _, tiles, units = items(contexts, counts, heads, kv_heads, prefix)
    assert int(got["tiles"].sum()) == int(tiles.sum()) * kv_heads
    total = int(units.sum()) * kv_heads
    share = max(-(-total // CTAS), 2)
    assert int(got["tiles"].max()) <= share + 2  # single tiles are not cut off
    busy = got[got["segments"] > 0]
    first, last = busy[0], busy[-1]
    some = [b for b, t in enumerate(counts) if t > 0]
    assert (first["b0"], first["row0"], first["head0"], first["begin0"]) == (some[0], 0, 0, 0)
    assert (last["b1"], last["head1"]) == (some[-1], kv_heads - 1) and last["end1"] == last["tiles1"]
    assert last["row1"] + last["rows1"] == counts[some[-1]] * (heads // kv_heads)
    for one, two in zip(busy[:-1], busy[1:]):  # where one ends the next begins
        if one["end1"] < one["tiles1"]:
            assert (two["b0"], two["row0"], two["head0"], two["begin0"]) == (one["b1"], one["row1"], one["head1"], one["end1"])
        else:
            assert two["begin0"] == 0 and (two["b0"], two["row0"], two["head0"]) > (one["b1"], one["row1"], one["head1"])
