"""Calls of the attention whose waits run out, for test_attention_give_up_gpu.py: run with a library whose CTAs give up after a few
looks at a barrier.  A call returns, reports it, and leaves every row of a head either right or as it was."""
import torch

import flash_llm_b200 as fl
from paged_cache import Batch, attention, random_tree

CASES = [
    # contexts, counts, heads, kv_heads, dim, tree, cap and slopes
    ([0], [5000], 16, 4, 128, False, False),                    # pairs of tiles, some cut
    ([0, 300, 7], [900, 500, 1300], 8, 8, 64, False, True),
    ([9000, 40, 20000], [1, 1, 1], 32, 8, 128, False, False),   # four times in the tile, many parts
    ([700 + 90 * i for i in range(20)], [16] * 20, 12, 2, 64, True, False),
    ([3000, 5000], [64, 50], 16, 2, 128, True, True),
    ([100, 100], [60, 1], 1, 1, 64, True, True),                # fewer CTAs than there are
]


def main():
    untouched = right = reported = 0
    for contexts, counts, heads, kv_heads, dim, tree, both in CASES:
        b = Batch(contexts, counts, heads, kv_heads, dim, 64, seed=5)
        masks, positions = random_tree(counts, contexts, 6)
        slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads) if both else None
        cap = 20.0 if both else 0.0
        want, bound = attention(b, masks if tree else None, positions if tree else None, cap=cap, slopes=slopes)
        workspace = torch.empty(fl.attention_workspace_bytes(dim), dtype=torch.uint8, device="cuda")
        batch = fl.PagedBatch(b.k_cache.data_ptr(), b.v_cache.data_ptr(), b.k_cache.shape[0], 64, kv_heads, dim, b.cu_tokens.data_ptr(),
                              b.context.data_ptr(), b.page_table.data_ptr(), b.page_table.shape[1], len(counts), b.rows)
        stream = torch.cuda.current_stream().cuda_stream
        before = reported
        options = dict(scale=None, cap=cap, slopes=slopes.data_ptr() if both else None)
        for _ in range(20):
            out = torch.full((b.rows, heads * dim), 7.0, dtype=torch.float16, device="cuda")
            if tree:
                fl.tree_attention(stream, b.q.data_ptr(), heads * dim, batch, heads, masks.data_ptr(), out.data_ptr(),
                                  workspace.data_ptr(), positions=positions.data_ptr(), **options)
            else:
                fl.prompt_attention(stream, b.q.data_ptr(), heads * dim, batch, heads, out.data_ptr(), workspace.data_ptr(), **options)
            status = fl.consume_status()
            left = (out.view(b.rows, heads, dim) == 7.0).all(2)
            off = ((out.double() - want).abs() <= bound).view(b.rows, heads, dim).all(2)
            assert bool((left | off).all()), f"{int((~(left | off)).sum())} rows of heads are neither right nor as they were"
            assert status in (0, 1) and (status == 1 or not bool(left.any()))
            untouched, right, reported = untouched + int(left.sum()), right + int(off.sum()), reported + status
        assert reported > before, "no call gave up"
    assert untouched > 0 and right > 0, (untouched, right)
    print(f"{reported} calls gave up, {untouched} rows of heads as they were, {right} right")


if __name__ == "__main__":
    main()
