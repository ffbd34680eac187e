"""Calls of the attention through a window and over a cache of 4 bits whose waits run out, for test_more_attention_give_up_gpu.py: run
with a library whose CTAs give up after a few looks at a barrier.  A call returns, reports it, and leaves every row of a head either
right or as it was."""
import torch

import flash_llm_b200 as fl
import four_bit_cache as four
from four_bit_cache import FourBitBatch
from paged_cache import Batch

CASES = [
    # contexts, counts, heads, kv_heads, dim, window, sinks, cap and slopes
    ([0], [5000], 16, 4, 128, 1500, 4, False),
    ([0, 300, 7], [900, 500, 1300], 8, 8, 64, 700, 200, True),
    ([9000, 40, 20000], [20, 3, 40], 32, 8, 128, 5000, 0, False),
    ([100, 100], [60, 41], 1, 1, 64, 64, 1, True),
]


def main():
    for kind in (Batch, FourBitBatch):
        untouched = right = reported = 0
        for contexts, counts, heads, kv_heads, dim, window, sinks, both in CASES:
            b = kind(contexts, counts, heads, kv_heads, dim, 64, seed=5)
            slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float32, device="cuda") / heads) if both else None
            cap = 20.0 if both else 0.0
            want, bound = four.attention(b, window, sinks, cap=cap, slopes=slopes)
            workspace = torch.empty(fl.attention_workspace_bytes(dim), dtype=torch.uint8, device="cuda")
            batch = fl.PagedBatch(b.k_cache.data_ptr(), b.v_cache.data_ptr(), b.k_cache.shape[0], 64, kv_heads, dim,
                                  b.cu_tokens.data_ptr(), b.context.data_ptr(), b.page_table.data_ptr(), b.page_table.shape[1],
                                  len(counts), b.rows)
            call = fl.four_bit_attention if kind is FourBitBatch else fl.window_attention
            before = reported
            for _ in range(20):
                out = torch.full((b.rows, heads * dim), 7.0, dtype=torch.float16, device="cuda")
                call(torch.cuda.current_stream().cuda_stream, b.q.data_ptr(), heads * dim, batch, heads, out.data_ptr(),
                     workspace.data_ptr(), window, sinks, cap=cap, slopes=slopes.data_ptr() if both else None)
                status = fl.consume_status()
                left = (out.view(b.rows, heads, dim) == 7.0).all(2)
                off = ((out.double() - want).abs() <= bound).view(b.rows, heads, dim).all(2)
                assert bool((left | off).all()), f"{int((~(left | off)).sum())} rows of heads are neither right nor as they were"
                assert status in (0, 1) and (status == 1 or not bool(left.any()))
                untouched, right, reported = untouched + int(left.sum()), right + int(off.sum()), reported + status
            assert reported > before, "no call gave up"
        assert untouched > 0 and right > 0, (untouched, right)
        print(f"{kind.__name__}: {reported} calls gave up, {untouched} rows of heads as they were, {right} right")


if __name__ == "__main__":
    main()
