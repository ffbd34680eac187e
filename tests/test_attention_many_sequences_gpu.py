"""Attention of many rows over 4 bits in calls of many sequences, some of several items, some that do not fit, on the GPU against the
definition in 64 bits."""
import pytest
import torch

import four_bit_cache as four
from four_bit_cache import FourBitBatch
from test_more_cache_operators_gpu import BAD_CACHE, healthy, near, ops  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
@pytest.mark.parametrize("sequences,heads,kv_heads,dim", [(12, 2, 1, 64), (13, 2, 1, 64), (40, 4, 2, 128), (400, 1, 1, 64), (60, 36, 1, 64)])
@pytest.mark.parametrize("misfits", [False, True])
def test_sequences_of_several_items_among_others(ops, lib, sequences, heads, kv_heads, dim, window, sinks, misfits):  # noqa: F811
    """Every fifth sequence has rows for several items, every seventh does not fit its table."""
    few = heads // kv_heads > 32  # every row is the tensor core's
    counts = [(15 if few else 270) if i % 5 == 2 else 1 + i % (3 if few else 40) for i in range(sequences)]
    b = FourBitBatch([(7 * i) % 60 for i in range(sequences)], counts, heads, kv_heads, dim, 16, extra_rows=2)
    want, bound = four.attention(b, window, sinks)
    context = b.context.clone()
    if misfits:
        context[3::7] = 1 << 30
    for _ in range(3):
        got = ops.four_bit_attention(b.q, b.k_cache, b.v_cache, b.cu_tokens, context, b.page_table, window, sinks)
        assert lib.consume_status() == (BAD_CACHE if misfits else 0)
        owner = torch.repeat_interleave(torch.arange(sequences, device="cuda"), torch.tensor(counts, device="cuda"))
        lost = (owner % 7 == 3) & misfits
        got, w, off = (x[:b.cut[-1]] for x in (got, want, bound))
        assert bool((got[lost] == 0).all())
        near(got[~lost], w[~lost], off[~lost])
