"""Norms with the rotary append, attention through a window and the cache of 4 bits on the host: refusals of the C ABI, shape
inference, what the layer chain's attention refuses, and the tests' own definition of the codes."""
import math

import pytest
import torch

import flash_llm_b200 as fl
from flash_llm_b200 import torch_op  # noqa: F401
import four_bit_cache as four
from four_bit_cache import FourBitBatch
from paged_cache import Batch
from test_cache_operators import BAD_BATCHES, INVALID, P, _batch


def _refused(lib, call):
    with pytest.raises(lib.FlashLLMError, match=f"cudaError_t {INVALID}$"):
        call()


@pytest.mark.parametrize("change", BAD_BATCHES, ids=[str(sorted(b.items())) for b in BAD_BATCHES])
def test_bad_caches_and_batches_are_refused(lib, change):
    batch = _batch(**change)
    _refused(lib, lambda: lib.norm_rotary_append(0, P, 1 << 20, P, 1 << 20, batch, 4, P, P))
    _refused(lib, lambda: lib.four_bit_append(0, P, 1 << 20, P, 1 << 20, batch, 4))
    _refused(lib, lambda: lib.window_attention(0, P, 1 << 20, batch, 4, P, P, 10, scale=1.0))
    _refused(lib, lambda: lib.four_bit_attention(0, P, 1 << 20, batch, 4, P, P, scale=1.0))
    _refused(lib, lambda: lib.four_bit_read(0, batch, P, P))


def test_bad_arguments_are_refused(lib):
    b = _batch()
    append = dict(QKV=P, ld_qkv=1024, Q=P + (1 << 30), ld_q=512, batch=b, heads=4, q_norm=P, k_norm=P, frequencies=P, rotary_dim=128)
    for change in (dict(QKV=None), dict(QKV=P + 2), dict(ld_qkv=1016), dict(ld_qkv=1025), dict(Q=None), dict(ld_q=504), dict(ld_q=516),
                   dict(heads=0), dict(heads=-4), dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=-16), dict(frequencies=None),
                   dict(magnitude=math.inf), dict(magnitude=math.nan), dict(q_norm=P + 8), dict(k_norm=P + 2), dict(eps=-1e-6),
                   dict(eps=math.nan), dict(eps=math.inf), dict(Q=P, ld_q=520)):
        _refused(lib, lambda: lib.norm_rotary_append(0, **{**append, **change}))
        _refused(lib, lambda: lib.four_bit_append(0, **{**append, **change}))
    for change in (dict(q_norm=None), dict(k_norm=None)):
        _refused(lib, lambda: lib.norm_rotary_append(0, **{**append, **change}))
    attend = dict(Q=P, ld_q=512, batch=b, heads=4, Out=P, workspace=P, window=10)
    for change in (dict(Q=None), dict(Q=P + 8), dict(ld_q=504), dict(ld_q=513), dict(heads=3), dict(heads=0),
                   dict(heads=258, ld_q=258 * 128), dict(Out=None), dict(Out=P + 4), dict(workspace=None), dict(workspace=P + 8),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.nan),
                   dict(cap=math.inf), dict(scale=3e38), dict(cap=3e38), dict(scale=1.0, cap=1e-39), dict(window=-1), dict(sinks=-1)):
        _refused(lib, lambda: lib.window_attention(0, **{**attend, **change}))
        _refused(lib, lambda: lib.four_bit_attention(0, **{**attend, **change}))
    _refused(lib, lambda: lib.window_attention(0, **{**attend, "window": 0}))
    for out in ((None, P), (P, None), (P + 8, P), (P, P + 2)):
        _refused(lib, lambda: lib.four_bit_read(0, b, *out))
    huge = _batch(page_size=1 << 25, table_width=1)
    _refused(lib, lambda: lib.four_bit_read(0, huge, P, P))
    _refused(lib, lambda: lib.four_bit_append(0, **{**append, "batch": huge}))
    _refused(lib, lambda: lib.four_bit_attention(0, **{**attend, "batch": huge}))


def test_empty_batches_are_accepted_without_a_device(lib):
    for b in (_batch(tokens=0), _batch(sequences=0)):
        lib.norm_rotary_append(0, P, 1024, P, 512, b, 4, P, P)
        lib.four_bit_append(0, P, 1024, P, 512, b, 4)
        lib.window_attention(0, P, 512, b, 4, P, P, 7)
        lib.four_bit_attention(0, P, 512, b, 4, P, P)
        lib.four_bit_read(0, b, P, P)


def test_operators_refuse_cpu_tensors_and_infer_shapes():
    ops = torch.ops.flashllm
    for kind, calls in ((Batch, lambda b, w, x: (lambda: ops.norm_rotary_append(x, *b.arrays, w, w), lambda: ops.window_attention(b.q, *b.arrays, 5))),
                        (FourBitBatch, lambda b, w, x: (lambda: ops.four_bit_append(x, *b.arrays), lambda: ops.four_bit_attention(b.q, *b.arrays),
                                                        lambda: ops.four_bit_read(*b.arrays, 5)))):
        b = kind([3, 20], [2, 3], 4, 2, 128, 16, device="cpu")
        x = torch.zeros((5, 8 * 128), dtype=torch.float16)
        for call in calls(b, x[0, :128], x):
            with pytest.raises(RuntimeError, match="no CPU implementation"):
                call()
        arrays = [t.to("meta") for t in b.arrays]
        meta, w = x.to("meta"), x[0, :128].to("meta")
        if kind is Batch:
            assert ops.norm_rotary_append(meta, *arrays, w, w).shape == (5, 512)
            assert ops.window_attention(b.q.to("meta"), *arrays, 9, 1).shape == (5, 512)
        else:
            assert ops.four_bit_append(meta, *arrays).shape == (5, 512)
            assert ops.four_bit_attention(b.q.to("meta"), *arrays).shape == (5, 512)
            keys, values = ops.four_bit_read(*arrays, 5)
            assert keys.shape == values.shape == (5, 256) and keys.dtype == torch.float16


def test_cached_attention_refuses_what_its_operators_do_not_have():
    from flash_llm_b200.tp_chain import CachedAttention
    x, half, four_bit = torch.zeros(1), torch.zeros(1, dtype=torch.float16), torch.zeros(1, dtype=torch.uint8)
    for cache, more, match in ((four_bit, dict(tree_mask=x, positions=x), "4 bits"), (four_bit, dict(prefix=x), "4 bits"),
                               (half, dict(window=5, prefix=x), "window"), (half, dict(window=5, tree_mask=x, positions=x), "window"),
                               (half, dict(q_norm=x), "both norms"), (half, dict(k_norm=x), "both norms")):
        with pytest.raises(ValueError, match=match):
            CachedAttention(cache, cache, x, x, x, **more)(x)


def test_the_codes_of_the_tests_stand_for_their_elements():
    """Elements are half a step away at most; groups that are not finite have none; a group of one value has that value."""
    x = torch.randn((7, 3, 128), generator=torch.Generator().manual_seed(3))
    x[0, 0, :64] = 0.75
    x[1, 1, 100] = math.inf
    cache = torch.zeros((1, 3, 16, 72), dtype=torch.uint8)
    at = (torch.zeros(7, dtype=torch.long), slice(None), torch.arange(7))
    four.put(cache, 128, at, x)
    kept, step, low = four.values(cache, 128, at)
    assert bool(torch.isnan(kept[1, 1, 64:]).all()) and not bool(torch.isnan(kept[1, 1, :64]).any())
    kept, step, x = (torch.where(torch.isnan(kept), torch.zeros_like(kept), t.double()) for t in (kept, step, x))
    # the lowest value and the step are rounded to fp16: 2^-11 of themselves, 15 steps at the top
    assert bool(((kept - x).abs() <= 0.5 * step + 2.0 ** -11 * (low.abs() + 15 * step) + 1e-12).all())
    assert bool((kept[0, 0, :64] == 0.75).all())


def test_the_window_of_the_tests_is_what_a_loop_sees():
    b = Batch([4, 0], [5, 3], 2, 1, 64, 16, device="cpu")
    for window, sinks in ((1, 0), (3, 1), (2, 7), (100, 0)):
        want, _ = four.attention(b, window, sinks)
        for s in range(2):
            k, v = b.rows_of(b.k_cache, s)[:, 0], b.rows_of(b.v_cache, s)[:, 0]
            for r in range(b.counts[s]):
                at = b.contexts[s] + r
                keys = [j for j in range(at + 1) if j < sinks or j > at - window]
                q = b.q[b.cut[s] + r, :64].double()
                p = torch.softmax(k[keys] @ q / 8, 0)
                assert torch.allclose(want[b.cut[s] + r, :64], p @ v[keys], atol=1e-12)
