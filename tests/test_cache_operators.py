"""The paged-cache operators on the host: refusals of the C ABI and of the PyTorch operators, shape inference, frequencies, and
the layer chain with an attention of its own."""
import math
import threading

import numpy as np
import pytest
import torch

import flash_llm_b200 as fl
from flash_llm_b200 import torch_op  # noqa: F401
from flash_llm_b200.tp_chain import ChainShape, reference_chain, run_chain, shard_weights
from paged_cache import Batch, attention, random_tree, rotate

INVALID = 1  # cudaErrorInvalidValue
P = 1 << 20  # a pointer that nothing dereferences: every refusal comes before the first use


def _batch(**changes):
    sizes = dict(K_cache=P, V_cache=P, pages=8, page_size=64, kv_heads=2, head_dim=128, cu_tokens=P, context=P, page_table=P,
                 table_width=4, sequences=2, tokens=5)
    sizes.update(changes)
    return fl.PagedBatch(**sizes)


BAD_BATCHES = [dict(K_cache=None), dict(V_cache=None), dict(K_cache=P + 8), dict(pages=0), dict(page_size=8), dict(page_size=48),
               dict(page_size=0), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=256), dict(cu_tokens=None), dict(context=None),
               dict(page_table=None), dict(table_width=0), dict(sequences=-1), dict(sequences=4097), dict(tokens=-1),
               dict(table_width=1 << 25), dict(pages=1 << 30, kv_heads=4)]


def _refused(lib, call):
    with pytest.raises(lib.FlashLLMError, match=f"cudaError_t {INVALID}$"):
        call()


@pytest.mark.parametrize("change", BAD_BATCHES, ids=[str(sorted(b.items())) for b in BAD_BATCHES])
def test_bad_caches_and_batches_are_refused(lib, change):
    batch = _batch(**change)
    _refused(lib, lambda: lib.rotary_append(0, P, 1 << 20, P, 1 << 20, batch, 4))
    _refused(lib, lambda: lib.tree_attention(0, P, 1 << 20, batch, 4, P, P, P, scale=1.0))
    _refused(lib, lambda: lib.prompt_attention(0, P, 1 << 20, batch, 4, P, P, scale=1.0))
    _refused(lib, lambda: lib.cache_accept(0, batch, P, P, 4))


def test_bad_arguments_of_each_operator_are_refused(lib):
    b = _batch()
    append = dict(QKV=P, ld_qkv=1024, Q=P, ld_q=512, batch=b, heads=4, frequencies=P, rotary_dim=128)
    for change in (dict(QKV=None), dict(QKV=P + 2), dict(ld_qkv=1016), dict(ld_qkv=1025), dict(Q=None), dict(ld_q=504), dict(ld_q=516),
                   dict(heads=0), dict(heads=-4), dict(rotary_dim=8), dict(rotary_dim=144), dict(rotary_dim=-16), dict(frequencies=None),
                   dict(magnitude=math.inf), dict(magnitude=math.nan)):
        _refused(lib, lambda: lib.rotary_append(0, **{**append, **change}))
    attend = dict(Q=P, ld_q=512, batch=b, heads=4, Out=P, workspace=P)
    for change in (dict(Q=None), dict(Q=P + 8), dict(ld_q=504), dict(ld_q=513), dict(heads=3), dict(heads=0), dict(heads=258, ld_q=258 * 128), dict(Out=None), dict(Out=P + 4),
                   dict(workspace=None), dict(workspace=P + 8), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                   dict(cap=-1.0), dict(cap=math.nan), dict(cap=math.inf)):
        _refused(lib, lambda: lib.prompt_attention(0, **{**attend, **change}))
        _refused(lib, lambda: lib.tree_attention(0, tree_mask=P, **{**attend, **change}))
    for change in (dict(scale=3e38), dict(cap=3e38), dict(scale=1.0, cap=1e-39), dict(scale=1e30, cap=1e-10)):  # what is made of them
        _refused(lib, lambda: lib.prompt_attention(0, **{**attend, **change}))
        _refused(lib, lambda: lib.tree_attention(0, tree_mask=P, **{**attend, **change}))
    _refused(lib, lambda: lib.tree_attention(0, tree_mask=None, **attend))
    _refused(lib, lambda: lib.tree_attention(0, tree_mask=P, slopes=P, **attend))  # distances need positions
    accept = dict(batch=b, accepted=P, accepted_lengths=P, accepted_width=4)
    for change in (dict(batch=_batch(layers=0)), dict(accepted=None), dict(accepted_lengths=None), dict(accepted_width=0),
                   dict(accepted_width=65)):
        _refused(lib, lambda: lib.cache_accept(0, **{**accept, **change}))


def test_appends_in_place_with_other_row_lengths_are_refused(lib):
    for ld_qkv, ld_q in ((1024, 512), (1024, 1032)):
        _refused(lib, lambda: lib.rotary_append(0, P, ld_qkv, P, ld_q, _batch(), 4, P, 128))


def test_scales_whose_largest_scores_are_not_finite_are_refused(lib):
    attend = dict(Q=P, ld_q=512, batch=_batch(), heads=4, Out=P, workspace=P)
    for change in (dict(scale=1e27), dict(scale=1e27, cap=1e20)):
        _refused(lib, lambda: lib.prompt_attention(0, **{**attend, **change}))
        _refused(lib, lambda: lib.tree_attention(0, tree_mask=P, **{**attend, **change}))


def test_empty_batches_are_accepted_without_a_device(lib):
    for change in (dict(tokens=0), dict(sequences=0)):
        b = _batch(**change)
        lib.rotary_append(0, P, 1024, P, 512, b, 4)
        lib.prompt_attention(0, P, 512, b, 4, P, P)
        lib.tree_attention(0, P, 512, b, 4, P, P, P)
        lib.cache_accept(0, b, P, P, 4)


def test_workspace_size_of_unsupported_heads_is_zero(lib):
    assert lib.attention_workspace_bytes(96) == 0


def test_operators_refuse_cpu_tensors_and_infer_shapes():
    ops = torch.ops.flashllm
    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    q = torch.zeros((3, 256), dtype=torch.float16)
    calls = [lambda: ops.rotary_append(q, k, k, *ints), lambda: ops.prompt_attention(q, k, k, *ints),
             lambda: ops.tree_attention(q, k, k, *ints, torch.zeros(3, dtype=torch.int64)),
             lambda: ops.cache_accept(k, k, *ints, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))]
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    meta = lambda t: t.to("meta")  # noqa: E731
    batch = [meta(k), meta(k)] + [meta(t) for t in ints]
    assert ops.rotary_append(meta(torch.zeros((3, (4 + 4) * 64), dtype=torch.float16)), *batch).shape == (3, 256)
    assert ops.prompt_attention(meta(q), *batch).shape == (3, 256)
    assert ops.tree_attention(meta(q), *batch, meta(torch.zeros(3, dtype=torch.int64))).shape == (3, 256)


def test_frequencies():
    f, magnitude = fl.rotary_frequencies(64)
    assert f.dtype == np.float64 and f.shape == (32,) and magnitude == 1.0
    assert f[0] == 1.0 and f[-1] == pytest.approx(10000.0 ** (-62 / 64), rel=1e-15)
    assert np.array_equal(fl.rotary_frequencies(64, scaling="linear", factor=4.0)[0], f / 4)
    slowed = fl.rotary_frequencies(64, scaling="base", factor=4.0)[0]
    assert slowed[0] == 1.0 and slowed[-1] == pytest.approx(f[-1] / 4, rel=1e-12)
    parts, magnitude = fl.rotary_frequencies(64, scaling="by parts", factor=4.0, original_length=2048)
    turns = 2048 * f / (2 * math.pi)
    assert np.array_equal(parts[turns > 32], f[turns > 32]) and np.allclose(parts[turns < 1], f[turns < 1] / 4, rtol=1e-15)
    between = (turns >= 1) & (turns <= 32)
    assert between.any() and ((parts[between] >= f[between] / 4) & (parts[between] <= f[between])).all()
    assert magnitude == pytest.approx(0.1 * math.log(4.0) + 1)
    for bad in (dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=64, base=0.0), dict(rotary_dim=64, factor=0.0),
                dict(rotary_dim=64, scaling="by parts"), dict(rotary_dim=64, scaling="other")):
        with pytest.raises(ValueError):
            fl.rotary_frequencies(**bad)


def test_the_oracle_gives_what_a_softmax_of_few_keys_gives():
    """The 64-bit definition against numbers written out by hand: two keys with scores ln 3 apart, one key, and none."""
    b = Batch([1], [2], 1, 1, 64, 16, device="cpu")
    rows = torch.zeros((3, 64), dtype=torch.float16)
    rows[0, 0], rows[1, 0], rows[2, 0] = 1.0, 2.0, 4.0
    page, at = b.pages_of(0, torch.arange(3))
    b.k_cache[page, 0, at] = rows
    b.v_cache[page, 0, at] = rows * 10
    b.q.zero_()
    b.q[:, 0] = 1.0
    out, _ = attention(b, scale=math.log(3.0))
    assert out[0, 0].item() == pytest.approx((1 * 10 + 3 * 20) / 4)                  # sees keys 0 and 1: weights 1 : 3
    assert out[1, 0].item() == pytest.approx((1 * 10 + 3 * 20 + 27 * 40) / 31)       # weights 1 : 3 : 27
    out, _ = attention(b, tree_mask=torch.tensor([0, 2]), scale=math.log(3.0))
    assert out[0, 0].item() == pytest.approx(10.0)                                   # the context alone
    assert out[1, 0].item() == pytest.approx((1 * 10 + 27 * 40) / 28)
    masks, positions = random_tree([5], [3], 0, device="cpu")
    assert all(m >> i & 1 for i, m in enumerate(masks.tolist())) and positions.min() == 3
    y, _ = rotate(torch.ones((1, 1, 64), dtype=torch.float64), torch.full((1, 8), math.pi / 2, dtype=torch.float64), 2.0, True, 16)
    assert torch.allclose(y[0, 0, :16], torch.tensor([-2.0, 2.0], dtype=torch.float64).repeat(8)) and bool((y[0, 0, 16:] == 1).all())


def test_cached_attention_refuses_trees_without_positions_or_with_a_prefix():
    from flash_llm_b200.tp_chain import CachedAttention
    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    ints = torch.tensor([0, 3], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    rows, masks = torch.zeros((3, 6 * 64), dtype=torch.float16), torch.ones(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="positions"):
        CachedAttention(k, k.clone(), *ints, tree_mask=masks, frequencies=torch.ones(32, dtype=torch.float64))(rows)
    with pytest.raises(ValueError, match="prefix"):
        CachedAttention(k, k.clone(), *ints, tree_mask=masks, prefix=torch.zeros(1, dtype=torch.int32))(rows)
    for more in (dict(frequencies=torch.ones(32, dtype=torch.float64), positions=torch.zeros(3, dtype=torch.int32)), {}):
        with pytest.raises(RuntimeError, match="no CPU implementation"):  # not refused here
            CachedAttention(k, k.clone(), *ints, tree_mask=masks, **more)(rows)


def test_chain_with_an_attention_of_its_own():
    """Two ranks' chains, each with the attention of its heads (a causal one over the batch's rows), add up to the whole layer."""
    shape, dim = ChainShape(hidden=256, ffn=512, tokens=8, world=2), 64
    g = torch.Generator().manual_seed(3)
    weights = [torch.randn(s, generator=g) * 0.05 for s in ((768, 256), (256, 256), (512, 256), (256, 512))]
    x = torch.randn((8, 256), generator=g)

    def attend(y):
        heads = y.shape[1] // 3 // dim
        q, k, v = (t.view(8, heads, dim).transpose(0, 1).float() for t in y.chunk(3, 1))
        score = (q @ k.transpose(1, 2) / 8).masked_fill(~torch.ones(8, 8).tril().bool(), -math.inf)
        return (torch.softmax(score, -1) @ v).transpose(0, 1).reshape(8, heads * dim)

    partial, gate, outs = {}, threading.Barrier(2), [None, None]

    def rank(r):
        shards = shard_weights(shape, r, *weights)

        def all_reduce(t):
            partial[r] = t
            gate.wait()
            total = partial[0] + partial[1]
            gate.wait()
            return total

        outs[r] = run_chain(shape, x, lambda name, t, relu=False: torch.relu(t @ shards[name].T) if relu else t @ shards[name].T,
                            all_reduce, attention=attend)

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    want = reference_chain(shape, x, *weights, attention=attend)
    assert torch.equal(outs[0], outs[1])
    assert float((outs[0] - want).abs().max()) <= 2e-3 * float(want.abs().max())  # the reference rounds to fp16 four times
