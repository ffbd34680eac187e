"""``torch.ops.flashllm``: the library's SpMM as PyTorch operators, for integration tests and for callers whose tensors
live in torch.  Importing this module registers

* ``flashllm::encode(Tensor A) -> (Tensor compressed, Tensor tile_offsets)``: a dense fp16 weight ``A[M][K]`` on a CUDA
  device to its tiled-CSL form (int32 words, int32 tile offsets) with the device encoder; what the reference does on
  the host with ``InitSparseMatrixA_API`` (reference csrc/SpMM_API.cu:449-494).
* ``flashllm::spmm(Tensor compressed, Tensor tile_offsets, Tensor B, int M, int split_k=1) -> Tensor``:
  ``C[N][M] = B[N][K] @ A[M][K]^T`` (reference ``SpMM_SplitK_API``, csrc/SpMM_API.cu:124-171).
* ``flashllm::spmm_epilogue(..., Tensor? bias, int activation, Tensor? residual) -> Tensor``: the same with
  ``act(. + bias[M]) + residual[N][M]`` applied to the fp32 sums before the one rounding.

* ``flashllm::rotary_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor cu_tokens, Tensor context, Tensor
  page_table, Tensor? frequencies=None, bool interleaved=False, float magnitude=1.0, Tensor? positions=None) -> Tensor``: the
  output of a QKV projection to turned queries ``[N][heads * head_dim]``, turned keys and values in a paged cache.
* ``flashllm::tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor cu_tokens, Tensor context, Tensor page_table,
  Tensor tree_mask, float? scale=None, float cap=0, Tensor? slopes=None, Tensor? positions=None) -> Tensor``: attention of up
  to 64 drafted tokens of each sequence (scale ``None``: 1 / sqrt(head_dim)).
* ``flashllm::prompt_attention(..., Tensor page_table, Tensor? prefix=None, float? scale=None, float cap=0, Tensor?
  slopes=None) -> Tensor``: causal attention of prompts, pieces of prompts and single tokens.
* ``flashllm::norm_rotary_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor cu_tokens, Tensor context, Tensor
  page_table, Tensor q_norm, Tensor k_norm, float eps=1e-6, Tensor? frequencies=None, bool interleaved=False, float magnitude=1.0,
  Tensor? positions=None) -> Tensor``: the rotary append of query and key heads that are normed first.
* ``flashllm::window_attention(..., Tensor page_table, int window, int sinks=0, float? scale=None, float cap=0, Tensor?
  slopes=None) -> Tensor``: prompt attention through a window, the first ``sinks`` positions of a sequence always in sight.
* ``flashllm::four_bit_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor cu_tokens, Tensor context, Tensor
  page_table, Tensor? q_norm=None, Tensor? k_norm=None, float eps=1e-6, Tensor? frequencies=None, bool interleaved=False, float
  magnitude=1.0, Tensor? positions=None) -> Tensor``: the append into a cache of 4 bits.
* ``flashllm::four_bit_attention(..., Tensor page_table, int window=0, int sinks=0, float? scale=None, float cap=0, Tensor?
  slopes=None) -> Tensor``: attention over a cache of 4 bits (window 0: none).
* ``flashllm::four_bit_read(Tensor k_cache, Tensor v_cache, Tensor cu_tokens, Tensor context, Tensor page_table, int tokens) ->
  (Tensor, Tensor)``: the batch's keys and values ``[tokens][kv_heads * head_dim]`` from a cache of 4 bits.
* ``flashllm::cache_accept(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor cu_tokens, Tensor context, Tensor page_table, Tensor
  accepted, Tensor accepted_lengths) -> ()``: moves an accepted path's keys and values behind the context, in one layer's cache
  or, with a leading dimension, in all layers' at once.

A cache is fp16 ``[pages][kv_heads][page_size][head_dim]``, one of 4 bits uint8 ``[pages][kv_heads][page_size][head_dim * 9 / 16]``,
sequence b owns rows ``cu_tokens[b]`` up to ``cu_tokens[b + 1]`` and
``context[b]`` positions of ``page_table[b]`` are filled before the call (int32; include/SpMM_API.cuh has the whole contract).
Rows of a result behind the last sequence are not written.

The operators run on the current CUDA stream of B's device and call the library through its C ABI; there is no CPU
implementation (a CPU tensor is refused), only shape inference for meta tensors.  Their CUDA side is native
(csrc/torch_ops.cpp, ``build/libflashllm_torch.so``): a decode step is launch-bound, and from Python the checks, the
result's allocation and the call took 18-22 us of host time around a 6 us kernel.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import api

OPERATORS_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "build", "libflashllm_torch.so")

_LIB = torch.library.Library("flashllm", "DEF")
_LIB.define("encode(Tensor A) -> (Tensor, Tensor)")
_LIB.define("spmm(Tensor compressed, Tensor tile_offsets, Tensor B, int M, int split_k=1) -> Tensor")
_LIB.define("spmm_epilogue(Tensor compressed, Tensor tile_offsets, Tensor B, int M, int split_k=1, Tensor? bias=None, "
            "int activation=0, Tensor? residual=None) -> Tensor")
_BATCH = "Tensor cu_tokens, Tensor context, Tensor page_table"
_LIB.define(f"rotary_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, {_BATCH}, Tensor? frequencies=None, "
            "bool interleaved=False, float magnitude=1.0, Tensor? positions=None) -> Tensor")
_LIB.define(f"tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, {_BATCH}, Tensor tree_mask, float? scale=None, "
            "float cap=0.0, Tensor? slopes=None, Tensor? positions=None) -> Tensor")
_LIB.define(f"prompt_attention(Tensor q, Tensor k_cache, Tensor v_cache, {_BATCH}, Tensor? prefix=None, float? scale=None, "
            "float cap=0.0, Tensor? slopes=None) -> Tensor")
_LIB.define(f"cache_accept(Tensor(a!) k_cache, Tensor(b!) v_cache, {_BATCH}, Tensor accepted, Tensor accepted_lengths) -> ()")
_NORM, _ROTARY = "float eps=1e-06", "Tensor? frequencies=None, bool interleaved=False, float magnitude=1.0, Tensor? positions=None"
_LIB.define(f"norm_rotary_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, {_BATCH}, Tensor q_norm, Tensor k_norm, "
            f"{_NORM}, {_ROTARY}) -> Tensor")
_LIB.define(f"window_attention(Tensor q, Tensor k_cache, Tensor v_cache, {_BATCH}, int window, int sinks=0, float? scale=None, "
            "float cap=0.0, Tensor? slopes=None) -> Tensor")
_LIB.define(f"four_bit_append(Tensor qkv, Tensor(a!) k_cache, Tensor(b!) v_cache, {_BATCH}, Tensor? q_norm=None, "
            f"Tensor? k_norm=None, {_NORM}, {_ROTARY}) -> Tensor")
_LIB.define(f"four_bit_attention(Tensor q, Tensor k_cache, Tensor v_cache, {_BATCH}, int window=0, int sinks=0, "
            "float? scale=None, float cap=0.0, Tensor? slopes=None) -> Tensor")
_LIB.define(f"four_bit_read(Tensor k_cache, Tensor v_cache, {_BATCH}, int tokens) -> (Tensor, Tensor)")
_OPERATORS = ("encode", "spmm", "spmm_epilogue", "rotary_append", "tree_attention", "prompt_attention", "cache_accept",
              "norm_rotary_append", "window_attention", "four_bit_append", "four_bit_attention", "four_bit_read")


def _load_operators() -> None:
    """Registers the CUDA implementations and binds them to the library build that :mod:`api` has loaded."""
    if not os.path.exists(OPERATORS_PATH):
        raise api.FlashLLMError(f"{OPERATORS_PATH} is missing: build it with `make -C flash-llm_b200/csrc all operators` "
                                "(or __graft_entry__.build()); there is no fallback implementation")
    library = api.library()
    torch.ops.load_library(OPERATORS_PATH)
    bind = ctypes.CDLL(OPERATORS_PATH).flashllm_torch_bind
    bind.restype, bind.argtypes = None, [ctypes.c_void_p] * 13 + [ctypes.py_object]
    bind(*(ctypes.cast(f, ctypes.c_void_p) for f in (library.FlashLLM_SpMM_SplitK_Epilogue,
                                                     library.FlashLLM_EncodeOnDevice_TileOffsets,
                                                     library.FlashLLM_EncodeOnDevice_Pack, library.FlashLLM_RotaryAppend,
                                                     library.FlashLLM_TreeAttention, library.FlashLLM_PromptAttention,
                                                     library.FlashLLM_CacheAccept,
                                                     library.FlashLLM_Attention_WorkspaceBytes,
                                                     library.FlashLLM_NormRotaryAppend, library.FlashLLM_WindowAttention,
                                                     library.FlashLLM_FourBitAppend, library.FlashLLM_FourBitAttention,
                                                     library.FlashLLM_FourBitRead)), api.FlashLLMError)


try:
    _load_operators()
except (api.FlashLLMError, OSError) as _error:
    # Schemas and shape inference work without the library (a build of torch without CUDA, a host that only traces);
    # whoever runs an operator is told.
    _reason = str(_error)

    def _refuse_cuda(*args, **kwargs):
        raise api.FlashLLMError(f"the flashllm operators could not be loaded: {_reason}")

    for _name in _OPERATORS:
        _LIB.impl(_name, _refuse_cuda, "CUDA")


def _refuse_cpu(*args, **kwargs):
    raise RuntimeError("flashllm operators have no CPU implementation: move the tensors to a CUDA device")


for _name in _OPERATORS:
    _LIB.impl(_name, _refuse_cpu, "CPU")


@torch.library.register_fake("flashllm::spmm")
def _spmm_fake(compressed, tile_offsets, B, M, split_k=1):
    return B.new_empty((B.shape[0], M))


@torch.library.register_fake("flashllm::spmm_epilogue")
def _spmm_epilogue_fake(compressed, tile_offsets, B, M, split_k=1, bias=None, activation=0, residual=None):
    return B.new_empty((B.shape[0], M))


@torch.library.register_fake("flashllm::rotary_append")
def _rotary_append_fake(qkv, k_cache, v_cache, cu_tokens, context, page_table, frequencies=None, interleaved=False, magnitude=1.0,
                        positions=None):
    return qkv.new_empty((qkv.shape[0], qkv.shape[1] - 2 * k_cache.shape[1] * k_cache.shape[3]))


@torch.library.register_fake("flashllm::tree_attention")
def _tree_attention_fake(q, k_cache, v_cache, cu_tokens, context, page_table, tree_mask, scale=None, cap=0.0, slopes=None,
                         positions=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("flashllm::prompt_attention")
def _prompt_attention_fake(q, k_cache, v_cache, cu_tokens, context, page_table, prefix=None, scale=None, cap=0.0, slopes=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("flashllm::cache_accept")
def _cache_accept_fake(k_cache, v_cache, cu_tokens, context, page_table, accepted, accepted_lengths):
    return None


@torch.library.register_fake("flashllm::norm_rotary_append")
def _norm_rotary_append_fake(qkv, k_cache, v_cache, cu_tokens, context, page_table, q_norm, k_norm, eps=1e-6, frequencies=None,
                             interleaved=False, magnitude=1.0, positions=None):
    return qkv.new_empty((qkv.shape[0], qkv.shape[1] - 2 * k_cache.shape[1] * k_cache.shape[3]))


@torch.library.register_fake("flashllm::window_attention")
def _window_attention_fake(q, k_cache, v_cache, cu_tokens, context, page_table, window, sinks=0, scale=None, cap=0.0, slopes=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("flashllm::four_bit_append")
def _four_bit_append_fake(qkv, k_cache, v_cache, cu_tokens, context, page_table, q_norm=None, k_norm=None, eps=1e-6,
                          frequencies=None, interleaved=False, magnitude=1.0, positions=None):
    return qkv.new_empty((qkv.shape[0], qkv.shape[1] - 2 * k_cache.shape[1] * (k_cache.shape[3] * 16 // 9)))


@torch.library.register_fake("flashllm::four_bit_attention")
def _four_bit_attention_fake(q, k_cache, v_cache, cu_tokens, context, page_table, window=0, sinks=0, scale=None, cap=0.0, slopes=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("flashllm::four_bit_read")
def _four_bit_read_fake(k_cache, v_cache, cu_tokens, context, page_table, tokens):
    shape = (tokens, k_cache.shape[1] * (k_cache.shape[3] * 16 // 9))
    return k_cache.new_empty(shape, dtype=torch.float16), k_cache.new_empty(shape, dtype=torch.float16)


def spmm(compressed: torch.Tensor, tile_offsets: torch.Tensor, B: torch.Tensor, M: int, split_k: int = 1) -> torch.Tensor:
    """Python spelling of ``torch.ops.flashllm.spmm``."""
    return torch.ops.flashllm.spmm(compressed, tile_offsets, B, M, split_k)
