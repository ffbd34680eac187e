// CUDA implementations of torch.ops.flashllm.{spmm, spmm_epilogue, encode, rotary_append, tree_attention, prompt_attention,
// cache_accept} (schemas, shape inference and the refusals for other devices are registered by torch_op.py).  Checks, result allocation and the call into libSpMM_API.so run here
// because a decode step is launch-bound: from Python the same work took 18-22 us per call, four times the kernel.
//
// The library's entry points are handed over as addresses (flashllm_torch_bind), so that the operators call whichever
// build of the library the package has loaded.
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <string>
#include <tuple>

#include "../../include/SpMM_API.cuh"

namespace {

using SpmmFn        = int (*)(void*, const void*, const int*, const void*, void*, int, int, int, void*, int, const void*, int,
                       const void*);
using TileOffsetsFn = int (*)(void*, const void*, int, int, int*);
using PackFn        = int (*)(void*, const void*, int, int, const int*, uint32_t*, int);

decltype(&FlashLLM_RotaryAppend)              g_rotary          = nullptr;
decltype(&FlashLLM_TreeAttention)             g_tree            = nullptr;
decltype(&FlashLLM_PromptAttention)           g_prompt          = nullptr;
decltype(&FlashLLM_CacheAccept)               g_accept          = nullptr;
decltype(&FlashLLM_Attention_WorkspaceBytes)  g_workspace_bytes = nullptr;

SpmmFn        g_spmm         = nullptr;
TileOffsetsFn g_tile_offsets = nullptr;
PackFn        g_pack         = nullptr;
PyObject*     g_error_class  = nullptr;  // FlashLLMError

[[noreturn]] void raise_library_error(const std::string& what, int code)
{
    pybind11::gil_scoped_acquire gil;
    PyErr_SetString(g_error_class, (what + " failed with cudaError_t " + std::to_string(code)).c_str());
    throw pybind11::error_already_set();
}

bool is_half_matrix(const at::Tensor& t)
{
    return t.scalar_type() == at::kHalf && t.dim() == 2 && t.is_contiguous();
}

at::Tensor spmm_epilogue(const at::Tensor& compressed, const at::Tensor& tile_offsets, const at::Tensor& B, int64_t M,
                         int64_t split_k, const std::optional<at::Tensor>& bias, int64_t activation,
                         const std::optional<at::Tensor>& residual)
{
    TORCH_CHECK(B.is_cuda(), "flashllm::spmm runs on CUDA tensors only");
    TORCH_CHECK(is_half_matrix(B), "B must be a contiguous fp16 matrix [N][K]");
    TORCH_CHECK(compressed.scalar_type() == at::kInt && tile_offsets.scalar_type() == at::kInt,
                "compressed and tile_offsets must be int32 tensors (tiled-CSL words, offsets in vectors)");
    TORCH_CHECK(compressed.device() == B.device() && tile_offsets.device() == B.device(),
                "all operands must live on one device");
    const int64_t N = B.size(0), K = B.size(1);
    TORCH_CHECK(M % 128 == 0 && K % 64 == 0, "M (", M, ") must be a multiple of 128 and K (", K, ") of 64");
    TORCH_CHECK(tile_offsets.numel() == (M / 128) * (K / 64) + 2, "tile_offsets does not belong to an M x K matrix of this shape");
    const bool has_bias = bias.has_value() && bias->defined(), has_residual = residual.has_value() && residual->defined();
    if (has_bias)
        TORCH_CHECK(bias->scalar_type() == at::kHalf && bias->dim() == 1 && bias->size(0) == M && bias->is_contiguous()
                        && bias->device() == B.device(),
                    "bias must be a contiguous fp16 tensor of shape (", M, ",) on B's device");
    if (has_residual)
        TORCH_CHECK(is_half_matrix(*residual) && residual->size(0) == N && residual->size(1) == M
                        && residual->device() == B.device(),
                    "residual must be a contiguous fp16 tensor of shape (", N, ", ", M, ") on B's device");
    const c10::cuda::CUDAGuard guard(B.device());
    const at::Tensor           C = at::empty({N, M}, B.options());
    at::Tensor                 workspace;
    if (split_k > 1)  // the room the reference's callers bring: Split_K fp16 matrices (reference csrc/SpMM_API.cu:150-152)
        workspace = at::empty({split_k, N, M}, B.options());
    const int code = g_spmm(c10::cuda::getCurrentCUDAStream().stream(), compressed.const_data_ptr(),
                            static_cast<const int*>(tile_offsets.const_data_ptr()), B.const_data_ptr(), C.mutable_data_ptr(),
                            static_cast<int>(M), static_cast<int>(N), static_cast<int>(K),
                            split_k > 1 ? workspace.mutable_data_ptr() : nullptr, static_cast<int>(split_k),
                            has_bias ? bias->const_data_ptr() : nullptr, static_cast<int>(activation),
                            has_residual ? residual->const_data_ptr() : nullptr);
    if (code != 0)
        raise_library_error("SpMM_SplitK_Epilogue(M=" + std::to_string(M) + ", N=" + std::to_string(N) + ", K=" + std::to_string(K)
                                + ", Split_K=" + std::to_string(split_k) + ")",
                            code);
    return C;
}

at::Tensor spmm(const at::Tensor& compressed, const at::Tensor& tile_offsets, const at::Tensor& B, int64_t M, int64_t split_k)
{
    return spmm_epilogue(compressed, tile_offsets, B, M, split_k, std::nullopt, 0, std::nullopt);
}

std::tuple<at::Tensor, at::Tensor> encode(const at::Tensor& A)
{
    TORCH_CHECK(is_half_matrix(A), "A must be a contiguous fp16 matrix [M][K]");
    const int64_t M = A.size(0), K = A.size(1);
    TORCH_CHECK(M % 128 == 0 && K % 64 == 0, "M (", M, ") must be a multiple of 128 and K (", K, ") of 64");
    const c10::cuda::CUDAGuard guard(A.device());
    const cudaStream_t         stream  = c10::cuda::getCurrentCUDAStream().stream();
    const auto                 options = A.options().dtype(at::kInt);
    const int64_t              tiles   = (M / 128) * (K / 64);
    const at::Tensor           offs    = at::empty({tiles + 2}, options);
    int* const                 offs_d  = static_cast<int*>(offs.mutable_data_ptr());
    int                        code    = g_tile_offsets(stream, A.const_data_ptr(), static_cast<int>(M), static_cast<int>(K), offs_d);
    if (code != 0)
        raise_library_error("EncodeOnDevice_TileOffsets", code);
    // The size of the result depends on the data: the one wait of an encoding.  Through page-locked memory (PyTorch's pool of
    // it), a copy to any other is staged.
    const at::Tensor size = at::empty({1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    code = cudaMemcpyAsync(size.mutable_data_ptr(), offs_d + tiles + 1, sizeof(int), cudaMemcpyDeviceToHost, stream);
    if (code == 0)
        code = cudaStreamSynchronize(stream);
    if (code != 0)
        raise_library_error("reading the size of the encoding", code);
    const int64_t    words = static_cast<int64_t>(*static_cast<const int*>(size.const_data_ptr())) * 4;
    const at::Tensor comp  = at::empty({words > 4 ? words : 4}, options);
    code = g_pack(stream, A.const_data_ptr(), static_cast<int>(M), static_cast<int>(K), offs_d,
                  static_cast<uint32_t*>(comp.mutable_data_ptr()), 1);
    if (code != 0)
        raise_library_error("EncodeOnDevice_Pack", code);
    return {words < 4 ? comp.narrow(0, 0, words) : comp, offs};
}

// ---------------------------------------------------------------- paged cache

// The sizes of a cache and a batch, checked; what the C ABI takes after the caches.
struct Paged {
    int        layers, pages, kv_heads, page_size, head_dim;  // layers: 1 for a cache without that dimension
    int        sequences, table_width;
    const int *cu_tokens, *context, *page_table;
};

const int* int_array(const at::Tensor& t, int64_t dims, const at::Device& device, const char* name)
{
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous() && t.device() == device, name,
                " must be a contiguous int32 tensor of ", dims, " dimension(s) on the cache's device");
    return static_cast<const int*>(t.const_data_ptr());
}

int as_int(int64_t value)
{
    TORCH_CHECK(value >= 0 && value <= std::numeric_limits<int>::max(), "size ", value, " does not fit into 32 bits");
    return static_cast<int>(value);
}

Paged paged(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& cu_tokens, const at::Tensor& context,
            const at::Tensor& page_table, bool may_have_layers = false)
{
    TORCH_CHECK(k_cache.is_cuda(), "the flashllm cache operators run on CUDA tensors only");
    const bool layers = may_have_layers && k_cache.dim() == 5;
    TORCH_CHECK(k_cache.scalar_type() == at::kHalf && k_cache.is_contiguous() && (k_cache.dim() == 4 || layers),
                "k_cache must be a contiguous fp16 tensor [pages][kv_heads][page_size][head_dim]",
                may_have_layers ? ", with or without a leading [layers]" : "");
    TORCH_CHECK(v_cache.scalar_type() == at::kHalf && v_cache.is_contiguous() && v_cache.sizes() == k_cache.sizes()
                    && v_cache.device() == k_cache.device(),
                "v_cache must be laid out like k_cache");
    Paged     p{};
    const int d = layers ? 1 : 0;
    p.layers    = layers ? as_int(k_cache.size(0)) : 1;
    p.pages     = as_int(k_cache.size(d));
    p.kv_heads  = as_int(k_cache.size(d + 1));
    p.page_size = as_int(k_cache.size(d + 2));
    p.head_dim  = as_int(k_cache.size(d + 3));
    TORCH_CHECK(p.head_dim == 64 || p.head_dim == 128, "head_dim (", p.head_dim, ") must be 64 or 128");
    TORCH_CHECK(p.page_size >= 16 && (p.page_size & (p.page_size - 1)) == 0, "page_size (", p.page_size,
                ") must be a power of two of at least 16");
    TORCH_CHECK(p.layers >= 1 && p.pages >= 1 && p.kv_heads >= 1, "the cache must not be empty");
    const at::Device device = k_cache.device();
    p.cu_tokens             = int_array(cu_tokens, 1, device, "cu_tokens");
    p.context               = int_array(context, 1, device, "context");
    p.page_table            = int_array(page_table, 2, device, "page_table");
    p.sequences             = as_int(context.size(0));
    p.table_width           = as_int(page_table.size(1));
    TORCH_CHECK(cu_tokens.size(0) == context.size(0) + 1 && page_table.size(0) == context.size(0),
                "cu_tokens, context and page_table must describe the same number of sequences (", context.size(0) + 1, ", ",
                context.size(0), " and ", context.size(0), " entries)");
    TORCH_CHECK(p.table_width >= 1 || p.sequences == 0, "page_table must have a column");
    return p;
}

// Checks an fp16 matrix whose rows may lie apart and returns the halves from one row to the next.
int row_length(const at::Tensor& t, const at::Device& device, const char* name)
{
    TORCH_CHECK(t.scalar_type() == at::kHalf && t.dim() == 2 && t.device() == device && (t.size(1) <= 1 || t.stride(1) == 1), name,
                " must be an fp16 matrix on the cache's device, its rows without gaps");
    if (t.size(0) <= 1)
        return as_int((t.size(1) + 7) / 8 * 8);
    TORCH_CHECK(t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1), "the rows of ", name, " must lie a multiple of 8 halves apart");
    return as_int(t.stride(0));
}

[[noreturn]] void raise_paged(const char* what, const Paged& p, int64_t tokens, int64_t heads, int code)
{
    raise_library_error(std::string(what) + "(tokens=" + std::to_string(tokens) + ", sequences=" + std::to_string(p.sequences)
                            + ", heads=" + std::to_string(heads) + ", kv_heads=" + std::to_string(p.kv_heads)
                            + ", head_dim=" + std::to_string(p.head_dim) + ", page_size=" + std::to_string(p.page_size) + ")",
                        code);
}

at::Tensor rotary_append(const at::Tensor& qkv, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& cu_tokens,
                         const at::Tensor& context, const at::Tensor& page_table, const std::optional<at::Tensor>& frequencies,
                         bool interleaved, double magnitude, const std::optional<at::Tensor>& positions)
{
    const Paged      p      = paged(k_cache, v_cache, cu_tokens, context, page_table);
    const at::Device device = k_cache.device();
    const int        ld     = row_length(qkv, device, "qkv");
    const int64_t    tokens = qkv.size(0), heads = qkv.size(1) / p.head_dim - 2 * static_cast<int64_t>(p.kv_heads);
    TORCH_CHECK(qkv.size(1) % p.head_dim == 0 && heads >= 1, "qkv must hold query heads and ", p.kv_heads,
                " key and value heads of ", p.head_dim, " each, but has ", qkv.size(1), " columns");
    const bool turned = frequencies.has_value() && frequencies->defined() && frequencies->numel() > 0;
    if (turned)
        TORCH_CHECK(frequencies->scalar_type() == at::kDouble && frequencies->dim() == 1 && frequencies->is_contiguous()
                        && frequencies->device() == device && frequencies->size(0) % 8 == 0 && 2 * frequencies->size(0) <= p.head_dim,
                    "frequencies must be a contiguous float64 tensor of 8, 16, ... head_dim / 2 angles on the cache's device");
    const bool has_positions = positions.has_value() && positions->defined();
    if (has_positions)
        TORCH_CHECK(positions->dim() == 1 && positions->size(0) == tokens, "positions must have one entry per row");
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor           q    = at::empty({tokens, heads * p.head_dim}, qkv.options());
    if (tokens == 0 || p.sequences == 0)
        return q;
    const int code = g_rotary(c10::cuda::getCurrentCUDAStream().stream(), qkv.const_data_ptr(), ld, q.mutable_data_ptr(),
                              as_int(q.size(1)), k_cache.mutable_data_ptr(), v_cache.mutable_data_ptr(), p.pages, p.page_size,
                              p.cu_tokens, p.context, p.page_table, p.table_width, p.sequences, as_int(tokens), as_int(heads),
                              p.kv_heads, p.head_dim, turned ? static_cast<const double*>(frequencies->const_data_ptr()) : nullptr,
                              turned ? as_int(2 * frequencies->size(0)) : 0, interleaved, static_cast<float>(magnitude),
                              has_positions ? int_array(*positions, 1, device, "positions") : nullptr);
    if (code != 0)
        raise_paged("RotaryAppend", p, tokens, heads, code);
    return q;
}

// What the two attention operators share; `call` is handed (workspace, out, ld_q, tokens, heads, scale, slopes).
template<typename Call>
at::Tensor attention(const char* what, const at::Tensor& q, const Paged& p, const at::Device& device, std::optional<double> scale,
                     double cap, const std::optional<at::Tensor>& slopes, Call&& call)
{
    const int     ld     = row_length(q, device, "q");
    const int64_t tokens = q.size(0), heads = q.size(1) / p.head_dim;
    TORCH_CHECK(q.size(1) % p.head_dim == 0 && heads >= 1 && heads % p.kv_heads == 0, "q must hold a multiple of ", p.kv_heads,
                " heads of ", p.head_dim, ", but has ", q.size(1), " columns");
    const double factor = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(p.head_dim));
    TORCH_CHECK(factor > 0 && std::isfinite(static_cast<float>(factor)) && static_cast<float>(factor) > 0, "scale must be positive and finite");
    TORCH_CHECK(cap >= 0 && std::isfinite(static_cast<float>(cap)) && (cap == 0 || static_cast<float>(cap) > 0),
                "cap must be positive and finite in 32 bits, or 0 for none");
    const float* slope = nullptr;
    if (slopes.has_value() && slopes->defined()) {
        TORCH_CHECK(slopes->scalar_type() == at::kFloat && slopes->dim() == 1 && slopes->size(0) == heads && slopes->is_contiguous()
                        && slopes->device() == device,
                    "slopes must be a contiguous float32 tensor with one entry per query head on the cache's device");
        slope = static_cast<const float*>(slopes->const_data_ptr());
    }
    const c10::cuda::CUDAGuard guard(device);
    const at::Tensor           out = at::empty({tokens, q.size(1)}, q.options());
    if (tokens == 0 || p.sequences == 0)
        return out;
    const at::Tensor workspace = at::empty({static_cast<int64_t>(g_workspace_bytes(p.head_dim))}, q.options().dtype(at::kByte));
    const int code = call(c10::cuda::getCurrentCUDAStream().stream(), ld, as_int(tokens), as_int(heads), static_cast<float>(factor),
                          slope, out.mutable_data_ptr(), workspace.mutable_data_ptr());
    if (code != 0)
        raise_paged(what, p, tokens, heads, code);
    return out;
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& cu_tokens,
                          const at::Tensor& context, const at::Tensor& page_table, const at::Tensor& tree_mask,
                          std::optional<double> scale, double cap, const std::optional<at::Tensor>& slopes,
                          const std::optional<at::Tensor>& positions)
{
    const Paged      p      = paged(k_cache, v_cache, cu_tokens, context, page_table);
    const at::Device device = k_cache.device();
    TORCH_CHECK(tree_mask.scalar_type() == at::kLong && tree_mask.dim() == 1 && tree_mask.is_contiguous() && tree_mask.device() == device
                    && tree_mask.size(0) == q.size(0),
                "tree_mask must be a contiguous int64 tensor with one mask per row on the cache's device");
    const bool has_positions = positions.has_value() && positions->defined();
    TORCH_CHECK(has_positions || !slopes.has_value() || !slopes->defined(), "slopes need the positions of the drafted tokens");
    if (has_positions)
        TORCH_CHECK(positions->dim() == 1 && positions->size(0) == q.size(0), "positions must have one entry per row");
    const int* place = has_positions ? int_array(*positions, 1, device, "positions") : nullptr;
    return attention("TreeAttention", q, p, device, scale, cap, slopes,
                     [&](void* stream, int ld, int tokens, int heads, float factor, const float* slope, void* out, void* workspace) {
                         return g_tree(stream, q.const_data_ptr(), ld, k_cache.const_data_ptr(), v_cache.const_data_ptr(), p.pages,
                                       p.page_size, p.cu_tokens, p.context, p.page_table, p.table_width, p.sequences, tokens, heads,
                                       p.kv_heads, p.head_dim, static_cast<const unsigned long long*>(tree_mask.const_data_ptr()),
                                       place, factor, static_cast<float>(cap), slope, out, workspace);
                     });
}

at::Tensor prompt_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& cu_tokens,
                            const at::Tensor& context, const at::Tensor& page_table, const std::optional<at::Tensor>& prefix,
                            std::optional<double> scale, double cap, const std::optional<at::Tensor>& slopes)
{
    const Paged      p          = paged(k_cache, v_cache, cu_tokens, context, page_table);
    const at::Device device     = k_cache.device();
    const bool       has_prefix = prefix.has_value() && prefix->defined();
    if (has_prefix)
        TORCH_CHECK(prefix->dim() == 1 && prefix->size(0) == p.sequences, "prefix must have one entry per sequence");
    const int* ahead = has_prefix ? int_array(*prefix, 1, device, "prefix") : nullptr;
    return attention("PromptAttention", q, p, device, scale, cap, slopes,
                     [&](void* stream, int ld, int tokens, int heads, float factor, const float* slope, void* out, void* workspace) {
                         return g_prompt(stream, q.const_data_ptr(), ld, k_cache.const_data_ptr(), v_cache.const_data_ptr(), p.pages,
                                         p.page_size, p.cu_tokens, p.context, p.page_table, p.table_width, p.sequences, tokens,
                                         heads, p.kv_heads, p.head_dim, ahead, factor, static_cast<float>(cap), slope, out, workspace);
                     });
}

void cache_accept(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& cu_tokens, const at::Tensor& context,
                  const at::Tensor& page_table, const at::Tensor& accepted, const at::Tensor& accepted_lengths)
{
    const Paged      p      = paged(k_cache, v_cache, cu_tokens, context, page_table, true);
    const at::Device device = k_cache.device();
    const int*       path   = int_array(accepted, 2, device, "accepted");
    const int*       length = int_array(accepted_lengths, 1, device, "accepted_lengths");
    TORCH_CHECK(accepted.size(0) == p.sequences && accepted_lengths.size(0) == p.sequences,
                "accepted and accepted_lengths must have one row and one entry per sequence");
    TORCH_CHECK(accepted.size(1) <= 64, "at most 64 tokens of a sequence can be accepted at a time, not ", accepted.size(1));
    if (p.sequences == 0 || accepted.size(1) == 0)
        return;
    const c10::cuda::CUDAGuard guard(device);
    const int code = g_accept(c10::cuda::getCurrentCUDAStream().stream(), k_cache.mutable_data_ptr(), v_cache.mutable_data_ptr(),
                              p.layers, p.pages, p.page_size, p.cu_tokens, p.context, p.page_table, p.table_width, p.sequences,
                              std::numeric_limits<int>::max(), p.kv_heads, p.head_dim, path, length, as_int(accepted.size(1)));
    if (code != 0)
        raise_paged("CacheAccept", p, 0, 0, code);
}

}  // namespace

extern "C" void flashllm_torch_bind(void* spmm_fn, void* tile_offsets_fn, void* pack_fn, void* rotary_fn, void* tree_fn,
                                    void* prompt_fn, void* accept_fn, void* workspace_bytes_fn, PyObject* error_class)
{
    g_rotary          = reinterpret_cast<decltype(g_rotary)>(rotary_fn);
    g_tree            = reinterpret_cast<decltype(g_tree)>(tree_fn);
    g_prompt          = reinterpret_cast<decltype(g_prompt)>(prompt_fn);
    g_accept          = reinterpret_cast<decltype(g_accept)>(accept_fn);
    g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(workspace_bytes_fn);
    g_spmm         = reinterpret_cast<SpmmFn>(spmm_fn);
    g_tile_offsets = reinterpret_cast<TileOffsetsFn>(tile_offsets_fn);
    g_pack         = reinterpret_cast<PackFn>(pack_fn);
    g_error_class  = error_class;  // kept alive by the package that defines it
}

TORCH_LIBRARY_IMPL(flashllm, CUDA, m)
{
    m.impl("spmm", &spmm);
    m.impl("spmm_epilogue", &spmm_epilogue);
    m.impl("encode", &encode);
    m.impl("rotary_append", &rotary_append);
    m.impl("tree_attention", &tree_attention);
    m.impl("prompt_attention", &prompt_attention);
    m.impl("cache_accept", &cache_accept);
}
