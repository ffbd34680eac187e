// Host side of the operators around a paged key/value cache: argument checks and launches.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/SpMM_API.cuh"
#include "attention_kernel_sm100.cuh"
#include "cache_kernels_sm100.cuh"
#include "launch.h"
#include "tiled_csl_host.h"

namespace flashllm {

static bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// What every operator's cache and batch have to be.
static bool describe_batch(CacheBatch* batch, const void* K_cache, const void* V_cache, int pages, int page_size,
                           const int* cu_tokens, const int* context, const int* page_table, int table_width, int sequences,
                           int tokens, int kv_heads, int head_dim)
{
    if (K_cache == nullptr || V_cache == nullptr || cu_tokens == nullptr || context == nullptr || page_table == nullptr
        || !aligned16(K_cache) || !aligned16(V_cache) || pages < 1 || kv_heads < 1 || (head_dim != 64 && head_dim != 128)
        || page_size < 16 || (page_size & (page_size - 1)) != 0 || table_width < 1 || sequences < 0
        || sequences > kMaxSequences || tokens < 0)
        return false;
    // Positions, and the pages of all heads, are counted in ints; a tile may reach 127 positions behind the last.
    if (static_cast<long long>(table_width) * page_size > 0x7fffffffll - 256
        || static_cast<long long>(pages) * kv_heads > 0x7fffffffll - 1)
        return false;
    batch->cu_tokens   = cu_tokens;
    batch->context     = context;
    batch->page_table  = page_table;
    batch->sequences   = sequences;
    batch->tokens      = tokens;
    batch->table_width = table_width;
    batch->pages       = pages;
    batch->page_shift  = __builtin_ctz(static_cast<unsigned>(page_size));
    batch->kv_heads    = kv_heads;
    return true;
}

static bool rows_fit(const void* matrix, int ld, int heads, int head_dim)
{
    return matrix != nullptr && aligned16(matrix) && ld % 8 == 0 && ld >= static_cast<long long>(heads) * head_dim;
}

static cudaError_t launch_rotary(cudaStream_t stream, const RotaryParams& p, int head_dim, bool interleaved)
{
    auto launch = [&](auto kernel) {
        return launch_in_stream_order(kernel, dim3(p.batch.tokens), dim3(kRotaryThreads), 0, stream, 1, p);
    };
    if (head_dim == 64)
        return interleaved ? launch(rotary_append_kernel<64, true>) : launch(rotary_append_kernel<64, false>);
    return interleaved ? launch(rotary_append_kernel<128, true>) : launch(rotary_append_kernel<128, false>);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled()
{
    static const EncodeTiledFn function = []() -> EncodeTiledFn {
        void*                           fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess
            || found != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeTiledFn>(fn);
    }();
    return function;
}

// Multiprocessors of the current device, and with them the shared-memory limits of the attention kernels raised: once per
// device.
static cudaError_t multiprocessors(int* count)
{
    constexpr int           kMaxDevices = 64;
    static std::atomic<int> known[kMaxDevices];
    int                     device = 0;
    cudaError_t             err    = cudaGetDevice(&device);
    if (err != cudaSuccess)
        return err;
    if (device < 0 || device >= kMaxDevices)
        return cudaErrorInvalidDevice;
    *count = known[device].load(std::memory_order_acquire);
    if (*count > 0)
        return cudaSuccess;
    err = cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device);
    auto raise = [&](auto kernel, int bytes) {
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    raise(attention_kernel<64, true>, attn_smem_bytes(64));
    raise(attention_kernel<64, false>, attn_smem_bytes(64));
    raise(attention_kernel<128, true>, attn_smem_bytes(128));
    raise(attention_kernel<128, false>, attn_smem_bytes(128));
    if (err == cudaSuccess)
        known[device].store(*count, std::memory_order_release);
    return err;
}

// A cache tensor as (head_dim, page_size, pages * kv_heads), copied in boxes of 64 columns and the rows of a page, 128 at most.
static bool encode_cache(CUtensorMap* map, const half* cache, const CacheBatch& batch, int head_dim)
{
    const EncodeTiledFn encode = encode_tiled();
    if (encode == nullptr)
        return false;
    const cuuint64_t page = cuuint64_t(1) << batch.page_shift, row = static_cast<cuuint64_t>(head_dim) * 2;
    const cuuint64_t dims[3]    = {static_cast<cuuint64_t>(head_dim), page, static_cast<cuuint64_t>(batch.pages) * batch.kv_heads};
    const cuuint64_t strides[2] = {row, page * row};
    const cuuint32_t box[3]     = {64, static_cast<cuuint32_t>(page < kAttnKeys ? page : kAttnKeys), 1};
    const cuuint32_t ones[3]    = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<half*>(cache), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
           == CUDA_SUCCESS;
}

// The queries as (head_dim, heads, tokens), copied in boxes of 64 columns, the heads of a group and as many tokens as `rows` hold.
static bool encode_rows(CUtensorMap* map, const AttentionParams& p, int head_dim, int rows)
{
    const EncodeTiledFn encode = encode_tiled();
    if (encode == nullptr)
        return false;
    const cuuint64_t dims[3]    = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(p.heads),
                                   static_cast<cuuint64_t>(p.batch.tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_dim) * 2, static_cast<cuuint64_t>(p.ld_q) * 2};
    const cuuint32_t box[3]     = {64, static_cast<cuuint32_t>(p.share), static_cast<cuuint32_t>(rows / p.share)};
    const cuuint32_t ones[3]    = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<half*>(p.q), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
           == CUDA_SUCCESS;
}

template<int HEAD_DIM>
static cudaError_t launch_attention(cudaStream_t stream, const AttentionParams& p)
{
    int         sms = 0;
    cudaError_t err = multiprocessors(&sms);
    if (err != cudaSuccess)
        return err;
    CUtensorMap map_q, map_q_few, map_k, map_v;
    if (!encode_rows(&map_q, p, HEAD_DIM, p.tile_rows) || !encode_rows(&map_q_few, p, HEAD_DIM, p.few_rows > 0 ? p.few_rows : p.tile_rows)
        || !encode_cache(&map_k, p.k_cache, p.batch, HEAD_DIM) || !encode_cache(&map_v, p.v_cache, p.batch, HEAD_DIM))
        return cudaErrorInvalidValue;
    const bool plain = p.cap == 0.0f && p.slopes == nullptr;
    err = launch_in_stream_order(plain ? attention_kernel<HEAD_DIM, true> : attention_kernel<HEAD_DIM, false>, dim3(sms), dim3(kAttnThreads), attn_smem_bytes(HEAD_DIM), stream, 1, map_q,
                                 map_q_few, map_k, map_v, p);
    if (err != cudaSuccess)
        return err;
    return launch_in_stream_order(attention_join_kernel<HEAD_DIM>, dim3(sms, kAttnSlotRows / 32), dim3(256), 0, stream, 1, p, sms);
}

// The checks that tree and prompt attention share, and the launch.
static cudaError_t attend(cudaStream_t stream, AttentionParams p, const void* Q, int ld_q, const void* K_cache,
                          const void* V_cache, int pages, int page_size, const int* cu_tokens, const int* context,
                          const int* page_table, int table_width, int sequences, int tokens, int heads, int kv_heads,
                          int head_dim, float scale, float cap, const float* slopes, void* Out, void* workspace)
{
    if (!describe_batch(&p.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || heads < 1 || heads % kv_heads != 0 || heads / kv_heads > kAttnRows || static_cast<long long>(heads) * head_dim > (1 << 24) || !rows_fit(Q, ld_q, heads, head_dim)
        || workspace == nullptr || !aligned16(workspace) || Out == nullptr || !aligned16(Out) || !(scale > 0.0f) || !std::isfinite(scale) || !(cap >= 0.0f) || !std::isfinite(cap)
        // What the kernels make of them is finite too, scores times log2 e of 128 products of the largest fp16 values among it.
        || !std::isfinite(scale * 8e11f) || !std::isfinite(cap * 1.45f) || (cap > 0.0f && !std::isfinite(scale / cap * 3.0f))
        || static_cast<long long>(tokens) * heads > 0x7fffffffll - 256)
        return cudaErrorInvalidValue;
    if (tokens == 0 || sequences == 0)
        return cudaSuccess;
    if (const int err = device_status_pointer(&p.batch.status))
        return static_cast<cudaError_t>(err);
    p.q       = static_cast<const half*>(Q);
    p.out     = static_cast<half*>(Out);
    p.k_cache = static_cast<const half*>(K_cache);
    p.v_cache = static_cast<const half*>(V_cache);
    p.slopes  = slopes;
    p.ld_q    = ld_q;
    p.scale   = scale;
    p.cap     = cap;
    p.workspace = static_cast<unsigned char*>(workspace);
    attn_set_heads(&p, heads, kv_heads);
    return head_dim == 64 ? launch_attention<64>(stream, p) : launch_attention<128>(stream, p);
}

}  // namespace flashllm

using namespace flashllm;

extern "C" {

int FlashLLM_RotaryAppend(void* stream, const void* QKV, int ld_qkv, void* Q, int ld_q, void* K_cache, void* V_cache, int pages,
                          int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                          int sequences, int tokens, int heads, int kv_heads, int head_dim, const double* frequencies,
                          int rotary_dim, int interleaved, float magnitude, const int* positions)
{
    RotaryParams p{};
    if (!describe_batch(&p.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || heads < 1 || static_cast<long long>(heads) * head_dim > (1 << 24) || static_cast<long long>(kv_heads) * head_dim > (1 << 24)
        || !rows_fit(QKV, ld_qkv, heads + 2 * kv_heads, head_dim) || !rows_fit(Q, ld_q, heads, head_dim) || rotary_dim < 0
        || rotary_dim > head_dim || rotary_dim % 16 != 0 || (rotary_dim > 0 && frequencies == nullptr) || !std::isfinite(magnitude))
        return static_cast<int>(cudaErrorInvalidValue);
    if (tokens == 0 || sequences == 0)
        return 0;
    if (Q == QKV && ld_q != ld_qkv)  // a row's queries would go where another CTA still reads
        return static_cast<int>(cudaErrorInvalidValue);
    if (const int err = device_status_pointer(&p.batch.status))
        return err;
    p.qkv         = static_cast<const half*>(QKV);
    p.q           = static_cast<half*>(Q);
    p.k_cache     = static_cast<half*>(K_cache);
    p.v_cache     = static_cast<half*>(V_cache);
    p.frequencies = frequencies;
    p.positions   = positions;
    p.ld_qkv      = ld_qkv;
    p.ld_q        = ld_q;
    p.heads       = heads;
    p.rotary_dim  = rotary_dim;
    p.magnitude   = magnitude;
    return static_cast<int>(launch_rotary(static_cast<cudaStream_t>(stream), p, head_dim, interleaved != 0));
}

unsigned long long FlashLLM_Attention_WorkspaceBytes(int head_dim)
{
    int sms = 0;
    if ((head_dim != 64 && head_dim != 128) || multiprocessors(&sms) != cudaSuccess)
        return 0;
    return attn_workspace_bytes(sms, head_dim);
}

int FlashLLM_TreeAttention(void* stream, const void* Q, int ld_q, const void* K_cache, const void* V_cache, int pages,
                           int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                           int sequences, int tokens, int heads, int kv_heads, int head_dim, const unsigned long long* tree_mask,
                           const int* positions, float scale, float cap, const float* slopes, void* Out, void* workspace)
{
    if (tree_mask == nullptr || (slopes != nullptr && positions == nullptr))
        return static_cast<int>(cudaErrorInvalidValue);
    AttentionParams p{};
    p.tree_mask = tree_mask;
    p.positions = positions;
    return static_cast<int>(attend(static_cast<cudaStream_t>(stream), p, Q, ld_q, K_cache, V_cache, pages, page_size, cu_tokens,
                                   context, page_table, table_width, sequences, tokens, heads, kv_heads, head_dim, scale, cap,
                                   slopes, Out, workspace));
}

int FlashLLM_PromptAttention(void* stream, const void* Q, int ld_q, const void* K_cache, const void* V_cache, int pages,
                             int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                             int sequences, int tokens, int heads, int kv_heads, int head_dim, const int* prefix, float scale,
                             float cap, const float* slopes, void* Out, void* workspace)
{
    AttentionParams p{};
    p.prefix = prefix;
    return static_cast<int>(attend(static_cast<cudaStream_t>(stream), p, Q, ld_q, K_cache, V_cache, pages, page_size, cu_tokens,
                                   context, page_table, table_width, sequences, tokens, heads, kv_heads, head_dim, scale, cap,
                                   slopes, Out, workspace));
}

int FlashLLM_CacheAccept(void* stream, void* K_cache, void* V_cache, int layers, int pages, int page_size, const int* cu_tokens,
                         const int* context, const int* page_table, int table_width, int sequences, int tokens, int kv_heads,
                         int head_dim, const int* accepted, const int* accepted_lengths, int accepted_width)
{
    AcceptParams p{};
    if (!describe_batch(&p.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || layers < 1 || static_cast<long long>(kv_heads) * layers > 0x7fffffffll || accepted == nullptr || accepted_lengths == nullptr || accepted_width < 1
        || accepted_width > kMaxDrafted)
        return static_cast<int>(cudaErrorInvalidValue);
    if (tokens == 0 || sequences == 0)
        return 0;
    if (const int err = device_status_pointer(&p.batch.status))
        return err;
    p.k_cache          = static_cast<half*>(K_cache);
    p.v_cache          = static_cast<half*>(V_cache);
    p.accepted         = accepted;
    p.accepted_lengths = accepted_lengths;
    p.accepted_width   = accepted_width;
    p.layer_elems      = static_cast<long long>(pages) * kv_heads * page_size * head_dim;
    p.layers           = layers;
    // Some four CTAs for each multiprocessor, of a sequence's heads and layers at most as many as there are.
    int sms = 0;
    if (const cudaError_t err = multiprocessors(&sms))
        return static_cast<int>(err);
    const long long heads = static_cast<long long>(kv_heads) * layers;
    const dim3      grid(sequences, static_cast<unsigned>(std::min(heads, (4ll * sms + sequences - 1) / sequences)));
    auto            launch = [&](auto kernel) {
        return launch_in_stream_order(kernel, grid, dim3(kAcceptThreads), 0, static_cast<cudaStream_t>(stream), 1, p);
    };
    return static_cast<int>(head_dim == 64 ? launch(cache_accept_kernel<64>) : launch(cache_accept_kernel<128>));
}

}  // extern "C"
