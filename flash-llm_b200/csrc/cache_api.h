// What the host sides of the paged cache's operators share: checks of a cache and a batch.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>

#include "../../include/SpMM_API.cuh"
#include "cache_batch.cuh"

namespace flashllm {

inline bool aligned16(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// What every operator's cache and batch have to be.
inline bool describe_batch(CacheBatch* batch, const void* K_cache, const void* V_cache, int pages, int page_size,
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

inline bool rows_fit(const void* matrix, int ld, int heads, int head_dim)
{
    return matrix != nullptr && aligned16(matrix) && ld % 8 == 0 && ld >= static_cast<long long>(heads) * head_dim;
}

// Multiprocessors of the current device; `prepare(kernel's attributes)` has been done once for it by then.
template<typename Prepare>
inline cudaError_t multiprocessors_once(std::atomic<int> (&known)[64], int* count, Prepare&& prepare)
{
    int         device = 0;
    cudaError_t err    = cudaGetDevice(&device);
    if (err != cudaSuccess)
        return err;
    if (device < 0 || device >= 64)
        return cudaErrorInvalidDevice;
    *count = known[device].load(std::memory_order_acquire);
    if (*count > 0)
        return cudaSuccess;
    err = cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device);
    if (err == cudaSuccess)
        err = prepare();
    if (err == cudaSuccess)
        known[device].store(*count, std::memory_order_release);
    return err;
}

// The scores' scale and cap, and what the kernels make of them, scores times log2 e of 128 products of the largest fp16 values among
// it, are finite.
inline bool scores_fit(float scale, float cap)
{
    return scale > 0.0f && std::isfinite(scale) && cap >= 0.0f && std::isfinite(cap) && std::isfinite(scale * 8e11f)
           && std::isfinite(cap * 1.45f) && (cap == 0.0f || std::isfinite(scale / cap * 3.0f))
           // (scores of three quarters of the cap take twice the cap times log2 e)
           && (std::isfinite(cap * 2.9f) || scale * 8e11f < 0.7f * cap);
}

}  // namespace flashllm
