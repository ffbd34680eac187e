// Host side of the operators around a paged cache of 4 bits, and of the appends with norms: argument checks and launches.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "append_kernels_sm100.cuh"
#include "attention_four_bit_sm100.cuh"
#include "attention_single_sm100.cuh"
#include "cache_api.h"
#include "launch.h"
#include "tiled_csl_host.h"

namespace flashllm {

// The attention kernel of many rows over a cache of 4 bits (attention_api.cu).
cudaError_t launch_rows_over_four_bits(cudaStream_t stream, const AttentionParams& p, int head_dim);

static cudaError_t four_multiprocessors(int* count)
{
    static std::atomic<int> known[64];
    return multiprocessors_once(known, count, []() {
        cudaError_t err   = cudaSuccess;
        auto        raise = [&](auto kernel, int bytes) {
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        };
        raise(four_bit_attention_kernel<64, 1, true>, four_smem_bytes(64, 1));
        raise(four_bit_attention_kernel<64, 1, false>, four_smem_bytes(64, 1));
        raise(four_bit_attention_kernel<64, 2, true>, four_smem_bytes(64, 2));
        raise(four_bit_attention_kernel<64, 2, false>, four_smem_bytes(64, 2));
        raise(four_bit_attention_kernel<128, 1, true>, four_smem_bytes(128, 1));
        raise(four_bit_attention_kernel<128, 1, false>, four_smem_bytes(128, 1));
        raise(four_bit_attention_kernel<128, 2, true>, four_smem_bytes(128, 2));
        raise(four_bit_attention_kernel<128, 2, false>, four_smem_bytes(128, 2));
        raise(window_single_kernel<64, true>, single_smem_bytes(64));
        raise(window_single_kernel<64, false>, single_smem_bytes(64));
        raise(window_single_kernel<128, true>, single_smem_bytes(128));
        raise(window_single_kernel<128, false>, single_smem_bytes(128));
        return err;
    });
}

// Bytes of what a head keeps of a page are counted in 32 bits.
static bool four_bit_page(int page_size)
{
    return page_size <= 1 << 24;
}

// The checks that the appends share, and the launch.
static cudaError_t append(cudaStream_t stream, bool four_bit, const void* QKV, int ld_qkv, void* Q, int ld_q, void* K_cache,
                          void* V_cache, int pages, int page_size, const int* cu_tokens, const int* context,
                          const int* page_table, int table_width, int sequences, int tokens, int heads, int kv_heads,
                          int head_dim, const double* frequencies, int rotary_dim, int interleaved, float magnitude,
                          const int* positions, const void* q_norm, const void* k_norm, float eps)
{
    AppendParams  p{};
    RotaryParams& r = p.rotary;
    if (!describe_batch(&r.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || heads < 1 || static_cast<long long>(heads) * head_dim > (1 << 24) || static_cast<long long>(kv_heads) * head_dim > (1 << 24)
        || !rows_fit(QKV, ld_qkv, heads + 2 * kv_heads, head_dim) || !rows_fit(Q, ld_q, heads, head_dim) || rotary_dim < 0
        || rotary_dim > head_dim || rotary_dim % 16 != 0 || (rotary_dim > 0 && frequencies == nullptr) || !std::isfinite(magnitude)
        || (four_bit && !four_bit_page(page_size)) || !aligned16(q_norm) || !aligned16(k_norm) || !(eps >= 0.0f) || !std::isfinite(eps))
        return cudaErrorInvalidValue;
    if (tokens == 0 || sequences == 0)
        return cudaSuccess;
    if (Q == QKV && ld_q != ld_qkv)  // a row's queries would go where another CTA still reads
        return cudaErrorInvalidValue;
    if (const int err = device_status_pointer(&r.batch.status))
        return static_cast<cudaError_t>(err);
    r.qkv         = static_cast<const half*>(QKV);
    r.q           = static_cast<half*>(Q);
    r.k_cache     = static_cast<half*>(K_cache);
    r.v_cache     = static_cast<half*>(V_cache);
    r.frequencies = frequencies;
    r.positions   = positions;
    r.ld_qkv      = ld_qkv;
    r.ld_q        = ld_q;
    r.heads       = heads;
    r.rotary_dim  = rotary_dim;
    r.magnitude   = magnitude;
    p.q_norm      = static_cast<const half*>(q_norm);
    p.k_norm      = static_cast<const half*>(k_norm);
    p.eps         = eps;
    int sms       = 0;
    if (const cudaError_t err = four_multiprocessors(&sms))
        return err;
    // As few rounds of CTAs over the multiprocessors, which hold four at a time, as kAppendRows allow, and tokens dealt out evenly over
    // them (6612 tokens, replayed from a graph: 41.5 us with 8 each, 1.4 rounds, 37.7 with 6, 36.0 to 36.8 with 12, all at once).
    const long long places = 4ll * sms, rounds = (tokens + kAppendRows * places - 1) / (kAppendRows * places);
    p.rows                 = static_cast<int>((tokens + rounds * places - 1) / (rounds * places));
    auto launch            = [&](auto kernel) {
        return launch_in_stream_order(kernel, dim3((tokens - 1) / p.rows + 1), dim3(kRotaryThreads), 0, stream, 1, p);
    };
    auto of_cache = [&](auto sixteen, auto four) { return four_bit ? launch(four) : launch(sixteen); };
    if (head_dim == 64)
        return interleaved ? of_cache(norm_append_kernel<64, true, false>, norm_append_kernel<64, true, true>)
                           : of_cache(norm_append_kernel<64, false, false>, norm_append_kernel<64, false, true>);
    return interleaved ? of_cache(norm_append_kernel<128, true, false>, norm_append_kernel<128, true, true>)
                       : of_cache(norm_append_kernel<128, false, false>, norm_append_kernel<128, false, true>);
}

// The warps' kernels make do with the workspace of the others.
static_assert(four_workspace_bytes(1, 64) <= attn_workspace_bytes(1, 64) && four_workspace_bytes(1, 128) <= attn_workspace_bytes(1, 128)
                  && four_workspace_bytes(256, 128) <= attn_workspace_bytes(256, 128),
              "workspace");

// Rows of a sequence (tokens x query heads of a key/value head) up to which it goes through the warps' kernel, sixteen at a time (16
// sequences of 2000 to 4000 positions, 32 rows each: 42 us, the other kernel 47; 64 rows: 63 and 51).
constexpr int kFourMostRows = 32;

template<int HEAD_DIM, int TILES>
static cudaError_t launch_four_bit(cudaStream_t stream, const FourBitParams& p, int ctas)
{
    const bool  plain = p.cap == 0.0f && p.slopes == nullptr;
    cudaError_t err   = launch_in_stream_order(plain ? four_bit_attention_kernel<HEAD_DIM, TILES, true> : four_bit_attention_kernel<HEAD_DIM, TILES, false>,
                                               dim3(ctas), dim3(four_warps(TILES) * 32), four_smem_bytes(HEAD_DIM, TILES), stream, 1, p);
    if (err != cudaSuccess)
        return err;
    return launch_in_stream_order(four_bit_join_kernel<HEAD_DIM>, dim3(ctas), dim3(256), 0, stream, 1, p);
}

template<int HEAD_DIM>
static cudaError_t launch_single(cudaStream_t stream, const FourBitParams& p, int ctas)
{
    const bool  plain = p.cap == 0.0f && p.slopes == nullptr;
    cudaError_t err   = launch_in_stream_order(plain ? window_single_kernel<HEAD_DIM, true> : window_single_kernel<HEAD_DIM, false>, dim3(ctas),
                                               dim3(kSingleWarps * 32), single_smem_bytes(HEAD_DIM), stream, 1, p);
    if (err != cudaSuccess)
        return err;
    return launch_in_stream_order(four_bit_join_kernel<HEAD_DIM>, dim3(ctas), dim3(256), 0, stream, 1, p);
}

// Single tokens through a window over a cache of fp16; `a` has been checked.
cudaError_t launch_single_tokens(cudaStream_t stream, const AttentionParams& a, int head_dim)
{
    int         sms = 0;
    cudaError_t err = four_multiprocessors(&sms);
    if (err != cudaSuccess)
        return err;
    FourBitParams p{};
    p.batch       = a.batch;
    p.q           = a.q;
    p.out         = a.out;
    p.k_cache     = reinterpret_cast<const unsigned char*>(a.k_cache);
    p.v_cache     = reinterpret_cast<const unsigned char*>(a.v_cache);
    p.slopes      = a.slopes;
    p.workspace   = a.workspace;
    p.ld_q        = a.ld_q;
    p.heads       = a.heads;
    p.share       = a.share;
    p.share_magic = a.share_magic;
    p.share_shift = a.share_shift;
    p.token_tiles = (a.share + 7) / 8;
    p.window      = a.window;
    p.sinks       = a.sinks;
    p.most_rows   = 0x7fffffff;
    p.scale       = a.scale;
    p.cap         = a.cap;
    p.unit        = a.cap == 0.0f && a.slopes == nullptr ? a.scale * CUDART_L2E_F : 1.0f;  // (plain kernels' maxima are of products)
    return head_dim == 64 ? launch_single<64>(stream, p, sms) : launch_single<128>(stream, p, sms);
}

}  // namespace flashllm

using namespace flashllm;

extern "C" {

int FlashLLM_NormRotaryAppend(void* stream, const void* QKV, int ld_qkv, void* Q, int ld_q, void* K_cache, void* V_cache, int pages,
                              int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                              int sequences, int tokens, int heads, int kv_heads, int head_dim, const double* frequencies,
                              int rotary_dim, int interleaved, float magnitude, const int* positions, const void* q_norm,
                              const void* k_norm, float eps)
{
    if (q_norm == nullptr || k_norm == nullptr)
        return static_cast<int>(cudaErrorInvalidValue);
    return static_cast<int>(append(static_cast<cudaStream_t>(stream), false, QKV, ld_qkv, Q, ld_q, K_cache, V_cache, pages, page_size,
                                   cu_tokens, context, page_table, table_width, sequences, tokens, heads, kv_heads, head_dim,
                                   frequencies, rotary_dim, interleaved, magnitude, positions, q_norm, k_norm, eps));
}

int FlashLLM_FourBitAppend(void* stream, const void* QKV, int ld_qkv, void* Q, int ld_q, void* K_cache, void* V_cache, int pages,
                           int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                           int sequences, int tokens, int heads, int kv_heads, int head_dim, const double* frequencies,
                           int rotary_dim, int interleaved, float magnitude, const int* positions, const void* q_norm,
                           const void* k_norm, float eps)
{
    return static_cast<int>(append(static_cast<cudaStream_t>(stream), true, QKV, ld_qkv, Q, ld_q, K_cache, V_cache, pages, page_size,
                                   cu_tokens, context, page_table, table_width, sequences, tokens, heads, kv_heads, head_dim,
                                   frequencies, rotary_dim, interleaved, magnitude, positions, q_norm, k_norm, eps));
}

int FlashLLM_FourBitRead(void* stream, const void* K_cache, const void* V_cache, int pages, int page_size, const int* cu_tokens,
                         const int* context, const int* page_table, int table_width, int sequences, int tokens, int kv_heads,
                         int head_dim, void* K_out, void* V_out)
{
    ReadParams p{};
    if (!describe_batch(&p.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || !four_bit_page(page_size) || static_cast<long long>(kv_heads) * head_dim > (1 << 24) || K_out == nullptr || V_out == nullptr || !aligned16(K_out)
        || !aligned16(V_out))
        return static_cast<int>(cudaErrorInvalidValue);
    if (tokens == 0 || sequences == 0)
        return 0;
    if (const int err = device_status_pointer(&p.batch.status))
        return err;
    int sms = 0;
    if (const cudaError_t err = four_multiprocessors(&sms))
        return static_cast<int>(err);
    p.cache[0] = static_cast<const unsigned char*>(K_cache);
    p.cache[1] = static_cast<const unsigned char*>(V_cache);
    p.out[0]   = static_cast<half*>(K_out);
    p.out[1]   = static_cast<half*>(V_out);
    // As many rows for a CTA as leave several CTAs for each multiprocessor.
    for (p.row_shift = 0; p.row_shift < 4 && tokens >> (p.row_shift + 1) >= 8 * sms;)
        ++p.row_shift;
    const int rows   = 1 << p.row_shift;
    auto      launch = [&](auto kernel) {
        return launch_in_stream_order(kernel, dim3((tokens - 1) / rows + 1), dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream), 1, p);
    };
    return static_cast<int>(head_dim == 64 ? launch(four_bit_read_kernel<64>) : launch(four_bit_read_kernel<128>));
}

int FlashLLM_FourBitAttention(void* stream, const void* Q, int ld_q, const void* K_cache, const void* V_cache, int pages,
                              int page_size, const int* cu_tokens, const int* context, const int* page_table, int table_width,
                              int sequences, int tokens, int heads, int kv_heads, int head_dim, int window, int sinks, float scale,
                              float cap, const float* slopes, void* Out, void* workspace)
{
    FourBitParams p{};
    if (!describe_batch(&p.batch, K_cache, V_cache, pages, page_size, cu_tokens, context, page_table, table_width, sequences, tokens,
                        kv_heads, head_dim)
        || !four_bit_page(page_size) || heads < 1 || heads % kv_heads != 0 || heads / kv_heads > kAttnRows || static_cast<long long>(heads) * head_dim > (1 << 24)
        || !rows_fit(Q, ld_q, heads, head_dim) || workspace == nullptr || !aligned16(workspace) || Out == nullptr || !aligned16(Out)
        || !scores_fit(scale, cap) || window < 0 || sinks < 0 || static_cast<long long>(tokens) * heads > 0x7fffffffll - 256)
        return static_cast<int>(cudaErrorInvalidValue);
    if (tokens == 0 || sequences == 0)
        return 0;
    if (const int err = device_status_pointer(&p.batch.status))
        return err;
    int sms = 0;
    if (const cudaError_t err = four_multiprocessors(&sms))
        return static_cast<int>(err);
    p.q         = static_cast<const half*>(Q);
    p.out       = static_cast<half*>(Out);
    p.k_cache   = static_cast<const unsigned char*>(K_cache);
    p.v_cache   = static_cast<const unsigned char*>(V_cache);
    p.slopes    = slopes;
    p.workspace = static_cast<unsigned char*>(workspace);
    p.ld_q      = ld_q;
    p.heads     = heads;
    AttentionParams a{};
    attn_set_heads(&a, heads, kv_heads);
    p.share       = a.share;
    p.share_magic = a.share_magic;
    p.share_shift = a.share_shift;
    p.window    = window > 0 ? window : 0x7fffffff;
    p.sinks     = window > 0 ? sinks : 0;
    // Sequences of more than kFourMostRows rows are the other kernel's.  The host does not know the rows of each: where one token has
    // more, all are (64 sequences of 1000 to 4000 positions, two key/value heads of 64 query heads of 128 each: 67 us, by warps 81); where
    // there is no more than a token for each sequence, or so many rows in all, none are (and rows that are more are right, if slower),
    // since the other kernel's launch and its join's are some 8 us though they find nothing to do.  Two tokens to a sequence are not
    // told from a long piece of one prompt among single tokens, which by warps would take as long as a sequence for every 16 rows.
    const bool all  = p.share > kFourMostRows;
    const bool many = all || (tokens > sequences && static_cast<long long>(tokens) * p.share > kFourMostRows);
    p.most_rows     = many ? kFourMostRows : 0x7fffffff;
    p.scale     = scale;
    p.cap       = cap;
    p.unit      = 1.0f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto few = [&](auto dim, auto tiles) { return launch_four_bit<decltype(dim)::value, decltype(tiles)::value>(s, p, sms); };
    using Dim64 = std::integral_constant<int, 64>;
    using Dim128 = std::integral_constant<int, 128>;
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    // Sixteen rows at a time where a sequence has more than eight.
    const bool  two = p.share > 8 || tokens > sequences;
    cudaError_t err = cudaSuccess;
    if (!all)
        err = head_dim == 64 ? (two ? few(Dim64{}, Two{}) : few(Dim64{}, One{})) : (two ? few(Dim128{}, Two{}) : few(Dim128{}, One{}));
    if (err != cudaSuccess || !many)
        return static_cast<int>(err);
    a.batch      = p.batch;
    a.q          = p.q;
    a.out        = p.out;
    a.k_cache    = reinterpret_cast<const half*>(p.k_cache);
    a.v_cache    = reinterpret_cast<const half*>(p.v_cache);
    a.slopes     = slopes;
    a.workspace  = p.workspace;
    a.ld_q       = ld_q;
    a.scale      = scale;
    a.cap        = cap;
    a.window     = p.window;
    a.sinks      = p.sinks;
    a.least_rows = all ? 0 : kFourMostRows + 1;
    return static_cast<int>(launch_rows_over_four_bits(s, a, head_dim));
}

}  // extern "C"
