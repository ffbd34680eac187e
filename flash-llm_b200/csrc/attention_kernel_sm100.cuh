// Attention of a batch's tokens over a paged key/value cache that holds their own keys and values already.
//
//   s_ij = scale q_i . k_j,  capped: cap tanh(s_ij / cap),  then + slope_h (position_j - position_i)
//   o_i  = sum over the keys j that i sees of softmax_j(s_ij) v_j;  zero for a row that sees none
//
// What token i of a sequence (rows first + i, place context + i in the cache) sees: the whole context, and of the batch's own
// tokens either those up to itself and those of the prefix (prompts), or those whose bit its mask has (trees).
#pragma once
#include "cache_batch.cuh"

namespace flashllm {

struct AttentionParams {
    CacheBatch                batch;
    const half*               q;    // [tokens][ld_q]
    half*                     out;  // [tokens][heads * head_dim]
    const half*               k_cache;
    const half*               v_cache;
    const unsigned long long* tree_mask;  // [tokens], or nullptr: prompts
    const int*                positions;  // [tokens] positions of tree tokens, for the distance
    const int*                prefix;     // [sequences] keys that all tokens of a prompt see, or nullptr
    const float*              slopes;     // [heads], or nullptr
    long long                 ld_q;
    int                       heads;
    float                     scale;
    float                     cap;  // 0: none
};

constexpr int kAttentionThreads = 128;

// One warp per row and head, key by key: a running maximum, the sum and the output in 32 bits.
template<int HEAD_DIM>
__global__ void __launch_bounds__(kAttentionThreads) attention_kernel(const AttentionParams p)
{
    constexpr int     kPairs = HEAD_DIM / 64;  // half2 per lane
    const CacheBatch& c      = p.batch;
    const int         n = blockIdx.x, lane = threadIdx.x & 31;
    const int         head = blockIdx.y * (kAttentionThreads / 32) + (threadIdx.x >> 5);
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    if (head >= p.heads)
        return;
    int owner = -1;
    for (int b = lane; b < c.sequences; b += 32) {
        const int begin = c.cu_tokens[b];
        if (begin >= 0 && begin <= n && n < c.cu_tokens[b + 1])
            owner = b;
    }
    owner = __reduce_max_sync(0xffffffffu, owner);
    if (owner < 0)
        return;
    const Sequence s       = load_sequence(c, owner);
    const int      i       = n - s.first;
    const int      kv_head = head / (p.heads / c.kv_heads);
    half2*         out     = reinterpret_cast<half2*>(p.out + (static_cast<long long>(n) * p.heads + head) * HEAD_DIM);
    const half2*   q       = reinterpret_cast<const half2*>(p.q + n * p.ld_q + static_cast<long long>(head) * HEAD_DIM);
    float2         x[kPairs], o[kPairs];
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
        x[k] = __half22float2(q[lane + 32 * k]);
        o[k] = make_float2(0.0f, 0.0f);
    }
    const unsigned long long mask = p.tree_mask ? p.tree_mask[n] : 0ull;
    int                      end  = s.count > 0 ? s.context + s.count : 0;
    int                      seen = s.context + i + 1;  // keys that are seen because of their place
    if (p.tree_mask) {
        seen = s.context;
        end  = min(end, s.context + kMaxDrafted);
    }
    else if (p.prefix)
        seen = max(seen, p.prefix[owner]);
    const float slope = p.slopes ? p.slopes[head] : 0.0f;
    const int   place = p.tree_mask && p.slopes ? p.positions[n] : s.context + i;
    float       top = -INFINITY, sum = 0.0f;
    for (int j = 0; j < end; ++j) {
        const int drafted = j - s.context;
        if (j >= seen && !(p.tree_mask && (mask >> drafted & 1)))
            continue;
        const long long row   = cache_row(c, owner, j, kv_head);
        const half2*    k_row = reinterpret_cast<const half2*>(p.k_cache + row * HEAD_DIM);
        const half2*    v_row = reinterpret_cast<const half2*>(p.v_cache + row * HEAD_DIM);
        float           dot   = 0.0f;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const float2 y = row < 0 ? make_float2(0.0f, 0.0f) : __half22float2(k_row[lane + 32 * k]);
            dot += x[k].x * y.x + x[k].y * y.y;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
            dot += __shfl_xor_sync(0xffffffffu, dot, d);
        dot *= p.scale;
        if (p.cap > 0.0f)
            dot = p.cap * tanhf(dot / p.cap);
        if (p.slopes)
            dot += slope * static_cast<float>((p.tree_mask && drafted >= 0 ? p.positions[s.first + drafted] : j) - place);
        const float new_top = fmaxf(top, dot);
        const float keep    = new_top == -INFINITY ? 1.0f : expf(top - new_top);
        const float weight  = new_top == -INFINITY ? 0.0f : expf(dot - new_top);
        top                 = new_top;
        sum                 = sum * keep + weight;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const float2 y = row < 0 ? make_float2(0.0f, 0.0f) : __half22float2(v_row[lane + 32 * k]);
            o[k].x         = o[k].x * keep + weight * y.x;
            o[k].y         = o[k].y * keep + weight * y.y;
        }
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < kPairs; ++k)
        out[lane + 32 * k] = sum == 0.0f ? __floats2half2_rn(0.0f, 0.0f) : __floats2half2_rn(o[k].x * inverse, o[k].y * inverse);
}

}  // namespace flashllm
