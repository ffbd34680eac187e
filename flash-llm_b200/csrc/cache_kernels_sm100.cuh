// Kernels that write a paged key/value cache: rotary positions with the append, and the acceptance of a drafted path.
#pragma once
#include "cache_batch.cuh"

namespace flashllm {

struct RotaryParams {
    CacheBatch    batch;
    const half*   qkv;          // [tokens][ld_qkv]: query heads, key heads, value heads
    half*         q;            // [tokens][ld_q]
    half*         k_cache;
    half*         v_cache;
    const double* frequencies;  // angle per position of each pair, radians
    const int*    positions;    // position of each row for the angle, or nullptr: its place in the sequence
    long long     ld_qkv;
    long long     ld_q;
    int           heads;
    int           rotary_dim;
    float         magnitude;
};

constexpr int kRotaryThreads = 256;

__device__ __forceinline__ void unpack_half8(const uint4& v, float (&x)[8])
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const half2*>(&w[i]));
        x[2 * i]       = f.x;
        x[2 * i + 1]   = f.y;
    }
}

__device__ __forceinline__ uint4 pack_half8(const float (&x)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i]          = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// y1 = x1 cos a - x2 sin a, y2 = x2 cos a + x1 sin a for every pair of the rotated part of a head, a = position * frequency;
// the rest of the head, and values, pass unchanged.  One CTA per token; a thread moves 32 bytes of a head at a time, which hold
// both members of eight pairs in either layout: (i, i + rotary_dim / 2), or INTERLEAVED (2 i, 2 i + 1).
// The angle is reduced in 64 bits: at position 1e6 its 32-bit product would be off by 0.06 radians.
template<int HEAD_DIM, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_append_kernel(const RotaryParams p)
{
    __shared__ float     s_cos[HEAD_DIM / 2], s_sin[HEAD_DIM / 2];
    __shared__ long long s_owner;  // sequence << 32 | first row; -1: nobody's
    const CacheBatch&    c = p.batch;
    const int            n = blockIdx.x;
    if (threadIdx.x == 0)
        s_owner = -1;
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    for (int b = threadIdx.x; b < c.sequences; b += kRotaryThreads) {
        const int begin = c.cu_tokens[b];
        if (begin >= 0 && begin <= n && n < c.cu_tokens[b + 1])
            s_owner = static_cast<long long>(b) << 32 | static_cast<unsigned>(begin);
    }
    __syncthreads();
    const long long owner = s_owner;
    if (owner < 0)
        return;
    const int       b        = static_cast<int>(owner >> 32), first = static_cast<int>(owner);
    const int       context  = c.context[b];
    const long long position = static_cast<long long>(context) + (n - first);
    const bool      fits     = context >= 0 && position < table_positions(c);
    const int       pairs    = p.rotary_dim / 2;
    if (threadIdx.x < pairs) {
        const double turns  = static_cast<double>(p.positions ? p.positions[n] : position) * (p.frequencies[threadIdx.x] * 0.15915494309189535);
        float        sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        s_cos[threadIdx.x] = cosine * p.magnitude;
        s_sin[threadIdx.x] = sine * p.magnitude;
    }
    if (!fits && threadIdx.x == 0)
        atomicOr(c.status, kStatusBadCache);
    long long row = fits ? cache_row(c, b, static_cast<int>(position), 0) : -1;  // of key/value head 0
    __syncthreads();

    constexpr int kUnits = HEAD_DIM / 16;  // of 32 bytes per head
    const int     units  = (p.heads + 2 * c.kv_heads) * kUnits;
    for (int u = threadIdx.x; u < units; u += kRotaryThreads) {
        const int   head = u / kUnits, part = u % kUnits;
        const half* src  = p.qkv + n * p.ld_qkv + static_cast<long long>(head) * HEAD_DIM;
        half*       dst;
        if (head < p.heads) {
            dst = p.q + n * p.ld_q + static_cast<long long>(head) * HEAD_DIM;
        }
        else {
            if (row < 0)
                continue;
            const bool key = head < p.heads + c.kv_heads;
            const int  h   = head - p.heads - (key ? 0 : c.kv_heads);
            dst            = (key ? p.k_cache : p.v_cache) + (row + (static_cast<long long>(h) << c.page_shift)) * HEAD_DIM;
        }
        const bool turned = head < p.heads + c.kv_heads && part * 16 < p.rotary_dim;
        const int  a      = turned && !INTERLEAVED ? part * 8 : part * 16;
        const int  z      = turned && !INTERLEAVED ? pairs + part * 8 : part * 16 + 8;
        uint4      va     = *reinterpret_cast<const uint4*>(src + a);
        uint4      vz     = *reinterpret_cast<const uint4*>(src + z);
        if (turned) {
            float x[8], y[8];
            unpack_half8(va, x);
            unpack_half8(vz, y);
            float co[8], si[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                co[i] = s_cos[part * 8 + i];
                si[i] = s_sin[part * 8 + i];
            }
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
                    x[2 * i]     = x0 * co[i] - x1 * si[i];
                    x[2 * i + 1] = x1 * co[i] + x0 * si[i];
                    y[2 * i]     = y0 * co[i + 4] - y1 * si[i + 4];
                    y[2 * i + 1] = y1 * co[i + 4] + y0 * si[i + 4];
                }
            }
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x0 = x[i], y0 = y[i];
                    x[i] = x0 * co[i] - y0 * si[i];
                    y[i] = y0 * co[i] + x0 * si[i];
                }
            }
            va = pack_half8(x);
            vz = pack_half8(y);
        }
        *reinterpret_cast<uint4*>(dst + a) = va;
        *reinterpret_cast<uint4*>(dst + z) = vz;
    }
}

struct AcceptParams {
    CacheBatch batch;
    half*      k_cache;  // [layers][pages][kv_heads][page_size][head_dim]
    half*      v_cache;
    const int* accepted;          // [sequences][accepted_width]: drafted tokens in the order in which they are kept
    const int* accepted_lengths;  // [sequences]
    int        accepted_width;    // 1 .. kMaxDrafted
    long long  layer_elems;
};

constexpr int kAcceptThreads = 256;

// Keys and values of drafted token accepted[b][i] move to position context[b] + i.  One CTA per sequence, head and layer, which
// holds everything in registers before it writes, so that sources and targets may overlap in any way.
template<int HEAD_DIM>
__global__ void __launch_bounds__(kAcceptThreads) cache_accept_kernel(const AcceptParams p)
{
    __shared__ long long s_from[kMaxDrafted], s_to[kMaxDrafted];  // rows of the cache; from = to: nothing moves
    const CacheBatch&    c = p.batch;
    const int            b = blockIdx.x, head = blockIdx.y;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Sequence s      = load_sequence(c, b);
    int            length = p.accepted_lengths[b];
    if (length < 0 || length > p.accepted_width || (s.count == 0 && length > 0)) {
        if (threadIdx.x == 0)
            atomicOr(c.status, kStatusBadCache);
        length = 0;
    }
    if (static_cast<int>(threadIdx.x) < length) {
        const int token = p.accepted[static_cast<long long>(b) * p.accepted_width + threadIdx.x];
        long long from = -1, to = -1;
        if (token >= 0 && token < s.count && static_cast<int>(threadIdx.x) < s.count) {
            from = cache_row(c, b, s.context + token, head);
            to   = cache_row(c, b, s.context + static_cast<int>(threadIdx.x), head);
        }
        else
            atomicOr(c.status, kStatusBadCache);
        if (from < 0 || to < 0)
            from = to = 0;
        s_from[threadIdx.x] = from;
        s_to[threadIdx.x]   = to;
    }
    __syncthreads();
    constexpr int kChunks = HEAD_DIM / 8;                                     // 16 bytes each
    constexpr int kPerThread = 2 * kMaxDrafted * kChunks / kAcceptThreads;
    half* const   caches[2] = {p.k_cache + blockIdx.z * p.layer_elems, p.v_cache + blockIdx.z * p.layer_elems};
    uint4         v[kPerThread];
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
        const int i = threadIdx.x + k * kAcceptThreads, row = i / (2 * kChunks), which = i / kChunks % 2;
        if (row < length && s_from[row] != s_to[row])
            v[k] = *reinterpret_cast<const uint4*>((which ? caches[1] : caches[0]) + s_from[row] * HEAD_DIM + i % kChunks * 8);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
        const int i = threadIdx.x + k * kAcceptThreads, row = i / (2 * kChunks), which = i / kChunks % 2;
        if (row < length && s_from[row] != s_to[row])
            *reinterpret_cast<uint4*>((which ? caches[1] : caches[0]) + s_to[row] * HEAD_DIM + i % kChunks * 8) = v[k];
    }
}

}  // namespace flashllm
