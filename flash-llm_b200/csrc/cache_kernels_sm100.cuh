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
// Bound by memory for prompts, for a few tokens by a chain of dependent loads: sequence, page, row.  A thread's first loads of the
// token's own row, which depend on none of them, are issued ahead of it.  Two moves in flight per thread instead of one cost
// registers and with them CTAs: prompts of a hidden-9216 layer 122 us instead of 119.
template<int HEAD_DIM, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_append_kernel(const RotaryParams p)
{
    constexpr int        kUnits = HEAD_DIM / 16;  // of 32 bytes per head
    __shared__ float     s_cos[HEAD_DIM / 2], s_sin[HEAD_DIM / 2];
    __shared__ int       s_sequence, s_position;  // of the token; -1: nobody's, or it does not fit
    const CacheBatch&    c     = p.batch;
    const int            n     = blockIdx.x;
    const int            pairs = p.rotary_dim / 2;
    const int            units = (p.heads + 2 * c.kv_heads) * kUnits;
    const half* const    row   = p.qkv + n * p.ld_qkv;
    if (threadIdx.x == 0)
        s_sequence = -1;
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    uint4 va{}, vz{};
    auto  turned_at = [&](int u) { return u / kUnits < p.heads + c.kv_heads && u % kUnits * 16 < p.rotary_dim; };
    // Where a unit's two halves lie in its head.
    auto offsets = [&](int u, int& a, int& z) {
        const int part = u % kUnits;
        const bool apart = turned_at(u) && !INTERLEAVED;
        a = apart ? part * 8 : part * 16;
        z = apart ? pairs + part * 8 : part * 16 + 8;
    };
    auto load = [&](int u) {
        int a, z;
        offsets(u, a, z);
        va = *reinterpret_cast<const uint4*>(row + u / kUnits * HEAD_DIM + a);
        vz = *reinterpret_cast<const uint4*>(row + u / kUnits * HEAD_DIM + z);
    };
    if (static_cast<int>(threadIdx.x) < units)
        load(threadIdx.x);
    const double frequency = threadIdx.x < pairs ? p.frequencies[threadIdx.x] : 0.0;
    const int    elsewhere = p.positions && threadIdx.x < pairs ? p.positions[n] : 0;
    for (int b = threadIdx.x; b < c.sequences; b += kRotaryThreads) {
        const int begin = max(c.cu_tokens[b], 0), end = min(c.cu_tokens[b + 1], c.tokens), context = c.context[b];
        if (begin <= n && n < end) {  // a sequence that does not fit is left out whole, as load_sequence has it
            const bool fits = context >= 0 && static_cast<long long>(context) + (end - begin) <= table_positions(c);
            s_sequence      = b;
            s_position      = fits ? context + (n - begin) : -1;
        }
    }
    __syncthreads();
    const int b = s_sequence, position = s_position;
    if (b < 0)
        return;
    if (position < 0 && threadIdx.x == 0)
        atomicOr(c.status, kStatusBadCache);
    const long long at = position >= 0 ? cache_row(c, b, position, 0) : -1;  // of key/value head 0
    if (threadIdx.x < pairs) {
        const double turns = static_cast<double>(p.positions ? elsewhere : position) * (frequency * 0.15915494309189535);
        float        sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        s_cos[threadIdx.x] = cosine * p.magnitude;
        s_sin[threadIdx.x] = sine * p.magnitude;
    }
    __syncthreads();

    for (int u = threadIdx.x; u < units; u += kRotaryThreads) {
        if (u != static_cast<int>(threadIdx.x))
            load(u);
        const int head = u / kUnits, part = u % kUnits;
        half*     dst;
        if (head < p.heads) {
            dst = p.q + n * p.ld_q + static_cast<long long>(head) * HEAD_DIM;
        }
        else {
            if (at < 0)
                continue;
            const bool key = head < p.heads + c.kv_heads;
            const int  h   = head - p.heads - (key ? 0 : c.kv_heads);
            dst            = (key ? p.k_cache : p.v_cache) + (at + (static_cast<long long>(h) << c.page_shift)) * HEAD_DIM;
        }
        int a, z;
        offsets(u, a, z);
        if (position < 0)  // queries of a sequence that does not fit
            va = vz = make_uint4(0, 0, 0, 0);
        else if (turned_at(u)) {
            float x[8], y[8], co[8], si[8];
            unpack_half8(va, x);
            unpack_half8(vz, y);
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
    int        layers;
    long long  layer_elems;
};

constexpr int kAcceptThreads = 256;

// Keys and values of drafted token accepted[b][i] move to position context[b] + i.  A CTA takes a share of one sequence's heads
// and layers, as many at a time as its registers hold whole: all of a head is read before any of it is written, so that sources
// and targets may overlap in any way.  Bound by the chain of loads that leads to the rows, which the heads and layers of a CTA
// share (24 sequences, 32 layers: a CTA for each head and layer 14.3 us, this 8.0).
template<int HEAD_DIM>
__global__ void __launch_bounds__(kAcceptThreads) cache_accept_kernel(const AcceptParams p)
{
    constexpr int        kChunks    = 2 * HEAD_DIM / 8;  // of 16 bytes in a row of keys and the row of values
    constexpr int        kPerThread = kMaxDrafted * kChunks / kAcceptThreads;
    __shared__ long long s_from[kMaxDrafted], s_to[kMaxDrafted];  // rows of the first head; from = to: nothing moves
    const CacheBatch&    c = p.batch;
    const int            b = blockIdx.x, i = threadIdx.x;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int      token  = i < p.accepted_width ? p.accepted[static_cast<long long>(b) * p.accepted_width + i] : 0;
    int            length = p.accepted_lengths[b];
    const Sequence s      = load_sequence(c, b);
    if (length < 0 || length > p.accepted_width || (s.count == 0 && length > 0)) {
        if (threadIdx.x == 0)
            atomicOr(c.status, kStatusBadCache);
        length = 0;
    }
    if (i < length) {
        long long from = -1, to = -1;
        if (token >= 0 && token < s.count && i < s.count) {
            from = cache_row(c, b, s.context + token, 0);
            to   = cache_row(c, b, s.context + i, 0);
        }
        else
            atomicOr(c.status, kStatusBadCache);
        if (from < 0 || to < 0)
            from = to = 0;
        s_from[i] = from;
        s_to[i]   = to;
    }
    __syncthreads();
    if (length == 0)
        return;
    const int heads    = c.kv_heads * p.layers;  // of all layers
    const int at_once  = max(1, kPerThread * kAcceptThreads / (length * kChunks));
    const int per_head = length * kChunks;
    for (int head0 = blockIdx.y * at_once; head0 < heads; head0 += gridDim.y * at_once) {
        uint4     v[kPerThread];
        long long to[kPerThread];  // element of the cache, -1: nothing moves
#pragma unroll
        for (int k = 0; k < kPerThread; ++k) {
            const int at = threadIdx.x + k * kAcceptThreads, head = head0 + at / per_head, in = at % per_head;
            to[k] = -1;
            if (at >= at_once * per_head || head >= heads)
                continue;
            const int row = in / kChunks, chunk = in % kChunks;
            if (s_from[row] == s_to[row])
                continue;
            const long long base = head / c.kv_heads * p.layer_elems + (static_cast<long long>(head % c.kv_heads) << c.page_shift) * HEAD_DIM
                                   + chunk % (kChunks / 2) * 8;
            const half* src = (chunk < kChunks / 2 ? p.k_cache : p.v_cache) + base + s_from[row] * HEAD_DIM;
            v[k]  = *reinterpret_cast<const uint4*>(src);
            to[k] = base + s_to[row] * HEAD_DIM;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPerThread; ++k)
            if (to[k] >= 0) {
                const int chunk = (threadIdx.x + k * kAcceptThreads) % per_head % kChunks;
                *reinterpret_cast<uint4*>((chunk < kChunks / 2 ? p.k_cache : p.v_cache) + to[k]) = v[k];
            }
    }
}

}  // namespace flashllm
