// Kernels that write and read the paged cache with more than a copy: norms of queries and keys with the rotary append, into a cache
// of fp16 or of 4 bits, and rows of a cache of 4 bits as fp16.
#pragma once
#include <math_constants.h>

#include "cache_kernels_sm100.cuh"
#include "four_bit_cache.cuh"

namespace flashllm {

struct AppendParams {
    RotaryParams rotary;  // its caches are bytes where they hold 4 bits
    const half*  q_norm;  // [head_dim] weights of the queries' and the keys' norm, or nullptr: none
    const half*  k_norm;
    float        eps;
};

// What eight elements add to the smallest and the largest of their 64; minus infinity if one of them fp16 does not hold.
__device__ __forceinline__ float2 four_bit_range(const float (&x)[8])
{
    float low = x[0], high = x[0], size = fabsf(x[0]);
    bool  bad = !(size <= 65504.0f);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        low  = fminf(low, x[i]);
        high = fmaxf(high, x[i]);
        bad  = bad || !(fabsf(x[i]) <= 65504.0f);
    }
    return make_float2(bad ? -CUDART_INF_F : low, high);
}

// Step and lowest value of 64 elements.
__device__ __forceinline__ half2 four_bit_scale(float2 range)
{
    const half low  = __float2half_rn(range.x);
    const half step = __float2half_rn(__fdiv_rn(range.y - __half2float(low), 15.0f));
    if (range.x == -CUDART_INF_F)
        return __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0));
    return __halves2half2(step, low);
}

__device__ __forceinline__ uint32_t four_bit_pack(const float (&x)[8], half2 scale)
{
    const float step = __low2float(scale), low = __high2float(scale);
    uint32_t    codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float code = fminf(fmaxf(rintf(__fdiv_rn(x[i] - low, step)), 0.0f), 15.0f);
        codes |= (step > 0.0f ? static_cast<uint32_t>(code) : 0u) << (4 * i);
    }
    return codes;
}

// rotary_append_kernel with norms: y = x w / sqrt(mean x^2 + eps) of each query and key head before it is turned, all in 32 bits, one
// rounding to what the cache holds.  One CTA per token, a thread takes 32 bytes of a head (both members of its pairs), the threads of
// a head (8 or 4 neighbours) add up its squares and find the smallest and the largest of its 64s by shuffles.
// Bound by memory for prompts, by a chain of dependent loads for a few tokens (sequence, page, row).
template<int HEAD_DIM, bool INTERLEAVED, bool FOUR_BIT>
__global__ void __launch_bounds__(kRotaryThreads) norm_append_kernel(const __grid_constant__ AppendParams p)
{
    constexpr int       kUnits  = HEAD_DIM / 16;  // of 32 bytes per head
    constexpr int       kGroups = four_bit_groups(HEAD_DIM);
    __shared__ float    s_cos[HEAD_DIM / 2], s_sin[HEAD_DIM / 2];
    __shared__ int      s_sequence, s_position;  // of the token; -1: nobody's, or it does not fit
    const RotaryParams& r     = p.rotary;
    const CacheBatch&   c     = r.batch;
    const int           n     = blockIdx.x;
    const int           pairs = r.rotary_dim / 2;
    const int           units = (r.heads + 2 * c.kv_heads) * kUnits;
    const half* const   row   = r.qkv + n * r.ld_qkv;
    const int           part  = threadIdx.x % kUnits;  // of every head that the thread takes
    if (threadIdx.x == 0)
        s_sequence = -1;
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    uint4 va{}, vz{};
    // Where a unit's two halves lie in its head: of query and key heads, and of value heads.
    const bool turned = part * 16 < r.rotary_dim;
    const int  a_turned = turned && !INTERLEAVED ? part * 8 : part * 16, z_turned = turned && !INTERLEAVED ? pairs + part * 8 : part * 16 + 8;
    auto       load = [&](int u) {
        const bool value = u / kUnits >= r.heads + c.kv_heads;
        const half* head = row + u / kUnits * HEAD_DIM;
        va               = *reinterpret_cast<const uint4*>(head + (value ? part * 16 : a_turned));
        vz               = *reinterpret_cast<const uint4*>(head + (value ? part * 16 + 8 : z_turned));
    };
    if (static_cast<int>(threadIdx.x) < units)
        load(threadIdx.x);
    const double frequency = threadIdx.x < pairs ? r.frequencies[threadIdx.x] : 0.0;
    const int    elsewhere = r.positions && threadIdx.x < pairs ? r.positions[n] : 0;
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
        const double turns = static_cast<double>(r.positions ? elsewhere : position) * (frequency * 0.15915494309189535);
        float        sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        s_cos[threadIdx.x] = cosine * r.magnitude;
        s_sin[threadIdx.x] = sine * r.magnitude;
    }
    __syncthreads();

    auto reduce = [](float v, auto&& with) {  // over the threads of a head
#pragma unroll
        for (int d = 1; d < kUnits; d <<= 1)
            v = with(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    };
    const int lane = threadIdx.x & 31;
    for (int u = threadIdx.x; u - lane < units; u += kRotaryThreads) {  // whole warps, for the shuffles
        const bool there = u < units;
        if (there && u != static_cast<int>(threadIdx.x))
            load(u);
        const int  head = u / kUnits;
        const bool query = head < r.heads, key = !query && head < r.heads + c.kv_heads, value = !query && !key;
        const int  a = value ? part * 16 : a_turned, z = value ? part * 16 + 8 : z_turned;
        float      x[8], y[8];
        unpack_half8(va, x);
        unpack_half8(vz, y);
        const half* const weights = query ? p.q_norm : key ? p.k_norm : nullptr;
        if (p.q_norm || p.k_norm) {
            float squares = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                squares = fmaf(x[i], x[i], fmaf(y[i], y[i], squares));
            squares = reduce(squares, [](float s, float t) { return s + t; });
            if (weights) {
                const float factor = 1.0f / sqrtf(fmaf(squares, 1.0f / HEAD_DIM, p.eps));
                float       wa[8], wz[8];
                unpack_half8(*reinterpret_cast<const uint4*>(weights + a), wa);
                unpack_half8(*reinterpret_cast<const uint4*>(weights + z), wz);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = x[i] * factor * wa[i];
                    y[i] = y[i] * factor * wz[i];
                }
            }
        }
        if (turned && !value) {
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
        }
        const int h = head - r.heads - (key ? 0 : c.kv_heads);  // key/value head
        if constexpr (FOUR_BIT) {
            if (__any_sync(0xffffffffu, !query)) {
                const float2 ra = four_bit_range(x), rz = four_bit_range(y);
                half2        scale[kGroups];
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    const bool ina = a / kFourBitGroup == g, inz = z / kFourBitGroup == g;
                    const float low  = reduce(fminf(ina ? ra.x : CUDART_INF_F, inz ? rz.x : CUDART_INF_F), [](float s, float t) { return fminf(s, t); });
                    const float high = reduce(fmaxf(ina ? ra.y : -CUDART_INF_F, inz ? rz.y : -CUDART_INF_F), [](float s, float t) { return fmaxf(s, t); });
                    scale[g]         = four_bit_scale(make_float2(low, high));
                }
                if (!query && there && at >= 0) {
                    unsigned char* const cache = reinterpret_cast<unsigned char*>(key ? r.k_cache : r.v_cache);
                    const long long      at_h  = at + (static_cast<long long>(h) << c.page_shift);
                    uint32_t* const      codes = reinterpret_cast<uint32_t*>(cache + four_bit_codes<HEAD_DIM>(c, at_h));
                    codes[a / 8]               = four_bit_pack(x, a < kFourBitGroup ? scale[0] : scale[kGroups - 1]);
                    codes[z / 8]               = four_bit_pack(y, z < kFourBitGroup ? scale[0] : scale[kGroups - 1]);
                    if (part < kGroups)
                        *reinterpret_cast<half2*>(cache + four_bit_scales<HEAD_DIM>(c, at_h) + 4 * part) = part == 0 ? scale[0] : scale[kGroups - 1];
                }
            }
            if (!query)
                continue;
        }
        if (!there || (!query && at < 0))
            continue;
        half* const dst = query ? r.q + n * r.ld_q + static_cast<long long>(head) * HEAD_DIM
                                : (key ? r.k_cache : r.v_cache) + (at + (static_cast<long long>(h) << c.page_shift)) * HEAD_DIM;
        const uint4 zero = make_uint4(0, 0, 0, 0);  // queries of a sequence that does not fit
        *reinterpret_cast<uint4*>(dst + a) = position < 0 ? zero : pack_half8(x);
        *reinterpret_cast<uint4*>(dst + z) = position < 0 ? zero : pack_half8(y);
    }
}

struct ReadParams {
    CacheBatch           batch;
    const unsigned char* cache[2];  // keys, values
    half*                out[2];    // [tokens][kv_heads * head_dim]
    int                  rows;      // of a CTA, kReadRows at most
};

constexpr int kReadThreads = 256, kReadRows = 16;

// Rows of the batch from a cache of 4 bits.  A CTA takes a few rows: for each its place is looked up once, then threads take eight
// elements at a time, the rows of one head, which lie one behind another in a page, before the next head's.  Bound by memory (most
// of it what is written).
template<int HEAD_DIM>
__global__ void __launch_bounds__(kReadThreads) four_bit_read_kernel(const __grid_constant__ ReadParams p)
{
    constexpr int        kWords = HEAD_DIM / 8;
    __shared__ long long s_row[kReadRows];  // of key/value head 0; -1: zeros, -2: nobody's
    const CacheBatch&    c  = p.batch;
    const int            n0 = blockIdx.x * p.rows;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = warp; i < p.rows; i += kReadThreads / 32) {  // a warp looks for a row's sequence, 32 at a time
        const int n = n0 + i;
        long long at = -2;
        for (int b0 = 0; n < c.tokens && b0 < c.sequences; b0 += 32) {
            const int      b     = b0 + lane;
            const int      begin = b < c.sequences ? max(c.cu_tokens[b], 0) : 0, end = b < c.sequences ? min(c.cu_tokens[b + 1], c.tokens) : 0;
            const unsigned found = __ballot_sync(0xffffffffu, begin <= n && n < end);
            if (!found)
                continue;
            if (lane == __ffs(found) - 1) {
                const int  context = c.context[b];
                const bool fits    = context >= 0 && static_cast<long long>(context) + (end - begin) <= table_positions(c);
                if (!fits)
                    atomicOr(c.status, kStatusBadCache);
                at = fits ? cache_row(c, b, context + (n - begin), 0) : -1;
                s_row[i] = at;
            }
            at = 0;
            break;
        }
        if (at == -2 && lane == 0)
            s_row[i] = -2;
    }
    __syncthreads();
    const int per_head = p.rows * kWords, units = 2 * c.kv_heads * per_head;
#pragma unroll 4
    for (int u = threadIdx.x; u < units; u += kReadThreads) {
        const int       which = u / per_head, i = u % per_head / kWords, word = u % kWords;
        const int       h = which >> 1, kind = which & 1;
        const long long at = s_row[i];
        if (at == -2)
            continue;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (at >= 0) {
            const long long row   = at + (static_cast<long long>(h) << c.page_shift);
            const uint32_t  codes = *reinterpret_cast<const uint32_t*>(p.cache[kind] + four_bit_codes<HEAD_DIM>(c, row) + 4 * word);
            const half2     scale = *reinterpret_cast<const half2*>(p.cache[kind] + four_bit_scales<HEAD_DIM>(c, row) + word / 8 * 4);
            v                     = four_bit_values<true>(codes, scale);
        }
        *reinterpret_cast<uint4*>(p.out[kind] + (static_cast<long long>(n0 + i) * c.kv_heads + h) * HEAD_DIM + 8 * word) = v;
    }
}

}  // namespace flashllm
