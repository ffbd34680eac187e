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
    int          rows;  // of a CTA, 1 .. kAppendRows
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

// Where `count` rows of the batch from row n0 on lie, for all threads of a CTA: at[i] is the cache row (cache_row) of key/value head
// 0, kLostRow for one whose sequence does not fit or whose page is none, kNobodysRow; position[i] the row's place in its sequence (-1
// where it does not fit).  Every sequence is looked at by one thread; a barrier ends it.
constexpr long long kLostRow = -1, kNobodysRow = -2;

template<int THREADS>
__device__ __forceinline__ void find_rows(const CacheBatch& c, int n0, int count, long long* at, int* position)
{
    for (int i = threadIdx.x; i < count; i += THREADS) {
        at[i]       = kNobodysRow;
        position[i] = -1;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < c.sequences; b += THREADS) {
        const int begin = max(c.cu_tokens[b], 0), end = min(c.cu_tokens[b + 1], c.tokens), context = c.context[b];
        if (begin >= n0 + count || end <= n0 || end <= begin)
            continue;
        // A sequence that does not fit is left out whole, as load_sequence has it.
        const bool fits = context >= 0 && static_cast<long long>(context) + (end - begin) <= table_positions(c);
        if (!fits)
            atomicOr(c.status, kStatusBadCache);
        for (int n = max(begin, n0); n < min(end, n0 + count); ++n) {
            position[n - n0] = fits ? context + (n - begin) : -1;
            at[n - n0]       = fits ? b : kLostRow;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += THREADS)
        if (at[i] >= 0)
            at[i] = cache_row(c, static_cast<int>(at[i]), position[i], 0);
    __syncthreads();
}

constexpr int kAppendRows = 8;  // of a CTA, at most

// rotary_append_kernel with norms: y = x w / sqrt(mean x^2 + eps) of each query and key head before it is turned, all in 32 bits, one
// rounding to what the cache holds.  A thread takes 32 bytes of a head (both members of its pairs), the threads of a head (8 or 4
// neighbours) add up its squares and find the smallest and the largest of its 64s by shuffles.
// Bound by memory for prompts, by a chain of dependent loads for a few tokens (sequence, page, row).  A CTA of many calls takes several
// tokens: their places and angles are found side by side, and the loads of the next 32 bytes are under way while these are worked on
// (APPENDNOTE).
template<int HEAD_DIM, bool INTERLEAVED, bool FOUR_BIT>
__global__ void __launch_bounds__(kRotaryThreads) norm_append_kernel(const __grid_constant__ AppendParams p)
{
    constexpr int        kUnits  = HEAD_DIM / 16;  // of 32 bytes per head
    constexpr int        kGroups = four_bit_groups(HEAD_DIM);
    __shared__ float2    s_turn[kAppendRows][HEAD_DIM / 2];  // cosine and sine
    __shared__ long long s_at[kAppendRows];
    __shared__ int       s_position[kAppendRows];
    const RotaryParams&  r     = p.rotary;
    const CacheBatch&    c     = r.batch;
    const int            n0    = blockIdx.x * p.rows, rows = min(p.rows, c.tokens - n0);
    const int            pairs = r.rotary_dim / 2;
    const int            units = (r.heads + 2 * c.kv_heads) * kUnits, all = rows * units;
    const int            part  = threadIdx.x % kUnits;  // of every head that the thread takes
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    // Where a unit's two halves lie in its head: of query and key heads, and of value heads.
    const bool turned   = part * 16 < r.rotary_dim;
    const int  a_turned = turned && !INTERLEAVED ? part * 8 : part * 16, z_turned = turned && !INTERLEAVED ? pairs + part * 8 : part * 16 + 8;
    // The thread's next unit: row of the CTA, unit of the row.
    int   i_next = 0, u_next = threadIdx.x;
    uint4 va_next{}, vz_next{};
    auto  load_next = [&]() {
        while (u_next >= units) {
            u_next -= units;
            ++i_next;
        }
        if (i_next < rows) {
            const bool        value = u_next / kUnits >= r.heads + c.kv_heads;
            const half* const head  = r.qkv + (n0 + i_next) * r.ld_qkv + u_next / kUnits * HEAD_DIM;
            va_next                 = *reinterpret_cast<const uint4*>(head + (value ? part * 16 : a_turned));
            vz_next                 = *reinterpret_cast<const uint4*>(head + (value ? part * 16 + 8 : z_turned));
        }
    };
    load_next();
    find_rows<kRotaryThreads>(c, n0, rows, s_at, s_position);
    for (int k = threadIdx.x; k < rows * pairs; k += kRotaryThreads) {
        const int    i = k / pairs, pair = k - i * pairs, position = r.positions ? r.positions[n0 + i] : s_position[i];
        const double turns = static_cast<double>(position) * (r.frequencies[pair] * 0.15915494309189535);
        float        sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        s_turn[i][pair] = make_float2(cosine * r.magnitude, sine * r.magnitude);
    }
    __syncthreads();

    auto reduce = [](float v, auto&& with) {  // over the threads of a head
#pragma unroll
        for (int d = 1; d < kUnits; d <<= 1)
            v = with(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    };
    const int lane = threadIdx.x & 31;
    for (int done = threadIdx.x - lane; done < all; done += kRotaryThreads) {  // whole warps, for the shuffles
        const bool  there = i_next < rows;
        const int   i = min(i_next, rows - 1), u = u_next;
        const uint4 va = va_next, vz = vz_next;
        u_next += kRotaryThreads;
        load_next();
        const long long at = s_at[i];
        const int       head = u / kUnits;
        const bool      query = head < r.heads, key = !query && head < r.heads + c.kv_heads, value = !query && !key;
        const int       a = value ? part * 16 : a_turned, z = value ? part * 16 + 8 : z_turned;
        float           x[8], y[8];
        unpack_half8(va, x);
        unpack_half8(vz, y);
        const half* const weights = query ? p.q_norm : key ? p.k_norm : nullptr;
        if (p.q_norm || p.k_norm) {
            float squares = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                squares = fmaf(x[k], x[k], fmaf(y[k], y[k], squares));
            squares = reduce(squares, [](float s, float t) { return s + t; });
            if (weights) {
                const float factor = 1.0f / sqrtf(fmaf(squares, 1.0f / HEAD_DIM, p.eps));
                float       wa[8], wz[8];
                unpack_half8(*reinterpret_cast<const uint4*>(weights + a), wa);
                unpack_half8(*reinterpret_cast<const uint4*>(weights + z), wz);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] = x[k] * factor * wa[k];
                    y[k] = y[k] * factor * wz[k];
                }
            }
        }
        if (turned && !value) {
            const float4* const turn = reinterpret_cast<const float4*>(&s_turn[i][part * 8]);  // of two pairs
            float               co[8], si[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 two = turn[k];
                co[2 * k] = two.x, si[2 * k] = two.y, co[2 * k + 1] = two.z, si[2 * k + 1] = two.w;
            }
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x0 = x[2 * k], x1 = x[2 * k + 1], y0 = y[2 * k], y1 = y[2 * k + 1];
                    x[2 * k]     = x0 * co[k] - x1 * si[k];
                    x[2 * k + 1] = x1 * co[k] + x0 * si[k];
                    y[2 * k]     = y0 * co[k + 4] - y1 * si[k + 4];
                    y[2 * k + 1] = y1 * co[k + 4] + y0 * si[k + 4];
                }
            }
            else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float x0 = x[k], y0 = y[k];
                    x[k] = x0 * co[k] - y0 * si[k];
                    y[k] = y0 * co[k] + x0 * si[k];
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
                    const bool  ina = a / kFourBitGroup == g, inz = z / kFourBitGroup == g;
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
        if (!there || at == kNobodysRow || (!query && at < 0))
            continue;
        half* const dst = query ? r.q + (n0 + i) * r.ld_q + static_cast<long long>(head) * HEAD_DIM
                                : (key ? r.k_cache : r.v_cache) + (at + (static_cast<long long>(h) << c.page_shift)) * HEAD_DIM;
        const bool  lost = s_position[i] < 0;  // queries of a sequence that does not fit
        const uint4 zero = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + a) = lost ? zero : pack_half8(x);
        *reinterpret_cast<uint4*>(dst + z) = lost ? zero : pack_half8(y);
    }
}

struct ReadParams {
    CacheBatch           batch;
    const unsigned char* cache[2];  // keys, values
    half*                out[2];    // [tokens][kv_heads * head_dim]
    int                  row_shift;  // a CTA takes 2^row_shift rows, kReadRows at most
};

constexpr int kReadThreads = 256, kReadRows = 16;

// Rows of the batch from a cache of 4 bits.  A CTA takes a few rows: for each its place is looked up once, then threads take eight
// elements at a time, the rows of one head, which lie one behind another in a page, before the next head's.  Bound by memory (most
// of it what is written): READNOTE.
template<int HEAD_DIM>
__global__ void __launch_bounds__(kReadThreads) four_bit_read_kernel(const __grid_constant__ ReadParams p)
{
    constexpr int        kWordShift = HEAD_DIM == 128 ? 4 : 3, kWords = 1 << kWordShift;
    __shared__ long long s_at[kReadRows];
    __shared__ int       s_position[kReadRows];
    const CacheBatch&    c  = p.batch;
    const int            n0 = blockIdx.x << p.row_shift, rows = min(1 << p.row_shift, c.tokens - n0);
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    find_rows<kReadThreads>(c, n0, rows, s_at, s_position);
    const int units = 2 * c.kv_heads << (p.row_shift + kWordShift), word = threadIdx.x % kWords;
    const long long width = static_cast<long long>(c.kv_heads) * HEAD_DIM;
#pragma unroll 4
    for (int u = threadIdx.x; u < units; u += kReadThreads) {
        const int i = (u >> kWordShift) & ((1 << p.row_shift) - 1), which = u >> (p.row_shift + kWordShift), h = which >> 1;
        if (i >= rows)
            continue;
        const long long at = s_at[i];
        if (at == kNobodysRow)
            continue;
        const unsigned char* const cache = which & 1 ? p.cache[1] : p.cache[0];
        half* const                out   = which & 1 ? p.out[1] : p.out[0];
        uint4                      v     = make_uint4(0, 0, 0, 0);
        if (at >= 0) {
            const long long row   = at + (static_cast<long long>(h) << c.page_shift);
            const uint32_t  codes = *reinterpret_cast<const uint32_t*>(cache + four_bit_codes<HEAD_DIM>(c, row) + 4 * word);
            const half2     scale = *reinterpret_cast<const half2*>(cache + four_bit_scales<HEAD_DIM>(c, row) + word / 8 * 4);
            v                     = four_bit_values<true>(codes, scale);
        }
        *reinterpret_cast<uint4*>(out + (n0 + i) * width + h * HEAD_DIM + 8 * word) = v;
    }
}

}  // namespace flashllm
