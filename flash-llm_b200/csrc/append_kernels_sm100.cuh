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
__device__ __forceinline__ float2 four_bit_range(const float2 (&x)[4])
{
    float low = fminf(x[0].x, x[0].y), high = fmaxf(x[0].x, x[0].y), probe = fmaf(x[0].x, 0.0f, x[0].y * 0.0f);
#pragma unroll
    for (int k = 1; k < 4; ++k) {
        low   = fminf(low, fminf(x[k].x, x[k].y));
        high  = fmaxf(high, fmaxf(x[k].x, x[k].y));
        probe = fmaf(x[k].x, 0.0f, fmaf(x[k].y, 0.0f, probe));  // no number if one is none or infinite (which min and max may pass over)
    }
    const bool bad = probe != 0.0f || low < -65504.0f || high > 65504.0f;
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

__device__ __forceinline__ uint32_t four_bit_pack(const float2 (&x)[4], half2 scale)
{
    const float step = __low2float(scale), low = __high2float(scale);
    uint32_t    codes = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float code = fminf(fmaxf(rintf(__fdiv_rn((k % 2 ? x[k / 2].y : x[k / 2].x) - low, step)), 0.0f), 15.0f);
        codes |= (step > 0.0f ? static_cast<uint32_t>(code) : 0u) << (4 * k);
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

constexpr int kAppendRows = 16;  // of a CTA, at most

// rotary_append_kernel with norms: y = x w / sqrt(mean x^2 + eps) of each query and key head before it is turned, all in 32 bits, one
// rounding to what the cache holds.  A thread takes 32 bytes of a head (both members of its pairs), the threads of a head (8 or 4
// neighbours) add up its squares and find the smallest and the largest of its 64s by shuffles.
// Bound by memory for prompts, by a chain of dependent loads for a few tokens (sequence, page, row).  A CTA of many calls takes several
// tokens: their places and angles are found side by side, and the loads of the next 32 bytes are under way while these are worked on.
// 6612 tokens of 56 heads of 128: 47.4 us with a CTA for each, 43.6 so, 41.5 with eights of neighbouring threads side by side in
// memory (wavefronts of the L1 74 to 49 % of what it can), 37.7 in two even rounds, 36.0 to 36.8 in one (up to 16 tokens a CTA), all
// replayed from a graph: 5.2 TB/s, 0.79 of the measured copy bandwidth; a call among others 38.5, 0.75.  What
// is left is the work on registers, 260 operations for a thread's 16 elements.
template<int HEAD_DIM, bool INTERLEAVED, bool FOUR_BIT>
__global__ void __launch_bounds__(kRotaryThreads) norm_append_kernel(const __grid_constant__ AppendParams p)
{
    constexpr int        kUnits  = HEAD_DIM / 16;  // of 32 bytes per head
    constexpr int        kGroups = four_bit_groups(HEAD_DIM);
    // Cosines and sines, of four pairs at a time: first those of the units' first (in the interleaved layout, first half's), so that
    // neighbouring units' are neighbours (banks).
    __shared__ float4    s_cos[kAppendRows][2][kUnits], s_sin[kAppendRows][2][kUnits];
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

    // Where the unit's two eights of elements lie in its head, such that neighbouring threads' are neighbours: of query and key heads, and
    // of value heads.  Interleaved pairs lie within an eight; others are one of each, and what is not turned is split in two as well.
    const int  a_value = part * 8, z_value = HEAD_DIM / 2 + part * 8;
    const bool paired = part * 16 < r.rotary_dim;
    const int  a_turned = INTERLEAVED || paired ? a_value : r.rotary_dim + part * 8 - pairs;
    const int  z_turned = INTERLEAVED ? z_value : paired ? pairs + part * 8 : (HEAD_DIM + r.rotary_dim) / 2 + part * 8 - pairs;
    const bool turn_a = INTERLEAVED ? a_value < r.rotary_dim : paired, turn_z = INTERLEAVED ? z_value < r.rotary_dim : paired;
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
            va_next                 = *reinterpret_cast<const uint4*>(head + (value ? a_value : a_turned));
            vz_next                 = *reinterpret_cast<const uint4*>(head + (value ? z_value : z_turned));
        }
    };
    load_next();
    find_rows<kRotaryThreads>(c, n0, rows, s_at, s_position);
    for (int k = threadIdx.x; k < rows * pairs; k += kRotaryThreads) {
        const int    i = k / pairs, pair = k - i * pairs, position = r.positions ? r.positions[n0 + i] : s_position[i];
        const double turns = static_cast<double>(position) * (r.frequencies[pair] * 0.15915494309189535);
        float        sine, cosine;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
        const int half = INTERLEAVED ? pair / 4 / kUnits : pair / 4 % 2, unit = INTERLEAVED ? pair / 4 % kUnits : pair / 8;
        reinterpret_cast<float*>(&s_cos[i][half][unit])[pair % 4] = cosine * r.magnitude;
        reinterpret_cast<float*>(&s_sin[i][half][unit])[pair % 4] = sine * r.magnitude;
    }
    __syncthreads();

    auto reduce = [](float v, auto&& with) {  // over the threads of a head
#pragma unroll
        for (int d = 1; d < kUnits; d <<= 1)
            v = with(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    };
    auto unpack = [](const uint4& v, float2 (&x)[4]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x[k] = __half22float2(*reinterpret_cast<const half2*>(&w[k]));
    };
    auto pack = [](const float2 (&x)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const half2 h = __floats2half2_rn(x[k].x, x[k].y);
            w[k]          = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto      minus = [](float2 v) { return make_float2(-v.x, -v.y); };
    const int lane  = threadIdx.x & 31;
    for (int done = threadIdx.x - lane; done < all; done += kRotaryThreads) {  // whole warps, for the shuffles
        const bool  there = i_next < rows;
        const int   i = min(i_next, rows - 1), u = u_next;
        const uint4 va = va_next, vz = vz_next;
        u_next += kRotaryThreads;
        load_next();
        const int  head = u / kUnits;
        const bool query = head < r.heads, key = !query && head < r.heads + c.kv_heads, value = !query && !key;
        const int  a = value ? a_value : a_turned, z = value ? z_value : z_turned;
        float2     x[4], y[4];
        unpack(va, x);
        unpack(vz, y);
        const half* const weights = query ? p.q_norm : key ? p.k_norm : nullptr;
        if (p.q_norm || p.k_norm) {
            float2 squares = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                squares = ptx::fma_x2(x[k], x[k], ptx::fma_x2(y[k], y[k], squares));
            const float all_squares = reduce(squares.x + squares.y, [](float s, float t) { return s + t; });
            if (weights) {
                const float  factor = rsqrtf(fmaf(all_squares, 1.0f / HEAD_DIM, p.eps));
                const float2 both   = make_float2(factor, factor);
                float2       wa[4], wz[4];
                unpack(*reinterpret_cast<const uint4*>(weights + a), wa);
                unpack(*reinterpret_cast<const uint4*>(weights + z), wz);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = ptx::mul_x2(ptx::mul_x2(x[k], both), wa[k]);
                    y[k] = ptx::mul_x2(ptx::mul_x2(y[k], both), wz[k]);
                }
            }
        }
        if (turn_a && !value) {
            const float4 c0 = s_cos[i][0][part], c1 = s_cos[i][1][part], s0 = s_sin[i][0][part], s1 = s_sin[i][1][part];
            const float2 co[4] = {make_float2(c0.x, c0.y), make_float2(c0.z, c0.w), make_float2(c1.x, c1.y), make_float2(c1.z, c1.w)};
            const float2 si[4] = {make_float2(s0.x, s0.y), make_float2(s0.z, s0.w), make_float2(s1.x, s1.y), make_float2(s1.z, s1.w)};
            if constexpr (INTERLEAVED) {
                auto turn = [](float2 v, float cosine, float sine) {
                    return ptx::fma_x2(v, make_float2(cosine, cosine), ptx::mul_x2(make_float2(v.y, v.x), make_float2(-sine, sine)));
                };
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = turn(x[k], k % 2 ? co[k / 2].y : co[k / 2].x, k % 2 ? si[k / 2].y : si[k / 2].x);
                    if (turn_z)
                        y[k] = turn(y[k], k % 2 ? co[2 + k / 2].y : co[2 + k / 2].x, k % 2 ? si[2 + k / 2].y : si[2 + k / 2].x);
                }
            }
            else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 x0 = x[k], y0 = y[k];
                    x[k] = ptx::fma_x2(x0, co[k], ptx::mul_x2(y0, minus(si[k])));
                    y[k] = ptx::fma_x2(y0, co[k], ptx::mul_x2(x0, si[k]));
                }
            }
        }
        const int       h  = head - r.heads - (key ? 0 : c.kv_heads);  // key/value head
        const long long at = s_at[i];
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
        *reinterpret_cast<uint4*>(dst + a) = lost ? zero : pack(x);
        *reinterpret_cast<uint4*>(dst + z) = lost ? zero : pack(y);
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
// of it what is written): 130000 rows of 8 heads of 128 122 us, 5.6 TB/s, 0.85 of the measured copy bandwidth (157 with addresses
// worked out for every eight elements).
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
    // A thread has one row's eight elements of every head, or, where rows are few, of every so many heads.
    const int       word = threadIdx.x % kWords, i = (threadIdx.x >> kWordShift) & ((1 << p.row_shift) - 1);
    const long long at = i < rows ? s_at[i] : kNobodysRow;
    if (at == kNobodysRow)
        return;
    const int            h0 = threadIdx.x >> (kWordShift + p.row_shift), step = kReadThreads >> (kWordShift + p.row_shift);
    const long long      page_bytes = static_cast<long long>(four_bit_row_bytes(HEAD_DIM)) << c.page_shift;  // of a head
    const long long      codes_at = at >= 0 ? four_bit_codes<HEAD_DIM>(c, at) + h0 * page_bytes + 4 * word : 0;
    const long long      scales_at = at >= 0 ? four_bit_scales<HEAD_DIM>(c, at) + h0 * page_bytes + word / 8 * 4 : 0;
    const unsigned char *k_codes = p.cache[0] + codes_at, *v_codes = p.cache[1] + codes_at;
    const unsigned char *k_scale = p.cache[0] + scales_at, *v_scale = p.cache[1] + scales_at;
    const long long      to = (static_cast<long long>(n0 + i) * c.kv_heads + h0) * HEAD_DIM + 8 * word;
    half *               k_out = p.out[0] + to, *v_out = p.out[1] + to;
#pragma unroll 4
    for (int h = h0; h < c.kv_heads; h += step) {
        uint32_t k = 0, v = 0;
        half2    ks = __float2half2_rn(0.0f), vs = ks;
        if (at >= 0) {
            k  = *reinterpret_cast<const uint32_t*>(k_codes);
            v  = *reinterpret_cast<const uint32_t*>(v_codes);
            ks = *reinterpret_cast<const half2*>(k_scale);
            vs = *reinterpret_cast<const half2*>(v_scale);
        }
        *reinterpret_cast<uint4*>(k_out) = four_bit_values<true>(k, ks);
        *reinterpret_cast<uint4*>(v_out) = four_bit_values<true>(v, vs);
        k_codes += step * page_bytes, v_codes += step * page_bytes, k_scale += step * page_bytes, v_scale += step * page_bytes;
        k_out += step * HEAD_DIM, v_out += step * HEAD_DIM;
    }
}

}  // namespace flashllm
