// A paged key/value cache of 4 bits: as cache_batch.cuh has it, but what one head keeps of one page, page_size x head_dim x 9 / 16
// bytes in one piece, are codes and what they stand for:
//
//   codes   [page_size][head_dim / 2] bytes, two to a byte, the even element in the low bits
//   scales  [page_size][head_dim / 64][2] fp16: step and lowest value of 64 elements
//
//   element = lowest + step x code
//
// lowest = fp16(min), step = fp16((max - lowest) / 15), code = (x - lowest) / step to the nearest, all from 32 bits: what a turned key is
// off there, some 2^-22 of it, makes the neighbouring code of some two in a million, no further from the element but a step from what
// 64 bits would have kept.  64 elements and
// not all 128 of a head: steps are 0.9 of what they would be for normally distributed elements, much less where few channels are
// large, for 0.25 bits an element.  A group that holds a value which is not finite, or beyond fp16's range, has a step of NaN, and so
// have its elements.
#pragma once
#include <math_constants.h>

#include "cache_batch.cuh"

namespace flashllm {

constexpr int kFourBitGroup = 64;

__host__ __device__ constexpr int four_bit_row_bytes(int head_dim)
{
    return head_dim * 9 / 16;
}

__host__ __device__ constexpr int four_bit_groups(int head_dim)
{
    return head_dim / kFourBitGroup;
}

// Where a row that cache_row names has its codes and its scales.
template<int HEAD_DIM>
__device__ __forceinline__ long long four_bit_codes(const CacheBatch& c, long long row)
{
    const long long in = row & ((1 << c.page_shift) - 1);
    return (row - in) * four_bit_row_bytes(HEAD_DIM) + in * (HEAD_DIM / 2);
}

template<int HEAD_DIM>
__device__ __forceinline__ long long four_bit_scales(const CacheBatch& c, long long row)
{
    const long long in = row & ((1 << c.page_shift) - 1);
    return (row - in) * four_bit_row_bytes(HEAD_DIM) + (static_cast<long long>(HEAD_DIM / 2) << c.page_shift)
           + in * (4 * four_bit_groups(HEAD_DIM));
}

// Eight elements, one rounding to fp16 each: product and sum are one operation, a code is exact (four bits put into the mantissa of 1024
// or, where they lie, of 64 are so much more).  BOUNDED: lowest value and step, rounded, can take the last codes past the largest
// number of fp16, which then is the element (unless the lowest value is infinite, which no append writes).
template<bool BOUNDED>
__device__ __forceinline__ uint4 four_bit_values(uint32_t codes, half2 scale)
{
    const half2    step = __low2half2(scale), low = __high2half2(scale);
    const half2    largest = __float2half2_rn(__hisinf(__high2half(scale)) ? CUDART_INF_F : 65504.0f);
    const uint32_t codes8 = codes >> 8;
    uint32_t       v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // elements i and i + 4
        const uint32_t w   = i < 2 ? codes : codes8;
        const uint32_t two = i % 2 == 0 ? (w & 0x000f000fu) | 0x64006400u : (w & 0x00f000f0u) | 0x54005400u;
        half2          h   = __hfma2(__hsub2(*reinterpret_cast<const half2*>(&two), __float2half2_rn(i % 2 == 0 ? 1024.0f : 64.0f)), step, low);
        if constexpr (BOUNDED)
            h = __hmin2_nan(h, largest);
        v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                      __byte_perm(v[2], v[3], 0x7632));
}

}  // namespace flashllm
