// Attention of single tokens through a window over a paged cache of fp16: the warps' kernel of attention_four_bit_sm100.cuh (its division
// of the work, its products with queries as the eight columns, its parts and their joining) with keys and values as they lie.
//
// A window is a few tiles of keys, and for a few of them the attention of many rows spends as long on beginning and ending as on its
// bytes (decoding of 64 sequences, window 1024: 70 us, here 40; 16 sequences, window 4096: 60 and 48).  A tile of rows is of one token, so all of it sees the same keys:
// what it does not see is not copied but left zero, and no product meets it.
//
// An infinite value times a weight of zero (too small for fp16) is no number: a piece that ends with one, though its weights have a
// sum, looks through its values again and writes what the definition gives, infinity for any weight.
#pragma once
#include "attention_four_bit_sm100.cuh"

namespace flashllm {

constexpr int kSingleWarps = 10;

__host__ __device__ constexpr int single_stage_bytes(int head_dim)
{
    return 2 * kFourKeys * head_dim * 2;
}

__host__ __device__ constexpr int single_stages(int head_dim)
{
    return 2 * 128 / head_dim;
}

__host__ __device__ constexpr int single_smem_bytes(int head_dim)
{
    return kSingleWarps * (single_stages(head_dim) * single_stage_bytes(head_dim) + four_rows_bytes(head_dim, 1))
           + static_cast<int>(sizeof(FourShared)) + 128;
}

// Four transposed 8 x 8 matrices: a lane's address is that of a row of one of them.
__device__ __forceinline__ void single_load_transposed(uint32_t at, uint32_t (&a)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
}

// Sums that are no numbers though their row's weights have a sum: infinities of the values that the rows see, whatever their weights
// are.  For a whole warp; `sums` are its rows' outputs, `seen(key)` tells which keys they see.
template<int HEAD_DIM, typename Seen, typename KeyOf>
__device__ __noinline__ void single_restore(const FourBitParams& p, int b, int head, int begin, int end, int rows, float* sums, const float2* stats, KeyOf key_of, Seen seen)
{
    const half* const cache = reinterpret_cast<const half*>(p.v_cache);
    const int         lane  = threadIdx.x & 31;
    for (int column = lane; column < HEAD_DIM; column += 32) {
        bool plus = false, minus = false;
        for (int block = begin; block < end; ++block)
            for (int k = 0; k < kFourKeys; ++k) {
                const int key = key_of(block) + k;
                if (!seen(key))
                    continue;
                const long long at = cache_row(p.batch, b, key, head);
                if (at < 0)
                    continue;
                const uint32_t h = __half_as_ushort(cache[at * HEAD_DIM + column]);
                if (!half_not_finite(h))
                    continue;
                const bool nan = (h & 0x3ffu) != 0u;
                plus           = plus || nan || h < 0x8000u;
                minus          = minus || nan || h >= 0x8000u;
            }
        for (int row = 0; row < rows; ++row) {
            float& o = sums[row * HEAD_DIM + column];
            if (o != o && stats[row].y == stats[row].y && (plus || minus))
                o = (plus ? CUDART_INF_F : 0.0f) + (minus ? -CUDART_INF_F : 0.0f);
        }
    }
}

// PLAIN: neither cap nor slopes.
template<int HEAD_DIM, bool PLAIN>
__global__ void __launch_bounds__(kSingleWarps * 32, 1) window_single_kernel(const __grid_constant__ FourBitParams p)
{
    constexpr int kRows = 8, kKeys = kFourKeys, kStages = single_stages(HEAD_DIM), kStageBytes = single_stage_bytes(HEAD_DIM);
    constexpr int kRowBytes = HEAD_DIM * 2, kTileBytes = kKeys * kRowBytes, kChunks = kRowBytes / 16, kChunkShift = HEAD_DIM == 128 ? 4 : 3;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t       raw  = ptx::smem_u32(smem_raw);
    const uint32_t       base = (raw + 127u) & ~127u;
    unsigned char* const smem = smem_raw + (base - raw);
    const int            warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const CacheBatch&    c    = p.batch;
    const uint32_t       ring = base + warp * (kStages * kStageBytes);
    unsigned char* const ring_ptr   = smem + warp * (kStages * kStageBytes);
    unsigned char* const first_sums = smem + kSingleWarps * (kStages * kStageBytes);
    FourShared&          sh = *reinterpret_cast<FourShared*>(first_sums + kSingleWarps * four_rows_bytes(HEAD_DIM, 1));

    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    unsigned long long u0, u1;
    if (!four_plan<HEAD_DIM, kRows, kKeys, kSingleWarps, true>(p, sh, u0, u1))
        return;

    // A lane copies 16 bytes of every second key (of every fourth where they are 128 bytes): where from, and where to in the ring.  Chunks
    // change places within a row, for the banks: those of keys by the key's lowest bit (four at a time, which a load of two keys
    // takes), those of values by its lowest three (a transposed load takes one of eight keys).
    constexpr int kStep = 32 / kChunks;  // keys of a copy
    const int     row_of_lane = lane >> kChunkShift, chunk_of_lane = lane & (kChunks - 1);
    const unsigned long long page_bytes = static_cast<unsigned long long>(kRowBytes) << c.page_shift;
    const unsigned char* const from_k = p.k_cache + 16 * lane;
    const unsigned char* const from_v = p.v_cache + 16 * lane;
    auto place_k = [](int row, int chunk) { return row * kRowBytes + 16 * (chunk ^ (row & 1) * 4); };
    auto place_v = [](int row, int chunk) { return row * kRowBytes + 16 * (chunk ^ (row & 7)); };

    if (u0 < u1) {
        FourWalk<kRows, kKeys, kSingleWarps, true> walk;
        walk.start(p, sh, u0, u1);
        do {
            walk.piece(p);
            const FourSequence& q     = walk.q;
            const FourTile      sight = walk.sight;
            const int b = walk.b, head = walk.head, row0 = walk.row0, rows = walk.rows, token = walk.token0, begin = walk.begin, end = walk.end;
            if (begin < end) {
                const int  place = q.context + token, low = place - p.window + 1;  // the rows' position; the first key of their window
                auto       sees   = [&](int key) { return key <= place && (key >= low || key < p.sinks); };
                auto       key_of = [&](int block) { return (block + (block < sight.skip_from ? 0 : sight.skip)) * kKeys; };
                auto       partly = [&](int key0) { return key0 + kKeys > place + 1 || (key0 < low && key0 + kKeys > p.sinks); };
                // Queries as the products' columns: 16 bytes of a key are elements of two products.
                uint32_t    qf[HEAD_DIM / 16][2];
                const half* q_row = p.q + (q.first + token) * p.ld_q + static_cast<long long>(head * p.share + row0 - token * p.share + g) * HEAD_DIM;
#pragma unroll
                for (int m = 0; m < HEAD_DIM / 32; ++m) {
                    const uint4 x = g < rows ? *reinterpret_cast<const uint4*>(q_row + 32 * m + 8 * t) : make_uint4(0, 0, 0, 0);
                    qf[2 * m][0] = x.x, qf[2 * m][1] = x.y, qf[2 * m + 1][0] = x.z, qf[2 * m + 1][1] = x.w;
                }
                const int* const table = c.page_table + static_cast<long long>(b) * c.table_width;
                auto ids_from = [&](int block) {  // pages of 32 blocks, a lane each; -1: reads as zeros
                    block += lane;
                    if (block >= end)
                        return -1;
                    const int id = table[key_of(block) >> c.page_shift];
                    if (static_cast<unsigned>(id) < static_cast<unsigned>(c.pages))
                        return id;
                    atomicOr(c.status, kStatusBadCache);
                    return -1;
                };
                int      ids = ids_from(begin), ids_next = ids_from(begin + 32);
                uint32_t copied = 0, at_hand = 0;
                auto copy = [&](int i) {  // the i-th block of the piece, to the next place of the ring
                    if (begin + i < end) {
                        if (i > 0 && i % 32 == 0) {
                            ids      = ids_next;
                            ids_next = ids_from(begin + i + 32);
                        }
                        const int          id = __shfl_sync(0xffffffffu, ids, i % 32), key0 = key_of(begin + i);
                        const unsigned long long at = static_cast<unsigned>(max(id, 0) * c.kv_heads + head) * page_bytes
                                                      + static_cast<unsigned>(key0 & ((1 << c.page_shift) - 1)) * static_cast<unsigned long long>(kRowBytes);
                        const bool some = partly(key0);
#pragma unroll
                        for (int k = 0; k < kKeys / kStep; ++k) {
                            const int  row   = row_of_lane + kStep * k;
                            const bool there = id >= 0 && (!some || sees(key0 + row));
                            four_copy16(ring + copied + place_k(row, chunk_of_lane), from_k + at + 512 * k, there);
                            four_copy16(ring + copied + kTileBytes + place_v(row, chunk_of_lane), from_v + at + 512 * k, there);
                        }
                        copied = copied == (kStages - 1) * kStageBytes ? 0 : copied + kStageBytes;
                    }
                    four_copies_done();
                };
                float slope[2] = {0.0f, 0.0f};
                if (!PLAIN && p.slopes)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        slope[e] = 2 * t + e < rows ? p.slopes[head * p.share + row0 - token * p.share + 2 * t + e] * CUDART_L2E_F : 0.0f;
                // PLAIN: maxima are of products, `factor` makes powers of two of them (where both are large, a difference of products keeps
                // what their multiples lose); otherwise of scores in units of log 2.  A maximum lags by `limit` at most: compared are
                // differences, since a large maximum's sum with it may be rounded to the next number.
                const float factor = PLAIN ? p.unit : 1.0f, limit = fminf(8.0f / factor, CUDART_MAX_NORMAL_F);
                const float cap_in = !PLAIN && p.cap > 0.0f ? p.scale / p.cap : 0.0f;

                float acc[HEAD_DIM / 16][4] = {};  // elements 16 m + g and 16 m + 8 + g, rows 2 t and 2 t + 1
                float top[2] = {-CUDART_INF_F, -CUDART_INF_F}, against[2] = {0.0f, 0.0f}, sum[2] = {0.0f, 0.0f};
#pragma unroll 1
                for (int i = 1 - kStages; i < end - begin; ++i) {
                    if (i >= 0) {
                        four_copies_wait<kStages - 2>();
                        __syncwarp();
                    }
                    copy(i + kStages - 1);
                    if (i < 0)
                        continue;
                    const unsigned char* const keys = ring_ptr + at_hand;
                    const uint32_t             vals = ring + at_hand + kTileBytes;
                    const int                  key0 = key_of(begin + i);
                    at_hand = at_hand == (kStages - 1) * kStageBytes ? 0 : at_hand + kStageBytes;

                    // ---- scores: keys g and g + 8, rows 2 t and 2 t + 1
                    float products[2][4];
#pragma unroll
                    for (int m = 0; m < HEAD_DIM / 32; ++m) {
                        const uint4 a = *reinterpret_cast<const uint4*>(keys + place_k(g, 4 * m + t)), z = *reinterpret_cast<const uint4*>(keys + place_k(g, 4 * m + t) + 8 * kRowBytes);
                        if (m == 0) {
                            four_mma_first(products[0], a.x, z.x, a.y, z.y, qf[0][0], qf[0][1]);
                            four_mma_first(products[1], a.z, z.z, a.w, z.w, qf[1][0], qf[1][1]);
                        }
                        else {
                            four_mma(products[0], a.x, z.x, a.y, z.y, qf[2 * m][0], qf[2 * m][1]);
                            four_mma(products[1], a.z, z.z, a.w, z.w, qf[2 * m + 1][0], qf[2 * m + 1][1]);
                        }
                    }
                    float s[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[e] = products[0][e] + products[1][e];
                        if constexpr (!PLAIN) {
                            s[e] = p.cap > 0.0f ? four_capped(s[e], cap_in, p.cap * CUDART_L2E_F) : s[e] * (p.scale * CUDART_L2E_F);
                            s[e] = fmaf(slope[e % 2], static_cast<float>(key0 + g + 8 * (e / 2) - place), s[e]);
                        }
                    }
                    if (partly(key0)) {
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (!sees(key0 + g + 8 * k))
                                s[2 * k] = s[2 * k + 1] = -CUDART_INF_F;
                    }
                    if (__any_sync(0xffffffffu, fmaxf(s[0], s[2]) - top[0] > limit || fmaxf(s[1], s[3]) - top[1] > limit)) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float newtop = fmaxf(top[e], fmaxf(s[e], s[e + 2]));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1)
                                newtop = fmaxf(newtop, __shfl_xor_sync(0xffffffffu, newtop, d));
                            const float keep = top[e] == newtop ? 1.0f : ptx::exp2_approx((top[e] - newtop) * factor);
                            top[e]           = newtop;
                            against[e]       = newtop == -CUDART_INF_F ? 0.0f : newtop;
                            sum[e] *= keep;
#pragma unroll
                            for (int m = 0; m < HEAD_DIM / 16; ++m) {
                                acc[m][e] *= keep;
                                acc[m][e + 2] *= keep;
                            }
                        }
                    }
                    // ---- weights (2^kAttnWeightExponent as large) as the second product's columns, keys g and g + 8
                    uint32_t pf[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float x = ptx::exp2_approx(fmaf(s[2 * k] - against[0], factor, kAttnWeightExponent));
                        const float y = ptx::exp2_approx(fmaf(s[2 * k + 1] - against[1], factor, kAttnWeightExponent));
                        sum[0] += x;
                        sum[1] += y;
                        const half2 h = __floats2half2_rn(x, y);
                        pf[k]         = four_transpose(*reinterpret_cast<const uint32_t*>(&h));
                    }
                    // ---- outputs: lanes 8 j to 8 j + 7 address the keys of matrix j, keys 0-7 or 8-15, elements 16 m or 16 m + 8 on
                    const int key = (lane & 7) + (lane & 16) / 2, of = lane >> 3 & 1;
#pragma unroll
                    for (int m = 0; m < HEAD_DIM / 16; ++m) {
                        uint32_t a[4];
                        single_load_transposed(vals + place_v(key, 2 * m + of), a);
                        four_mma(acc[m], a[0], a[1], a[2], a[3], pf[0], pf[1]);
                    }
                }
                four_copies_wait<0>();
                __syncwarp();

                // ---- the end of the piece: sums by way of shared memory, rows one behind another
                const bool     item = begin == 0 && end == sight.blocks;
                const unsigned kind = begin == 0 ? kPartBegins : end == sight.blocks ? kPartEnds : kPartContinues;
                const int      slot = item || kind == kPartBegins ? 1 : 0;
                float* const   to   = reinterpret_cast<float*>(slot ? ring_ptr : first_sums + warp * four_rows_bytes(HEAD_DIM, 1));
                bool           nan  = false;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 2 * t + e;
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1)
                        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], d);
                    if (row < rows) {
#pragma unroll
                        for (int m = 0; m < HEAD_DIM / 16; ++m) {
                            to[row * HEAD_DIM + 16 * m + g]     = acc[m][e];
                            to[row * HEAD_DIM + 16 * m + 8 + g] = acc[m][e + 2];
                            nan = nan || (sum[e] == sum[e] && (acc[m][e] != acc[m][e] || acc[m][e + 2] != acc[m][e + 2]));
                        }
                        if (g == 0)
                            sh.stats[warp][slot][row] = make_float2(top[e], sum[e]);
                    }
                }
                __syncwarp();
                if (__any_sync(0xffffffffu, nan))
                    single_restore<HEAD_DIM>(p, b, head, begin, end, rows, to, sh.stats[warp][slot], key_of, sees);
                __syncwarp();
                if (item) {
                    for (int u = lane; u < rows * (HEAD_DIM / 4); u += 32) {
                        const int row = u / (HEAD_DIM / 4), column = u % (HEAD_DIM / 4) * 4;
                        *reinterpret_cast<uint2*>(four_out<HEAD_DIM>(p, q.first, head, row0 + row) + column) =
                            four_outputs(*reinterpret_cast<const float4*>(to + row * HEAD_DIM + column), sh.stats[warp][slot][row].y);
                    }
                    __syncwarp();
                }
                else if (lane == 0)
                    sh.part[warp][slot] = FourPart{kind, q.first, row0, rows, head, {0, 0, 0}};
            }
            else if (begin > 0) {
                // A share so small that none of the item's blocks is its own: a part all the same, for the others' chain.
                float* const to = reinterpret_cast<float*>(first_sums + warp * four_rows_bytes(HEAD_DIM, 1));
                for (int i = lane; i < rows * HEAD_DIM; i += 32)
                    to[i] = 0.0f;
                if (lane < rows)
                    sh.stats[warp][0][lane] = make_float2(-CUDART_INF_F, 0.0f);
                if (lane == 0)
                    sh.part[warp][0] = FourPart{kPartContinues, q.first, row0, rows, head, {0, 0, 0}};
            }
        } while (walk.next(p, sh));
    }
    __syncthreads();
    four_finish<HEAD_DIM, kRows, kSingleWarps>(p, sh, smem, kStages * kStageBytes, first_sums);
}

}  // namespace flashllm
