// Attention over a paged cache of 4 bits (four_bit_cache.cuh) of few rows per key/value head: single tokens, a few of them.
//
//   s_ij = scale q_i . k_j,  capped: cap tanh(s_ij / cap),  then + slope_h (j - i)
//   o_i  = sum over the keys j that i sees of softmax_j(s_ij) v_j;  zero for a row that sees none
//
// Codes are not turned into elements before they are multiplied: with k = low + step n for each 64 elements g of a head
//
//   q . k       = sum_g step_g (q_g . n_g) + low_g sum(q_g)
//   sum_j p_j v = sum_j (p_j step_j) n_j + sum_j p_j low_j
//
// so that an element costs 0.6 to 0.75 operations: four bits masked out of a word are the mantissa of a subnormal fp16 number, n x 2^-24
// (or, where they lie four bits up, sixteen times that), which the tensor core multiplies exactly.  Products are transposed, S^T = K Q^T and O^T = V^T P^T
// (m16n8k16): 16 keys, then 16 elements of a head, are the rows, the queries the 8 columns, so that eight queries waste nothing
// (the tensor core is busy a quarter of the time).  tcgen05 would want dense tiles in shared memory:
// 64 KB written and read for each 18 KB of codes, half of the memory's time by itself.
//
// Every warp works by itself: it copies 32 keys and values at a time (16 where it has sixteen rows) into its own ring in shared memory
// (cp.async, no barriers) and keeps maximum, sum and outputs of its rows in registers.  The work of a call, blocks of so many keys of
// all sequences, tiles of rows and heads, is one linear sequence dealt out evenly over all warps; warps that share an item leave sums, which their CTA adds up in key
// order, and CTAs that do leave theirs in the workspace for four_bit_join_kernel.
//
// Bound by the issue of operations next to memory (9/16 of a byte per element): 310 for 16 keys in the loop, with all that is before
// and behind it 322 in 16 sequences of 4000 to 40000 positions in 8 heads of 128, and 352 in 64 of 100 to 9000.  The former, 274 MB, are
// 72 us a call, 67 replayed from a graph, of which 50 are the loop (42 at the measured copy bandwidth), the latter, 138 MB, 42 and 41.
#pragma once
#include <math_constants.h>

#include "attention_kernel_sm100.cuh"
#include "four_bit_cache.cuh"

namespace flashllm {

struct FourBitParams {
    CacheBatch           batch;
    const half*          q;    // [tokens][ld_q]
    half*                out;  // [tokens][heads * head_dim]
    const unsigned char* k_cache;
    const unsigned char* v_cache;
    const float*         slopes;  // [heads], or nullptr
    unsigned char*       workspace;
    long long            ld_q;
    int                  heads;
    int                  share;  // query heads per key/value head, and what divides by it (see AttentionParams)
    unsigned             share_magic;
    int                  share_shift;
    int                  token_tiles;  // tiles of eight rows of a token: kernels whose tiles are of one token each
    int                  window;  // keys up to itself that a row sees
    int                  sinks;   // ... and of its sequence's first
    int                  most_rows;  // sequences with more rows (tokens x share) are somebody else's
    float                scale;
    float                cap;  // 0: none
    float                unit;  // times a difference of the maxima that parts leave: the exponent of a power of two
};

constexpr int kFourKeys = 16;  // keys of a product: a page holds whole sixteens

// TILES of eight rows each.
// (Three or two for each scheduler.  Four, with registers spilled: 16 long sequences 70.4 us instead of 67.3; 13, unevenly: 82.)
__host__ __device__ constexpr int four_warps(int tiles)
{
    return tiles == 1 ? 12 : 8;
}

// Sixteens of keys that a warp takes at a time, a block: two are independent work side by side and share what a step costs, for
// more rows the registers hold one.
__host__ __device__ constexpr int four_sixteens(int tiles)
{
    return tiles == 1 ? 2 : 1;
}

__host__ __device__ constexpr int four_stage_bytes(int head_dim, int tiles)
{
    return 2 * kFourKeys * four_sixteens(tiles) * four_bit_row_bytes(head_dim);
}

// Blocks in flight or at hand per warp: 110 to 150 KB of an SM.  (One on its way while another is worked on is enough: 16 long sequences
// 67.3 us, 67.9 with two.)
__host__ __device__ constexpr int four_stages(int head_dim, int tiles)
{
    return (tiles == 1 ? 2 : 8) * 128 / head_dim;
}

struct FourPart {
    unsigned kind;  // kPartNone ...
    int      first;  // first row of the sequence in the batch
    int      row0;   // first row of the item in the sequence's
    int      rows;   // rows of the item
    int      head;   // key/value head
    int      pad[3];
};

constexpr int kFourKnown = 384;  // sequences whose sizes are kept in shared memory

struct FourShared {
    unsigned long long before[512];  // units before a thread's sequences
    int4               known[kFourKnown];  // first row, rows, context, units of the first sequences
    unsigned long long total;
    unsigned long long warp_sums[16];
    FourPart           part[16][2];       // of each warp: a piece of an item begun before it, and one that others end
    float2             stats[16][2][16];  // maximum and sum of a part's rows
};

__host__ __device__ constexpr int four_rows_bytes(int head_dim, int tiles)
{
    return 8 * tiles * head_dim * 4;
}

// The ring of each warp (where the sums of its last part go in the end), the sums of its first part, and FourShared.
__host__ __device__ constexpr int four_smem_bytes(int head_dim, int tiles)
{
    return four_warps(tiles) * (four_stages(head_dim, tiles) * four_stage_bytes(head_dim, tiles) + four_rows_bytes(head_dim, tiles))
           + static_cast<int>(sizeof(FourShared)) + 128;
}

// Workspace: two parts of each CTA, [cta][2] FourPart, then their rows' statistics, then their sums.
__host__ __device__ constexpr size_t four_stats_offset(int ctas)
{
    return size_t(2) * ctas * sizeof(FourPart);
}

__host__ __device__ constexpr size_t four_sums_offset(int ctas)
{
    return four_stats_offset(ctas) + size_t(2) * ctas * 16 * sizeof(float2);
}

__host__ __device__ constexpr size_t four_workspace_bytes(int ctas, int head_dim)
{
    return four_sums_offset(ctas) + size_t(2) * ctas * 16 * head_dim * sizeof(float);
}

// ---------------------------------------------------------------- the work of a call

// Beginning and ending an item takes a warp about as long as so many blocks.
constexpr int kFourExtra = 3;

// A tile of rows of a sequence, and the blocks of keys that any of them sees: those before `skip_from`, and from there on those
// `skip` further on.
struct FourTile {
    int blocks, skip_from, skip;
};

template<int KEYS>
__device__ __forceinline__ FourTile four_tile(const FourBitParams& p, int context, int token0, int token1)
{
    const int keys = context + token1 + 1, first = max(0, context + token0 - p.window + 1);
    FourTile  t;
    t.skip_from = static_cast<int>((static_cast<long long>(min(p.sinks, keys)) + KEYS - 1) / KEYS);
    t.skip      = max(0, first / KEYS - t.skip_from);
    t.blocks    = static_cast<int>((static_cast<long long>(keys) + KEYS - 1) / KEYS) - t.skip;
    return t;
}

// Token of a row of a sequence's (tokens x share) rows.
__device__ __forceinline__ int four_token(const FourBitParams& p, int row)
{
    return static_cast<int>((__umulhi(static_cast<unsigned>(row), p.share_magic) + static_cast<unsigned>(row)) >> p.share_shift);
}

// A sequence's tiles of rows, and the units that each of them counts: at least its blocks and what beginning it takes, the same for
// all (exact for a single tile; the tiles of longer prompts share a bound).
struct FourSequence {
    int first, count, context;  // first row, rows of the batch, position of the first
    int rows, tiles, units;
};

// BY_TOKEN: no tile has rows of two tokens.
template<int ROWS, int KEYS, bool BY_TOKEN>
__device__ __forceinline__ FourSequence four_sequence(const FourBitParams& p, int b, int* lost = nullptr)
{
    const Sequence s = load_sequence(p.batch, b);
    FourSequence   q{s.first, s.count, s.context, s.count * p.share, 0, 0};
    if (lost)
        *lost = s.lost;
    if (q.rows > p.most_rows)
        q.rows = q.count = 0;
    q.tiles = BY_TOKEN ? q.count * p.token_tiles : (q.rows + ROWS - 1) / ROWS;
    if (q.tiles == 1 || q.count == 1)
        q.units = four_tile<KEYS>(p, q.context, 0, q.count - 1).blocks + kFourExtra;
    else if (q.tiles > 1) {
        const long long all = (static_cast<long long>(q.context) + q.count + KEYS - 1) / KEYS;
        // Behind the sinks: a window's keys and those of the tile's tokens, wherever blocks begin.
        const long long seen = (static_cast<long long>(min(p.sinks, q.context + q.count)) + KEYS - 1) / KEYS
                               + (static_cast<long long>(p.window) + ROWS + 2 * KEYS) / KEYS;
        q.units = static_cast<int>(min(all, seen)) + kFourExtra;
    }
    return q;
}

template<int ROWS, int KEYS, bool BY_TOKEN>
__device__ __noinline__ FourSequence four_sequence_again(const FourBitParams& p, int b)
{
    return four_sequence<ROWS, KEYS, BY_TOKEN>(p, b);
}

// ... what the plan has kept of it.
template<int ROWS, int KEYS, bool BY_TOKEN>
__device__ __forceinline__ FourSequence four_sequence(const FourBitParams& p, const FourShared& sh, int b)
{
    if (b >= kFourKnown)
        return four_sequence_again<ROWS, KEYS, BY_TOKEN>(p, b);
    const int4 known = sh.known[b];
    const int  rows  = known.y * p.share;
    return FourSequence{known.x, known.y, known.z, rows, BY_TOKEN ? known.y * p.token_tiles : (rows + ROWS - 1) / ROWS, known.w};
}

// a / b, of 32 bits where they are that.
__device__ __forceinline__ unsigned long long four_divide(unsigned long long a, unsigned long long b)
{
    return ((a | b) >> 32) == 0 ? static_cast<unsigned>(a) / static_cast<unsigned>(b) : a / b;
}

// ---------------------------------------------------------------- pieces of the kernel

__device__ __forceinline__ void four_copy16(uint32_t dst, const void* src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void four_copies_done()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}

template<int PENDING>
__device__ __forceinline__ void four_copies_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ void four_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ... of two operands alone.
__device__ __forceinline__ void four_mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t four_transpose(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

__device__ __forceinline__ float four_weight(float top, float newtop, float unit = 1.0f)
{
    return top == newtop ? 1.0f : ptx::exp2_approx((top - newtop) * unit);
}

// Place of a key's values among the 16 of a block: a thread's four keys, 2 t, 2 t + 1, 2 t + 8 and 2 t + 9, lie four places apart.
__device__ __forceinline__ int four_value_place(int key)
{
    return (key & 8) | (key & 1) << 2 | (key >> 1 & 3);
}

// Adds up four columns of a row of one item's parts, in key order: `stats(i)` is the i-th part's maximum and sum of the row, `sums(i)`
// its outputs of these columns, `unit` FourBitParams'.  AT_ONCE parts' loads are under way at a time.
template<int AT_ONCE, typename Stats, typename Sums>
__device__ __forceinline__ float4 four_add_up(int count, float unit, Stats&& stats, Sums&& sums, float2& all)
{
    float  top = -CUDART_INF_F, sum = 0.0f;
    float4 o   = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += AT_ONCE) {
        float2 s[AT_ONCE];
        float4 x[AT_ONCE];
        float  newtop = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            s[i] = make_float2(-CUDART_INF_F, 0.0f);
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 + i < count) {
                s[i] = stats(i0 + i);
                x[i] = *sums(i0 + i);
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            newtop = fmaxf(newtop, s[i].x);
        // (Never zero: a part's infinity stays one.)
        const float before = fmaxf(four_weight(top, newtop, unit), 0x1p-126f);
        sum *= before;
        o   = make_float4(o.x * before, o.y * before, o.z * before, o.w * before);
        top = newtop;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const float keep = fmaxf(four_weight(s[i].x, top, unit), 0x1p-126f);
            sum              = fmaf(s[i].y, keep, sum);
            o                = make_float4(fmaf(x[i].x, keep, o.x), fmaf(x[i].y, keep, o.y), fmaf(x[i].z, keep, o.z), fmaf(x[i].w, keep, o.w));
        }
    }
    all = make_float2(top, sum);
    return o;
}

// Four outputs of a row, divided by its sum.
__device__ __forceinline__ uint2 four_outputs(float4 o, float sum)
{
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    return make_uint2(attn_pack_bounded(o.x * inverse, o.y * inverse), attn_pack_bounded(o.z * inverse, o.w * inverse));
}

// Eight outputs of a row, divided by its sum.
__device__ __forceinline__ uint4 four_outputs(const float (&o)[8], float sum)
{
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    return make_uint4(attn_pack_bounded(o[0] * inverse, o[1] * inverse), attn_pack_bounded(o[2] * inverse, o[3] * inverse),
                      attn_pack_bounded(o[4] * inverse, o[5] * inverse), attn_pack_bounded(o[6] * inverse, o[7] * inverse));
}

template<int HEAD_DIM>
__device__ __forceinline__ half* four_out(const FourBitParams& p, int first, int head, int row)
{
    const int token = four_token(p, row);
    return p.out + (static_cast<long long>(first + token) * p.heads + head * p.share + (row - token * p.share)) * HEAD_DIM;
}

// cap tanh(x / cap) in units of log 2, `in` = 1 / cap x what x lacks, `cap` = the cap times log2 e.
__device__ __forceinline__ float four_capped(float x, float in, float cap)
{
    const float y = x * in, z = y * y;
    if (fabsf(y) <= kAttnTanhRange) {
        float t = kAttnTanh[kAttnTanhTerms - 1];
#pragma unroll
        for (int k = kAttnTanhTerms - 2; k >= 0; --k)
            t = fmaf(t, z, kAttnTanh[k]);
        return cap * (y * t);
    }
    return fmaf(-2.0f * cap, ptx::rcp_approx(1.0f + ptx::exp2_approx(2.0f * CUDART_L2E_F * y)), cap);
}

// Where each warp's share of the work begins and ends; false if there is none at all.  For all threads: each counts the units of a few
// sequences in a row.
template<int HEAD_DIM, int ROWS, int KEYS, int WARPS, bool BY_TOKEN>
__device__ __forceinline__ bool four_plan(const FourBitParams& p, FourShared& sh, unsigned long long& u0, unsigned long long& u1)
{
    const CacheBatch& c    = p.batch;
    const int         warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_thread = c.sequences <= (WARPS * 32) ? 1 : (c.sequences + (WARPS * 32) - 1) / (WARPS * 32);
    {
        unsigned long long mine = 0;
        bool               lost = false;
        for (int k = 0; k < per_thread; ++k) {
            const int b = threadIdx.x * per_thread + k;
            if (b >= c.sequences)
                break;
            int                rows_lost;
            const FourSequence q = four_sequence<ROWS, KEYS, BY_TOKEN>(p, b, &rows_lost);
            mine += static_cast<unsigned long long>(q.tiles) * (static_cast<unsigned long long>(q.units) * c.kv_heads);
            lost = lost || rows_lost > 0;
            if (b < kFourKnown)
                sh.known[b] = make_int4(q.first, q.count, q.context, q.units);
        }
        const unsigned long long upto = attn_warp_scan(mine);
        if (lane == 31)
            sh.warp_sums[warp] = upto;
        if (lane == 0)
            sh.part[warp][0].kind = sh.part[warp][1].kind = kPartNone;
        if (__syncthreads_or(lost ? 1 : 0)) {  // rows of sequences that do not fit
            for (int b = blockIdx.x; b < c.sequences; b += gridDim.x) {
                const Sequence  q   = load_sequence(c, b);
                const long long row = static_cast<long long>(p.heads) * HEAD_DIM;
                for (long long i = threadIdx.x * 8; i < q.lost * row; i += (WARPS * 32) * 8)
                    *reinterpret_cast<uint4*>(p.out + q.first * row + i) = make_uint4(0, 0, 0, 0);
            }
        }
        unsigned long long before = upto - mine;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            before += w < warp ? sh.warp_sums[w] : 0;
        sh.before[threadIdx.x] = before;
        if (threadIdx.x == (WARPS * 32) - 1)
            sh.total = before + mine;
        __syncthreads();
    }
    const unsigned long long total = sh.total;
    if (total == 0) {
        if (threadIdx.x < 2)
            reinterpret_cast<FourPart*>(p.workspace)[2 * blockIdx.x + threadIdx.x].kind = kPartNone;
        return false;
    }
    // Small calls take as few warps of each CTA as leave them a few blocks each.
    constexpr unsigned       kLeast = kFourExtra + 2;
    const int                busy   = total >= static_cast<unsigned long long>(kLeast) * WARPS * gridDim.x ? WARPS : static_cast<int>(total) / static_cast<int>(kLeast * gridDim.x) + 1;
    const unsigned           workers = gridDim.x * busy;
    const unsigned long long share   = four_divide(total + workers - 1, workers);
    const unsigned long long worker  = static_cast<unsigned long long>(blockIdx.x) * busy + warp;
    u0 = min(total, share * worker);
    u1 = warp < busy ? min(total, u0 + share) : u0;
    return true;

}

// Walks a warp's share: pieces of items, order (sequence, tile of rows, key/value head, blocks of keys).
template<int ROWS, int KEYS, int WARPS, bool BY_TOKEN>
struct FourWalk {
    FourSequence       q;
    FourTile           sight;
    int                b, tile, head, unit, upto;
    int                row0, rows, token0, token1;  // of the tile
    int                begin, end;                  // blocks of the piece
    unsigned long long left;

    __device__ __forceinline__ void start(const FourBitParams& p, const FourShared& sh, unsigned long long u0, unsigned long long u1)
    {
        const int per_thread = p.batch.sequences <= WARPS * 32 ? 1 : (p.batch.sequences + WARPS * 32 - 1) / (WARPS * 32);
        // The thread that counted the sequence of unit u0, and that sequence.
        int lo = 0;
#pragma unroll 1
        for (int step = 256; step > 0; step >>= 1)
            if (lo + step < WARPS * 32 && sh.before[lo + step] <= u0)
                lo += step;
        // (several threads may have the same count: the last of them has units)
        unsigned long long at = sh.before[lo];
        b = lo * per_thread;
        q = four_sequence<ROWS, KEYS, BY_TOKEN>(p, sh, b);
        auto               whole = [&]() { return static_cast<unsigned long long>(q.tiles) * (static_cast<unsigned long long>(q.units) * p.batch.kv_heads); };
        while (at + whole() <= u0 && b + 1 < p.batch.sequences) {
            at += whole();
            q = four_sequence<ROWS, KEYS, BY_TOKEN>(p, sh, ++b);
        }
        const unsigned long long in       = u0 - at;  // unit of the sequence
        const unsigned long long per_tile = static_cast<unsigned long long>(max(q.units, 1)) * p.batch.kv_heads;
        tile = q.tiles > 1 ? static_cast<int>(four_divide(in, per_tile)) : 0;
        const unsigned long long in_tile  = in - tile * per_tile;
        head = static_cast<int>(four_divide(in_tile, max(q.units, 1)));
        unit = static_cast<int>(in_tile - static_cast<unsigned long long>(head) * max(q.units, 1));
        left = u1 - u0;

    }
    __device__ __forceinline__ void piece(const FourBitParams& p)
    {
        if constexpr (BY_TOKEN) {
            token0 = token1 = p.token_tiles == 1 ? tile : tile / p.token_tiles;
            row0            = token0 * p.share + (tile - token0 * p.token_tiles) * ROWS;
            rows            = min(ROWS, (token0 + 1) * p.share - row0);
        }
        else {
            row0   = tile * ROWS;
            rows   = min(ROWS, q.rows - row0);
            token0 = four_token(p, row0);
            token1 = four_token(p, row0 + rows - 1);
        }
        sight = four_tile<KEYS>(p, q.context, token0, token1);
        upto  = static_cast<int>(min(static_cast<unsigned long long>(q.units), unit + left));
        // Units of the tile to its blocks: exact where the tile's blocks are what it counts, in proportion where they are fewer.
        auto cut = [&](int x) {
            const int counted = q.units - kFourExtra, behind = max(0, x - kFourExtra);
            return counted == sight.blocks ? behind : static_cast<int>(static_cast<long long>(behind) * sight.blocks / counted);
        };
        begin = cut(unit);
        end   = cut(upto);
        left -= upto - unit;
    }
    // On to the next item; false at the end.
    __device__ __forceinline__ bool next(const FourBitParams& p, const FourShared& sh)
    {
        if (left == 0)
            return false;
        unit = upto;
        if (unit == q.units) {
            unit = 0;
            if (++head == p.batch.kv_heads) {
                head = 0;
                if (++tile == q.tiles) {
                    tile = 0;
                    do {
                        if (++b >= p.batch.sequences)
                            return false;
                        q = four_sequence<ROWS, KEYS, BY_TOKEN>(p, sh, b);
                    } while (q.tiles == 0);
                }
            }
        }
        return true;
    }
};

// Items that several warps of a CTA have worked on, in key order; what began before this CTA, or ends behind it, to the workspace.  For all
// threads; sums of a warp's first part lie in `first_sums`, those of its last in its ring (`ring_bytes` each).
template<int HEAD_DIM, int ROWS, int WARPS>
__device__ __forceinline__ void four_finish(const FourBitParams& p, const FourShared& sh, const unsigned char* smem, int ring_bytes, const unsigned char* first_sums)
{
    const int lane = threadIdx.x & 31;
    // Parts in key order, of warp i / 2: that is their kinds, and which of them belong to an item.  All items side by side.
    const unsigned kind_here = lane < 2 * WARPS ? sh.part[lane >> 1][lane & 1].kind : kPartNone;
    const unsigned begins = __ballot_sync(0xffffffffu, kind_here == kPartBegins), ends = __ballot_sync(0xffffffffu, kind_here == kPartEnds);
    const unsigned all_present = __ballot_sync(0xffffffffu, kind_here != kPartNone);
    constexpr int  kPerItem = ROWS * (HEAD_DIM / 4);
    unsigned       present = all_present;
    int            number  = 0;  // of the item that `present` begins with
#pragma unroll 1
    for (int u = threadIdx.x;; u += (WARPS * 32)) {
        unsigned mine = 0;
#pragma unroll 1
        for (;;) {
            // Up to the part that ends the item, or before the next that begins one.
            const unsigned ending = ends & present, other = begins & present & (present - 1);
            mine = present;
            if (ending)
                mine &= ending ^ (ending - 1);
            if (other)
                mine &= (other & -other) - 1;
            if (number == u / kPerItem || present == 0)
                break;
            present &= ~mine;
            ++number;
        }
        if (mine == 0)
            break;
        const int       row = u / (HEAD_DIM / 4) % ROWS, column = u % (HEAD_DIM / 4) * 4;
        // The parts are those of neighbouring warps, the first of which may be the last piece of its warp; the others are first pieces.
        const int       begin = (__ffs(mine) - 1) >> 1, tail = (__ffs(mine) - 1) & 1, count = (31 - __clz(mine)) / 2 - begin + 1;
        const FourPart& from  = sh.part[begin][tail];
        const bool      ended = (mine & ends) != 0, item = from.kind == kPartBegins && ended;
        const unsigned  kind  = from.kind == kPartBegins ? kPartBegins : ended ? kPartEnds : kPartContinues;
        const int       slot  = kind == kPartBegins ? 1 : 0;
        if (row < from.rows) {
            float2       all;
            const float4 o = four_add_up<1>(
                count, p.unit, [&](int k) { return sh.stats[begin + k][k == 0 ? tail : 0][row]; },
                [&](int k) {
                    const int            w  = begin + k;
                    const unsigned char* at = k == 0 && tail ? smem + w * ring_bytes : first_sums + w * four_rows_bytes(HEAD_DIM, ROWS / 8);
                    return reinterpret_cast<const float4*>(at) + row * (HEAD_DIM / 4) + column / 4;
                },
                all);
            if (item)
                *reinterpret_cast<uint2*>(four_out<HEAD_DIM>(p, from.first, from.head, from.row0 + row) + column) = four_outputs(o, all.y);
            else {
                const size_t at = static_cast<size_t>(2 * blockIdx.x + slot) * 16 + row;
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.workspace + four_sums_offset(gridDim.x)) + at * HEAD_DIM + column) = o;
                if (column == 0)
                    reinterpret_cast<float2*>(p.workspace + four_stats_offset(gridDim.x))[at] = all;
            }
        }
        if (!item && u % kPerItem == 0)
            reinterpret_cast<FourPart*>(p.workspace)[2 * blockIdx.x + slot] = FourPart{kind, from.first, from.row0, from.rows, from.head, {0, 0, 0}};
    }
    if (threadIdx.x < 2) {
        // What this CTA leaves for others: a first piece where the first part began elsewhere, a last one where the last part has not
        // ended and its item began here.
        const unsigned first = all_present & -all_present, last_begins = begins ? 31 - __clz(begins) : -1;
        const bool     has   = threadIdx.x == 0 ? (first & ~begins) != 0 : begins != 0 && (ends >> last_begins) == 0;
        if (!has)
            reinterpret_cast<FourPart*>(p.workspace)[2 * blockIdx.x + threadIdx.x].kind = kPartNone;
    }
}

// PLAIN: neither cap nor slopes.  TILES of eight rows at a time.
template<int HEAD_DIM, int TILES, bool PLAIN>
__global__ void __launch_bounds__(four_warps(TILES) * 32, 1) four_bit_attention_kernel(const __grid_constant__ FourBitParams p)
{
    constexpr int  kRows = 8 * TILES, kWarps = four_warps(TILES), kThreads = kWarps * 32, kGroups = four_bit_groups(HEAD_DIM);
    constexpr int  kSixteens = four_sixteens(TILES), kKeys = kFourKeys * kSixteens;  // of a block
    constexpr int  kStages = four_stages(HEAD_DIM, TILES), kStageBytes = four_stage_bytes(HEAD_DIM, TILES);
    constexpr int  kSixteenCodes = kFourKeys * HEAD_DIM / 2, kSixteenScales = kFourKeys * 4 * kGroups;  // bytes
    constexpr int  kCodeBytes = kSixteens * kSixteenCodes, kScaleBytes = kSixteens * kSixteenScales;    // of a block's keys
    constexpr float kOne = 16777216.0f;  // 2^24: what a product with n x 2^-24 lacks
    extern __shared__ unsigned char smem_raw[];
    const uint32_t       raw  = ptx::smem_u32(smem_raw);
    const uint32_t       base = (raw + 127u) & ~127u;
    unsigned char* const smem = smem_raw + (base - raw);
    const int            warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const CacheBatch&    c    = p.batch;
    const uint32_t       ring = base + warp * (kStages * kStageBytes);
    unsigned char* const ring_ptr = smem + warp * (kStages * kStageBytes);
    unsigned char* const first_sums = smem + kWarps * (kStages * kStageBytes);  // [warp][rows][head_dim] floats
    FourShared&          sh = *reinterpret_cast<FourShared*>(first_sums + kWarps * four_rows_bytes(HEAD_DIM, TILES));

    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    unsigned long long u0, u1;
    if (!four_plan<HEAD_DIM, kRows, kKeys, kWarps, false>(p, sh, u0, u1))
        return;

    // What the copies of a lane have in common: 16 bytes of the codes of a key (and of the one eight further on), and of the scales.
    // Rows of 64 bytes have their chunks 2 and 3 first in every other pair of rows, for the banks.
    const uint32_t page_bytes = static_cast<uint32_t>(four_bit_row_bytes(HEAD_DIM)) << c.page_shift;
    constexpr int  kRowBytes  = HEAD_DIM / 2, kChunks = kRowBytes / 16;
    auto           place      = [](int row, int chunk) { return row * kRowBytes + 16 * (HEAD_DIM == 128 ? chunk ^ (row & 2) : chunk); };
    const unsigned char* const from_k = p.k_cache + 16 * lane;
    const unsigned char* const from_v = p.v_cache + 16 * lane;
    const int scale_chunk = lane % (kScaleBytes / 16), second = scale_chunk / (kSixteenScales / 16);  // of the second sixteen keys
    const unsigned char* const from_scales = (lane < kScaleBytes / 16 ? p.k_cache : p.v_cache) + 16 * scale_chunk
                                             + (static_cast<long long>(kRowBytes) << c.page_shift);
    const uint32_t to_k = ring + place(lane / kChunks, lane % kChunks), to_scales = ring + 2 * kCodeBytes + 16 * lane;
    const uint32_t to_v = ring + kCodeBytes + place(four_value_place(lane / kChunks), lane % kChunks);
    // ... and its loads: of keys g and g + 8, and of values at four places; chunks of the second 64 elements lie at the address with
    // bit 5 turned.
    const uint32_t at_k = place(g, t / 2) + 8 * (t & 1), at_v = kCodeBytes + place(t, g / 4) + 4 * (g & 3);
    uint32_t       copied = 0;

    if (u0 < u1) {
        FourWalk<kRows, kKeys, kWarps, false> walk;
        walk.start(p, sh, u0, u1);
        do {
            // ---- a piece of an item
            walk.piece(p);
            const FourSequence& q    = walk.q;
            const FourTile      sight = walk.sight;
            const int b = walk.b, head = walk.head, row0 = walk.row0, rows = walk.rows, token0 = walk.token0, token1 = walk.token1, begin = walk.begin, end = walk.end;
            if (begin < end) {
                // The rows of Q, on their way while pages are looked up.
                uint4 q_raw[TILES][kGroups][2];
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    const int         row = 8 * n + g, token = four_token(p, row0 + row);
                    const half* const from = p.q + (q.first + token) * p.ld_q + static_cast<long long>(head * p.share + row0 + row - token * p.share) * HEAD_DIM;
#pragma unroll
                    for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
                        for (int w = 0; w < 2; ++w)
                            q_raw[n][gr][w] = row < rows ? *reinterpret_cast<const uint4*>(from + gr * kFourBitGroup + 16 * t + 8 * w) : make_uint4(0, 0, 0, 0);
                }
                const int* const table = c.page_table + static_cast<long long>(b) * c.table_width;
                auto key_of = [&](int block) { return (block + (block < sight.skip_from ? 0 : sight.skip)) * kKeys; };
                const int keys = q.context + token1 + 1;  // none at or behind this is seen
                // Page ids of 32 sixteens at a time, a lane each, the next 32 ahead of their use; -1: reads as zeros.
                auto ids_from = [&](int block) {
                    block += lane / kSixteens;
                    if (block >= end)
                        return -1;
                    const int key = key_of(block) + lane % kSixteens * kFourKeys;
                    if (key >= keys)
                        return -1;
                    const int id = table[key >> c.page_shift];
                    if (static_cast<unsigned>(id) < static_cast<unsigned>(c.pages))
                        return id;
                    atomicOr(c.status, kStatusBadCache);
                    return -1;
                };
                constexpr int kAhead = 32 / kSixteens;
                int  ids = ids_from(begin), ids_next = ids_from(begin + kAhead);
                auto copy = [&](int i) {  // the i-th block of the piece, to the next place of the ring
                    if (begin + i < end) {
                        if (i > 0 && i % kAhead == 0) {
                            ids      = ids_next;
                            ids_next = ids_from(begin + i + kAhead);
                        }
                        // (32-bit factors: multiply-adds with wide sums, no shifts and additions of 64 bits)
                        auto sixteens = [&](int id, uint32_t in, int first, int count, bool scales) {
                            const uint32_t piece = max(id, 0) * c.kv_heads + head;  // of the cache's pages and heads
                            const unsigned char* const k = from_k + static_cast<unsigned long long>(piece) * page_bytes + static_cast<unsigned long long>(in) * kRowBytes;
                            const unsigned char* const v = from_v + static_cast<unsigned long long>(piece) * page_bytes + static_cast<unsigned long long>(in) * kRowBytes;
                            const unsigned char* const w = from_scales + static_cast<unsigned long long>(piece) * page_bytes + static_cast<unsigned long long>(in) * (4 * kGroups);
#pragma unroll
                            for (int k8 = 0; k8 < count * (kSixteenCodes / 512); ++k8) {
                                four_copy16(to_k + copied + first * kSixteenCodes + 512 * k8, k + 512 * k8, id >= 0);
                                four_copy16(to_v + copied + first * kSixteenCodes + 512 * k8, v + 512 * k8, id >= 0);
                            }
                            if (scales)
                                four_copy16(to_scales + copied, w, id >= 0);
                        };
                        const uint32_t in = key_of(begin + i) & ((1 << c.page_shift) - 1);
                        const int      id = __shfl_sync(0xffffffffu, ids, i * kSixteens % 32);
                        const bool     scales = lane < 2 * kScaleBytes / 16;
                        if (kSixteens == 1 || c.page_shift > 4)
                            sixteens(id, in, 0, kSixteens, scales);
                        else {  // pages of sixteen positions
                            const int id2 = __shfl_sync(0xffffffffu, ids, i * kSixteens % 32 + 1);
                            sixteens(id, 0, 0, 1, scales && second == 0);
                            // (the second sixteen's scales are the first of their page)
                            sixteens(id2, 0, 1, 1, false);
                            if (scales && second == 1)
                                four_copy16(to_scales + copied, from_scales - kSixteenScales + static_cast<unsigned long long>(static_cast<uint32_t>(max(id2, 0) * c.kv_heads + head)) * page_bytes, id2 >= 0);
                        }
                        copied = copied == (kStages - 1) * kStageBytes ? 0 : copied + kStageBytes;
                    }
                    four_copies_done();
                };
                copied = 0;

                // ---- the rows: queries as the products' columns, and what they see
                uint32_t qf[TILES][4 * kGroups][2];
                float    qsum[TILES][kGroups][2];  // of a group's elements, of the rows whose scores the lane has
                int      limit[TILES][2], low[TILES][2];
                float    slope[TILES][2];
                // Keys from the one on (or sinks) and before the other are seen by all rows.
                const int seen_from = q.context + token1 - p.window + 1, seen_upto = q.context + token0 + 1;
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int gr = 0; gr < kGroups; ++gr) {
                        float sum = 0.0f;
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const uint4 x = q_raw[n][gr][w];
                            // Elements i and i + 4 of a word's eight are neighbours in the products: even ones, odd ones.
                            qf[n][4 * gr + 2 * w][0]     = __byte_perm(x.x, x.z, 0x5410);
                            qf[n][4 * gr + 2 * w][1]     = __byte_perm(x.y, x.w, 0x5410);
                            qf[n][4 * gr + 2 * w + 1][0] = __byte_perm(x.x, x.z, 0x7632);
                            qf[n][4 * gr + 2 * w + 1][1] = __byte_perm(x.y, x.w, 0x7632);
                            float e[8];
                            unpack_half8(x, e);
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                sum += e[k];
                        }
                        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                        qsum[n][gr][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                        qsum[n][gr][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * n + 2 * t + e, tok = four_token(p, row0 + min(r, rows - 1)), at_key = q.context + tok;
                        limit[n][e] = r < rows ? at_key + 1 : 0;
                        low[n][e]   = at_key - p.window + 1;
                        if constexpr (!PLAIN)
                            slope[n][e] = p.slopes && r < rows ? p.slopes[head * p.share + row0 + r - tok * p.share] * CUDART_L2E_F : 0.0f;
                    }
                }
                // Scores are sums in units of log 2 at once, an operation less for each: steps and sums of queries times the factor are off by
                // 2^-24 of a score, about as much as its sum in 32 bits is (of scores of 2^24 and more that is a power of two).
                const float factor = PLAIN ? p.scale * CUDART_L2E_F : p.cap > 0.0f ? 1.0f : p.scale * CUDART_L2E_F;
                const float cap_in = !PLAIN && p.cap > 0.0f ? p.scale / p.cap : 0.0f;
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int gr = 0; gr < kGroups; ++gr) {
                        qsum[n][gr][0] *= factor;
                        qsum[n][gr][1] *= factor;
                    }

                float acc[TILES][4 * kGroups][4];  // [elements 8 g + 2 k and (times 16) 8 g + 2 k + 1 of a group, k = 0..3][row]
                // A weight is rounded to fp16 for its product, and what that is off is multiplied by a code.  So that it is by a code
                // less 7.5, elements are (low + 7.5 step) + step (n - 7.5): `mids` adds up the first, `ones` what the second subtracts,
                // the rounded weights' sum, by a product with ones (0.0005 of the output instead of 0.0003).
                float ones[TILES][kGroups][4];
                float top[TILES][2], sum[TILES][2], mids[TILES][kGroups][2];
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
#pragma unroll
                    for (int m = 0; m < 4 * kGroups; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[n][m][e] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        top[n][e] = -CUDART_INF_F;
                        sum[n][e] = 0.0f;
#pragma unroll
                        for (int gr = 0; gr < kGroups; ++gr)
                            mids[n][gr][e] = ones[n][gr][e] = ones[n][gr][e + 2] = 0.0f;
                    }
                }
                // Steps of values are multiplied by `unit_v`, a power of two that makes the largest so far 2^5 to 2^6: with weights
                // up to 2^8, where a maximum lags, their products stay below 2^15, and hold all bits down to 2^-20 of the largest.
                float    unit_v = 1.0f;
                uint32_t limit_v = 0;  // fp16 bits of the largest step that may be: four times that, at most
                float    against[TILES][2] = {};  // the maximum, 0 where there is none
                uint32_t at_hand = 0;             // the block's place in the ring

                // The first steps only copy: code that is executed once costs its fetch, and this is not there twice.
#pragma unroll 1
                for (int i = 1 - kStages; i < end - begin; ++i) {
                    if (i >= 0) {
                        four_copies_wait<kStages - 2>();
                        __syncwarp();  // the block is there, and the one before it no longer read
                    }
                    copy(i + kStages - 1);
                    if (i < 0)
                        continue;
                    const unsigned char* const stage = ring_ptr + at_hand;
                    const int                  key0  = key_of(begin + i);
                    at_hand = at_hand == (kStages - 1) * kStageBytes ? 0 : at_hand + kStageBytes;

                    // ---- scores: keys g and g + 8 of each sixteen, rows 2 t and 2 t + 1 of each tile.  Odd codes are left where they
                    // are, four bits up: their products are sixteen times as large.
                    struct alignas(4 * kGroups) Scales {
                        half2 of[kGroups];
                    };
                    const unsigned char* const scales = stage + 2 * kCodeBytes;
                    float2                     s[kSixteens][TILES][2];  // [key g, g + 8], rows 2 t and 2 t + 1
#pragma unroll
                    for (int j = 0; j < kSixteens; ++j) {
                        float products[TILES][kGroups][2][4];  // [even codes, odd codes]
#pragma unroll
                        for (int gr = 0; gr < kGroups; ++gr) {
                            const unsigned char* const from = stage + j * kSixteenCodes + (at_k ^ 32 * gr);
                            const uint2 ka = *reinterpret_cast<const uint2*>(from), kb = *reinterpret_cast<const uint2*>(from + 8 * kRowBytes);
#pragma unroll
                            for (int w = 0; w < 2; ++w) {
                                const uint32_t a = w ? ka.y : ka.x, b2 = w ? kb.y : kb.x, a8 = a >> 8, b8 = b2 >> 8;
#pragma unroll
                                for (int odd = 0; odd < 2; ++odd) {
                                    const uint32_t mask = odd ? 0x00f000f0u : 0x000f000fu;
#pragma unroll
                                    for (int n = 0; n < TILES; ++n) {
                                        const uint32_t(&columns)[2] = qf[n][4 * gr + 2 * w + odd];
                                        if (w == 0)
                                            four_mma_first(products[n][gr][odd], a & mask, b2 & mask, a8 & mask, b8 & mask, columns[0], columns[1]);
                                        else
                                            four_mma(products[n][gr][odd], a & mask, b2 & mask, a8 & mask, b8 & mask, columns[0], columns[1]);
                                    }
                                }
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const Scales ks = *reinterpret_cast<const Scales*>(scales + j * kSixteenScales + (g + 8 * k) * (4 * kGroups));
#pragma unroll
                            for (int gr = 0; gr < kGroups; ++gr) {
                                const float2 scale = __half22float2(ks.of[gr]);
                                const float  step  = fmaf(scale.y, 0.0f, scale.x * (kOne * factor));  // no number unless both are
#pragma unroll
                                for (int n = 0; n < TILES; ++n) {
                                    const float(&even)[4] = products[n][gr][0], (&odd)[4] = products[n][gr][1];
                                    const float2 product = ptx::fma_x2(make_float2(odd[2 * k], odd[2 * k + 1]), make_float2(0.0625f, 0.0625f), make_float2(even[2 * k], even[2 * k + 1]));
                                    const float2 sums    = make_float2(qsum[n][gr][0], qsum[n][gr][1]);
                                    const float2 lowest  = make_float2(scale.y, scale.y);
                                    s[j][n][k] = ptx::fma_x2(product, make_float2(step, step), gr == 0 ? ptx::mul_x2(lowest, sums) : ptx::fma_x2(lowest, sums, s[j][n][k]));
                                }
                            }
                        }
                    }
                    if constexpr (!PLAIN) {
#pragma unroll
                        for (int j = 0; j < kSixteens; ++j)
#pragma unroll
                            for (int n = 0; n < TILES; ++n)
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    float2& x = s[j][n][k];
                                    if (p.cap > 0.0f)
                                        x = make_float2(four_capped(x.x, cap_in, p.cap * CUDART_L2E_F), four_capped(x.y, cap_in, p.cap * CUDART_L2E_F));
                                    const int key = key0 + j * kFourKeys + g + 8 * k;
                                    x.x           = fmaf(slope[n][0], static_cast<float>(key - limit[n][0] + 1), x.x);
                                    x.y           = fmaf(slope[n][1], static_cast<float>(key - limit[n][1] + 1), x.y);
                                }
                    }
                    Scales vs[kSixteens][2];
#pragma unroll
                    for (int j = 0; j < kSixteens; ++j)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            vs[j][k] = *reinterpret_cast<const Scales*>(scales + kScaleBytes + j * kSixteenScales + (g + 8 * k) * (4 * kGroups));
                    // ---- blocks that some row does not see all of (code by itself, not selections in all others)
                    uint32_t hidden  = 0;  // bit (j TILES + n) 4 + 2 k + row: the row does not see the key
                    bool     careful = false, grown = false;
                    auto     larger  = [&](uint32_t bits) { return bits - limit_v - 1u < 0x7c00u - limit_v; };  // and a number
                    if (key0 + kKeys > seen_upto || (key0 < seen_from && key0 + kKeys > p.sinks)) {
                        __syncwarp();
                        bool bad = false;
#pragma unroll
                        for (int j = 0; j < kSixteens; ++j)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int key = key0 + j * kFourKeys + g + 8 * k;
                                bool      any = false, all = true;  // of the lane's rows see it
#pragma unroll
                                for (int n = 0; n < TILES; ++n) {
                                    const bool x = key < limit[n][0] && (key >= low[n][0] || key < p.sinks);
                                    const bool y = key < limit[n][1] && (key >= low[n][1] || key < p.sinks);
                                    s[j][n][k].x = x ? s[j][n][k].x : -CUDART_INF_F;
                                    s[j][n][k].y = y ? s[j][n][k].y : -CUDART_INF_F;
                                    hidden |= (x ? 0u : 1u) << ((j * TILES + n) * 4 + 2 * k) | (y ? 0u : 2u) << ((j * TILES + n) * 4 + 2 * k);
                                    any = any || x || y;
                                    all = all && x && y;
                                }
#pragma unroll
                                for (int gr = 0; gr < kGroups; ++gr) {
                                    const float2 scale = __half22float2(vs[j][k].of[gr]);
                                    if (!any)  // what a key that nobody sees holds must not matter
                                        vs[j][k].of[gr] = __half2half2(__ushort_as_half(0));
                                    else if (!all && !(fabsf(scale.x) + fabsf(scale.y) < CUDART_INF_F))
                                        bad = true;  // nor one that only some see
                                    grown = grown || larger(__half_as_ushort(__low2half(vs[j][k].of[gr])));
                                }
                            }
                        careful = __any_sync(0xffffffffu, bad);
                    }
                    else {
#pragma unroll
                        for (int j = 0; j < (kSixteens * kFourKeys * kGroups + 31) / 32; ++j)  // (a lane looks at the step of a key and group)
                            grown = grown || larger(*reinterpret_cast<const uint32_t*>(scales + kScaleBytes + 4 * ((lane + 32 * j) % (kKeys * kGroups))) & 0xffffu);
                    }
                    // ---- a larger maximum, or larger steps, than the sums at hand are against: rarely after the first blocks
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        float2 most = make_float2(-CUDART_INF_F, -CUDART_INF_F);
#pragma unroll
                        for (int j = 0; j < kSixteens; ++j) {
                            most.x = fmaxf(most.x, fmaxf(s[j][n][0].x, s[j][n][1].x));
                            most.y = fmaxf(most.y, fmaxf(s[j][n][0].y, s[j][n][1].y));
                        }
                        grown = grown || most.x - top[n][0] > 8.0f || most.y - top[n][1] > 8.0f;  // (a sum with 8 may be rounded to the next number)
                    }
                    if (__any_sync(0xffffffffu, grown)) {
                        float largest = 0.0f;
#pragma unroll
                        for (int j = 0; j < kSixteens; ++j)
#pragma unroll
                            for (int k = 0; k < 2; ++k)
#pragma unroll
                                for (int gr = 0; gr < kGroups; ++gr)
                                    largest = fmaxf(largest, __low2float(vs[j][k].of[gr]));
#pragma unroll
                        for (int d = 1; d < 32; d <<= 1)
                            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, d));
                        float keep_v = 1.0f;
                        if (__half_as_ushort(__float2half_rn(largest)) > limit_v) {
                            const int   exponent = min((__float_as_int(largest) >> 23) - 127, 15);  // NaN has not become the largest
                            const float unit     = __int_as_float((127 + 5 - exponent) << 23);
                            keep_v               = unit / unit_v;  // (of lowest values there are sums before the first step)
                            unit_v               = unit;
                            limit_v              = __half_as_ushort(__float2half_rn(128.0f / unit));
                        }
#pragma unroll
                        for (int n = 0; n < TILES; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float newtop = top[n][e];
#pragma unroll
                                for (int j = 0; j < kSixteens; ++j)
#pragma unroll
                                    for (int k = 0; k < 2; ++k)
                                        newtop = fmaxf(newtop, e ? s[j][n][k].y : s[j][n][k].x);
#pragma unroll
                                for (int d = 4; d < 32; d <<= 1)
                                    newtop = fmaxf(newtop, __shfl_xor_sync(0xffffffffu, newtop, d));
                                const float keep = four_weight(top[n][e], newtop);
                                top[n][e]        = newtop;
                                against[n][e]    = newtop == -CUDART_INF_F ? 0.0f : -newtop;
                                sum[n][e] *= keep;
#pragma unroll
                                for (int gr = 0; gr < kGroups; ++gr) {
                                    mids[n][gr][e] *= keep * keep_v;
                                    ones[n][gr][e] *= keep * keep_v;
                                }
#pragma unroll
                                for (int m = 0; m < 4 * kGroups; ++m) {
                                    acc[n][m][e] *= keep * keep_v;
                                    acc[n][m][e + 2] *= keep * keep_v;
                                }
                            }
                    }
                    // ---- weights, times the steps of their values, as the second product's columns; outputs: elements 8 g + 2 k and
                    // 8 g + 2 k + 1 of each group, keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
                    for (int j = 0; j < kSixteens; ++j) {
                        uint32_t pf[TILES][kGroups][2];
#pragma unroll
                        for (int n = 0; n < TILES; ++n)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const float2 x = ptx::add_x2(s[j][n][k], make_float2(against[n][0], against[n][1]));
                                s[j][n][k]     = make_float2(ptx::exp2_approx(x.x), ptx::exp2_approx(x.y));
                                const float2 all = ptx::add_x2(make_float2(sum[n][0], sum[n][1]), s[j][n][k]);
                                sum[n][0] = all.x, sum[n][1] = all.y;
                            }
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int gr = 0; gr < kGroups; ++gr) {
                                const float2 scale = __half22float2(vs[j][k].of[gr]);
                                const float  step = scale.x * unit_v, mid = fmaf(7.5f, step, scale.y * unit_v);
#pragma unroll
                                for (int n = 0; n < TILES; ++n) {
                                    const float2 weights = s[j][n][k];
                                    float2       x = ptx::mul_x2(weights, make_float2(step, step)), all = make_float2(mids[n][gr][0], mids[n][gr][1]);
                                    if (careful) {
                                        __syncwarp();
                                        const uint32_t no = hidden >> ((j * TILES + n) * 4 + 2 * k);
                                        x     = make_float2(no & 1u ? 0.0f : x.x, no & 2u ? 0.0f : x.y);
                                        all.x = no & 1u ? all.x : fmaf(weights.x, mid, all.x);
                                        all.y = no & 2u ? all.y : fmaf(weights.y, mid, all.y);
                                    }
                                    else
                                        all = ptx::fma_x2(weights, make_float2(mid, mid), all);
                                    mids[n][gr][0] = all.x, mids[n][gr][1] = all.y;
                                    const half2 h = __floats2half2_rn(x.x, x.y);
                                    pf[n][gr][k]  = four_transpose(*reinterpret_cast<const uint32_t*>(&h));
                                }
                            }
#pragma unroll
                        for (int gr = 0; gr < kGroups; ++gr) {
                            uint32_t v[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                v[k] = *reinterpret_cast<const uint32_t*>(stage + j * kSixteenCodes + (at_v ^ 32 * gr) + 4 * k * kRowBytes);
#pragma unroll
                            for (int n = 0; n < TILES; ++n)
                                four_mma(ones[n][gr], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, pf[n][gr][0], pf[n][gr][1]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {  // a byte of each of two keys: two elements
                                const uint32_t x = __byte_perm(v[0], v[1], 0x0400 + 0x0101 * k), y = __byte_perm(v[2], v[3], 0x0400 + 0x0101 * k);
#pragma unroll
                                for (int n = 0; n < TILES; ++n)
                                    four_mma(acc[n][4 * gr + k], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, pf[n][gr][0], pf[n][gr][1]);
                            }
                        }
                    }
                }
                four_copies_wait<0>();
                __syncwarp();

                // ---- the end of the piece
                const bool     item = begin == 0 && end == sight.blocks;
                const unsigned kind = begin == 0 ? kPartBegins : end == sight.blocks ? kPartEnds : kPartContinues;
                const int      slot = kind == kPartBegins ? 1 : 0;
                float* const   to   = reinterpret_cast<float*>(slot ? ring_ptr : first_sums + warp * four_rows_bytes(HEAD_DIM, TILES));
                const float    back = 1.0f / unit_v;
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = 8 * n + 2 * t + e;
                        float     all_sum = sum[n][e];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1)
                            all_sum += __shfl_xor_sync(0xffffffffu, all_sum, d);
#pragma unroll
                        for (int gr = 0; gr < kGroups; ++gr) {
                            float low_sum = mids[n][gr][e];
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1)
                                low_sum += __shfl_xor_sync(0xffffffffu, low_sum, d);
                            low_sum = fmaf(-7.5f, ones[n][gr][e], low_sum);
                            float o[8];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                o[2 * k]     = fmaf(acc[n][4 * gr + k][e], kOne, low_sum) * back;
                                o[2 * k + 1] = fmaf(acc[n][4 * gr + k][e + 2], kOne / 16, low_sum) * back;
                            }
                            if (row >= rows)
                                continue;
                            const int column = gr * kFourBitGroup + 8 * g;
                            if (item) {
                                const uint2 x = four_outputs(make_float4(o[0], o[1], o[2], o[3]), all_sum), y = four_outputs(make_float4(o[4], o[5], o[6], o[7]), all_sum);
                                *reinterpret_cast<uint4*>(four_out<HEAD_DIM>(p, q.first, head, row0 + row) + column) = make_uint4(x.x, x.y, y.x, y.y);
                            }
                            else {
                                float4* const at4 = reinterpret_cast<float4*>(to + row * HEAD_DIM + column);
                                at4[0]            = make_float4(o[0], o[1], o[2], o[3]);
                                at4[1]            = make_float4(o[4], o[5], o[6], o[7]);
                            }
                        }
                        if (!item && g == 0)
                            sh.stats[warp][slot][row] = make_float2(top[n][e], all_sum);
                    }
                if (!item && lane == 0)
                    sh.part[warp][slot] = FourPart{kind, q.first, row0, rows, head, {0, 0, 0}};
                __syncwarp();
            }
            else if (begin > 0) {
                // A share so small that none of the item's blocks is its own: a part all the same, for the others' chain.
                float* const to = reinterpret_cast<float*>(first_sums + warp * four_rows_bytes(HEAD_DIM, TILES));
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

    four_finish<HEAD_DIM, kRows, kWarps>(p, sh, smem, kStages * kStageBytes, first_sums);
}

// Adds up the parts of the item that CTA blockIdx.x ended but did not begin, in key order.
template<int HEAD_DIM>
__global__ void __launch_bounds__(256) four_bit_join_kernel(const __grid_constant__ FourBitParams p)
{
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const FourPart* const parts = reinterpret_cast<const FourPart*>(p.workspace);
    const int             cta = blockIdx.x, lane = threadIdx.x & 31;
    // The CTA that began the item: the nearest before that did not only continue it.  (What tells is loaded at once: a call of few
    // sequences is a chain of such loads.)
    const FourPart last  = parts[2 * cta];
    int            begin = cta;
    unsigned       begun = 0;
    do {
        const int      c     = begin - 1 - lane;
        const unsigned kind  = c < 0 ? kPartNone : parts[2 * c].kind, next = c < 0 ? kPartNone : parts[2 * c + 1].kind;
        const unsigned other = __ballot_sync(0xffffffffu, kind != kPartContinues);
        begun                = __ballot_sync(0xffffffffu, next == kPartBegins);
        if (last.kind != kPartEnds)
            return;
        begin -= other ? __ffs(other) : 32;
        if (other) {
            begun = begun >> (__ffs(other) - 1) & 1u;
            break;
        }
    } while (true);
    if (begin < 0 || !begun)
        return;
    auto                slot  = [&](int i) { return static_cast<size_t>(2 * (begin + i) + (i == 0 ? 1 : 0)); };
    const float2* const stats = reinterpret_cast<const float2*>(p.workspace + four_stats_offset(gridDim.x));
    const float* const  sums  = reinterpret_cast<const float*>(p.workspace + four_sums_offset(gridDim.x));
    for (int u = threadIdx.x; u < last.rows * (HEAD_DIM / 4); u += blockDim.x) {
        const int    row = u / (HEAD_DIM / 4), column = u % (HEAD_DIM / 4) * 4;
        float2       all;
        const float4 o = four_add_up<8>(
            cta - begin + 1, p.unit, [&](int i) { return stats[slot(i) * 16 + row]; },
            [&](int i) { return reinterpret_cast<const float4*>(sums + (slot(i) * 16 + row) * HEAD_DIM + column); }, all);
        *reinterpret_cast<uint2*>(four_out<HEAD_DIM>(p, last.first, last.head, last.row0 + row) + column) = four_outputs(o, all.y);
    }
}

}  // namespace flashllm
