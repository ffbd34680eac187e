// Attention of a batch's tokens over a paged key/value cache that holds their own keys and values already.
//
//   s_ij = scale q_i . k_j,  capped: cap tanh(s_ij / cap),  then + slope_h (position_j - position_i)
//   o_i  = sum over the keys j that i sees of softmax_j(s_ij) v_j;  zero for a row that sees none
//
// What token i of a sequence (rows first + i, place context + i in the cache) sees: the whole context, and of the batch's own
// tokens either those up to itself and those of the prefix (prompts), or those whose bit its mask has (trees).  With a window
// it sees, of those up to itself, the last `window` and the first `sinks` of the sequence.
//
// One pass over the keys in tiles of 128 with the running maximum and sum of a softmax: S = Q K^T on the tensor cores, P =
// exp(S - maximum) in registers, one thread per row, rounded to fp16 (the type of the other operand of its product; kAttnWeightExponent
// says what that takes off a weight) and back to tensor memory, O += P V from there.  The query heads that share a key/value head
// are rows of one tile: row r of a sequence's (tokens x share) rows is token r / share, head r % share of the group.  A tile holds
// the rows of as many whole tokens as its 128 have room for: one tensor copy brings 64 columns of them.
//
// An item is two such tiles of one sequence and one key/value head.  Its two tiles of rows are two groups of softmax warps that
// take turns on the tensor core; an item of one tile (single tokens, drafted trees) is the same tile for both groups,
// each takes every other tile of keys, and the two results are joined at the end.  An item of at most 32 rows, which would leave
// one warp of four with all the work, lies in the tile four times: every warp has all rows and a quarter of the tile's keys
// (weights of zero for the others), and the joined results are eight.  The work of a call is the linear sequence
// of all items' tiles of keys, dealt out evenly over one CTA per SM whatever the sequences' lengths; an item that is cut leaves
// partial sums in the workspace, which attention_join_kernel adds up in key order.
#pragma once
#include <math_constants.h>

#include "cache_batch.cuh"
#include "four_bit_cache.cuh"
#include "tiling.h"

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
    unsigned char*            workspace;
    long long                 ld_q;
    int                       heads;
    int                       share;  // query heads per key/value head, and what divides by it: (mulhi(n, magic) + n) >> shift
    unsigned                  share_magic;
    int                       share_shift;
    int                       tile_rows;  // rows of a tile: whole tokens, at most 128
    int                       few_rows;   // ... at most 32; 0 where not one fits
    float                     scale;
    float                     cap;  // 0: none
    int                       window;  // keys up to itself that a row sees, kernels with a window alone
    int                       sinks;   // ... and of its sequence's first
    int                       least_rows;  // sequences with fewer rows (tokens x share) are somebody else's
};

// What follows from the heads: how rows are tokens and heads, and how many of them tiles hold (kAttnRows at most).
inline void attn_set_heads(AttentionParams* p, int heads, int kv_heads)
{
    p->heads          = heads;
    p->batch.kv_heads = kv_heads;
    p->share          = heads / kv_heads;
    p->tile_rows      = 128 / p->share * p->share;
    p->few_rows       = 32 / p->share * p->share;
    for (p->share_shift = 0; (1 << p->share_shift) < p->share;)
        ++p->share_shift;
    p->share_magic = static_cast<unsigned>(((1ull << 32) * ((1ull << p->share_shift) - p->share)) / p->share + 1);
}

// Token of a row of a sequence's (tokens x share) rows.
__device__ __forceinline__ int attn_token(const AttentionParams& p, int row)
{
    return static_cast<int>((__umulhi(static_cast<unsigned>(row), p.share_magic) + static_cast<unsigned>(row)) >> p.share_shift);
}

constexpr int kAttnKeys      = 128;  // keys per tile
constexpr int kAttnRows      = 128;  // rows per tile: one per lane of tensor memory
constexpr int kAttnSlotRows  = 2 * kAttnRows;  // rows that the workspace has room for in a part of an item
constexpr int kAttnMmaWarp   = 8;  // warps 0..3 and 4..7: the two groups of rows
constexpr int kAttnLoadWarp  = 9;
constexpr int kAttnHelpWarp  = 10;  // and 11
constexpr int kAttnThreads   = 12 * 32;
constexpr int kAttnTmemCols  = 512;
constexpr int kAttnKnown     = 512;  // sequences whose sizes are kept in shared memory from the plan on
constexpr int kAttnSegments  = 8;  // segments that shared memory holds at a time
// Registers of a thread, 256 x 208 + 128 x 88 = 384 x 168: a softmax thread keeps 64 plain scores of its row, or 32 that are masked,
// capped or biased, and what their transformation and the ends of an item (32 outputs of its row) take besides.
constexpr int kAttnSoftmaxRegisters = 208, kAttnOtherRegisters = 88;

// Over a cache of 4 bits four more warps turn codes into the elements that the products take.  256 x 152 + 128 x 104 + 128 x 104 = 512 x
// 128: what the softmax gives up costs it little, registers that the warps of products and work lack spill in their loops (a prompt of
// 7000 tokens, before other steps: 184, 64 and 80 registers 738 us, 168, 72 and 104 691, 160, 88 and 104 653, 152, 96 and 112 624).
constexpr int kAttnTurnWarp     = 12;
constexpr int kAttnFourThreads  = 16 * 32;
constexpr int kAttnFourSoftmaxRegisters = 152, kAttnFourOtherRegisters = 104, kAttnFourTurnRegisters = 104;

// Looks at a barrier before a CTA gives up: a second.  A look suspends the thread until the barrier changes, for 4.0 us at most
// (measured on B200).  (Counted and not timed: the waits stand in many places, and code that the instruction cache need not hold is
// time: ragged prompts 60 us with a clock in each, 55 without.)  A CTA that gave up leaves rows as they were, those of items that
// others share with it too; all other rows are right.
#ifndef FLASHLLM_ATTENTION_LOOKS  // the tests have a build that gives up early, elsewhere in each CTA
#define FLASHLLM_ATTENTION_LOOKS (1u << 18)
#define FLASHLLM_ATTENTION_LOOKS_AT_ONCE 32u
#define FLASHLLM_ATTENTION_LOOK ptx::mbar_try_wait
#endif

// Tiles of keys (and as many of values) in shared memory at a time.
__host__ __device__ constexpr int attn_stages(int head_dim)
{
    return head_dim == 128 ? 2 : 4;
}

__host__ __device__ constexpr int attn_tile_bytes(int head_dim)
{
    return kAttnKeys * head_dim * 2;
}

// What an item sees through a window.  Tiles of keys between the sinks and the window of its first row are left out: its tiles are
// numbered without them.
template<bool WINDOW>
struct AttnSight {};

template<>
struct AttnSight<true> {
    int sinks;
    int sink_tiles;  // tiles before those that are left out
    int skip;        // tiles that are left out
    int low[2];      // first key, sinks aside, that every row of a group sees: the last row's
};

// The part of an item that one CTA takes in one go.
template<bool WINDOW>
struct AttnSegmentOf : AttnSight<WINDOW> {
    int  b;
    int  first, count, context, prefix;  // of the sequence: first row, rows, position of the first row, keys that all see
    int  head;     // key/value head
    int  row0;     // first row of the item in the sequence's rows (tokens x share)
    int  rows;     // rows of the item
    int  keys;     // keys that any row of the item sees: none at or behind this
    int  open[2];  // keys that every row of a group sees: the first tile that needs a mask ends behind them
    int  tiles;    // of keys, the whole item
    int  begin;    // first tile of the segment
    int  end;      // behind its last; 0: no more segments
    int  tiles0;   // pair: tiles of keys that the first tile of rows needs
    bool pair;     // two tiles of rows; otherwise both groups share the one
    bool fourfold;  // few rows: four copies of them in the tile

    // Tiles of keys that a group goes through, and the i-th of them.
    __device__ __forceinline__ int count_of(int group) const
    {
        if (pair)
            return group == 0 ? max(min(end, tiles0) - begin, 0) : end - begin;
        return (end - begin + 1 - group) / 2;
    }
    __device__ __forceinline__ int tile(int group, int i) const
    {
        return pair ? begin + i : begin + group + 2 * i;
    }
    // First key of a tile.
    __device__ __forceinline__ int key_of(int tile) const
    {
        if constexpr (WINDOW)
            tile += tile < this->sink_tiles ? 0 : this->skip;
        return tile * kAttnKeys;
    }
    // Whether some row of the group does not see all of the tile that begins with that key (of the item: see `mixed`).
    __device__ __forceinline__ bool masked(int key0, int group) const
    {
        if constexpr (WINDOW)
            if (key0 < this->low[group] && key0 + kAttnKeys > this->sinks)
                return true;
        return key0 + kAttnKeys > open[group];
    }
    __device__ __forceinline__ bool mixed(int tile) const
    {
        const int key0 = key_of(tile);
        if constexpr (WINDOW)
            if (key0 < this->low[1] && key0 + kAttnKeys > this->sinks)
                return true;
        return key0 + kAttnKeys > open[0];
    }
    // Such tiles are few: the last three, and with a window the one that the sinks end in and the three that begin it (an item's
    // rows are at most 256 tokens).  Which of them a tile is, and back.
    static constexpr int kMixed = WINDOW ? 7 : 3;
    __device__ __forceinline__ int mixed_of(int tile) const
    {
        const int last = tiles - 1 - tile;
        if constexpr (WINDOW) {
            if (last < 3)
                return last;
            const int behind = tile - this->sink_tiles;
            return behind < 0 ? 3 : behind < 3 ? 4 + behind : kMixed;
        }
        return last < 3 ? last : kMixed;
    }
    __device__ __forceinline__ int tile_of(int mixed) const
    {
        if constexpr (WINDOW)
            if (mixed >= 3)
                return this->sink_tiles + mixed - 4;
        return tiles - 1 - mixed;
    }
};
using AttnSegment = AttnSegmentOf<false>;

// Dynamic shared memory: two tiles of Q, the stages, and what AttnShared holds.
template<bool WINDOW>
struct AttnSharedOf {
    unsigned long long k_full[4], k_empty[4], v_full[4], v_clean[4], v_empty[4];
    unsigned long long s_full[2], p_full[2][2], o_done[2], q_full[2], q_empty[2], segment_full[kAttnSegments];
    uint32_t           tmem;
    volatile uint32_t  abort_flag;
    // Written by the loader, which is ahead of everybody, by at most the stages and one: a segment's values cannot be loaded
    // before those of the one so many tiles earlier have been multiplied, and its place here is taken again only after
    // kAttnSegments more.
    AttnSegmentOf<WINDOW> segment[kAttnSegments];
    float              top[2][kAttnRows], sum[2][kAttnRows];
    uint32_t           any_not_finite[kAttnSegments];
    uint32_t           not_finite[kAttnSegments][AttnSegmentOf<WINDOW>::kMixed][4];  // keys of such tiles whose values are not finite
    int                drafted[2][kMaxDrafted];          // positions of drafted tokens, by group
    union {
        unsigned int units[kMaxSequences];  // of all items of a sequence's first key/value head; the plan's alone
        float4       staged[2][512];        // by group: outputs on their way out
    };
    int4               known[kAttnKnown];                // first row, rows, context and prefix of the first sequences
};
using AttnShared = AttnSharedOf<false>;

template<bool WINDOW = false>
__host__ __device__ constexpr int attn_smem_bytes(int head_dim)
{
    return (2 + 2 * attn_stages(head_dim)) * attn_tile_bytes(head_dim) + static_cast<int>(sizeof(AttnSharedOf<WINDOW>)) + 1024;
}

// The workspace: for each CTA two slots, the segment that continues an item that another CTA began, and the one that begins an
// item that another CTA continues.
constexpr unsigned kPartNone = 0, kPartBegins = 1, kPartContinues = 2, kPartEnds = 3;

struct AttnPart {
    unsigned kind;
    int      first;  // first row of the sequence in the batch
    int      row0;   // first row of the item in the sequence
    int      rows;   // rows of the item
    int      head;   // key/value head
    int      pad[3];
};

__host__ __device__ constexpr size_t attn_stats_offset(int ctas)
{
    return size_t(2) * ctas * sizeof(AttnPart);
}

__host__ __device__ constexpr size_t attn_sums_offset(int ctas)
{
    return attn_stats_offset(ctas) + size_t(2) * ctas * kAttnSlotRows * sizeof(float2);
}

// Sums lie as [slot][tile of rows][head_dim / 4][row] float4: a warp's rows are neighbours.
__host__ __device__ constexpr size_t attn_workspace_bytes(int ctas, int head_dim)
{
    return attn_sums_offset(ctas) + size_t(2) * ctas * kAttnSlotRows * head_dim * sizeof(float);
}

__device__ __forceinline__ bool attn_wait_longer(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, unsigned int* status)
{
#pragma unroll 1
    for (uint32_t it = 1;; ++it) {
        if (FLASHLLM_ATTENTION_LOOK(bar, parity))
            return true;
        if (it % FLASHLLM_ATTENTION_LOOKS_AT_ONCE == 0u) {
            if (it >= FLASHLLM_ATTENTION_LOOKS) {
                *abort_flag = 1u;
                atomicOr(status, kStatusWaitExpired);
            }
            if (*abort_flag)
                return false;
        }
    }
}

// A bounded wait; false once the CTA gives up.
template<bool WINDOW>
__device__ __forceinline__ bool attn_wait(const unsigned long long* barrier, uint32_t parity, AttnSharedOf<WINDOW>& sh, unsigned int* status)
{
    const uint32_t bar = ptx::smem_u32(barrier);
    return FLASHLLM_ATTENTION_LOOK(bar, parity) || attn_wait_longer(bar, parity, &sh.abort_flag, status);
}

// ---------------------------------------------------------------- the work of a call

// One sequence as the rows of its items see it.
struct AttnSequence {
    Sequence s;
    int      prefix;  // keys of the sequence that all of its rows see, beyond the context
    int      rows;    // count * share
};

template<bool WINDOW>
__device__ __forceinline__ AttnSequence attn_sequence(const AttentionParams& p, int b)
{
    AttnSequence a;
    a.s      = load_sequence(p.batch, b);
    if (WINDOW && a.s.count * p.share < p.least_rows)
        a.s.count = 0;
    a.prefix = p.prefix ? min(p.prefix[b], a.s.context + a.s.count) : 0;
    a.rows   = a.s.count * p.share;
    return a;
}

// ... what the plan has kept of it.
template<bool WINDOW>
__device__ __forceinline__ AttnSequence attn_sequence(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh, int b)
{
    if (b >= kAttnKnown)
        return attn_sequence<WINDOW>(p, b);
    const int4 known = sh.known[b];
    return AttnSequence{{known.x, known.y, known.z, 0}, known.w, known.y * p.share};
}

// Keys that rows before `row_end` (of the sequence's rows) see at most: no row sees the key of that index or one behind it.
__device__ __forceinline__ int attn_keys(const AttentionParams& p, const AttnSequence& a, int row_end)
{
    if (p.tree_mask)
        return a.s.context + min(a.s.count, kMaxDrafted);
    return max(a.s.context + attn_token(p, row_end - 1) + 1, a.prefix);
}

// Keys that all rows from `row` on see.
__device__ __forceinline__ int attn_open_keys(const AttentionParams& p, const AttnSequence& a, int row)
{
    return p.tree_mask ? a.s.context : max(a.s.context + attn_token(p, row) + 1, a.prefix);
}

__device__ __forceinline__ int attn_tiles(int keys)
{
    return (keys + kAttnKeys - 1) / kAttnKeys;
}

// What an item whose first row is `row` and whose rows see `keys` keys at most leaves out between sinks and window.
__device__ __forceinline__ void attn_set_sight(const AttentionParams& p, const AttnSequence& a, int row, int keys, AttnSight<true>& sight)
{
    const int first  = max(0, a.s.context + attn_token(p, row) - p.window + 1);
    sight.sinks      = p.sinks;
    sight.sink_tiles = attn_tiles(min(p.sinks, keys));
    sight.skip       = max(0, first / kAttnKeys - sight.sink_tiles);
}

// Tiles of keys of the item with rows `row` up to `row_end`.
template<bool WINDOW>
__device__ __forceinline__ int attn_item_tiles(const AttentionParams& p, const AttnSequence& a, int row, int row_end)
{
    const int keys = attn_keys(p, a, row_end);
    if constexpr (WINDOW) {
        AttnSight<true> sight;
        attn_set_sight(p, a, row, keys, sight);
        return attn_tiles(keys) - sight.skip;
    }
    return attn_tiles(keys);
}

// Beginning an item, and ending it, takes about as long as two of its tiles of keys, and as four where its groups share their rows
// and join their sums (us a call with 2 / 3 / 4 for all: decoding of 64 sequences 128 / 124 / 122, prompts with a prefix 73 / 76 /
// 79; with 4 / 5 for the latter alone: decoding 114 / 116): an item counts as so many units more than it has tiles when the work is dealt
// out.
__device__ __forceinline__ int attn_extra_units(const AttentionParams& p, int rows)
{
    return rows > p.tile_rows ? 2 : 4;
}

// The tile of an item with `tiles` before which unit x of it cuts it; no piece of `least` tiles or fewer is cut off.
__device__ __forceinline__ int attn_cut(int x, int tiles, int extra, int least)
{
    const int t = x - extra;
    return t >= tiles ? tiles : t <= least ? 0 : tiles - t <= least ? tiles : t;
}

// Where a CTA's share is but a few tiles, one for each group is the least that pays: a single tile is not cut off.  (Larger
// shares even out better with every cut where it falls: capped trees of 64 tokens 76 us, 80 with cuts moved by up to an eighth of
// the share.)
__device__ __forceinline__ int attn_least(unsigned long long share)
{
    return share <= 4 ? 1 : 0;
}

// Units of the item whose rows begin with row0 of the sequence's.
template<bool WINDOW>
__device__ __forceinline__ unsigned attn_units(const AttentionParams& p, const AttnSequence& a, int row0)
{
    const int end = min(row0 + 2 * p.tile_rows, a.rows);
    return static_cast<unsigned>(attn_item_tiles<WINDOW>(p, a, row0, end) + attn_extra_units(p, end - row0));
}

// The segment of that number, once the loader has written it; nullptr at the end and when the CTA gives up.
template<bool WINDOW>
__device__ __forceinline__ const AttnSegmentOf<WINDOW>* attn_segment(AttnSharedOf<WINDOW>& sh, int number, unsigned int* status)
{
    const int place = number % kAttnSegments;
    if (!attn_wait(&sh.segment_full[place], number / kAttnSegments & 1, sh, status) || sh.segment[place].end == 0)
        return nullptr;
    return &sh.segment[place];
}

// In place of a sequence's units: several items, to be counted by a warp; rows to be cleared; in the end, more than 32 bits hold.
constexpr unsigned kAttnSeveralItems = 0xffffffffu, kAttnLostRows = 0xfffffffeu, kAttnManyUnits = 0xffffffffu;

// A sum over a warp's lanes that 64 bits hold.
__device__ __forceinline__ unsigned long long attn_warp_sum(unsigned long long mine)
{
    const unsigned low = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(mine) & 0xffffffu);
    const unsigned mid = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(mine >> 24) & 0xffffffu);
    const unsigned top = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(mine >> 48));
    return low + (static_cast<unsigned long long>(mid) << 24) + (static_cast<unsigned long long>(top) << 48);
}

// Sums over a warp's lanes up to each lane.
template<typename COUNT>
__device__ __forceinline__ COUNT attn_warp_scan(COUNT mine)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const COUNT other = __shfl_up_sync(0xffffffffu, mine, d);
        if (lane >= d)
            mine += other;
    }
    return mine;
}

// Units of all items of a sequence's first key/value head, for a whole warp.  A sequence can have up to 2^49 of them, a call with
// all heads of all sequences more: a prompt of 2 million tokens with 64 heads has 2^32, some 80 seconds' work.
template<bool WINDOW>
__device__ __forceinline__ unsigned long long attn_sequence_units(const AttentionParams& p, const AttnSequence& a)
{
    const int          item_rows = 2 * p.tile_rows;
    unsigned long long mine      = 0;
#pragma unroll 1
    for (long long r = (threadIdx.x & 31) * item_rows; r < a.rows; r += 32 * item_rows)
        mine += attn_units<WINDOW>(p, a, static_cast<int>(r));
    return attn_warp_sum(mine);
}

// Units of every sequence; all threads, ends with a barrier.  The rows of a sequence that does not fit into the page table are
// cleared here, by one CTA.  Each sequence is one thread's, then one warp's: what stands in sh.units tells a warp whether it is to be
// counted and is overwritten with the count (kernels differ in their threads).
template<bool WINDOW>
__device__ __forceinline__ void attn_count_units(const AttentionParams& p, AttnSharedOf<WINDOW>& sh, int head_dim)
{
    const int B = p.batch.sequences, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int item_rows = 2 * p.tile_rows;
    bool      several   = false;
#pragma unroll 1
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        const AttnSequence a = attn_sequence<WINDOW>(p, b);
        if (b < kAttnKnown)
            sh.known[b] = make_int4(a.s.first, a.s.count, a.s.context, a.prefix);
        const unsigned units = a.s.lost > 0         ? kAttnLostRows
                               : a.rows == 0        ? 0u
                               : a.rows > item_rows ? kAttnSeveralItems
                                                    : attn_units<WINDOW>(p, a, 0);
        sh.units[b]          = units;
        several              = several || units >= kAttnLostRows;
    }
    if (__syncthreads_or(several ? 1 : 0)) {
#pragma unroll 1
        for (int b = warp; b < B; b += blockDim.x / 32) {
            if (sh.units[b] < kAttnLostRows)
                continue;
            const AttnSequence a = attn_sequence<WINDOW>(p, b);
            if (a.s.lost > 0 && b % gridDim.x == blockIdx.x) {
                const long long row = static_cast<long long>(p.heads) * head_dim;
#pragma unroll 1
                for (long long i = lane * 8; i < a.s.lost * row; i += 32 * 8)
                    *reinterpret_cast<uint4*>(p.out + a.s.first * row + i) = make_uint4(0, 0, 0, 0);
            }
            const unsigned long long units = attn_sequence_units<WINDOW>(p, a);
            __syncwarp();
            if (lane == 0)
                sh.units[b] = static_cast<unsigned>(min(units, static_cast<unsigned long long>(kAttnManyUnits)));
        }
        __syncthreads();
    }
}

// Where this CTA's share begins and how long it is, for a whole warp.
struct AttnStart {
    unsigned long long units;
    int                least, sequence, row0, head, unit;
};

// Units of this lane's sequence of the 32 from `base` on, first key/value head, for a whole warp.
template<bool WINDOW>
__device__ __forceinline__ unsigned long long attn_units_of(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh, int base)
{
    const int          b    = base + (threadIdx.x & 31);
    const unsigned     kept = b < p.batch.sequences ? sh.units[b] : 0;
    unsigned long long mine = kept;
#pragma unroll 1
    for (unsigned many = __ballot_sync(0xffffffffu, kept == kAttnManyUnits); many; many &= many - 1) {
        const int                at    = base + __ffs(many) - 1;
        const unsigned long long units = attn_sequence_units<WINDOW>(p, attn_sequence(p, sh, at));
        mine                           = b == at ? units : mine;
    }
    return mine;
}

// The item that holds unit u0 of the call.  COUNT holds all units: 32 bits if they do (small trees 12.2 us with 64 bits throughout,
// 11.9 with 32; capped trees of 64 tokens 73.8 and 72.7).
template<typename COUNT, bool WINDOW>
__device__ __forceinline__ void attn_find(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh, COUNT u0, AttnStart& start)
{
    const int   B = p.batch.sequences, lane = threadIdx.x & 31, item_rows = 2 * p.tile_rows;
    const COUNT heads = p.batch.kv_heads;
    // The sequence that holds it: the first whose running sum passes it.
    COUNT before = 0;
    int   b      = 0;
#pragma unroll 1
    for (int base = 0; base < B; base += 32) {
        COUNT mine;
        if constexpr (sizeof(COUNT) == 4)
            mine = base + lane < B ? sh.units[base + lane] * heads : 0;
        else
            mine = attn_units_of(p, sh, base) * heads;
        const COUNT    upto = attn_warp_scan(mine);
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > u0);
        if (past) {
            const int l = __ffs(past) - 1;
            b           = base + l;
            before += __shfl_sync(0xffffffffu, upto - mine, l);
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const AttnSequence a    = attn_sequence(p, sh, b);
    int                row0 = 0;
    unsigned           item = 1;
    if (a.rows <= item_rows)
        item = attn_units<WINDOW>(p, a, 0);
    else {
#pragma unroll 1
        for (long long base = 0;; base += 32 * item_rows) {  // ... and of its items the first
            const long long r    = base + lane * item_rows;
            const unsigned  size = r < a.rows ? attn_units<WINDOW>(p, a, static_cast<int>(r)) : 0;
            const COUNT     mine = size * heads, upto = attn_warp_scan(mine);
            const unsigned  past = __ballot_sync(0xffffffffu, before + upto > u0);
            if (past || base + 32 * item_rows >= a.rows) {
                const int l = past ? __ffs(past) - 1 : 0;
                row0        = static_cast<int>(base) + l * item_rows;
                item        = max(1u, __shfl_sync(0xffffffffu, size, l));
                before += __shfl_sync(0xffffffffu, upto - mine, l);
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    start.sequence = b;
    start.row0     = row0;
    start.head     = static_cast<int>((u0 - before) / item);
    start.unit     = static_cast<int>((u0 - before) % item);
}

// ... where 32 bits do not hold them: code of its own, out of the way of the usual calls'.
template<bool WINDOW>
__device__ __noinline__ AttnStart attn_start_many(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh)
{
    AttnStart          start{0, 0, 0, 0, 0, 0};
    unsigned long long total = 0;
#pragma unroll 1
    for (int base = 0; base < p.batch.sequences; base += 32)
        total += attn_units_of(p, sh, base) * p.batch.kv_heads;
    const unsigned long long units = attn_warp_sum(total), share = (units + gridDim.x - 1) / gridDim.x;
    const unsigned long long u0 = min(units, share * blockIdx.x), u1 = min(units, u0 + share);
    if (u1 > u0)
        attn_find<unsigned long long>(p, sh, u0, start);
    start.units = u1 - u0;
    start.least = attn_least(share);
    return start;
}

template<bool WINDOW>
__device__ __forceinline__ AttnStart attn_start(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh)
{
    const int          lane = threadIdx.x & 31;
    AttnStart          start{0, 0, 0, 0, 0, 0};
    unsigned long long total = 0;
#pragma unroll 1
    for (int b = lane; b < p.batch.sequences; b += 32)  // kAttnManyUnits among them makes many, too
        total += static_cast<unsigned long long>(sh.units[b]) * p.batch.kv_heads;
    const unsigned long long units = attn_warp_sum(total);
    if (units >= kAttnManyUnits)
        return attn_start_many(p, sh);
    const unsigned share = max(static_cast<unsigned>((units + gridDim.x - 1) / gridDim.x), 2u);  // a tile for each group
    const unsigned u0    = static_cast<unsigned>(min(units, static_cast<unsigned long long>(share) * blockIdx.x));
    const unsigned u1    = static_cast<unsigned>(min(units, static_cast<unsigned long long>(u0) + share));
    if (u1 > u0)
        attn_find<unsigned>(p, sh, u0, start);
    start.units = u1 - u0;
    start.least = attn_least(share);
    return start;
}

// Walks a CTA's share of the linear sequence of units, order (sequence, rows, key/value head, keys).
template<bool WINDOW>
struct AttnCursorOf {
    AttnSequence a;
    AttnSegmentOf<WINDOW> seg;
    unsigned long long left;
    int          next_unit;  // of the item
    int          extra;      // units of the item beyond its tiles
    int          least;      // tiles that are not cut off

    bool         new_sequence, new_rows;  // what `seg` does not describe yet

    __device__ __forceinline__ explicit AttnCursorOf(const AttnStart& start)
    {
        left         = start.units;
        least        = start.least;
        seg.b        = start.sequence;
        seg.row0     = start.row0;
        seg.head     = start.head;
        next_unit    = start.unit;
        new_sequence = true;
        new_rows     = false;
        seg.tiles    = 0x7fffff00;  // until the sequence is entered
        extra        = 0;
    }
    // The next segment that has a tile; its `end` is 0 at the end of the share.
    __device__ __forceinline__ void next(const AttentionParams& p, const AttnSharedOf<WINDOW>& sh)
    {
        do {
            if (next_unit >= seg.tiles + extra) {
                next_unit = 0;
                if (++seg.head == p.batch.kv_heads) {
                    seg.head = 0;
                    seg.row0 += 2 * p.tile_rows;
                    new_rows = true;
                    if (seg.row0 >= a.rows) {
                        seg.row0 = 0;
                        ++seg.b;
                        new_sequence = true;
                    }
                }
            }
            if (left > 0 && new_sequence) {
#pragma unroll 1
                for (;; ++seg.b) {
                    if (seg.b >= p.batch.sequences) {  // only if somebody writes the arrays during the call
                        left = 0;
                        break;
                    }
                    a = attn_sequence(p, sh, seg.b);
                    if (a.rows > 0)
                        break;
                }
                seg.first    = a.s.first;
                seg.count    = a.s.count;
                seg.context  = a.s.context;
                seg.prefix   = a.prefix;
                new_sequence = false;
                new_rows     = true;
            }
            if (left > 0 && new_rows) {
                const int end = min(seg.row0 + 2 * p.tile_rows, a.rows);
                seg.rows      = end - seg.row0;
                seg.pair      = seg.rows > p.tile_rows;
                seg.fourfold  = seg.rows <= p.few_rows;
                extra         = attn_extra_units(p, seg.rows);
                seg.keys      = attn_keys(p, a, end);
                seg.tiles     = attn_tiles(seg.keys);
                seg.tiles0    = seg.pair ? attn_tiles(attn_keys(p, a, seg.row0 + p.tile_rows)) : seg.tiles;
                if constexpr (WINDOW) {
                    attn_set_sight(p, a, seg.row0, seg.keys, seg);
                    const int low = seg.context - p.window + 1;  // of the sequence's first row
                    seg.tiles -= seg.skip;
                    seg.tiles0 -= seg.skip;
                    seg.low[1] = low + attn_token(p, end - 1);
                    seg.low[0] = seg.pair ? low + attn_token(p, seg.row0 + p.tile_rows - 1) : seg.low[1];
                }
                seg.open[0]   = attn_open_keys(p, a, seg.row0);
                seg.open[1]   = seg.pair ? attn_open_keys(p, a, seg.row0 + p.tile_rows) : seg.open[0];
                new_rows      = false;
            }
            seg.begin = seg.end = 0;
            if (left == 0)
                return;
            const int upto  = static_cast<int>(min(static_cast<unsigned long long>(seg.tiles + extra), next_unit + left));
            seg.begin       = attn_cut(next_unit, seg.tiles, extra, least);
            seg.end         = attn_cut(upto, seg.tiles, extra, least);
            left -= upto - next_unit;
            next_unit = upto;
        } while (seg.end == seg.begin);
    }
};
using AttnCursor = AttnCursorOf<false>;

// ---------------------------------------------------------------- masks

// The bits of 32 keys that lie before the n-th of them.
__device__ __forceinline__ uint32_t attn_bits_before(int n)
{
    return n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
}

// What a row sees.
template<bool WINDOW>
struct AttnRowOf;

template<>
struct AttnRowOf<true> {
    int limit;  // keys before this one that are
    int low;    // at or behind this one
    int sinks;  // or before this one

    __device__ __forceinline__ bool sees(int key) const { return key < limit && (key >= low || key < sinks); }
    __device__ __forceinline__ uint32_t word(int key0) const
    {
        return attn_bits_before(limit - key0) & (~attn_bits_before(low - key0) | attn_bits_before(sinks - key0));
    }
};

template<>
struct AttnRowOf<false> {
    int                limit;   // all keys before this one
    int                drafts;  // ... and, for trees, key drafts + i where bit i is set
    unsigned long long bits;

    __device__ __forceinline__ bool sees(int key) const
    {
        const int i = key - drafts;
        return key < limit || (i >= 0 && i < kMaxDrafted && (bits >> i & 1));
    }
    // Bit c: the row sees key `key0` + c.
    __device__ __forceinline__ uint32_t word(int key0) const
    {
        uint32_t  w = attn_bits_before(limit - key0);
        const int d = drafts - key0;
        if (d >= 0 && d < 32)
            w |= static_cast<uint32_t>(bits << d);
        else if (d < 0 && d > -kMaxDrafted)
            w |= static_cast<uint32_t>(bits >> -d);
        return w;
    }
};

__device__ __forceinline__ AttnRowOf<true> attn_row(const AttentionParams& p, const AttnSegmentOf<true>& seg, int row, bool valid)
{
    const int place = seg.context + (valid ? attn_token(p, row) : 0);
    return AttnRowOf<true>{valid ? place + 1 : 0, place - p.window + 1, p.sinks};
}

__device__ __forceinline__ AttnRowOf<false> attn_row(const AttentionParams& p, const AttnSegmentOf<false>& seg, int row, bool valid)
{
    AttnRowOf<false> r;
    r.limit  = 0;
    r.drafts = seg.context;
    r.bits   = 0;
    if (!valid)
        return r;
    const int token = attn_token(p, row);
    if (p.tree_mask) {
        r.limit = seg.context;
        r.bits  = p.tree_mask[seg.first + token];
        if (seg.count < kMaxDrafted)
            r.bits &= (1ull << seg.count) - 1;
    }
    else
        r.limit = max(seg.context + token + 1, seg.prefix);
    return r;
}

// ---------------------------------------------------------------- the kernel

__device__ __forceinline__ bool half_not_finite(uint32_t h)
{
    return (h & 0x7c00u) == 0x7c00u;
}

// Not zero if one of two halves is not finite.
__device__ __forceinline__ uint32_t halves_not_finite(uint32_t u)
{
    return ((u & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
}

// Two outputs as fp16.  Weights of 11 bits and their sum of 24 can take an average past the largest value that fp16 holds, which then
// is the average: only infinities become one.
__device__ __forceinline__ uint32_t attn_pack_bounded(float x, float y)
{
    auto bounded = [](float v) { return fabsf(v) < 131072.0f ? fminf(fmaxf(v, -65504.0f), 65504.0f) : v; };
    const half2 h = __floats2half2_rn(bounded(x), bounded(y));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Elements `column` up to `column` + 4 of a row of values.
template<int HEAD_DIM, bool FOUR_BIT>
__device__ __forceinline__ uint2 attn_values(const AttentionParams& p, long long row, int column)
{
    if constexpr (FOUR_BIT) {
        const unsigned char* const cache = reinterpret_cast<const unsigned char*>(p.v_cache);
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(cache + four_bit_codes<HEAD_DIM>(p.batch, row) + column / 8 * 4);
        const half2    scale = *reinterpret_cast<const half2*>(cache + four_bit_scales<HEAD_DIM>(p.batch, row) + column / kFourBitGroup * 4);
        const uint4    v     = four_bit_values<true>(codes, scale);
        return column % 8 == 0 ? make_uint2(v.x, v.y) : make_uint2(v.z, v.w);
    }
    return *reinterpret_cast<const uint2*>(p.v_cache + row * HEAD_DIM + column);
}

template<bool WINDOW>
using AttnList = uint32_t[AttnSegmentOf<WINDOW>::kMixed][4];

// Adds to o[c], element column + c of a row's output, the values that are not finite of keys that the row sees (the products
// took zeros in their place: a weight of zero times infinity is not zero).
template<int HEAD_DIM, bool FOUR_BIT, int COLUMNS, bool WINDOW>
__device__ __forceinline__ void attn_add_not_finite(const AttentionParams& p, const AttnSegmentOf<WINDOW>& seg,
                                                    const AttnRowOf<WINDOW>& row, const AttnList<WINDOW>& list, int column,
                                                    float (&o)[COLUMNS])
{
#pragma unroll 1
    for (int i = 0; i < 4 * AttnSegmentOf<WINDOW>::kMixed; ++i)
#pragma unroll 1
        for (uint32_t w = list[i / 4][i % 4]; w != 0; w &= w - 1) {
            const int key = seg.key_of(seg.tile_of(i / 4)) + 32 * (i % 4) + __ffs(w) - 1;
            if (!row.sees(key))
                continue;
            const long long at = cache_row(p.batch, seg.b, key, seg.head);
            if (at < 0)
                continue;
#pragma unroll
            for (int c = 0; c < COLUMNS; c += 4) {
                const uint2 v = attn_values<HEAD_DIM, FOUR_BIT>(p, at, column + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t h = (k < 2 ? v.x : v.y) >> (16 * (k & 1)) & 0xffffu;
                    if (half_not_finite(h))
                        o[c + k] += __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
                }
            }
        }
}

// The same for keys of tiles that all rows of the segment see, which the products take as they are: infinity times a weight of zero,
// another copy's key or one too small for fp16, has made NaN of the sums there.  Bits of columns `column` on that have a positive
// infinity or NaN among these keys, and a negative infinity or NaN; for a whole warp.
template<int HEAD_DIM, bool FOUR_BIT, int COLUMNS, bool WINDOW>
__device__ __forceinline__ uint2 attn_seen_not_finite(const AttentionParams& p, const AttnSegmentOf<WINDOW>& seg, int column)
{
    uint2     found = make_uint2(0u, 0u);
    const int end   = (WINDOW ? seg.end : min(seg.end, seg.open[0] / kAttnKeys)) * kAttnKeys;
#pragma unroll 4
    for (int place = seg.begin * kAttnKeys + (threadIdx.x & 31); place < end; place += 32) {
        if (WINDOW && seg.mixed(place / kAttnKeys))
            continue;
        const int       key = seg.key_of(place / kAttnKeys) + place % kAttnKeys;
        const long long at  = cache_row(p.batch, seg.b, key, seg.head);
        if (at < 0)
            continue;
#pragma unroll
        for (int c = 0; c < COLUMNS; c += 4) {
            const uint2 v = attn_values<HEAD_DIM, FOUR_BIT>(p, at, column + c);
            if (halves_not_finite(v.x) | halves_not_finite(v.y))
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    const uint32_t h = (k < 2 ? v.x : v.y) >> (16 * (k & 1)) & 0xffffu;
                    if (!half_not_finite(h))
                        continue;
                    const bool nan = (h & 0x3ffu) != 0u;
                    found.x |= nan || h < 0x8000u ? 1u << (c + k) : 0u;
                    found.y |= nan || h >= 0x8000u ? 1u << (c + k) : 0u;
                }
        }
    }
    return make_uint2(__reduce_or_sync(0xffffffffu, found.x), __reduce_or_sync(0xffffffffu, found.y));
}

template<int COLUMNS>
struct AttnSums {
    float o[COLUMNS];
};

// A row's sums of columns `column` on, put right where values are not finite; for a whole warp.  A row whose weights have no finite
// sum stays without a number.
template<int HEAD_DIM, bool FOUR_BIT, int COLUMNS, bool WINDOW>
__device__ __forceinline__ AttnSums<COLUMNS> attn_restore(const AttentionParams& p, const AttnSegmentOf<WINDOW>& seg,
                                                          const AttnRowOf<WINDOW>& row, const AttnList<WINDOW>& list, bool listed,
                                                          float sum, int column,
                                                          AttnSums<COLUMNS> sums)
{
    bool nan = false;
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
        nan = nan || sums.o[c] != sums.o[c];
    if (__any_sync(0xffffffffu, nan && sum == sum)) {
        const uint2 found = attn_seen_not_finite<HEAD_DIM, FOUR_BIT, COLUMNS>(p, seg, column);
#pragma unroll
        for (int c = 0; c < COLUMNS; ++c) {
            const float plus = found.x >> c & 1u ? CUDART_INF_F : 0.0f, minus = found.y >> c & 1u ? -CUDART_INF_F : 0.0f;
            sums.o[c]        = sums.o[c] == sums.o[c] ? sums.o[c] : plus + minus;
        }
    }
    if (listed)
        attn_add_not_finite<HEAD_DIM, FOUR_BIT, COLUMNS>(p, seg, row, list, column, sums.o);
    return sums;
}

// What the end of a segment adds up to a lane's row: its group's output and, where the groups share the rows, the other's.
struct AttnOutputs {
    uint32_t mine_tmem, other_tmem;  // of this warp's lanes
    float    mine_keep, other_keep;
    bool     mine, other;  // there at all

    // 16 columns from `c` on.
    __device__ __forceinline__ void load(int c, bool shared, float (&o)[16]) const
    {
        uint32_t x[16], y[16];
        ptx::tmem_ld_x16(mine_tmem + c, x);
        if (shared)
            ptx::tmem_ld_x16(other_tmem + c, y);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            asm volatile("" : "+r"(x[k]), "+r"(y[k]));
            o[k] = mine ? __uint_as_float(x[k]) * mine_keep : 0.0f;
            o[k] = other ? fmaf(__uint_as_float(y[k]), other_keep, o[k]) : o[k];
        }
    }
};

// The end of a segment for a warp with an output that is not finite, or may not be: its rows (`out` of a whole item's, or `sums` of a
// part's; neither for a lane without a row) are written anew.  Code of its own, out of the way of the usual ends: in their midst it
// cost ragged prompts 2 us of 55.
template<int HEAD_DIM, bool FOUR_BIT, bool WINDOW>
__device__ __noinline__ void attn_end_carefully(const AttentionParams& p, const AttnSegmentOf<WINDOW>& seg, const AttnRowOf<WINDOW> row,
                                                const AttnList<WINDOW>& list, bool listed, AttnOutputs outputs, float sum, int column0,
                                                int column1, half* out, float4* sums)
{
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
    for (int c = column0; c < column1; c += 16) {
        AttnSums<16> s;
        outputs.load(c, !seg.pair, s.o);
        s = attn_restore<HEAD_DIM, FOUR_BIT, 16>(p, seg, row, list, listed, sum, c, s);
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
            if (out)
                *reinterpret_cast<uint4*>(out + c + k) =
                    make_uint4(attn_pack_bounded(s.o[k] * inverse, s.o[k + 1] * inverse),
                               attn_pack_bounded(s.o[k + 2] * inverse, s.o[k + 3] * inverse),
                               attn_pack_bounded(s.o[k + 4] * inverse, s.o[k + 5] * inverse),
                               attn_pack_bounded(s.o[k + 6] * inverse, s.o[k + 7] * inverse));
            else if (sums) {
                sums[(c + k) / 4 * kAttnRows]     = make_float4(s.o[k], s.o[k + 1], s.o[k + 2], s.o[k + 3]);
                sums[(c + k + 4) / 4 * kAttnRows] = make_float4(s.o[k + 4], s.o[k + 5], s.o[k + 6], s.o[k + 7]);
            }
        }
    }
}

// ... of 4 columns of rows that lie in the tile four times, added up already.
template<int HEAD_DIM, bool FOUR_BIT, bool WINDOW>
__device__ __noinline__ AttnSums<4> attn_restore_four(const AttentionParams& p, const AttnSegmentOf<WINDOW>& seg,
                                                      const AttnRowOf<WINDOW> row, const AttnList<WINDOW>& list, bool listed, float sum,
                                                      int column, AttnSums<4> sums)
{
    return attn_restore<HEAD_DIM, FOUR_BIT, 4>(p, seg, row, list, listed, sum, column, sums);
}

// tanh x on [-0.75, 0.75] to 2.7e-7, rounding included: x times a polynomial in x^2, fitted to it for the smallest largest error
// (weights depend on the differences of scores; of a small score it is 2.9e-6).  A call has the coefficients times its cap.
constexpr float kAttnTanhRange = 0.75f;
constexpr int   kAttnTanhTerms = 5;
__device__ constexpr float kAttnTanh[kAttnTanhTerms] = {0.9999971985816956f, -0.33323076367378235f, 0.13226091861724854f, -0.04928046092391014f, 0.012318842113018036f};

// What a softmax thread keeps of its row from tile to tile, and what the transformation of its scores takes.
struct AttnState {
    float top, sum;      // the maximum that weights are taken against (of q.k, or of scores times log2 e), their sum
    float factor;        // what turns the scores at hand into powers of two
    float scale, cap;    // of scores in units of log 2; cap 0: none
    float cap_in;        // products times this are what the tanh takes
    float tanh[kAttnTanhTerms];  // cap times the polynomial's coefficients
    float slope;         // in units of log 2
    bool  biased;        // by slopes
    int   place;         // the row's position
    const int* drafted;  // positions of drafted tokens in shared memory, or nullptr
    bool  valid;         // the row is somebody's
    bool  far;           // a row of the warp has a maximum beyond kAttnFarExponent
};

// The largest of a row's scores, NaN if one of them is.
template<int COLUMNS>
__device__ __forceinline__ float attn_largest(const float (&s)[COLUMNS], float m0)
{
    float m[4] = {m0, s[1], s[2], s[3]};
    m[0]       = ptx::max3_nan(m0, s[0], s[0]);
#pragma unroll
    for (int c = 4; c < COLUMNS - 4; c += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            m[k] = ptx::max3_nan(m[k], s[c + k], s[c + 4 + k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        m[k] = ptx::max3_nan(m[k], s[COLUMNS - 4 + k], m[k]);
    return ptx::max3_nan(ptx::max3_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// 32 products of a row to scores in units of log 2, capped and biased: those with the keys from `key0` on.  `drafted`: keys at and
// behind `open` may stand elsewhere than they lie.
__device__ __forceinline__ void attn_transform(const AttnState& st, float (&s)[32], int key0, int open, bool drafted)
{
    if (st.cap > 0.0f) {
        // Scores are mostly small against the cap: then a polynomial, a third of the cost of two approximations by the special
        // function unit, which the weights need too.
        float2 largest = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            largest.x = ptx::max3_nan(largest.x, fabsf(s[c]), fabsf(s[c + 1]));
            largest.y = ptx::max3_nan(largest.y, fabsf(s[c + 2]), fabsf(s[c + 3]));
        }
        const float in = st.cap_in;
        if (__all_sync(0xffffffffu, !st.valid || ptx::max3_nan(largest.x, largest.y, largest.y) * in <= kAttnTanhRange)) {
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const float2 x = ptx::mul_x2(make_float2(s[c], s[c + 1]), make_float2(in, in)), y = ptx::mul_x2(x, x);
                float2       t = make_float2(st.tanh[kAttnTanhTerms - 1], st.tanh[kAttnTanhTerms - 1]);
#pragma unroll
                for (int k = kAttnTanhTerms - 2; k >= 0; --k)
                    t = ptx::fma_x2(t, y, make_float2(st.tanh[k], st.tanh[k]));
                t        = ptx::mul_x2(x, t);
                s[c]     = t.x;
                s[c + 1] = t.y;
            }
        }
        else {
            const float twice = 2.0f * CUDART_L2E_F * in;  // tanh x = 1 - 2 / (1 + e^2x), to some 2^-21
#pragma unroll
            for (int c = 0; c < 32; ++c)
                s[c] = fmaf(-2.0f * st.cap, ptx::rcp_approx(1.0f + ptx::exp2_approx(s[c] * twice)), st.cap);
        }
    }
    else {
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            const float2 t = ptx::mul_x2(make_float2(s[c], s[c + 1]), make_float2(st.scale, st.scale));
            s[c]           = t.x;
            s[c + 1]       = t.y;
        }
    }
    if (!st.biased)
        return;
    if (drafted) {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            const int key   = key0 + c, i = key - open;
            const int where = i >= 0 && i < kMaxDrafted ? st.drafted[i] : key;
            s[c]            = fmaf(st.slope, static_cast<float>(where - st.place), s[c]);
        }
    }
    else {
        const float  away  = st.slope * static_cast<float>(key0 - st.place);
        const float2 slope = make_float2(st.slope, st.slope), base = make_float2(away, away);
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            const float2 far = ptx::fma_x2(slope, make_float2(static_cast<float>(c), static_cast<float>(c + 1)), base);
            const float2 t   = ptx::add_x2(make_float2(s[c], s[c + 1]), far);
            s[c]             = t.x;
            s[c + 1]         = t.y;
        }
    }
}

// Minus infinity for the keys, from `key0` on, that the row does not see.
template<int COLUMNS, bool WINDOW>
__device__ __forceinline__ void attn_mask(const AttnRowOf<WINDOW>& row, float (&s)[COLUMNS], int key0)
{
#pragma unroll
    for (int k = 0; k < COLUMNS / 32; ++k) {
        const uint32_t seen = row.word(key0 + 32 * k);
#pragma unroll
        for (int c = 0; c < 32; ++c)
            s[32 * k + c] = seen >> c & 1u ? s[32 * k + c] : -CUDART_INF_F;
    }
}

// Where the maximum times `factor` is this large, its rounding takes a power of two and more off the weights, in the end all they have:
// then scores are taken against the maximum before they are multiplied.  One operation per pair of scores more; the code stands by
// itself.
constexpr float kAttnFarExponent = 8388608.0f;

// The maximum that weights are taken against, from the largest score of a tile.  `rescale(keep)` multiplies the row's output by
// `keep`, and is called by whole warps.
template<bool PLAIN, typename Rescale>
__device__ __forceinline__ void attn_new_top(AttnState& st, float new_top, bool first, Rescale&& rescale)
{
    auto far = [&]() {
        return PLAIN && __any_sync(0xffffffffu, st.valid && st.top != -CUDART_INF_F && fabsf(st.top) * st.factor > kAttnFarExponent);
    };
    if (!(new_top < CUDART_INF_F)) {  // a score that is no number, or infinity less itself: neither has the row's output a number
        st.sum  = CUDART_NAN_F;
        new_top = st.top;
    }
    if (first) {
        st.top = new_top;
        st.far = far();
    }
    else if (__any_sync(0xffffffffu, st.valid && (new_top - st.top) * st.factor > 8.0f)) {  // rows of nobody have no say
        // It moves only when it has grown by more than 2^8, which 32-bit sums and fp16 weights have room for: rarely after the
        // first tiles.
        const float keep = new_top == st.top ? 1.0f : ptx::exp2_approx((st.top - new_top) * st.factor);
        st.top           = new_top;
        st.sum *= keep;
        st.far = far();
        rescale(keep);
    }
}

// 32 scores to weights, rounded to fp16 in pairs; `part` takes their sums before the rounding.
template<bool PLAIN>
__device__ __forceinline__ void attn_weights(const float* s, float factor, float minus, float2 (&part)[2], uint32_t (&w)[16])
{
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        float2 x = make_float2(s[2 * k], s[2 * k + 1]);
        if constexpr (PLAIN)
            x = ptx::fma_x2(x, make_float2(factor, factor), make_float2(minus, minus));
        else
            x = ptx::add_x2(x, make_float2(minus, minus));
        x             = make_float2(ptx::exp2_approx(x.x), ptx::exp2_approx(x.y));
        part[k & 1]   = ptx::add_x2(part[k & 1], x);
        const half2 h = __floats2half2_rn(x.x, x.y);
        w[k]          = *reinterpret_cast<const uint32_t*>(&h);
    }
}

template<int COLUMNS>
__device__ __forceinline__ void attn_load_scores(uint32_t s_tmem, float (&s)[COLUMNS])
{
    uint32_t(&raw)[COLUMNS] = reinterpret_cast<uint32_t(&)[COLUMNS]>(s);
#pragma unroll
    for (int c = 0; c < COLUMNS; c += 32)
        ptx::tmem_ld_x32(s_tmem + c, raw + c);
    ptx::tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
        asm volatile("" : "+r"(raw[c]));  // not read before the wait
}

// Weights are 2^7 times what they are against the maximum: fp16 holds the largest, 2^15 where the maximum lags by 2^8, and those down
// to 2^-21 of it in full, down to 2^-32 at all.  Without the factor, which the sum has too, a long flat tail is lost: 40000 keys of 2^-26
// each are 6e-4 of the sum.
constexpr float kAttnWeightExponent = 7.0f;

// What is added to a score times `factor` to make the exponent of its weight; rounded down, so that no weight passes 2^15.
__device__ __forceinline__ float attn_minus(const AttnState& st)
{
    return st.top == -CUDART_INF_F ? 0.0f : __fmaf_rd(-st.top, st.factor, kAttnWeightExponent);
}

// Plain scores of one row in tensor memory, 128 of them, to weights there; their sum.  For a whole warp.
inline __device__ __noinline__ float attn_far_weights(uint32_t s_tmem, float top, float factor)
{
    const float minus = top == -CUDART_INF_F ? 0.0f : -top;
    float2      part  = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (int c = 0; c < kAttnKeys; c += 32) {  // weights take the place of scores already read
        float    s[32];
        uint32_t w[16];
        attn_load_scores(s_tmem + c, s);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            float2 x = ptx::add_x2(make_float2(s[2 * k], s[2 * k + 1]), make_float2(minus, minus));
            x        = ptx::fma_x2(x, make_float2(factor, factor), make_float2(kAttnWeightExponent, kAttnWeightExponent));
            x        = make_float2(ptx::exp2_approx(x.x), ptx::exp2_approx(x.y));
            part     = ptx::add_x2(part, x);

            const half2 h = __floats2half2_rn(x.x, x.y);
            w[k]          = *reinterpret_cast<const uint32_t*>(&h);
        }
        ptx::tmem_st_x16(s_tmem + c / 2, w);
    }
    return part.x + part.y;
}

// One tile of scores of one row, from tensor memory to weights there: all 128 of them, or, where the row lies in the tile four
// times, the 32 from `column` on and zeros for the others.  The tile's first key is `key0`; `masked` unless all rows see all of
// it, as keys before `open` are seen.  `part_done(half)` tells that the weights of that half of the tile are in place.
template<bool PLAIN, bool FOURFOLD, bool WINDOW, typename Rescale, typename PartDone>
__device__ __forceinline__ void attn_softmax(AttnState& st, const AttnRowOf<WINDOW>& row, uint32_t s_tmem, int column, int key0, int open,
                                             bool masked, bool first, Rescale&& rescale, PartDone&& part_done)
{
    float2     part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    auto       stored  = [&]() {
        ptx::tmem_wait_st();
        ptx::tc_fence_before_sync();
        __syncwarp();
    };
    if constexpr (FOURFOLD) {
        float s[32];
        attn_load_scores(s_tmem + column, s);
        if constexpr (!PLAIN)
            attn_transform(st, s, key0 + column, open, masked && st.drafted != nullptr);
        if (masked)
            attn_mask(row, s, key0 + column);
        attn_new_top<PLAIN>(st, attn_largest(s, st.top), first, rescale);
        if constexpr (PLAIN) {  // (as attn_far_weights, always)
            const float top = st.top == -CUDART_INF_F ? 0.0f : st.top;
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const float2 x = ptx::add_x2(make_float2(s[c], s[c + 1]), make_float2(-top, -top));
                s[c]           = x.x;
                s[c + 1]       = x.y;
            }
        }
        const float    minus     = PLAIN ? kAttnWeightExponent : attn_minus(st);
        const uint32_t zeros[16] = {0};
        uint32_t       w[16];
#pragma unroll
        for (int c = 0; c < kAttnKeys; c += 32)  // the other copies' keys
            if (c != column)
                ptx::tmem_st_x16(s_tmem + c / 2, zeros);
        attn_weights<PLAIN>(s, st.factor, minus, part, w);
        ptx::tmem_st_x16(s_tmem + column / 2, w);
        stored();
        part_done(0);
        part_done(1);
    }
    else {
        float new_top = st.top;
        if (PLAIN && !masked) {
            // 64 columns at a time: half the waits for loads of the other way, which has more to do per column (prompt of 7000 tokens
            // 444 us instead of 461, ragged prompts 55.0 instead of 55.7; all 128 in registers 467 and 60.9).
#pragma unroll 1
            for (int c = 0; c < kAttnKeys; c += 64) {
                float s[64];
                attn_load_scores(s_tmem + c, s);
                new_top = attn_largest(s, new_top);
            }
        }
        else {
            // 32 columns at a time, masked or transformed scores back to tensor memory in between: with all 128 in registers the code of
            // one tile does not fit the instruction cache (capped trees of 64 tokens took 90 us instead of 77, ragged prompts 71
            // instead of 60).
#pragma unroll 1
            for (int c = 0; c < kAttnKeys; c += 32) {
                float s[32];
                attn_load_scores(s_tmem + c, s);
                if constexpr (!PLAIN)
                    attn_transform(st, s, key0 + c, open, masked && st.drafted != nullptr);
                if (masked)
                    attn_mask(row, s, key0 + c);
                new_top = attn_largest(s, new_top);
                ptx::tmem_st_x32(s_tmem + c, reinterpret_cast<const uint32_t*>(s));
            }
            ptx::tmem_wait_st();
        }
        attn_new_top<PLAIN>(st, new_top, first, rescale);
        if (PLAIN && st.far) {
            st.sum += attn_far_weights(s_tmem, st.top, st.factor);
            stored();
            part_done(0);
            part_done(1);
            return;
        }
        // Weights take the place of scores already read.
        const float   minus    = attn_minus(st);
        constexpr int kColumns = PLAIN ? 64 : 32;
#pragma unroll (PLAIN ? 1 : 2)
        for (int c = 0; c < kAttnKeys; c += kColumns) {
            float s[kColumns];
            attn_load_scores(s_tmem + c, s);
#pragma unroll
            for (int k = 0; k < kColumns; k += 32) {
                uint32_t w[16];
                attn_weights<PLAIN>(s + k, st.factor, minus, part, w);
                ptx::tmem_st_x16(s_tmem + (c + k) / 2, w);
            }
            if ((c + kColumns) % 64 == 0) {
                stored();
                part_done(c / 64);
            }
        }
    }
    st.sum += (part[0].x + part[1].x) + (part[0].y + part[1].y);
}

// Warps 12 to 15 over a cache of 4 bits: a tile's codes to elements of fp16 in the stages of K and V, as the tensor copies would lay
// them.  Codes are read straight into registers, those of the next tile while this one's wait for its room: a thread has 32 elements
// of a key, neighbours have the rest of it and the keys behind.  Elements are rounded to fp16 once, as four_bit_read gives them: both
// operands of a product are of one type, and queries are fp16 (5.5e-4 of the output; 3e-4 where codes are multiplied as they are, which
// takes a product and a pass over its scores for each 64 elements and was not tried here).
template<int HEAD_DIM, bool WINDOW>
__device__ __forceinline__ void attn_turn_codes(const AttentionParams& p, AttnSharedOf<WINDOW>& sh, unsigned char* k_stages, unsigned char* v_stages)
{
    constexpr int kStages = attn_stages(HEAD_DIM), kTileBytes = attn_tile_bytes(HEAD_DIM), kBlock = kAttnKeys * 128;
    constexpr int kChunks = HEAD_DIM / 32, kRows = 32 / kChunks, kJobs = 32 / kRows;  // of 16 bytes of a key; keys of a job; jobs of a warp
    const CacheBatch& c = p.batch;
    const int warp = (threadIdx.x >> 5) - kAttnTurnWarp, lane = threadIdx.x & 31, q = lane % kChunks, r0 = 32 * warp + lane / kChunks;
    const uint32_t page_bytes = static_cast<uint32_t>(four_bit_row_bytes(HEAD_DIM)) << c.page_shift;
    const uint32_t scales_at  = static_cast<uint32_t>(HEAD_DIM / 2) << c.page_shift;
    const uint32_t offset     = (q >> 1) * kBlock + r0 * 128 + (((q & 1) * 4 + (q >> 1) * 2) ^ (r0 & 7)) * 16;
    uint32_t n  = 0;
    bool     ok = true;
#pragma unroll 1
    for (int number = 0;; ++number) {
        const AttnSegmentOf<WINDOW>* const current = attn_segment(sh, number, c.status);
        AttnList<WINDOW>& list = sh.not_finite[number % kAttnSegments];
        const int         t128 = threadIdx.x - kAttnTurnWarp * 32;
        if (t128 < 4 * AttnSegmentOf<WINDOW>::kMixed)
            (&list[0][0])[t128] = 0u;
        if (t128 == 0)
            sh.any_not_finite[number % kAttnSegments] = 0u;
        if (ptx::named_barrier_any(5, 128, current == nullptr || !ok))  // all or none
            break;
        const AttnSegmentOf<WINDOW>& seg = *current;
        const int* const table = c.page_table + static_cast<long long>(seg.b) * c.table_width;
        // Pages of the warp's two sixteens of keys, looked up a tile ahead of the loads that need them.
        auto pages = [&](int t, int (&ids)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = seg.key_of(t) + 32 * warp + 16 * h;
                ids[h]        = t < seg.end && key < seg.keys ? table[key >> c.page_shift] : 0;
            }
        };
        // Codes and scales of the thread's keys; zeros, which stand for zeros, where there are none.
        auto load = [&](const half* cache, int t, const int (&ids)[2], uint4 (&codes)[kJobs], half2 (&scale)[kJobs]) {
            const int key0 = seg.key_of(t) + 32 * warp;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int      id = ids[h], left = t < seg.end ? seg.keys - key0 - 16 * h : 0;  // keys of the sixteen that there are
                const bool     there = static_cast<unsigned>(id) < static_cast<unsigned>(c.pages);
                const uint32_t in = ((key0 + 16 * h) & ((1 << c.page_shift) - 1)) + lane / kChunks;
                const unsigned char* const page = reinterpret_cast<const unsigned char*>(cache) + static_cast<unsigned long long>(static_cast<uint32_t>(id) * c.kv_heads + seg.head) * page_bytes;
                const unsigned char* const from = page + in * (HEAD_DIM / 2) + 16 * q;
                const unsigned char* const from_scales = page + scales_at + in * (4 * four_bit_groups(HEAD_DIM)) + q / 2 * 4;
#pragma unroll
                for (int k = 0; k < kJobs / 2; ++k) {
                    const int j = h * (kJobs / 2) + k;
                    codes[j]    = make_uint4(0, 0, 0, 0);
                    scale[j]    = __float2half2_rn(0.0f);
                    if (there && lane / kChunks + kRows * k < left) {
                        codes[j] = *reinterpret_cast<const uint4*>(from + kRows * k * (HEAD_DIM / 2));
                        scale[j] = *reinterpret_cast<const half2*>(from_scales + kRows * k * (4 * four_bit_groups(HEAD_DIM)));
                    }
                }
                if (!there && left > 0)
                    atomicOr(c.status, kStatusBadCache);
            }
        };
        // Where the i-th eight elements of a job's keys go, and the word that has them: threads with a head's second 64 elements begin
        // with their third, for the banks.
        auto at = [&](unsigned char* stage, int j, int i) -> uint4& {
            return *reinterpret_cast<uint4*>(stage + (offset ^ 16 * i) + j * kRows * 128);
        };
        auto word = [&](const uint4& w, int i) {
            const uint32_t x = q < 2 ? (i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w) : (i == 0 ? w.z : i == 1 ? w.w : i == 2 ? w.x : w.y);
            return x;
        };
        auto turn = [&](unsigned char* stage, const uint4 (&codes)[kJobs], const half2 (&scale)[kJobs]) {
            half last = __ushort_as_half(0);  // the largest last element: see four_bit_values
#pragma unroll
            for (int j = 0; j < kJobs; ++j)
                last = __hmax(last, __hfma(__float2half_rn(15.0f), __low2half(scale[j]), __high2half(scale[j])));
            if (__any_sync(0xffffffffu, __half_as_ushort(last) == 0x7c00u)) {
#pragma unroll 1
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kJobs; ++j)
                        at(stage, j, i) = four_bit_values<true>(word(codes[j], i), scale[j]);
                return;
            }
#pragma unroll 1  // (whole 557 us, half of the words at a time 535, a word at a time 666)
            for (int half = 0; half < 4; half += 2)
#pragma unroll
                for (int j = 0; j < kJobs; ++j) {
                    const bool     second = (half == 0) != (q < 2);  // of the words' two halves
                    const uint32_t w0 = second ? codes[j].z : codes[j].x, w1 = second ? codes[j].w : codes[j].y;
                    at(stage, j, half)     = four_bit_values<false>(w0, scale[j]);
                    at(stage, j, half + 1) = four_bit_values<false>(w1, scale[j]);
                }
        };
        // A tile's keys, its values, the next tile's keys and so on through the same code: twice of it do not fit the instruction cache
        // beside the softmax's (a prompt of 7000 tokens 626 us, so 557).
        int   ids[2], ids_next[2];
        uint4 codes[kJobs], codes_next[kJobs];
        half2 scale[kJobs], scale_next[kJobs];
        pages(seg.begin, ids);
        load(p.k_cache, seg.begin, ids, codes, scale);
        load(p.v_cache, seg.begin, ids, codes_next, scale_next);
        pages(seg.begin + 1, ids_next);
        const int steps = 2 * (seg.end - seg.begin);
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            const int            which = step & 1, t = seg.begin + step / 2;
            const uint32_t       in = n + step / 2, stage = in % kStages, parity = (in / kStages & 1u) ^ 1u;
            unsigned char* const to = (which ? v_stages : k_stages) + stage * kTileBytes;
            ok = __all_sync(0xffffffffu, attn_wait(which ? &sh.v_empty[stage] : &sh.k_empty[stage], parity, sh, c.status));
            if (!ok)
                break;
            bool odd = false;
            if (which && seg.mixed(t)) {
#pragma unroll
                for (int j = 0; j < kJobs; ++j)
                    odd = odd || halves_not_finite(*reinterpret_cast<const uint32_t*>(&scale[j])) != 0u;
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd)
                turn(to, codes, scale);
            else {  // values that not all rows see, and that are not finite: zeros in their place
                const int mixed = seg.mixed_of(t);
#pragma unroll
                for (int j = 0; j < kJobs; ++j) {
                    const int  r   = r0 + kRows * j;
                    const bool bad = halves_not_finite(*reinterpret_cast<const uint32_t*>(&scale[j])) != 0u;
#pragma unroll 1
                    for (int i = 0; i < 4; ++i)
                        at(to, j, i) = bad ? make_uint4(0, 0, 0, 0) : four_bit_values<true>(word(codes[j], i), scale[j]);
                    if (bad && mixed < AttnSegmentOf<WINDOW>::kMixed) {
                        atomicOr(&list[mixed][r / 32], 1u << r % 32);
                        sh.any_not_finite[number % kAttnSegments] = 1u;
                    }
                }
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0)
                ptx::mbar_arrive(ptx::smem_u32(which ? &sh.v_clean[stage] : &sh.k_full[stage]));
#pragma unroll
            for (int j = 0; j < kJobs; ++j) {
                codes[j] = codes_next[j];
                scale[j] = scale_next[j];
            }
            if (which == 0) {
                ids[0] = ids_next[0];
                ids[1] = ids_next[1];
            }
            load(which ? p.v_cache : p.k_cache, t + 1, ids, codes_next, scale_next);
            if (which)
                pages(t + 2, ids_next);
        }
        n += steps / 2;
    }
}

// PLAIN: neither cap nor slopes.
template<int HEAD_DIM, bool PLAIN, bool WINDOW = false, bool FOUR_BIT = false>
__global__ void __launch_bounds__(FOUR_BIT ? kAttnFourThreads : kAttnThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q_few,
                 const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ AttentionParams p)
{
    constexpr int      kStages    = attn_stages(HEAD_DIM);
    constexpr int      kTileBytes = attn_tile_bytes(HEAD_DIM);
    constexpr int      kBlock     = kAttnKeys * 128;  // bytes of 64 columns of a tile
    constexpr int      kBlocks    = HEAD_DIM / 64;
    constexpr uint32_t kS = 0, kO = 256;  // tensor memory: scores (weights in their first half) and outputs, 128 columns a group
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw  = ptx::smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    const uint32_t       q_base = base, k_base = base + 2 * kTileBytes, v_base = k_base + kStages * kTileBytes;
    AttnSharedOf<WINDOW>& sh    = *reinterpret_cast<AttnSharedOf<WINDOW>*>(smem + (2 + 2 * kStages) * kTileBytes);
    unsigned int* const  status = p.batch.status;
    const int            warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            ptx::mbar_init(ptx::smem_u32(&sh.k_full[i]), FOUR_BIT ? 4 : 1);
            ptx::mbar_init(ptx::smem_u32(&sh.k_empty[i]), 1);
            ptx::mbar_init(ptx::smem_u32(&sh.v_full[i]), 1);
            ptx::mbar_init(ptx::smem_u32(&sh.v_clean[i]), FOUR_BIT ? 4 : 64);
            ptx::mbar_init(ptx::smem_u32(&sh.v_empty[i]), 1);
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(ptx::smem_u32(&sh.s_full[i]), 1);
            ptx::mbar_init(ptx::smem_u32(&sh.p_full[i][0]), 4);
            ptx::mbar_init(ptx::smem_u32(&sh.p_full[i][1]), 4);
            ptx::mbar_init(ptx::smem_u32(&sh.o_done[i]), 1);
            ptx::mbar_init(ptx::smem_u32(&sh.q_full[i]), 1);
            ptx::mbar_init(ptx::smem_u32(&sh.q_empty[i]), 1);
        }
#pragma unroll 1
        for (int i = 0; i < kAttnSegments; ++i)
            ptx::mbar_init(ptx::smem_u32(&sh.segment_full[i]), 1);
        sh.abort_flag = 0u;
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&map_q);
        ptx::prefetch_tensormap(&map_q_few);
        if constexpr (!FOUR_BIT) {
            ptx::prefetch_tensormap(&map_k);
            ptx::prefetch_tensormap(&map_v);
        }
    }
    if (warp == kAttnMmaWarp) {
        ptx::tmem_alloc(ptx::smem_u32(&sh.tmem), kAttnTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::grid_dependency_wait();
    ptx::tc_fence_before_sync();
    attn_count_units(p, sh, HEAD_DIM);
    ptx::tc_fence_after_sync();
    const uint32_t tmem = sh.tmem;
    if (threadIdx.x == 0)
        ptx::grid_launch_dependents();

    if (warp < kAttnMmaWarp)
        ptx::take_registers<FOUR_BIT ? kAttnFourSoftmaxRegisters : kAttnSoftmaxRegisters>();
    else if (FOUR_BIT && warp >= kAttnTurnWarp)
        ptx::give_registers<kAttnFourTurnRegisters>();
    else
        ptx::give_registers<FOUR_BIT ? kAttnFourOtherRegisters : kAttnOtherRegisters>();

    if (warp < kAttnMmaWarp) {
        // ================================================================ softmax: one thread per row
        const int       group = warp >> 2, thread = threadIdx.x & 127;
        const uint32_t  lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's lanes of tensor memory
        const uint32_t  s_tmem = tmem + kS + group * 128 + lanes, o_tmem = tmem + kO + group * 128 + lanes;
        uint32_t        s_parity = 0, o_parity = 0;  // phases of s_full and o_done
        AttnPart* const parts = reinterpret_cast<AttnPart*>(p.workspace) + 2 * blockIdx.x;
        bool            ok = true, written[2] = {false, false};
        for (int number = 0;; ++number) {
            const AttnSegmentOf<WINDOW>* const current = attn_segment(sh, number, status);
            // All or none: the barriers below count every thread of the two groups.
            if (ptx::named_barrier_any(1, 256, current == nullptr || !ok))
                break;
            ptx::tc_fence_after_sync();
            const AttnSegmentOf<WINDOW>& seg = *current;
            const bool         pair = seg.pair, fourfold = seg.fourfold;
            const int          in_tile = fourfold ? lane : thread, tile0 = pair ? group * p.tile_rows : 0;
            const int          row_id  = seg.row0 + tile0 + in_tile;  // of the sequence
            const int          rows    = min(seg.rows - tile0, p.tile_rows);
            const bool         valid   = in_tile < rows;
            const bool         busy    = (in_tile & ~31) < rows;  // the warp has a row
            const int          token   = valid ? attn_token(p, row_id) : 0;
            const int          head    = seg.head * p.share + (valid ? row_id - token * p.share : 0);
            const long long    in_row  = static_cast<long long>(head) * HEAD_DIM;
            const AttnRowOf<WINDOW> row = attn_row(p, seg, row_id, valid);
            const int open  = seg.open[group];
            const int tiles = seg.count_of(group);
            AttnState st{};
            st.top    = -CUDART_INF_F;
            st.valid  = valid;
            st.factor = PLAIN ? p.scale * CUDART_L2E_F : 1.0f;
            if constexpr (!PLAIN) {
                st.scale = p.scale * CUDART_L2E_F;
                st.cap    = p.cap * CUDART_L2E_F;
                st.cap_in = p.cap > 0.0f ? p.scale / p.cap : 0.0f;
#pragma unroll
                for (int k = 0; k < kAttnTanhTerms; ++k)
                    st.tanh[k] = kAttnTanh[k] * st.cap;
                st.place = seg.context + token;
                if (p.slopes) {
                    st.biased = true;
                    st.slope  = p.slopes[head] * CUDART_L2E_F;
                    if (p.tree_mask) {
                        st.place   = valid ? p.positions[seg.first + token] : 0;
                        st.drafted = sh.drafted[group];
                        if (thread < min(seg.count, kMaxDrafted))
                            sh.drafted[group][thread] = p.positions[seg.first + thread];
                        ptx::named_barrier_sync(2 + group, 128);  // the group's threads, none of which reads the last segment's any more
                    }
                }
            }
            auto rescale = [&](float keep) {  // the product before has ended: these scores come after it
#pragma unroll 1
                for (int c = 0; c < HEAD_DIM; c += 32) {
                    uint32_t o[32];
                    ptx::tmem_ld_x32(o_tmem + c, o);
                    ptx::tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        asm volatile("" : "+r"(o[k]));
                        o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                    }
                    ptx::tmem_st_x32(o_tmem + c, o);
                }
            };
            auto part_done = [&](int half_tile) {  // the product with the first 64 values may begin before the rest is there
                if (lane == 0)
                    ptx::mbar_arrive(ptx::smem_u32(&sh.p_full[group][half_tile]));
            };
            const int key_begin = seg.tile(group, 0) * kAttnKeys, key_step = (pair ? 1 : 2) * kAttnKeys;
            for (int i = 0; i < tiles; ++i) {
                const int  key0   = WINDOW ? seg.key_of(seg.tile(group, i)) : key_begin + i * key_step;
                const bool masked = WINDOW ? seg.masked(key0, group) : key0 + kAttnKeys > open;
                ok             = attn_wait(&sh.s_full[group], s_parity, sh, status) && ok;
                s_parity ^= 1u;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                ptx::tc_fence_after_sync();
                if (busy && !fourfold)
                    attn_softmax<PLAIN, false>(st, row, s_tmem, 0, key0, open, masked, i == 0, rescale, part_done);
                else if (fourfold)
                    attn_softmax<PLAIN, true>(st, row, s_tmem, thread & ~31, key0, open, masked, i == 0, rescale, part_done);
                else {
                    part_done(0);
                    part_done(1);
                }
            }
            if (tiles > 0) {
                ok = __all_sync(0xffffffffu, ok && attn_wait(&sh.o_done[group], o_parity, sh, status));
                o_parity ^= 1u;
            }
            ptx::tc_fence_after_sync();

            // ---- the end of the segment: what is added up to a row lies in up to eight places, 2 groups x 4 copies
            int   column0 = 0, column1 = HEAD_DIM;
            float keep = 1.0f, keep_other = 0.0f;  // on this group's output of this lane, on the other group's
            bool  join = false;
            if (!pair) {
                sh.top[group][thread] = st.top;
                sh.sum[group][thread] = st.sum;
                ptx::tc_fence_before_sync();
                ok = !ptx::named_barrier_any(1, 256, !ok);
                ptx::tc_fence_after_sync();
                const int step   = fourfold ? 32 : kAttnRows;
                float     newtop = -CUDART_INF_F, newsum = 0.0f;
#pragma unroll 1
                for (int r = fourfold ? lane : thread; r < kAttnRows; r += step)
                    newtop = fmaxf(newtop, fmaxf(sh.top[0][r], sh.top[1][r]));
                auto weight = [&](float top) { return top == newtop ? 1.0f : ptx::exp2_approx((top - newtop) * st.factor); };
#pragma unroll 1
                for (int r = fourfold ? lane : thread; r < kAttnRows; r += step)
                    newsum += sh.sum[0][r] * weight(sh.top[0][r]) + sh.sum[1][r] * weight(sh.top[1][r]);
                keep       = weight(st.top);
                keep_other = weight(sh.top[group ^ 1][thread]);
                join       = seg.count_of(1) > 0;
                st.top     = newtop;
                st.sum     = newsum;
                column0    = group * (HEAD_DIM / 2);
                column1    = column0 + HEAD_DIM / 2;
            }
            const bool      whole = seg.begin == 0 && seg.end == seg.tiles;
            const unsigned  kind  = whole ? kPartNone : seg.begin == 0 ? kPartBegins : seg.end == seg.tiles ? kPartEnds : kPartContinues;
            const int       slot  = kind == kPartBegins ? 1 : 0;
            const int       tile_row = pair ? group : 0;
            const long long to       = static_cast<long long>(seg.first + token) * p.heads * HEAD_DIM + in_row;
            float4* const   sums     = reinterpret_cast<float4*>(p.workspace + attn_sums_offset(gridDim.x))
                                 + (static_cast<size_t>(2 * blockIdx.x + slot) * 2 + tile_row) * (HEAD_DIM / 4) * kAttnRows;
            const AttnList<WINDOW>& list = sh.not_finite[number % kAttnSegments];
            const float inverse         = st.sum == 0.0f ? 0.0f : 1.0f / st.sum;
            const bool  any             = sh.any_not_finite[number % kAttnSegments] != 0;
            // An accumulator that no product has written may hold anything: this group's without a tile of its own, where the groups
            // share the rows the second group's with a single tile.
            const AttnOutputs outputs{o_tmem, tmem + kO + (group ^ 1) * 128 + lanes, keep, keep_other,
                                      pair ? tiles > 0 : group == 0 || join, !pair && (group == 1 || join)};
            if (fourfold) {
                float4* const staged = sh.staged[group];  // [4 x 4 columns][lane]
#pragma unroll 1
                for (int c = column0; c < column1; c += 16) {
                    float o[16];
                    outputs.load(c, true, o);
#pragma unroll
                    for (int k = 0; k < 16; k += 4)
                        staged[k / 4 * kAttnRows + thread] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    ptx::named_barrier_sync(2 + group, 128);
                    const int     column = c + 4 * (warp & 3);
                    const float4* four   = staged + (warp & 3) * kAttnRows + lane;
                    float         sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int copy = 0; copy < 4; ++copy) {
                        const float4 v = four[32 * copy];
                        sum4[0] += v.x, sum4[1] += v.y, sum4[2] += v.z, sum4[3] += v.w;
                    }
                    const float probe = (sum4[0] + sum4[1] + (sum4[2] + sum4[3])) * 0.0f;  // NaN if one of them is not finite
                    if (any || __any_sync(0xffffffffu, valid && probe != probe)) {
                        AttnSums<4> sums4;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            sums4.o[k] = sum4[k];
                        sums4 = attn_restore_four<HEAD_DIM, FOUR_BIT>(p, seg, row, list, any, st.sum, column, sums4);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            sum4[k] = sums4.o[k];
                    }
                    if (valid && ok && whole) {
                        *reinterpret_cast<uint2*>(p.out + to + column) =
                            make_uint2(attn_pack_bounded(sum4[0] * inverse, sum4[1] * inverse),
                                       attn_pack_bounded(sum4[2] * inverse, sum4[3] * inverse));
                    }
                    else if (valid && ok)
                        sums[column / 4 * kAttnRows + lane] = make_float4(sum4[0], sum4[1], sum4[2], sum4[3]);
                    ptx::named_barrier_sync(2 + group, 128);
                }
            }
            // Of the others 32 rows are written at a time, and written again if one of them is not finite.
            bool again = any;
            if (fourfold || !ok || !busy)
                again = false;
            else if (!any && pair && whole) {
                // 32 rows x 32 columns at a time through 2 KB of the warp's own, so that neighbouring lanes store neighbours
                uint4* const    staged = reinterpret_cast<uint4*>(sh.staged[group]) + (warp & 3) * 128;
                const long long mine   = valid ? to : -1;
                const int       r      = lane / 4;
                const long long at[4]  = {__shfl_sync(0xffffffffu, mine, r), __shfl_sync(0xffffffffu, mine, r + 8),
                                          __shfl_sync(0xffffffffu, mine, r + 16), __shfl_sync(0xffffffffu, mine, r + 24)};
                half2           largest = __float2half2_rn(0.0f);
#pragma unroll 1
                for (int c = 0; c < HEAD_DIM; c += 32) {
                    uint32_t x[32];
                    ptx::tmem_ld_x32(o_tmem + c, x);
                    ptx::tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        asm volatile("" : "+r"(x[k]));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const half2 h = __floats2half2_rn(__uint_as_float(x[8 * k + 2 * e]) * inverse,
                                                              __uint_as_float(x[8 * k + 2 * e + 1]) * inverse);
                            w[e]          = *reinterpret_cast<const uint32_t*>(&h);
                            largest       = __hmax2_nan(largest, __habs2(h));
                        }
                        staged[lane * 4 + (k ^ (lane >> 1 & 3))] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
                    uint4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[k] = staged[(8 * k + r) * 4 + ((lane ^ (r >> 1)) & 3)];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (at[k] >= 0)
                            *reinterpret_cast<uint4*>(p.out + at[k] + c + lane % 4 * 8) = v[k];
                    __syncwarp();
                }
                again = __any_sync(0xffffffffu, valid && halves_not_finite(*reinterpret_cast<const uint32_t*>(&largest)) != 0u);
            }
            else if (!any) {
                // 32 rows x 16 columns at a time through 1 KB of the warp's own, so that neighbouring lanes store neighbours
                uint4* const    staged = reinterpret_cast<uint4*>(sh.staged[group]) + (warp & 3) * 128;
                const long long mine   = valid ? to : -1;
                float           probe  = 0.0f;  // NaN if one of the row's sums is not finite
                half2           largest = __float2half2_rn(0.0f);
#pragma unroll 1
                for (int c = column0; c < column1; c += 16) {
                    float o[16];
                    outputs.load(c, !pair, o);
                    if (whole) {
#pragma unroll
                        for (int k = 0; k < 16; k += 8) {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {  // a row that sees no key: what its sums hold are zeros
                                const half2 h = __floats2half2_rn(o[k + 2 * e] * inverse, o[k + 2 * e + 1] * inverse);
                                w[e]          = *reinterpret_cast<const uint32_t*>(&h);
                                largest       = __hmax2_nan(largest, __habs2(h));
                            }
                            staged[lane * 2 + (k / 8 ^ (lane >> 2 & 1))] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int       r  = 16 * k + lane / 2;
                            const long long at = __shfl_sync(0xffffffffu, mine, r);
                            const uint4     v  = staged[r * 2 + ((lane ^ r >> 2) & 1)];
                            if (at >= 0)
                                *reinterpret_cast<uint4*>(p.out + at + c + lane % 2 * 8) = v;
                        }
                    }
                    else if (valid) {
#pragma unroll
                        for (int k = 0; k < 16; k += 4)
                            sums[(c + k) / 4 * kAttnRows + thread] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            probe = fmaf(o[k], 0.0f, probe);
                    }
                    __syncwarp();
                }
                const bool bad = probe != probe || halves_not_finite(*reinterpret_cast<const uint32_t*>(&largest)) != 0u;
                again          = __any_sync(0xffffffffu, valid && bad);
            }
            if (again)
                attn_end_carefully<HEAD_DIM, FOUR_BIT>(p, seg, row, list, any, outputs, st.sum, column0, column1,
                                             valid && whole ? p.out + to : nullptr, valid && !whole ? sums + thread : nullptr);
            if (ok && !whole && valid && column0 == 0 && (!fourfold || thread < 32))
                reinterpret_cast<float2*>(p.workspace + attn_stats_offset(gridDim.x))[static_cast<size_t>(2 * blockIdx.x + slot) * kAttnSlotRows
                                                                                      + tile_row * kAttnRows + thread] =
                    make_float2(st.top, st.sum);  // (times the factor it would lose what it differs by from others')
            if (kind != kPartNone) {
                written[slot] = true;
                const bool all = !ptx::named_barrier_any(1, 256, !ok);  // a part is there for all rows or for none
                if (threadIdx.x == 0)
                    parts[slot] = AttnPart{all ? kind : kPartNone, seg.first, seg.row0, seg.rows, seg.head, {0, 0, 0}};
            }
            // The barrier before the next segment: both groups are done with both outputs and with the joined sums' room.
            ptx::tc_fence_before_sync();
        }
        if (threadIdx.x == 0) {
            for (int slot = 0; slot < 2; ++slot)
                if (!written[slot])
                    parts[slot].kind = kPartNone;
        }
    }
    else if (warp == kAttnMmaWarp) {
        // ================================================================ products: one converged warp issues them all
        const uint32_t idesc_s = ptx::umma_idesc_f16_f32(kAttnRows, kAttnKeys);
        const uint32_t idesc_o = ptx::umma_idesc_f16_f32(kAttnRows, HEAD_DIM) | ptx::kUmmaBNMajor;
        const uint64_t q_desc = ptx::umma_desc_kmajor_sw128(q_base), k_desc = ptx::umma_desc_kmajor_sw128(k_base);
        const uint64_t v_desc  = ptx::umma_desc_nmajor_sw128(v_base, kBlock);
        uint32_t       loaded  = 0;  // tiles of keys before this segment
        uint32_t       q_parity = 0, p_parity = 0;
        bool           ok = true;
        // Both groups take the same code, parities of their barriers are the bits of a register: the instruction cache holds it more
        // often (code for each group: ragged prompts 64 us instead of 57).
        int  tiles0 = 0, tiles1 = 0;
        bool pair = false;
        auto have     = [&](const unsigned long long* barrier, uint32_t parity) {
            const uint32_t bar = ptx::smem_u32(barrier);  // one look first (prompt of 7000 tokens 438 us instead of 444)
            return __all_sync(0xffffffffu, FLASHLLM_ATTENTION_LOOK(bar, parity)) != 0
                   || __all_sync(0xffffffffu, attn_wait_longer(bar, parity, &sh.abort_flag, status)) != 0;
        };
        auto stage_of = [&](int group, int i) { return loaded + static_cast<uint32_t>(pair ? i : group + 2 * i); };
        const AttnSegmentOf<WINDOW>* current = nullptr;
#pragma unroll 1
        for (int number = 0; ok; ++number) {
            current = attn_segment(sh, number, status);
            if (__any_sync(0xffffffffu, current == nullptr))
                break;
            tiles0 = current->count_of(0);
            tiles1 = current->count_of(1);
            pair   = current->pair;
            const int length = current->end - current->begin;
            // Step i of a group: the product of its i-th weights and values, and the scores of its next tile; step -1 has no product.
#pragma unroll 1
            for (int i = -1; ok && (i < tiles0 || i < tiles1); ++i)
#pragma unroll 1
                for (int group = 0; ok && group < 2; ++group) {
                    const int tiles = group == 0 ? tiles0 : tiles1;
                    if (i >= tiles)
                        continue;
                    const uint32_t d = tmem + group * 128;
                    if (i >= 0) {
                        const uint32_t n = stage_of(group, i), stage = n % kStages, parity = p_parity >> group & 1u;
                        const uint64_t v = v_desc + stage * (kTileBytes >> 4);
                        ok = have(&sh.v_clean[stage], n / kStages & 1u) && have(&sh.p_full[group][0], parity);
                        if (!ok)
                            break;
                        ptx::tc_fence_after_sync();
                        ptx::umma_f16_ts_x4_elect(d + kO, d + kS, v, idesc_o, i > 0);
                        ok = have(&sh.p_full[group][1], parity);
                        if (!ok)
                            break;
                        ptx::tc_fence_after_sync();
                        ptx::umma_f16_ts_x4_elect(d + kO, d + kS + 32, v + (4 * 2048 >> 4), idesc_o, 1u);
                        p_parity ^= 1u << group;
                        // Scores that are complete mean that the product before them is: o_done tells of a segment's last alone.
                        if (i + 1 == tiles)
                            ptx::umma_commit_elect(ptx::smem_u32(&sh.o_done[group]));
                        if (!pair || group == 1)
                            ptx::umma_commit_elect(ptx::smem_u32(&sh.v_empty[stage]));
                    }
                    else if (pair || group == 0) {
                        if (tiles == 0)
                            continue;
                        ok = have(&sh.q_full[group], q_parity >> group & 1u);
                        q_parity ^= 1u << group;
                    }
                    if (!ok || i + 1 >= tiles)
                        continue;
                    const uint32_t n = stage_of(group, i + 1), stage = n % kStages;
                    const uint64_t q = q_desc + (pair ? group * (kTileBytes >> 4) : 0), k = k_desc + stage * (kTileBytes >> 4);
                    ok = have(&sh.k_full[stage], n / kStages & 1u);
                    if (!ok)
                        break;
                    ptx::tc_fence_after_sync();
#pragma unroll
                    for (int block = 0; block < kBlocks; ++block)
                        ptx::umma_f16_ss_x4_elect(d + kS, q + block * (kBlock >> 4), k + block * (kBlock >> 4), idesc_s, block > 0);
                    ptx::umma_commit_elect(ptx::smem_u32(&sh.s_full[group]));
                    if (!pair || group == 1)  // the last to need this tile of keys
                        ptx::umma_commit_elect(ptx::smem_u32(&sh.k_empty[stage]));
                    // Q's room is free for the next segment's after the group's last scores; where the groups share it, after the
                    // last of both (the groups take turns: the second's if their numbers are even, else the first's).
                    if (i + 2 == tiles && (pair || (tiles0 == tiles1) == (group == 1)))
                        ptx::umma_commit_elect(ptx::smem_u32(&sh.q_empty[pair ? group : 0]));
                }
            loaded += length;
        }
        __syncwarp();
    }
    else if (warp == kAttnLoadWarp) {
        // ================================================================ tiles of keys and values, one tensor copy per page and 64 columns
        const CacheBatch& c        = p.batch;
        const int         page     = 1 << c.page_shift;
        const int         box      = min(page, kAttnKeys);  // rows of a copy
        const int         pieces   = kAttnKeys / box;
        const int         piece    = lane / kBlocks, block = lane % kBlocks;
        const bool        active   = piece < pieces;
        const uint32_t    offset   = block * kBlock + piece * box * 128;
        AttnCursorOf<WINDOW> cursor(attn_start(p, sh));
        const AttnSegmentOf<WINDOW>& seg = cursor.seg;
        uint32_t          n        = 0;
        bool              ok       = true;
        for (int number = 0; ok; ++number) {
            cursor.next(p, sh);
            if (lane == 0) {
                sh.segment[number % kAttnSegments] = seg;
                ptx::mbar_arrive(ptx::smem_u32(&sh.segment_full[number % kAttnSegments]));
            }
            if (seg.end == 0)
                break;
            const int* table = c.page_table + static_cast<long long>(seg.b) * c.table_width;
            for (int t = seg.begin; ok && t < seg.end; ++t, ++n) {
                if constexpr (FOUR_BIT) {  // only as far ahead as the copies would be: the segments' places
                    ok = __all_sync(0xffffffffu, attn_wait(&sh.v_empty[n % kStages], (n / kStages & 1u) ^ 1u, sh, status));
                    continue;
                }
                const int key   = seg.key_of(t) + piece * box;
                int       z     = c.pages * c.kv_heads;  // behind the cache: reads as zeros
                if (active && key < seg.keys) {
                    const int id = table[key >> c.page_shift];
                    if (static_cast<unsigned>(id) < static_cast<unsigned>(c.pages))
                        z = id * c.kv_heads + seg.head;
                    else
                        atomicOr(status, kStatusBadCache);
                }
                const uint32_t stage = n % kStages, parity = (n / kStages & 1u) ^ 1u;
                for (int which = 0; which < 2; ++which) {
                    ok = attn_wait(which ? &sh.v_empty[stage] : &sh.k_empty[stage], parity, sh, status);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = ptx::smem_u32(which ? &sh.v_full[stage] : &sh.k_full[stage]);
                    if (lane == 0)
                        ptx::mbar_arrive_expect_tx(bar, kTileBytes);
                    __syncwarp();
                    if (active)
                        ptx::tma_load_3d((which ? v_base : k_base) + stage * kTileBytes + offset, which ? &map_v : &map_k, block * 64,
                                         key & (page - 1), z, bar);
                }
            }
        }
    }
    else if (FOUR_BIT && warp >= kAttnTurnWarp) {
        // ================================================================ codes to elements
        if constexpr (FOUR_BIT)
            attn_turn_codes<HEAD_DIM>(p, sh, smem + 2 * kTileBytes, smem + (2 + kStages) * kTileBytes);
    }
    else {
        // ================================================================ rows of Q, and values that no product may see
        const int t64         = threadIdx.x - kAttnHelpWarp * 32;
        uint32_t  n           = 0, q_parity[2] = {1, 1};
        bool      ok          = true;
        for (int number = 0;; ++number) {
            const AttnSegmentOf<WINDOW>* const current = attn_segment(sh, number, status);
            AttnList<WINDOW>& list = sh.not_finite[number % kAttnSegments];
            if (!FOUR_BIT && t64 < 4 * AttnSegmentOf<WINDOW>::kMixed)
                (&list[0][0])[t64] = 0u;
            if (!FOUR_BIT && t64 == 0)
                sh.any_not_finite[number % kAttnSegments] = 0u;
            if (ptx::named_barrier_any(4, 64, current == nullptr || !ok))  // all or none
                break;
            const AttnSegmentOf<WINDOW>& seg = *current;
            if (t64 == 0) {
                const CUtensorMap* map   = seg.fourfold ? &map_q_few : &map_q;
                const int          bytes = (seg.fourfold ? 4 * p.few_rows : p.tile_rows) * HEAD_DIM * 2;
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    if ((tile == 1 && !seg.pair) || seg.count_of(tile) == 0)
                        continue;
                    ok = ok && attn_wait(&sh.q_empty[tile], q_parity[tile], sh, status);
                    q_parity[tile] ^= 1u;
                    if (!ok)
                        continue;
                    const uint32_t bar   = ptx::smem_u32(&sh.q_full[tile]), dst = q_base + tile * kTileBytes;
                    const int      token = seg.first + attn_token(p, seg.row0 + tile * p.tile_rows);
                    ptx::mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
                    for (int block = 0; block < kBlocks; ++block)
                        for (int copy = 0; copy < (seg.fourfold ? 4 : 1); ++copy)
                            ptx::tma_load_3d(dst + block * kBlock + copy * 32 * 128, map, block * 64, seg.head * p.share, token, bar);
                }
            }
            for (int t = seg.begin; !FOUR_BIT && t < seg.end; ++t, ++n) {
                const uint32_t stage = n % kStages;
                ok                   = ok && attn_wait(&sh.v_full[stage], n / kStages & 1u, sh, status);
                if (!ok)  // nor without the rows of Q: those of the next segment would be taken for them
                    break;
                if (seg.mixed(t)) {
                    const int key0 = seg.key_of(t), mixed = seg.mixed_of(t);
#pragma unroll 1
                    for (int r = t64; r < kAttnKeys; r += 64) {
                        const int key = key0 + r;
                        uint4*    v   = reinterpret_cast<uint4*>(smem + (2 + kStages) * kTileBytes + stage * kTileBytes + r * 128);
                        bool      bad = false;
#pragma unroll 2
                        for (int x = 0; x < HEAD_DIM / 8; ++x) {
                            uint4& at = v[(x / 8) * (kBlock / 16) + ((x + r) & 7)];  // any order of chunks: banks
                            uint4  w  = key < seg.keys ? at : make_uint4(0, 0, 0, 0);
                            if (key >= seg.keys)
                                at = w;
                            else if (halves_not_finite(w.x) | halves_not_finite(w.y) | halves_not_finite(w.z) | halves_not_finite(w.w)) {
                                bad        = true;
                                auto clean = [&](uint32_t u) {
                                    return (half_not_finite(u) ? 0u : u & 0xffffu) | (half_not_finite(u >> 16) ? 0u : u & 0xffff0000u);
                                };
                                at = make_uint4(clean(w.x), clean(w.y), clean(w.z), clean(w.w));
                            }
                        }
                        if (bad && mixed < AttnSegmentOf<WINDOW>::kMixed) {
                            atomicOr(&list[mixed][r / 32], 1u << r % 32);
                            sh.any_not_finite[number % kAttnSegments] = 1u;
                        }
                    }
                    ptx::fence_proxy_async_smem();
                }
                ptx::mbar_arrive(ptx::smem_u32(&sh.v_clean[stage]));
            }
        }
    }

    if (sh.abort_flag) {  // copies and products already issued get a bounded chance to end before the CTA may exit
        const uint64_t t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 2000000ull) {}
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == kAttnMmaWarp)
        ptx::tmem_dealloc(tmem, kAttnTmemCols);
}

// Adds up the parts of the item that CTA blockIdx.x of the attention ended but did not begin, in key order, for 32 rows and all
// columns of it.
template<int HEAD_DIM>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttentionParams p, int ctas)
{
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const AttnPart* const parts = reinterpret_cast<const AttnPart*>(p.workspace);
    const float2* const   stats = reinterpret_cast<const float2*>(p.workspace + attn_stats_offset(ctas));
    const float4* const   sums  = reinterpret_cast<const float4*>(p.workspace + attn_sums_offset(ctas));
    const int             cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const AttnPart        last = parts[2 * cta];
    const int             place = blockIdx.y * 32 + lane;  // in a part: tile of rows, row of the tile
    const int             row   = place / kAttnRows * p.tile_rows + place % kAttnRows;  // of the item
    const bool            valid = place % kAttnRows < p.tile_rows && row < last.rows;
    if (last.kind != kPartEnds || !__any_sync(0xffffffffu, valid))
        return;
    // The CTA whose segment began the item: the nearest before that did not continue it.
    int begin = cta;
#pragma unroll 1
    do {
        const int c = begin - 1 - lane;
        const unsigned other = __ballot_sync(0xffffffffu, c < 0 || parts[2 * c].kind != kPartContinues);
        begin -= other ? __ffs(other) : 32;
        if (other)
            break;
    } while (true);
    if (begin < 0 || parts[2 * begin + 1].kind != kPartBegins)
        return;  // a CTA gave up
    // Maxima are of products where scores are plain, else of scores in units of log 2.
    const float unit = p.cap == 0.0f && p.slopes == nullptr ? p.scale * CUDART_L2E_F : 1.0f;
    auto        slot = [&](int c) { return static_cast<size_t>(2 * c + (c == begin ? 1 : 0)); };
    float       top  = -CUDART_INF_F;
    for (int c = begin; c <= cta; ++c)
        top = fmaxf(top, stats[slot(c) * kAttnSlotRows + place].x);
    constexpr int kPer = HEAD_DIM / 4 / 8;  // float4 columns of a warp
    float4        o[kPer];
    float         sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k)
        o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = begin; c <= cta; ++c) {
        const float2 stat = stats[slot(c) * kAttnSlotRows + place];
        // Never zero: a part's infinity stays one.
        const float  keep = stat.x == top ? 1.0f : fmaxf(ptx::exp2_approx((stat.x - top) * unit), 0x1p-126f);
        sum += stat.y * keep;
        const float4* src = sums + ((slot(c) * 2 + place / kAttnRows) * (HEAD_DIM / 4) + warp * kPer) * kAttnRows + place % kAttnRows;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const float4 v = src[k * kAttnRows];
            o[k].x         = fmaf(v.x, keep, o[k].x);
            o[k].y         = fmaf(v.y, keep, o[k].y);
            o[k].z         = fmaf(v.z, keep, o[k].z);
            o[k].w         = fmaf(v.w, keep, o[k].w);
        }
    }
    if (!valid)
        return;
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int   r       = last.row0 + row;
    half* out = p.out + (static_cast<long long>(last.first + attn_token(p, r)) * p.heads + last.head * p.share + r - attn_token(p, r) * p.share) * HEAD_DIM
                + warp * kPer * 4;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        *reinterpret_cast<uint2*>(out + 4 * k) = make_uint2(attn_pack_bounded(o[k].x * inverse, o[k].y * inverse),
                                                            attn_pack_bounded(o[k].z * inverse, o[k].w * inverse));
    }
}

}  // namespace flashllm
