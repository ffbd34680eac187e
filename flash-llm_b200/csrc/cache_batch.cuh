// A paged key/value cache and the batch of sequences that a call works on, as the kernels see them.
//
// A cache tensor is [pages][kv_heads][page_size][head_dim] fp16: what one head keeps of one page lies in one piece, so that a
// tensor copy of a page's rows of one head reads whole lines.  Position j of sequence b lives in place j % page_size of page
// page_table[b][j / page_size].  Tokens of the batch lie one behind another: sequence b owns rows cu_tokens[b] up to
// cu_tokens[b + 1], and its first row stands at position context[b].  Rows behind the last sequence belong to nobody.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace flashllm {

// A page id outside the cache, a length that does not fit into the page table, or an accepted token that the sequence does not
// have: such keys read as zeros, such tokens are not written.
constexpr unsigned kStatusBadCache = 64u;

constexpr int kMaxDrafted   = 64;    // drafted tokens of a sequence that a tree mask can name
constexpr int kMaxSequences = 4096;  // sequences of a call

struct CacheBatch {
    const int*    cu_tokens;   // [sequences + 1]
    const int*    context;     // [sequences]
    const int*    page_table;  // [sequences][table_width]
    unsigned int* status;
    int           sequences;
    int           tokens;  // rows of the batch
    int           table_width;
    int           pages;
    int           page_shift;  // log2 of the page size
    int           kv_heads;
};

// Sequence b's rows and first position, made to fit the batch and the page table whatever the arrays hold.
struct Sequence {
    int first;    // first row
    int count;    // rows; 0 for a sequence that does not fit
    int context;  // position of the first row
    int lost;     // rows of a sequence that does not fit
};

__device__ __forceinline__ long long table_positions(const CacheBatch& c)
{
    return static_cast<long long>(c.table_width) << c.page_shift;
}

__device__ __forceinline__ Sequence load_sequence(const CacheBatch& c, int b)
{
    const int begin = c.cu_tokens[b], end = c.cu_tokens[b + 1], context = c.context[b];
    Sequence  s;
    s.first   = min(max(begin, 0), c.tokens);
    s.count   = min(max(end, s.first), c.tokens) - s.first;
    s.context = context;
    s.lost    = 0;
    if (context < 0 || static_cast<long long>(context) + s.count > table_positions(c)) {
        if (s.count > 0)
            atomicOr(c.status, kStatusBadCache);
        s.lost    = s.count;
        s.count   = 0;
        s.context = 0;
    }
    return s;
}

// Row (in elements of head_dim) of a position's page entry and head in a cache tensor, or -1.
__device__ __forceinline__ long long cache_row(const CacheBatch& c, int b, int position, int head)
{
    const int page = c.page_table[static_cast<long long>(b) * c.table_width + (position >> c.page_shift)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages)) {
        atomicOr(c.status, kStatusBadCache);
        return -1;
    }
    return ((static_cast<long long>(page) * c.kv_heads + head) << c.page_shift) + (position & ((1 << c.page_shift) - 1));
}

}  // namespace flashllm
