// The attention's division of a call's work among its CTAs, by itself: what each CTA would take, without taking it.  It reads a
// batch's lengths alone, so a test can ask for sizes whose caches no GPU holds.  Built as build/libattention_plan.so.
#include <cuda.h>

#include "../flash-llm_b200/csrc/attention_kernel_sm100.cuh"

using namespace flashllm;

struct PlanCta {
    long long tiles, segments;                       // of keys; pieces of items
    int       b0, row0, head0, begin0;               // where the first piece begins
    int       b1, row1, head1, end1, tiles1, rows1;  // where the last ends: in which item, before which of its tiles, its rows
};

__global__ void __launch_bounds__(kAttnThreads, 1) plan_kernel(const __grid_constant__ AttentionParams p, PlanCta* out)
{
    extern __shared__ __align__(16) unsigned char raw[];
    AttnShared& sh = *reinterpret_cast<AttnShared*>(raw);
    attn_count_units(p, sh, 128);
    if (threadIdx.x >> 5 != kAttnLoadWarp)
        return;
    AttnCursor         cursor(attn_start(p, sh));
    const AttnSegment& seg = cursor.seg;
    PlanCta            cta{};
    for (;;) {
        cursor.next(p, sh);
        if (seg.end == 0)
            break;
        if (cta.segments++ == 0)
            cta.b0 = seg.b, cta.row0 = seg.row0, cta.head0 = seg.head, cta.begin0 = seg.begin;
        cta.b1 = seg.b, cta.row1 = seg.row0, cta.head1 = seg.head, cta.end1 = seg.end, cta.tiles1 = seg.tiles, cta.rows1 = seg.rows;
        cta.tiles += seg.end - seg.begin;
    }
    if ((threadIdx.x & 31) == 0)
        out[blockIdx.x] = cta;
}

// Device arrays as the operators take them; `out` holds `ctas` PlanCta, `status` one word.
extern "C" int attention_plan(int ctas, const int* cu_tokens, const int* context, const int* prefix, int table_width, int page_shift,
                              int sequences, int tokens, int heads, int kv_heads, unsigned int* status, void* out)
{
    AttentionParams p{};
    p.batch.cu_tokens   = cu_tokens;
    p.batch.context     = context;
    p.batch.status      = status;
    p.batch.sequences   = sequences;
    p.batch.tokens      = tokens;
    p.batch.table_width = table_width;
    p.batch.page_shift  = page_shift;
    p.batch.pages       = 1;
    p.prefix            = prefix;
    attn_set_heads(&p, heads, kv_heads);
    const int   smem = static_cast<int>(sizeof(AttnShared));
    cudaError_t err  = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err == cudaSuccess) {
        plan_kernel<<<ctas, kAttnThreads, smem>>>(p, static_cast<PlanCta*>(out));
        err = cudaGetLastError();
    }
    if (err == cudaSuccess)
        err = cudaDeviceSynchronize();
    return static_cast<int>(err);
}
