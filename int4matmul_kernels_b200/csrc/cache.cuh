// What the kernels of the paged 8-bit key-value cache share: its geometry and the bytes' two codings.
//
// A byte q of a page and head stands for q * scale.  int8: q in [-127, 127] (the writer leaves -128 unused); e4m3: 4 exponent and 3
// mantissa bits, largest 448, no infinities.  Both convert to fp16 without rounding, which is what the attention kernels multiply with.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace i4mm {

struct CacheView {
    uint8_t* k;
    uint8_t* v;
    float2* scales;                                   // [page][head]: of keys, of values
    long long k_page, k_head, k_token;                // strides in bytes
    long long v_page, v_head, v_token;
    int pages, heads;
    int page_shift;                                   // log2(tokens of a page), 4 .. 7
    int dim;                                          // 64 or 128
};

// rows of activations (tokens, heads, dim): strides in elements, a multiple of 8 (16 bytes)
struct RowsView {
    const void* p;
    long long token, head;
};

struct PlanParams {
    const int* seq_lens;
    const int* new_lens;
    int* table;
    int* free_pages;
    const int* free_count;
    int *lens_after, *cu_lens, *slots, *positions, *request_of, *counts;
    long long table_stride;
    int requests, table_width, free_capacity, page_shift, max_tokens;
};

struct AttentionParams {
    CacheView cache;
    RowsView q;
    void* out;                                        // (tokens, q_heads, dim) contiguous
    const int* table;
    const int* seq_lens;
    const int* cu_lens;                               // or nullptr: one row for each request
    void* workspace;
    size_t prompt_parts;                              // where in it the prompt kernel's parts lie
    long long table_stride;
    int table_width, requests, tokens, q_heads, group; // group = q_heads / cache.heads
    int window;                                       // 0: none
    float scale;
};

cudaError_t cache_plan_launch(const PlanParams& p, cudaStream_t stream);
cudaError_t cache_write_launch(const CacheView& c, bool e4m3, const RowsView& k, const RowsView& v, bool bf16, int tokens, const int* slots,
                               cudaStream_t stream);
cudaError_t cache_read_launch(const CacheView& c, bool e4m3, void* k_out, void* v_out, bool bf16, int tokens, const int* slots,
                              cudaStream_t stream);

}  // namespace i4mm
