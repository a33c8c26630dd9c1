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
    size_t prompt_parts, prefix_parts;                // where in it the prompt kernel's and the prefix kernel's parts lie
    long long table_stride;
    int table_width, requests, tokens, q_heads, group; // group = q_heads / cache.heads
    int window;                                       // 0: none
    float scale;
    // shared prefixes (`shared` below): of request b, the place of the batch whose tokens come before its own, or -1; the list of the
    // rows that read place p is rows[starts[p]] .. rows[starts[p + 1] - 1]
    const int* prefix_of;
    const int* prefix_starts;
    const int* prefix_rows;
    int prefix_listed;                                // entries of the list
    // what the rows' prefixes come to, by packed row and head: (m, sum of 2^(s - m)) and the sums of 2^(s - m) v
    float2* prefix_total;
    float* prefix_sums;
};

struct AppendParams {
    CacheView cache;
    RowsView q, k, v;
    void* q_out;                                      // (tokens, q_heads, dim) contiguous
    const int* slots;
    const float2* angles;                             // (tokens, pairs): cos, sin
    const void *q_weight, *k_weight;                  // (dim) in the activations' type, or nullptr: no norm
    int tokens, q_heads, pairs;                       // pairs 0: no rotation
    float eps;
};

struct ShareParams {
    const int *prefix_of, *seq_lens, *cu_lens;
    int *effective, *starts, *rows, *positions;
    int requests, max_tokens;
};

cudaError_t cache_plan_launch(const PlanParams& p, cudaStream_t stream);
cudaError_t cache_write_launch(const CacheView& c, bool e4m3, const RowsView& k, const RowsView& v, bool bf16, int tokens, const int* slots,
                               cudaStream_t stream);
cudaError_t cache_append_launch(const AppendParams& p, bool e4m3, bool bf16, bool pairs_beside, cudaStream_t stream);
cudaError_t cache_angles_launch(void* out, const int* positions, const float* freqs, int tokens, int pairs, cudaStream_t stream);
cudaError_t cache_share_launch(const ShareParams& p, cudaStream_t stream);
cudaError_t cache_read_launch(const CacheView& c, bool e4m3, void* k_out, void* v_out, bool bf16, int tokens, const int* slots,
                              cudaStream_t stream);

}  // namespace i4mm
