// extern "C" entry points of the paged 8-bit key-value cache: argument validation and launches.
#include "../../include/int4matmul_b200.h"

#include <algorithm>

#include "cache_attention.cuh"
#include "common.cuh"

namespace {

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int64_t kMost = 0x7FFFFFFF;                 // lengths, slots and page numbers are int32

int finish(cudaError_t e) {
    if (e == cudaSuccess) return I4MM_OK;
    i4mm::record_cuda_error((int)e);
    return I4MM_ERR_LAUNCH;
}

// log2 of a page's tokens, -1 for a size that there is not
int shift_of(int64_t page_size) {
    switch (page_size) {
        case 16: return 4;
        case 32: return 5;
        case 64: return 6;
        case 128: return 7;
        default: return -1;
    }
}

// rows of activations (tokens, heads, dim); the stride of a single token or head says nothing
i4mm::RowsView rows_of(const void* p, int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride) {
    return {p, tokens > 1 ? token_stride : 0, heads > 1 ? head_stride : 0};
}
bool aligned(const i4mm::RowsView& r) { return aligned(r.p, 16) && ((r.token | r.head) & 7) == 0; }

int view_of(const i4mm_cache* c, i4mm::CacheView& w) {
    if (!c) return I4MM_ERR_NULL;
    if (c->type != I4MM_CACHE_INT8 && c->type != I4MM_CACHE_E4M3) return I4MM_ERR_UNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128) return I4MM_ERR_UNSUPPORTED;
    if (shift_of(c->page_size) < 0) return I4MM_ERR_UNSUPPORTED;
    if (c->pages <= 0 || c->heads <= 0 || c->heads > 65535 || c->pages > kMost / c->page_size) return I4MM_ERR_SHAPE;
    if (!c->k || !c->v || !c->scales) return I4MM_ERR_NULL;
    // (the stride of a single page or head says nothing)
    const int64_t one = c->head_dim;
    const auto stride = [&](int64_t n, int64_t s) { return n > 1 ? s : one; };
    const int64_t k_page = stride(c->pages, c->k_page_stride), k_head = stride(c->heads, c->k_head_stride);
    const int64_t v_page = stride(c->pages, c->v_page_stride), v_head = stride(c->heads, c->v_head_stride);
    for (const int64_t s : {k_page, k_head, c->k_token_stride, v_page, v_head, c->v_token_stride})
        if (s < 0 || s > kMost) return I4MM_ERR_SHAPE;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 8) ||
        ((k_page | k_head | c->k_token_stride | v_page | v_head | c->v_token_stride) & 15))
        return I4MM_ERR_ALIGN;
    for (const int64_t s : {k_page, k_head, c->k_token_stride, v_page, v_head, c->v_token_stride})
        if (s < one) return I4MM_ERR_SHAPE;
    w.k = (uint8_t*)c->k;
    w.v = (uint8_t*)c->v;
    w.scales = (float2*)c->scales;
    w.k_page = k_page;
    w.k_head = k_head;
    w.k_token = c->k_token_stride;
    w.v_page = v_page;
    w.v_head = v_head;
    w.v_token = c->v_token_stride;
    w.pages = (int)c->pages;
    w.heads = (int)c->heads;
    w.page_shift = shift_of(c->page_size);
    w.dim = (int)c->head_dim;
    return I4MM_OK;
}

thread_local int g_attention_kernels = 0;             // i4mm_last_attention_kernels

size_t attention_workspace() { return i4mm::kCacheHeaderBytes + i4mm::cache_rows_workspace() + i4mm::cache_prompt_workspace(); }

// Which kernel.  A request's rows are its new tokens times the query heads of a key head.  The few-row kernel takes 8 or 16 of them at a time
// and reads the cache again (from the second-level cache) for the next ones, the prompt kernel works on 256 whatever they are: 16 requests of one
// token with contexts around 2250, 8 key heads of 128, 8 / 16 / 32 / 64 rows: 27 / 41 / 61 / 101 us and always 118; 2 requests 16 / 23 / 27 / 29
// and 35; 64 requests around 2000 65 / 99 / 168 / 295 and 259.  Where a batch may have both kinds, both run, each on its own requests.
// Little work is the few-row kernel's alone, more rows or not: it begins 5 to 10 us earlier, and a second launch costs 10.  `tiles` bounds its tiles
// of 32 tokens and 16 rows by what the host knows (lengths are on the GPU).  Single tokens beside a chunk: up to 12000 (bound 2250: 20 us and
// 34 for both, 5780: 34 and 45, 10192: 43 and 65, 12480: 40 and 44, 17680: 60 and 51).  Prompts alone: up to 8000 (1360: 25 and 33, 4160: 31 and
// 34, 10640: 44 and 36), but not those whose rows are more than twice their tokens, which fill the prompt kernel's tiles (1764: 26 and
// 25, 2576: 31 and 22, 4644: 31 and 19).
cudaError_t attend(const i4mm::AttentionParams& p, bool e4m3, bool bf16, int64_t max_len, cudaStream_t stream) {
    const int64_t len = p.cu_lens ? std::max<int64_t>(max_len, 1) : 1, rows = len * p.group;
    int64_t span = (int64_t)p.table_width << p.cache.page_shift;
    if (p.window) span = std::min(span, (int64_t)p.window + len);
    const int64_t tiles = ((int64_t)p.tokens * p.group / 16 + p.requests) * p.cache.heads * (span / 32 + 1);
    const bool mixed = (int64_t)p.tokens * 2 < p.requests * len;
    const bool little = mixed ? tiles <= 12000 : tiles <= 8000 && (rows < 2 * span || tiles <= 1000);
    const auto few = [&](int most_rows, bool to_8) {
        g_attention_kernels |= I4MM_ATTENTION_FEW_ROWS;
        return i4mm::cache_rows_launch(p, e4m3, bf16, most_rows, to_8, stream);
    };
    const auto prompt = [&](int least_rows, bool alone) {
        g_attention_kernels |= I4MM_ATTENTION_PROMPT;
        return i4mm::cache_prompt_launch(p, e4m3, bf16, least_rows, alone, stream);
    };
    if (rows <= i4mm::kFewRows || little) return few(0x7FFFFFFF, rows <= 8);
    if (p.group > i4mm::kFewRows) return prompt(1, true);
    const cudaError_t e = few(i4mm::kFewRows, p.group <= 8);
    return e != cudaSuccess ? e : prompt(i4mm::kFewRows + 1, false);
}

}  // namespace

extern "C" {

int i4mm_cache_plan(int64_t requests, const void* seq_lens, const void* new_lens, void* block_table, int64_t table_width,
                    int64_t table_stride, void* free_pages, int64_t free_capacity, const void* free_count, int64_t page_size,
                    int64_t max_tokens, void* lens_after, void* cu_lens, void* slots, void* positions, void* request_of, void* counts,
                    void* stream) {
    if (shift_of(page_size) < 0) return I4MM_ERR_UNSUPPORTED;
    // the kernel's loops over tokens and table entries step by up to 296 * 512 in 32 bits
    constexpr int64_t kMostSteps = int64_t(1) << 30;
    if (requests < 0 || requests > 16384 || table_width < 0 || table_width > kMost || requests * table_width > kMostSteps ||
        table_stride < table_width || free_capacity < 0 || free_capacity > kMost || max_tokens < 0 || max_tokens > kMostSteps)
        return I4MM_ERR_SHAPE;
    if (!cu_lens || !counts || !free_count) return I4MM_ERR_NULL;
    if (requests > 0 && (!seq_lens || !new_lens || !lens_after || (table_width > 0 && !block_table))) return I4MM_ERR_NULL;
    if ((max_tokens > 0 && (!slots || !positions || !request_of)) || (free_capacity > 0 && !free_pages)) return I4MM_ERR_NULL;
    for (const void* p : {seq_lens, new_lens, (const void*)block_table, (const void*)free_pages, free_count, (const void*)lens_after,
                          (const void*)cu_lens, (const void*)slots, (const void*)positions, (const void*)request_of, (const void*)counts})
        if (!aligned(p, 4)) return I4MM_ERR_ALIGN;
    i4mm::PlanParams p{};
    p.seq_lens = (const int*)seq_lens;
    p.new_lens = (const int*)new_lens;
    p.table = (int*)block_table;
    p.free_pages = (int*)free_pages;
    p.free_count = (const int*)free_count;
    p.lens_after = (int*)lens_after;
    p.cu_lens = (int*)cu_lens;
    p.slots = (int*)slots;
    p.positions = (int*)positions;
    p.request_of = (int*)request_of;
    p.counts = (int*)counts;
    p.table_stride = table_stride;
    p.requests = (int)requests;
    p.table_width = (int)table_width;
    p.free_capacity = (int)free_capacity;
    p.page_shift = shift_of(page_size);
    p.max_tokens = (int)max_tokens;
    return finish(i4mm::cache_plan_launch(p, (cudaStream_t)stream));
}

int i4mm_cache_write(const i4mm_cache* cache, const void* k, const void* v, int type, int64_t tokens, int64_t k_token_stride,
                     int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const void* slots, void* stream) {
    i4mm::CacheView c{};
    const int status = view_of(cache, c);
    if (status != I4MM_OK) return status;
    if (type != I4MM_TYPE_FP16 && type != I4MM_TYPE_BF16) return I4MM_ERR_UNSUPPORTED;
    if (tokens < 0 || tokens > kMost) return I4MM_ERR_SHAPE;
    if (tokens == 0) return I4MM_OK;
    if (!k || !v || !slots) return I4MM_ERR_NULL;
    const i4mm::RowsView k_rows = rows_of(k, tokens, k_token_stride, c.heads, k_head_stride);
    const i4mm::RowsView v_rows = rows_of(v, tokens, v_token_stride, c.heads, v_head_stride);
    if (!aligned(k_rows) || !aligned(v_rows) || !aligned(slots, 4)) return I4MM_ERR_ALIGN;
    return finish(i4mm::cache_write_launch(c, cache->type == I4MM_CACHE_E4M3, k_rows, v_rows, type == I4MM_TYPE_BF16, (int)tokens,
                                           (const int*)slots, (cudaStream_t)stream));
}

int i4mm_cache_read(const i4mm_cache* cache, void* k_out, void* v_out, int type, int64_t tokens, const void* slots, void* stream) {
    i4mm::CacheView c{};
    const int status = view_of(cache, c);
    if (status != I4MM_OK) return status;
    if (type != I4MM_TYPE_FP16 && type != I4MM_TYPE_BF16) return I4MM_ERR_UNSUPPORTED;
    if (tokens < 0 || tokens > kMost) return I4MM_ERR_SHAPE;
    if (tokens == 0) return I4MM_OK;
    if (!k_out || !v_out || !slots) return I4MM_ERR_NULL;
    if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(slots, 4)) return I4MM_ERR_ALIGN;
    return finish(i4mm::cache_read_launch(c, cache->type == I4MM_CACHE_E4M3, k_out, v_out, type == I4MM_TYPE_BF16, (int)tokens,
                                          (const int*)slots, (cudaStream_t)stream));
}

int i4mm_last_attention_kernels(void) { return g_attention_kernels; }

size_t i4mm_cache_attention_workspace_bytes(void) { return attention_workspace(); }

int i4mm_cache_attention(const i4mm_cache* cache, void* out, const void* q, int type, int64_t tokens, int64_t q_heads,
                         int64_t q_token_stride, int64_t q_head_stride, const void* block_table, int64_t table_width,
                         int64_t table_stride, const void* seq_lens, const void* cu_lens, int64_t requests, int64_t max_len, float scale,
                         int64_t window, void* workspace, size_t workspace_bytes, void* stream) {
    g_attention_kernels = 0;
    i4mm::AttentionParams p{};
    const int status = view_of(cache, p.cache);
    if (status != I4MM_OK) return status;
    if (type != I4MM_TYPE_FP16 && type != I4MM_TYPE_BF16) return I4MM_ERR_UNSUPPORTED;
    if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->heads) return I4MM_ERR_SHAPE;
    // (tokens of a table's row: a tile of 128 that begins among them ends below 2^31)
    if (tokens < 0 || tokens > kMost / q_heads || requests < 0 || requests > 16384 || table_width < 0 || table_width > (kMost - 127) / cache->page_size ||
        table_stride < table_width || max_len < 0 || max_len > kMost || window < 0 || window > kMost)
        return I4MM_ERR_SHAPE;
    if (!cu_lens && tokens < requests) return I4MM_ERR_SHAPE;
    if (tokens == 0) return I4MM_OK;
    if (!out || !q || (requests > 0 && (!seq_lens || (table_width > 0 && !block_table)))) return I4MM_ERR_NULL;
    p.q = rows_of(q, tokens, q_token_stride, q_heads, q_head_stride);
    if (!aligned(out, 16) || !aligned(p.q) || !aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(cu_lens, 4)) return I4MM_ERR_ALIGN;
    if (!workspace || workspace_bytes < attention_workspace()) return I4MM_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return I4MM_ERR_ALIGN;
    p.out = out;
    p.table = (const int*)block_table;
    p.seq_lens = (const int*)seq_lens;
    p.cu_lens = (const int*)cu_lens;
    p.workspace = workspace;
    p.prompt_parts = i4mm::kCacheHeaderBytes + i4mm::cache_rows_workspace();
    p.table_stride = table_stride;
    p.table_width = (int)table_width;
    p.requests = (int)requests;
    p.tokens = (int)tokens;
    p.q_heads = (int)q_heads;
    p.group = (int)(q_heads / cache->heads);
    p.window = (int)window;
    p.scale = scale;
    return finish(attend(p, cache->type == I4MM_CACHE_E4M3, type == I4MM_TYPE_BF16, max_len, (cudaStream_t)stream));
}

}  // extern "C"
