// Attention over the paged 8-bit cache (i4mm_cache_attention), many rows per request: prompts and chunks of them.
//
//   x_j = log2(e) * scale * s_key * (q . k_j) + log2(s_value),  P_j = 2^(x_j - M)   (fp16)
//   with a reference M, an x_j of the row,
//   o = sum_j P_j v_j / sum_j (P_j / s_value),  k_j and v_j the cache's bytes, s_key and s_value their page's scales
// so the value scale is in the weight that is rounded anyway, and the bytes go into the tensor cores as they are.
//
// With hundreds of rows for each byte the tensor cores and the exponentials bound it: per tile of 256 rows and 128 tokens at head_dim 128,
// 16 score instructions of 128 x 128 x 16 with both operands in shared memory (106 cycles each, measured alone), 16 of the second product
// with the weights in tensor memory (76), 2900 cycles together, and 32768 exponentials (16 a cycle and SM: 2048 cycles).  They have to run
// at the same time, so they belong to different warps:
//
//   warps 0..3, 4..7   softmax of 128 rows each (A and B): a thread owns a row; scores come from tensor memory, weights go back there,
//                      where they are the A operand of the second product
//   warps 8..11        read the pages, turn bytes into fp16 (exact) and lay out K and V^T for the tensor cores (128-byte swizzle);
//                      K and V tiles are decoded once for 256 rows
//   warp 12            issues the products: while the softmax of A runs, the tensor cores work for B
//   warp 13            takes the next item (request, key head, 256 rows, a range of tokens), one ahead
//
// The rows of all query heads of a key head are packed into one tile: row r is token r / group, head r % group.  Sums stay in
// tensor memory in fp32 and are rescaled only when a row's weights would outgrow fp16 (below that their relative precision is the
// same), which costs no maximum on the way: the weights' sum, which is needed anyhow, tells.  Long contexts under few rows are cut along the
// tokens into items of their own; the block that finishes a segment's last part joins them in order.  Every wait is bounded; a block that
// gives up records it in the status word.
//
// Measured: 2 x 1024 new tokens after 8000, 64 heads in groups of 8: 750 us, 720 TFLOP/s; a prompt of 2048 tokens, 40 heads: 102 us, the few-row
// kernel's empty launch before it included.  A tile
// takes about 5000 cycles: the chain of one half (scores 850 and more, 400 until they are in registers, 2 x 1000 for weights, 2 x 250 to pack and
// publish them, the second product) against the other half's, and the decoding warps' chain, which is as long.  Without exponentials it is
// 2 % faster, without decoding 17 %, with neither softmax nor decoding 40 %.  Slower: scores of 64 tokens at a time in two halves of their
// columns (1000 us: 75 cycles an instruction, and loads from tensor memory wait for products), one thread waiting and issuing instead of
// an elected lane of a whole warp (900).
#include <algorithm>
#include <type_traits>

#include "cache_attention.cuh"

namespace i4mm {
namespace {

constexpr int kTokens = 128;                          // of a tile
constexpr int kHalf = 128;                            // rows of A and of B
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 4;
constexpr int kDecode0 = kSoftmaxWarps, kMma = kDecode0 + kDecodeWarps, kSchedule = kMma + 1;
constexpr int kThreads = 32 * (kSchedule + 1);
constexpr int kScaleSlots = 4;
constexpr int kMinTiles = 4;                          // a part of a segment has at least so many tiles
constexpr float kLeastFactor = 1e-30f;                // in the place of a key scale of 0: scores are 0 either way
constexpr float kMostWeight = 16384.f;                // fp16 holds 65504

template <int D>
struct Layout {
    static constexpr int kQ = kHalf * D * 2, kK = kTokens * D * 2, kV = D * kTokens * 2;
    static constexpr int kQ0 = 0, kK0 = 2 * kQ, kV0 = kK0 + 2 * kK, kBytes = kV0 + 2 * kV + 1024;
    static constexpr int kPartFloats = kHalf * D + 2 * kHalf;                // of one half: [D / 4][row][4], maxima, totals
};

struct Item {
    int valid;
    int b, row0, position, all_rows, head, base;      // base: first row of the tile
    int lo, limit;                                    // tokens that may be seen
    int tile0;                                        // first tile of the item
    int tiles[2];                                     // of A and B (0: none)
    int rows[2];                                      // rows of A and B
    int part, parts, which;                           // first part of the segment in the workspace (-1: not cut), their number, this item's
};

struct Barriers {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], scale_full[kScaleSlots], item_full[2], item_empty[2];
    unsigned long long q_full[2], s_full[2], p_full[2][2], pv_half[2], pv_done[2], group[2], drained;
};

// A whole warp waits; false (in all of its lanes) once the block gives up.
__device__ __forceinline__ bool wait_on(unsigned long long* bar, uint32_t parity, volatile int* abort) {
    const uint32_t at = ptx::smem_u32(bar);
    for (uint32_t i = 0; i < ptx::kSpinLimit; ++i) {
        if (__all_sync(kAll, ptx::mbar_try_wait(at, parity))) return true;
        if (__any_sync(kAll, *abort)) return false;
    }
    *abort = 1;
    return false;
}
__device__ __forceinline__ void arrive(unsigned long long* bar) { ptx::mbar_arrive(ptx::smem_u32(bar)); }

// What a launch is for: rows over their own tokens; the same, and what a shared prefix came to is added at the end; or all rows that read a prefix,
// over that prefix, whose sums and totals are kept for that.
enum Kind { kOwn, kJoining, kPrefixes };

// The segments' owner: a request, or a place and its readers (row0: their first in the list of readers).  All of a prefix is seen by every reader, but
// for what a window hides.
template <int KIND>
__device__ __forceinline__ Request load_owner(const AttentionParams& p, int b) {
    if (KIND != kPrefixes) return load_request(p, b);
    Request r;
    const int from = min(max(p.prefix_starts[b], 0), p.prefix_listed), to = min(max(p.prefix_starts[b + 1], 0), p.prefix_listed), seq = p.seq_lens[b];
    r.row0 = from;
    r.rows = min(max(to - from, 0), p.tokens);
    r.limit = max(min(seq, p.table_width << p.cache.page_shift), 0);
    r.position = r.limit;
    r.lo = p.window && seq >= p.window ? min(seq - p.window + 1, r.limit) : 0;
    return r;
}

// ---- items ---------------------------------------------------------------------------------------------------------------------
// A segment is a key head and a tile of 256 rows of a request.  Segments are items of their own, or cut along the tokens into parts:
//   * long ones, so that none has more than its share of the GPU's work;
//   * those that are left over when all blocks have had the same number of whole ones (of 512 equal segments 444 make three rounds of 148
//     blocks; the other 68, cut in two, make half a round instead of a whole one), unless they are short.
// A part costs about two tiles' time for writing its sums and joining them.
struct Split {
    int part_tiles;                                   // of the first kind
    long long whole;                                  // segments (in their order) before those that are left over
    int spread;                                       // parts of one that is left over
};
struct Cut {
    int row_tiles, segments, parts, last, last_parts; // the last `last` segments are cut into last_parts, the others into `parts`
};
__device__ __forceinline__ int row_tiles_of(const AttentionParams& p, const Request& r, int least_rows) {
    const long long rows = (long long)r.rows * p.group;
    return rows < least_rows ? 0 : (int)((rows + 2 * kHalf - 1) / (2 * kHalf));
}
__device__ __forceinline__ int tiles_of(const Request& r) { return r.limit > r.lo ? (r.limit + kTokens - 1) / kTokens - r.lo / kTokens : 0; }
// `before`: segments of the requests before this one
__device__ __forceinline__ Cut cut_of(const AttentionParams& p, const Request& r, int least_rows, const Split& s, long long before) {
    Cut c;
    const int tiles = tiles_of(r);
    c.row_tiles = row_tiles_of(p, r, least_rows);
    c.segments = c.row_tiles * p.cache.heads;
    c.parts = max(1, (tiles + s.part_tiles - 1) / s.part_tiles);
    // the segments at the end of a request are those of its first rows: what they see
    const int few = min(tiles, max(0, (r.position + (2 * kHalf + p.group - 1) / p.group + kTokens - 1) / kTokens - r.lo / kTokens));
    c.last_parts = max(c.parts, min(s.spread, few / (2 * kMinTiles)));
    c.last = c.last_parts > c.parts ? (int)max(0ll, min((long long)c.segments, before + c.segments - s.whole)) : 0;
    return c;
}
__device__ __forceinline__ long long items_of(const Cut& c) { return (long long)(c.segments - c.last) * c.parts + (long long)c.last * c.last_parts; }
__device__ __forceinline__ long long parts_of(const Cut& c) {             // of segments that are cut
    return (c.parts > 1 ? (long long)(c.segments - c.last) * c.parts : 0) + (c.last_parts > 1 ? (long long)c.last * c.last_parts : 0);
}

// How all segments are cut, and the number of items.  Parts must find room in the workspace.
template <int KIND>
__device__ __forceinline__ Split choose_split(const AttentionParams& p, int least_rows, int blocks, long long* items) {
    const int lane = threadIdx.x & 31;
    long long tiles = 0, segments = 0;
    for (int b = lane; b < p.requests; b += 32) {
        const Request r = load_owner<KIND>(p, b);
        const long long n = (long long)row_tiles_of(p, r, least_rows) * p.cache.heads;
        segments += n;
        tiles += n * tiles_of(r);
    }
    tiles = warp_sum(tiles);
    segments = warp_sum(segments);
    Split s;
    s.whole = segments / blocks * blocks;
    s.spread = segments > s.whole ? (int)(blocks / (segments - s.whole)) : 1;
    long long part = max((long long)kMinTiles, (tiles * 9 / 8 + blocks - 1) / blocks);
    for (;; part *= 2) {
        s.part_tiles = (int)min(part, (long long)0x3FFFFFFF);
        long long all = 0, cut = 0, before = 0;
        for (int base = 0; base < p.requests; base += 32) {
            Cut c{};
            c.parts = c.last_parts = 1;
            Request r{};
            if (base + lane < p.requests) r = load_owner<KIND>(p, base + lane);
            const long long own = base + lane < p.requests ? (long long)row_tiles_of(p, r, least_rows) * p.cache.heads : 0, upto = warp_prefix(own);
            if (base + lane < p.requests) c = cut_of(p, r, least_rows, s, before + upto - own);
            before += __shfl_sync(kAll, upto, 31);
            all += items_of(c);
            cut += parts_of(c);
        }
        all = warp_sum(all);
        cut = warp_sum(cut);
        if (cut <= kPromptParts || part > 0x3FFFFFFF) {
            *items = all;
            return s;
        }
        if (part > tiles) s.spread = 1;
    }
}

// Item `index` in the order of requests, from each one's last rows to its first (they see the most).  The whole warp calls.
template <int KIND>
__device__ __forceinline__ void find_item(const AttentionParams& p, int least_rows, const Split& split, long long index, Item* out) {
    const int lane = threadIdx.x & 31;
    long long before = 0, parts_before = 0, segments_before = 0;
    for (int base = 0; base < p.requests; base += 32) {
        Request r{};
        Cut c{};
        c.parts = c.last_parts = 1;
        if (base + lane < p.requests) r = load_owner<KIND>(p, base + lane);
        const long long segments = base + lane < p.requests ? (long long)row_tiles_of(p, r, least_rows) * p.cache.heads : 0, upto = warp_prefix(segments);
        if (base + lane < p.requests) c = cut_of(p, r, least_rows, split, segments_before + upto - segments);
        segments_before += __shfl_sync(kAll, upto, 31);
        const long long own = items_of(c), own_parts = parts_of(c), sum = warp_prefix(own), parts = warp_prefix(own_parts);
        const uint32_t here = __ballot_sync(kAll, before + sum > index);
        if (here == 0) {
            before += __shfl_sync(kAll, sum, 31);
            parts_before += __shfl_sync(kAll, parts, 31);
            continue;
        }
        if (lane == __ffs(here) - 1) {
            long long in = index - (before + sum - own), first_part = parts_before + parts - own_parts;
            const long long plain = (long long)(c.segments - c.last) * c.parts;
            int n_parts = c.parts;
            long long segment = 0;
            if (in >= plain) {
                in -= plain;
                segment = c.segments - c.last;
                if (c.parts > 1) first_part += plain;
                n_parts = c.last_parts;
            }
            const int which = (int)(in % n_parts);
            segment += in / n_parts;
            const int head = (int)(segment % p.cache.heads), tile = c.row_tiles - 1 - (int)(segment / p.cache.heads);
            Item t;
            t.valid = 1;
            t.b = base + lane;
            t.row0 = r.row0;
            t.position = r.position;
            t.all_rows = r.rows * p.group;
            t.head = head;
            t.base = tile * 2 * kHalf;
            t.parts = n_parts;
            t.which = which;
            t.part = n_parts > 1 ? (int)(first_part + in - which) : -1;
            // the tokens that the rows of A and of B see, in tiles
            const int first = t.base / p.group;
            t.lo = KIND != kPrefixes && p.window && r.position + first >= p.window ? min(r.position + first - p.window + 1, r.limit) : r.lo;
            int end[2] = {0, 0};
            for (int h = 0; h < 2; ++h) {
                t.rows[h] = min(max(t.all_rows - t.base - h * kHalf, 0), kHalf);
                if (t.rows[h] == 0) continue;
                const int limit = min(r.limit, r.position + (t.base + h * kHalf + t.rows[h] - 1) / p.group + 1);
                if (limit > t.lo) end[h] = (limit + kTokens - 1) / kTokens;
                t.limit = limit;
            }
            const int begin = t.lo / kTokens, n = max(max(end[0], end[1]) - begin, 0);
            t.tile0 = begin + (int)((long long)n * which / n_parts);
            const int stop = begin + (int)((long long)n * (which + 1) / n_parts);
            for (int h = 0; h < 2; ++h) t.tiles[h] = max(min(end[h], stop) - t.tile0, 0);
            *out = t;
        }
        __syncwarp();
        return;
    }
    if (lane == 0) out->valid = 0;                    // (not unless the lengths change under the kernel)
    __syncwarp();
}

// ---- two fp32 at a time ----
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// address of 16 bytes (8 values) `unit` of `row` in an operand tile of `rows` rows: sub-tiles of 64 values, 128-byte rows, swizzled
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int rows, int row, int unit) {
    return tile + (unit >> 3) * (rows * 128) + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
}

template <bool E4M3, bool BF16, int D, int KIND>
__global__ void __launch_bounds__(kThreads, 1) cache_prompt_kernel(const AttentionParams p, int least_rows, int alone) {
    using L = Layout<D>;
    extern __shared__ uint8_t dynamic[];
    __shared__ Barriers bars;
    __shared__ Item items[2];
    __shared__ float4 scales[kScaleSlots][kTokens / 16];   // of 16 tokens: key scale, log2 of the value scale, its inverse
    __shared__ volatile int s_abort;
    __shared__ int s_last[2];
    __shared__ uint32_t tmem_smem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem = (ptx::smem_u32(dynamic) + 1023u) & ~1023u;
    const uint32_t q_tile[2] = {smem + L::kQ0, smem + L::kQ0 + L::kQ};
    const uint32_t k_tile = smem + L::kK0, v_tile = smem + L::kV0;
    uint8_t* const header = static_cast<uint8_t*>(p.workspace);
    int* const status = reinterpret_cast<int*>(header + kStatusOffset);

    if (threadIdx.x == 0) {
        const auto init = [](unsigned long long& b, uint32_t n) { ptx::mbar_init(ptx::smem_u32(&b), n); };
        for (int i = 0; i < 2; ++i) {
            init(bars.k_full[i], kDecodeWarps);
            init(bars.v_full[i], kDecodeWarps);
            init(bars.k_empty[i], 1);
            init(bars.v_empty[i], 1);
            init(bars.item_full[i], 1);
            init(bars.item_empty[i], kSoftmaxWarps + kDecodeWarps + 1);
            init(bars.q_full[i], 4);
            init(bars.s_full[i], 1);
            init(bars.p_full[i][0], 4);
            init(bars.p_full[i][1], 4);
            init(bars.pv_half[i], 1);
            init(bars.pv_done[i], 1);
            init(bars.group[i], 4);
        }
        for (int i = 0; i < kScaleSlots; ++i) init(bars.scale_full[i], 1);
        init(bars.drained, 1);
        ptx::fence_mbar_init();
        s_abort = 0;
    }
    if (warp == kMma) {
        ptx::tmem_alloc(ptx::smem_u32(&tmem_smem), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = tmem_smem;
    const auto s_col = [&](int h) { return tmem + h * 128; };
    const auto o_col = [&](int h) { return tmem + 256 + h * 128; };
    // (kPrefixes: the kernel before is that of places with few readers, which let this one begin once it knew all before it complete.  They write different
    // rows and share nothing else, so it is only waited for before a block leaves: this kernel must not be complete before that one is.)
    if (KIND != kPrefixes) ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    if (alone) {                                      // rows of no request
        const int first = p.requests == 0 ? 0 : p.cu_lens ? min(max(p.cu_lens[p.requests], 0), p.tokens) : p.requests;
        const long long from = (long long)first * p.q_heads * D, to = (long long)p.tokens * p.q_heads * D;
        for (long long i = from + 8ll * (blockIdx.x * kThreads + threadIdx.x); i < to; i += 8ll * gridDim.x * kThreads)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i) = make_uint4(0, 0, 0, 0);
    }

    // every role walks the same items: slot n & 1, filled for the (n / 2)-th time
    const auto next_item = [&](uint32_t n) { return wait_on(&bars.item_full[n & 1], (n >> 1) & 1, &s_abort) && items[n & 1].valid; };
    const auto done_with_item = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) arrive(&bars.item_empty[n & 1]);
    };

    if (warp == kSchedule) {
        long long count = 0;
        const Split split = choose_split<KIND>(p, least_rows, gridDim.x, &count);
        unsigned int* const next = reinterpret_cast<unsigned int*>(header + kPromptNext);
        for (uint32_t n = 0;; ++n) {
            if (!wait_on(&bars.item_empty[n & 1], ((n >> 1) & 1) ^ 1, &s_abort)) break;
            // the first item is the block's own number, the others come off the counter
            long long i = blockIdx.x;
            if (n > 0) {
                unsigned int taken = 0;
                if (lane == 0) taken = atomicAdd(next, 1u);
                i = (long long)gridDim.x + __shfl_sync(kAll, taken, 0);
            }
            const bool more = i < count;
            if (more) find_item<KIND>(p, least_rows, split, i, &items[n & 1]);
            else if (lane == 0) items[n & 1].valid = 0;
            __syncwarp();
            if (lane == 0) {
                arrive(&bars.item_full[n & 1]);
                // every block that had an item takes one number too many, `count` numbers in all; the last one leaves the counter as the next
                // launch expects it
                if (!more && n > 0 && i == count + gridDim.x - 1) atomicExch(next, 0u);
            }
            if (!more) break;
        }
    } else if (warp == kMma) {
        // ---- products ----
        const uint32_t idesc_s = ptx::idesc_f16_m128(kTokens), idesc_o = ptx::idesc_f16_m128(D);
        uint32_t k_stage = 0, v_stage = 0;            // tiles of K and V that have been used
        uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
        bool ok = true;
        for (uint32_t n = 0; ok && next_item(n); ++n) {
            const Item& t = items[n & 1];
            const int tiles[2] = {t.tiles[0], t.tiles[1]}, most = max(tiles[0], tiles[1]);
            const auto score = [&](int h, int j) {    // S_h = Q_h K_j^T
                if (j == 0) {
                    ok = ok && wait_on(&bars.q_full[h], q_phase[h], &s_abort);
                    q_phase[h] ^= 1;
                }
                ok = ok && wait_on(&bars.k_full[k_stage & 1], (k_stage >> 1) & 1, &s_abort);
                if (!ok) return;
                ptx::tc_fence_after_sync();
                if (ptx::elect_one()) {
                    const uint64_t a = ptx::smem_desc_sw128(q_tile[h]), b = ptx::smem_desc_sw128(k_tile + (k_stage & 1) * L::kK);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t step = (uint64_t)((k >> 2) * (128 * 128 >> 4) + (k & 3) * 2);
                        ptx::umma_f16_ss(s_col(h), a + step, b + step, idesc_s, k > 0);
                    }
                    ptx::tc_commit(ptx::smem_u32(&bars.s_full[h]));
                }
                __syncwarp();
            };
            const auto k_done = [&]() {
                if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars.k_empty[k_stage & 1]));
                __syncwarp();
                ++k_stage;
            };
            if (most > 0) {
                for (int h = 0; h < 2; ++h)
                    if (tiles[h] > 0) score(h, 0);
                k_done();
            }
            for (int j = 0; j < most && ok; ++j) {
                for (int h = 0; h < 2; ++h) {
                    if (j >= tiles[h]) continue;
                    // O_h += P_h V_j, as far as the weights are there
                    ok = ok && wait_on(&bars.v_full[v_stage & 1], (v_stage >> 1) & 1, &s_abort);
                    for (int part = 0; part < 2 && ok; ++part) {
                        ok = wait_on(&bars.p_full[h][part], p_phase[h], &s_abort);
                        if (!ok) break;
                        ptx::tc_fence_after_sync();
                        if (ptx::elect_one()) {
                            const uint64_t b = ptx::smem_desc_sw128(v_tile + (v_stage & 1) * L::kV) + (uint64_t)part * (D * 128 >> 4);
                            const uint32_t a = s_col(h) + 32 * part;
#pragma unroll
                            for (int k = 0; k < kTokens / 32; ++k) ptx::umma_f16_ts(o_col(h), a + 8 * k, b + k * 2, idesc_o, j > 0 || part > 0 || k > 0);
                            ptx::tc_commit(ptx::smem_u32(part == 0 ? &bars.pv_half[h] : &bars.pv_done[h]));
                        }
                        __syncwarp();
                    }
                    p_phase[h] ^= 1;
                    if (!ok) break;
                    if (j + 1 < tiles[h]) score(h, j + 1);
                }
                if (!ok) break;
                if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars.v_empty[v_stage & 1]));
                __syncwarp();
                ++v_stage;
                if (j + 1 < most) k_done();
            }
            done_with_item(n);
        }
        // nothing of this block may be in flight when its tensor memory goes
        if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars.drained));
        __syncwarp();
        for (uint32_t i = 0; i < ptx::kSpinLimit && !ptx::mbar_try_wait(ptx::smem_u32(&bars.drained), 0); ++i) {}
    } else if (warp >= kDecode0) {
        // ---- bytes to operands ----
        const CacheView& cache = p.cache;
        const int w = warp - kDecode0;
        constexpr int kKeyRows = D / 16;              // 16 bytes of so many key rows a thread
        const int k_unit = D == 128 ? 4 * (w & 1) + (lane >> 3) : lane >> 3;                    // of 16 bytes
        const int k_block = D == 128 ? 8 * (w >> 1) : 4 * w;                                    // rows 8 * (k_block + i) + (lane & 7)
        const int v_unit = 4 * (w & 1) + (lane >> 3), v_group = 8 * (w >> 1) + (lane & 7);      // D / 8 bytes of tokens 8 * v_group ..
        using VBytes = std::conditional_t<D == 128, uint4, uint2>;
        uint32_t stage = 0;
        bool ok = true;
        for (uint32_t n = 0; ok && next_item(n); ++n) {
            const Item t = items[n & 1];
            const int most = max(t.tiles[0], t.tiles[1]);
            const int* const table = p.table + t.b * p.table_stride;
            uint4 k[kKeyRows];
            VBytes v[8];
            int ids = -1, later = -1;                 // lane l: the page of tokens 16 * (l & 7) of the tile that is fetched next, and of the one after
            float2 both = {}, later_both = {}, now = {};                      // their scales, and those of the tile that is decoded
            const auto load_pages = [&](int j) {
                const int token = (t.tile0 + j) * kTokens + 16 * (lane & 7), at = token >> cache.page_shift;
                later = -1;
                if (j < most && at < p.table_width && token + 16 > t.lo && token < t.limit) later = table[at];
            };
            const auto load_scales = [&]() {          // of `later`
                if ((unsigned int)later >= (unsigned int)cache.pages) later = -1;
                if (later >= 0) later_both = cache.scales[(long long)later * cache.heads + t.head];
            };
            const auto next_pages = [&]() {
                ids = later;
                both = later_both;
            };
            // (32-bit strides: 64-bit products for each row would take longer than the decoding)
            const uint8_t* const k_base = cache.k + t.head * cache.k_head + (lane & 7) * cache.k_token + 16 * k_unit;
            const uint8_t* const v_base = cache.v + t.head * cache.v_head + (D / 8) * v_unit;
            const int page_mask = (1 << cache.page_shift) - 1;
            const int k_page = (int)cache.k_page, v_page = (int)cache.v_page, k_token = (int)cache.k_token, v_token = (int)cache.v_token;
            const auto load_keys = [&](int j) {
                const int first = (t.tile0 + j) * kTokens;
                const bool all = first >= t.lo && first + kTokens <= t.limit;
#pragma unroll
                for (int i = 0; i < kKeyRows; ++i) {
                    const int token = first + 8 * (k_block + i);              // and lane & 7
                    const int id = __shfl_sync(kAll, ids, (k_block + i) >> 1);
                    k[i] = make_uint4(0, 0, 0, 0);
                    if (id >= 0 && (all || (token + (lane & 7) >= t.lo && token + (lane & 7) < t.limit)))
                        k[i] = *reinterpret_cast<const uint4*>(k_base + (long long)id * k_page + (long long)(token & page_mask) * k_token);
                }
            };
            const auto load_values = [&](int j) {
                const int first = (t.tile0 + j) * kTokens + 8 * v_group;
                const int id = __shfl_sync(kAll, ids, v_group >> 1);
                const uint8_t* const from = v_base + (long long)max(id, 0) * v_page + (long long)(first & page_mask) * v_token;
                if (id >= 0 && first >= t.lo && first + 8 <= t.limit) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const VBytes*>(from + (long long)i * v_token);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[i] = VBytes{};
                        if (id >= 0 && first + i >= t.lo && first + i < t.limit) v[i] = *reinterpret_cast<const VBytes*>(from + (long long)i * v_token);
                    }
                }
            };
            if (most > 0) {
                load_pages(0);
                load_scales();
                next_pages();
                load_keys(0);
                load_values(0);
                load_pages(1);
            }
            for (int j = 0; j < most && ok; ++j, ++stage) {
                const bool there = ids >= 0;
                now = both;
                load_scales();                        // of tile j + 1, whose pages were asked for a tile ago
                next_pages();
                load_pages(j + 2);
                const int s = stage & 1;
                const uint32_t phase = ((stage >> 1) & 1) ^ 1;
                if (w == 0 && lane < 8) {
                    const float value = fmaxf(now.y, kLeastScale);
                    scales[stage % kScaleSlots][lane] = there ? make_float4(now.x, log2f(value), 1.f / value, 0.f) : make_float4(0.f, -INFINITY, 0.f, 0.f);
                }
                ok = wait_on(&bars.k_empty[s], phase, &s_abort);
                if (!ok) break;
                const uint32_t k_to = k_tile + s * L::kK, v_to = v_tile + s * L::kV;
#pragma unroll
                for (int i = 0; i < kKeyRows; ++i) {
                    const int row = 8 * (k_block + i) + (lane & 7);
                    uint4 a, b;
                    decode4<E4M3>(k[i].x, a.x, a.y);
                    decode4<E4M3>(k[i].y, a.z, a.w);
                    decode4<E4M3>(k[i].z, b.x, b.y);
                    decode4<E4M3>(k[i].w, b.z, b.w);
                    ptx::sts128(swizzled(k_to, kTokens, row, 2 * k_unit), a);
                    ptx::sts128(swizzled(k_to, kTokens, row, 2 * k_unit + 1), b);
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    arrive(&bars.k_full[s]);
                    if (w == 0) arrive(&bars.scale_full[stage % kScaleSlots]);
                }
                if (j + 1 < most) load_keys(j + 1);
                ok = wait_on(&bars.v_empty[s], phase, &s_abort);
                if (!ok) break;
                const auto word = [&](int i, int c) {
                    if constexpr (D == 128) return c == 0 ? v[i].x : c == 1 ? v[i].y : c == 2 ? v[i].z : v[i].w;
                    else return c == 0 ? v[i].x : v[i].y;
                };
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint4 a, b;
                        decode_pair<E4M3>(word(0, c), word(1, c), half, a.x, b.x);
                        decode_pair<E4M3>(word(2, c), word(3, c), half, a.y, b.y);
                        decode_pair<E4M3>(word(4, c), word(5, c), half, a.z, b.z);
                        decode_pair<E4M3>(word(6, c), word(7, c), half, a.w, b.w);
                        const int row = (D / 8) * v_unit + 4 * c + 2 * half;
                        ptx::sts128(swizzled(v_to, D, row, v_group), a);
                        ptx::sts128(swizzled(v_to, D, row + 1, v_group), b);
                    }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&bars.v_full[s]);
                if (j + 1 < most) load_values(j + 1);
            }
            done_with_item(n);
        }
    } else {
        // ---- softmax ----
        const int h = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = s_col(h) + lanes, o_at = o_col(h) + lanes;
        uint32_t s_phase = 0, pv_count = 0, tile_count = 0, group_phase = 0;
        bool ok = true;
        const auto meet = [&]() {                     // the four warps of a half; bounded, unlike a named barrier
            __syncwarp();
            if (lane == 0) arrive(&bars.group[h]);
            ok = ok && wait_on(&bars.group[h], group_phase, &s_abort);
            group_phase ^= 1;
        };
        for (uint32_t n = 0; ok && next_item(n); ++n) {
            const Item& t = items[n & 1];
            const int tiles = t.tiles[h], most = max(t.tiles[0], t.tiles[1]);
            const int mine = t.base + h * kHalf + row;                        // the row
            bool real = row < t.rows[h];
            int token = mine / p.group;
            const int head = t.head * p.group + mine - token * p.group;
            int position = real ? t.position + token : -1;
            if constexpr (KIND == kPrefixes) {        // the row that the list names, at its place behind the prefix
                const int entry = t.row0 + token;
                token = real && entry < p.prefix_listed ? p.prefix_rows[entry] : -1;
                real = token >= 0 && token < p.tokens;
                position = real ? t.position : -1;
                if (real && p.window) position = behind_prefix(p, t.b, token);
                token -= t.row0;
            }
            float2 prefix = make_float2(-INFINITY, 0.f);
            if constexpr (KIND == kJoining) {         // (asked for long before it is used)
                if (real && sees_prefix(p, t.b, position)) prefix = p.prefix_total[(long long)(t.row0 + token) * p.q_heads + head];
            }
            float factor = p.scale * kLog2e;
            if (tiles > 0) {
                // q -> shared memory; a negative scale goes into q, so that larger scores are larger weights
                const uint16_t* const from = static_cast<const uint16_t*>(p.q.p) + (t.row0 + token) * p.q.token + head * p.q.head;
                float down = 1.f, up = 1.f;
                uint4 x[D / 8];
#pragma unroll
                for (int u = 0; u < D / 8; ++u) {
                    x[u] = make_uint4(0, 0, 0, 0);
                    if (real) x[u] = *reinterpret_cast<const uint4*>(from + 8 * u);
                }
                if (BF16) {
                    float top = 0.f;
#pragma unroll
                    for (int u = 0; u < D / 8; ++u) top = fmaxf(top, fmaxf(bf16_most(make_uint2(x[u].x, x[u].y)), bf16_most(make_uint2(x[u].z, x[u].w))));
                    bf16_powers(top, up, down);
                }
                const uint32_t flip = factor < 0.f ? 0x80008000u : 0u;
                factor = fabsf(factor) * up;
#pragma unroll
                for (int u = 0; u < D / 8; ++u) {
                    uint2 a = make_uint2(x[u].x ^ flip, x[u].y ^ flip), b = make_uint2(x[u].z ^ flip, x[u].w ^ flip);
                    if (BF16) {
                        a = bf16_scaled(a, down);
                        b = bf16_scaled(b, down);
                    }
                    a = key_order<E4M3>(a);
                    b = key_order<E4M3>(b);
                    ptx::sts128(swizzled(q_tile[h], kHalf, row, u), make_uint4(a.x, a.y, b.x, b.y));
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&bars.q_full[h]);
            }
            float top = real ? -INFINITY : 0.f, sum = 0.f;                    // the reference that weights are taken relative to; their total
            // the warp's rows see a tile whole if the first of them does and, with a window, the last
            const int first_position = __shfl_sync(kAll, position, 0), last_position = __reduce_max_sync(kAll, position);
            for (int j = 0; j < tiles; ++j) {
                const int slot = (tile_count + j) % kScaleSlots;
                const int first = (t.tile0 + j) * kTokens;
                ok = wait_on(&bars.scale_full[slot], ((tile_count + j) / kScaleSlots) & 1, &s_abort) && wait_on(&bars.s_full[h], s_phase, &s_abort);
                if (!ok) break;
                s_phase ^= 1;
                ptx::tc_fence_after_sync();
                const bool all_real = __all_sync(kAll, real);
                const bool whole = all_real && (KIND == kPrefixes || first + kTokens - 1 <= first_position) && first + kTokens <= t.limit && first >= t.lo &&
                                   (!p.window || first > last_position - p.window);
                // tokens below `from` and at `to` and beyond are hidden from this row (relative to the tile)
                const int from = max(p.window ? position - p.window + 1 : 0, t.lo) - first, to = (KIND == kPrefixes ? (real ? t.limit : 0) : min(position + 1, t.limit)) - first;
                // Half a tile of tokens at a time: x = a * score + b of each 16 (a is not 0: hidden scores are -infinity), weights 2^x.  They are
                // taken relative to a reference that is no maximum any more once scores exceed it, which does no harm until the half's
                // weights add up to more than kMostWeight; then the reference moves, sums follow it, and the half is taken again.
                uint32_t x[2][32];
                const auto load = [&](int half) {
                    ptx::tmem_ld32(s_at + 64 * half, x[0]);
                    ptx::tmem_ld32(s_at + 64 * half + 32, x[1]);
                };
                const auto hide = [&](int half) {
                    if (whole) return;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (64 * half + 32 * c + i < from || 64 * half + 32 * c + i >= to) x[c][i] = 0xFF800000u;
                };
                load(0);
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    float total;
                    bool again = false;
#pragma unroll 1
                    for (;;) {
                        ptx::tc_wait_ld();
                        hide(half);
                        if (again || __any_sync(kAll, top == -INFINITY)) {
                            float high = -INFINITY;
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                float m = -INFINITY;
#pragma unroll
                                for (int i = 0; i < 16; i += 2) m = max3(m, __uint_as_float(x[g >> 1][16 * (g & 1) + i]), __uint_as_float(x[g >> 1][16 * (g & 1) + i + 1]));
                                const float4 sc = scales[slot][4 * half + g];
                                high = fmaxf(high, fmaf(m, fmaxf(factor * sc.x, kLeastFactor), sc.y));
                            }
                            const float next = fmaxf(top, high), keep = next == top ? 1.f : exp2_approx(top - next);     // (0 from -infinity on)
                            if ((j > 0 || half > 0) && __any_sync(kAll, keep != 1.f)) {
                                // (the scores of a tile come after the sums of the one before it)
                                if (half > 0) ok = wait_on(&bars.pv_half[h], pv_count & 1, &s_abort);
                                if (!ok) break;
                                ptx::tc_fence_after_sync();
#pragma unroll 1
                                for (int c = 0; c < D / 16; ++c) {
                                    uint32_t y[16];
                                    ptx::tmem_ld16(o_at + 16 * c, y);
                                    ptx::tc_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * keep);
                                    ptx::tmem_st16(o_at + 16 * c, y);
                                }
                            }
                            sum *= keep;
                            top = next;
                        }
                        // all exponents, then all exponentials, then sums and packing: the exponential pipe is fed without a pause
                        const float base = top == -INFINITY ? 0.f : top;
                        float2 part[4];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float4 sc = scales[slot][4 * half + g];
                            const float a = fmaxf(factor * sc.x, kLeastFactor), b = sc.y - base;
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                uint32_t* const s2 = &x[g >> 1][16 * (g & 1) + i];
                                const float2 y = fma2(make_float2(__uint_as_float(s2[0]), __uint_as_float(s2[1])), make_float2(a, a), make_float2(b, b));
                                s2[0] = __float_as_uint(y.x);
                                s2[1] = __float_as_uint(y.y);
                            }
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i) x[c][i] = __float_as_uint(exp2_approx(__uint_as_float(x[c][i])));
                        total = 0.f;
                        float largest = 0.f;
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            part[g] = make_float2(0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                part[g] = add2(part[g], make_float2(__uint_as_float(x[g >> 1][16 * (g & 1) + i]), __uint_as_float(x[g >> 1][16 * (g & 1) + i + 1])));
                            const float all = part[g].x + part[g].y;
                            largest = fmaxf(largest, all);
                            total = fmaf(all, scales[slot][4 * half + g].z, total);
                        }
                        if (again || !__any_sync(kAll, largest > kMostWeight)) break;
                        again = true;
                        load(half);
                    }
                    if (!ok) break;
                    sum += total;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = h2_as_u32(__floats2half2_rn(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1])));
                        ptx::tmem_st16(s_at + 32 * half + 16 * c, w);
                        if (half == 0) ptx::tmem_ld32(s_at + 64 + 32 * c, x[c]);
                    }
                    ptx::tc_wait_st();
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) arrive(&bars.p_full[h][half]);
                }
                if (!ok) break;
                ++pv_count;
            }
            tile_count += most;
            if (!ok) break;
            if (tiles > 0) {
                ok = wait_on(&bars.pv_done[h], (pv_count - 1) & 1, &s_abort);
                if (!ok) break;
                ptx::tc_fence_after_sync();
            }
            if (t.rows[h] > 0) {
                const long long to = ((long long)(t.row0 + token) * p.q_heads + head) * D;
                uint16_t* const out = static_cast<uint16_t*>(p.out) + to;
                // what the sums are multiplied with, once there are all of the row's own; the same of its prefix's
                const auto joint = [&](float m, float sum) {
                    if constexpr (KIND == kJoining) {
                        if (prefix.y < 0.f) {         // parts: joined where their sums would lie, for this thread alone
                            const float2 told = prefix;
#pragma unroll 1
                            for (int c = 0; c < D; c += 4) {
                                alignas(16) float x[4];
                                prefix = prefix_sums(p, told, 0, c, x);
                                *reinterpret_cast<float4*>(p.prefix_sums + to + c) = make_float4(x[0], x[1], x[2], x[3]);
                            }
                        }
                        return join_prefix(m, sum, prefix);
                    }
                    return Joint{sum > 0.f ? 1.f / sum : sum, 0.f};                           // (a NaN stays one)
                };
                float* const kept = KIND == kPrefixes ? p.prefix_sums + to : nullptr;
                const auto prefix4 = [&](int at) { return *reinterpret_cast<const float4*>(p.prefix_sums + to + at); };
                if (t.part < 0) {
                    const Joint both = joint(top, sum);
                    const float f = both.own;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t x[32] = {};
                        if (tiles > 0) {
                            ptx::tmem_ld32(o_at + 32 * c, x);
                            ptx::tc_wait_ld();
                        }
                        if constexpr (KIND == kPrefixes) {
                            if (real)
#pragma unroll
                                for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(kept + 32 * c + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                        } else if (KIND == kJoining && both.prefix != 0.f) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                const float4 a = prefix4(32 * c + i), b = prefix4(32 * c + i + 4);
                                const float z[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                                uint32_t y[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    y[k] = pack_out<BF16>(fmaf(__uint_as_float(x[i + 2 * k]), f, z[2 * k] * both.prefix),
                                                          fmaf(__uint_as_float(x[i + 2 * k + 1]), f, z[2 * k + 1] * both.prefix));
                                *reinterpret_cast<uint4*>(out + 32 * c + i) = make_uint4(y[0], y[1], y[2], y[3]);
                            }
                        } else if (real) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                uint32_t y[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) y[k] = pack_out<BF16>(__uint_as_float(x[i + 2 * k]) * f, __uint_as_float(x[i + 2 * k + 1]) * f);
                                *reinterpret_cast<uint4*>(out + 32 * c + i) = make_uint4(y[0], y[1], y[2], y[3]);
                            }
                        }
                        if (KIND != kOwn) __syncwarp();
                    }
                    if constexpr (KIND == kPrefixes) {
                        if (real) p.prefix_total[(long long)(t.row0 + token) * p.q_heads + head] = make_float2(top, sum);
                    }
                } else {
                    float* const parts = reinterpret_cast<float*>(header + p.prompt_parts) + (size_t)h * L::kPartFloats;
                    const auto part_at = [&](int i) { return parts + (size_t)(t.part + i) * 2 * L::kPartFloats; };
                    float* const own = part_at(t.which);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t x[32] = {};
                        if (tiles > 0) {
                            ptx::tmem_ld32(o_at + 32 * c, x);
                            ptx::tc_wait_ld();
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4*>(own + ((8 * c + i) * kHalf + row) * 4) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                    }
                    own[kHalf * D + row] = top;
                    own[kHalf * D + kHalf + row] = sum;
                    __threadfence();
                    meet();
                    if (!ok) break;
                    if (row == 0) {
                        unsigned int* const counter = reinterpret_cast<unsigned int*>(header + kPromptCounters) + 2 * t.part + h;
                        const bool last = atomicAdd(counter, 1u) == (unsigned int)(t.parts - 1);
                        if (last) atomicExch(counter, 0u);
                        s_last[h] = last;
                        __threadfence();
                    }
                    meet();
                    if (!ok) break;
                    if (s_last[h] && real) {
                        __threadfence();
                        // (every pass over the parts has independent loads only: what it costs is their latency)
                        float m = -INFINITY, total = 0.f;
#pragma unroll 4
                        for (int i = 0; i < t.parts; ++i) m = fmaxf(m, __ldcg(part_at(i) + kHalf * D + row));
                        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll 4
                        for (int i = 0; i < t.parts; ++i)
                            total += exp2_approx(__ldcg(part_at(i) + kHalf * D + row) - from) * __ldcg(part_at(i) + kHalf * D + kHalf + row);
                        const Joint both = joint(m, total);
                        const float f = KIND == kPrefixes ? 1.f : both.own;
                        if constexpr (KIND == kPrefixes) p.prefix_total[(long long)(t.row0 + token) * p.q_heads + head] = make_float2(m, total);
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float y[32] = {};
                            if constexpr (KIND == kJoining) {
                                if (both.prefix != 0.f)
#pragma unroll
                                    for (int k = 0; k < 8; ++k) {
                                        const float4 x = prefix4(c + 4 * k);
                                        y[4 * k] = x.x * both.prefix;
                                        y[4 * k + 1] = x.y * both.prefix;
                                        y[4 * k + 2] = x.z * both.prefix;
                                        y[4 * k + 3] = x.w * both.prefix;
                                    }
                            }
#pragma unroll 2
                            for (int i = 0; i < t.parts; ++i) {
                                const float take = exp2_approx(__ldcg(part_at(i) + kHalf * D + row) - from) * f;
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float4 x = __ldcg(reinterpret_cast<const float4*>(part_at(i) + ((c / 4 + k) * kHalf + row) * 4));
                                    y[4 * k] += take * x.x;
                                    y[4 * k + 1] += take * x.y;
                                    y[4 * k + 2] += take * x.z;
                                    y[4 * k + 3] += take * x.w;
                                }
                            }
                            if constexpr (KIND == kPrefixes) {
#pragma unroll
                                for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(kept + c + k) = make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
                                continue;
                            }
#pragma unroll
                            for (int k = 0; k < 32; k += 8)
                                *reinterpret_cast<uint4*>(out + c + k) = make_uint4(pack_out<BF16>(y[k], y[k + 1]), pack_out<BF16>(y[k + 2], y[k + 3]),
                                                                                    pack_out<BF16>(y[k + 4], y[k + 5]), pack_out<BF16>(y[k + 6], y[k + 7]));
                        }
                    }
                    meet();                                                   // (s_last is free again)
                    if (!ok) break;
                }
            }
            // what was read of the sums is read before the next item's products overwrite them
            ptx::tc_fence_before_sync();
            done_with_item(n);
        }
    }

    if (KIND == kPrefixes) ptx::grid_dependency_wait();
    if (lane == 0 && s_abort) atomicExch(status, 61);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    if (warp == kMma) ptx::tmem_dealloc(tmem, 512);
}

template <bool E4M3, bool BF16, int D, int KIND>
cudaError_t launch_prompt(const AttentionParams& p, int least_rows, bool alone, cudaStream_t stream) {
    const auto kernel = cache_prompt_kernel<E4M3, BF16, D, KIND>;
    constexpr int kSmem = Layout<D>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(kMaxBlocks, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p, least_rows, alone ? 1 : 0);
    if (e == cudaSuccess) count_launch();
    return e;
}

template <int KIND>
cudaError_t by_types(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, bool alone, cudaStream_t stream) {
    const auto by_dim = [&](auto e, auto h) {
        constexpr bool E = decltype(e)::value, H = decltype(h)::value;
        return p.cache.dim == 128 ? launch_prompt<E, H, 128, KIND>(p, least_rows, alone, stream) : launch_prompt<E, H, 64, KIND>(p, least_rows, alone, stream);
    };
    const auto by_type = [&](auto e) { return bf16 ? by_dim(e, std::true_type{}) : by_dim(e, std::false_type{}); };
    return e4m3 ? by_type(std::true_type{}) : by_type(std::false_type{});
}

}  // namespace

size_t cache_prompt_workspace() { return (size_t)kPromptParts * 2 * Layout<128>::kPartFloats * 4; }

cudaError_t cache_prompt_launch(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, bool alone, cudaStream_t stream) {
    return p.prefix_of ? by_types<kJoining>(p, e4m3, bf16, least_rows, alone, stream) : by_types<kOwn>(p, e4m3, bf16, least_rows, alone, stream);
}

cudaError_t cache_many_readers_launch(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, cudaStream_t stream) {
    return by_types<kPrefixes>(p, e4m3, bf16, least_rows, false, stream);
}

}  // namespace i4mm
