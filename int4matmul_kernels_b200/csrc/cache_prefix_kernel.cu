// Attention of all rows that read a shared prefix over that prefix (the first half of i4mm_cache_attention_shared).
//
//   x_j = log2(e) * scale * s_key * (q . k_j) + log2(s_value),  P_j = 2^(x_j - M)   (fp16), with a reference M, an x_j of the row,
//   total = sum_j P_j / s_value,  sums = sum_j P_j v_j      over the prefix's tokens that the row sees, k_j and v_j the cache's bytes
// M, total and sums of each row are what the kernel of its own tokens adds to its own.  Weights are rounded to fp16 for the product, as the prompt kernel's are
// (2^-11 of each, and they are rounded apart from one another): against 64 bits an fp16 output is off by 2.5e-4 to 2.9e-4 of its norm, by 2.1e-4 where it alone
// is rounded.  Carrying the rounding errors, as the few-row kernel does, would double the weights' shared memory and the second product.
//
// The rows of all readers of a place, times the query heads of a key head, are the rows of tiles of up to 64.  With so few rows for each byte the floor is DRAM's (a
// tile of 128 tokens is 32 KB at head_dim 128, 1400 cycles of an SM's share; what bounds the kernel instead stands below), and many columns are what the
// tensor cores do not have to be given, so tokens are the 128 rows of both products and the readers their columns, as many as there are:
//
//   S^T = K Q^T      K: bytes -> fp16 -> tensor memory, a thread a token (no trip through shared memory, no transposition); Q: shared memory
//   O^T = V^T P^T    V: bytes -> fp16 -> shared memory as they lie (dim fastest); P: shared memory, a thread a token
// A thread of the softmax has one token, so a page's scales are its constants; it keeps its part of each row's total in a register, and nothing is summed
// over threads until the end.  The largest score is looked for only where a weight would exceed 2^14: then sums follow to a new reference.
//
//   warps 0..15        softmax: two sets, which take tiles in turns, of four warps (32 tokens each) for either half of the rows
//   warps 16..19       the rows' queries; bytes to operands
//   warp 20            issues the products
//   warps 21, 22       fetch pages into rings, a TMA copy a page, keys and values; the first deals out the work
//
// The tiles of all segments (place, key head, up to 64 rows) in a row are dealt out in equal contiguous ranges to the blocks.  What a range cuts goes through
// the workspace: few parts are added up by the block that comes last, many by those who read the rows (kJoined).  Nobody waits for another block.  Waits
// are bounded: a warp that gives up sets the abort flag, which ends every other wait of the block, and the status word.
//
// What bounds it: the steps of a tile one after the other.  A set takes 6200 cycles for one of its tiles (64 rows, head_dim 64): scores 450, weights 3700, the
// product with the values 800; the decoding warps are busy for 2600 of the 3100 a tile (at head_dim 128 as long as the softmax).  A block's first scores
// come after 12000 cycles (loads that depend on one another, code that is not there yet), and a further segment costs 6000 to 20000.  Issue slots are
// filled to 42 %, the tensor cores to 8.  One set of softmax warps instead of two: 64 readers with 40 heads, 4000 tokens 151 us
// with the kernel of own tokens, for 132.
#include <algorithm>
#include <type_traits>

#include "cache_attention.cuh"

namespace i4mm {
namespace {

constexpr int kTokens = 128;                          // of a tile
constexpr int kMostRows = kPrefixRows;
constexpr int kHalves = 2, kColumns = kMostRows / kHalves;                   // of a tile's rows; columns of each
constexpr int kSoftmaxWarps = 4 * 2 * kHalves, kDecode0 = kSoftmaxWarps, kDecodeWarps = 4, kMma = kDecode0 + 4, kCopy = kMma + 1, kCopyValues = kCopy + 1;
constexpr int kThreads = 32 * (kCopyValues + 1);
constexpr int kStages = 3;                            // of either ring
constexpr int kItems = 4, kScales = 4, kRawScales = 8;
constexpr int kPieces = kTokens / 16;                 // pages of a tile, at most
// Parts of a segment that one block adds up; 3 / 6 / 10, us with the kernel of own tokens: 64 rows over 4000 tokens, 40 heads (4 parts) 176 / 128 / 128, 8 rows of
// 8 heads (8 parts) 26.8 / 26.9 / 30.0, 16 over 16000 49.4 / 49.5 / 53.8
constexpr int kJoined = 6;
constexpr int kMinBlockTiles = 4;                     // fewer tiles than this are not cut further, nor twice as many of whole segments
constexpr float kNone = -3e38f;                       // a reference below any score
constexpr float kMostLog = 14.f;                      // fp16 holds 2^16
constexpr uint32_t kNoPage = 0x7FC0DEADu;             // in the place of a scale: there is no such page
constexpr uint32_t kMnStride = 16384;                 // 128 tokens of 64 columns

template <int D>
struct Layout {
    static constexpr int kHalf = kTokens * D;                                 // bytes of a tile's keys or values
    static constexpr int kV = 2 * kMnStride, kP = kMnStride, kQ = kMostRows * D * 2;         // V and P: one of two
    static constexpr int kV0 = 0, kP0 = kV0 + 2 * kV, kQ0 = kP0 + 2 * kP, kKeys0 = kQ0 + kQ, kValues0 = kKeys0 + kStages * kHalf,
                         kBytes = kValues0 + kStages * kHalf + 1024;
    static constexpr int kPartFloats = kMostRows * D + 2 * kMostRows;         // sums [row][dim], (reference, total) [row]
};
constexpr size_t kPartsBytes = (size_t)kMaxBlocks * 2 * Layout<128>::kPartFloats * 4;

struct Item {
    int valid, place, head, base, rows, n;            // base: first row of the tile; n: rows, rounded up to 16
    int first;                                        // of the place's readers in the list
    int lo, limit;                                    // tokens that may be seen
    int tile0, tiles;
    int first_block, last_block;                      // that have a part of its segment; one alone: the item is all of it
};

struct Barriers {
    unsigned long long item_full[kItems], item_empty[kItems], q_full[kItems], scale_full[kScales];
    unsigned long long keys_full[kStages], keys_empty[kStages], values_full[kStages], values_empty[kStages];
    unsigned long long k_full[2], s_full[2], p_full[2], v_full[2], pv_done[2], drained;
};

// A whole warp waits; false (in all of its lanes) once the block gives up.
__device__ __noinline__ bool wait_longer(uint32_t at, uint32_t parity, volatile int* abort) {
    for (uint32_t i = 0; i < ptx::kSpinLimit; ++i) {
        if (__all_sync(kAll, ptx::mbar_try_wait(at, parity))) return true;
        if (__any_sync(kAll, *abort)) return false;
    }
    *abort = 1;
    return false;
}
__device__ __forceinline__ bool wait_on(unsigned long long* bar, uint32_t parity, volatile int* abort) {
    const uint32_t at = ptx::smem_u32(bar);
    if (__all_sync(kAll, ptx::mbar_try_wait(at, parity & 1))) return true;
    return wait_longer(at, parity & 1, abort);
}
__device__ __forceinline__ void arrive(unsigned long long* bar) { ptx::mbar_arrive(ptx::smem_u32(bar)); }

// ---- work ----------------------------------------------------------------------------------------------------------------------
struct Place {
    int first, rows;                                  // of its readers in the list; readers times query heads of a key head
    int lo, limit, tiles;                             // tokens that any row sees; at least one tile, so that all rows are written
    int row_tiles, height;                            // rows of a row tile: all of a place alike
};
__device__ __forceinline__ Place load_place(const AttentionParams& p, int most_rows, int b) {
    Place r;
    const int from = min(max(p.prefix_starts[b], 0), p.prefix_listed), to = min(max(p.prefix_starts[b + 1], 0), p.prefix_listed), seq = p.seq_lens[b];
    r.first = from;
    r.rows = min(max(to - from, 0), p.tokens) * p.group;                      // (tokens * q_heads is below 2^31)
    if (r.rows > most_rows) r.rows = 0;                                       // the other kernel's
    r.limit = max(min(seq, p.table_width << p.cache.page_shift), 0);
    r.lo = p.window && seq >= p.window ? min(seq - p.window + 1, r.limit) : 0;
    r.tiles = max((r.limit + kTokens - 1) / kTokens - r.lo / kTokens, 1);
    r.row_tiles = (r.rows + kMostRows - 1) / kMostRows;
    r.height = (r.rows + 15) & ~15;
    if (r.row_tiles > 1) r.height = (int)(((uint32_t)r.rows + 16u * r.row_tiles - 1) / (16u * r.row_tiles)) * 16;
    return r;
}
// (the host has made sure that all of these together are below 2^31)
__device__ __forceinline__ uint32_t segments_of(const AttentionParams& p, const Place& r) { return (uint32_t)(r.row_tiles * p.cache.heads); }

// ---- two fp32 at a time ----
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
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

// 32 values of each lane -> lane l has the result over all lanes of value l
template <int DISTANCE, typename F>
__device__ __forceinline__ void reduce_step(uint32_t (&x)[32], F op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < DISTANCE; ++i) {
        const uint32_t send = lane & DISTANCE ? x[i] : x[i + DISTANCE], keep = lane & DISTANCE ? x[i + DISTANCE] : x[i];
        x[i] = __float_as_uint(op(__uint_as_float(keep), __uint_as_float(__shfl_xor_sync(kAll, send, DISTANCE))));
    }
}
template <typename F>
__device__ __forceinline__ float reduce32(uint32_t (&x)[32], F op) {
    reduce_step<16>(x, op);
    reduce_step<8>(x, op);
    reduce_step<4>(x, op);
    reduce_step<2>(x, op);
    reduce_step<1>(x, op);
    return __uint_as_float(x[0]);
}

// address of 16 bytes (8 values) `unit` of `row` in Q: sub-tiles of 64 values, 128-byte rows, swizzled
__device__ __forceinline__ uint32_t swizzled(uint32_t tile, int row, int unit) {
    return tile + (unit >> 3) * (kMostRows * 128) + row * 128 + (((unit & 7) ^ (row & 7)) << 4);
}
// V and P: blocks of 64 columns, a token's 128 bytes to a row, swizzled in the same way.
// Matrix descriptor of such an operand: its columns are the M or N of a product, its tokens the K.  8 tokens 1024 bytes apart, blocks of 64 columns kMnStride
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(kMnStride >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
constexpr uint32_t kBothMn = (1u << 15) | (1u << 16); // of an instruction descriptor: A and B lie so

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(kThreads, 1) cache_prefix_kernel(const AttentionParams p, int most_rows, const __grid_constant__ CUtensorMap k_map,
                                                                   const __grid_constant__ CUtensorMap v_map) {
    using L = Layout<D>;
    extern __shared__ uint8_t dynamic[];
    __shared__ Barriers bars;
    __shared__ Item items[kItems];
    __shared__ float2 s_raw[kRawScales][kPieces];
    __shared__ float4 s_scale[kScales][kPieces];      // key scale, log2 of the value scale, its inverse, whether there is such a page
    __shared__ int s_row[kItems][kMostRows];          // packed row times query heads plus head; -1: none
    __shared__ long long s_query[kItems][kMostRows];  // where its query lies (a warp may write the next item's while another one reads this one's)
    __shared__ int s_low[kItems][kMostRows];          // the first token that the row sees
    __shared__ __align__(16) float s_up[kItems][kMostRows];                   // what its scores are multiplied with (bf16; read four at a time)
    __shared__ int s_most_low[kItems];
    // (by set and half)
    __shared__ __align__(16) float s_minus_top[2 * kHalves][kColumns];        // the rows' references, their signs turned over
    __shared__ __align__(16) float s_keep[2 * kHalves][kColumns];
    __shared__ float s_warps[2 * kHalves][4][kColumns];
    __shared__ volatile uint32_t s_need[2 * kHalves][2];
    __shared__ float2 s_take[kMostRows];              // of a row, what either set's sums are multiplied with
    __shared__ volatile int s_abort, s_last[kHalves];
    __shared__ uint32_t tmem_smem;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem = (ptx::smem_u32(dynamic) + 1023u) & ~1023u;
    const uint32_t q_tile = smem + L::kQ0, v_tile = smem + L::kV0, p_tile = smem + L::kP0, keys_ring = smem + L::kKeys0, values_ring = smem + L::kValues0;
    uint8_t* const header = static_cast<uint8_t*>(p.workspace);
    const CacheView& cache = p.cache;
    const int page_shift = cache.page_shift, pieces = kTokens >> page_shift;

    if (threadIdx.x == 0) {
        const auto init = [](unsigned long long& b, uint32_t n) { ptx::mbar_init(ptx::smem_u32(&b), n); };
#pragma unroll 1
        for (int i = 0; i < kItems; ++i) {
            init(bars.item_full[i], 1);
            init(bars.item_empty[i], kSoftmaxWarps + kDecodeWarps + 2);
            init(bars.q_full[i], kDecodeWarps);
        }
#pragma unroll 1
        for (int i = 0; i < kStages; ++i) {
            init(bars.keys_full[i], 2 * pieces);      // each lane's bytes, and its scales
            init(bars.keys_empty[i], kDecodeWarps);
        }
#pragma unroll 1
        for (int i = 0; i < kStages; ++i) {
            init(bars.values_full[i], pieces);
            init(bars.values_empty[i], kDecodeWarps);
        }
#pragma unroll 1
        for (int i = 0; i < kScales; ++i) init(bars.scale_full[i], 1);
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            init(bars.k_full[i], kDecodeWarps);
            init(bars.s_full[i], 1);
            init(bars.p_full[i], kSoftmaxWarps / 2);
            init(bars.pv_done[i], 1);
            init(bars.v_full[i], kDecodeWarps);
        }
        init(bars.drained, 1);
        ptx::fence_mbar_init();
        s_abort = 0;
#pragma unroll 1
        for (int i = 0; i < 4 * kHalves; ++i) s_need[i >> 1][i & 1] = 0;
    }
    if (D == 64)                                      // the columns of V that there are not
#pragma unroll 1
        for (int i = threadIdx.x; i < (int)kMnStride / 16; i += kThreads) {
            ptx::sts128(v_tile + kMnStride + 16 * i, make_uint4(0, 0, 0, 0));
            ptx::sts128(v_tile + L::kV + kMnStride + 16 * i, make_uint4(0, 0, 0, 0));
        }
    ptx::fence_proxy_async_smem();
    if (warp == kMma) {
        ptx::tmem_alloc(ptx::smem_u32(&tmem_smem), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = tmem_smem;
    const auto s_col = [&](uint32_t g) { return tmem + (g & 1) * kMostRows; };
    const auto o_col = [&](uint32_t g) { return tmem + (2 + (g & 1)) * kMostRows; };
    const auto k_col = [&](uint32_t g) { return tmem + 4 * kMostRows + (g & 1) * 64; };
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    // Named barriers among four warps.  One that gives up arrives once more as it leaves (s_abort is set by then), which lets the others through to see it.
    const auto meet = [&](int id, int threads) -> bool {
        ptx::named_bar_sync(id, threads);
        return !__any_sync(kAll, s_abort);
    };
    const auto done_with_item = [&](uint32_t n) {
        __syncwarp();
        if (lane == 0) arrive(&bars.item_empty[n % kItems]);
    };
    const auto next_item = [&](uint32_t n) { return wait_on(&bars.item_full[n % kItems], n / kItems, &s_abort); };
    // Fetches an item's keys or values into a ring, a page to a lane; g: tiles before it.
    uint32_t fetched = 0;
    const auto copy = [&](const Item& t, uint32_t g, const CUtensorMap* map, uint32_t ring, unsigned long long* full, unsigned long long* empty, uint32_t stages,
                          bool scales) -> bool {
        const int* const table = p.table + t.place * p.table_stride;
        int page = -1;
        const auto find_page = [&](int j) {           // lane l: the tile's l-th
            const int token = (t.tile0 + j) * kTokens + (lane << page_shift), i = token >> page_shift;
            page = -1;
            if (lane < pieces && token < t.limit && token + (1 << page_shift) > t.lo && i < p.table_width) page = table[i];
        };
        find_page(0);
#pragma unroll 1
        for (int j = 0; j < t.tiles; ++j, ++g) {
            const int id = (unsigned int)page < (unsigned int)cache.pages ? page : -1;
            if (j + 1 < t.tiles) find_page(j + 1);
            const uint32_t slot = g % stages, bar = ptx::smem_u32(&full[slot]);
            if (!wait_on(&empty[slot], (g / stages) ^ 1, &s_abort)) return false;
            if (lane < pieces) {
                if (id >= 0) {
                    ptx::mbar_arrive_expect_tx(bar, D << page_shift);
                    ptx::tma_load_4d(ring + slot * L::kHalf + lane * (D << page_shift), map, 0, 0, t.head, id, bar);
                } else {
                    ptx::mbar_arrive(bar);
                }
                if (scales) {
                    if (id >= 0) {
                        ptx::cp_async_8(ptx::smem_u32(&s_raw[g % kRawScales][lane]), cache.scales + (long long)id * cache.heads + t.head);
                        ptx::cp_async_arrive(bar);
                    } else {
                        s_raw[g % kRawScales][lane] = make_float2(__uint_as_float(kNoPage), 0.f);
                        ptx::mbar_arrive(bar);
                    }
                }
            }
            __syncwarp();
            fetched = g + 1;
        }
        return true;
    };
    // A block that gives up waits, bounded again, for what is on its way to its rings: the shared memory is someone else's once it has ended.
    const auto landed = [&](unsigned long long* full, uint32_t stages) {
#pragma unroll 1
        for (uint32_t i = fetched > stages ? fetched - stages : 0; i < fetched; ++i) (void)ptx::mbar_wait(ptx::smem_u32(&full[i % stages]), (i / stages) & 1);
    };

    if (warp == kCopy) {
        // the block's range: all have the same number of tiles, but for those at the end.  The first 32 places stay in the lanes' registers.
        Place mine{};
        uint32_t segments = 0, all_tiles = 0, longest = 0;
        if (lane < p.requests) {
            mine = load_place(p, most_rows, lane);
            segments = segments_of(p, mine);
            all_tiles = segments * mine.tiles;
            longest = segments ? mine.tiles : 0;
        }
#pragma unroll 1
        for (int b = lane + 32; b < p.requests; b += 32) {
            const Place r = load_place(p, most_rows, b);
            segments += segments_of(p, r);
            all_tiles += segments_of(p, r) * r.tiles;
            if (r.row_tiles) longest = max(longest, (uint32_t)r.tiles);
        }
        segments = __reduce_add_sync(kAll, segments);
        all_tiles = __reduce_add_sync(kAll, all_tiles);
        longest = __reduce_max_sync(kAll, longest);
        const uint32_t begin = segments * 8 < gridDim.x ? 0 : kPrefixBegin, total = all_tiles + segments * begin;
        const uint32_t least = (longest <= 2 * kMinBlockTiles ? longest : kMinBlockTiles) + begin;
        const auto units_of = [&](const Place& r) { return segments_of(p, r) * (r.tiles + begin); };
        const uint32_t share = max((total + gridDim.x - 1) / gridDim.x, max(least, 1u));
        uint32_t own = units_of(mine), at = min(blockIdx.x * share, total);
        const uint32_t end = min(at + share, total);
        // the place that the range begins in
        uint32_t before = 0;
        int b = 0;
        Place r{};
        const auto find_place = [&]() {               // from request b (a multiple of 32) on, `before` tiles before it
#pragma unroll 1
            for (; b < p.requests; b += 32) {
                if (b > 0) {
                    mine = b + lane < p.requests ? load_place(p, most_rows, b + lane) : Place{};
                    own = units_of(mine);
                }
                uint32_t upto = own;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const uint32_t o = __shfl_up_sync(kAll, upto, d);
                    if (lane >= d) upto += o;
                }
                const uint32_t here = __ballot_sync(kAll, before + upto > at);
                if (here) {
                    const int l = __ffs(here) - 1;
                    before += __shfl_sync(kAll, upto - own, l);
                    b += l;
                    r.first = __shfl_sync(kAll, mine.first, l);
                    r.rows = __shfl_sync(kAll, mine.rows, l);
                    r.lo = __shfl_sync(kAll, mine.lo, l);
                    r.limit = __shfl_sync(kAll, mine.limit, l);
                    r.tiles = __shfl_sync(kAll, mine.tiles, l);
                    r.row_tiles = __shfl_sync(kAll, mine.row_tiles, l);
                    r.height = __shfl_sync(kAll, mine.height, l);
                    return;
                }
                before += __shfl_sync(kAll, upto, 31);
            }
        };
        uint32_t n = 0, g = 0;                        // items, tiles so far
        bool ok = true, placed = false;
#pragma unroll 1
        while (ok && at < end) {
            if (!placed || at >= before + units_of(r)) {
                // (the next place with rows: from the multiple of 32 at or below the current one, whose earlier tiles are counted again)
                if (placed) {
                    before += units_of(r);
                    ++b;
#pragma unroll 1
                    for (; b < p.requests && (b & 31); ++b) {
                        r = load_place(p, most_rows, b);
                        if (r.rows > 0) break;
                    }
                    if (b < p.requests && !(b & 31)) find_place();
                } else {
                    find_place();
                }
                if (b >= p.requests) break;           // (not unless the lengths change under the kernel)
                placed = true;
            }
            Item t;
            {
                const uint32_t length = r.tiles + begin, segment = (at - before) / length, from = before + segment * length, stop = min(from + length, end);
                const int tile = max((int)(at - from - begin), 0), tiles = (int)(stop - from - begin) - tile;
                at = stop;
                if (tiles <= 0) continue;             // (what it costs to begin is this block's, the tiles are the next one's)
                const int head = (int)segment / r.row_tiles, row_tile = (int)segment - head * r.row_tiles;
                t.valid = 1;
                t.place = b;
                t.head = head;
                t.base = row_tile * r.height;
                t.rows = max(min(r.height, r.rows - t.base), 0);
                t.n = max((t.rows + 15) & ~15, 16);
                t.first = r.first;
                t.lo = r.lo;
                t.limit = r.limit;
                t.tile0 = r.lo / kTokens + tile;
                t.tiles = tiles;
                t.first_block = t.last_block = (int)blockIdx.x;
                if (t.tiles < r.tiles) {
                    t.first_block = (int)((from + begin) / share);
                    t.last_block = (int)((from + length - 1) / share);
                }
            }
            ok = wait_on(&bars.item_empty[n % kItems], (n / kItems) ^ 1, &s_abort);
            if (!ok) break;
            if (lane == 0) {
                items[n % kItems] = t;
                arrive(&bars.item_full[n % kItems]);
            }
            __syncwarp();
            ++n;
            ok = copy(t, g, &k_map, keys_ring, bars.keys_full, bars.keys_empty, kStages, true);
            g += t.tiles;
        }
        if (ok) ok = wait_on(&bars.item_empty[n % kItems], (n / kItems) ^ 1, &s_abort);
        if (ok && lane == 0) {
            items[n % kItems].valid = 0;
            arrive(&bars.item_full[n % kItems]);
        }
        if (!ok) landed(bars.keys_full, kStages);
    } else if (warp == kCopyValues) {
        uint32_t g = 0;
        bool ok = true;
#pragma unroll 1
        for (uint32_t n = 0; ok; ++n) {
            ok = next_item(n);
            if (!ok || !items[n % kItems].valid) break;
            const Item t = items[n % kItems];
            ok = copy(t, g, &v_map, values_ring, bars.values_full, bars.values_empty, kStages, false);
            g += t.tiles;
            done_with_item(n);
        }
        if (!ok) landed(bars.values_full, kStages);
    } else if (warp == kMma) {
        // ---- products ----
        uint32_t g = 0;
        bool ok = true;
#pragma unroll 1
        for (uint32_t n = 0; ok; ++n) {
            ok = next_item(n);
            if (!ok || !items[n % kItems].valid) break;
            const int tiles = items[n % kItems].tiles, columns = items[n % kItems].n;
            const uint32_t idesc = ptx::idesc_f16_m128(columns), idesc_mn = idesc | kBothMn;
            ok = wait_on(&bars.q_full[n % kItems], n / kItems, &s_abort);
            const auto score = [&](uint32_t i) {      // S_i = K_i Q^T; the weights of tile i - 2 are there by now, so its scores have been read
                ok = ok && wait_on(&bars.k_full[i & 1], i >> 1, &s_abort);
                if (!ok) return;
                ptx::tc_fence_after_sync();
                if (ptx::elect_one()) {
                    const uint64_t b = ptx::smem_desc_sw128(q_tile);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        ptx::umma_f16_ts(s_col(i), k_col(i) + 8 * k, b + (uint64_t)((k >> 2) * (kMostRows * 128 >> 4) + (k & 3) * 2), idesc, k > 0);
                    ptx::tc_commit(ptx::smem_u32(&bars.s_full[i & 1]));
                }
                __syncwarp();
            };
            score(g);
            if (tiles > 1) score(g + 1);
#pragma unroll 1
            for (int j = 0; j < tiles && ok; ++j) {
                const uint32_t i = g + j;
                ok = wait_on(&bars.v_full[i & 1], i >> 1, &s_abort) && wait_on(&bars.p_full[i & 1], i >> 1, &s_abort);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                if (ptx::elect_one()) {
                    const uint64_t a = smem_desc_mn(v_tile + (i & 1) * L::kV), b = smem_desc_mn(p_tile + (i & 1) * L::kP);
#pragma unroll
                    for (int k = 0; k < kTokens / 16; ++k) ptx::umma_f16_ss(o_col(i), a + (uint64_t)(k * 2048 >> 4), b + (uint64_t)(k * 2048 >> 4), idesc_mn, j > 1 || k > 0);
                    ptx::tc_commit(ptx::smem_u32(&bars.pv_done[i & 1]));
                }
                __syncwarp();
                if (j + 2 < tiles) score(i + 2);
            }
            g += tiles;
            done_with_item(n);
        }
        // nothing of this block may be in flight when its tensor memory goes
        if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars.drained));
        __syncwarp();
#pragma unroll 1
        for (uint32_t i = 0; i < ptx::kSpinLimit && !ptx::mbar_try_wait(ptx::smem_u32(&bars.drained), 0); ++i) {}
    } else if (warp >= kDecode0) {
        // ---- queries; bytes to operands ----
        constexpr int kMeet = 7;
        const int w = warp - kDecode0, tid = w * 32 + lane;
        constexpr int kUnits = D / 8;                 // of 16 bytes in a query
        uint32_t g = 0;
        bool ok = true;
#pragma unroll 1
        for (uint32_t n = 0; ok; ++n) {
            ok = next_item(n);
            if (!ok || !items[n % kItems].valid) break;
            const uint32_t slot = n % kItems;
            const Item t = items[slot];
            // whose rows they are
            {
                int id = -1, low = 0;
                long long query = 0;
                if (tid < t.rows) {
                    const int in = t.base + tid, entry = t.first + in / p.group, token = entry < p.prefix_listed ? p.prefix_rows[entry] : -1;
                    if (token >= 0 && token < p.tokens) {
                        const int h = t.head * p.group + in % p.group;
                        id = token * p.q_heads + h;
                        query = token * p.q.token + h * p.q.head;
                        if (p.window) {
                            low = min(max(behind_prefix(p, t.place, token) - p.window + 1, 0), t.limit);
                        }
                    }
                }
                if (tid < kMostRows) {
                    s_row[slot][tid] = id;
                    s_query[slot][tid] = query;
                    s_low[slot][tid] = low;
                }
                const int most = __reduce_max_sync(kAll, low);
                if (p.window) {
                    if (tid == 0) s_most_low[slot] = 0;
                    if (!(ok = meet(kMeet, 128))) break;
                    if (lane == 0) atomicMax(&s_most_low[slot], most);
                } else if (tid == 0) {
                    s_most_low[slot] = 0;
                }
            }
            if (!(ok = meet(kMeet, 128))) break;
            // (the scores of the item before are complete)
            if (g > 0 && !(ok = wait_on(&bars.s_full[(g - 1) & 1], (g - 1) >> 1, &s_abort))) break;
            constexpr int kAtOnce = 4, kRowsAtOnce = 32 / kUnits;             // of a warp
#pragma unroll 1
            for (int r0 = w * kRowsAtOnce; r0 < t.n; r0 += kAtOnce * 4 * kRowsAtOnce) {
                uint4 x[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const int r = r0 + i * 4 * kRowsAtOnce + lane / kUnits, id = r < t.n ? s_row[slot][r] : -1;
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (id >= 0) x[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q.p) + s_query[slot][r] + 8 * (lane % kUnits));
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const int r = r0 + i * 4 * kRowsAtOnce + lane / kUnits;
                    uint2 a = make_uint2(x[i].x, x[i].y), b = make_uint2(x[i].z, x[i].w);
                    if (BF16) {
                        float most = fmaxf(bf16_most(a), bf16_most(b)), up, down;
#pragma unroll
                        for (int d = kUnits / 2; d; d /= 2) most = fmaxf(most, __shfl_xor_sync(kAll, most, d));
                        bf16_powers(most, up, down);
                        a = bf16_scaled(a, down);
                        b = bf16_scaled(b, down);
                        if (lane % kUnits == 0 && r < t.n) s_up[slot][r] = up;
                    }
                    a = key_order<E4M3>(a);
                    b = key_order<E4M3>(b);
                    if (r < t.n) ptx::sts128(swizzled(q_tile, r, lane % kUnits), make_uint4(a.x, a.y, b.x, b.y));
                }
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&bars.q_full[slot]);

            const auto seen_at = [&](uint32_t g, int first, int token) {
                return first + token >= t.lo && first + token < t.limit && __float_as_uint(s_raw[g % kRawScales][token >> page_shift].x) != kNoPage;
            };
            const auto all_there = [&](uint32_t g, int first) {
                return __all_sync(kAll, __float_as_uint(s_raw[g % kRawScales][lane & (pieces - 1)].x) != kNoPage) && first >= t.lo && first + kTokens <= t.limit;
            };
            // keys: a thread a token
            const auto keys = [&](int j) -> bool {
                const uint32_t i = g + j, at = i % kStages;
                const int first = (t.tile0 + j) * kTokens;
                if (!wait_on(&bars.keys_full[at], i / kStages, &s_abort)) return false;
                if (w == 0 && lane < pieces) {
                    const float2 raw = s_raw[i % kRawScales][lane];
                    const float value = fmaxf(raw.y, kLeastScale);
                    s_scale[i % kScales][lane] = __float_as_uint(raw.x) != kNoPage ? make_float4(raw.x, log2_approx(value), 1.f / value, 1.f) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const bool all = all_there(i, first), seen = all || seen_at(i, first, tid);
                if (i >= 2 && !wait_on(&bars.s_full[i & 1], (i >> 1) - 1, &s_abort)) return false;             // (the keys that lay there have been used)
                const uint32_t from = keys_ring + at * L::kHalf + tid * D, to = k_col(i) + ((uint32_t)(w * 32) << 16);
                const uint32_t swizzle = D == 128 ? (lane & 7) << 4 : ((lane >> 1) & 3) << 4;
#pragma unroll
                for (int c0 = 0; c0 < D / 16; c0 += 4) {
                    uint32_t out[32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint4 x = ptx::lds128(from + ((16 * (c0 + c)) ^ swizzle));
                        decode4<E4M3>(x.x, out[8 * c], out[8 * c + 1]);
                        decode4<E4M3>(x.y, out[8 * c + 2], out[8 * c + 3]);
                        decode4<E4M3>(x.z, out[8 * c + 4], out[8 * c + 5]);
                        decode4<E4M3>(x.w, out[8 * c + 6], out[8 * c + 7]);
                    }
                    if (!all) {                       // (bytes of tokens that nobody sees may be anything)
#pragma unroll
                        for (int k = 0; k < 32; ++k) out[k] = seen ? out[k] : 0;
                    }
                    ptx::tmem_st32(to + 8 * c0, out);
                }
                ptx::tc_wait_st();
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    arrive(&bars.k_full[i & 1]);
                    arrive(&bars.keys_empty[at]);
                    if (w == 0) arrive(&bars.scale_full[i % kScales]);
                }
                return true;
            };
            // values: 8 tokens and 4 units of 16 at a time, in an order whose lanes meet in no bank
            const auto values = [&](int j) -> bool {
                const uint32_t i = g + j, at = i % kStages;
                const int first = (t.tile0 + j) * kTokens;
                if (!wait_on(&bars.values_full[at], i / kStages, &s_abort)) return false;
                if (i >= 2 && !wait_on(&bars.pv_done[i & 1], (i >> 1) - 1, &s_abort)) return false;              // (the values that lay there have been used)
                const bool all = all_there(i, first);
                const int in8 = (lane >> 3) ^ (lane & 4 ? 5 : 0), token0 = w * 32 + in8, unit = lane & 3;
                const uint32_t from = values_ring + at * L::kHalf + token0 * D + ((16 * unit) ^ (D == 128 ? in8 << 4 : ((in8 >> 1) & 3) << 4));
                const uint32_t to = v_tile + (i & 1) * L::kV + token0 * 128 + ((32 * unit) ^ (in8 << 4));
#pragma unroll 2
                for (int q = 0; q < 4; ++q) {
                    const bool seen = all || seen_at(i, first, token0 + 8 * q);
#pragma unroll
                    for (int half = 0; half < D / 64; ++half) {
                        uint4 x = ptx::lds128((from ^ (64 * half)) + q * 8 * D);
                        if (!seen) x = make_uint4(0, 0, 0, 0);                // (0 * NaN is NaN)
                        uint4 a, b;
                        decode4<E4M3>(x.x, a.x, a.y);
                        decode4<E4M3>(x.y, a.z, a.w);
                        decode4<E4M3>(x.z, b.x, b.y);
                        decode4<E4M3>(x.w, b.z, b.w);
                        ptx::sts128(to + half * kMnStride + q * 1024, a);
                        ptx::sts128((to ^ 16) + half * kMnStride + q * 1024, b);
                    }
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    arrive(&bars.v_full[i & 1]);
                    arrive(&bars.values_empty[at]);
                }
                return true;
            };
            // (the next tile's keys come first, so that its scores do not wait for this one's products)
#pragma unroll 1
            for (int j = 0; j <= t.tiles && ok; ++j) ok = (j == t.tiles || keys(j)) && (j == 0 || values(j - 1));
            g += t.tiles;
            if (ok) done_with_item(n);
        }
        if (!ok) ptx::named_bar_arrive(kMeet, 128);
    } else {
        // ---- softmax ----
        // A set of eight warps has every other tile, with references, totals and sums of its own, so that one set's chain of steps runs beside the other's.
        const int set = warp >> 3, h = (warp >> 2) & 1, me = warp >> 2, w = warp & 3, tid = w * 32 + lane;
        const int id_set = 1 + me, id_half = 5 + h;   // named barriers: of four warps, and of both sets' for a half
        const uint32_t lanes = (uint32_t)(w * 32) << 16;
        uint32_t g = 0, pass = 0;
        bool ok = true;
        const float factor = p.scale * kLog2e;
#pragma unroll 1
        for (uint32_t n = 0; ok; ++n) {
            ok = next_item(n);
            if (!ok || !items[n % kItems].valid) break;
            const uint32_t item_slot = n % kItems;
            const Item& t = items[item_slot];
            ok = wait_on(&bars.q_full[item_slot], n / kItems, &s_abort);
            if (!ok) break;
            const int columns = t.n / kHalves, row0 = h * columns, groups = columns / 8, tiles = t.tiles;       // groups of 8
            const int most_low = s_most_low[item_slot];
            if (tid < kColumns) s_minus_top[me][tid] = tid < columns ? -kNone : -INFINITY;   // (columns that are the other half's, or nobody's, have no weights)
            float sums[kColumns];
#pragma unroll
            for (int i = 0; i < kColumns; ++i) sums[i] = 0.f;
            if (!(ok = meet(id_set, 128))) break;
            const int j0 = (set ^ g) & 1;
#pragma unroll 1
            for (int j = j0; j < tiles; j += 2) {
                const uint32_t i = g + j;
                ok = wait_on(&bars.scale_full[i % kScales], i / kScales, &s_abort) && wait_on(&bars.s_full[set], i >> 1, &s_abort);
                // (what lay in the weights' place has been used, and is in the sums)
                if (ok && j >= 2) ok = wait_on(&bars.pv_done[set], (i >> 1) - 1, &s_abort);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const float4 sc = s_scale[i % kScales][tid >> page_shift];
                const int first = (t.tile0 + j) * kTokens, token = first + tid;
                const bool there = sc.w != 0.f && token >= t.lo && token < t.limit, hide = first < most_low;
                // (keys of tokens that are not there are 0)
                const float a = there ? factor * sc.x : 0.f, b = there ? sc.y : -INFINITY, inverse = sc.z;
                const uint32_t s_at = s_col(i) + lanes + row0;
                const uint32_t p_at = p_tile + set * L::kP + tid * 128, unit0 = row0 / 8;
                // exponents of N columns from `at` on, relative to the rows' references or not
                const auto exponents = [&](auto& x, int at, bool relative) {
                    constexpr int N = sizeof(x) / 4;
#pragma unroll
                    for (int k = 0; k < N; k += 4) {
                        float4 from = make_float4(b, b, b, b);
                        float2 a0 = make_float2(a, a), a1 = a0, f0 = make_float2(b, b), f1 = f0;
                        if (BF16) {
                            const float4 up = *reinterpret_cast<const float4*>(&s_up[item_slot][row0 + at + k]);
                            a0 = mul2(a0, make_float2(up.x, up.y));
                            a1 = mul2(a1, make_float2(up.z, up.w));
                        }
                        if (relative) {
                            from = *reinterpret_cast<const float4*>(&s_minus_top[me][at + k]);
                            f0 = add2(f0, make_float2(from.x, from.y));
                            f1 = add2(f1, make_float2(from.z, from.w));
                        }
                        const float2 y0 = fma2(make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), a0, f0);
                        const float2 y1 = fma2(make_float2(__uint_as_float(x[k + 2]), __uint_as_float(x[k + 3])), a1, f1);
                        x[k] = __float_as_uint(y0.x);
                        x[k + 1] = __float_as_uint(y0.y);
                        x[k + 2] = __float_as_uint(y1.x);
                        x[k + 3] = __float_as_uint(y1.y);
                    }
                    if (hide) {
#pragma unroll
                        for (int k = 0; k < N; ++k) x[k] = token < s_low[item_slot][row0 + at + k] ? 0xFF800000u : x[k];
                    }
                };
                // 16 columns at a time; a warp that comes upon a weight that outgrows fp16 stops there.  Then the rows' references move, and all begin again;
                // what is in the totals already is not added twice.
                int added = 0;
                bool again = false;
#pragma unroll 1
                for (;;) {
                    bool over = j < 2 && !again;     // (the rows have no reference yet: to that at once)
#pragma unroll
                    for (int c = 0; c < kColumns / 16; ++c)
                        if (2 * c < groups && !over) {
                            uint32_t x[16];
                            ptx::tmem_ld16(s_at + 16 * c, x);
                            ptx::tc_wait_ld();
                            exponents(x, 16 * c, true);
                            if (!again) {
                                float most = -INFINITY;
#pragma unroll
                                for (int k = 0; k < 16; k += 2) most = max3(most, __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                                over = __any_sync(kAll, most > kMostLog);
                            }
                            if (!over) {
#pragma unroll
                                for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(exp2_approx(__uint_as_float(x[k])));
                                if (c >= added) {
                                    added = c + 1;
#pragma unroll
                                    for (int k = 0; k < 16; k += 2) {
                                        const float2 s2 = fma2(make_float2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), make_float2(inverse, inverse),
                                                               make_float2(sums[16 * c + k], sums[16 * c + k + 1]));
                                        sums[16 * c + k] = s2.x;
                                        sums[16 * c + k + 1] = s2.y;
                                    }
                                }
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    uint32_t y[4];
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        y[k] = h2_as_u32(__floats2half2_rn(__uint_as_float(x[8 * q + 2 * k]), __uint_as_float(x[8 * q + 2 * k + 1])));
                                    const uint32_t unit = unit0 + 2 * c + q;
                                    if (2 * c + q < groups) ptx::sts128(p_at + ((unit ^ (tid & 7)) << 4), make_uint4(y[0], y[1], y[2], y[3]));
                                }
                            }
                        }
                    if (again) break;
                    if (j >= 2) {
                        ++pass;
                        if (over) s_need[me][pass & 1] = pass;
                        if (!(ok = meet(id_set, 128))) break;
                        if (s_need[me][pass & 1] != pass) break;
                    }
                    {
                        uint32_t x[kColumns];
                        ptx::tmem_ld32(s_at, x);
                        ptx::tc_wait_ld();
                        exponents(x, 0, false);
                        s_warps[me][w][lane] = reduce32(x, [](float u, float v) { return fmaxf(u, v); });
                    }
                    if (!(ok = meet(id_set, 128))) break;
                    if (tid < columns) {
                        const float old = -s_minus_top[me][tid];
                        float top = old;
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = fmaxf(top, s_warps[me][k][tid]);
                        s_minus_top[me][tid] = -top;
                        s_keep[me][tid] = top == old ? 1.f : exp2_approx(old - top);
                    }
                    if (!(ok = meet(id_set, 128))) break;
                    if (j >= 2) {
#pragma unroll
                        for (int k = 0; k < kColumns; ++k) sums[k] *= s_keep[me][k];
#pragma unroll 1
                        for (int q = 0; q < groups; ++q) {
                            uint32_t x[8];
                            ptx::tmem_ld8(o_col(set) + lanes + row0 + 8 * q, x);
                            ptx::tc_wait_ld();
#pragma unroll
                            for (int k = 0; k < 8; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * s_keep[me][8 * q + k]);
                            ptx::tmem_st8(o_col(set) + lanes + row0 + 8 * q, x);
                        }
                        ptx::tc_wait_st();
                    }
                    again = true;
                }
                if (!ok) break;
                ptx::tc_fence_before_sync();
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&bars.p_full[set]);
            }
            if (!ok) break;
            g += tiles;
            for (uint32_t i = tiles > 1 ? g - 2 : g - 1; i != g && ok; ++i) ok = wait_on(&bars.pv_done[i & 1], i >> 1, &s_abort);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            // totals: over the lanes, then over the warps, then of both sets
            {
                uint32_t x[kColumns];
#pragma unroll
                for (int k = 0; k < kColumns; ++k) x[k] = __float_as_uint(sums[k]);
                s_warps[me][w][lane] = reduce32(x, [](float u, float v) { return u + v; });
            }
            if (!(ok = meet(id_half, 256))) break;
            // A part: the block's first item continues another block's, its last is continued.  Few parts are added up by the block that comes last; more of
            // them would take it longer than they take those who read the rows.
            const int a = t.first_block, z = t.last_block;
            const bool whole = a == z, joins = !whole && z - a < kJoined;
            float* const parts = reinterpret_cast<float*>(header + p.prefix_parts);
            const auto part_of = [&](int block) { return parts + ((size_t)block * 2 + (block == a ? 1 : 0)) * L::kPartFloats; };
            float* const own = part_of(blockIdx.x);
            if (set == 0 && tid < columns) {
                float top[2], total[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int of = 2 * k + h;
                    const float minus = s_minus_top[of][tid];
                    top[k] = minus == -kNone ? -INFINITY : -minus;
                    total[k] = (s_warps[of][0][tid] + s_warps[of][1][tid]) + (s_warps[of][2][tid] + s_warps[of][3][tid]);
                }
                const float most = fmaxf(top[0], top[1]), from = most == -INFINITY ? 0.f : most;
                const float2 take = make_float2(exp2_approx(top[0] - from), exp2_approx(top[1] - from));
                const float2 both = make_float2(most, total[0] * take.x + total[1] * take.y);
                const int id = s_row[item_slot][row0 + tid];
                s_take[row0 + tid] = take;
                if (!whole) *reinterpret_cast<float2*>(own + kMostRows * D + 2 * (row0 + tid)) = both;
                if (id >= 0 && whole) p.prefix_total[id] = both;
                if (id >= 0 && !whole && !joins && (int)blockIdx.x == a) p.prefix_total[id] = in_parts(a, z - a + 1, row0 + tid);
            }
            if (!(ok = meet(id_half, 256))) break;
            // (int8: the products' rows are the dims in decode4's order)
            const int dim = E4M3 ? tid : (tid & ~3) | ((tid & 1) << 1) | ((tid >> 1) & 1);
            const bool real = tid < D;
#pragma unroll 1
            for (int q = set; q < groups; q += 2) {   // (a set that had no tile has no sums)
                uint32_t x[8], y[8];
                ptx::tmem_ld8(o_col(g - 1) + lanes + row0 + 8 * q, x);
                ptx::tmem_ld8(o_col(tiles > 1 ? g : g - 1) + lanes + row0 + 8 * q, y);
                ptx::tc_wait_ld();
                if (real)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int row = row0 + 8 * q + k, id = s_row[item_slot][row];
                        const float2 take = s_take[row];
                        const float last = (g - 1) & 1 ? take.y : take.x, other = (g - 1) & 1 ? take.x : take.y;
                        float* const to = whole ? p.prefix_sums + (long long)id * D : own + row * D;
                        float sum = __uint_as_float(x[k]) * last;
                        if (tiles > 1) sum = fmaf(__uint_as_float(y[k]), other, sum);
                        if (id >= 0) to[dim] = sum;
                    }
                __syncwarp();
            }
            if (joins) {
                __threadfence();
                if (!(ok = meet(id_half, 256))) break;
                if (set == 0 && tid == 0) {
                    unsigned int* const counter = reinterpret_cast<unsigned int*>(header + kPrefixCounters) + kHalves * a + h;
                    const bool last = atomicAdd(counter, 1u) == (unsigned int)(z - a);
                    if (last) atomicExch(counter, 0u);                        // as the next launch expects it
                    s_last[h] = last;
                    __threadfence();
                }
                if (!(ok = meet(id_half, 256))) break;
                if (s_last[h]) {
                    __threadfence();
                    using Columns = std::conditional_t<D == 128, float4, float2>;             // of a lane
#pragma unroll 1
                    for (int r = 4 * set + w; r < columns; r += 8) {
                        const int row = row0 + r, id = s_row[item_slot][row];
                        if (id < 0) continue;
                        const auto both = [&](int b) { return __ldcg(reinterpret_cast<const float2*>(part_of(b) + kMostRows * D + 2 * row)); };
                        float m = -INFINITY;
#pragma unroll 1
                        for (int b = a + lane; b <= z; b += 32) m = fmaxf(m, both(b).x);
#pragma unroll
                        for (int d = 16; d; d /= 2) m = fmaxf(m, __shfl_xor_sync(kAll, m, d));
                        const float from = m == -INFINITY ? 0.f : m;
                        float all_total = 0.f;
                        Columns o{};
#pragma unroll 1
                        for (int b0 = a; b0 <= z; b0 += 32) {
                            float2 mine = make_float2(-INFINITY, 0.f);
                            if (b0 + lane <= z) mine = both(b0 + lane);
                            const float take = exp2_approx(mine.x - from);
                            all_total = fmaf(take, mine.y, all_total);
                            const int count = min(32, z - b0 + 1);
#pragma unroll 4
                            for (int i = 0; i < count; ++i) {
                                const Columns x = __ldcg(reinterpret_cast<const Columns*>(part_of(b0 + i) + row * D) + lane);
                                const float f = __shfl_sync(kAll, take, i);
                                o.x = fmaf(f, x.x, o.x);
                                o.y = fmaf(f, x.y, o.y);
                                if constexpr (D == 128) {
                                    o.z = fmaf(f, x.z, o.z);
                                    o.w = fmaf(f, x.w, o.w);
                                }
                            }
                        }
#pragma unroll
                        for (int d = 16; d; d /= 2) all_total += __shfl_xor_sync(kAll, all_total, d);
                        reinterpret_cast<Columns*>(p.prefix_sums + (long long)id * D)[lane] = o;
                        if (lane == 0) p.prefix_total[id] = make_float2(m, all_total);
                    }
                }
            }
            // what was read of the sums is read before the next item's products overwrite them, whichever set it was of
            ptx::tc_fence_before_sync();
            if (!(ok = meet(id_half, 256))) break;
            done_with_item(n);
        }
        if (!ok) {
            ptx::named_bar_arrive(id_set, 128);
            ptx::named_bar_arrive(id_half, 256);
        }
    }

    if (lane == 0 && s_abort) atomicExch(reinterpret_cast<int*>(header + kStatusOffset), 63);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    if (warp == kMma) ptx::tmem_dealloc(tmem, 512);
}

template <bool E4M3, bool BF16, int D>
cudaError_t launch_prefix(const AttentionParams& p, int most_rows, cudaStream_t stream) {
    const auto kernel = cache_prefix_kernel<E4M3, BF16, D>;
    constexpr int kSmem = Layout<D>::kBytes;
    CUtensorMap k_map, v_map;
    if (!cache_map(&k_map, p.cache, true, 1 << p.cache.page_shift) || !cache_map(&v_map, p.cache, false, 1 << p.cache.page_shift)) return cudaErrorNotSupported;
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
    e = cudaLaunchKernelEx(&cfg, kernel, p, most_rows, k_map, v_map);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

size_t cache_prefix_workspace() { return kPartsBytes; }

cudaError_t cache_prefix_launch(const AttentionParams& p, bool e4m3, bool bf16, int most_rows, cudaStream_t stream) {
    const auto by_dim = [&](auto e, auto h) {
        constexpr bool E = decltype(e)::value, H = decltype(h)::value;
        return p.cache.dim == 128 ? launch_prefix<E, H, 128>(p, most_rows, stream) : launch_prefix<E, H, 64>(p, most_rows, stream);
    };
    const auto by_type = [&](auto e) { return bf16 ? by_dim(e, std::true_type{}) : by_dim(e, std::false_type{}); };
    return e4m3 ? by_type(std::true_type{}) : by_type(std::false_type{});
}

}  // namespace i4mm
