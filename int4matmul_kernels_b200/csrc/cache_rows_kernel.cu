// Attention over the paged 8-bit cache (i4mm_cache_attention), few rows per request: decoding.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j, over the tokens j that the row sees,
// in one pass with the running maximum and sum.  Every byte of the cache is read once and enters 2 multiply-adds for each of a head's few
// rows, so DRAM bounds it: 24 bytes a cycle and SM.  What the rest is made for is to keep that many bytes in flight and to decode them
// in less than that time:
//
// * Work.  The tokens of a request and head (a segment) are cut into tiles of 32.  All tiles of all segments in a row are dealt out in
//   equal contiguous ranges, to the blocks (one to an SM) and within them to the warps, whatever the lengths are.  What a
//   range cuts is joined: warps of a block through shared memory, blocks through the workspace, where the block that comes last adds up
//   all parts in their order (so results do not depend on which one it is).  Nobody waits for anybody.
// * Bytes.  Each warp fetches its own tiles, two ahead, into a ring of its own (a TMA copy for each 16 keys and 16 values, swizzled, one
//   barrier for a tile): warps do not wait for one another, and no registers are held by loads in flight.  Copies alone, with nothing
//   done to what they bring, take 207 us for 1.32 GB (64 requests of up to 4000 tokens, 40 heads of 128); the same bytes by 16-byte
//   copies of each thread took 314.
// * Products.  S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: the cache is the 16-row operand, the head's rows are the 8 columns.  The
//   order of the 16 k of an instruction is free as long as both operands agree, so a thread takes 16 consecutive bytes of a key row (and
//   the same places of q), and 16 consecutive bytes of each of its value rows; two value rows become operand words by byte
//   permutes.  int8 becomes fp16 by placing the byte in the mantissa of 1024 (exact), e4m3 by the conversion instruction (exact).  The
//   weights go from the accumulator layout to the operand layout by a transpose of 8 x 8 matrices.
// * Scales.  x = s + log2(value scale) of the page: weights are 2^(x - the tile's largest x), rounded to fp16, and a tile's product joins the
//   fp32 sums with the factor 2^(largest x - reference): pages of any scales, none of it lost to fp16's range; the totals take each weight
//   divided by its page's value scale again.  A second product with the weights' rounding errors (their low halves) brings the output to
//   fp32's exactness for 16 more tensor instructions a tile, which the tensor pipe (20 % busy) has spare.
//
// Measured: the requests above 285 us (4.6 TB/s; some 830 instructions a tile of 32 tokens, half of them for the bytes' decoding, are what is left
// to hide); 12 requests of 20000 to 34000 tokens, 8 heads, e4m3, 8 rows: 120 us (5.6 TB/s); one request of 1011 tokens: 13.5 us, of which
// 5 find and fetch the first tile, 3.6 join parts over blocks.  (Whole segments to blocks, without that join: 14.8.)
#include <algorithm>
#include <type_traits>

#include "cache_attention.cuh"
#include "tensor_map.cuh"

namespace i4mm {
namespace {

constexpr int kTile = 32;                             // tokens: two halves of 16, each within one page
constexpr int kMinBlockTiles = 4, kMinWarpTiles = 1;  // fewer tiles than this are not cut further
constexpr uint32_t kNoPage = 0x7FC0DEADu;             // in the place of a scale: there is no such page

template <int D, int NT>
struct Shape {
    // Registers (234 to 243 for one column tile at head_dim 128, nothing spilled; two column tiles take all 255 and spill 100 to 128 bytes,
    // which 360 to 456 bytes of loads bring back) allow 8 warps; with half the bytes to a token, 12 warps of 168 hide more of a tile's
    // dependent steps than they lose, though two column tiles spill 124 bytes there (524 of loads) and one, of 155 to 158 registers, nothing
    // (33 drafts, head_dim 64: 63.5 us with 8, 61.6 with 12; 64 single tokens, head_dim 128: 284 and 279
    // with a ring of two stages, 118 and 122 on long contexts).
    static constexpr int kWarps = D == 64 ? 12 : 8;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kRows = 8 * NT;
    static constexpr int kHalfBytes = 32 * D;                                 // 16 tokens: keys, then values
    static constexpr int kStageBytes = 2 * kHalfBytes;
    static constexpr int kStages = D == 128 ? 3 : 4;
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kPartFloats = kRows * D + 2 * kRows;                 // sums, maxima, totals of a part of a segment
    static_assert(kPartFloats * 4 <= kWarpBytes, "a warp leaves its last part in its ring");
};

// ---- behind the workspace's header: [a part per warp][two parts per block] ----
constexpr size_t kWarpPartsBytes = (size_t)kMaxBlocks * Shape<128, 2>::kWarps * Shape<128, 2>::kPartFloats * 4;
static_assert(Shape<64, 2>::kWarps * Shape<64, 2>::kPartFloats <= Shape<128, 2>::kWarps * Shape<128, 2>::kPartFloats, "room for any shape");
constexpr size_t kBlockPartsBytes = (size_t)kMaxBlocks * 2 * Shape<128, 2>::kPartFloats * 4;

// a request and its tiles of tokens: at least one if there are rows (rows that see nothing are written too)
struct Few : Request {
    int tiles;
};
__device__ __forceinline__ Few load_few(const AttentionParams& p, int most_rows, int b) {
    Few r;
    static_cast<Request&>(r) = load_request(p, b);
    if ((long long)r.rows * p.group > most_rows) r.rows = 0;    // the other kernel's
    r.tiles = max((r.limit + kTile - 1) / kTile - r.lo / kTile, 1);
    return r;
}

// segments of a request: one for each head and tile of rows
template <int ROWS>
__device__ __forceinline__ int row_tiles(const AttentionParams& p, const Request& r) {
    return (r.rows * p.group + ROWS - 1) / ROWS;
}

template <int ROWS>
__device__ __forceinline__ long long units_of(const AttentionParams& p, const Few& r) {
    if (r.rows == 0) return 0;
    return (long long)r.tiles * p.cache.heads * row_tiles<ROWS>(p, r);
}

// ---- decoding and products -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {   // onto zeros
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// The token of a half that the products' row (and k) index i stands for.  Any order is right as long as keys, values and masks agree;
// in this one the lanes of a quarter warp, which read the swizzled rows of i = 2 j, 2 j + 1 (keys) and of i = 0, 2, 4, 6 (values), meet
// in no bank (head_dim 128).
__device__ __forceinline__ int token_of(int i) {
    const int pair = (i & 7) >> 1;
    return (i & 8) + ((2 * pair + (pair >> 1)) ^ ((i & 1) << 2));
}

template <bool BF16>
__device__ __forceinline__ void store4(void* out, long long at, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(pack_out<BF16>(a, b), pack_out<BF16>(c, d));
}

// a part of a segment that a range has cut: where the segment lies among all tiles, and which one it is
struct Piece {
    long long from, to;                               // from < 0: none
    int b, segment, rows;                             // rows of its row tile
};

template <bool E4M3, bool BF16, int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 1) cache_rows_kernel(const AttentionParams p, int most_rows,
                                                                              const __grid_constant__ CUtensorMap k_map,
                                                                              const __grid_constant__ CUtensorMap v_map) {
    using S = Shape<D, NT>;
    constexpr int kSteps = D / 16, kWords = D / 32;   // k steps of 16; words of 4 bytes that a thread has of a value row
    extern __shared__ uint8_t dynamic[];
    uint8_t* const ring = dynamic + (1024 - (ptx::smem_u32(dynamic) & 1023)) % 1024;
    __shared__ unsigned long long s_full[S::kWarps][S::kStages];
    __shared__ float2 s_scales[S::kWarps][S::kStages][2];
    __shared__ Piece s_head[S::kWarps], s_tail[S::kWarps];
    __shared__ int s_last[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const CacheView& cache = p.cache;
    if (lane == 0) {
        // two lanes fetch a half each: each of them arrives with the bytes that it expects, and once its scales are there
        for (int i = 0; i < S::kStages; ++i) ptx::mbar_init(ptx::smem_u32(&s_full[warp][i]), 4);
        ptx::fence_mbar_init();
    }
    __syncwarp();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    // rows of no request
    {
        const int first = p.requests == 0 ? 0 : p.cu_lens ? min(max(p.cu_lens[p.requests], 0), p.tokens) : p.requests;
        const long long from = (long long)first * p.q_heads * D, to = (long long)p.tokens * p.q_heads * D;
        for (long long i = from + 8ll * (blockIdx.x * S::kThreads + threadIdx.x); i < to; i += 8ll * gridDim.x * S::kThreads)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i) = make_uint4(0, 0, 0, 0);
    }

    // all tiles; the block's range and the warp's.  The first 32 requests stay in the lanes' registers.
    Few mine{};
    long long own = 0;
    if (lane < p.requests) {
        mine = load_few(p, most_rows, lane);
        own = units_of<S::kRows>(p, mine);
    }
    long long total = own;
    for (int b = lane + 32; b < p.requests; b += 32) total += units_of<S::kRows>(p, load_few(p, most_rows, b));
    const long long own_upto = warp_prefix(own);
    total = warp_sum(total);
    const long long blocks = min((long long)gridDim.x, (total + kMinBlockTiles - 1) / kMinBlockTiles);
    if (blockIdx.x >= blocks) return;
    const long long c0 = range_lo(total, blocks, blockIdx.x), c1 = range_lo(total, blocks, blockIdx.x + 1);
    const long long warps = min((long long)S::kWarps, (c1 - c0 + kMinWarpTiles - 1) / kMinWarpTiles);
    const long long u0 = warp < warps ? c0 + range_lo(c1 - c0, warps, warp) : c1, u1 = warp < warps ? c0 + range_lo(c1 - c0, warps, warp + 1) : c1;
    if (lane == 0) {
        s_head[warp].from = -1;
        s_tail[warp].from = -1;
    }

    float* const warp_part = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + kCacheHeaderBytes) + ((size_t)blockIdx.x * S::kWarps + warp) * S::kPartFloats;
    const uint32_t my_ring = ptx::smem_u32(ring) + warp * S::kWarpBytes;

    if (u0 < u1) {
        // the request that the range begins in, the segment within it and the tile within that
        int b = 0, segment, tile;
        Few r;
        {
            long long before = 0, here_own = own, upto = own_upto;
            for (;;) {
                const uint32_t here = __ballot_sync(kAll, before + upto > u0);
                if (here) {
                    const int l = __ffs(here) - 1;
                    before += __shfl_sync(kAll, upto - here_own, l);
                    b += l;
                    break;
                }
                before += __shfl_sync(kAll, upto, 31);
                b += 32;
                if (b >= p.requests) break;           // (not unless the lengths change under the kernel)
                here_own = b + lane < p.requests ? units_of<S::kRows>(p, load_few(p, most_rows, b + lane)) : 0;
                upto = warp_prefix(here_own);
            }
            b = min(b, p.requests - 1);
            if (b < 32) {
                r.row0 = __shfl_sync(kAll, mine.row0, b);
                r.rows = __shfl_sync(kAll, mine.rows, b);
                r.position = __shfl_sync(kAll, mine.position, b);
                r.lo = __shfl_sync(kAll, mine.lo, b);
                r.limit = __shfl_sync(kAll, mine.limit, b);
                r.tiles = __shfl_sync(kAll, mine.tiles, b);
            } else {
                r = load_few(p, most_rows, b);
            }
            segment = (int)((u0 - before) / r.tiles);
            tile = (int)(u0 - before - (long long)segment * r.tiles);
        }

        // ---- copies: the same tiles, kStages - 1 of them ahead.  Lanes 0 and 1 take a half each. ----
        struct {
            int left;                                 // tiles to be copied
            int b, segment, segments, row_tiles, head;
            int tile, end, lo, limit;                 // the tile (from the request's token 0), the segment's end, its tokens
            const int* table;
            int id;                                   // the page of the lane's half of the tile
            int stage;
        } c = {};
        const int page_mask = (1 << cache.page_shift) - 1;
        const auto enter_request = [&](const Few& r) {
            c.row_tiles = row_tiles<S::kRows>(p, r);
            c.segments = cache.heads * c.row_tiles;
            c.tile = r.lo / kTile;
            c.end = c.tile + r.tiles;
            c.lo = r.lo;
            c.limit = r.limit;
            c.table = p.table + c.b * p.table_stride;
        };
        const auto find_page = [&]() {                // (nothing is done with what is loaded before the next copy)
            const int first = c.tile * kTile + 16 * (lane & 1), j = first >> cache.page_shift;
            c.id = -1;
            if (lane < 2 && first < c.limit && first + 16 > c.lo && c.limit > c.lo && j < p.table_width) c.id = c.table[j];
        };
        c.left = (int)(u1 - u0);
        c.b = b;
        c.segment = segment;
        enter_request(r);
        c.tile += tile;
        c.head = segment / c.row_tiles;
        find_page();
        const auto copy = [&]() {
            if (c.left <= 0) return;
            if (lane < 2) {
                const uint32_t bar = ptx::smem_u32(&s_full[warp][c.stage]), to = my_ring + c.stage * S::kStageBytes + lane * S::kHalfBytes;
                if ((unsigned int)c.id < (unsigned int)cache.pages) {
                    const int place = (c.tile * kTile + 16 * lane) & page_mask;
                    ptx::mbar_arrive_expect_tx(bar, S::kHalfBytes);
                    ptx::tma_load_4d(to, &k_map, 0, place, c.head, c.id, bar);
                    ptx::tma_load_4d(to + 16 * D, &v_map, 0, place, c.head, c.id, bar);
                    ptx::cp_async_8(ptx::smem_u32(&s_scales[warp][c.stage][lane]), cache.scales + (long long)c.id * cache.heads + c.head);
                    ptx::cp_async_arrive(bar);
                } else {
                    s_scales[warp][c.stage][lane] = make_float2(__uint_as_float(kNoPage), 0.f);
                    ptx::mbar_arrive(bar);
                    ptx::mbar_arrive(bar);
                }
            }
            c.stage = c.stage + 1 == S::kStages ? 0 : c.stage + 1;
            if (--c.left == 0) return;
            if (++c.tile == c.end) {
                if (++c.segment < c.segments) {
                    c.tile = c.lo / kTile;
                } else {
                    c.segment = 0;
                    Few next;
                    do {
                        ++c.b;
                        if (c.b < p.requests) next = load_few(p, most_rows, c.b);
                    } while (c.b < p.requests && next.rows == 0);
                    if (c.b < p.requests) enter_request(next);
                    else c.left = 0;                  // (as above)
                }
                c.head = c.segment / c.row_tiles;
            }
            find_page();
        };
        for (int i = 0; i < S::kStages - 1; ++i) copy();

        // where the lane's bytes lie in a half
        const int k_row = token_of(g), v_row0 = token_of(2 * t), v_row1 = token_of(2 * t + 1);
        const auto keys_at = [&](int j) {             // chunk 4 * j + t of 16 bytes
            return D == 128 ? k_row * 128 + (((4 * j + t) ^ (k_row & 7)) << 4) : k_row * 64 + ((t ^ ((k_row >> 1) & 3)) << 4);
        };
        const auto values_at = [&](int row) {         // D / 8 bytes from place D / 8 * g on
            return 16 * D + (D == 128 ? row * 128 + ((g ^ (row & 7)) << 4) : row * 64 + (((g >> 1) ^ ((row >> 1) & 3)) << 4) + 8 * (g & 1));
        };
        const uint32_t keys_lane[2] = {(uint32_t)keys_at(0), (uint32_t)keys_at(D / 64 - 1)};
        const uint32_t values_lane[2] = {(uint32_t)values_at(v_row0), (uint32_t)values_at(v_row1)};

        // ---- the segments of the range ----
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        long long at = u0;
        while (at < u1 && ok) {
            const int tiles_here = (int)min((long long)(r.tiles - tile), u1 - at);
            const int row_tile_count = row_tiles<S::kRows>(p, r), head = segment / row_tile_count, base = (segment - head * row_tile_count) * S::kRows;
            const int all_rows = r.rows * p.group;
            // q as the second operand of the score products: the lane's row is base + 8 * n + g
            uint32_t q[NT][2 * kSteps];
            float factor[NT][2], m[NT][2], sum[NT][2], o[NT][2 * kWords][4];
            int position[NT][2];                      // of the lane's rows of the products' results, base + 8 * n + 2 * t and the next: -1 if there is none
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int row = base + 8 * n + g;
                float mine = 1.f;
                if (row < all_rows) {
                    const int token = row / p.group, h = head * p.group + row - token * p.group;
                    const uint16_t* const from = static_cast<const uint16_t*>(p.q.p) + (r.row0 + token) * p.q.token + h * p.q.head + 16 * t;
                    uint2 w[kSteps];
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) w[s] = *reinterpret_cast<const uint2*>(from + 64 * (s >> 2) + 4 * (s & 3));
                    if (BF16) {
                        float most = 0.f, down;
#pragma unroll
                        for (int s = 0; s < kSteps; ++s) most = fmaxf(most, bf16_most(w[s]));
                        const uint32_t peers = 0xFu << (lane & 28);
                        most = fmaxf(most, __shfl_xor_sync(peers, most, 1));
                        most = fmaxf(most, __shfl_xor_sync(peers, most, 2));
                        bf16_powers(most, mine, down);
#pragma unroll
                        for (int s = 0; s < kSteps; ++s) w[s] = bf16_scaled(w[s], down);
                    }
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        const uint2 x = key_order<E4M3>(w[s]);
                        q[n][2 * s] = x.x;
                        q[n][2 * s + 1] = x.y;
                    }
                } else {
#pragma unroll
                    for (int s = 0; s < 2 * kSteps; ++s) q[n][s] = 0;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    factor[n][i] = __shfl_sync(kAll, mine, 4 * (2 * t + i)) * (p.scale * kLog2e);
                    const int row = base + 8 * n + 2 * t + i;
                    position[n][i] = row < all_rows ? r.position + row / p.group : -1;
                    m[n][i] = -INFINITY;
                    sum[n][i] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 2 * kWords; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
            }

            // tiles that begin in [whole_from, whole_to] are seen whole by all rows of the tile of rows
            const int whole_from = p.window ? max(r.position + r.rows - p.window, r.lo) : r.lo;
            const int whole_to = base + S::kRows <= all_rows ? min(r.position + 1, r.limit) - kTile : -1;
            int first = (r.lo / kTile + tile) * kTile;
            for (int i = 0; i < tiles_here; ++i, first += kTile) {
                __syncwarp();                         // (the stage that the copy goes to has been read)
                copy();
                ok = __all_sync(kAll, ptx::mbar_wait(ptx::smem_u32(&s_full[warp][stage]), phase));
                if (!ok) {
                    if (lane == 0) atomicExch(reinterpret_cast<int*>(static_cast<uint8_t*>(p.workspace) + kStatusOffset), 62);
                    break;
                }
                const uint32_t half0 = my_ring + stage * S::kStageBytes;
                // scores
                float s[NT][2][4];
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        const uint32_t keys = half0 + half * S::kHalfBytes + keys_lane[j];
                        const uint4 ka = ptx::lds128(keys), kb = ptx::lds128(keys + 8 * D);
                        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            uint32_t a0, a1, a2, a3;
                            decode4<E4M3>(wa[w], a0, a2);
                            decode4<E4M3>(wb[w], a1, a3);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint32_t b0 = q[n][2 * (4 * j + w)], b1 = q[n][2 * (4 * j + w) + 1];
                                if (j == 0 && w == 0) mma_first(s[n][half], a0, a1, a2, a3, b0, b1);
                                else mma(s[n][half], a0, a1, a2, a3, b0, b1);
                            }
                        }
                    }
                bool there[2];
                float k_scale[2], v_log2[2], v_inverse[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float2 both = s_scales[warp][stage][half];
                    there[half] = __float_as_uint(both.x) != kNoPage;
                    const float v_scale = there[half] ? fmaxf(both.y, kLeastScale) : 1.f;
                    k_scale[half] = there[half] ? both.x : 0.f;
                    v_log2[half] = log2_approx(v_scale);
                    v_inverse[half] = exp2_approx(-v_log2[half]);
                }
                const bool whole = there[0] && there[1] && first >= whole_from && first <= whole_to;
                uint32_t high[NT][2][2], low[NT][2][2];
                float weight[NT][2];                  // of the tile's sums in the segment's
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float most[2];
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) s[n][half][i2] = fmaf(s[n][half][i2], factor[n][i2 & 1] * k_scale[half], v_log2[half]);
                    if (!whole) {
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int i2 = 0; i2 < 4; ++i2) {
                                const int token = first + 16 * half + k_row + 8 * (i2 >> 1), at_row = position[n][i2 & 1];
                                const bool sees = there[half] && token <= at_row && token < r.limit && token >= r.lo && (!p.window || token > at_row - p.window);
                                if (!sees) s[n][half][i2] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        float x = fmaxf(fmaxf(s[n][0][i2], s[n][0][2 + i2]), fmaxf(s[n][1][i2], s[n][1][2 + i2]));
                        x = fmaxf(x, __shfl_xor_sync(kAll, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(kAll, x, 8));
                        most[i2] = fmaxf(x, __shfl_xor_sync(kAll, x, 16));
                    }
                    // the reference of the sums moves only when a tile exceeds it by much: they are fp32 and have room
                    if (__any_sync(kAll, most[0] > m[n][0] + 16.f || most[1] > m[n][1] + 16.f)) {
#pragma unroll
                        for (int i2 = 0; i2 < 2; ++i2) {
                            const float next = fmaxf(m[n][i2], most[i2]), keep = m[n][i2] == -INFINITY ? 0.f : exp2_approx(m[n][i2] - next);
                            m[n][i2] = next;
                            sum[n][i2] *= keep;
#pragma unroll
                            for (int j = 0; j < 2 * kWords; ++j) {
                                o[n][j][i2] *= keep;
                                o[n][j][2 + i2] *= keep;
                            }
                        }
                    }
                    float e[2][4];
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        const bool any = most[i2] != -INFINITY;
                        const float from = any ? most[i2] : 0.f;
                        weight[n][i2] = any ? exp2_approx(most[i2] - m[n][i2]) : 0.f;
                        float all = 0.f;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            e[half][i2] = exp2_approx(s[n][half][i2] - from);
                            e[half][2 + i2] = exp2_approx(s[n][half][2 + i2] - from);
                            all = fmaf(e[half][i2] + e[half][2 + i2], v_inverse[half], all);
                        }
                        sum[n][i2] = fmaf(weight[n][i2], all, sum[n][i2]);
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int i2 = 0; i2 < 2; ++i2) {
                            const __half2 h = __floats2half2_rn(e[half][2 * i2], e[half][2 * i2 + 1]);
                            const float2 back = __half22float2(h);
                            high[n][half][i2] = transpose8x8(h2_as_u32(h));
                            low[n][half][i2] = transpose8x8(h2_as_u32(__floats2half2_rn(e[half][2 * i2] - back.x, e[half][2 * i2 + 1] - back.y)));
                        }
                }
                // values
                uint32_t v[2][4][kWords];
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i2 = 0; i2 < 4; ++i2) {
                        const uint32_t values = half0 + half * S::kHalfBytes + values_lane[i2 & 1] + (i2 >> 1) * 8 * D;
                        if constexpr (D == 128) {
                            const uint4 w = ptx::lds128(values);
                            v[half][i2][0] = w.x; v[half][i2][1] = w.y; v[half][i2][2] = w.z; v[half][i2][3] = w.w;
                        } else {
                            const uint2 w = ptx::lds64(values);
                            v[half][i2][0] = w.x; v[half][i2][1] = w.y;
                        }
                    }
                if (!(there[0] && there[1] && first >= r.lo && first + kTile <= r.limit)) {
                    // bytes of tokens that nobody sees may be anything, and 0 * NaN is NaN
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) {
                            const int token = first + 16 * half + (i2 & 1 ? v_row1 : v_row0) + 8 * (i2 >> 1);
                            if (!(there[half] && token >= r.lo && token < r.limit))
#pragma unroll
                                for (int w = 0; w < kWords; ++w) v[half][i2][w] = 0;
                        }
                }
#pragma unroll
                for (int j = 0; j < 2 * kWords; ++j) {
                    float d[NT][4];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t a0, a1, a2, a3;
                        decode_pair<E4M3>(v[half][0][j >> 1], v[half][1][j >> 1], j & 1, a0, a1);
                        decode_pair<E4M3>(v[half][2][j >> 1], v[half][3][j >> 1], j & 1, a2, a3);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (half == 0) mma_first(d[n], a0, a1, a2, a3, low[n][half][0], low[n][half][1]);
                            else mma(d[n], a0, a1, a2, a3, low[n][half][0], low[n][half][1]);
                            mma(d[n], a0, a1, a2, a3, high[n][half][0], high[n][half][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) o[n][j][i2] = fmaf(weight[n][i2 & 1], d[n][i2], o[n][j][i2]);
                }
                if (++stage == S::kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
            at += tiles_here;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) sum[n][i] += __shfl_xor_sync(kAll, sum[n][i], d);

            if (tiles_here == r.tiles) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = base + 8 * n + 2 * t + i;
                        if (row >= all_rows) continue;
                        const int token = row / p.group, h = head * p.group + row - token * p.group;
                        const long long to = ((long long)(r.row0 + token) * p.q_heads + h) * D + (D / 8) * g;
                        const float f = sum[n][i] > 0.f ? 1.f / sum[n][i] : sum[n][i];       // (a NaN stays one)
#pragma unroll
                        for (int j = 0; j < kWords; ++j)
                            store4<BF16>(p.out, to + 4 * j, o[n][2 * j][i] * f, o[n][2 * j][2 + i] * f, o[n][2 * j + 1][i] * f, o[n][2 * j + 1][2 + i] * f);
                    }
            } else {
                // a part: the range's last one stays in the ring (nothing is on its way there any more), its first goes to the workspace
                const bool last = at == u1;
                __syncwarp();
                float* const part = last ? reinterpret_cast<float*>(ring + warp * S::kWarpBytes) : warp_part;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 8 * n + 2 * t + i;
                        if (base + row >= all_rows) continue;
#pragma unroll
                        for (int j = 0; j < kWords; ++j)
                            *reinterpret_cast<float4*>(part + row * D + (D / 8) * g + 4 * j) =
                                make_float4(o[n][2 * j][i], o[n][2 * j][2 + i], o[n][2 * j + 1][i], o[n][2 * j + 1][2 + i]);
                        if (g == 0) {
                            part[S::kRows * D + row] = m[n][i];
                            part[S::kRows * D + S::kRows + row] = sum[n][i];
                        }
                    }
                if (lane == 0) {
                    const long long from = at - tiles_here - tile;
                    (last ? s_tail : s_head)[warp] = Piece{from, from + r.tiles, b, segment, min(S::kRows, all_rows - base)};
                }
            }
            // the next segment
            tile = 0;
            if (++segment == cache.heads * row_tile_count && at < u1) {
                segment = 0;
                do {
                    ++b;
                    if (b < p.requests) r = load_few(p, most_rows, b);
                } while (b < p.requests && r.rows == 0);
                if (b >= p.requests) break;           // (as above)
            }
        }
        // A warp that stops early waits, bounded again, for what is on its way to its ring: the shared memory is someone else's once the block
        // has ended.  (All kStages are where it gave up on the tile that lies as many behind the next copy.)
        int in_flight = c.stage - stage + (c.stage < stage || (c.stage == stage && !ok) ? S::kStages : 0);
        for (; in_flight > 0; --in_flight) {
            (void)ptx::mbar_wait(ptx::smem_u32(&s_full[warp][stage]), phase);
            if (++stage == S::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
    }
    __syncthreads();

    // ---- parts of one segment are added up, a row by a warp ----
    constexpr int kMine = D / 32;                     // columns of a lane
    struct Joined {
        float m, sum, o[kMine];
    };
    // (parts of other blocks are read past the first-level cache)
    const auto add = [&](Joined& a, const float* part, int row, bool mine) {
        const auto load = [&](int i) { return mine ? part[i] : __ldcg(part + i); };
        using Columns = std::conditional_t<kMine == 4, float4, float2>;
        const Columns* const at = reinterpret_cast<const Columns*>(part + row * D) + lane;
        const Columns x = mine ? *at : __ldcg(at);
        const float pm = load(S::kRows * D + row), ps = load(S::kRows * D + S::kRows + row);
        const float next = fmaxf(a.m, pm);
        const float keep = a.m == -INFINITY ? 0.f : exp2_approx(a.m - next), take = pm == -INFINITY ? 0.f : exp2_approx(pm - next);
        a.m = next;
        a.sum = a.sum * keep + ps * take;
        a.o[0] = a.o[0] * keep + x.x * take;
        a.o[1] = a.o[1] * keep + x.y * take;
        if constexpr (kMine == 4) {
            a.o[2] = a.o[2] * keep + x.z * take;
            a.o[3] = a.o[3] * keep + x.w * take;
        }
    };
    const auto finish = [&](const Joined& a, const Piece& piece, int row) {
        const Request r = load_request(p, piece.b);
        const int count = row_tiles<S::kRows>(p, r), head = piece.segment / count, in = (piece.segment - head * count) * S::kRows + row;
        const int token = in / p.group, h = head * p.group + in - token * p.group;
        const long long to = ((long long)(r.row0 + token) * p.q_heads + h) * D + kMine * lane;
        const float f = a.sum > 0.f ? 1.f / a.sum : a.sum;
        if constexpr (kMine == 4) {
            store4<BF16>(p.out, to, a.o[0] * f, a.o[1] * f, a.o[2] * f, a.o[3] * f);
        } else {
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + to) = pack_out<BF16>(a.o[0] * f, a.o[1] * f);
        }
    };
    float* const block_parts = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + kCacheHeaderBytes + kWarpPartsBytes);
    const auto ring_part = [&](int w) { return reinterpret_cast<const float*>(ring + w * S::kWarpBytes); };
    const auto workspace_part = [&](int w) {
        return reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.workspace) + kCacheHeaderBytes) + ((size_t)blockIdx.x * S::kWarps + w) * S::kPartFloats;
    };
    int item = 0;
    for (int l = -1; l < S::kWarps; ++l) {
        // segments by their first part in this block: the first warp's first part, or a warp's last part that the warp before does not share
        const Piece piece = l < 0 ? s_head[0] : s_tail[l];
        if (piece.from < 0 || (l > 0 && s_tail[l - 1].from == piece.from)) continue;
        const bool inside = piece.from >= c0 && piece.to <= c1;
        for (int row = 0; row < piece.rows; ++row) {
            if (item++ % S::kWarps != warp) continue;
            Joined a{-INFINITY, 0.f, {}};
            add(a, l < 0 ? workspace_part(0) : ring_part(l), row, true);
            for (int w = l + 1; l >= 0 && w < S::kWarps; ++w) {
                if (s_head[w].from == piece.from) {
                    add(a, workspace_part(w), row, true);
                    break;
                }
                if (s_tail[w].from != piece.from) break;
                add(a, ring_part(w), row, true);
            }
            if (inside) {
                finish(a, piece, row);
            } else {
                float* const to = block_parts + ((size_t)blockIdx.x * 2 + (piece.from >= c0 ? 1 : 0)) * S::kPartFloats;
#pragma unroll
                for (int i = 0; i < kMine; ++i) to[row * D + kMine * lane + i] = a.o[i];
                if (lane == 0) {
                    to[S::kRows * D + row] = a.m;
                    to[S::kRows * D + S::kRows + row] = a.sum;
                }
            }
        }
    }

    // ---- and across blocks: whoever comes last adds them up ----
    Piece cut[2];                                     // the segment that began before this block's range; the one that goes on after it
    cut[0].from = cut[1].from = -1;
    for (int l = -1; l < S::kWarps; ++l) {
        const Piece piece = l < 0 ? s_head[0] : s_tail[l];
        if (piece.from < 0) continue;
        if (piece.from < c0) cut[0] = piece;
        else if (piece.to > c1) cut[1] = piece;
    }
    if (cut[0].from < 0 && cut[1].from < 0) return;
    __syncthreads();
    if (threadIdx.x < 2) {
        int last = 0;
        const Piece& piece = cut[threadIdx.x];
        if (piece.from >= 0) {
            const int a = range_owner(total, blocks, piece.from), z = range_owner(total, blocks, piece.to - 1);
            unsigned int* const counter = reinterpret_cast<unsigned int*>(static_cast<uint8_t*>(p.workspace) + kRowsCounters) + a;
            __threadfence();
            if (atomicAdd(counter, 1u) == (unsigned int)(z - a)) {
                last = 1;
                *counter = 0;                         // as the next launch expects it
            }
            __threadfence();
        }
        s_last[threadIdx.x] = last;
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i) {
        if (!s_last[i]) continue;
        const int a = range_owner(total, blocks, cut[i].from), z = range_owner(total, blocks, cut[i].to - 1);
        for (int row = warp; row < cut[i].rows; row += S::kWarps) {
            Joined j{-INFINITY, 0.f, {}};
            for (int c = a; c <= z; ++c) add(j, block_parts + ((size_t)c * 2 + (c == a ? 1 : 0)) * S::kPartFloats, row, false);
            finish(j, cut[i], row);
        }
    }
}

// the cache's keys or values as (dim, token, head, page), read 16 tokens at a time in rows whose 16-byte chunks are swizzled
bool cache_map(CUtensorMap* out, const CacheView& c, bool keys) {
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.dim, 1ull << c.page_shift, (cuuint64_t)c.heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(keys ? c.k_token : c.v_token), (cuuint64_t)(keys ? c.k_head : c.v_head), (cuuint64_t)(keys ? c.k_page : c.v_page)};
    const cuuint32_t box[4] = {(cuuint32_t)c.dim, 16, 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode_with_context([&] {
        return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, keys ? c.k : c.v, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

template <bool E4M3, bool BF16, int D, int NT>
cudaError_t launch_rows(const AttentionParams& p, int most_rows, cudaStream_t stream) {
    using S = Shape<D, NT>;
    const auto kernel = cache_rows_kernel<E4M3, BF16, D, NT>;
    constexpr int kSmem = S::kWarps * S::kWarpBytes + 1024;
    CUtensorMap k_map, v_map;
    if (!cache_map(&k_map, p.cache, true) || !cache_map(&v_map, p.cache, false)) return cudaErrorNotSupported;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(kMaxBlocks, 1, 1);
    cfg.blockDim = dim3(S::kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p, most_rows, k_map, v_map);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

size_t cache_rows_workspace() { return kWarpPartsBytes + kBlockPartsBytes; }

// Two column tiles (16 rows) where a request may have more than 8 rows: its bytes are decoded once for both.
cudaError_t cache_rows_launch(const AttentionParams& p, bool e4m3, bool bf16, int most_rows, bool few, cudaStream_t stream) {
    const auto by_rows = [&](auto e, auto h, auto d) {
        constexpr bool E = decltype(e)::value, H = decltype(h)::value;
        constexpr int D = decltype(d)::value;
        return few ? launch_rows<E, H, D, 1>(p, most_rows, stream) : launch_rows<E, H, D, 2>(p, most_rows, stream);
    };
    const auto by_dim = [&](auto e, auto h) {
        return p.cache.dim == 128 ? by_rows(e, h, std::integral_constant<int, 128>{}) : by_rows(e, h, std::integral_constant<int, 64>{});
    };
    const auto by_type = [&](auto e) { return bf16 ? by_dim(e, std::true_type{}) : by_dim(e, std::false_type{}); };
    return e4m3 ? by_type(std::true_type{}) : by_type(std::false_type{});
}

}  // namespace i4mm
