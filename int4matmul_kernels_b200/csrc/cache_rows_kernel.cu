// Attention over the paged 8-bit cache (i4mm_cache_attention), few rows per request: decoding.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j, over the tokens j that the row sees,
// in one pass with the running maximum and sum.  Every byte of the cache is read once and enters 2 multiply-adds for each of a head's few
// rows, so DRAM bounds it: 24 bytes a cycle and SM.  What the rest is made for is to keep that many bytes in flight and to decode them
// in less than that time:
//
// * Work.  The tokens of a request and head (a segment) are cut into tiles of 16.  All tiles of all segments in a row are dealt out in
//   equal contiguous ranges, to the blocks (one to an SM) and within them to the warps, whatever the lengths are.  What a
//   range cuts is joined: warps of a block through shared memory, blocks through the workspace, where the block that comes last adds up
//   all parts in their order (so results do not depend on which one it is).  Nobody waits for anybody.
// * Bytes.  A thread copies (cp.async) exactly the bytes that it will decode itself into a ring of its own, several tiles
//   ahead: no barrier anywhere in the loop, and no registers are held by loads in flight.
// * Products.  S^T = K Q^T and O^T = V^T P^T with mma.m16n8k16: the cache is the 16-row operand, the head's rows are the 8 columns, so a
//   tile costs 16 instructions for 8 rows.  The order of the 16 k of an instruction is free as long as both operands agree, so a thread
//   takes 16 consecutive bytes of a key row (and the same places of q), and 16 consecutive bytes of each of its four value rows; two
//   value rows become operand words by byte permutes.  int8 becomes fp16 by placing the byte in the mantissa of 1024 (exact), e4m3 by
//   the conversion instruction (exact).  The weights go from the accumulator layout to the operand layout by a transpose of 8 x 8 matrices.
// * Scales.  The page's key scale multiplies the scores.  Weights are rounded to fp16 relative to the largest of their tile, and each
//   tile's product joins the fp32 sums with the factor 2^(m_tile - m) * value scale: pages of any scales, none of it lost to fp16's
//   range.  A second product with the weights' rounding errors (their low halves) brings the output to fp32's exactness for 8 more
//   tensor instructions a tile, which the tensor pipe has spare.
#include <algorithm>
#include <type_traits>

#include "cache_attention.cuh"

namespace i4mm {
namespace {

constexpr int kTile = 16;                             // tokens; divides every page size
constexpr int kMinBlockTiles = 8, kMinWarpTiles = 2;  // fewer tiles than this are not cut further
constexpr uint32_t kNoPage = 0x7FC0DEADu;             // in the place of a scale: there is no such page

template <int D, int NT>
struct Shape {
    static constexpr int kWarps = NT == 1 ? 16 : 12;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kRows = 8 * NT;
    static constexpr int kStageBytes = 32 * D + 256;                          // a tile's keys, values, and 8 bytes of scales for each lane
    static constexpr int kStages = D == 128 ? (NT == 1 ? 3 : 4) : (NT == 1 ? 5 : 6);
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kPartFloats = kRows * D + 2 * kRows;                 // sums, maxima, totals of a part of a segment
    static_assert(kPartFloats * 4 <= kWarpBytes, "a warp leaves its last part in its ring");
};

// ---- behind the workspace's header: [a part per warp][two parts per block] ----
constexpr size_t kWarpPartsBytes = (size_t)kMaxBlocks * 12 * Shape<128, 2>::kPartFloats * 4;
static_assert(16 * Shape<128, 1>::kPartFloats <= 12 * Shape<128, 2>::kPartFloats, "room for either shape");
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
__device__ __forceinline__ long long units_of(const AttentionParams& p, int most_rows, int b) {
    const Few r = load_few(p, most_rows, b);
    if (r.rows == 0) return 0;
    return (long long)r.tiles * p.cache.heads * row_tiles<ROWS>(p, r);
}

// A place in the row of all tiles.
struct Cursor {
    long long left;                                   // tiles of the range from here on
    Few r;
    int b, segment, segments, tile;                   // the segment within the request, the tile within the segment
};

template <int ROWS>
__device__ __forceinline__ void enter_request(const AttentionParams& p, int most_rows, Cursor& c) {
    c.r = load_few(p, most_rows, c.b);
    c.segments = p.cache.heads * row_tiles<ROWS>(p, c.r);
    c.segment = 0;
    c.tile = 0;
}

template <int ROWS>
__device__ __forceinline__ void advance(const AttentionParams& p, int most_rows, Cursor& c) {
    if (--c.left == 0) return;
    if (++c.tile < c.r.tiles) return;
    c.tile = 0;
    if (++c.segment < c.segments) return;
    do {
        if (++c.b >= p.requests) {                    // (not unless the lengths change under the kernel)
            c.left = 0;
            return;
        }
        enter_request<ROWS>(p, most_rows, c);
    } while (c.r.rows == 0);
}

// ---- decoding and products -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
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
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 1) cache_rows_kernel(const AttentionParams p, int most_rows) {
    using S = Shape<D, NT>;
    constexpr int kSteps = D / 16, kWords = D / 32;   // k steps of 16; words of 4 bytes that a thread has of a value row
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ Piece s_head[S::kWarps], s_tail[S::kWarps];
    __shared__ int s_last[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const CacheView& cache = p.cache;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();

    // rows of no request
    {
        const int first = p.requests == 0 ? 0 : p.cu_lens ? min(max(p.cu_lens[p.requests], 0), p.tokens) : p.requests;
        const long long from = (long long)first * p.q_heads * D, to = (long long)p.tokens * p.q_heads * D;
        for (long long i = from + 8ll * (blockIdx.x * S::kThreads + threadIdx.x); i < to; i += 8ll * gridDim.x * S::kThreads)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i) = make_uint4(0, 0, 0, 0);
    }

    // all tiles; the block's range and the warp's
    long long total = 0;
    for (int b = lane; b < p.requests; b += 32) total += units_of<S::kRows>(p, most_rows, b);
#pragma unroll
    for (int d = 16; d; d /= 2) total += __shfl_xor_sync(kAll, total, d);
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
        // the request that the range begins in
        Cursor cur;
        {
            long long before = 0;
            int base = 0;
            for (;; base += 32) {
                const long long own = base + lane < p.requests ? units_of<S::kRows>(p, most_rows, base + lane) : 0;
                long long sum = own;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const long long o = __shfl_up_sync(kAll, sum, d);
                    if (lane >= d) sum += o;
                }
                const uint32_t here = __ballot_sync(kAll, before + sum > u0);
                if (here) {
                    const int l = __ffs(here) - 1;
                    before += __shfl_sync(kAll, sum - own, l);
                    base += l;
                    break;
                }
                before += __shfl_sync(kAll, sum, 31);
                if (base + 32 >= p.requests) break;   // (as above)
            }
            cur.b = min(base, p.requests - 1);
            enter_request<S::kRows>(p, most_rows, cur);
            const long long in = u0 - before;
            cur.segment = (int)(in / cur.r.tiles);
            cur.tile = (int)(in - (long long)cur.segment * cur.r.tiles);
            cur.left = u1 - u0;
        }

        // ---- copies ----
        Cursor ahead = cur;
        int rt = row_tiles<S::kRows>(p, ahead.r);
        const auto page_of = [&](const Cursor& c) {
            const int j = (c.r.lo / kTile + c.tile) >> (cache.page_shift - 4);
            return j < p.table_width && c.r.limit > c.r.lo ? p.table[c.b * p.table_stride + j] : -1;
        };
        int id = page_of(ahead);
        uint32_t fill = my_ring;
        const auto copy = [&]() {
            if (ahead.left > 0) {
                const int first = (ahead.r.lo / kTile + ahead.tile) * kTile, place = first & ((1 << cache.page_shift) - 1);
                const int head = ahead.segment / rt;
                const bool there = id >= 0 && id < cache.pages;
                const long long page = there ? id : 0;
                const uint8_t* const k = cache.k + page * cache.k_page + head * cache.k_head + (place + g) * cache.k_token + 16 * t;
                const uint8_t* const v = cache.v + page * cache.v_page + head * cache.v_head + (place + 2 * t) * cache.v_token + (D / 8) * g;
                // bytes of tokens that nobody sees are not brought in: they may be anything, and 0 * NaN is NaN
                const auto seen = [&](int i) { return there && first + i >= ahead.r.lo && first + i < ahead.r.limit; };
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < D / 64; ++j)
                        ptx::cp_async_16(fill + (h * (D / 64) + j) * 512 + lane * 16, k + 8 * h * cache.k_token + 64 * j, there ? 16 : 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = (i & 1) + 8 * (i >> 1);
                    const uint8_t* const from = v + token * cache.v_token;
                    if (D == 128) ptx::cp_async_16(fill + 2048 + i * 512 + lane * 16, from, seen(2 * t + token) ? 16 : 0);
                    else cp_async_8(fill + 1024 + i * 256 + lane * 8, from, seen(2 * t + token) ? 8 : 0);
                }
                if (there) cp_async_8(fill + 32 * D + lane * 8, cache.scales + page * cache.heads + head, 8);
                else sts64(fill + 32 * D + lane * 8, kNoPage, kNoPage);
                const int b = ahead.b;
                advance<S::kRows>(p, most_rows, ahead);
                if (ahead.left > 0) {
                    if (ahead.b != b) rt = row_tiles<S::kRows>(p, ahead.r);
                    id = page_of(ahead);
                }
            }
            ptx::cp_async_commit();
            fill = fill + S::kStageBytes == my_ring + S::kWarpBytes ? my_ring : fill + S::kStageBytes;
        };
        for (int i = 0; i < S::kStages - 1; ++i) copy();

        // ---- the segments of the range ----
        uint32_t stage = my_ring;
        long long at = u0;
        while (at < u1) {
            const Few r = cur.r;
            const int tiles_here = (int)min((long long)(r.tiles - cur.tile), u1 - at), first_tile = cur.tile;
            const int row_tile_count = row_tiles<S::kRows>(p, r), head = cur.segment / row_tile_count, base = (cur.segment - head * row_tile_count) * S::kRows;
            const int b = cur.b, segment = cur.segment, all_rows = r.rows * p.group;
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

            for (int i = 0; i < tiles_here; ++i) {
                copy();
                ptx::cp_async_wait_group<S::kStages - 1>();
                const int first = (r.lo / kTile + first_tile + i) * kTile;
                // scores
                float s[NT][4] = {};
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    const uint4 ka = ptx::lds128(stage + j * 512 + lane * 16), kb = ptx::lds128(stage + (D / 64 + j) * 512 + lane * 16);
                    const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t a0, a1, a2, a3;
                        decode4<E4M3>(wa[w], a0, a2);
                        decode4<E4M3>(wb[w], a1, a3);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma(s[n], a0, a1, a2, a3, q[n][2 * (4 * j + w)], q[n][2 * (4 * j + w) + 1]);
                    }
                }
                const uint2 both = ptx::lds64(stage + 32 * D + lane * 8);
                const bool there = both.x != kNoPage;
                const float k_scale = there ? __uint_as_float(both.x) : 0.f, v_scale = there ? __uint_as_float(both.y) : 0.f;
                const bool whole = there && first >= r.lo && first + kTile - 1 <= r.position && first + kTile <= r.limit &&
                                   (!p.window || first > r.position + r.rows - 1 - p.window) && base + S::kRows <= all_rows;
                uint32_t high[NT][2], low[NT][2];
                float weight[NT][2];                  // of the tile's sums in the segment's
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float most[2];
#pragma unroll
                    for (int i2 = 0; i2 < 4; ++i2) s[n][i2] *= factor[n][i2 & 1] * k_scale;
                    if (!whole) {
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) {
                            const int token = first + g + 8 * (i2 >> 1), at_row = position[n][i2 & 1];
                            const bool sees = there && token <= at_row && token < r.limit && token >= r.lo && (!p.window || token > at_row - p.window);
                            if (!sees) s[n][i2] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        float x = fmaxf(s[n][i2], s[n][2 + i2]);
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
                    float e[4];
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        const bool any = most[i2] != -INFINITY;
                        const float from = any ? most[i2] : 0.f, up = any ? exp2_approx(most[i2] - m[n][i2]) : 0.f;
                        e[i2] = exp2_approx(s[n][i2] - from);
                        e[2 + i2] = exp2_approx(s[n][2 + i2] - from);
                        sum[n][i2] += up * (e[i2] + e[2 + i2]);
                        weight[n][i2] = up * v_scale;
                    }
#pragma unroll
                    for (int i2 = 0; i2 < 2; ++i2) {
                        const __half2 h = __floats2half2_rn(e[2 * i2], e[2 * i2 + 1]);
                        const float2 back = __half22float2(h);
                        high[n][i2] = transpose8x8(h2_as_u32(h));
                        low[n][i2] = transpose8x8(h2_as_u32(__floats2half2_rn(e[2 * i2] - back.x, e[2 * i2 + 1] - back.y)));
                    }
                }
                // values
                uint32_t v[4][kWords];
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                    if constexpr (D == 128) {
                        const uint4 w = ptx::lds128(stage + 2048 + i2 * 512 + lane * 16);
                        v[i2][0] = w.x; v[i2][1] = w.y; v[i2][2] = w.z; v[i2][3] = w.w;
                    } else {
                        const uint2 w = ptx::lds64(stage + 1024 + i2 * 256 + lane * 8);
                        v[i2][0] = w.x; v[i2][1] = w.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < 2 * kWords; ++j) {
                    uint32_t a0, a1, a2, a3;
                    decode_pair<E4M3>(v[0][j >> 1], v[1][j >> 1], j & 1, a0, a1);
                    decode_pair<E4M3>(v[2][j >> 1], v[3][j >> 1], j & 1, a2, a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float d[4] = {};
                        mma(d, a0, a1, a2, a3, low[n][0], low[n][1]);
                        mma(d, a0, a1, a2, a3, high[n][0], high[n][1]);
#pragma unroll
                        for (int i2 = 0; i2 < 4; ++i2) o[n][j][i2] += weight[n][i2 & 1] * d[i2];
                    }
                }
                stage = stage + S::kStageBytes == my_ring + S::kWarpBytes ? my_ring : stage + S::kStageBytes;
                advance<S::kRows>(p, most_rows, cur);
            }
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
                if (last) ptx::cp_async_wait_group<0>();
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
                    const long long from = at - tiles_here - first_tile;
                    (last ? s_tail : s_head)[warp] = Piece{from, from + r.tiles, b, segment, min(S::kRows, all_rows - base)};
                }
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
        const float pm = load(S::kRows * D + row), ps = load(S::kRows * D + S::kRows + row);
        const float next = fmaxf(a.m, pm);
        const float keep = a.m == -INFINITY ? 0.f : exp2_approx(a.m - next), take = pm == -INFINITY ? 0.f : exp2_approx(pm - next);
        a.m = next;
        a.sum = a.sum * keep + ps * take;
#pragma unroll
        for (int i = 0; i < kMine; ++i) a.o[i] = a.o[i] * keep + load(row * D + kMine * lane + i) * take;
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

template <bool E4M3, bool BF16, int D, int NT>
cudaError_t launch_rows(const AttentionParams& p, int most_rows, cudaStream_t stream) {
    using S = Shape<D, NT>;
    const auto kernel = cache_rows_kernel<E4M3, BF16, D, NT>;
    constexpr int kSmem = S::kWarps * S::kWarpBytes;
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
    e = cudaLaunchKernelEx(&cfg, kernel, p, most_rows);
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
