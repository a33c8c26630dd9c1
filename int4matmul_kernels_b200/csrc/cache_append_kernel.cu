// A step's queries and keys on their way from the projection to the attention (i4mm_cache_append): norm of each head, rotation, and keys and values
// quantised into their pages, in one launch.
//
//   y = x / sqrt(mean(x^2) + eps) * w      (without weights: y = x)
//   (a, b) -> (a cos - b sin, b cos + a sin)      for the pairs (i, i + F) or (2 i, 2 i + 1) of the first 2 F values, cos and sin from the step's table
// in fp32, rounded once to the activations' type; queries are stored so, keys go on to the cache as cache_write_kernel.cu says, and so do values,
// which are not changed.  So the bytes are those of a write of the rotated keys.
// What bounds it: with few tokens the chain of launch, slots, rows and old scales (1 token, 40 heads 4.0 us, 150 tokens, 32 on 8 heads 5.3; a write alone 2.3 and
// 3.6).  These are of steps in which no scale grows.  Where one does, a warp holds the page's earlier rows in the new scale one after the other, a load and a store
// each (append_singles; the writer takes two at a time), and the launch takes as long as the longest of these: 150 requests that decode on with normal values, pages of 64,
// grow 14 (int8, fp16) or 34 (e4m3, bf16) of 2400 scales a step, and take 29 or 26 us by events around the call, where the same without growth takes 10 (a write 14 to
// 16, and 7).
// With many tokens, issue slots (3 prompts, 4500 tokens, 40 heads 71 us where 16-bit rows in and out and bytes out are 36, a write alone 31).
#include <algorithm>

#include "cache_bytes.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr int kWarps = 8;
constexpr int kHeld = 8;                              // rows (two at head_dim 128, four at 64) that a warp holds at once
constexpr uint32_t kAll = 0xFFFFFFFFu;

enum Turn { kStraight, kHalves, kPairs };             // no rotation; pairs (i, i + F); pairs (2 i, 2 i + 1)

constexpr int kWindow = 16;                           // tokens whose runs a block looks at
constexpr int kMostGroups = 16;                       // more blocks of a window than these would each bring its angles to shared memory (cache_append_launch)
constexpr int kManyWarps = 8;
constexpr int kStaged = 32;                           // tokens whose angles a block keeps in shared memory

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}

// 1 / s; the writers' scales are powers of two, whose exponents turn over
__device__ __forceinline__ float inverse_of(float s) {
    const uint32_t bits = __float_as_uint(s);
    if (bits == 0) return 1.f;
    return (bits & 0x7FFFFFu) || bits >= 0x7F000000u ? 1.f / s : __uint_as_float(0x7F000000u - bits);
}
// 8 bytes of a page whose scale grows
template <bool E4M3>
__device__ __forceinline__ void requantise(uint8_t* at, float ratio) {
    const uint2 b = *reinterpret_cast<const uint2*>(at);
    const uint32_t u[2] = {b.x, b.y};
    uint32_t r[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j >> 2] |= to_byte<E4M3>(from_byte<E4M3>(u[j >> 2] >> (8 * (j & 3)) & 0xFFu) * ratio) << (8 * (j & 3));
    *reinterpret_cast<uint2*>(at) = make_uint2(r[0], r[1]);
}
template <bool E4M3, bool BF16>
__device__ __forceinline__ uint2 to_bytes_of(uint4 w, float inverse, bool finite) {
    if (!finite) return to_bytes_any<E4M3, BF16>(w, inverse);
    if (!BF16 && normal_half(inverse)) return half_to_bytes<E4M3>(w, h2_as_u32(__float2half2_rn(inverse)));
    float f[8];
    unpack8<BF16>(w, f);
    return to_bytes<E4M3>(f, inverse);
}

// the largest finite magnitude among 8 values
template <bool BF16>
__device__ __noinline__ float largest_finite(uint4 w) {
    float f[8], a = 0.f;
    unpack8<BF16>(w, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) a = fabsf(f[j]) <= 3.4e38f ? fmaxf(a, fabsf(f[j])) : a;
    return a;
}

// What a lane does to its 8 values of a row; the lanes of a row call together.
template <bool BF16, int TURN>
struct Turned {
    static constexpr int kTable = TURN == kHalves ? 4 : TURN == kPairs ? 2 : 1;         // 16 bytes of angles of a lane: two pairs each
    float2 weight[4];
    bool norm, turns;
    int partner, lanes;                               // the lane with the other halves; lanes of a row
    float sign;                                       // of the other value's part (kHalves)
    float eps, per;                                   // 1 / head_dim
    int first;                                        // the lane's first pair

    __device__ __forceinline__ Turned(const AppendParams& p, const void* w, int lane) {
        lanes = p.cache.dim >> 3;
        const int at = lane % lanes, col = 8 * at, pairs = p.pairs;
        norm = w != nullptr;
        eps = p.eps;
        per = 1.f / (float)p.cache.dim;
        turns = TURN != kStraight && col < 2 * pairs;
        const bool second = TURN == kHalves && col >= pairs;
        partner = !turns ? lane : second ? lane - (pairs >> 3) : lane + (pairs >> 3);
        sign = second ? 1.f : -1.f;
        first = !turns ? 0 : TURN == kPairs ? col / 2 : second ? col - pairs : col;
        if (norm) {
            float f[8];
            unpack8<BF16>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + col), f);
#pragma unroll
            for (int i = 0; i < 4; ++i) weight[i] = make_float2(f[2 * i], f[2 * i + 1]);
        }
    }
    // A token's angles, (cos, cos, sin, sin) of two pairs at a time: from shared memory, where the i-th 16 bytes of all lanes lie side by side, or
    // from the table
    __device__ __forceinline__ void angles(float4 (&t)[kTable], const float4* staged, int token, int pairs) const {
        if (TURN == kStraight) return;
        const int per_lane = 2 * kTable, across = pairs / per_lane;
#pragma unroll
        for (int i = 0; i < kTable; ++i) t[i] = staged[(token * kTable + i) * across + first / per_lane];
    }
    __device__ __forceinline__ void angles(float4 (&t)[kTable], const float2* table, long long token, int pairs) const {
        if (TURN == kStraight) return;
        const float4* const from = reinterpret_cast<const float4*>(table + token * pairs + first);
#pragma unroll
        for (int i = 0; i < kTable; ++i) {
            const float4 x = __ldg(from + i);
            t[i] = make_float4(x.x, x.z, x.y, x.w);
        }
    }

    __device__ __forceinline__ uint4 operator()(uint4 w, const float4 (&t)[kTable]) const {
        float g[8];
        unpack8<BF16>(w, g);
        float2 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = make_float2(g[2 * i], g[2 * i + 1]);
        if (norm) {
            float2 squares = mul2(f[0], f[0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) squares = fma2(f[i], f[i], squares);
            float sum = squares.x + squares.y;
            sum += __shfl_xor_sync(kAll, sum, 4);
            sum += __shfl_xor_sync(kAll, sum, 2);
            sum += __shfl_xor_sync(kAll, sum, 1);
            if (lanes == 16) sum += __shfl_xor_sync(kAll, sum, 8);
            const float r = rsqrtf(fmaf(sum, per, eps));
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = mul2(f[i], mul2(weight[i], make_float2(r, r)));
        }
        if constexpr (TURN == kHalves) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 other = make_float2(__shfl_sync(kAll, f[i].x, partner), __shfl_sync(kAll, f[i].y, partner));
                const float2 y = fma2(f[i], make_float2(t[i].x, t[i].y), mul2(mul2(other, make_float2(sign, sign)), make_float2(t[i].z, t[i].w)));
                if (turns) f[i] = y;
            }
        } else if constexpr (TURN == kPairs) {
            if (turns) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = i & 1 ? t[i / 2].y : t[i / 2].x, s = i & 1 ? t[i / 2].w : t[i / 2].z;
                    f[i] = make_float2(fmaf(f[i].x, c, -f[i].y * s), fmaf(f[i].y, c, f[i].x * s));
                }
            }
        }
        return make_uint4(pack2<BF16>(f[0].x, f[0].y), pack2<BF16>(f[1].x, f[1].y), pack2<BF16>(f[2].x, f[2].y), pack2<BF16>(f[3].x, f[3].y));
    }
};

// A block's view of its window: neighbouring tokens with ascending slots of one page are a run, the window's if it begins there.
struct Window {
    int t0, slot;                                     // lane i: the slot of token t0 - 1 + i
    uint32_t on, singles, runs;                       // lanes that go on with a run; where runs of one token and of several begin
    __device__ __forceinline__ Window(const AppendParams& p, int first) {
        const int lane = threadIdx.x & 31, t = first - 1 + lane, page = 1 << p.cache.page_shift;
        t0 = first;
        slot = t >= 0 && t < p.tokens ? p.slots[t] : -1;
        const int before = __shfl_up_sync(kAll, slot, 1);
        const bool goes_on = lane > 0 && before >= 0 && slot == before + 1 && (slot & (page - 1)) != 0;
        const bool begins = lane > 0 && lane <= kWindow && slot >= 0 && (slot >> p.cache.page_shift) < p.cache.pages && !goes_on;
        on = __ballot_sync(kAll, goes_on);
        const uint32_t starts = __ballot_sync(kAll, begins);
        singles = starts & ~(on >> 1);
        runs = starts & ~singles;
    }
    // the place of the n-th bit of a mask
    __device__ __forceinline__ static int nth_of(uint32_t mask, int n) {
        for (; n > 0; --n) mask &= mask - 1;
        return __ffs(mask) - 1;
    }
    // tokens of the run that begins at lane `from`: up to the first lane that does not go on; beyond the 32 lanes it is looked for
    __device__ __forceinline__ int length(const AppendParams& p, int from, int first_slot) const {
        const int lane = threadIdx.x & 31, page = 1 << p.cache.page_shift, left = page - (first_slot & (page - 1)), run = t0 - 1 + from;
        const uint32_t stop = ~on & (~0u << (from + 1));
        int n = stop ? __ffs(stop) - 1 - from : 32 - from;
#pragma unroll 1
        while (!stop && n < left) {
            const int i = n + lane;
            const bool more = i < left && run + i < p.tokens && p.slots[run + i] == first_slot + i;
            const uint32_t end = __ballot_sync(kAll, !more);
            if (end) {
                n += __ffs(end) - 1;
                break;
            }
            n += 32;
        }
        return n;
    }
};

__device__ __forceinline__ uint32_t largest_bits(uint32_t most, uint4 w) {                    // of magnitudes, two 16-bit values at a time
    return __vmaxu2(most, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
}
template <bool BF16>
__device__ __forceinline__ float from_bits(uint32_t most) {
    return BF16 ? __uint_as_float(most << 16) : __half2float(__ushort_as_half((unsigned short)most));
}

// Keys, then values, of tokens that are runs of their own: a warp takes `rows` heads of a token, each with its own scale.  `unit`: the warp's next one of
// units that all warps take in turns, counted from the first of these; it is moved on behind them.
template <bool E4M3, bool BF16, int TURN>
__device__ __forceinline__ void append_singles(const AppendParams& p, const Window& window, const Turned<BF16, TURN>& turned, int steps, int stride, int& unit) {
    using T = Turned<BF16, TURN>;
    const CacheView& c = p.cache;
    const int lane = threadIdx.x & 31, page = 1 << c.page_shift, lanes_per_row = c.dim >> 3, rows_per_step = 32 / lanes_per_row;
    const int row = lane / lanes_per_row, col = (lane % lanes_per_row) * 8, rows = steps * rows_per_step, per_token = (c.heads + rows - 1) / rows;
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const RowsView view = which ? p.v : p.k;
        const int count = __popc(window.singles) * per_token;
#pragma unroll 1
        for (; unit < count; unit += stride) {
            int part = unit, nth = 0;
            for (; part >= per_token; part -= per_token) ++nth;
            const int from = Window::nth_of(window.singles, nth), token = window.t0 - 1 + from, from_slot = __shfl_sync(kAll, window.slot, from);
            const int id = from_slot >> c.page_shift, at = from_slot & (page - 1), first = part * rows + row;
            const uint16_t* const x = static_cast<const uint16_t*>(view.p) + token * view.token + col;
            uint8_t* const held0 = (which ? c.v + id * c.v_page : c.k + id * c.k_page) + col;
            const long long held_token = which ? c.v_token : c.k_token, held_head = which ? c.v_head : c.k_head;
            float* const scales = reinterpret_cast<float*>(c.scales + (long long)id * c.heads) + which;
            uint4 w[kHeld];
            float olds[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i >= steps) break;
                const int head = first + i * rows_per_step;
                w[i] = make_uint4(0, 0, 0, 0);
                olds[i] = 0.f;
                if (head < c.heads) {
                    w[i] = *reinterpret_cast<const uint4*>(x + head * view.head);
                    if (at) olds[i] = scales[2 * head];
                }
            }
            float4 table[T::kTable];
            if (!which) turned.angles(table, p.angles, (long long)token, p.pairs);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i >= steps) break;
                const int head = first + i * rows_per_step;
                const bool real = head < c.heads;
                if (!which) w[i] = turned(w[i], table);
                uint32_t most = largest_bits(0, w[i]);
                most = max(most & 0xFFFFu, most >> 16);
                const bool finite = most < (BF16 ? 0x7F80u : 0x7C00u);        // (the lane's; what is not is left out of the row's largest)
                float a = from_bits<BF16>(most);
                if (!finite) a = largest_finite<BF16>(w[i]);
                for (int d = lanes_per_row >> 1; d; d >>= 1) a = fmaxf(a, __shfl_xor_sync(kAll, a, d));
                const float old = olds[i], s = fmaxf(old, scale_for<E4M3>(a));
                uint8_t* const held = held0 + head * held_head;
                if (real && s > old && at > 0) {
                    const float ratio = old / s;      // (0 where the scale was: bytes of infinities beside zeros go on standing for 0)
#pragma unroll 1
                    for (int j = 0; j < at; ++j) requantise<E4M3>(held + j * held_token, ratio);
                }
                const uint2 q = to_bytes_of<E4M3, BF16>(w[i], inverse_of(s), finite);
                if (real) {
                    *reinterpret_cast<uint2*>(held + at * held_token) = q;
                    if (col == 0) scales[2 * head] = s;
                }
            }
        }
        unit -= count;
    }
}

// Few tokens: a block's share of a window of 16, a warp a unit at a time.  Runs of a head's keys or values as the writer takes them, single tokens by
// heads, and the window's queries in the order of tokens and heads: `steps` times as many rows as the warp has at once.
template <bool E4M3, bool BF16, int TURN>
__global__ void __launch_bounds__(kWarps * 32, 2) cache_append_kernel(const AppendParams p, int groups, int steps) {
    using T = Turned<BF16, TURN>;
    const int lane = threadIdx.x & 31;
    const int block = (int)(blockIdx.x / groups), group = (int)(blockIdx.x - block * groups);
    const CacheView& c = p.cache;
    const int page = 1 << c.page_shift, lanes_per_row = c.dim >> 3, rows_per_step = 32 / lanes_per_row;
    const int row = lane / lanes_per_row, col = (lane % lanes_per_row) * 8, chunk = kHeld * rows_per_step, t0 = block * kWindow;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Window window(p, t0);
    const int rows = steps * rows_per_step, here = min(kWindow, p.tokens - t0), stride = groups * kWarps;
    int unit = group * kWarps + (threadIdx.x >> 5);   // the warp's next one, counted from the first of the kind that is being worked on
    uint4 w[kHeld];
    const int others = 2 * (__popc(window.runs) * c.heads + __popc(window.singles) * ((c.heads + rows - 1) / rows));

    // ---- runs of a head's keys, then of its values; single tokens ----
    if (unit < others) {
        const T turned(p, p.k_weight, lane);
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
            const RowsView view = which ? p.v : p.k;
            const long long page_stride = which ? c.v_page : c.k_page, head_stride = which ? c.v_head : c.k_head, token_stride = which ? c.v_token : c.k_token;
            const int count = __popc(window.runs) * c.heads;
#pragma unroll 1
            for (; unit < count; unit += stride) {
                int head = unit, nth = 0;
                for (; head >= c.heads; head -= c.heads) ++nth;
                const int from = Window::nth_of(window.runs, nth), run = t0 - 1 + from, first_slot = __shfl_sync(kAll, window.slot, from);
                const int id = first_slot >> c.page_shift, at = first_slot & (page - 1), n = window.length(p, from, first_slot);
                float* const scale = reinterpret_cast<float*>(c.scales + (long long)id * c.heads + head) + which;
                const float old = at ? *scale : 0.f;
                // the lane's part of kHeld rows at a time; a run that fits (a page of 16 tokens does) is read once
                const uint16_t* const first = static_cast<const uint16_t*>(view.p) + head * view.head + (run + row) * view.token + col;
                const auto fetch = [&](int i0) {
                    const uint16_t* x = first + i0 * view.token;
                    const int left = n - i0 - row;        // of the lane's rows: those with i * rows_per_step < left
#pragma unroll
                    for (int i = 0; i < kHeld; ++i, x += rows_per_step * view.token) {
                        w[i] = make_uint4(0, 0, 0, 0);
                        if (i * rows_per_step < left) w[i] = *reinterpret_cast<const uint4*>(x);
                    }
                    if (which) return;
#pragma unroll
                    for (int i = 0; i < kHeld; ++i) {     // (rows beyond the run are not used)
                        if (i0 + i * rows_per_step >= n) break;
                        float4 table[T::kTable];
                        turned.angles(table, p.angles, (long long)run + min(i0 + i * rows_per_step + row, n - 1), p.pairs);
                        const uint4 y = turned(w[i], table);
                        if (i * rows_per_step < left) w[i] = y;
                    }
                };
                uint32_t most = 0;
#pragma unroll 1
                for (int i0 = 0; i0 < n; i0 += chunk) {
                    fetch(i0);
#pragma unroll
                    for (int i = 0; i < kHeld; ++i) most = largest_bits(most, w[i]);
                }
                most = __reduce_max_sync(kAll, max(most & 0xFFFFu, most >> 16));
                const bool finite = most < (BF16 ? 0x7F80u : 0x7C00u);
                float a = from_bits<BF16>(most);
                if (!finite) {                                                   // the largest of the others
                    a = 0.f;
#pragma unroll 1
                    for (int i0 = 0; i0 < n; i0 += chunk) {
                        if (n > chunk) fetch(i0);
#pragma unroll
                        for (int i = 0; i < kHeld; ++i) a = fmaxf(a, largest_finite<BF16>(w[i]));
                    }
#pragma unroll
                    for (int d = 16; d; d /= 2) a = fmaxf(a, __shfl_xor_sync(kAll, a, d));
                }
                const float s = fmaxf(old, scale_for<E4M3>(a));
                uint8_t* const held = (which ? c.v : c.k) + id * page_stride + head * head_stride + col;
                if (s > old && at > 0) {
                    const float ratio = old / s;
#pragma unroll 1
                    for (int i = row; i < at; i += rows_per_step) requantise<E4M3>(held + i * token_stride, ratio);
                }
                const float inverse = inverse_of(s);
#pragma unroll 1
                for (int i0 = 0; i0 < n; i0 += chunk) {
                    if (n > chunk) fetch(i0);
                    const int left = n - i0 - row;
                    uint8_t* to = held + (at + i0 + row) * token_stride;
#pragma unroll
                    for (int i = 0; i < kHeld; ++i, to += rows_per_step * token_stride)
                        if (i * rows_per_step < left) *reinterpret_cast<uint2*>(to) = to_bytes_of<E4M3, BF16>(w[i], inverse, finite);
                }
                __syncwarp();
                if (lane == 0) *scale = s;
            }
            unit -= count;
        }
        append_singles<E4M3, BF16, TURN>(p, window, turned, steps, stride, unit);
    } else {
        unit -= others;
    }

    // ---- queries: rows of the window in the order of tokens and heads ----
    const int end = here * p.q_heads, count = (end + rows - 1) / rows;
    if (unit >= count) return;
    const T turned(p, p.q_weight, lane);
#pragma unroll 1
    for (; unit < count; unit += stride) {
        const int first = unit * rows + row, token0 = first / p.q_heads, head0 = first - token0 * p.q_heads;
        const uint16_t* const q = static_cast<const uint16_t*>(p.q.p) + t0 * p.q.token + col;
        const int left = end - first;                 // of the lane's rows: those with i * rows_per_step < left
        int token = token0, head = head0;
        const auto next = [&]() {
            for (head += rows_per_step; head >= p.q_heads; head -= p.q_heads) ++token;
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            if (i >= steps) break;
            if (i * rows_per_step < left) w[i] = *reinterpret_cast<const uint4*>(q + token * p.q.token + head * p.q.head);
            next();
        }
        token = token0;
        head = head0;
        uint16_t* to = static_cast<uint16_t*>(p.q_out) + ((long long)t0 * p.q_heads + first) * c.dim + col;
#pragma unroll
        for (int i = 0; i < kHeld; ++i, to += rows_per_step * c.dim) {
            if (i >= steps) break;
            const bool real = i * rows_per_step < left;
            float4 table[T::kTable];
            turned.angles(table, p.angles, (long long)t0 + (real ? token : 0), p.pairs);
            const uint4 y = turned(w[i], table);
            if (real) *reinterpret_cast<uint4*>(to) = y;
            next();
        }
    }
}

// Many tokens: the window's angles are brought to shared memory once for all heads, and a unit's rows (a head's run of keys or values, or a head's
// queries of the window) while the one before is worked on, each lane its own part of them, so that no registers hold them and no lane waits for another.
template <bool E4M3, bool BF16, int TURN>
__global__ void __launch_bounds__(kManyWarps * 32, 2) cache_append_many_kernel(const AppendParams p, int groups) {
    using T = Turned<BF16, TURN>;
    extern __shared__ uint4 s_rows[];                 // [warp][2][kHeld][lane], then the angles
    float4* const s_angles = reinterpret_cast<float4*>(s_rows + kManyWarps * 2 * kHeld * 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int block = (int)(blockIdx.x / groups), group = (int)(blockIdx.x - block * groups);
    const CacheView& c = p.cache;
    const int page = 1 << c.page_shift, lanes_per_row = c.dim >> 3, rows_per_step = 32 / lanes_per_row;
    const int row = lane / lanes_per_row, col = (lane % lanes_per_row) * 8, chunk = kHeld * rows_per_step, t0 = block * kWindow;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const Window window(p, t0);
    const int here = min(kWindow, p.tokens - t0), stride = groups * kManyWarps, run_units = __popc(window.runs) * c.heads, units = 2 * run_units + p.q_heads;
    uint4* const mine = s_rows + warp * 2 * kHeld * 32 + lane;

    struct Unit {
        int kind, n;                                  // 0 keys, 1 values, 2 queries; rows
        int head, run, id, at;                        // run: the first token
        float old;
        const uint16_t* x;                            // the lane's first row
        long long token;                              // stride
    };
    const auto describe = [&](int unit) {
        Unit u;
        u.kind = unit < run_units ? 0 : unit < 2 * run_units ? 1 : 2;
        u.head = unit - u.kind * run_units;
        u.run = t0;
        u.n = here;
        u.old = 0.f;
        u.id = u.at = 0;
        if (u.kind < 2) {
            int nth = 0;
            for (; u.head >= c.heads; u.head -= c.heads) ++nth;
            const int from = Window::nth_of(window.runs, nth), first_slot = __shfl_sync(kAll, window.slot, from);
            u.run = t0 - 1 + from;
            u.id = first_slot >> c.page_shift;
            u.at = first_slot & (page - 1);
            u.n = window.length(p, from, first_slot);
            if (u.at) u.old = *(reinterpret_cast<const float*>(c.scales + (long long)u.id * c.heads + u.head) + u.kind);
        }
        const RowsView& view = u.kind == 0 ? p.k : u.kind == 1 ? p.v : p.q;
        u.token = view.token;
        u.x = static_cast<const uint16_t*>(view.p) + u.head * view.head + (u.run + row) * u.token + col;
        return u;
    };
    const auto ask = [&](const Unit& u, int i0, uint4* to) {
        const uint16_t* x = u.x + i0 * u.token;
        const int left = u.n - i0 - row;              // of the lane's rows: those with i * rows_per_step < left
#pragma unroll
        for (int i = 0; i < kHeld; ++i, x += rows_per_step * u.token)
            if (i * rows_per_step < left) ptx::cp_async_16(ptx::smem_u32(to + 32 * i), x, 16);
    };

    int unit = group * kManyWarps + warp, buffer = 0;
    Unit now{};
    if (unit < units) {
        now = describe(unit);
        ask(now, 0, mine);
    }
    ptx::cp_async_commit();
    if constexpr (TURN != kStraight) {
        const int two = p.pairs / 2, across = p.pairs / (2 * T::kTable), all = min(kStaged, p.tokens - t0) * two;
        const float4* const from = reinterpret_cast<const float4*>(p.angles + (long long)t0 * p.pairs);
        for (int i = threadIdx.x; i < all; i += kManyWarps * 32) {
            const float4 x = __ldg(from + i);
            const int token = i / two, j = i - token * two;
            s_angles[(token * T::kTable + j % T::kTable) * across + j / T::kTable] = make_float4(x.x, x.z, x.y, x.w);
        }
        __syncthreads();
    }
    T turned(p, now.kind == 2 ? p.q_weight : p.k_weight, lane);
    bool of_queries = now.kind == 2;

#pragma unroll 1
    for (; unit < units; unit += stride) {
        Unit next{};
        uint4* const rows = mine + buffer * kHeld * 32;
        buffer ^= 1;
        if (unit + stride < units) {
            next = describe(unit + stride);
            ask(next, 0, mine + buffer * kHeld * 32);
        }
        ptx::cp_async_commit();
        ptx::cp_async_wait_group<1>();
        const int n = now.n;
        if (now.kind == 2) {
            if (!of_queries) turned = T(p, p.q_weight, lane);
            of_queries = true;
            uint16_t* to = static_cast<uint16_t*>(p.q_out) + ((long long)(t0 + row) * p.q_heads + now.head) * c.dim + col;
#pragma unroll 2
            for (int i = 0; i < kHeld; ++i, to += (long long)rows_per_step * p.q_heads * c.dim) {
                if (i * rows_per_step >= n) break;
                const int r = i * rows_per_step + row;
                float4 table[T::kTable];
                turned.angles(table, s_angles, min(r, n - 1), p.pairs);
                const uint4 y = turned(rows[32 * i], table);
                if (r < n) *reinterpret_cast<uint4*>(to) = y;
            }
            now = next;
            continue;
        }
        const bool near = now.run + n <= t0 + kStaged;
        uint32_t most = 0;
        // a run that does not fit in the lane's places is read again, and its keys are treated again, for the second pass
        const auto again = [&](int i0) {
            ask(now, i0, rows);
            ptx::cp_async_commit();
            ptx::cp_async_wait_group<0>();
        };
        const auto treat = [&](int i0) {
            if (now.kind) return;
#pragma unroll 2
            for (int i = 0; i < kHeld; ++i) {
                const int r = i0 + i * rows_per_step + row, token = now.run + min(r, n - 1);
                if (i0 + i * rows_per_step >= n) break;
                float4 table[T::kTable];
                if (near) turned.angles(table, s_angles, token - t0, p.pairs);
                else turned.angles(table, p.angles, (long long)token, p.pairs);
                rows[32 * i] = turned(rows[32 * i], table);
            }
        };
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += chunk) {
            if (i0 > 0) again(i0);
            treat(i0);
            const int left = n - i0 - row;
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (i * rows_per_step < left) most = largest_bits(most, rows[32 * i]);
        }
        most = __reduce_max_sync(kAll, max(most & 0xFFFFu, most >> 16));
        const bool finite = most < (BF16 ? 0x7F80u : 0x7C00u);
        float a = from_bits<BF16>(most);
        if (!finite) {                                                       // the largest of the others
            a = 0.f;
#pragma unroll 1
            for (int i0 = 0; i0 < n; i0 += chunk) {
                if (n > chunk) {
                    again(i0);
                    treat(i0);
                }
                const int left = n - i0 - row;
#pragma unroll 1
                for (int i = 0; i * rows_per_step < left && i < kHeld; ++i) a = fmaxf(a, largest_finite<BF16>(rows[32 * i]));
            }
            __syncwarp();
#pragma unroll
            for (int d = 16; d; d /= 2) a = fmaxf(a, __shfl_xor_sync(kAll, a, d));
        }
        const float old = now.old, s = fmaxf(old, scale_for<E4M3>(a));
        const long long token_stride = now.kind ? c.v_token : c.k_token;
        uint8_t* const held = (now.kind ? c.v + now.id * c.v_page + now.head * c.v_head : c.k + now.id * c.k_page + now.head * c.k_head) + col;
        if (s > old && now.at > 0) {
            const float ratio = old / s;              // (0 where the scale was: bytes of infinities beside zeros go on standing for 0)
#pragma unroll 1
            for (int i = row; i < now.at; i += rows_per_step) requantise<E4M3>(held + i * token_stride, ratio);
        }
        const float inverse = inverse_of(s);
        const uint32_t inverse2 = h2_as_u32(__float2half2_rn(inverse));
        const bool by_halves = !BF16 && finite && normal_half(inverse);
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += chunk) {
            if (n > chunk) {
                again(i0);
                treat(i0);
            }
            const int left = n - i0 - row;
            uint8_t* to = held + (now.at + i0 + row) * token_stride;
            if (by_halves) {
#pragma unroll
                for (int i = 0; i < kHeld; ++i, to += rows_per_step * token_stride)
                    if (i * rows_per_step < left) *reinterpret_cast<uint2*>(to) = half_to_bytes<E4M3>(rows[32 * i], inverse2);
            } else {
#pragma unroll 2
                for (int i = 0; i < kHeld; ++i, to += rows_per_step * token_stride)
                    if (i * rows_per_step < left) *reinterpret_cast<uint2*>(to) = to_bytes_of<E4M3, BF16>(rows[32 * i], inverse, finite);
            }
        }
        __syncwarp();
        if (lane == 0) *(reinterpret_cast<float*>(c.scales + (long long)now.id * c.heads + now.head) + now.kind) = s;
        now = next;
    }
    ptx::cp_async_wait_group<0>();
    if (window.singles == 0) return;
    unit -= units;
    append_singles<E4M3, BF16, TURN>(p, window, T(p, p.k_weight, lane), kHeld, stride, unit);
}

template <typename F>
cudaError_t launch_many(F* kernel, long long blocks, cudaStream_t stream, const AppendParams& p, int groups) {
    constexpr int kSmem = (kManyWarps * 2 * kHeld + kStaged) * 32 * 16;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kManyWarps * 32);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, p, groups);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

// Blocks enough for the GPU, a window to several of them, and no more rows to a warp than leave it full: a few tokens are spread over all of it.
// The second kernel where that gives a window 16 blocks or fewer (577 tokens and more): with more of them what it brings to shared memory is used too
// little.  First / second, dim 128, us: a prompt of 250 tokens, 40 on 40 heads 11.4 / 11.1, 600 18.3 / 15.7, 800 25.4 / 20.7, 1100 with 32 on 8 heads
// 16.7 / 14.0; single tokens, 32 on 8 heads: 250 8.5 / 12.0, 400 11.3 / 14.0, 600 16.1 / 16.1, 1000 20.5 / 18.9.
cudaError_t cache_append_launch(const AppendParams& p, bool e4m3, bool bf16, bool pairs_beside, cudaStream_t stream) {
    constexpr int kBlocks = 148 * 4;
    const int windows = (p.tokens + kWindow - 1) / kWindow, here = std::min(p.tokens, kWindow), rows_per_step = 256 / p.cache.dim;
    const long long all_steps = (long long)p.tokens * (p.q_heads + 2 * p.cache.heads) / rows_per_step;
    const int steps = (int)std::min<long long>(kHeld, all_steps / (kBlocks * kWarps / 2) + 1), rows = steps * rows_per_step;
    // (units of a window at most: tokens that are runs of their own, or runs of two)
    const long long singles = (long long)here * 2 * ((p.cache.heads + rows - 1) / rows), runs = (long long)(here + 1) / 2 * 2 * p.cache.heads;
    const long long units = std::max(singles, runs) + ((long long)here * p.q_heads + rows - 1) / rows;
    const int groups = (int)std::max<long long>(1, std::min<long long>((units + kWarps - 1) / kWarps, (kBlocks + windows - 1) / windows));
    const long long blocks = (long long)windows * groups;
    const auto by_size = [&](auto e, auto h, auto t) {
        constexpr bool E = decltype(e)::value, H = decltype(h)::value;
        constexpr int turn = decltype(t)::value;
        if ((kBlocks + windows - 1) / windows > kMostGroups) return launch_overlapping(cache_append_kernel<E, H, turn>, dim3((unsigned)blocks), kWarps * 32, stream, p, groups, steps);
        return launch_many(cache_append_many_kernel<E, H, turn>, blocks, stream, p, groups);
    };
    const auto by_turn = [&](auto e, auto h) {
        if (p.pairs == 0) return by_size(e, h, std::integral_constant<int, kStraight>{});
        return pairs_beside ? by_size(e, h, std::integral_constant<int, kPairs>{}) : by_size(e, h, std::integral_constant<int, kHalves>{});
    };
    const auto by_type = [&](auto e) { return bf16 ? by_turn(e, std::true_type{}) : by_turn(e, std::false_type{}); };
    return e4m3 ? by_type(std::true_type{}) : by_type(std::false_type{});
}

}  // namespace i4mm
