// What the attention kernels of the paged 8-bit cache share: a request as they see it, the decoding of bytes, the workspace.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"
#include "tensor_map.cuh"

namespace i4mm {

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxBlocks = 148;                       // one block to an SM
// ---- PTX that only these kernels use ---------------------------------------------------------------------------------------------------------
namespace ptx {
// 8 bytes; cp_async_arrive: this thread arrives on the barrier (which counts it) once its copies so far are done
__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_l1(const void* at) { asm volatile("prefetch.global.L1 [%0];" ::"l"(at)); }
// 4-D tiled tensor-map copy, coordinates (x = innermost, y, z, w)
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// D[tmem] (+)= A[smem descriptor] * B[smem descriptor]; kind::f16; one thread issues
__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
}  // namespace ptx

// Requests of at most this many rows (new tokens times query heads of a key head) are the few-row kernel's, wherever both run
constexpr int kFewRows = 64;

// ---- the workspace: [counters, with the status word where i4mm_device_status looks for it][parts of the few-row kernel][of the other] ----
constexpr size_t kCacheHeaderBytes = kCounterBytes;
constexpr size_t kRowsCounters = 0;                   // one per block
constexpr size_t kPromptNext = 4096;                  // the next item to be worked on
constexpr size_t kPromptCounters = 8192;              // two per part
constexpr int kPromptParts = 320;
constexpr size_t kPrefixCounters = 16384;             // two per block
// Tiles' worth of a block's time that it takes to begin a segment of the prefix kernel, where there are enough of them that many blocks begin a second one
// (an eighth of the blocks).  0 / 3 / 6, us: 64 rows, 40 heads, 4000 tokens 128.6 / 124.1 / 125.0, 16 rows 39.0 / 36.5 / 38.0, 5 prefixes of 48 rows, 8 heads
// of 64 41.4 / 37.6 / 39.2; 16 rows of 8 heads, 4000 tokens, with and without 26.5 / 23.4.
constexpr int kPrefixBegin = 3;
constexpr int kPrefixRows = 64;                       // rows of a tile of the prefix kernel

struct Request {
    int row0, rows;                                   // its packed rows
    int position;                                     // of the first of them
    int lo, limit;                                    // tokens lo .. limit - 1 may be seen
};

__device__ __forceinline__ Request load_request(const AttentionParams& p, int b) {
    Request r;
    const int seq = p.seq_lens[b];
    int n = 1;
    if (p.cu_lens) {
        const int from = p.cu_lens[b], to = p.cu_lens[b + 1];
        n = to - from;
        r.row0 = min(max(from, 0), p.tokens);
        r.rows = max(min(to, p.tokens) - r.row0, 0);
    } else {
        r.row0 = b;
        r.rows = 1;
    }
    r.position = seq - n;
    r.limit = max(min(min(seq, r.position + r.rows), p.table_width << p.cache.page_shift), 0);
    r.lo = p.window && r.position >= p.window ? r.position - p.window + 1 : 0;
    if (r.lo > r.limit) r.lo = r.limit;
    return r;
}

// ---- sums over a warp
__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int d = 16; d; d /= 2) v += __shfl_xor_sync(kAll, v, d);
    return v;
}
__device__ __forceinline__ long long warp_prefix(long long v) {             // sum over this lane and those before it
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long o = __shfl_up_sync(kAll, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// ---- decoding --------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLeastScale = 7.888609e-31f;          // 2^-100 in the place of a value scale of 0: its bytes are 0, its tokens still have weight
// two e4m3 bytes (low and high) -> two fp16
__device__ __forceinline__ uint32_t e4m3_to_h2(uint32_t two) {
    uint32_t d;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(two));
    return d;
}
// bytes 0 and 2 of w -> two fp16: in the mantissa of 1024, with the sign bit turned over, q is 1152 + q
__device__ __forceinline__ uint32_t int8_to_h2(uint32_t w) {
    uint32_t x;
    asm("lop3.b32 %0, %1, 0x00FF00FF, %2, 0x6A;" : "=r"(x) : "r"(w), "r"(0x64806480u));    // (w & 0x00FF00FF) ^ 0x64806480
    return hsub2_u(x, 0x64806480u);
}
// 4 bytes -> 2 x 2 fp16.  int8: bytes (0, 2) and (1, 3); e4m3: (0, 1) and (2, 3)
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& x, uint32_t& y) {
    if (E4M3) {
        x = e4m3_to_h2(w);
        y = e4m3_to_h2(w >> 16);
    } else {
        x = int8_to_h2(w);
        y = int8_to_h2(w >> 8);
    }
}
// four fp16 of a query in the order that decode4 gives the keys
template <bool E4M3>
__device__ __forceinline__ uint2 key_order(uint2 w) {
    return E4M3 ? w : make_uint2(prmt(w.x, w.y, 0x5410), prmt(w.x, w.y, 0x7632));
}
// bytes 2 * half, 2 * half + 1 of two rows a, b -> fp16 pairs (a, b) of the one place and of the next
template <bool E4M3>
__device__ __forceinline__ void decode_pair(uint32_t a, uint32_t b, int half, uint32_t& x, uint32_t& y) {
    if (E4M3) {
        const uint32_t w = prmt(a, b, half ? 0x7362 : 0x5140);
        x = e4m3_to_h2(w);
        y = e4m3_to_h2(w >> 16);
    } else {
        const uint32_t w = prmt(a, b, half ? 0x7632 : 0x5410);
        x = int8_to_h2(w);
        y = int8_to_h2(w >> 8);
    }
}

// ---- bf16 queries are brought into fp16's range by a power of two for each row: 2^e <= most < 2^(e + 1), q * 2^-e is below 2 --------------
__device__ __forceinline__ float bf16_most(uint2 w) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(w.x << 16)), fabsf(__uint_as_float(w.x & 0xFFFF0000u))),
                 fmaxf(fabsf(__uint_as_float(w.y << 16)), fabsf(__uint_as_float(w.y & 0xFFFF0000u))));
}
__device__ __forceinline__ void bf16_powers(float most, float& up, float& down) {
    const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126);
    down = __uint_as_float((uint32_t)(127 - e) << 23);
    up = __uint_as_float((uint32_t)(127 + e) << 23);
}
__device__ __forceinline__ uint2 bf16_scaled(uint2 w, float down) {
    return make_uint2(h2_as_u32(__floats2half2_rn(__uint_as_float(w.x << 16) * down, __uint_as_float(w.x & 0xFFFF0000u) * down)),
                      h2_as_u32(__floats2half2_rn(__uint_as_float(w.y << 16) * down, __uint_as_float(w.y & 0xFFFF0000u) * down)));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&x);
    }
    return h2_as_u32(__floats2half2_rn(a, b));
}

// ---- a row's own sums and those of its shared prefix -------------------------------------------------------------------------------
// (m, sum, o) of disjoint sets of tokens add up as in (max m; factors 2^(m - max) on sum and o): `own` and `prefix` are those factors over the whole sum
struct Joint {
    float own, prefix;
};
__device__ __forceinline__ Joint join_prefix(float m, float sum, float2 prefix) {
    const float top = fmaxf(m, prefix.x);
    const float a = m == -INFINITY ? 0.f : exp2_approx(m - top), b = prefix.x == -INFINITY ? 0.f : exp2_approx(prefix.x - top);
    const float total = fmaf(sum, a, prefix.y * b), f = total > 0.f ? 1.f / total : total;      // (a NaN stays one)
    return {a * f, b * f};
}
// ---- what a row's prefix came to: joined, or in parts -----------------------------------------------------------------------------
// The prefix kernel leaves a row's (m, total) and sums.  Where many blocks had a part of the prefix each, `total` is negative and m's bits name
// them: blocks a .. a + count - 1, and the row's place in their tiles.  Whoever reads the row adds them up: all SMs do that at once, where a block that
// joined 18 parts of 64 rows read 0.6 MB alone (8 us).  A few parts are better joined there (64 requests of 300 tokens of their own behind 4000
// of 40 heads, 4 parts: 130 us, and 175 where each row's reader looks for them at the end of its tokens).
__device__ __forceinline__ float2 in_parts(int a, int count, int row) { return make_float2(__int_as_float(a | count << 8 | row << 16), -1.f); }
struct PrefixParts {
    const float* base;
    int a, count, row, dim;
    __device__ __forceinline__ PrefixParts(const AttentionParams& p, float2 told) {
        const int bits = __float_as_int(told.x);
        a = bits & 0xFF;
        count = bits >> 8 & 0xFF;
        row = bits >> 16 & 0xFF;
        // A row that no list names, or whose prefix kernel gave up, has in this place whatever the caller's scratch holds: what names no parts is no prefix.
        if (bits >> 24 || a + count > kMaxBlocks || row >= kPrefixRows) count = 0;
        dim = p.cache.dim;
        base = reinterpret_cast<const float*>(static_cast<const uint8_t*>(p.workspace) + p.prefix_parts);
    }
    // a block's two places: of a segment that it goes on with, and of one that begins with it
    __device__ __forceinline__ const float* part(int i) const { return base + (size_t)(2 * (a + i) + (i == 0 ? 1 : 0)) * (kPrefixRows * dim + 2 * kPrefixRows); }
    __device__ __forceinline__ const float* sums(int i) const { return part(i) + row * dim; }
    __device__ __forceinline__ float2 total(int i) const { return __ldcg(reinterpret_cast<const float2*>(part(i) + kPrefixRows * dim + 2 * row)); }
    __device__ __forceinline__ float most() const {
        float m = -INFINITY;
#pragma unroll 8
        for (int i = 0; i < count; ++i) m = fmaxf(m, total(i).x);
        return m;
    }
};
// N of the row's sums, from column `col` on, and its (m, total)
template <int N>
__device__ __forceinline__ float2 prefix_sums(const AttentionParams& p, float2 told, long long at, int col, float (&sums)[N]) {
    static_assert(N % 2 == 0, "two at a time at least");
    using Some = std::conditional_t<N % 4 == 0, float4, float2>;
    constexpr int kSome = sizeof(Some) / 4;
    if (!(told.y < 0.f)) {
#pragma unroll
        for (int k = 0; k < N; k += kSome) *reinterpret_cast<Some*>(sums + k) = *reinterpret_cast<const Some*>(p.prefix_sums + at * p.cache.dim + col + k);
        return told;
    }
    const PrefixParts parts(p, told);
    const float m = parts.most(), from = m == -INFINITY ? 0.f : m;
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) sums[k] = 0.f;
#pragma unroll 2
    for (int i = 0; i < parts.count; ++i) {
        const float2 of = parts.total(i);
        const float take = exp2_approx(of.x - from);
        total = fmaf(take, of.y, total);
#pragma unroll
        for (int k = 0; k < N; k += kSome) {
            alignas(16) float x[kSome];
            *reinterpret_cast<Some*>(x) = __ldcg(reinterpret_cast<const Some*>(parts.sums(i) + col + k));
#pragma unroll
            for (int e = 0; e < kSome; ++e) sums[k + e] = fmaf(take, x[e], sums[k + e]);
        }
    }
    return make_float2(m, total);
}

// the position of packed row `token`, which reads the prefix at `place`, that prefix counted
__device__ __forceinline__ int behind_prefix(const AttentionParams& p, int place, int token) {
    int b = min(token, p.requests - 1);
    if (p.cu_lens) {
        int hi = p.requests - 1;
#pragma unroll 1
        for (b = 0; b < hi;) {
            const int mid = (b + hi + 1) >> 1;
            if (p.cu_lens[mid] <= token) b = mid;
            else hi = mid - 1;
        }
    }
    const long long position = (long long)p.seq_lens[place] + p.seq_lens[b] - (p.cu_lens ? p.cu_lens[b + 1] : b + 1) + token;
    return (int)min(max(position, 0ll), 0x7FFFFFFEll);
}
// whether a row of request b at this position sees a prefix
__device__ __forceinline__ bool sees_prefix(const AttentionParams& p, int b, int position) { return position >= 0 && p.prefix_of[b] >= 0; }

// the cache's keys or values as (dim, token, head, page), read `tokens` tokens at a time in rows whose 16-byte chunks are swizzled
inline bool cache_map(CUtensorMap* out, const CacheView& c, bool keys, int tokens) {
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.dim, 1ull << c.page_shift, (cuuint64_t)c.heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(keys ? c.k_token : c.v_token), (cuuint64_t)(keys ? c.k_head : c.v_head), (cuuint64_t)(keys ? c.k_page : c.v_page)};
    const cuuint32_t box[4] = {(cuuint32_t)c.dim, (cuuint32_t)tokens, 1, 1}, steps[4] = {1, 1, 1, 1};
    return encode_with_context([&] {
        return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, keys ? c.k : c.v, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

// The two kernels of requests' own tokens.  Few rows: requests of more than most_rows rows are left to the other one; `few`: no request has more than 8.
// Prompts: requests of fewer than least_rows rows are left to the other one; `alone`: it is not launched.
// With p.prefix_of set, both add what p.prefix_total and p.prefix_sums say to each row that has a prefix.
cudaError_t cache_rows_launch(const AttentionParams& p, bool e4m3, bool bf16, int most_rows, bool few, cudaStream_t stream);
cudaError_t cache_prompt_launch(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, bool alone, cudaStream_t stream);
// Rows of all requests that share a prefix over that prefix, into p.prefix_total and p.prefix_sums: of prefixes that up to most_rows rows of a key
// head read, and of those that least_rows read or more.
cudaError_t cache_prefix_launch(const AttentionParams& p, bool e4m3, bool bf16, int most_rows, cudaStream_t stream);
cudaError_t cache_many_readers_launch(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, cudaStream_t stream);
size_t cache_rows_workspace();                        // bytes behind the header
size_t cache_prompt_workspace();                      // bytes behind those
size_t cache_prefix_workspace();                      // and behind those

}  // namespace i4mm
