// What the two attention kernels of the paged 8-bit cache share: a request as they see it, the decoding of bytes, the workspace.
#pragma once

#include <cuda.h>

#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"

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
// 4-D tiled tensor-map copy, coordinates (x = innermost, y, z, w)
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
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

// The two kernels.  Few rows: requests of more than most_rows rows are left to the other one; `few`: no request has more than 8.
// Prompts: requests of fewer than least_rows rows are left to the other one; `alone`: it is not launched.
cudaError_t cache_rows_launch(const AttentionParams& p, bool e4m3, bool bf16, int most_rows, bool few, cudaStream_t stream);
cudaError_t cache_prompt_launch(const AttentionParams& p, bool e4m3, bool bf16, int least_rows, bool alone, cudaStream_t stream);
size_t cache_rows_workspace();                        // bytes behind the header
size_t cache_prompt_workspace();                      // bytes behind those

}  // namespace i4mm
