// The cache's writer and its inverse (i4mm_cache_write, i4mm_cache_read).
//
// Per page and head, and for keys and values apart: a = the largest finite |x| of the tokens that the call adds,
//   s_new = min { 2^e : a <= most * 2^e },  s = max(s_old, s_new),  q = round(x / s),  q_held = round(q_held * s_old / s) where s grew.
// All scales are powers of two, so x / s and q * s are exact and the only rounding is the one to the byte: every implementation of these
// lines gives the same bytes.  A held value has been rounded at steps s, s / 2, s / 4 ... at most, so it is off by less than s.
// What bounds it: 16-bit rows in, bytes out, and each page's scale is needed before its first byte can be written.
#include <algorithm>

#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr int kWarps = 8;
constexpr uint32_t kAll = 0xFFFFFFFFu;

template <bool BF16>
__device__ __forceinline__ void unpack8(uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (BF16) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        } else {
            const float2 h = __half22float2(u32_as_h2(u[i]));
            f[2 * i] = h.x;
            f[2 * i + 1] = h.y;
        }
    }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    return h2_as_u32(__floats2half2_rn(a, b));
}

// the byte nearest to f, |f| within the type's range but for infinities; NaN -> 0
template <bool E4M3>
__device__ __forceinline__ uint32_t to_byte(float f) {
    constexpr float kMost = E4M3 ? 448.f : 127.f;
    f = f != f ? 0.f : fminf(fmaxf(f, -kMost), kMost);
    if (E4M3) return (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)__float2int_rn(f) & 0xFFu;
}
template <bool E4M3>
__device__ __forceinline__ float from_byte(uint32_t b) {
    if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
    return (float)(int)(signed char)b;
}

// The least power of two s with a <= most * s (0 for a = 0).  With a in [2^e, 2^(e+1)): most = 127 = 1.984 * 2^6 and 448 = 1.75 * 2^8, so
// s is 2^(e-6) (2^(e-8)) or the next one.  Not below 2^-100, so that 1 / s is a finite number whatever the input.
template <bool E4M3>
__device__ __forceinline__ float scale_for(float a) {
    if (a == 0.f) return 0.f;
    constexpr int kTop = E4M3 ? 8 : 6;
    constexpr float kMost = E4M3 ? 448.f : 127.f;
    const int e = max((int)(__float_as_uint(a) >> 23) - 127 - kTop, -100);   // (a subnormal a lies below the limit anyhow)
    const float s = __uint_as_float((uint32_t)(e + 127) << 23);
    return a > kMost * s ? 2.f * s : s;
}

// A warp takes one head's keys or values (blockIdx.y * kWarps + warp: 2 * head + which) of the runs that begin in a window of `window`
// tokens (window <= 16).  A run: neighbouring tokens with ascending slots of one page; it ends with the page, so it has at most 128 tokens.
template <bool E4M3, bool BF16>
__global__ void __launch_bounds__(kWarps * 32) cache_write_kernel(const CacheView c, const RowsView k, const RowsView v, int tokens,
                                                                  const int* slots, int window) {
    const int lane = threadIdx.x & 31;
    const int unit = blockIdx.y * kWarps + (threadIdx.x >> 5), head = unit >> 1, which = unit & 1;
    if (head >= c.heads) return;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int page = 1 << c.page_shift, lanes_per_row = c.dim >> 3, rows_per_step = 32 / lanes_per_row;
    const int row = lane / lanes_per_row, col = (lane % lanes_per_row) * 8;
    const uint16_t* x = (const uint16_t*)(which ? v.p : k.p) + head * (which ? v.head : k.head) + col;
    const long long x_token = which ? v.token : k.token;

    const int t0 = blockIdx.x * window;
    // lane i: the slot of token t0 - 1 + i
    const int t = t0 - 1 + lane;
    const int slot = lane <= window && t >= 0 && t < tokens ? slots[t] : -1;
    const int before = __shfl_up_sync(kAll, slot, 1);
    const bool valid = slot >= 0 && (slot >> c.page_shift) < c.pages;
    const bool begins = lane > 0 && valid && !(before >= 0 && slot == before + 1 && (slot & (page - 1)) != 0);
    for (uint32_t starts = __ballot_sync(kAll, begins); starts; starts &= starts - 1) {
        const int from = __ffs(starts) - 1, run = t0 - 1 + from;
        const int first_slot = __shfl_sync(kAll, slot, from);
        const int id = first_slot >> c.page_shift, place = first_slot & (page - 1);
        // its length
        int n = 1;
        while (n < page - place) {
            const int i = n + lane;
            const bool more = i < page - place && run + i < tokens && slots[run + i] == first_slot + i;
            const uint32_t stop = __ballot_sync(kAll, !more);
            if (stop) {
                n += __ffs(stop) - 1;
                break;
            }
            n += 32;
        }
        const uint16_t* rows = x + (long long)run * x_token;
        float a = 0.f;
        for (int i = row; i < n; i += rows_per_step) {
            float f[8];
            unpack8<BF16>(*reinterpret_cast<const uint4*>(rows + i * x_token), f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = fabsf(f[j]);
                a = m > a && m <= 3.4e38f ? m : a;                       // (neither infinities nor NaN)
            }
        }
#pragma unroll
        for (int d = 16; d; d /= 2) a = fmaxf(a, __shfl_xor_sync(kAll, a, d));
        float* const scale = reinterpret_cast<float*>(c.scales + (long long)id * c.heads + head) + which;
        const float old = place ? *scale : 0.f;
        const float s = fmaxf(old, scale_for<E4M3>(a));
        uint8_t* const held = (which ? c.v : c.k) + id * (which ? c.v_page : c.k_page) + head * (which ? c.v_head : c.k_head);
        const long long held_token = which ? c.v_token : c.k_token;
        if (s > old && old > 0.f) {
            const float ratio = old / s;
            for (int i = row; i < place; i += rows_per_step) {
                uint2* const at = reinterpret_cast<uint2*>(held + i * held_token + col);
                uint2 w = *at;
                uint32_t u[2] = {w.x, w.y}, r[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j >> 2] |= to_byte<E4M3>(from_byte<E4M3>(u[j >> 2] >> (8 * (j & 3)) & 0xFFu) * ratio) << (8 * (j & 3));
                *at = make_uint2(r[0], r[1]);
            }
        }
        const float inverse = s > 0.f ? 1.f / s : 1.f;
        for (int i = row; i < n; i += rows_per_step) {
            float f[8];
            unpack8<BF16>(*reinterpret_cast<const uint4*>(rows + i * x_token), f);
            uint32_t r[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j >> 2] |= to_byte<E4M3>(f[j] * inverse) << (8 * (j & 3));
            *reinterpret_cast<uint2*>(held + (place + i) * held_token + col) = make_uint2(r[0], r[1]);
        }
        __syncwarp();
        if (lane == 0) *scale = s;
    }
}

// a thread takes 8 values of one token, head and of keys or values
template <bool E4M3, bool BF16>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheView c, uint4* k_out, uint4* v_out, long long units, const int* slots) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int per_row = c.dim >> 3;
    for (long long u = blockIdx.x * 256ll + threadIdx.x; u < units; u += gridDim.x * 256ll) {
        const long long row = u / per_row;
        const int col = (int)(u - row * per_row) * 8;
        const long long t = row / c.heads;
        const int head = (int)(row - t * c.heads), which = blockIdx.y;
        const int slot = slots[t], id = slot >> c.page_shift;
        uint32_t r[4] = {0, 0, 0, 0};
        if (slot >= 0 && id < c.pages) {
            const int place = slot & ((1 << c.page_shift) - 1);
            const uint8_t* at = which ? c.v + id * c.v_page + head * c.v_head + place * c.v_token : c.k + id * c.k_page + head * c.k_head + place * c.k_token;
            const uint2 w = *reinterpret_cast<const uint2*>(at + col);
            const float2 both = c.scales[(long long)id * c.heads + head];
            const float s = which ? both.y : both.x;
            const uint32_t b[2] = {w.x, w.y};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = b[j >> 1] >> (16 * (j & 1));
                r[j] = pack2<BF16>(from_byte<E4M3>(two & 0xFFu) * s, from_byte<E4M3>(two >> 8 & 0xFFu) * s);
            }
        }
        (which ? v_out : k_out)[u] = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

template <typename F, typename... Args>
cudaError_t launch(F* kernel, dim3 grid, int threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

cudaError_t cache_write_launch(const CacheView& c, bool e4m3, const RowsView& k, const RowsView& v, bool bf16, int tokens, const int* slots,
                               cudaStream_t stream) {
    const int window = tokens > 1024 ? 16 : 1;
    const dim3 grid((unsigned)((tokens + window - 1) / window), (unsigned)((2 * c.heads + kWarps - 1) / kWarps), 1);
    const auto kernel = e4m3 ? (bf16 ? cache_write_kernel<true, true> : cache_write_kernel<true, false>)
                             : (bf16 ? cache_write_kernel<false, true> : cache_write_kernel<false, false>);
    return launch(kernel, grid, kWarps * 32, stream, c, k, v, tokens, slots, window);
}

cudaError_t cache_read_launch(const CacheView& c, bool e4m3, void* k_out, void* v_out, bool bf16, int tokens, const int* slots,
                              cudaStream_t stream) {
    const long long units = (long long)tokens * c.heads * (c.dim >> 3);
    const dim3 grid((unsigned)std::min((units + 255) / 256, 148ll * 64), 2, 1);
    const auto kernel = e4m3 ? (bf16 ? cache_read_kernel<true, true> : cache_read_kernel<true, false>)
                             : (bf16 ? cache_read_kernel<false, true> : cache_read_kernel<false, false>);
    return launch(kernel, grid, 256, stream, c, (uint4*)k_out, (uint4*)v_out, units, slots);
}

}  // namespace i4mm
