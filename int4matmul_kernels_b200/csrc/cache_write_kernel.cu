// The cache's writer and its inverse (i4mm_cache_write, i4mm_cache_read).
//
// Per page and head, and for keys and values apart: a = the largest finite |x| of the tokens that the call adds,
//   s_new = min { 2^e : a <= most * 2^e },  s = max(s_old, s_new),  q = round(x / s),  q_held = round(q_held * s_old / s) where s grew.
// All scales are powers of two, so x / s and q * s are exact and the only rounding is the one to the byte: every implementation of these
// lines gives the same bytes.  A held value has been rounded at steps s, s / 2, s / 4 ... at most, so it is off by less than s.
// What bounds it: 16-bit rows in, bytes out, and each page's scale is needed before its first byte can be written.  A warp holds the 16 rows of
// a page in registers between the two, so they are read once; magnitudes are compared as 16-bit integers.  4500 tokens of 40 heads of 128: 33 us
// (4.2 TB/s; 1000 instructions for 16 rows), and 25 us (5.6 TB/s) for the reader; one token 3 and 2 us.
#include <algorithm>

#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr int kWarps = 8;
constexpr int kHeld = 8;                              // rows (two at head_dim 128, four at 64) that a warp of the writer holds at once
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

// 8 values times `inverse` as bytes, all of them within the type's range: int8 in the low bits of 1.5 * 2^23 + q, whose addition rounds to
// nearest even (the product with a power of two is exact)
template <bool E4M3>
__device__ __forceinline__ uint2 to_bytes(const float (&f)[8], float inverse) {
    uint32_t r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float* const g = f + 4 * h;
        if (E4M3) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(g[0] * inverse, g[1] * inverse), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(g[2] * inverse, g[3] * inverse), __NV_SATFINITE, __NV_E4M3);
            r[h] = lo | hi << 16;
        } else {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(fmaf(g[j], inverse, 12582912.f));
            r[h] = prmt(prmt(b[0], b[1], 0x0040), prmt(b[2], b[3], 0x0040), 0x5410);
        }
    }
    return make_uint2(r[0], r[1]);
}
// the same of 8 packed 16-bit values, some of them infinite or NaN
template <bool E4M3, bool BF16>
__device__ __noinline__ uint2 to_bytes_any(uint4 w, float inverse) {
    float f[8];
    unpack8<BF16>(w, f);
    uint32_t r[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j >> 2] |= to_byte<E4M3>(f[j] * inverse) << (8 * (j & 3));
    return make_uint2(r[0], r[1]);
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

// A warp takes one head's keys or values (2 * head + which) of the runs that begin in a window of `window` tokens (window <= 16), of every
// gridDim.y-th of them; neighbouring blocks take the heads of the same tokens, which lie side by side in memory.  A run: neighbouring tokens with ascending slots of one page; it ends with the page, so it has at most 128 tokens.
template <bool E4M3, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 4) cache_write_kernel(const CacheView c, const RowsView k, const RowsView v, int tokens,
                                                                  const int* slots, int window) {
    const int lane = threadIdx.x & 31;
    const int groups = (2 * c.heads + kWarps - 1) / kWarps, block = (int)(blockIdx.x / groups), unit = (int)(blockIdx.x - block * groups) * kWarps + (threadIdx.x >> 5), head = unit >> 1, which = unit & 1;
    if (head >= c.heads) return;
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int page = 1 << c.page_shift, lanes_per_row = c.dim >> 3, rows_per_step = 32 / lanes_per_row;
    const int row = lane / lanes_per_row, col = (lane % lanes_per_row) * 8;
    const uint16_t* x = (const uint16_t*)(which ? v.p : k.p) + head * (which ? v.head : k.head) + col;
    const long long x_token = which ? v.token : k.token;

    const int t0 = block * window;
    // lane i: the slot of token t0 - 1 + i, and whether it goes on with the run of the one before
    const int t = t0 - 1 + lane;
    const int slot = t >= 0 && t < tokens ? slots[t] : -1;
    const int before = __shfl_up_sync(kAll, slot, 1);
    const bool goes_on = lane > 0 && before >= 0 && slot == before + 1 && (slot & (page - 1)) != 0;
    const bool begins = lane > 0 && lane <= window && slot >= 0 && (slot >> c.page_shift) < c.pages && !goes_on;
    const uint32_t on = __ballot_sync(kAll, goes_on);
    int turn = 0;
    for (uint32_t starts = __ballot_sync(kAll, begins); starts; starts &= starts - 1) {
        if (turn++ % (int)gridDim.y != (int)blockIdx.y) continue;
        const int from = __ffs(starts) - 1, run = t0 - 1 + from;
        const int first_slot = __shfl_sync(kAll, slot, from);
        const int id = first_slot >> c.page_shift, place = first_slot & (page - 1);
        // its length: up to the first lane that does not go on; beyond the 32 lanes it is looked for
        const uint32_t stop = ~on & (from == 31 ? 0u : ~0u << (from + 1));
        int n = stop ? __ffs(stop) - 1 - from : 32 - from;
        while (!stop && n < page - place) {
            const int i = n + lane;
            const bool more = i < page - place && run + i < tokens && slots[run + i] == first_slot + i;
            const uint32_t end = __ballot_sync(kAll, !more);
            if (end) {
                n += __ffs(end) - 1;
                break;
            }
            n += 32;
        }
        // the lane's part of kHeld rows at a time; a run that fits (a page of 16 tokens does) is read once
        const uint16_t* rows = x + (long long)run * x_token;
        uint4 w[kHeld];
        const auto fetch = [&](int i0) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const int r = i0 + i * rows_per_step + row;
                w[i] = make_uint4(0, 0, 0, 0);
                if (r < n) w[i] = *reinterpret_cast<const uint4*>(rows + r * x_token);
            }
        };
        const int chunk = kHeld * rows_per_step;
        // magnitudes of either 16-bit type are ordered as their bits are, infinities and NaN on top
        uint32_t most = 0;
        for (int i0 = 0; i0 < n; i0 += chunk) {
            fetch(i0);
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                most = __vmaxu2(most, __vmaxu2(__vmaxu2(w[i].x & 0x7FFF7FFFu, w[i].y & 0x7FFF7FFFu), __vmaxu2(w[i].z & 0x7FFF7FFFu, w[i].w & 0x7FFF7FFFu)));
        }
        most = __reduce_max_sync(kAll, max(most & 0xFFFFu, most >> 16));
        const bool finite = most < (BF16 ? 0x7F80u : 0x7C00u);
        float a = BF16 ? __uint_as_float(most << 16) : __half2float(__ushort_as_half((unsigned short)most));
        if (!finite) {                                                   // the largest of the others
            a = 0.f;
            for (int i0 = 0; i0 < n; i0 += chunk) {
                if (n > chunk) fetch(i0);
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    float f[8];
                    unpack8<BF16>(w[i], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) a = fabsf(f[j]) <= 3.4e38f ? fmaxf(a, fabsf(f[j])) : a;
                }
            }
#pragma unroll
            for (int d = 16; d; d /= 2) a = fmaxf(a, __shfl_xor_sync(kAll, a, d));
        }
        float* const scale = reinterpret_cast<float*>(c.scales + (long long)id * c.heads + head) + which;
        const float old = place ? *scale : 0.f;
        const float s = fmaxf(old, scale_for<E4M3>(a));
        uint8_t* const held = (which ? c.v : c.k) + id * (which ? c.v_page : c.k_page) + head * (which ? c.v_head : c.k_head);
        const long long held_token = which ? c.v_token : c.k_token;
        if (s > old && place > 0) {
            const float ratio = old / s;              // (0 where the scale was: bytes of infinities beside zeros go on standing for 0)
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
        for (int i0 = 0; i0 < n; i0 += chunk) {
            if (n > chunk) fetch(i0);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i0 + i * rows_per_step >= n) break;
                const int r = i0 + i * rows_per_step + row;
                uint2 q;
                if (finite) {
                    float f[8];
                    unpack8<BF16>(w[i], f);
                    q = to_bytes<E4M3>(f, inverse);
                } else {
                    q = to_bytes_any<E4M3, BF16>(w[i], inverse);
                }
                if (r < n) *reinterpret_cast<uint2*>(held + (place + r) * held_token + col) = q;
            }
        }
        __syncwarp();
        if (lane == 0) *scale = s;
    }
}

// A block takes a token: its threads take 8 values each, of all heads' keys and then values, several of them in flight.
template <bool E4M3, bool BF16>
__global__ void __launch_bounds__(256) cache_read_kernel(const CacheView c, uint4* k_out, uint4* v_out, const int* slots) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    constexpr int kAtOnce = 4;
    const int shift = c.dim == 128 ? 4 : 3, per_which = c.heads << shift, units = 2 * per_which;
    const long long t = blockIdx.x;
    const int slot = slots[t], id = slot >> c.page_shift, place = slot & ((1 << c.page_shift) - 1);
    const bool there = slot >= 0 && id < c.pages;
    const uint8_t* const k = c.k + (there ? id * c.k_page + place * c.k_token : 0);
    const uint8_t* const v = c.v + (there ? id * c.v_page + place * c.v_token : 0);
    const float* const scales = reinterpret_cast<const float*>(c.scales + (there ? (long long)id * c.heads : 0));
    for (int u0 = threadIdx.x; u0 < units; u0 += kAtOnce * blockDim.x) {
        uint2 w[kAtOnce];
        float s[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int u = u0 + i * blockDim.x, which = u >= per_which, in = which ? u - per_which : u, head = in >> shift, col = (in & ((1 << shift) - 1)) * 8;
            w[i] = make_uint2(0, 0);
            s[i] = 0.f;
            if (there && u < units) {
                w[i] = *reinterpret_cast<const uint2*>((which ? v + head * c.v_head : k + head * c.k_head) + col);
                s[i] = scales[2 * head + which];
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int u = u0 + i * blockDim.x, which = u >= per_which;
            if (u >= units) break;
            const uint32_t b[2] = {w[i].x, w[i].y};
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = b[j >> 1] >> (16 * (j & 1));
                r[j] = there ? pack2<BF16>(from_byte<E4M3>(two & 0xFFu) * s[i], from_byte<E4M3>(two >> 8 & 0xFFu) * s[i]) : 0;
            }
            (which ? v_out - per_which : k_out)[t * per_which + u] = make_uint4(r[0], r[1], r[2], r[3]);
        }
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
    const long long blocks = (long long)((tokens + window - 1) / window) * ((2 * c.heads + kWarps - 1) / kWarps);
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)blocks, window > 1 ? 2 : 1, 1);
    const auto kernel = e4m3 ? (bf16 ? cache_write_kernel<true, true> : cache_write_kernel<true, false>)
                             : (bf16 ? cache_write_kernel<false, true> : cache_write_kernel<false, false>);
    return launch(kernel, grid, kWarps * 32, stream, c, k, v, tokens, slots, window);
}

cudaError_t cache_read_launch(const CacheView& c, bool e4m3, void* k_out, void* v_out, bool bf16, int tokens, const int* slots,
                              cudaStream_t stream) {
    // four units a thread, a warp to a full block
    const int threads = std::min(256, std::max(32, (2 * c.heads * (c.dim >> 3) / 4 + 31) / 32 * 32));
    const auto kernel = e4m3 ? (bf16 ? cache_read_kernel<true, true> : cache_read_kernel<true, false>)
                             : (bf16 ? cache_read_kernel<false, true> : cache_read_kernel<false, false>);
    return launch(kernel, dim3((unsigned)tokens, 1, 1), threads, stream, c, (uint4*)k_out, (uint4*)v_out, slots);
}

}  // namespace i4mm
