// How 16-bit values become the cache's bytes: what its writers and its reader share.
//
//   a = the largest finite |x| that a call adds to a page and head,  s = max(s_old, min { 2^e : a <= most * 2^e }),  q = round(x / s)
// All scales are powers of two, so x / s and q * s are exact and the only rounding is the one to the byte.
#pragma once

#include "cache.cuh"
#include "common.cuh"

namespace i4mm {

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

// The same bytes of 8 packed fp16 values that are all finite, two at a time, where `inverse` is a normal fp16 number.  int8: 1536 + x * inverse is rounded
// once, to whole numbers, and its low byte is q.  e4m3: the product is exact down to 2^-14, and what is below that is 0 either way.
template <bool E4M3>
__device__ __forceinline__ uint2 half_to_bytes(uint4 w, uint32_t inverse2) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (E4M3) {
            unsigned short two;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(two) : "r"(hmul2_u(u[i], inverse2)));
            r[i] = two;
        } else {
            r[i] = hfma2_u(u[i], inverse2, 0x66006600u);
        }
    }
    if (E4M3) return make_uint2(r[0] | r[1] << 16, r[2] | r[3] << 16);
    return make_uint2(prmt(r[0], r[1], 0x6420), prmt(r[2], r[3], 0x6420));
}
__device__ __forceinline__ bool normal_half(float power) { return power >= 6.103515625e-5f && power <= 32768.f; }

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

// A launch that may begin while the kernel before it ends: every kernel launched with it waits before it touches anything.
template <typename F, typename... Args>
inline cudaError_t launch_overlapping(F* kernel, dim3 grid, int threads, cudaStream_t stream, Args... args) {
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

}  // namespace i4mm
