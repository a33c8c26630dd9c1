// Attention over the paged 8-bit cache (i4mm_cache_attention).
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j,  m = max_j s_j, over the tokens j that the row sees
// in one pass with the running maximum and sum.  One warp per row and head; every lane holds its share of the head's values.
#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr int kWarps = 8;

template <bool BF16>
__device__ __forceinline__ float load16(const void* p, long long i) {
    return BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : __half2float(static_cast<const __half*>(p)[i]);
}

template <bool E4M3>
__device__ __forceinline__ float value(uint8_t b) {
    if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
    return (float)(signed char)b;
}

// the request that packed row t belongs to, or -1
__device__ __forceinline__ int request_of(const AttentionParams& p, int t) {
    if (!p.cu_lens) return t < p.requests ? t : -1;
    if (p.requests == 0 || t >= p.cu_lens[p.requests]) return -1;
    int lo = 0, hi = p.requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.cu_lens[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(kWarps * 32) cache_attention_kernel(const AttentionParams p) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const long long unit = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int t = (int)(unit / p.q_heads), h = (int)(unit % p.q_heads);
    if (t >= p.tokens) return;
    const CacheView& c = p.cache;
    const int kv = h / p.group, b = request_of(p, t);
    float q[N], o[N], m = -INFINITY, sum = 0.f;
    for (int i = 0; i < N; ++i) {
        q[i] = load16<BF16>(p.q.p, t * p.q.token + h * p.q.head + lane * N + i) * p.scale;
        o[i] = 0.f;
    }
    if (b >= 0) {
        const int seq = min(p.seq_lens[b], p.table_width << c.page_shift);
        const int last = p.cu_lens ? p.seq_lens[b] - (p.cu_lens[b + 1] - t) : p.seq_lens[b] - 1;     // the row's position
        for (int j = p.window ? max(0, last - p.window + 1) : 0; j <= last && j < seq; ++j) {
            const int id = p.table[b * p.table_stride + (j >> c.page_shift)], place = j & ((1 << c.page_shift) - 1);
            if (id < 0 || id >= c.pages) continue;
            const uint8_t* k = c.k + id * c.k_page + kv * c.k_head + place * c.k_token + lane * N;
            const uint8_t* v = c.v + id * c.v_page + kv * c.v_head + place * c.v_token + lane * N;
            const float2 scale = c.scales[(long long)id * c.heads + kv];
            float s = 0.f;
            for (int i = 0; i < N; ++i) s += q[i] * value<E4M3>(k[i]);
            for (int d = 16; d; d /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
            s *= scale.x;
            const float next = fmaxf(m, s), keep = m == -INFINITY ? 0.f : __expf(m - next), w = __expf(s - next);
            sum = sum * keep + w;
            for (int i = 0; i < N; ++i) o[i] = o[i] * keep + w * scale.y * value<E4M3>(v[i]);
            m = next;
        }
    }
    const float inverse = sum > 0.f ? 1.f / sum : 0.f;
    for (int i = 0; i < N; ++i) {
        const long long at = ((long long)t * p.q_heads + h) * D + lane * N + i;
        if (BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16(o[i] * inverse);
        else static_cast<__half*>(p.out)[at] = __float2half(o[i] * inverse);
    }
}

}  // namespace

size_t cache_attention_workspace() { return 16; }

cudaError_t cache_attention_launch(const AttentionParams& p, bool e4m3, bool bf16, int, cudaStream_t stream) {
    const auto pick = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return e4m3 ? (bf16 ? cache_attention_kernel<true, true, D> : cache_attention_kernel<true, false, D>)
                    : (bf16 ? cache_attention_kernel<false, true, D> : cache_attention_kernel<false, false, D>);
    };
    const auto kernel = p.cache.dim == 128 ? pick(std::integral_constant<int, 128>{}) : pick(std::integral_constant<int, 64>{});
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)(((long long)p.tokens * p.q_heads + kWarps - 1) / kWarps), 1, 1);
    cfg.blockDim = dim3(kWarps * 32, 1, 1);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace i4mm
