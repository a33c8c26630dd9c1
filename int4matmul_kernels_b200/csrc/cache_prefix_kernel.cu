// Attention of all rows that read a shared prefix over that prefix (the first half of i4mm_cache_attention_shared).
//
//   m = max_j s_j,  total = sum_j 2^(s_j - m),  sums = sum_j 2^(s_j - m) v_j,  s_j = log2(e) * scale * q . k_j, over the prefix's tokens that the row sees
// Simplest form: a warp for a row and head, a token to a lane.
#include "cache_attention.cuh"
#include "cache_bytes.cuh"

namespace i4mm {
namespace {

template <bool E4M3, bool BF16, int D>
__global__ void __launch_bounds__(256) cache_prefix_kernel(const AttentionParams p) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const CacheView& c = p.cache;
    const int page_mask = (1 << c.page_shift) - 1;
    const long long units = (long long)min(max(p.prefix_starts[p.requests], 0), p.prefix_listed) * p.q_heads;
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long long)gridDim.x * 8) {
        const int entry = (int)(u / p.q_heads), h = (int)(u - (long long)entry * p.q_heads), head = h / p.group, t = p.prefix_rows[entry];
        if (t < 0 || t >= p.tokens) continue;
        const auto owner = [&](const int* sums, int x) {
            int lo = 0, hi = p.requests - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (sums[mid] <= x) lo = mid;
                else hi = mid - 1;
            }
            return lo;
        };
        const int place = owner(p.prefix_starts, entry), b = p.cu_lens ? owner(p.cu_lens, t) : t;
        const int length = min(p.seq_lens[place], p.table_width << c.page_shift);
        const long long position = (long long)p.seq_lens[place] + p.seq_lens[b] - (p.cu_lens ? p.cu_lens[b + 1] : t + 1) + t;
        const int lo = p.window ? (int)min(max(position - p.window + 1, 0ll), (long long)max(length, 0)) : 0;
        const uint16_t* const q = static_cast<const uint16_t*>(p.q.p) + t * p.q.token + h * p.q.head;
        float m = -INFINITY, total = 0.f, o[D / 32] = {};
        for (int base = lo; base < length; base += 32) {
            const int j = base + lane;
            const int id = j < length ? p.table[place * p.table_stride + (j >> c.page_shift)] : -1;
            const bool there = id >= 0 && id < c.pages;
            float s = -INFINITY, v_scale = 0.f;
            if (there) {
                const uint8_t* const k = c.k + id * c.k_page + head * c.k_head + (j & page_mask) * c.k_token;
                const float2 scales = c.scales[(long long)id * c.heads + head];
                float dot = 0.f;
                for (int d = 0; d < D; d += 8) {
                    float f[8];
                    unpack8<BF16>(*reinterpret_cast<const uint4*>(q + d), f);
                    for (int i = 0; i < 8; ++i) dot = fmaf(f[i], from_byte<E4M3>(k[d + i]), dot);
                }
                s = dot * scales.x * (p.scale * kLog2e);
                v_scale = scales.y;
            }
            float top = s;
            for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
            const float next = fmaxf(m, top), from = next == -INFINITY ? 0.f : next, keep = m == -INFINITY ? 0.f : exp2f(m - next), e = exp2f(s - from);
            m = next;
            float sum = e;
            for (int d = 16; d; d /= 2) sum += __shfl_xor_sync(kAll, sum, d);
            total = total * keep + sum;
            for (int i = 0; i < D / 32; ++i) o[i] *= keep;
            for (int l = 0; l < 32; ++l) {
                const int at = __shfl_sync(kAll, there ? id : -1, l);
                const float w = __shfl_sync(kAll, e * v_scale, l);
                if (at < 0) continue;
                const uint8_t* const v = c.v + at * c.v_page + head * c.v_head + ((base + l) & page_mask) * c.v_token + lane * (D / 32);
                for (int i = 0; i < D / 32; ++i) o[i] = fmaf(w, from_byte<E4M3>(v[i]), o[i]);
            }
        }
        const long long row = (long long)t * p.q_heads + h;
        if (lane == 0) p.prefix_total[row] = make_float2(m, total);
        for (int i = 0; i < D / 32; ++i) p.prefix_sums[row * D + lane * (D / 32) + i] = o[i];
    }
}

}  // namespace

cudaError_t cache_prefix_launch(const AttentionParams& p, bool e4m3, bool bf16, cudaStream_t stream) {
    const auto by_dim = [&](auto e, auto h) {
        constexpr bool E = decltype(e)::value, H = decltype(h)::value;
        const auto kernel = p.cache.dim == 128 ? cache_prefix_kernel<E, H, 128> : cache_prefix_kernel<E, H, 64>;
        return launch_overlapping(kernel, dim3(148 * 8), 256, stream, p);
    };
    const auto by_type = [&](auto e) { return bf16 ? by_dim(e, std::true_type{}) : by_dim(e, std::false_type{}); };
    return e4m3 ? by_type(std::true_type{}) : by_type(std::false_type{});
}

}  // namespace i4mm
