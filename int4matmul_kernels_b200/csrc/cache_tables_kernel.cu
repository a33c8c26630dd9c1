// Tables that a step is given once and all its layers use: angles of positions (i4mm_cache_angles), and which rows read which shared
// prefix (i4mm_cache_share).
#include <algorithm>

#include "cache_bytes.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr uint32_t kAll = 0xFFFFFFFFu;

// (cos, sin) of position * freq.  The product of two fp32-sized numbers in fp64 is exact up to positions of 2^29, and so good to 2^-52 above; whole
// turns are taken off in fp64, which leaves the fp32 functions an argument of at most one turn: positions of a million are as good as those
// below ten, and from 2^28 radians on the fp64 roundings show (2^-51 of the angle).  Two angles a thread, 16 bytes a store.  What bounds it: instructions. Each
// 16 bytes cost a 64-bit division, a load and conversion of the position, conversions of two frequencies, fp64 products and the fp32 functions: 36000
// tokens of 64 pairs 7.3 us (18.4 MB, 2.5 TB/s; the stores alone would be 2.8), 64 tokens 1.6.
__global__ void __launch_bounds__(256) cache_angles_kernel(float4* out, const int* positions, const float* freqs, long long twos, int per_token) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    constexpr double kTurns = 0.15915494309189533577;                         // 1 / (2 pi)
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < twos; i += (long long)gridDim.x * blockDim.x) {
        const long long t = i / per_token;
        const int j = (int)(i - t * per_token), position = positions[t];
        const float2 f = *reinterpret_cast<const float2*>(freqs + 2 * j);
        float4 v = make_float4(1.f, 0.f, 1.f, 0.f);                           // of padding
        if (position >= 0) {
            const auto turn = [&](float freq, float& c, float& s) {
                const double turns = (double)position * (double)freq * kTurns;
                sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
            };
            turn(f.x, v.x, v.y);
            turn(f.y, v.z, v.w);
        }
        out[i] = v;
    }
}

// Requests b with their effective prefix of(b): -1 unless it is another place that holds tokens, as b does itself.
//   rows(b) = packed rows of b at positions >= 0,  starts(p) = sum of rows(b) over the b with of(b) < p,
//   offset(b) = starts(of(b)) + sum of rows(b') over the b' < b with of(b') = of(b)
// and row i of b is entry offset(b) + i of the list.  Every block takes the sums itself (they are a few loads per thread) and keeps its own part
// of the rows.  The sums over equal prefixes are taken in order by one warp, 32 requests at a time, so that the list's order is always the same.
// What bounds it: the launch, and a chain of loads, sums, that one warp's pass and a search for each token (4 requests 3.0 us, 500 requests 8.5).
constexpr int kShareThreads = 512;

__global__ void __launch_bounds__(kShareThreads) cache_share_kernel(const ShareParams p) {
    extern __shared__ int shared[];
    __shared__ int warp_sums[kShareThreads / 32];
    const int n = p.requests, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int *s_starts = shared, *s_offset = shared + n + 1, *s_cu = shared + 2 * n + 1;
    short* const s_of = reinterpret_cast<short*>(shared + 3 * n + 2);         // (there are 16384 places at most)
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    // first row that counts, and their number
    const auto rows_of = [&](int seq, int cu, int next, int& from) {
        const long long lo = cu, hi = next, skip = max(hi - lo - max(seq, 0), 0ll);
        from = (int)min(max(lo + skip, 0ll), (long long)p.max_tokens);
        return (int)max(min(hi, (long long)p.max_tokens) - from, 0ll);
    };
    for (int b = threadIdx.x; b <= n; b += kShareThreads) s_starts[b] = 0;
    __syncthreads();
    for (int b = threadIdx.x; b <= n; b += kShareThreads) {
        const int cu = p.cu_lens[b];
        s_cu[b] = cu;
        if (b == n) break;
        const int seq = p.seq_lens[b], next = p.cu_lens[b + 1];
        int of = p.prefix_of[b];
        if (of < 0 || of >= n || of == b || seq <= 0 || p.seq_lens[of] <= 0) of = -1;
        int from;
        const int count = rows_of(seq, cu, next, from);
        s_of[b] = (short)of;
        s_offset[b] = count;
        if (of >= 0 && count > 0) atomicAdd(&s_starts[of], count);
    }
    __syncthreads();
    // s_starts: numbers of rows -> exclusive sums
    int carry = 0;
    for (int base = 0; base <= n; base += kShareThreads) {
        const int b = base + threadIdx.x, own = b < n ? s_starts[b] : 0;
        int v = own;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int o = __shfl_up_sync(kAll, v, d);
            if (lane >= d) v += o;
        }
        if (lane == 31) warp_sums[warp] = v;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < kShareThreads / 32; ++w) {
            if (w < warp) before += warp_sums[w];
            carry += warp_sums[w];
        }
        if (b <= n) s_starts[b] = before + v - own;
        __syncthreads();
    }
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= n; b += kShareThreads) p.starts[b] = s_starts[b];
    __syncthreads();
    // s_offset: numbers of rows -> where they begin; s_starts[p] moves on to the end of what has been given out of p's
    if (warp == 0)
        for (int base = 0; base < n; base += 32) {
            const int b = base + lane, of = b < n ? s_of[b] : -1, count = b < n ? s_offset[b] : 0;
            const uint32_t peers = __match_any_sync(kAll, of);
            // counts of the peers in lower lanes, bit by bit
            const uint32_t lower = peers & ((1u << lane) - 1), bits = __reduce_or_sync(kAll, (uint32_t)count);
            int before = 0;
            for (int i = 0; bits >> i; ++i) before += __popc(__ballot_sync(kAll, count >> i & 1) & lower) << i;
            const int at = of >= 0 ? s_starts[of] : 0;
            __syncwarp();
            if (of >= 0 && 31 - __clz(peers) == lane) s_starts[of] = at + before + count;
            if (b < n) s_offset[b] = at + before;
            __syncwarp();
        }
    __syncthreads();
    const int listed = s_starts[n], first = blockIdx.x * kShareThreads + threadIdx.x, step = gridDim.x * kShareThreads;
    for (int b = first; b < n; b += step) p.effective[b] = s_of[b];
    for (int t = first; t < p.max_tokens; t += step) {
        if (t >= listed) p.rows[t] = -1;
        int position = -1;
        if (n > 0 && t < s_cu[n] && t >= s_cu[0]) {
            int lo = 0, hi = n - 1;                   // the b with cu_lens[b] <= t < cu_lens[b + 1]
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_cu[mid] <= t) lo = mid;
                else hi = mid - 1;
            }
            const int of = s_of[lo], seq = p.seq_lens[lo];
            int from;
            const int count = rows_of(seq, s_cu[lo], s_cu[lo + 1], from);
            const long long pos = (long long)seq - s_cu[lo + 1] + t;
            if (t >= from && t < from + count && pos >= 0) {
                position = (int)min(pos + (of >= 0 ? p.seq_lens[of] : 0), 0x7FFFFFFFll);
                const long long at = (long long)s_offset[lo] + (t - from);
                if (of >= 0 && at >= 0 && at < p.max_tokens) p.rows[at] = t;
            }
        }
        p.positions[t] = position;
    }
}

}  // namespace

cudaError_t cache_angles_launch(void* out, const int* positions, const float* freqs, int tokens, int pairs, cudaStream_t stream) {
    const long long twos = (long long)tokens * (pairs / 2);
    const long long blocks = std::min<long long>((twos + 255) / 256, 148 * 8);
    return launch_overlapping(cache_angles_kernel, dim3((unsigned)blocks), 256, stream, (float4*)out, positions, freqs, twos, pairs / 2);
}

cudaError_t cache_share_launch(const ShareParams& p, cudaStream_t stream) {
    const size_t smem = (3 * (size_t)p.requests + 2) * sizeof(int) + (size_t)p.requests * sizeof(short);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(cache_share_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    const int blocks = (std::max(p.max_tokens, p.requests + 1) + kShareThreads - 1) / kShareThreads;
    cfg.gridDim = dim3((unsigned)std::min(blocks, 148), 1, 1);
    cfg.blockDim = dim3(kShareThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, cache_share_kernel, p);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace i4mm
