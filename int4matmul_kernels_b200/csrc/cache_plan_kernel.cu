// Block tables and slot maps of one step, from the requests' lengths (i4mm_cache_plan).
//
//   add(b)   = max(new(b), 0), after(b) = seq(b) + add(b)            (a request that ends: both 0)
//   freed(b) = ceil(seq(b) / P) if b ends, else 0;  need(b) = ceil(after(b) / P) - ceil(seq(b) / P), both within the table's row
//   stack    = free_pages[0 .. count), then the pages of the requests that end; the i-th new page is stack[top - 1 - i]
//   slot(t)  = table[b][pos / P] * P + pos % P for the packed token t of request b at position pos
// Everything follows from three prefix sums over the requests.  A few kilobytes go in and out, so what bounds it is the launch and one
// chain of dependent steps (lengths -> sums -> search -> table entry -> slot).  A grid that had to hand the sums from one block to the
// others would add a device-wide hand-shake to that chain; instead every block takes all the sums itself (they are a few loads per
// thread) and keeps its own part of the tokens and pages.  Nothing that a block reads is written by another one: entries of pages that
// the step begins are computed again from the stack wherever they are needed, and pushes lie above every entry that is popped by value.
// Measured: 4 us for 4 requests of one token, 7 us for 500 requests with 36000 new tokens (in a graph; a call from Python takes 7.5).
#include <algorithm>

#include "cache.cuh"
#include "common.cuh"
#include "ptx.cuh"

namespace i4mm {
namespace {

constexpr int kThreads = 512;

__device__ __forceinline__ int clamp_int(long long v) { return (int)min(v, (long long)0x7FFFFFFF); }

// the b with sums[b] <= x < sums[b + 1]; x < sums[n]
__device__ __forceinline__ int owner(const int* sums, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// s[0 .. n] = exclusive sums of three quantities per request; every thread of the block takes part
__device__ __forceinline__ void prefix_sums(const PlanParams& p, int* s_add, int* s_need, int* s_freed) {
    __shared__ long long warp_sums[3][kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int page = 1 << p.page_shift;
    long long carry[3] = {0, 0, 0};
    for (int base = 0; base < p.requests; base += kThreads) {
        const int b = base + threadIdx.x;
        long long v[3] = {0, 0, 0};
        if (b < p.requests) {
            const long long seq = max(p.seq_lens[b], 0), add = p.new_lens[b];
            const long long held = min((seq + page - 1) >> p.page_shift, (long long)p.table_width);
            if (add < 0) {
                v[2] = held;
            } else {
                v[0] = add;
                v[1] = min((seq + add + page - 1) >> p.page_shift, (long long)p.table_width) - held;
            }
        }
        long long own[3] = {v[0], v[1], v[2]};
#pragma unroll
        for (int d = 1; d < 32; d *= 2)
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const long long o = __shfl_up_sync(0xFFFFFFFFu, v[i], d);
                if (lane >= d) v[i] += o;
            }
        if (lane == 31)
#pragma unroll
            for (int i = 0; i < 3; ++i) warp_sums[i][warp] = v[i];
        __syncthreads();
        long long before[3], total[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            before[i] = carry[i];
            total[i] = carry[i];
            for (int w = 0; w < kThreads / 32; ++w) {
                if (w < warp) before[i] += warp_sums[i][w];
                total[i] += warp_sums[i][w];
            }
            carry[i] = total[i];
        }
        if (b < p.requests) {
            s_add[b] = clamp_int(before[0] + v[0] - own[0]);
            s_need[b] = clamp_int(before[1] + v[1] - own[1]);
            s_freed[b] = clamp_int(before[2] + v[2] - own[2]);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        s_add[p.requests] = clamp_int(carry[0]);
        s_need[p.requests] = clamp_int(carry[1]);
        s_freed[p.requests] = clamp_int(carry[2]);
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) cache_plan_kernel(const PlanParams p) {
    extern __shared__ int sums[];
    const int n = p.requests, page = 1 << p.page_shift;
    int *s_add = sums, *s_need = sums + n + 1, *s_freed = sums + 2 * (n + 1);
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    prefix_sums(p, s_add, s_need, s_freed);
    const int count = min(max(*p.free_count, 0), p.free_capacity), freed = s_freed[n], needed = s_need[n];
    const long long top = (long long)count + freed;

    // the page at place i of the stack, pushes included
    const auto at = [&](long long i) {
        if (i < 0) return -1;
        if (i < count) return p.free_pages[i];
        const int j = (int)(i - count), b = owner(s_freed, n, j);
        return p.table[b * p.table_stride + (j - s_freed[b])];
    };
    const int first = blockIdx.x * kThreads + threadIdx.x, step = gridDim.x * kThreads;
    for (int i = first; i < freed; i += step)
        if (count + (long long)i < p.free_capacity) p.free_pages[count + i] = at((long long)count + i);
    for (int i = first; i < needed; i += step) {
        const int b = owner(s_need, n, i);
        const int held = (int)(((long long)max(p.seq_lens[b], 0) + page - 1) >> p.page_shift);
        p.table[b * p.table_stride + held + (i - s_need[b])] = at(top - 1 - i);
    }
    for (int t = first; t < p.max_tokens; t += step) {
        int slot = -1, pos = -1, b = -1;
        if (t < s_add[n]) {
            b = owner(s_add, n, t);
            const int seq = max(p.seq_lens[b], 0);
            const long long place = (long long)seq + (t - s_add[b]);
            const long long j = place >> p.page_shift;
            pos = clamp_int(place);
            if (j < p.table_width) {
                const int held = (int)(((long long)seq + page - 1) >> p.page_shift);
                const int id = j < held ? p.table[b * p.table_stride + j] : at(top - 1 - ((long long)s_need[b] + (j - held)));
                if (id >= 0) slot = (id << p.page_shift) + (int)(place & (page - 1));
            }
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
        p.request_of[t] = b;
    }
    for (int b = first; b <= n; b += step) {
        p.cu_lens[b] = s_add[b];
        if (b < n) p.lens_after[b] = p.new_lens[b] < 0 ? 0 : clamp_int((long long)max(p.seq_lens[b], 0) + p.new_lens[b]);
    }
    if (blockIdx.x == 0) {
        // pages that the lengths ask for and that do not come: beyond the table's row, or the stack's bottom
        __shared__ unsigned long long beyond;
        if (threadIdx.x == 0) beyond = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int b = threadIdx.x; b < n; b += kThreads)
            if (p.new_lens[b] >= 0) {
                const long long seq = max(p.seq_lens[b], 0);
                const long long wanted = ((seq + p.new_lens[b] + page - 1) >> p.page_shift) - ((seq + page - 1) >> p.page_shift);
                mine += (unsigned long long)(wanted - (s_need[b + 1] - s_need[b]));
            }
        if (mine) atomicAdd(&beyond, mine);
        __syncthreads();
        if (threadIdx.x == 0) {
            const long long left = max(top - needed, 0ll), given = top - left;
            p.counts[0] = (int)min(left, (long long)p.free_capacity);
            p.counts[1] = clamp_int((long long)beyond + (needed - given));
        }
    }
}

}  // namespace

cudaError_t cache_plan_launch(const PlanParams& p, cudaStream_t stream) {
    const size_t smem = 3 * (size_t)(p.requests + 1) * sizeof(int);
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(cache_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    // one block per 512 tokens; the pages of a step are at most as many, unless a prompt's pages are freed (then each thread takes a few)
    const int blocks = (std::max(p.max_tokens, p.requests + 1) + kThreads - 1) / kThreads;
    cfg.gridDim = dim3((unsigned)std::min(blocks, 296), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, cache_plan_kernel, p);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace i4mm
