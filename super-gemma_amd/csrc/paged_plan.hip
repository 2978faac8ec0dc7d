// Block tables and the slot map of a step, built on the GPU from the requests'
// lengths, and the return of finished requests' pages.
//
// With c_s tokens cached and n_s new ones, request s holds ceil(c_s/P) pages and
// needs ceil((c_s+n_s)/P).  The pages it lacks are popped from a stack of free
// pages in request order, the i-th pop being free_list[n_free-1-i], so the
// tables follow from the inputs alone.  Row cu_s + i of the packed step is
// position c_s + i, whose slot is table[s][pos/P]·P + pos%P.
//
// A few kilobytes: what counts is the launch and the chain of dependent
// loads.  One workgroup scans both sums in LDS and fills everything: the
// thread of a row (or of a popped page) finds its request by bisection in the
// LDS sums.
#include "paged.h"

namespace sgq {
namespace {

constexpr int kPlanThreads = 1024;

// Inclusive sums over the workgroup of one value a thread.
template <int NT>
__device__ __forceinline__ long long block_scan(long long v, long long *wave_s, long long *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();  // wave_s of the last call has been read
    if (lane == 63) wave_s[wave] = v;
    __syncthreads();
    long long base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        if (w < wave) base += wave_s[w];
        all += wave_s[w];
    }
    *total = all;
    return v + base;
}

// The largest s of 0..n-1 with sums[s] <= i (sums[0] = 0, ascending).
__device__ __forceinline__ int find_owner(const int *sums, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int clamp_len(long long v) {
    return v < 0 ? 0 : v > 0x7fffffff ? 0x7fffffff : (int)v;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlan p) {
    __shared__ int cu_s[kPagedMaxSeqs + 1];
    __shared__ int pg_s[kPagedMaxSeqs + 1];
    __shared__ int cached_s[kPagedMaxSeqs];
    __shared__ long long wave_s[kPlanThreads / 64];
    __shared__ int missing_s;
    const int P = 1 << p.page_log2, tid = threadIdx.x;
    const int n_free = min(max(*p.n_free, 0), p.n_pages);
    if (tid == 0) missing_s = 0;
    long long tok0 = 0, pg0 = 0;
    for (int b = 0; b < p.n_seqs; b += kPlanThreads) {
        const int s = b + tid;
        int c = 0, n = 0, more = 0;
        if (s < p.n_seqs) {
            c = max(p.cached[s], 0);
            n = max(p.add[s], 0);
            const long long cap = (long long)p.max_pages;
            long long have = ((long long)c + P - 1) >> p.page_log2;
            long long want = ((long long)c + n + P - 1) >> p.page_log2;
            have = have < cap ? have : cap;
            want = want < cap ? want : cap;
            more = (int)(want - have);
        }
        long long tok_all, pg_all;
        const long long tok = tok0 + block_scan<kPlanThreads>(n, wave_s, &tok_all);
        const long long pg = pg0 + block_scan<kPlanThreads>(more, wave_s, &pg_all);
        if (s < p.n_seqs) {
            cached_s[s] = c;
            cu_s[s] = clamp_len(tok - n);
            pg_s[s] = clamp_len(pg - more);
            p.cu[s] = cu_s[s];
            p.kv_lens[s] = clamp_len((long long)c + n);
        }
        tok0 += tok_all;
        pg0 += pg_all;
    }
    const int n_rows = clamp_len(tok0), n_new = clamp_len(pg0);
    if (tid == 0) {
        cu_s[p.n_seqs] = n_rows;
        pg_s[p.n_seqs] = n_new;
        p.cu[p.n_seqs] = n_rows;
    }
    __syncthreads();
    // the popped pages
    for (int i = tid; i < n_new; i += kPlanThreads) {
        const int s = find_owner(pg_s, p.n_seqs, i);
        const int have = (int)(((long long)cached_s[s] + P - 1) >> p.page_log2);
        const int at = n_free - 1 - i;
        p.tables[(size_t)s * p.max_pages + have + (i - pg_s[s])] = at >= 0 ? p.free_list[at] : -1;
    }
    __syncthreads();
    // the rows
    int lost = 0;
    for (int r = tid; r < p.n_tokens; r += kPlanThreads) {
        int slot = -1;
        if (r < n_rows) {
            const int s = find_owner(cu_s, p.n_seqs, r);
            const long long pos = (long long)cached_s[s] + (r - cu_s[s]);
            const long long e = pos >> p.page_log2;
            const int page = e < p.max_pages ? p.tables[(size_t)s * p.max_pages + e] : -1;
            if ((unsigned)page < (unsigned)p.n_pages)
                slot = (page << p.page_log2) + (int)(pos & (P - 1));
            else
                lost++;
        }
        p.slots[r] = slot;
    }
    if (lost) atomicAdd(&missing_s, lost);
    __syncthreads();
    if (tid == 0) {
        *p.missing = missing_s + max(n_rows - p.n_tokens, 0);
        *p.n_free_out = max(n_free - n_new, 0);
    }
}

// Pages go back in request order, a request's pages in table order.
__global__ __launch_bounds__(kPlanThreads) void paged_release_kernel(PagedRelease p) {
    __shared__ int pg_s[kPagedMaxSeqs + 1];
    __shared__ long long wave_s[kPlanThreads / 64];
    const int P = 1 << p.page_log2, tid = threadIdx.x;
    const int n_free = min(max(*p.n_free, 0), p.n_pages);
    long long pg0 = 0;
    for (int b = 0; b < p.n_seqs; b += kPlanThreads) {
        const int s = b + tid;
        int held = 0;
        if (s < p.n_seqs && p.done[s]) {
            const long long h = ((long long)max(p.kv_lens[s], 0) + P - 1) >> p.page_log2;
            held = (int)(h < p.max_pages ? h : p.max_pages);
        }
        long long all;
        const long long pg = pg0 + block_scan<kPlanThreads>(held, wave_s, &all);
        if (s < p.n_seqs) pg_s[s] = clamp_len(pg - held);
        pg0 += all;
    }
    const int n_held = clamp_len(pg0);
    if (tid == 0) pg_s[p.n_seqs] = n_held;
    __syncthreads();
    // entries outside the pool are dropped: the pushed ones are counted in order
    int top = n_free;
    for (int b = 0; b < n_held; b += kPlanThreads) {
        const int i = b + tid;
        int page = -1;
        if (i < n_held) {
            const int s = find_owner(pg_s, p.n_seqs, i);
            page = p.tables[(size_t)s * p.max_pages + (i - pg_s[s])];
        }
        const bool ok = (unsigned)page < (unsigned)p.n_pages;
        long long all;
        const long long at = top + block_scan<kPlanThreads>(ok, wave_s, &all) - 1;
        if (ok && at < p.n_pages) p.free_list[at] = page;
        top = (int)min((long long)p.n_pages, top + all);
    }
    __syncthreads();
    for (int s = 0; s < p.n_seqs; s++) {
        if (!p.done[s]) continue;
        for (int j = tid; j < p.max_pages; j += kPlanThreads)
            p.tables[(size_t)s * p.max_pages + j] = -1;
    }
    for (int s = tid; s < p.n_seqs; s += kPlanThreads)
        if (p.done[s]) p.kv_lens[s] = 0;
    if (tid == 0) *p.n_free = top;
}

}  // namespace

int launch_paged_plan(hipStream_t st, const PagedPlan &p) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

int launch_paged_release(hipStream_t st, const PagedRelease &p) {
    hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

}  // namespace sgq
