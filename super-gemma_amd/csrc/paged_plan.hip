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
// loads (64 requests: 4.9 us, of which an empty kernel takes 2.4).  One workgroup
// scans both sums in LDS and pops the pages: the thread of a page (or of a row)
// finds its request by bisection in the LDS sums.  It fills the slot map too up to
// four rows a thread; a longer one goes to a second launch over the whole GPU
// (64 rows: 9.0 us in one launch, 11.5 in two; with a release before them and the
// copies that it works on, 4060 rows: 30.1 and 31.6; 8100: 27.9 and 28.8; 32000: 62 and 34).
#include "paged.h"

namespace sgq {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 4 * kPlanThreads;

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

__device__ __forceinline__ int clamp_new(int n) { return min(max(n, 0), 1 << 22); }

// Rows first, first + step, ... of the slot map; how many of them got no slot.
template <typename Cached>
__device__ __forceinline__ int fill_rows(const PagedPlan &p, const int *cu_s, int n_rows, int first,
                                         int step, Cached cached) {
    int lost = 0;
    for (int r = first; r < p.n_tokens; r += step) {
        int slot = -1;
        if (r < n_rows) {
            const int s = find_owner(cu_s, p.n_seqs, r);
            const long long pos = (long long)cached(s) + (r - cu_s[s]);
            const long long e = pos >> p.page_log2;
            const int page = e < p.max_pages ? p.tables[(size_t)s * p.max_pages + e] : -1;
            if ((unsigned)page < (unsigned)p.n_pages)
                slot = (page << p.page_log2) + (int)(pos & ((1 << p.page_log2) - 1));
            else
                lost++;
        }
        p.slots[r] = slot;
    }
    return lost;
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
            n = min(clamp_new(p.add[s]), 0x7fffffff - c);  // c + n and, up to 2^22 rows, cu are exact
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
    for (uint32_t u = tid; u < (uint32_t)n_new; u += kPlanThreads) {  // n_new < 2^31
        const int i = (int)u, s = find_owner(pg_s, p.n_seqs, i);
        const int have = (int)(((long long)cached_s[s] + P - 1) >> p.page_log2);
        const int at = n_free - 1 - i;
        p.tables[(size_t)s * p.max_pages + have + (i - pg_s[s])] = at >= 0 ? p.free_list[at] : -1;
    }
    __syncthreads();
    if (tid == 0) *p.n_free_out = max(n_free - n_new, 0);
    const int over = max(n_rows - p.n_tokens, 0);  // rows that the map does not hold
    if (p.n_tokens > kPlanRows) {
        if (tid == 0) *p.missing = over;  // the next launch adds to it
        return;
    }
    const int lost = fill_rows(p, cu_s, n_rows, tid, kPlanThreads, [&](int s) { return cached_s[s]; });
    if (lost) atomicAdd(&missing_s, lost);
    __syncthreads();
    if (tid == 0) *p.missing = missing_s + over;
}

// The slot map of many rows; kv_lens and cu are the scan's.
constexpr int kRowsThreads = 256;
__global__ __launch_bounds__(kRowsThreads) void paged_plan_rows_kernel(PagedPlan p) {
    __shared__ int cu_s[kPagedMaxSeqs + 1];
    for (int s = threadIdx.x; s <= p.n_seqs; s += kRowsThreads) cu_s[s] = p.cu[s];
    __syncthreads();
    int lost = fill_rows(p, cu_s, cu_s[p.n_seqs], blockIdx.x * kRowsThreads + threadIdx.x,
                         gridDim.x * kRowsThreads,
                         [&](int s) { return p.kv_lens[s] - (cu_s[s + 1] - cu_s[s]); });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lost += __shfl_xor(lost, d);
    if (lost && (threadIdx.x & 63) == 0) atomicAdd(p.missing, lost);  // whole numbers: any order
}

// Pages go back in request order, a request's pages in table order.  The finished
// requests are listed first, and a wave writes where its requests' entries are:
// what follows is bound by chains of LDS reads and loads.  1024 requests, 128 of them
// finished with 64 pages each: 11.6 us (a bisection per page, and counts summed by
// every thread: 18).
__global__ __launch_bounds__(kPlanThreads) void paged_release_kernel(PagedRelease p) {
    __shared__ int pg_s[kPagedMaxSeqs + 1];             // a finished request's first page
    __shared__ unsigned short seq_s[kPagedMaxSeqs];
    __shared__ long long wave_s[kPlanThreads / 64];
    const int P = 1 << p.page_log2, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_free = min(max(*p.n_free, 0), p.n_pages);
    constexpr int kCount = 40;  // a sum holds the pages below this bit, the requests from it on
    long long sum0 = 0;
    for (int b = 0; b < p.n_seqs; b += kPlanThreads) {
        const int s = b + tid;
        bool done = false;
        long long held = 0;
        if (s < p.n_seqs) {
            const long long h = ((long long)max(p.kv_lens[s], 0) + P - 1) >> p.page_log2;
            done = p.done[s] != 0;
            if (done) held = h < p.max_pages ? h : p.max_pages;
        }
        long long all;
        const long long mine = held | (long long)done << kCount;
        const long long before = sum0 + block_scan<kPlanThreads>(mine, wave_s, &all) - mine;
        if (done) {
            const int at = (int)(before >> kCount);
            seq_s[at] = (unsigned short)s;
            pg_s[at] = (int)(before & ((1ll << kCount) - 1));  // below 2^31, as the table's entries
        }
        sum0 += all;
    }
    const int n_held = (int)(sum0 & ((1ll << kCount) - 1)), n_done = (int)(sum0 >> kCount);
    if (tid == 0) pg_s[n_done] = n_held;
    __syncthreads();
    // entries outside the pool are dropped: the pushed ones are counted in order,
    // 8 rounds of a thread per page at a time
    constexpr int kRounds = 8, kWaves = kPlanThreads / 64;
    static_assert(kRounds * kWaves == 128, "two a lane");
    __shared__ int count_s[kRounds * kWaves];
    __shared__ int entry_s[kRounds * kPlanThreads];  // of these rounds' pages, in the tables
    int top = n_free;
    for (uint32_t b = 0; b < (uint32_t)n_held; b += kRounds * kPlanThreads) {  // n_held < 2^31
        int page[kRounds];
        uint64_t in[kRounds];
        const uint32_t end = min(b + kRounds * kPlanThreads, (uint32_t)n_held);
        for (int d = wave; d < n_done; d += kWaves) {
            const uint32_t lo = max((uint32_t)pg_s[d], b), hi = min((uint32_t)pg_s[d + 1], end);
            const uint32_t first = (uint32_t)(seq_s[d] * p.max_pages) - (uint32_t)pg_s[d];  // wraps, and back
            for (uint32_t i = lo + lane; i < hi; i += 64) entry_s[i - b] = (int)(first + i);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kRounds; k++) {
            const int at = k * kPlanThreads + tid;
            page[k] = b + at < end ? p.tables[entry_s[at]] : -1;
        }
#pragma unroll
        for (int k = 0; k < kRounds; k++) in[k] = __ballot((unsigned)page[k] < (unsigned)p.n_pages);
        __syncthreads();  // count_s of the last rounds has been read
        if (lane < kRounds) {
            uint64_t mine = in[0];
#pragma unroll
            for (int k = 1; k < kRounds; k++) mine = lane == k ? in[k] : mine;
            count_s[lane * kWaves + wave] = __popcll(mine);
        }
        __syncthreads();
        // sums over the 128 counts, two a lane
        const int c0 = count_s[lane], c1 = count_s[64 + lane];
        int s0 = c0, s1 = c1;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o0 = __shfl_up(s0, d), o1 = __shfl_up(s1, d);
            s0 += lane >= d ? o0 : 0;
            s1 += lane >= d ? o1 : 0;
        }
        const int half = __builtin_amdgcn_readlane(s0, 63);
#pragma unroll
        for (int k = 0; k < kRounds; k++) {
            const int before = k < kRounds / 2 ? __builtin_amdgcn_readlane(s0 - c0, k * kWaves + wave)
                                               : half + __builtin_amdgcn_readlane(s1 - c1, k * kWaves - 64 + wave);
            const int to = top + before + __popcll(in[k] & ((1ull << lane) - 1));
            if (in[k] >> lane & 1 && to < p.n_pages) p.free_list[to] = page[k];
        }
        top = min(top + half + __builtin_amdgcn_readlane(s1, 63), p.n_pages);
    }
    __syncthreads();  // the tables have been read
    for (int d = wave; d < n_done; d += kWaves) {
        const int s = seq_s[d];
        if (lane == 0) p.kv_lens[s] = 0;
        int32_t *row = p.tables + (size_t)s * p.max_pages;
        for (int j = lane; j < p.max_pages; j += 64) row[j] = -1;
    }
    if (tid == 0) *p.n_free = top;
}

}  // namespace

int launch_paged_plan(hipStream_t st, const PagedPlan &p) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    SGQ_HIP(hipGetLastError());
    if (p.n_tokens > kPlanRows) {
        const int wgs = (p.n_tokens + kRowsThreads - 1) / kRowsThreads;
        hipLaunchKernelGGL(paged_plan_rows_kernel, dim3(wgs < 512 ? wgs : 512), dim3(kRowsThreads), 0,
                           st, p);
        SGQ_HIP(hipGetLastError());
    }
    return SGQ_OK;
}

int launch_paged_release(hipStream_t st, const PagedRelease &p) {
    hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

}  // namespace sgq
