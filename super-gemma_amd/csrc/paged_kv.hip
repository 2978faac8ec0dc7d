// Appending K and V rows to the paged 8-bit cache, and reading slots back.
//
// A run is a maximal sequence of consecutive rows that go to one page; the rows
// of a step's slot map form at most rows/P + 2·requests of them.  Per head, with
// d = max|x| / 127 over the run (one IEEE division):
//   the run holds the page's slot 0    the block begins anew, scale = d
//   else                               scale = max(old, d); when it grows, the
//                                      block's quants become rte(q·old/scale)
//   quants of the run's rows           rte(x/scale), 0 where scale is 0
// rte of the real quotient, ties to even: the fp32 product with the reciprocal
// gives the integer up to one, and the exact residual x - t·scale decides.
// A row with an infinity or a NaN makes the scale NaN, so that attention over
// the block is NaN too instead of quietly wrong.
#include "paged.h"

namespace sgq {
namespace {

constexpr int kAppThreads = 256;
constexpr uint32_t kInfBits = 0x7f800000u;

// rte((x + xe)/d) for d > 0, |x| <= 127.5·d and an xe below x's last place:
// t = rint(x·(1/d)) is off by at most one.  The residual x - t·d is a multiple of
// the smaller of both units in the last place and below 2·d, so the fma is
// exact, and so is its difference from ±d/2 where that is small enough for xe to
// matter.
__device__ __forceinline__ int quant_rte(float x, float xe, float d, float inv) {
    float t = rintf(x * inv);
    const float r = fmaf(-t, d, x), h = 0.5f * d;
    const float over = (r - h) + xe, under = (r + h) + xe;
    const bool odd = (int)t & 1;
    t += over > 0.f || (over == 0.f && odd) ? 1.f : 0.f;
    t -= under < 0.f || (under == 0.f && odd) ? 1.f : 0.f;
    return (int)fminf(fmaxf(t, -127.f), 127.f);
}

// 16 quants q as rte(q·old/d), old <= d: the product has up to 31 bits, its
// rounded value and the error of that go in.
__device__ __forceinline__ uint4 regrid(uint4 w, float old, float d, float inv) {
    uint32_t *p = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t o = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float q = (float)(int8_t)(p[i] >> (8 * j)), x = q * old;
            o |= ((uint32_t)quant_rte(x, fmaf(q, old, -x), d, inv) & 0xffu) << (8 * j);
        }
        p[i] = o;
    }
    return w;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Two consecutive activations starting at element 2j.
__device__ __forceinline__ float2 act_ld2(const float *p, size_t j) {
    return reinterpret_cast<const float2 *>(p)[j];
}
__device__ __forceinline__ float2 act_ld2(const uint16_t *p, size_t j) {
    const uint32_t w = reinterpret_cast<const uint32_t *>(p)[j];
    return make_float2(f16_bits_to_f32(w & 0xffffu), f16_bits_to_f32(w >> 16));
}

// One workgroup writes one run at a time for one head, K (y = 0) or V (y = 1):
// the runs that begin in its window of `window` rows.  Every wave finds the runs by
// itself (a load of 64 slots and ballots), the rows are read twice (the second
// time from the caches): once for the maximum, once to be rounded.
// K: a thread rounds 8 dims of a row.  V, stored by dim: a thread rounds 2 dims
// of 16 tokens, so a wave reads whole rows and stores 16 bytes a lane; a dword
// or byte at a time the stores alone took four times as long as the reads.
template <typename T, int HD>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(
    const T *__restrict__ k, uint64_t k_stride, const T *__restrict__ v, uint64_t v_stride,
    const int32_t *__restrict__ slots, int n_tokens, int window, PagedPages pg) {
    constexpr int U = HD / 8;    // 8-dim units of a row
    __shared__ int row_of[128];  // offset in the page -> row of the run, -1: none
    __shared__ uint32_t amax_s[kAppThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.x % pg.n_kv;
    const bool is_v = blockIdx.y != 0;
    const int lg = pg.page_log2, P = 1 << lg;
    const T *src = (is_v ? v : k) + (size_t)head * HD;
    const uint64_t stride = is_v ? v_stride : k_stride;
    const uint32_t n_slots = (uint32_t)pg.n_pages << lg;
    const auto slot_of = [&](int r) { return r >= 0 && r < n_tokens ? slots[r] : -1; };
    // page of a slot, -1: the row is not stored
    const auto page_of = [&](int slot) { return (uint32_t)slot < n_slots ? slot >> lg : -1; };
    const int r0 = (int)(blockIdx.x / pg.n_kv) * window;
    // lane i: row r0 - 1 + i, of which the window is the rows 1 .. window
    const int near = slot_of(r0 - 1 + lane), near_page = page_of(near);
    const int before = __shfl_up(near_page, 1);
    uint64_t starts = __ballot(lane >= 1 && lane <= window && near_page >= 0 && near_page != before);
    while (starts) {
        const int first = __builtin_ctzll(starts);
        starts &= starts - 1;
        const int r = r0 - 1 + first, page = __builtin_amdgcn_readlane(near_page, first);
        const int off0 = __builtin_amdgcn_readlane(near, first) & (P - 1);
        // the run's rows r .. r+len-1, and whether their slots ascend one by one
        uint64_t out = __ballot(near_page != page) >> first;
        int len = out ? __builtin_ctzll(out) : 64 - first;  // below 64
        bool ascend = !((__ballot(near - off0 != (page << lg) + lane - first) >> first) & ((1ull << len) - 1));
        while (!out) {  // ends: rows past the last one are out
            const int s = slot_of(r + len + lane);
            out = __ballot(page_of(s) != page);
            const uint64_t in = out ? (1ull << __builtin_ctzll(out)) - 1 : ~0ull;
            ascend = ascend && !(__ballot(s - off0 != (page << lg) + len + lane) & in);
            len += out ? __builtin_ctzll(out) : 64;
        }
        int lo = off0, hi = off0 + len - 1;  // the offsets that the run covers
        __syncthreads();                     // row_of and amax_s of the last run have been read
        if (!ascend) {
            if (tid < P) row_of[tid] = -1;
            __syncthreads();
            lo = P, hi = 0;
            for (int i = lane; i < len; i += 64) {
                const int off = slots[r + i] & (P - 1);
                atomicMax(&row_of[off], r + i);  // a slot named twice: the later row
                lo = min(lo, off);
                hi = max(hi, off);
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                lo = min(lo, __shfl_xor(lo, d));
                hi = max(hi, __shfl_xor(hi, d));
            }
        }
        const size_t block = (size_t)page * pg.n_kv + head;
        float *scale_p = (is_v ? pg.vs : pg.ks) + block;
        int8_t *quants = (is_v ? pg.vq : pg.kq) + ((block * HD) << lg);
        const float old = *scale_p;
        uint32_t amax = 0;
#pragma unroll 4
        for (int i = tid; i < len * U; i += kAppThreads) {
            const T *x = src + (size_t)(r + i / U) * stride + i % U * 8;
            const float4 a = act_ld4(x, 0), b = act_ld4(x, 1);
            // as bits: NaN > infinity > finite
            amax = max(amax, max(max(abs_bits(a.x), abs_bits(a.y)), max(abs_bits(a.z), abs_bits(a.w))));
            amax = max(amax, max(max(abs_bits(b.x), abs_bits(b.y)), max(abs_bits(b.z), abs_bits(b.w))));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
        if (lane == 0) amax_s[tid >> 6] = amax;
        __syncthreads();
        amax = max(max(amax_s[0], amax_s[1]), max(amax_s[2], amax_s[3]));
        // the run's row at an offset of lo .. hi, -1: none
        const auto row_at = [&](int off) {
            return ascend ? (off >= lo && off <= hi ? r + (off - lo) : -1) : row_of[off];
        };
        const float need = amax >= kInfBits ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax) / 127.f;
        float scale = need;
        // scale and what it divides both times 2^64 where 1/scale could overflow
        const auto raise = [](float s) { return s < 0x1p-64f ? 0x1p64f : 1.f; };
        if (row_at(0) < 0) {
            if (need != need || old != old) {
                scale = __uint_as_float(0x7fc00000u);
            } else if (need > old) {
                uint4 *w = reinterpret_cast<uint4 *>(quants);
                const float up = raise(need), d = need * up, inv = 1.f / d;
                for (int i = tid; i < (HD << lg) / 16; i += kAppThreads) w[i] = regrid(w[i], old * up, d, inv);
                __syncthreads();  // the run's quants go over the old ones
            } else {
                scale = old;
            }
        }
        if (tid == 0) *scale_p = scale;  // every thread has read the old one
        const bool live = scale > 0.f;   // neither 0 nor NaN
        const float up = raise(scale), d = scale * up, inv = live ? 1.f / d : 0.f;
        const auto quant = [&](float x) {
            return live ? (uint32_t)quant_rte(x * up, 0.f, d, inv) & 0xffu : 0u;
        };
        if (!is_v) {
#pragma unroll 4
            for (int i = tid; i < (hi - lo + 1) * U; i += kAppThreads) {
                const int off = lo + i / U, c = i % U, row = row_at(off);
                const T *x = src + (size_t)max(row, r) * stride + c * 8;
                const float4 a = act_ld4(x, 0), b = act_ld4(x, 1);
                uint2 o;
                o.x = quant(a.x) | quant(a.y) << 8 | quant(a.z) << 16 | quant(a.w) << 24;
                o.y = quant(b.x) | quant(b.y) << 8 | quant(b.z) << 16 | quant(b.w) << 24;
                if (row >= 0) reinterpret_cast<uint2 *>(quants + (size_t)off * HD)[c] = o;
            }
        } else {
            for (int i = tid; i < (hi / 16 - lo / 16 + 1) * (HD / 2); i += kAppThreads) {
                const int o16 = lo / 16 + i / (HD / 2), c = i % (HD / 2);
                int8_t *dst = quants + ((size_t)(o16 / 2) * HD + c * 2) * 32 + o16 % 2 * 16;
                uint32_t w[2][4] = {}, in = 0;
                const int j0 = max(lo - o16 * 16, 0), j1 = min(hi - o16 * 16, 15);
                if (j1 - j0 < 2) {  // single tokens, the end of a run: only what is there
                    for (int j = j0; j <= j1; j++) {
                        const int row = row_at(o16 * 16 + j);
                        if (row < 0) continue;
                        const float2 x = act_ld2(src + (size_t)row * stride, c);
                        dst[j] = (int8_t)quant(x.x);
                        dst[32 + j] = (int8_t)quant(x.y);
                    }
                    continue;
                }
                float2 x[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int row = row_at(o16 * 16 + j);
                    in |= (row >= 0 ? 1u : 0u) << j;
                    x[j] = act_ld2(src + (size_t)max(row, r) * stride, c);
                }
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    w[0][j / 4] |= quant(x[j].x) << (j % 4 * 8);
                    w[1][j / 4] |= quant(x[j].y) << (j % 4 * 8);
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (in == 0xffffu) {
                        *reinterpret_cast<uint4 *>(dst + e * 32) = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (in >> j & 1) dst[e * 32 + j] = (int8_t)(w[e][j / 4] >> (j % 4 * 8));
                    }
                }
            }
        }
    }
}

// Slots as values: a half wave reads 4 dims a lane (HD/4 lanes a row) of
// kGatherRows rows in turn.  V's dword holds 4 tokens of a dim: it is loaded
// again only when a row leaves it, so consecutive slots read V once.
constexpr int kGatherRows = 8;

template <typename T, int HD>
__global__ __launch_bounds__(kAppThreads) void paged_gather_kernel(
    T *__restrict__ k, uint64_t k_stride, T *__restrict__ v, uint64_t v_stride,
    const int32_t *__restrict__ slots, int n_tokens, PagedPages pg) {
    constexpr int kLanes = HD / 4;  // of a row
    const int head = blockIdx.x % pg.n_kv, lg = pg.page_log2, c = threadIdx.x % kLanes;
    const uint32_t n_slots = (uint32_t)pg.n_pages << lg;
    const int r0 = ((int)(blockIdx.x / pg.n_kv) * (kAppThreads / kLanes) + threadIdx.x / kLanes) * kGatherRows;
    const auto put = [&](T *p, float a, float b, float c4, float d) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(p) = make_float4(a, b, c4, d);
        } else {
            const uint2 w = make_uint2(f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16,
                                       f32_to_f16_bits(c4) | (uint32_t)f32_to_f16_bits(d) << 16);
            *reinterpret_cast<uint2 *>(p) = w;
        }
    };
    int slot_j[kGatherRows];
#pragma unroll
    for (int j = 0; j < kGatherRows; j++) slot_j[j] = r0 + j < n_tokens ? slots[r0 + j] : -1;
    uint32_t word = ~0u, w[4] = {};
#pragma unroll
    for (int j = 0; j < kGatherRows; j++) {
        const uint32_t slot = (uint32_t)slot_j[j];
        if (slot >= n_slots) continue;
        const int off = slot & ((1u << lg) - 1);
        const size_t block = (size_t)(slot >> lg) * pg.n_kv + head;
        const float ks = pg.ks[block], vs = pg.vs[block];
        const uint32_t q = *reinterpret_cast<const uint32_t *>(pg.kq + ((block * HD) << lg) + (size_t)off * HD + c * 4);
        if (word != slot / 4) {
            const int8_t *vp = pg.vq + ((block * HD) << lg) + ((size_t)(off / 32) * HD + c * 4) * 32 + off % 32 / 4 * 4;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = *reinterpret_cast<const uint32_t *>(vp + e * 32);
            word = slot / 4;
        }
        const int b = slot % 4 * 8;
        const size_t r = (size_t)(r0 + j), at = (size_t)head * HD + c * 4;
        put(k + r * k_stride + at, (float)(int8_t)q * ks, (float)(int8_t)(q >> 8) * ks,
            (float)(int8_t)(q >> 16) * ks, (float)(int8_t)(q >> 24) * ks);
        put(v + r * v_stride + at, (float)(int8_t)(w[0] >> b) * vs, (float)(int8_t)(w[1] >> b) * vs,
            (float)(int8_t)(w[2] >> b) * vs, (float)(int8_t)(w[3] >> b) * vs);
    }
}

template <typename T, int HD>
int append(hipStream_t st, const PagedPages &pg, const void *k, uint64_t k_stride, const void *v,
           uint64_t v_stride, const int32_t *slots, int n) {
    // few rows: one a workgroup, as they are likely single tokens of many
    // requests; many: runs of up to a page
    const int window = n <= 512 ? 1 : n <= 2048 ? 4 : 16;
    // the heads of a row side by side, as they lie
    const dim3 grid((n + window - 1) / window * pg.n_kv, 2);
    hipLaunchKernelGGL((paged_append_kernel<T, HD>), grid, dim3(kAppThreads), 0, st,
                       static_cast<const T *>(k), k_stride, static_cast<const T *>(v), v_stride, slots,
                       n, window, pg);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

template <typename T, int HD>
int gather(hipStream_t st, const PagedPages &pg, const int32_t *slots, int n, void *k,
           uint64_t k_stride, void *v, uint64_t v_stride) {
    constexpr int rows = kAppThreads / (HD / 4) * kGatherRows;
    hipLaunchKernelGGL((paged_gather_kernel<T, HD>), dim3((n + rows - 1) / rows * pg.n_kv),
                       dim3(kAppThreads), 0, st, static_cast<T *>(k), k_stride, static_cast<T *>(v),
                       v_stride, slots, n, pg);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

}  // namespace

#define SGQ_BY_TYPE(f, ...)                                                                     \
    switch (pg.head_dim) {                                                                      \
        case 128: return f16 ? f<uint16_t, 128>(__VA_ARGS__) : f<float, 128>(__VA_ARGS__);      \
        case 256: return f16 ? f<uint16_t, 256>(__VA_ARGS__) : f<float, 256>(__VA_ARGS__);      \
        case 512: return f16 ? f<uint16_t, 512>(__VA_ARGS__) : f<float, 512>(__VA_ARGS__);      \
    }                                                                                           \
    return fail(SGQ_ERR_VALIDATION, "paged cache: head_dim %d unsupported", pg.head_dim)

int launch_paged_append(hipStream_t st, const PagedPages &pg, const void *k, uint64_t k_stride,
                        const void *v, uint64_t v_stride, bool f16, const int32_t *slots,
                        uint32_t n_tokens) {
    SGQ_BY_TYPE(append, st, pg, k, k_stride, v, v_stride, slots, (int)n_tokens);
}

int launch_paged_gather(hipStream_t st, const PagedPages &pg, const int32_t *slots,
                        uint32_t n_tokens, bool f16, void *k, uint64_t k_stride, void *v,
                        uint64_t v_stride) {
    SGQ_BY_TYPE(gather, st, pg, slots, (int)n_tokens, k, k_stride, v, v_stride);
}

}  // namespace sgq
