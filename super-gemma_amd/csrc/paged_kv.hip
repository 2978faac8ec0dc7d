// Appending K and V rows to the paged 8-bit cache, and reading slots back.
//
// A run is a maximal sequence of consecutive rows that go to one page; the rows
// of a step's slot map form at most rows/P + 2·requests of them.  Per head, with
// d = max|x| / 127 over the run (one IEEE division):
//   the run holds the page's slot 0    the block begins anew, scale = d
//   else, d <= old                     scale = old
//   else                               scale = max(d, growth·old), and the
//                                      block's quants become rte(q·old/scale)
//   quants of the run's rows           rte(x/scale), 0 where scale is 0
// rte of the real quotient, ties to even: the fp32 product with the reciprocal
// gives the integer up to one, and the exact residual x - t·scale decides.
// Each growth moves the older values by up to half a step, s_i/2 of the i-th scale.
// With s_i >= growth·s_(i-1) that is growth/(2·(growth-1)) steps of the last together at
// most; with growth 1, as many halves as there were.
// A row with an infinity or a NaN makes the scale NaN, so that attention over
// the block is NaN too instead of quietly wrong.
#include <algorithm>

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

// A block's grid, and four values on it as the bytes of a word.  The low byte of
// x·(1/scale) + 1.5·2^23 is the rounded quotient, and the residual says whether it may
// be off: not while it stays below 0.49999 of the scale.  The largest residual goes
// to `far`; a thread whose unit has one above, or whose grid is so fine that
// 1/scale may overflow, rounds the unit again the exact way (about one value in 10^5).
struct Grid {
    float scale, inv, near_half;
    uint32_t keep;  // 0 where the scale is 0 or NaN
    __device__ __forceinline__ explicit Grid(float s)
        : scale(s), inv(1.f / s), near_half(s < 0x1p-64f ? -1.f : 0.49999f * s), keep(s > 0.f ? ~0u : 0u) {}
    static __device__ __forceinline__ float raise(float s) { return s < 0x1p-64f ? 0x1p64f : 1.f; }
    __device__ __forceinline__ bool again(float far) const { return keep && far > near_half; }
    __device__ __forceinline__ int8_t exact(float x) const {
        const float up = raise(scale), d = scale * up;
        return (int8_t)quant_rte(x * up, 0.f, d, 1.f / d);
    }
    __device__ __forceinline__ uint32_t quants(float x, float y, float z, float w, float &far) const {
        constexpr float kMagic = 12582912.f;
        const float a = fmaf(x, inv, kMagic), b = fmaf(y, inv, kMagic), c = fmaf(z, inv, kMagic), e = fmaf(w, inv, kMagic);
        far = fmaxf(fmaxf(far, fabsf(fmaf(kMagic - a, scale, x))), fabsf(fmaf(kMagic - b, scale, y)));
        far = fmaxf(fmaxf(far, fabsf(fmaf(kMagic - c, scale, z))), fabsf(fmaf(kMagic - e, scale, w)));
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(e), __float_as_uint(c), 0x04000c0cu);
        return (lo | hi) & keep;
    }
};

// Two consecutive activations as they lie, and as numbers.
template <typename T>
struct Pair;
template <>
struct Pair<float> {
    typedef float2 Raw;
    static __device__ __forceinline__ float2 value(Raw x) { return x; }
};
template <>
struct Pair<uint16_t> {
    typedef uint32_t Raw;
    static __device__ __forceinline__ float2 value(Raw x) {
        return make_float2(f16_bits_to_f32(x & 0xffffu), f16_bits_to_f32(x >> 16));
    }
};

__device__ __forceinline__ uint32_t most(uint32_t m, float4 x) {  // as bits: NaN > infinity > finite
    return max(m, max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w))));
}

// One workgroup writes one run at a time for one head, K (y = 0) or V (y = 1):
// the runs that begin in its window of `window` rows.  Every wave finds the runs by
// itself (a load of 64 slots and ballots); the rows are read twice, the second
// time from the caches: once for the maximum, once to be rounded.  K: a thread
// rounds 8 dims of a row.  V, stored by dim: a thread rounds 2 dims of 16 tokens,
// so a wave reads whole rows and stores 16 bytes a lane (a dword or byte at a time
// the stores alone took four times as long as the reads); only the rows before
// and behind whole groups of 16 go byte by byte.  Keeping the rows in registers
// between the two passes halved the waves in flight: 4096 rows and their read-back
// 80 us, not 42.  Bound by the two dependent passes: 4096 f16 rows of 16 heads of 128
// take 22 us, 2.2 TB/s of what must move.
template <typename T, int HD>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(
    const T *__restrict__ k, uint64_t k_stride, const T *__restrict__ v, uint64_t v_stride,
    const int32_t *__restrict__ slots, int n_tokens, int window, float growth, PagedPages pg) {
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
            amax = most(most(amax, act_ld4(x, 0)), act_ld4(x, 1));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
        if (lane == 0) amax_s[tid >> 6] = amax;
        __syncthreads();
        amax = max(max(amax_s[0], amax_s[1]), max(amax_s[2], amax_s[3]));
        const float need = amax >= kInfBits ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax) / 127.f;
        float scale = need;
        if (ascend ? lo > 0 : row_of[0] < 0) {
            if (need != need || old != old) {
                scale = __uint_as_float(0x7fc00000u);
            } else if (need > old) {
                scale = fmaxf(need, old * growth);
                uint4 *w = reinterpret_cast<uint4 *>(quants);
                const float up = Grid::raise(scale), d = scale * up, inv = 1.f / d;
                for (int i = tid; i < (HD << lg) / 16; i += kAppThreads) w[i] = regrid(w[i], old * up, d, inv);
                __syncthreads();  // the run's quants go over the old ones
            } else {
                scale = old;
            }
        }
        if (tid == 0) *scale_p = scale;  // every thread has read the old one
        const Grid grid(scale);
        // The offset of row r + i; -1 where another row has its slot.
        const auto offset_of = [&](int i) {
            if (ascend) return lo + i;
            const int off = slots[r + i] & (P - 1);
            return row_of[off] == r + i ? off : -1;
        };
        if (!is_v) {
#pragma unroll 2
            for (int i = tid; i < len * U; i += kAppThreads) {
                const int off = offset_of(i / U);
                const T *x = src + (size_t)(r + i / U) * stride + i % U * 8;
                const float4 a = act_ld4(x, 0), b = act_ld4(x, 1);
                float far = 0.f;
                const uint2 o = make_uint2(grid.quants(a.x, a.y, a.z, a.w, far), grid.quants(b.x, b.y, b.z, b.w, far));
                if (off < 0) continue;
                int8_t *dst = quants + (size_t)off * HD + i % U * 8;
                *reinterpret_cast<uint2 *>(dst) = o;
                if (grid.again(far))
                    for (int e = 0; e < 8; e++) dst[e] = grid.exact(act_ld(x, e));
            }
            continue;
        }
        const int g0 = (lo + 15) / 16, groups = ascend ? max((hi + 1) / 16 - g0, 0) : 0;
        for (int i = tid; i < groups * (HD / 2); i += kAppThreads) {
            const int o16 = g0 + i / (HD / 2), c = i % (HD / 2);
            const T *x = src + (size_t)(r + o16 * 16 - lo) * stride + c * 2;
            typename Pair<T>::Raw raw[16];
#pragma unroll
            for (int j = 0; j < 16; j++) raw[j] = *reinterpret_cast<const typename Pair<T>::Raw *>(x + j * stride);
            uint32_t w[2][4];
            float far = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 a = Pair<T>::value(raw[j * 4]), b = Pair<T>::value(raw[j * 4 + 1]);
                const float2 e = Pair<T>::value(raw[j * 4 + 2]), f = Pair<T>::value(raw[j * 4 + 3]);
                w[0][j] = grid.quants(a.x, b.x, e.x, f.x, far);
                w[1][j] = grid.quants(a.y, b.y, e.y, f.y, far);
            }
            int8_t *dst = quants + ((size_t)(o16 / 2) * HD + c * 2) * 32 + o16 % 2 * 16;
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
            *reinterpret_cast<uint4 *>(dst + 32) = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
            if (grid.again(far))
                for (int j = 0; j < 32; j++)
                    dst[(j >> 4) * 32 + (j & 15)] = grid.exact(act_ld(x + (j & 15) * stride, j >> 4));
        }
        const int before_groups = groups ? g0 * 16 - lo : len;
        for (int i = tid; i < (len - groups * 16) * (HD / 4); i += kAppThreads) {
            const int e = i / (HD / 4), c = i % (HD / 4), k = e < before_groups ? e : e + groups * 16;
            const int off = offset_of(k);
            const T *x = src + (size_t)(r + k) * stride + c * 4;
            const float4 a = act_ld4(x, 0);
            float far = 0.f;
            const uint32_t q = grid.quants(a.x, a.y, a.z, a.w, far);
            if (off < 0) continue;
            int8_t *dst = quants + ((size_t)(off / 32) * HD + c * 4) * 32 + off % 32;
            const bool again = grid.again(far);
#pragma unroll
            for (int j = 0; j < 4; j++) dst[j * 32] = (int8_t)(q >> (8 * j));
            if (again)
                for (int j = 0; j < 4; j++) dst[j * 32] = grid.exact(act_ld(x, j));
        }
    }
}

// Slots as values: a half wave reads 4 dims a lane (HD/4 lanes a row) of
// kGatherRows rows in turn.  V's dword holds 4 tokens of a dim: it is loaded
// again only when a row leaves it, so consecutive slots read V once.  Bound by its
// stores: 4096 slots of 16 heads of 128 as fp32 15 us, 5.4 TB/s (with one row a half wave
// 22).
constexpr int kGatherRows = 4;

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
           uint64_t v_stride, float growth, const int32_t *slots, int n) {
    // Single tokens want a workgroup each (16 heads of 128, 64 requests: 16 us with windows
    // of 1, 24 of 8, 59 of 32), runs as few empty workgroups as possible (a prompt of
    // 2040 rows: 56 us of 1, 34 of 8, 27 of 32; 4096 rows: 42 of 63, 53 of 32).  Many
    // rows are more often prompts: 64 windows, until a wave's 64 slots hold no more.
    const int window = std::clamp(n / 64, 1, 63);
    // the heads of a row side by side, as they lie
    const dim3 grid((n + window - 1) / window * pg.n_kv, 2);
    hipLaunchKernelGGL((paged_append_kernel<T, HD>), grid, dim3(kAppThreads), 0, st,
                       static_cast<const T *>(k), k_stride, static_cast<const T *>(v), v_stride, slots,
                       n, window, growth, pg);
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
                        const void *v, uint64_t v_stride, bool f16, float growth,
                        const int32_t *slots, uint32_t n_tokens) {
    SGQ_BY_TYPE(append, st, pg, k, k_stride, v, v_stride, growth, slots, (int)n_tokens);
}

int launch_paged_gather(hipStream_t st, const PagedPages &pg, const int32_t *slots,
                        uint32_t n_tokens, bool f16, void *k, uint64_t k_stride, void *v,
                        uint64_t v_stride) {
    SGQ_BY_TYPE(gather, st, pg, slots, (int)n_tokens, k, k_stride, v, v_stride);
}

}  // namespace sgq
