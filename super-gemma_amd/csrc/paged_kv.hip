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

// rte(x/d) for finite x and d > 0, |x| <= 127.5·d: t = rint(x·(1/d)) is off by
// at most one, and then x - t·d is a multiple of the smaller of both units in
// the last place and below 2·d, so the fma is exact and compares with d/2.
__device__ __forceinline__ int quant_rte(float x, float d, float inv) {
    float t = rintf(x * inv);
    const float r = fmaf(-t, d, x), h = 0.5f * d;
    const int odd = (int)t & 1;
    if (r > h || (r == h && odd)) t += 1.f;
    else if (r < -h || (r == -h && odd)) t -= 1.f;
    return (int)fminf(fmaxf(t, -127.f), 127.f);
}

template <typename T>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(
    const T *__restrict__ k, uint64_t k_stride, const T *__restrict__ v, uint64_t v_stride,
    const int32_t *__restrict__ slots, int n_tokens, int rows_per_wg, PagedPages pg) {
    __shared__ int row_of[128];      // offset in the page -> row of the run, -1: none
    __shared__ uint32_t amax_s[kAppThreads / 64];
    __shared__ int len_s;
    const int tid = threadIdx.x, head = blockIdx.y, hd = pg.head_dim;
    const bool is_v = blockIdx.z != 0;
    const int P = 1 << pg.page_log2;
    const int r0 = blockIdx.x * rows_per_wg, r1 = min(r0 + rows_per_wg, n_tokens);
    const T *src = (is_v ? v : k) + (size_t)head * hd;
    const uint64_t stride = is_v ? v_stride : k_stride;
    const uint32_t n_slots = (uint32_t)pg.n_pages << pg.page_log2;
    for (int r = r0; r < r1; r++) {
        const int slot = slots[r];
        if ((uint32_t)slot >= n_slots) continue;
        const int page = slot >> pg.page_log2;
        if (r > 0) {
            const int before = slots[r - 1];
            if ((uint32_t)before < n_slots && before >> pg.page_log2 == page) continue;
        }
        // the run's rows: r .. r+len-1
        __syncthreads();  // row_of, amax_s and len_s of the last run have been read
        if (tid < P) row_of[tid] = -1;
        if (tid == 0) len_s = n_tokens - r;
        __syncthreads();
        for (int b = r;; b += kAppThreads) {  // ends: past n_tokens nothing is in the run
            const int i = b + tid;
            const int s = i < n_tokens ? slots[i] : -1;
            const bool in = (uint32_t)s < n_slots && s >> pg.page_log2 == page;
            if (!in) atomicMin(&len_s, max(i - r, 0));
            __syncthreads();
            const int len = len_s;
            __syncthreads();
            if (len < b + kAppThreads - r || b + kAppThreads >= n_tokens) break;
        }
        const int len = len_s;
        for (int i = tid; i < len; i += kAppThreads)
            atomicMax(&row_of[slots[r + i] & (P - 1)], r + i);  // a slot named twice: the later row
        uint32_t amax = 0;
        const int u = hd / 4;  // 4 dims a unit
        for (int i = tid; i < len * u; i += kAppThreads) {
            const int row = i / u, c = i - row * u;
            const float4 x = act_ld4(src + (size_t)(r + row) * stride, c);
            const uint32_t a = max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu);
            const uint32_t b = max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu);
            amax = max(amax, max(a, b));  // as bits: NaN > infinity > finite
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
        if ((tid & 63) == 0) amax_s[tid >> 6] = amax;
        __syncthreads();
        amax = max(max(amax_s[0], amax_s[1]), max(amax_s[2], amax_s[3]));
        const float need = amax >= kInfBits ? __uint_as_float(0x7fc00000u) : __uint_as_float(amax) / 127.f;
        const size_t block = (size_t)page * pg.n_kv + head;
        float *scale_p = (is_v ? pg.vs : pg.ks) + block;
        int8_t *quants = (is_v ? pg.vq : pg.kq) + ((block * hd) << pg.page_log2);
        float scale = need;
        if (row_of[0] < 0) {
            const float old = *scale_p;
            if (need != need || old != old) {
                scale = __uint_as_float(0x7fc00000u);
            } else if (need > old) {
                // q·old has up to 31 bits: the quotient is taken in fp64
                for (int i = tid; i < (hd << pg.page_log2) / 4; i += kAppThreads) {
                    uint32_t w = reinterpret_cast<uint32_t *>(quants)[i], o = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int q = (int8_t)(w >> (8 * j));
                        const int t = (int)rint((double)q * (double)old / (double)need);
                        o |= ((uint32_t)t & 0xffu) << (8 * j);
                    }
                    reinterpret_cast<uint32_t *>(quants)[i] = o;
                }
            } else {
                scale = old;
            }
        }
        __syncthreads();  // every thread has read the old scale and written its old quants
        if (tid == 0) *scale_p = scale;
        const bool live = scale > 0.f;  // neither 0 nor NaN
        // x and scale both times 2^64 where 1/scale could overflow (|x| <= 127.5·scale)
        const float up = scale < 0x1p-64f ? 0x1p64f : 1.f, d = scale * up;
        const float inv = live ? 1.f / d : 0.f;
        if (!is_v) {
            for (int i = tid; i < P * u; i += kAppThreads) {
                const int off = i / u, c = i - off * u, row = row_of[off];
                if (row < 0) continue;
                const float4 x = act_ld4(src + (size_t)row * stride, c);
                uint32_t o = 0;
                if (live)
                    o = ((uint32_t)quant_rte(x.x * up, d, inv) & 0xffu) |
                        ((uint32_t)quant_rte(x.y * up, d, inv) & 0xffu) << 8 |
                        ((uint32_t)quant_rte(x.z * up, d, inv) & 0xffu) << 16 |
                        ((uint32_t)quant_rte(x.w * up, d, inv) & 0xffu) << 24;
                reinterpret_cast<uint32_t *>(quants + (size_t)off * hd)[c] = o;
            }
        } else {
            for (int i = tid; i < P / 4 * hd; i += kAppThreads) {
                const int o4 = i / hd, c = i - o4 * hd;  // 4 offsets from 4·o4 on, one dim
                int8_t *dst = quants + ((size_t)(o4 / 8) * hd + c) * 32 + (o4 % 8) * 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = row_of[o4 * 4 + j];
                    if (row < 0) continue;
                    const float x = act_ld(src + (size_t)row * stride, c);
                    dst[j] = (int8_t)(live ? quant_rte(x * up, d, inv) : 0);
                }
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kAppThreads) void paged_gather_kernel(
    T *__restrict__ k, uint64_t k_stride, T *__restrict__ v, uint64_t v_stride,
    const int32_t *__restrict__ slots, int n_tokens, PagedPages pg) {
    const int hd = pg.head_dim, head = blockIdx.y, P = 1 << pg.page_log2;
    const uint32_t n_slots = (uint32_t)pg.n_pages << pg.page_log2;
    for (int r = blockIdx.x; r < n_tokens; r += gridDim.x) {
        const int slot = slots[r];
        if ((uint32_t)slot >= n_slots) continue;
        const int off = slot & (P - 1);
        const size_t block = (size_t)(slot >> pg.page_log2) * pg.n_kv + head;
        const float ks = pg.ks[block], vs = pg.vs[block];
        const int8_t *kq = pg.kq + ((block * hd) << pg.page_log2) + (size_t)off * hd;
        const int8_t *vq = pg.vq + ((block * hd) << pg.page_log2) + (size_t)(off / 32) * hd * 32 + off % 32;
        for (int d = threadIdx.x; d < hd; d += kAppThreads) {
            act_st(k + (size_t)r * k_stride + (size_t)head * hd, d, (float)kq[d] * ks);
            act_st(v + (size_t)r * v_stride + (size_t)head * hd, d, (float)vq[(size_t)d * 32] * vs);
        }
    }
}

}  // namespace

int launch_paged_append(hipStream_t st, const PagedPages &pg, const void *k, uint64_t k_stride,
                        const void *v, uint64_t v_stride, bool f16, const int32_t *slots,
                        uint32_t n_tokens) {
    const int rows = n_tokens > 1024 ? 8 : 1;
    const dim3 grid((n_tokens + rows - 1) / rows, pg.n_kv, 2);
    if (f16)
        hipLaunchKernelGGL(paged_append_kernel<uint16_t>, grid, dim3(kAppThreads), 0, st,
                           static_cast<const uint16_t *>(k), k_stride,
                           static_cast<const uint16_t *>(v), v_stride, slots, (int)n_tokens, rows, pg);
    else
        hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(kAppThreads), 0, st,
                           static_cast<const float *>(k), k_stride, static_cast<const float *>(v),
                           v_stride, slots, (int)n_tokens, rows, pg);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

int launch_paged_gather(hipStream_t st, const PagedPages &pg, const int32_t *slots,
                        uint32_t n_tokens, bool f16, void *k, uint64_t k_stride, void *v,
                        uint64_t v_stride) {
    const dim3 grid(n_tokens < 65536 ? n_tokens : 65536, pg.n_kv);
    if (f16)
        hipLaunchKernelGGL(paged_gather_kernel<uint16_t>, grid, dim3(kAppThreads), 0, st,
                           static_cast<uint16_t *>(k), k_stride, static_cast<uint16_t *>(v),
                           v_stride, slots, (int)n_tokens, pg);
    else
        hipLaunchKernelGGL(paged_gather_kernel<float>, grid, dim3(kAppThreads), 0, st,
                           static_cast<float *>(k), k_stride, static_cast<float *>(v), v_stride,
                           slots, (int)n_tokens, pg);
    SGQ_HIP(hipGetLastError());
    return SGQ_OK;
}

}  // namespace sgq
