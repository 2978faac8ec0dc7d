// Attention over the paged 8-bit cache for a batch of requests of different
// lengths.
//
// Query row i of a request at position p_i attends the keys j <= p_i (and
// j > p_i - window) of its pages:
//   s_ij = scale·ks[page(j)]·(q_i · kq_j)
//   out_i = Σ_j e^(s_ij)·vs[page(j)]·vq_j / Σ_j e^(s_ij)
// In log2 units t_ij = s_ij·log2(e) + log2(vs): one FMA folds V's block scale
// into the weight w_ij = 2^(t_ij - M_i), so the accumulator is Σ w·vq and the
// denominator Σ w/vs, and M bounds each key's part in the output whatever the
// blocks' scales.
#include "paged.h"

namespace sgq {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -1e30f;      // the reference M before the first key
// M moves only when a tile's maximum is over it by this (log2); weights are
// taken against M - kHead, so f16 weights lie below 2^(kLazy + kHead) = 2^14
// and their subnormals begin 2^20 below M.
constexpr float kLazy = 8.f, kHead = 6.f;
constexpr float kMinScale = 0x1p-100f;  // V scales below weigh as this one

struct AttnArgs {
    PagedPages pg;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const int32_t *tables, *kv_lens, *cu;
    float *part;    // [row][split][hd]
    float2 *part_ml;  // [row][split] (M, l)
    int max_pages, n_seqs, n_tokens, n_q, group, max_new, window, n_splits;
    float scale_log2;
};

// A tile of query rows of one request and kv head: row r is token r/group of
// the request's new ones, query head head·group + r%group.
struct RowTile {
    int seq, tok0, new_len, row0, rows, kv_len;
};

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Tile `id` of BM rows.  Request s owns the ids from floor(cu_s·group/BM) + s
// on, which is room for its ceil(new·group/BM) tiles; ids left over are empty.
template <int BM>
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int id, RowTile *t) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const long long c = clamped(a.cu[mid], 0, a.n_tokens);
        if (c * a.group / BM + mid <= id) lo = mid;
        else hi = mid;
    }
    const int c0 = clamped(a.cu[lo], 0, a.n_tokens);
    const int c1 = clamped(a.cu[lo + 1], c0, a.n_tokens);
    t->seq = lo;
    t->tok0 = c0;
    t->new_len = min(c1 - c0, a.max_new);
    t->row0 = (id - (int)((long long)c0 * a.group / BM) - lo) * BM;
    t->rows = min(t->new_len * a.group - t->row0, BM);
    t->kv_len = a.kv_lens[lo];
    return t->row0 >= 0 && t->rows > 0;
}

// Keys [lo, hi) of the query at position pos.
__device__ __forceinline__ int key_lo(const AttnArgs &a, int pos) {
    return a.window > 0 ? max(pos - a.window + 1, 0) : 0;
}
__device__ __forceinline__ int key_hi(const AttnArgs &a, int pos, int kv_len) {
    const int cap = a.max_pages << a.pg.page_log2;
    return clamped(min(pos + 1, kv_len), 0, cap);
}

// Which 32-key tiles a row tile attends, and into how many parts of `per`
// tiles they are cut (at most n_splits, each of 8 tiles or more).
struct KeySpan {
    int t0, t1, parts, per;
};
__device__ __forceinline__ KeySpan key_span(const AttnArgs &a, const RowTile &rt) {
    const int first = rt.kv_len - rt.new_len + rt.row0 / a.group;
    const int last = rt.kv_len - rt.new_len + (rt.row0 + rt.rows - 1) / a.group;
    KeySpan k;
    k.t0 = key_lo(a, first) >> 5;
    k.t1 = max((key_hi(a, last, rt.kv_len) + 31) >> 5, k.t0);
    const int n = k.t1 - k.t0;
    const int want = clamped((n + 7) / 8, 1, a.n_splits);
    k.per = max((n + want - 1) / want, 1);
    k.parts = max((n + k.per - 1) / k.per, 1);
    return k;
}

// 8 quants (two words) as f16: byte u = q + 128 under the exponent of 1024
// makes 1024 + u exactly, minus 1152 is q.
__device__ __forceinline__ h8 quants_f16(uint32_t w0, uint32_t w1) {
    const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u, e = 0x64646464u;
    const uint32_t p[4] = {__builtin_amdgcn_perm(e, x0, 0x04010400u),
                           __builtin_amdgcn_perm(e, x0, 0x04030402u),
                           __builtin_amdgcn_perm(e, x1, 0x04010400u),
                           __builtin_amdgcn_perm(e, x1, 0x04030402u)};
    const h2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h2 v = __builtin_bit_cast(h2, p[i]) + off;
        r[2 * i] = v[0];
        r[2 * i + 1] = v[1];
    }
    return r;
}

__device__ __forceinline__ float lane_f(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

constexpr int kRowWaves = 4;

// 16 query rows against one part of the keys; 4 waves take 32-key tiles in
// turn.  Sᵀ = K·Qᵀ (v_mfma_f32_16x16x32_f16): row m of key half t is key
// 8·(m/4) + 4·t + m%4 of the tile, which leaves lane (g, n) = (lane/16,
// lane%16) with the scores of row n against keys 8g .. 8g+7 - the B operand
// of Oᵀ = Vᵀ·Pᵀ as it is.  fp32 rows go in as two f16 halves (22 bits), q
// scaled by a power of two per row, and so do their weights.
template <typename T, int HD>
__global__ __launch_bounds__(kRowWaves * 64) void paged_attn_rows_kernel(AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NC = HD / 64, ND = HD / 16;
    __shared__ float ml_s[kRowWaves][2][16];
    __shared__ __align__(16) float o_s[kRowWaves][16][64 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % a.n_splits, head = blockIdx.y;
    RowTile rt;
    if (!find_tile<16>(a, blockIdx.x / a.n_splits, &rt)) return;
    const KeySpan ks = key_span(a, rt);
    if (split >= ks.parts) return;
    const int t0 = ks.t0 + split * ks.per, t1 = min(t0 + ks.per, ks.t1);

    // this lane's query row (columns past the last row repeat it, unread)
    const int row = rt.row0 + min(n, rt.rows - 1);
    const int tok = rt.tok0 + row / a.group, qh = head * a.group + row % a.group;
    const int pos = rt.kv_len - rt.new_len + row / a.group;
    const int lo = key_lo(a, pos), hi = key_hi(a, pos, rt.kv_len);
    // tiles inside [all_lo, all_hi) need no mask
    const int first = rt.kv_len - rt.new_len + rt.row0 / a.group;
    const int last = rt.kv_len - rt.new_len + (rt.row0 + rt.rows - 1) / a.group;
    const int all_lo = key_lo(a, last), all_hi = key_hi(a, first, rt.kv_len);

    h8 qa[NC][2], ql[F32 ? NC : 1][2];
    float row_scale = a.scale_log2;
    {
        const T *src = static_cast<const T *>(a.q) + (size_t)tok * a.q_stride + (size_t)qh * HD;
        if constexpr (F32) {
            float x[NC][2][8], amax = 0.f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(src + c * 64 + g * 16 + h * 8 + j);
                        x[c][h][j] = v.x, x[c][h][j + 1] = v.y, x[c][h][j + 2] = v.z, x[c][h][j + 3] = v.w;
                        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                    }
            amax = fmaxf(amax, __shfl_xor(amax, 16));
            amax = fmaxf(amax, __shfl_xor(amax, 32));
            int e = 0;
            if (amax > 0.f && amax < INFINITY) (void)frexpf(amax, &e);
            const int up = 15 - e;  // the largest value into [2^14, 2^15)
            row_scale = ldexpf(row_scale, -up);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float v = ldexpf(x[c][h][j], up);
                        const _Float16 hi16 = (_Float16)v;
                        qa[c][h][j] = hi16;
                        ql[c][h][j] = (_Float16)(v - (float)hi16);
                    }
        } else {
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    qa[c][h] = *reinterpret_cast<const h8 *>(src + c * 64 + g * 16 + h * 8);
        }
    }

    f4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d] = f4{0.f, 0.f, 0.f, 0.f};
    float M = kNoMax, l = 0.f;
    const int32_t *table = a.tables + (size_t)rt.seq * a.max_pages;
    const int tile_page = a.pg.page_log2 - 5;  // tiles per page, log2
    // the page, and its scales, of this wave's next 64 tiles: one a lane
    int my_page = 0;
    float my_ks = 0.f, my_lv = 0.f, my_rv = 0.f;
    for (int i = 0, t = t0 + wave; t < t1; i++, t += kRowWaves) {
        if (i % 64 == 0) {
            const int mine = t + lane * kRowWaves;
            const int p = mine < t1 ? table[mine >> tile_page] : -1;
            const bool ok = (unsigned)p < (unsigned)a.pg.n_pages;
            my_page = ok ? p : 0;
            const size_t b = (size_t)my_page * a.pg.n_kv + head;
            const float vs = fmaxf(a.pg.vs[b], kMinScale) + (a.pg.vs[b] - a.pg.vs[b]);  // NaN stays
            my_ks = ok ? a.pg.ks[b] : 0.f;
            my_lv = ok ? __builtin_amdgcn_logf(vs) : -INFINITY;  // no page: no weight
            my_rv = ok && vs == vs ? 1.f / vs : 1.f;  // finite: a masked key's 0·rv stays 0
        }
        const int page = __builtin_amdgcn_readlane(my_page, i % 64);
        const float tks = lane_f(my_ks, i % 64), lv = lane_f(my_lv, i % 64), rv = lane_f(my_rv, i % 64);
        const int sub = t & ((1 << tile_page) - 1);  // the tile within its page
        const size_t base = (((size_t)page * a.pg.n_kv + head) << a.pg.page_log2) * HD + (size_t)sub * 32 * HD;
        const int8_t *kp = a.pg.kq + base + (size_t)((n >> 2) * 8 + (n & 3)) * HD + g * 16;
        const int8_t *vp = a.pg.vq + base + n * 32 + g * 8;
        uint4 kr[NC][2];
        uint2 vr[ND];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                kr[c][h] = *reinterpret_cast<const uint4 *>(kp + c * 64 + h * 4 * HD);
#pragma unroll
        for (int d = 0; d < ND; d++) vr[d] = *reinterpret_cast<const uint2 *>(vp + d * 16 * 32);

        f4 s[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const h8 k0 = quants_f16(kr[c][h].x, kr[c][h].y), k1 = quants_f16(kr[c][h].z, kr[c][h].w);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qa[c][0], s[h], 0, 0, 0);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qa[c][1], s[h], 0, 0, 0);
                if constexpr (F32) {
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[c][0], s[h], 0, 0, 0);
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[c][1], s[h], 0, 0, 0);
                }
            }
        const float c = row_scale * tks;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = fmaf(s[j >> 2][j & 3], c, lv);
        if (t * 32 < all_lo || t * 32 + 32 > all_hi) {
            const int key = t * 32 + g * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = key + j >= lo && key + j < hi ? x[j] : -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) mx = fmaxf(mx, x[j]);
        if (__any(mx > M + kLazy)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m1 = fmaxf(M, mx), f = __builtin_amdgcn_exp2f(M - m1);
            M = m1;
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; d++) acc[d] *= f;
        }
        h8 w, wl;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float p = __builtin_amdgcn_exp2f(x[j] - (M - kHead));
            sum += p;
            w[j] = (_Float16)p;
            if constexpr (F32) wl[j] = (_Float16)(p - (float)w[j]);
        }
        l = fmaf(sum, rv, l);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            const h8 v = quants_f16(vr[d].x, vr[d].y);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w, acc[d], 0, 0, 0);
            if constexpr (F32) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wl, acc[d], 0, 0, 0);
        }
    }
    // the four lanes of a row, then the four waves, in their order
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        ml_s[wave][0][n] = M;
        ml_s[wave][1][n] = l;
    }
    __syncthreads();
    float m_all = kNoMax;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) m_all = fmaxf(m_all, ml_s[w][0][n]);
    const float f = __builtin_amdgcn_exp2f(M - m_all);
    const int orow = threadIdx.x >> 4, od = (threadIdx.x & 15) * 4;
    float om = kNoMax, ol = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; w++) om = fmaxf(om, ml_s[w][0][orow]);
#pragma unroll
    for (int w = 0; w < kRowWaves; w++)
        ol += ml_s[w][1][orow] * __builtin_amdgcn_exp2f(ml_s[w][0][orow] - om);
    const int r = rt.row0 + orow;
    const int otok = rt.tok0 + r / a.group, oh = head * a.group + r % a.group;
    const size_t prow = ((size_t)otok * a.n_q + oh) * a.n_splits + split;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; d++) *reinterpret_cast<f4 *>(&o_s[wave][n][d * 16 + g * 4]) = acc[c * 4 + d] * f;
        __syncthreads();
        f4 o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kRowWaves; w++) o += *reinterpret_cast<const f4 *>(&o_s[w][orow][od]);
        if (orow < rt.rows) {
            if (ks.parts == 1) {
                // a row that attends nothing is zero
                const float inv = ol == 0.f ? 0.f : 1.f / ol;
                T *dst = static_cast<T *>(a.out) + (size_t)otok * a.out_stride + (size_t)oh * HD + c * 64 + od;
#pragma unroll
                for (int j = 0; j < 4; j++) dst[j] = (T)(o[j] * inv);
            } else {
                *reinterpret_cast<f4 *>(a.part + prow * HD + c * 64 + od) = o;
                if (c == 0 && od == 0) a.part_ml[prow] = make_float2(om, ol);
            }
        }
    }
}

// Joins the parts of a row tile's rows, in their order.
template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
    RowTile rt;
    if (!find_tile<16>(a, blockIdx.x, &rt)) return;
    const KeySpan ks = key_span(a, rt);
    if (ks.parts == 1) return;
    const int head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = wave; i < rt.rows; i += 4) {
        const int r = rt.row0 + i;
        const int tok = rt.tok0 + r / a.group, qh = head * a.group + r % a.group;
        const size_t prow = ((size_t)tok * a.n_q + qh) * a.n_splits;
        float m = kNoMax, l = 0.f, o[HD / 64];
        for (int s = 0; s < ks.parts; s++) m = fmaxf(m, a.part_ml[prow + s].x);
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] = 0.f;
        for (int s = 0; s < ks.parts; s++) {
            const float2 ml = a.part_ml[prow + s];
            const float f = __builtin_amdgcn_exp2f(ml.x - m);
            l = fmaf(ml.y, f, l);
#pragma unroll
            for (int d = 0; d < HD / 64; d++) o[d] = fmaf(a.part[(prow + s) * HD + d * 64 + lane], f, o[d]);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) dst[d * 64 + lane] = (T)(o[d] * inv);
    }
}

template <typename T, int HD>
int launch(hipStream_t st, const AttnArgs &a) {
    const int tiles = (int)((long long)a.n_tokens * a.group / 16) + a.n_seqs;
    hipLaunchKernelGGL((paged_attn_rows_kernel<T, HD>), dim3(tiles * a.n_splits, a.pg.n_kv),
                       dim3(kRowWaves * 64), 0, st, a);
    SGQ_HIP(hipGetLastError());
    if (a.n_splits > 1) {
        hipLaunchKernelGGL((paged_attn_join_kernel<T, HD>), dim3(tiles, a.pg.n_kv), dim3(256), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    return SGQ_OK;
}

// Parts that the keys are cut into: enough workgroups for two on each of the
// 256 CUs, each part of 256 keys or more.
int wanted_splits(int n_tokens, int n_seqs, int n_q, int n_kv, int max_kv) {
    const long long tiles = (long long)n_tokens * (n_q / n_kv) / 16 + n_seqs;
    const long long by_fill = (2 * 256 + tiles * n_kv - 1) / (tiles * n_kv);
    const long long by_keys = ((long long)max_kv + 255) / 256;
    const long long s = by_fill < by_keys ? by_fill : by_keys;
    return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

}  // namespace

uint64_t paged_attn_workspace(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim,
                              int max_new, int max_kv) {
    (void)max_new;
    const int s = wanted_splits(n_tokens, n_seqs, n_q, n_kv, max_kv);
    return s <= 1 ? 0 : (uint64_t)n_tokens * n_q * s * (head_dim + 2) * 4;
}

int launch_paged_attn(hipStream_t st, const PagedAttn &p) {
    AttnArgs a{};
    a.pg = p.pg;
    a.q = p.q, a.out = p.out, a.q_stride = p.q_stride, a.out_stride = p.out_stride;
    a.tables = p.tables, a.kv_lens = p.kv_lens, a.cu = p.cu;
    a.max_pages = p.max_pages, a.n_seqs = p.n_seqs, a.n_tokens = p.n_tokens, a.n_q = p.n_q;
    a.group = p.n_q / p.pg.n_kv, a.max_new = p.max_new, a.window = p.window;
    a.scale_log2 = p.scale * kLog2e;
    const uint64_t row_bytes = (uint64_t)p.n_tokens * p.n_q * (p.pg.head_dim + 2) * 4;
    const uint64_t fit = p.workspace ? p.workspace_bytes / row_bytes : 0;
    const int want = wanted_splits(p.n_tokens, p.n_seqs, p.n_q, p.pg.n_kv, p.max_kv);
    a.n_splits = fit < 2 ? 1 : fit < (uint64_t)want ? (int)fit : want;
    a.part = static_cast<float *>(p.workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part + (uint64_t)p.n_tokens * p.n_q * a.n_splits * p.pg.head_dim);
    switch (p.pg.head_dim * 2 + (p.f16 ? 1 : 0)) {
        case 128 * 2: return launch<float, 128>(st, a);
        case 128 * 2 + 1: return launch<_Float16, 128>(st, a);
        case 256 * 2: return launch<float, 256>(st, a);
        case 256 * 2 + 1: return launch<_Float16, 256>(st, a);
        case 512 * 2: return launch<float, 512>(st, a);
        case 512 * 2 + 1: return launch<_Float16, 512>(st, a);
    }
    return fail(SGQ_ERR_VALIDATION, "attn_paged_q8: head_dim %d unsupported (128, 256, 512)", p.pg.head_dim);
}

}  // namespace sgq
