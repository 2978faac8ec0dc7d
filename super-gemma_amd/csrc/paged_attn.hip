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
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace sgq {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

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
    float *part;      // [row][split][hd]
    float2 *part_ml;  // [row][split] (M, l)
    int max_pages, n_seqs, n_tokens, n_q, group, max_new, window;
    int few_splits, many_splits;  // parts at most, of requests with few and with many rows
    int few_per, many_per;        // their length in 32-key tiles, if that makes no more of them
    int part_slots;               // parts that the workspace holds for a row
    bool few;                     // requests with few rows go to their own kernel
    float scale_log2;
};

// A tile of query rows of one request and kv head: row r is token r/group of
// the request's new ones, query head head·group + r%group.
struct RowTile {
    int seq, tok0, new_len, row0, rows, kv_len;
};

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Requests with at most kFewRows rows a kv head (single tokens) share a wave's
// 16 columns; their keys are what is spread over the GPU.
constexpr int kFewRows = 16;

__device__ __forceinline__ bool request_rows(const AttnArgs &a, int seq, RowTile *t) {
    const int c0 = clamped(a.cu[seq], 0, a.n_tokens);
    const int c1 = clamped(a.cu[seq + 1], c0, a.n_tokens);
    t->seq = seq;
    t->tok0 = c0;
    t->new_len = min(c1 - c0, a.max_new);
    t->kv_len = a.kv_lens[seq];
    return t->new_len > 0;
}

// The rows of request `seq` when they are few.
__device__ __forceinline__ bool few_rows(const AttnArgs &a, int seq, RowTile *t) {
    if (!request_rows(a, seq, t) || t->new_len * a.group > kFewRows) return false;
    t->row0 = 0;
    t->rows = t->new_len * a.group;
    return true;
}

// Tile `id` of BM rows.  Request s owns the ids from floor(cu_s·group/BM) + s
// on, which is room for its ceil(new·group/BM) tiles; ids left over are empty.
template <int BM>
__device__ __forceinline__ bool many_rows(const AttnArgs &a, int id, RowTile *t) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const long long c = clamped(a.cu[mid], 0, a.n_tokens);
        if (c * a.group / BM + mid <= id) lo = mid;
        else hi = mid;
    }
    if (!request_rows(a, lo, t) || (a.few && t->new_len * a.group <= kFewRows)) return false;
    t->row0 = (id - (int)((long long)t->tok0 * a.group / BM) - lo) * BM;
    t->rows = min(t->new_len * a.group - t->row0, BM);
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
// tiles they are cut: parts of one length for all requests, so that a long one
// has more of them, unless that makes more than `splits`.
struct KeySpan {
    int t0, t1, parts, per;
};
__device__ __forceinline__ KeySpan key_span(const AttnArgs &a, const RowTile &rt, int splits, int per) {
    const int first = rt.kv_len - rt.new_len + rt.row0 / a.group;
    const int last = rt.kv_len - rt.new_len + (rt.row0 + rt.rows - 1) / a.group;
    KeySpan k;
    k.t0 = key_lo(a, first) >> 5;
    k.t1 = max((key_hi(a, last, rt.kv_len) + 31) >> 5, k.t0);
    const int n = k.t1 - k.t0;
    k.per = max(per, (n + splits - 1) / splits);
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

// 8 quants as the f16 numbers (q + 128)·2^-24: the byte is a subnormal's bits.
// Exact, at 6 operations in place of 10; who takes these subtracts the 128.
__device__ __forceinline__ h8 quants_f16_raised(uint32_t w0, uint32_t w1) {
    const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u;
    const uint4 p = make_uint4(__builtin_amdgcn_perm(0, x0, 0x0c010c00u), __builtin_amdgcn_perm(0, x0, 0x0c030c02u),
                               __builtin_amdgcn_perm(0, x1, 0x0c010c00u), __builtin_amdgcn_perm(0, x1, 0x0c030c02u));
    return __builtin_bit_cast(h8, p);
}

__device__ __forceinline__ float lane_f(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

template <bool STREAM, typename V>
__device__ __forceinline__ V load(const int8_t *p) {
    const V *v = reinterpret_cast<const V *>(p);
    return STREAM ? __builtin_nontemporal_load(v) : *v;
}

__device__ __forceinline__ float fmax16(float v) {  // over the lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// One wave: 16·NT query rows (columns n of NT column tiles) against 32 keys at a
// time.  Sᵀ = K·Qᵀ (v_mfma_f32_16x16x32_f16): row m of key half h is key
// 8·(m/4) + 4·h + m%4 of the tile, which leaves lane (g, n) = (lane/16, lane%16)
// with the scores of row n against keys 8g .. 8g+7 - the B operand of
// Oᵀ = Vᵀ·Pᵀ as it is, so neither P nor a quant passes through LDS or a
// shuffle.  The quants become f16 once for the NT column tiles.  fp32 rows go in
// as two f16 halves (22 bits), q scaled by a power of two per row, and so do
// their weights.
template <typename T, int HD, int NT>
struct Wave {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NC = HD / 64, ND = HD / 16;
    h8 qa[NT][NC][2], ql[F32 ? NT : 1][F32 ? NC : 1][2];
    // x = s·(row_scale·ks) + row_raise·ks: f16 rows meet K raised by 128, and the
    // second term takes 128·Σq away.  Its rounding is 2^-24 of numbers some
    // four times the scores: far below an f16 weight's, not below an fp32 one's.
    float row_scale[NT], row_raise[NT];
    f4 acc[NT][ND];
    float M[NT], l[NT];

    __device__ __forceinline__ void load_q(const AttnArgs &a, const RowTile &rt, int head, int n, int g) {
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int row = rt.row0 + min(i * 16 + n, rt.rows - 1);  // columns past the last row repeat it
            const T *src = static_cast<const T *>(a.q) + (size_t)(rt.tok0 + row / a.group) * a.q_stride +
                           (size_t)(head * a.group + row % a.group) * HD + g * 16;
            row_scale[i] = a.scale_log2;
            M[i] = kNoMax;
            l[i] = 0.f;
#pragma unroll
            for (int d = 0; d < ND; d++) acc[i][d] = f4{0.f, 0.f, 0.f, 0.f};
            if constexpr (F32) {
                float x[NC][2][8], amax = 0.f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(src + c * 64 + j);
                        float *y = &x[c][j / 8][j % 8];
                        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
                        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                    }
                amax = fmax16(amax);
                int e = 0;
                if (amax > 0.f && amax < INFINITY) (void)frexpf(amax, &e);
                const int up = 15 - e;  // the largest value into [2^14, 2^15)
                row_scale[i] = ldexpf(row_scale[i], -up);
                row_raise[i] = 0.f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float v = ldexpf(x[c][h][j], up);
                            const _Float16 hi16 = (_Float16)v;
                            qa[i][c][h][j] = hi16;
                            ql[i][c][h][j] = (_Float16)(v - (float)hi16);
                        }
            } else {
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        qa[i][c][h] = *reinterpret_cast<const h8 *>(src + c * 64 + h * 8);
#pragma unroll
                        for (int j = 0; j < 8; j++) sum += (float)qa[i][c][h][j];
                    }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                row_raise[i] = -128.f * sum * row_scale[i];
                row_scale[i] *= 0x1p24f;
            }
        }
    }

    // Tiles t0, t0 + step, ... below t1.  STREAM: no other wave reads these pages
    // soon, so they are not kept in the caches.
    template <bool STREAM>
    __device__ __forceinline__ void attend(const AttnArgs &a, const RowTile &rt, int head, int t0, int t1,
                                           int step, int lane) {
        const int n = lane & 15, g = lane >> 4;
        const int base_pos = rt.kv_len - rt.new_len;
        const int last_row = rt.row0 + rt.rows - 1;
        // tiles inside [all_lo, all_hi] need no mask
        const int all_lo = key_lo(a, base_pos + last_row / a.group);
        const int all_hi = key_hi(a, base_pos + rt.row0 / a.group, rt.kv_len);
        const int32_t *table = a.tables + (size_t)rt.seq * a.max_pages;
        const int lg = a.pg.page_log2;
        // the page, and its scales, of this wave's next 64 tiles: one a lane
        int my_page = 0;
        float my_ks = 0.f, my_lv = 0.f, my_rv = 0.f;
        const auto load_pages = [&](int t) {
            const int mine = t + lane * step;
            const int p = mine < t1 ? table[mine >> (lg - 5)] : -1;
            const bool ok = (unsigned)p < (unsigned)a.pg.n_pages;
            my_page = ok ? p : 0;
            const size_t b = (size_t)my_page * a.pg.n_kv + head;
            const float raw = a.pg.vs[b];
            const float vs = fmaxf(raw, kMinScale) + (raw - raw);  // NaN stays
            my_ks = ok ? a.pg.ks[b] : 0.f;
            my_lv = ok ? __builtin_amdgcn_logf(vs) : -INFINITY;  // no page: no weight
            my_rv = ok && vs == vs ? 1.f / vs : 1.f;             // finite: a masked key's 0·rv stays 0
        };
        const size_t lane_k = (size_t)((n >> 2) * 8 + (n & 3)) * HD + g * 16;
        const size_t lane_v = n * 32 + g * 8;
        const auto block = [&](int t, int i) {  // the quants of tile t, the wave's i-th
            const int page = __builtin_amdgcn_readlane(my_page, i % 64);
            return ((((size_t)page * a.pg.n_kv + head) << (lg - 5)) + (t & ((1 << (lg - 5)) - 1))) * (32 * HD);
        };
        u4 kr[NC][2];
        u2 vr[ND];
        const auto load_k = [&](size_t b) {
            const int8_t *p = a.pg.kq + b + lane_k;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) kr[c][h] = load<STREAM, u4>(p + c * 64 + h * 4 * HD);
        };
        if (t0 >= t1) return;
        load_pages(t0);
        size_t blk = block(t0, 0);
        load_k(blk);
        // One tile.  Its V and then the next tile's K are on their way while it is
        // worked on; the last tile has a copy of this code without that K, as a
        // load under a condition would be waited for at once.
        const auto tile = [&](int i, int t, auto more) {
            const float tks = lane_f(my_ks, i % 64), lv = lane_f(my_lv, i % 64), rv = lane_f(my_rv, i % 64);
            const int8_t *vp = a.pg.vq + blk + lane_v;
#pragma unroll
            for (int d = 0; d < ND; d++) vr[d] = load<STREAM, u2>(vp + d * 16 * 32);
            f4 s[NT][2];
#pragma unroll
            for (int j = 0; j < NT; j++) s[j][0] = s[j][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const h8 k0 = F32 ? quants_f16(kr[c][h].x, kr[c][h].y) : quants_f16_raised(kr[c][h].x, kr[c][h].y);
                    const h8 k1 = F32 ? quants_f16(kr[c][h].z, kr[c][h].w) : quants_f16_raised(kr[c][h].z, kr[c][h].w);
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qa[j][c][0], s[j][h], 0, 0, 0);
                        if constexpr (F32)
                            s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[j][c][0], s[j][h], 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qa[j][c][1], s[j][h], 0, 0, 0);
                        if constexpr (F32)
                            s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[j][c][1], s[j][h], 0, 0, 0);
                    }
                }
            if constexpr (decltype(more)::value) {
                if (i % 64 == 63) load_pages(t + step);
                blk = block(t + step, i + 1);
                load_k(blk);
            }
            float x[NT][8], mx = -INFINITY;
            const bool edge = t * 32 < all_lo || t * 32 + 32 > all_hi;
            const auto weights = [&]() {
                mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const float c = row_scale[j] * tks, b = fmaf(row_raise[j], tks, lv + (kHead - M[j]));
#pragma unroll
                    for (int e = 0; e < 8; e++) x[j][e] = fmaf(s[j][e >> 2][e & 3], c, b);
                    if (edge) {
                        const int row = rt.row0 + min(j * 16 + n, rt.rows - 1);
                        const int pos = base_pos + row / a.group;
                        const int lo = key_lo(a, pos), hi = key_hi(a, pos, rt.kv_len), key = t * 32 + g * 8;
#pragma unroll
                        for (int e = 0; e < 8; e++) x[j][e] = key + e >= lo && key + e < hi ? x[j][e] : -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) mx = fmaxf(mx, x[j][e]);
                }
            };
            weights();
            if (__any(mx > kLazy + kHead)) {
                // a larger reference: from the scores again, as x may hold them against none
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const float c = row_scale[j] * tks, b = fmaf(row_raise[j], tks, lv);
                    float m = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        m = fmaxf(m, x[j][e] == -INFINITY ? x[j][e] : fmaf(s[j][e >> 2][e & 3], c, b));
                    const float m1 = fmaxf(M[j], fmax16(m)), f = __builtin_amdgcn_exp2f(M[j] - m1);
                    M[j] = m1;
                    l[j] *= f;
#pragma unroll
                    for (int d = 0; d < ND; d++) acc[j][d] *= f;
                }
                weights();
            }
            h8 w[NT], wl[F32 ? NT : 1];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = __builtin_amdgcn_exp2f(x[j][e]);
                    sum += p;  // not the f16 weight: over a block of small V scale that may be 0
                    w[j][e] = (_Float16)p;
                    if constexpr (F32) wl[j][e] = (_Float16)(p - (float)w[j][e]);
                }
                l[j] = fmaf(sum, rv, l[j]);
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const h8 v = quants_f16(vr[d].x, vr[d].y);
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    acc[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[j], acc[j][d], 0, 0, 0);
                    if constexpr (F32) acc[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wl[j], acc[j][d], 0, 0, 0);
                }
            }
        };
        int i = 0, t = t0;
        for (; t + step < t1; i++, t += step) tile(i, t, std::true_type{});
        tile(i, t, std::false_type{});
#pragma unroll
        for (int j = 0; j < NT; j++) {  // the lanes of a row have the same M
            l[j] += __shfl_xor(l[j], 16);
            l[j] += __shfl_xor(l[j], 32);
        }
    }
};

__device__ __forceinline__ float4 scaled(f4 o, float f) { return make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f); }
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store4(_Float16 *p, float4 v) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4 *>(p) = h4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
}
// a row that attends nothing is zero
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Few rows: one request and kv head against one part of the keys, the tiles dealt
// to 4 waves in turn and their sums joined in LDS in wave order.
constexpr int kFewWaves = 4;

template <typename T, int HD>
__global__ __launch_bounds__(kFewWaves * 64, HD == 128 ? 3 : HD == 256 ? 2 : 1) void paged_attn_few_kernel(AttnArgs a) {
    constexpr int NC = HD / 64;
    __shared__ float ml_s[kFewWaves][2][16];
    __shared__ __align__(16) float o_s[kFewWaves][16][64 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    // the heads of a page lie side by side, and so do their workgroups
    const int head = blockIdx.x % a.pg.n_kv, unit = blockIdx.x / a.pg.n_kv;
    const int split = unit % a.few_splits;
    RowTile rt;
    if (!few_rows(a, unit / a.few_splits, &rt)) return;
    const KeySpan ks = key_span(a, rt, a.few_splits, a.few_per);
    if (split >= ks.parts) return;
    const int t0 = ks.t0 + split * ks.per, t1 = min(t0 + ks.per, ks.t1);
    Wave<T, HD, 1> w;
    w.load_q(a, rt, head, n, g);
    w.template attend<true>(a, rt, head, t0 + wave, t1, kFewWaves, lane);
    if (g == 0) {
        ml_s[wave][0][n] = w.M[0];
        ml_s[wave][1][n] = w.l[0];
    }
    __syncthreads();
    float m_all = kNoMax;
#pragma unroll
    for (int i = 0; i < kFewWaves; i++) m_all = fmaxf(m_all, ml_s[i][0][n]);
    const float f = __builtin_amdgcn_exp2f(w.M[0] - m_all);
    const int orow = threadIdx.x >> 4, od = (threadIdx.x & 15) * 4;
    float om = kNoMax, ol = 0.f;
#pragma unroll
    for (int i = 0; i < kFewWaves; i++) om = fmaxf(om, ml_s[i][0][orow]);
#pragma unroll
    for (int i = 0; i < kFewWaves; i++)
        ol += ml_s[i][1][orow] * __builtin_amdgcn_exp2f(ml_s[i][0][orow] - om);
    const int otok = rt.tok0 + orow / a.group, oh = head * a.group + orow % a.group;
    const size_t prow = ((size_t)otok * a.n_q + oh) * a.part_slots + split;
    const float inv = inverse(ol);
#pragma unroll
    for (int c = 0; c < NC; c++) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; d++) store4(&o_s[wave][n][d * 16 + g * 4], scaled(w.acc[0][c * 4 + d], f));
        __syncthreads();
        f4 o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kFewWaves; i++) o += *reinterpret_cast<const f4 *>(&o_s[i][orow][od]);
        if (orow < rt.rows) {
            if (ks.parts == 1) {
                store4(static_cast<T *>(a.out) + (size_t)otok * a.out_stride + (size_t)oh * HD + c * 64 + od,
                       scaled(o, inv));
            } else {
                store4(a.part + prow * HD + c * 64 + od, scaled(o, 1.f));
                if (c == 0 && od == 0) a.part_ml[prow] = make_float2(om, ol);
            }
        }
    }
}

// Many rows: each wave has 16·NT rows of its own and walks all keys of its part.
constexpr int kManyWaves = 4;
template <typename T, int HD>
constexpr int many_tiles() {  // column tiles that the registers hold
    return HD == 128 ? 2 : HD == 256 ? (sizeof(T) == 2 ? 2 : 1) : 1;
}

template <typename T, int HD>
__global__ __launch_bounds__(kManyWaves * 64, HD < 512 ? 2 : 1) void paged_attn_many_kernel(AttnArgs a, int n_wgs) {
    constexpr int NT = many_tiles<T, HD>();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    // XCD = id % 8 takes heads congruent to it, so its L2 holds their pages; the
    // last tiles, which attend most keys, go first
    const int split = blockIdx.y % a.many_splits;
    const int head = blockIdx.x % a.pg.n_kv, wg = n_wgs - 1 - blockIdx.x / a.pg.n_kv;
    RowTile rt;
    if (!many_rows<NT * 16>(a, wg * kManyWaves + wave, &rt)) return;
    const KeySpan ks = key_span(a, rt, a.many_splits, a.many_per);
    if (split >= ks.parts) return;
    const int t0 = ks.t0 + split * ks.per, t1 = min(t0 + ks.per, ks.t1);
    Wave<T, HD, NT> w;
    w.load_q(a, rt, head, n, g);
    w.template attend<false>(a, rt, head, t0, t1, 1, lane);
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int row = rt.row0 + j * 16 + n;
        if (j * 16 + n >= rt.rows) continue;
        const int tok = rt.tok0 + row / a.group, qh = head * a.group + row % a.group;
        if (ks.parts == 1) {
            const float inv = inverse(w.l[j]);
            T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD + g * 4;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) store4(dst + d * 16, scaled(w.acc[j][d], inv));
        } else {
            const size_t prow = ((size_t)tok * a.n_q + qh) * a.part_slots + split;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) store4(a.part + prow * HD + d * 16 + g * 4, scaled(w.acc[j][d], 1.f));
            if (g == 0) a.part_ml[prow] = make_float2(w.M[j], w.l[j]);
        }
    }
}

// Joins the parts of a row tile's rows, in their order: a wave a row, its lanes
// first share out the parts' references and sums, then the dims.
template <typename T, int HD>
__device__ __forceinline__ void join_rows(const AttnArgs &a, const RowTile &rt, int head, int parts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = wave; i < rt.rows; i += 4) {
        const int r = rt.row0 + i;
        const int tok = rt.tok0 + r / a.group, qh = head * a.group + r % a.group;
        const size_t prow = ((size_t)tok * a.n_q + qh) * a.part_slots;
        float m = kNoMax, l = 0.f, o[HD / 64];
        for (int s = lane; s < parts; s += 64) m = fmaxf(m, a.part_ml[prow + s].x);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
#pragma unroll
        for (int d = 0; d < HD / 64; d++) o[d] = 0.f;
        for (int b = 0; b < parts; b += 64) {
            const float2 ml = b + lane < parts ? a.part_ml[prow + b + lane] : make_float2(kNoMax, 0.f);
            const float mine = __builtin_amdgcn_exp2f(ml.x - m), ls = ml.y * mine;
            const int e = min(parts - b, 64);
            for (int s = 0; s < e; s++) {
                const float f = lane_f(mine, s);
                l += lane_f(ls, s);
#pragma unroll
                for (int d = 0; d < HD / 64; d++)
                    o[d] = fmaf(a.part[(prow + b + s) * HD + d * 64 + lane], f, o[d]);
            }
        }
        const float inv = inverse(l);
        T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) dst[d * 64 + lane] = (T)(o[d] * inv);
    }
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_attn_join_few_kernel(AttnArgs a) {
    RowTile rt;
    if (!few_rows(a, blockIdx.x, &rt)) return;
    const KeySpan ks = key_span(a, rt, a.few_splits, a.few_per);
    if (ks.parts > 1) join_rows<T, HD>(a, rt, blockIdx.y, ks.parts);
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_attn_join_many_kernel(AttnArgs a) {
    RowTile rt;
    if (!many_rows<many_tiles<T, HD>() * 16>(a, blockIdx.x, &rt)) return;
    const KeySpan ks = key_span(a, rt, a.many_splits, a.many_per);
    if (ks.parts > 1) join_rows<T, HD>(a, rt, blockIdx.y, ks.parts);
}

// How a call is laid out: which kernels run, and into how many parts at most
// they cut the keys of a row.
constexpr int kFewWgs = 1024;
struct Layout {
    bool few, many;
    int few_splits, many_splits, many_wgs;
};

// Parts of 256 keys or more, so many that `units` workgroups of one part each
// become `wanted` of them.
int splits_for(long long units, long long wanted, int max_kv) {
    const long long by_fill = (wanted + units - 1) / units, by_keys = ((long long)max_kv + 255) / 256;
    const long long s = by_fill < by_keys ? by_fill : by_keys;
    return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

Layout layout(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim, bool f16, int max_new, int max_kv) {
    const int group = n_q / n_kv;
    Layout y{};
    // requests with many rows exist only if max_new says so; a lone request
    // needs one kernel
    y.many = (long long)max_new * group > kFewRows;
    y.few = !y.many || n_seqs > 1;
    y.few_splits = y.many_splits = 1;
    if (y.few) y.few_splits = splits_for((long long)n_seqs * n_kv, kFewWgs, max_kv);
    if (y.many) {
        const int bm = 16 * (head_dim == 128 ? 2 : head_dim == 256 ? (f16 ? 2 : 1) : 1);
        const long long tiles = (long long)n_tokens * group / bm + n_seqs;
        y.many_wgs = (int)((tiles + kManyWaves - 1) / kManyWaves);
        y.many_splits = splits_for((long long)y.many_wgs * n_kv, 512, max_kv);
    }
    return y;
}

template <typename T, int HD>
int launch(hipStream_t st, const AttnArgs &a, const Layout &y) {
    if (y.many) {
        hipLaunchKernelGGL((paged_attn_many_kernel<T, HD>), dim3(y.many_wgs * a.pg.n_kv, a.many_splits),
                           dim3(kManyWaves * 64), 0, st, a, y.many_wgs);
        SGQ_HIP(hipGetLastError());
    }
    if (y.few) {
        hipLaunchKernelGGL((paged_attn_few_kernel<T, HD>), dim3(a.n_seqs * a.few_splits * a.pg.n_kv),
                           dim3(kFewWaves * 64), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    if (y.many && a.many_splits > 1) {
        hipLaunchKernelGGL((paged_attn_join_many_kernel<T, HD>),
                           dim3(y.many_wgs * kManyWaves, a.pg.n_kv), dim3(256), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    if (y.few && a.few_splits > 1) {
        hipLaunchKernelGGL((paged_attn_join_few_kernel<T, HD>), dim3(a.n_seqs, a.pg.n_kv), dim3(256), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    return SGQ_OK;
}

}  // namespace

uint64_t paged_attn_workspace(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim, int max_new,
                              int max_kv) {
    // for rows of either type
    int s = 1;
    for (int f16 = 0; f16 < 2; f16++) {
        const Layout y = layout(n_tokens, n_seqs, n_q, n_kv, head_dim, f16, max_new, max_kv);
        s = std::max(s, std::max(y.few_splits, y.many_splits));
    }
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
    const int reach = p.window > 0 ? (int)std::min<long long>(p.max_kv, (long long)p.window + p.max_new) : p.max_kv;
    const Layout y = layout(p.n_tokens, p.n_seqs, p.n_q, p.pg.n_kv, p.pg.head_dim, p.f16, p.max_new, reach);
    const uint64_t row_bytes = (uint64_t)p.n_tokens * p.n_q * (p.pg.head_dim + 2) * 4;
    const uint64_t fit = std::max<uint64_t>(p.workspace ? p.workspace_bytes / row_bytes : 0, 1);
    a.few = y.few;
    a.few_splits = (int)std::min<uint64_t>(y.few_splits, fit);
    a.many_splits = (int)std::min<uint64_t>(y.many_splits, fit);
    const int tiles = std::max((int)(((long long)reach + 31) / 32), 1);
    a.few_per = std::max((tiles + a.few_splits - 1) / a.few_splits, 8);
    a.many_per = std::max((tiles + a.many_splits - 1) / a.many_splits, 8);
    a.part_slots = std::max(a.few_splits, a.many_splits);
    a.part = static_cast<float *>(p.workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part + (uint64_t)p.n_tokens * p.n_q * a.part_slots * p.pg.head_dim);
    switch (p.pg.head_dim * 2 + (p.f16 ? 1 : 0)) {
        case 128 * 2: return launch<float, 128>(st, a, y);
        case 128 * 2 + 1: return launch<_Float16, 128>(st, a, y);
        case 256 * 2: return launch<float, 256>(st, a, y);
        case 256 * 2 + 1: return launch<_Float16, 256>(st, a, y);
        case 512 * 2: return launch<float, 512>(st, a, y);
        case 512 * 2 + 1: return launch<_Float16, 512>(st, a, y);
    }
    return fail(SGQ_ERR_VALIDATION, "attn_paged_q8: head_dim %d unsupported (128, 256, 512)", p.pg.head_dim);
}

}  // namespace sgq
