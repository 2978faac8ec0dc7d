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
constexpr float kNoMax = -3.4e38f;    // the reference M before the first key: below any score
// M moves only when a tile's maximum is over it by this (log2); weights are
// taken against M - kHead, so f16 weights lie below 2^(kLazy + kHead) = 2^14
// and their subnormals begin 2^20 below M.  (Two prompts of 4001 rows: 335 us;
// with M moved at every larger score 389.)
constexpr float kLazy = 8.f, kHead = 6.f;
// V scales below this one weigh as it: an error below 127·2^-80 = 1.1e-22 in the output.
// The sum of w/vs then stays finite whatever the number of keys (2^14·2^80·2^31),
// also over blocks of zeros, and a weight that underflows (2^-126) has no more than
// 2^-52·vs of that sum, vs the scale of the largest weight's block.
constexpr float kMinScale = 0x1p-80f;

struct AttnArgs {
    PagedPages pg;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const int32_t *tables, *kv_lens, *cu;
    // the parts' sums [row][part][hd] and (M, l) [row][part]: rows (request, kv head, row)
    // of few rows, (cut tile and kv head, row of the tile) of many
    float *few_part, *many_part;
    float2 *few_ml, *many_ml;
    int max_pages, n_seqs, n_tokens, n_q, group, max_new, window;
    int few_splits, few_per;      // parts at most, of requests with few rows; their 32-key tiles, if
                                  // that makes no more of them
    int few_cap;                  // rows a request of few has at most
    int many_tiles, many_room;    // row tiles at most; parts that the workspace holds
    bool few;                     // requests with few rows go to their own kernel
    float scale_log2;
};

// A tile of query rows of one request and kv head: row r is token r/group of
// the request's new ones, query head head·group + r%group, at position
// pos0 + r/group.
struct RowTile {
    int seq, tok0, new_len, row0, rows, kv_len, pos0;
};

__device__ __forceinline__ int clamped(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Requests with at most kFewRows rows a kv head (single tokens) share a wave's
// 16 columns; their keys are what is spread over the GPU, and their quants go from
// memory to registers.  Through the kernel of many rows, whose waves share keys
// in LDS, 64 single tokens over up to 8192 keys take 624 us in place of 244.  Two kinds of
// single tokens go there all the same: those with more than 16 query heads a kv head
// (64 of 32 heads over up to 2000 keys: 32 us), and a lone request's where max_new
// announces more rows, as the keys are then cut for those (8191 keys of 128 dims 27 us,
// with max_new 1 12.7; 32768 of 512 dims 2061 and 37).
constexpr int kFewRows = 16;

__device__ __forceinline__ bool request_rows(const AttnArgs &a, int seq, RowTile *t) {
    const int c0 = clamped(a.cu[seq], 0, a.n_tokens);
    const int c1 = clamped(a.cu[seq + 1], c0, a.n_tokens);
    t->seq = seq;
    t->tok0 = c0;
    t->new_len = min(c1 - c0, a.max_new);
    t->kv_len = a.kv_lens[seq];
    // of the whole request, also where max_new or n_tokens cuts its rows off
    t->pos0 = t->kv_len - (a.cu[seq + 1] - a.cu[seq]);
    return t->new_len > 0;
}

// The rows of request `seq` when they are few.
__device__ __forceinline__ bool few_rows(const AttnArgs &a, int seq, RowTile *t) {
    if (!request_rows(a, seq, t) || t->new_len * a.group > kFewRows) return false;
    t->row0 = 0;
    t->rows = t->new_len * a.group;
    return true;
}

// 256 requests' tiles of BM rows, four requests a lane.
template <int BM>
struct ManyScan {
    int n[4], end;  // of each; of all up to this lane's last
    int reach;      // keys that a row tile attends at most
    __device__ __forceinline__ void load(const AttnArgs &a, int b) {
        const int lane = threadIdx.x & 63;
        int cu[5], kv[4];
#pragma unroll
        for (int k = 0; k < 5; k++) cu[k] = clamped(a.cu[min(b + lane * 4 + k, a.n_seqs)], 0, a.n_tokens);
#pragma unroll
        for (int k = 0; k < 4; k++) kv[k] = a.kv_lens[min(b + lane * 4 + k, a.n_seqs - 1)];
        end = reach = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int rows = min(max(cu[k + 1] - cu[k], 0), a.max_new) * a.group;
            n[k] = a.few && rows <= kFewRows ? 0 : (rows + BM - 1) / BM;
            end += n[k];
            const int wide = kv[k] - (BM - 1) / a.group;
            if (n[k]) reach = max(reach, a.window > 0 && wide > a.window ? kv[k] - wide + a.window : kv[k]);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(end, d);
            end += lane >= d ? o : 0;
        }
    }
};

// How a call's row tiles are launched: the last ones, which attend most keys, first.
// As many as fill the GPU a whole number of times (a workgroup a CU) stay whole; the
// keys of what is left are cut into `splits` parts of `per` 32-key tiles.  Every
// wave works it out from the lengths (a lane a number of parts): the host knows
// bounds only.
struct ManyPlan {
    int tiles, whole, splits, per;
};
constexpr int kCus = 256;
__host__ __device__ __forceinline__ int whole_tiles(int tiles, int n_kv) { return tiles * n_kv / kCus * kCus / n_kv; }

// The microseconds of `units` workgroups of `area` rows x dims with p parts of `per`
// tiles: a round costs its tiles, 1.3 each (1.1 to 2.1 measured), and four for its
// start; joining moves the parts twice, at 4 TB/s.
__host__ __device__ __forceinline__ float parts_cost(int units, int p, int per, int area) {
    return 1.3f * ((units * p + kCus - 1) / kCus) * (per + 4) + (p > 1 ? 5.f + 2e-6f * area * units * p : 0.f);
}

template <int BM, int HD>
__device__ __forceinline__ ManyPlan many_plan(const AttnArgs &a, ManyScan<BM> &scan) {
    ManyPlan m;
    m.tiles = 0;
    int reach = 0;
    for (int b = 0; b < a.n_seqs; b += 256) {
        scan.load(a, b);
        m.tiles += __builtin_amdgcn_readlane(scan.end, 63);
        reach = max(reach, scan.reach);
    }
    m.tiles = clamped(m.tiles, 0, a.many_tiles);
    m.whole = m.tiles, m.splits = 1, m.per = INT32_MAX;
    const int whole = whole_tiles(m.tiles, a.pg.n_kv), units = (m.tiles - whole) * a.pg.n_kv;
    if (a.many_room < 2 * units || units == 0) return m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) reach = max(reach, __shfl_xor(reach, d));
    const int p = (threadIdx.x & 63) + 1, keys = min(reach, a.max_pages << a.pg.page_log2) / 32 + 1;
    const int per = (keys + p - 1) / p;
    float us = parts_cost(units, p, per, BM * HD);
    if (p > 1 && (per < 4 || units * p > a.many_room)) us = INFINITY;
    float least = us;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
    const int best = __builtin_ctzll(__ballot(us == least));
    if (best == 0) return m;
    m.whole = whole, m.splits = best + 1, m.per = __builtin_amdgcn_readlane(per, best);
    return m;
}

// Tile `id` of the plan that `scan` was made for.
template <int BM>
__device__ __forceinline__ bool many_rows(const AttnArgs &a, ManyScan<BM> &scan, int id, RowTile *t) {
    int before = 0;
    for (int b = 0; b < a.n_seqs; b += 256) {
        if (a.n_seqs > 256) scan.load(a, b);
        if (const uint64_t past = __ballot(before + scan.end > id)) {
            int k = 0, first = before + scan.end - (scan.n[0] + scan.n[1] + scan.n[2] + scan.n[3]);
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (k == i && first + scan.n[i] <= id) first += scan.n[i], k++;
            const int owner = __builtin_ctzll(past);
            first = __builtin_amdgcn_readlane(first, owner);
            if (!request_rows(a, b + owner * 4 + __builtin_amdgcn_readlane(k, owner), t)) return false;
            t->row0 = (id - first) * BM;
            t->rows = min(t->new_len * a.group - t->row0, BM);
            return t->row0 >= 0 && t->rows > 0;
        }
        before += __builtin_amdgcn_readlane(scan.end, 63);
    }
    return false;
}

// Keys [lo, hi) of the query at position pos.
__device__ __forceinline__ int key_lo(const AttnArgs &a, int pos) {
    return a.window > 0 ? max(pos - a.window + 1, 0) : 0;
}
__device__ __forceinline__ int key_hi(const AttnArgs &a, int pos, int kv_len) {
    const int cap = a.max_pages << a.pg.page_log2;
    return clamped(min(pos + 1, kv_len), 0, cap);
}

// The positions of a row tile's first and last row.
__device__ __forceinline__ int first_pos(const AttnArgs &a, const RowTile &rt) {
    return rt.pos0 + rt.row0 / a.group;
}
__device__ __forceinline__ int last_pos(const AttnArgs &a, const RowTile &rt) {
    return rt.pos0 + (rt.row0 + rt.rows - 1) / a.group;
}

// Which 32-key tiles a row tile attends, and into how many parts of `per`
// tiles they are cut: parts of one length for all requests, so that a long one
// has more of them, unless that makes more than `splits`.
struct KeySpan {
    int t0, t1, parts, per;
};
__device__ __forceinline__ KeySpan key_span(const AttnArgs &a, const RowTile &rt, int splits, int per) {
    KeySpan k;
    k.t0 = key_lo(a, first_pos(a, rt)) >> 5;
    k.t1 = max((key_hi(a, last_pos(a, rt), rt.kv_len) + 31) >> 5, k.t0);
    const int n = k.t1 - k.t0;
    k.per = max(per, (n + splits - 1) / splits);
    k.parts = max((n + k.per - 1) / k.per, 1);
    return k;
}

// 8 quants (two words) as f16: byte u = q + 128 under the exponent of 1024
// makes 1024 + u exactly, minus 1152 is q.  (As the subnormal u·2^-24, with 128·Σq taken
// from the scores, 4 of the 10 operations go: 30 single tokens over up to 9000 keys of 512
// dims 174 us for 177, of other dims the same.  But where q has a mean and a block's quants
// are small beside an outlier, that term is far larger than the scores and takes their digits.)
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

template <bool STREAM, typename V>
__device__ __forceinline__ V load(const int8_t *p) {
    const V *v = reinterpret_cast<const V *>(p);
    return STREAM ? __builtin_nontemporal_load(v) : *v;
}

// The pages of 64 tiles and what their scales make of the scores: one tile a lane,
// read lane by lane.  LEAN keeps the V scale and takes its log2 and reciprocal tile by
// tile, a register less: with it single f16 tokens of 512 dims spill nothing in their loop
// (30 of up to 9000 keys 177 us, else 185).  The loop of many rows, bound by vector work, is
// faster without (2048 f16 rows of 512 dims 336 us, else 350).
template <bool LEAN>
struct TilePages {
    int page;            // 0 where there is none
    float ks, lv, rv;    // K scale; log2 and reciprocal of the V scale (LEAN: lv is the scale)
    // Lane i: tile t + i·step, if that is below t1.
    __device__ __forceinline__ void load(const AttnArgs &a, const int32_t *table, int head, int t, int step, int t1) {
        const int mine = t + (threadIdx.x & 63) * step;
        const int p = mine < t1 ? table[mine >> (a.pg.page_log2 - 5)] : -1;
        const bool ok = (unsigned)p < (unsigned)a.pg.n_pages;
        page = ok ? p : 0;
        const size_t b = (size_t)page * a.pg.n_kv + head;
        const float raw = a.pg.vs[b];
        const float vs = fmaxf(raw, kMinScale) + (raw - raw);  // NaN stays
        ks = ok ? a.pg.ks[b] : 0.f;
        if constexpr (LEAN) {
            lv = ok ? vs : 0.f;
        } else {
            lv = ok ? __builtin_amdgcn_logf(vs) : -INFINITY;  // no page: no weight
            rv = ok && vs == vs ? 1.f / vs : 1.f;             // finite: a masked key's 0·rv stays 0
        }
    }
    __device__ __forceinline__ void scales(int lane, float (&sc)[3]) const {
        sc[0] = lane_f(ks, lane);
        if constexpr (LEAN) {
            const float vs = lane_f(lv, lane);
            sc[1] = __builtin_amdgcn_logf(vs);                     // of 0: -infinity
            sc[2] = __builtin_amdgcn_rcpf(fmaxf(vs, kMinScale));  // of a NaN or 0: finite, as above
        } else {
            sc[1] = lane_f(lv, lane), sc[2] = lane_f(rv, lane);
        }
    }
};

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
    h8 (*ql_s)[64];  // fp32 rows of 512 dims, few: ql [fragment][lane] in LDS
    float row_scale[NT];  // of the scores, in log2 units
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
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) qa[i][c][h] = *reinterpret_cast<const h8 *>(src + c * 64 + h * 8);
            }
        }
    }

    // The weights w (fp32 rows: w + wl) of K tiles from t on from their scores, with l,
    // and with M and acc where the reference has to move.  edge: some row does not
    // attend all keys; keys from key_end on are not this part's.  sc: each tile's K
    // scale, log2 and reciprocal of its V scale.
    template <int K>
    __device__ __forceinline__ void weigh(const AttnArgs &a, const RowTile &rt, int t, bool edge, int key_end,
                                          const float (&sc)[K][3], const f4 (&s)[K][NT][2], h8 (&w)[K][NT],
                                          h8 (&wl)[K][F32 ? NT : 1], int n, int g) {
        float x[K][NT][8], mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float c = row_scale[j] * sc[k][0];
                const float b = sc[k][1] + (kHead - M[j]);
#pragma unroll
                for (int e = 0; e < 8; e++) x[k][j][e] = fmaf(s[k][j][e >> 2][e & 3], c, b);
            }
        if (edge) {
            asm volatile("");  // a branch: as selects the masks would be half of the loop's VALU work
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int row = rt.row0 + min(j * 16 + n, rt.rows - 1);
                const int pos = rt.pos0 + row / a.group;
                const int lo = key_lo(a, pos), hi = min(key_hi(a, pos, rt.kv_len), key_end);
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int key = (t + k) * 32 + g * 8 + e;
                        x[k][j][e] = key >= lo && key < hi ? x[k][j][e] : -INFINITY;
                    }
            }
        }
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, x[k][j][e]);
        if (__any(mx > kLazy + kHead)) {
            // a larger reference: from the scores again, as x may hold them against none
#pragma unroll
            for (int j = 0; j < NT; j++) {
                float m = -INFINITY;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const float c = row_scale[j] * sc[k][0], b = sc[k][1];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        m = fmaxf(m, x[k][j][e] == -INFINITY ? x[k][j][e] : fmaf(s[k][j][e >> 2][e & 3], c, b));
                }
                const float m1 = fmaxf(M[j], fmax16(m)), f = __builtin_amdgcn_exp2f(M[j] - m1);
                M[j] = m1;
                l[j] *= f;
#pragma unroll
                for (int d = 0; d < ND; d++) acc[j][d] *= f;
                // the rounded scores against M, so that its own key is at kHead: in the FMA
                // M's rounding would remain, which for scores past 2^27 is more than an f16
                // weight holds
#pragma unroll
                for (int k = 0; k < K; k++) {
                    const float c = row_scale[j] * sc[k][0], b = sc[k][1];
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        x[k][j][e] = x[k][j][e] == -INFINITY ? x[k][j][e] : fmaf(s[k][j][e >> 2][e & 3], c, b) - m1 + kHead;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p = __builtin_amdgcn_exp2f(x[k][j][e]);
                    sum += p;  // not the f16 weight: over a block of small V scale that may be 0
                    w[k][j][e] = (_Float16)p;
                    if constexpr (F32) wl[k][j][e] = (_Float16)(p - (float)w[k][j][e]);
                }
                l[j] = fmaf(sum, sc[k][2], l[j]);
            }
    }

    // The four lanes of a row have the same M; its l is their sum.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            l[j] += __shfl_xor(l[j], 16);
            l[j] += __shfl_xor(l[j], 32);
        }
    }

    // Tiles t0, t0 + step, ... below t1.  STREAM: no other wave reads these pages
    // soon, so they are not kept in the caches (64 requests of up to 8192 keys, 16 heads
    // of 128: 243 us, kept 256; one of 32768: 29 and 33).  Not at 512 dims, where that
    // is the slower way for all but a lone request (4 heads: 12 requests of up to 32768 207 us,
    // kept 192; 30 of up to 9000 187 and 174; 40 of up to 1000 52.5 and 50.5; 7 of up to
    // 9000 47.5 and 46.9; one of 32768 37.1 and 39.7).
    template <bool STREAM>
    __device__ __forceinline__ void attend(const AttnArgs &a, const RowTile &rt, int head, int t0, int t1,
                                           int step, int lane) {
        const int n = lane & 15, g = lane >> 4;
        // tiles inside [all_lo, all_hi] need no mask
        const int all_lo = key_lo(a, last_pos(a, rt)), all_hi = key_hi(a, first_pos(a, rt), rt.kv_len);
        const int32_t *table = a.tables + (size_t)rt.seq * a.max_pages;
        const int lg = a.pg.page_log2;
        TilePages<HD == 512> pages;
        const size_t lane_k = (size_t)((n >> 2) * 8 + (n & 3)) * HD + g * 16;
        const size_t lane_v = n * 32 + g * 8;
        const auto block = [&](int t, int i) {  // the quants of tile t, the wave's i-th
            const int page = __builtin_amdgcn_readlane(pages.page, i % 64);
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
        pages.load(a, table, head, t0, step, t1);
        size_t blk = block(t0, 0);
        load_k(blk);
        // One tile.  Its V and then the next tile's K are on their way while it is
        // worked on; the last tile has a copy of this code without that K, as a
        // load under a condition would be waited for at once.
        const auto low = [&](int j, int c, int e) {
            if constexpr (F32 && HD == 512) return ql_s[c * 2 + e][lane];
            else return ql[j][c][e];
        };
        const auto tile = [&](int i, int t, auto more) {
            float sc[1][3];
            pages.scales(i % 64, sc[0]);
            const int8_t *vp = a.pg.vq + blk + lane_v;
#pragma unroll
            for (int d = 0; d < ND; d++) vr[d] = load<STREAM, u2>(vp + d * 16 * 32);
            f4 sk[1][NT][2], (&s)[NT][2] = sk[0];
#pragma unroll
            for (int j = 0; j < NT; j++) s[j][0] = s[j][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const h8 k0 = quants_f16(kr[c][h].x, kr[c][h].y), k1 = quants_f16(kr[c][h].z, kr[c][h].w);
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qa[j][c][0], s[j][h], 0, 0, 0);
                        if constexpr (F32)
                            s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, low(j, c, 0), s[j][h], 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qa[j][c][1], s[j][h], 0, 0, 0);
                        if constexpr (F32)
                            s[j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, low(j, c, 1), s[j][h], 0, 0, 0);
                    }
                }
            if constexpr (decltype(more)::value) {
                if (i % 64 == 63) pages.load(a, table, head, t + step, step, t1);
                blk = block(t + step, i + 1);
                load_k(blk);
            }
            h8 wk[1][NT], wlk[1][F32 ? NT : 1], (&w)[NT] = wk[0], (&wl)[F32 ? NT : 1] = wlk[0];
            weigh<1>(a, rt, t, t * 32 < all_lo || t * 32 + 32 > all_hi, INT32_MAX, sc, sk, wk, wlk, n, g);
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
        finish();
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

// A row's place in the workspace.
__device__ __forceinline__ size_t few_row(const AttnArgs &a, const RowTile &rt, int head, int i) {
    return ((size_t)rt.seq * a.pg.n_kv + head) * a.few_cap + i;
}

// Few rows: one request and kv head against one part of the keys, the tiles dealt
// to 4 waves in turn and their sums joined in LDS in wave order.  Bound by reading
// the pages: 64 single tokens over up to 8192 keys (16 heads of 128, f16) 244 us,
// 5.5 TB/s; 12 over up to 32768 (4 heads of 512) 184 us, 5.6 TB/s; one over 8191
// (fp32) 13 us with the join, of which the launches and the latency of the first loads
// are 8.
constexpr int kFewWaves = 4;

template <typename T, int HD>
__global__ __launch_bounds__(kFewWaves * 64, HD == 128 ? 3 : HD == 256 ? 2 : 1) void paged_attn_few_kernel(AttnArgs a) {
    // dims that the waves' sums meet in LDS at a time: few barriers, and room for the
    // workgroups that a CU's registers hold
    constexpr int CW = HD == 512 ? 256 : 128;
    __shared__ float ml_s[kFewWaves][2][16];
    __shared__ __align__(16) float o_s[kFewWaves][16][CW + 4];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    // 512 dims: in a scalar register, and so are its tiles and their addresses (30 f16 tokens
    // of up to 9000 keys 177 us, else 181; 200 of 2000 of 128 dims 187, else 184)
    const int wave = HD == 512 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : threadIdx.x >> 6;
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
    if constexpr (Wave<T, HD, 1>::F32 && HD == 512) {
        // both halves of q, the accumulator and a tile on its way are more registers than
        // a wave has (84 spilled): the waves' common low half from LDS, 174 -> 119 us
        // for 16 requests of 8192 keys
        constexpr int NC = HD / 64;
        __shared__ h8 ql_s[NC * 2][64];
        if (wave == 0)
#pragma unroll
            for (int c = 0; c < NC; c++) ql_s[c * 2][lane] = w.ql[0][c][0], ql_s[c * 2 + 1][lane] = w.ql[0][c][1];
        __syncthreads();
        w.ql_s = ql_s;
    }
    w.template attend<HD != 512>(a, rt, head, t0 + wave, t1, kFewWaves, lane);
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
    const size_t prow = few_row(a, rt, head, orow) * a.few_splits + split;
    const float inv = inverse(ol);
#pragma unroll
    for (int c = 0; c < HD / CW; c++) {
        if (c) __syncthreads();
#pragma unroll
        for (int d = 0; d < CW / 16; d++)
            store4(&o_s[wave][n][d * 16 + g * 4], scaled(w.acc[0][c * (CW / 16) + d], f));
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CW; k += 64) {
            if (orow >= rt.rows) break;
            f4 o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kFewWaves; i++) o += *reinterpret_cast<const f4 *>(&o_s[i][orow][k + od]);
            const int dim = c * CW + k + od;
            if (ks.parts == 1) {
                store4(static_cast<T *>(a.out) + (size_t)otok * a.out_stride + (size_t)oh * HD + dim, scaled(o, inv));
            } else {
                store4(a.few_part + prow * HD + dim, scaled(o, 1.f));
                if (dim == 0) a.few_ml[prow] = make_float2(om, ol);
            }
        }
    }
}

// Many rows: a workgroup's waves have 16·NT rows each and share the keys.  A step
// of kStep 32-key tiles is turned into f16 once, by all waves, into LDS.
// The two waves of a SIMD take turns: while one multiplies (the last step's P·V,
// then this step's Q·K, with the conversion of its share of the next quants in
// the products' shadow) the other weighs its scores, with a barrier at each
// change, so that the matrix cores and the vector units both have work all the
// time.  Phase 2t+w is the multiplication of step t for waves of group w = 0, 1,
// phase 2t+1+w their weighing.  K(t+1) and V(t) are stored in the phases 2t and
// 2t+1: complete before phase 2t+2, which reads them first, and over K(t-1) and
// V(t-2), which phase 2t-1 read last, so two buffers of each do.
//   K [key][HD]: the 16-byte units of a row are stored at unit ^ swizzle(key), so
//                that the 16 keys of a fragment read fall on different banks
//   V [tile][dim][32 keys]: a fragment is one kilobyte, its four units of a dim
//                likewise exchanged (2048 rows of 256 dims: 113 us, else 120)
// The products of f16 rows of 128 dims have 32 rows a wave, at half the LDS reads
// of 16 (two prompts of 4001 rows: 335 us and 440), four reads ahead (two: 356); wider
// rows' accumulators leave no room for that.  Bound by LDS reads and the
// scores' vector work beside the products.  In TFLOP/s, f16: two prompts of 4001 rows of 128
// dims 820, 2048 rows of 256 dims 600 and of 512 dims 411 (there each wave of 16 rows reads
// all of K and V from LDS, and the one wave of a SIMD weighs alone).  fp32, at two
// products each: 2048 rows of 128 dims 353 (706 done), 1111 of 256 dims with a window
// 320 (640), 1024 of 512 dims over 2048 keys 342 (684).
template <typename T, int HD>
struct Many {
    static constexpr bool F32 = sizeof(T) == 4;
    // the accumulator (64·NT·HD/128 registers) and q bound the rows of a wave
    static constexpr int NT = HD == 128 && !F32 ? 2 : 1;
    static constexpr int kWaves = HD == 512 ? 4 : 8;  // 512 dims take the registers of two
    static constexpr int kRows = kWaves * NT * 16;
    static constexpr int kStep = HD == 128 ? 2 : 1;
    static constexpr int kThreads = kWaves * 64;
    static constexpr int kGroups = kWaves / 4;
    static constexpr int kLoads = kStep * 2 * HD / kThreads;  // 16-byte loads a thread, for K and for V
    static_assert(kLoads * kThreads == kStep * 2 * HD && 2 * HD % 64 == 0, "whole waves load a tile");
    static constexpr int kFrags = kStep * HD / 16;  // fragments of a step's K, and of its V
    static constexpr int kAhead = 4;                // fragment reads under way
    struct Lds {
        h8 k[2][kStep][32][HD / 8];
        h8 v[2][kStep][HD][4];
    };
    static __device__ __forceinline__ int swizzle_v(int dim) { return -(dim >> 2) & 3; }
    static __device__ __forceinline__ int swizzle(int key) { return (key & 3) | (key >> 3 & 3) << 2; }
};

template <typename T, int HD>
__global__ __launch_bounds__((Many<T, HD>::kThreads), (Many<T, HD>::kWaves / 4)) void paged_attn_many_kernel(AttnArgs a) {
    using C = Many<T, HD>;
    constexpr int NT = C::NT, KT = C::kStep;
    __shared__ __align__(16) typename C::Lds lds;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    // in a scalar register: what follows from it, barriers among it, branches for the
    // whole wave
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCD = id % 8 takes heads congruent to it, so its L2 holds their pages
    ManyScan<C::kRows> scan;
    const ManyPlan plan = many_plan<C::kRows, HD>(a, scan);
    const int n_whole = plan.whole * a.pg.n_kv, n_cut = (plan.tiles - plan.whole) * a.pg.n_kv;
    const bool whole = (int)blockIdx.x < n_whole;
    if (!whole && (int)blockIdx.x - n_whole >= n_cut * plan.splits) return;
    const int unit = whole ? blockIdx.x : (blockIdx.x - n_whole) % n_cut;
    const int split = whole ? 0 : (blockIdx.x - n_whole) / n_cut;
    const int head = unit % a.pg.n_kv, rank = unit / a.pg.n_kv + (whole ? 0 : plan.whole);
    RowTile rt;
    if (!many_rows(a, scan, plan.tiles - 1 - rank, &rt)) return;
    const KeySpan ks = key_span(a, rt, whole ? 1 : plan.splits, whole ? 1 : plan.per);
    if (split >= ks.parts) return;
    const int t0 = ks.t0 + split * ks.per, t1 = min(t0 + ks.per, ks.t1);

    // this wave's rows
    RowTile wt = rt;
    const bool idle = wave * NT * 16 >= rt.rows;
    wt.row0 = rt.row0 + (idle ? 0 : wave * NT * 16);
    wt.rows = idle ? 1 : min(rt.rows - wave * NT * 16, NT * 16);
    const int all_lo = key_lo(a, last_pos(a, wt)), all_hi = min(key_hi(a, first_pos(a, wt), rt.kv_len), t1 * 32);
    Wave<T, HD, NT> w;
    w.load_q(a, wt, head, n, g);

    const int32_t *table = a.tables + (size_t)rt.seq * a.max_pages;
    const int lg = a.pg.page_log2 - 5;  // tiles of a page, log2
    // What this wave loads of a step: kLoads pieces of K and V, each of one tile.
    u4 kr[C::kLoads], vr[C::kLoads];
    int page_k[C::kLoads], page_v[C::kLoads];
    const auto tile_of = [&](int step, int p) {  // past the end: the last one again, unused
        return min(t0 + step * KT + (p * C::kThreads + wave * 64) / (2 * HD), t1 - 1);
    };
    int pages[C::kLoads];  // of 64 steps: one a lane
    // Steps are looked up one after another.
    const auto look_up = [&](int step, int (&page)[C::kLoads]) {
        if ((step & 63) == 0) {
#pragma unroll
            for (int p = 0; p < C::kLoads; p++) {
                const int v = table[tile_of(step + lane, p) >> lg];
                pages[p] = (unsigned)v < (unsigned)a.pg.n_pages ? v : 0;  // none: any, as it weighs nothing
            }
        }
#pragma unroll
        for (int p = 0; p < C::kLoads; p++) page[p] = __builtin_amdgcn_readlane(pages[p], step & 63);
    };
    const auto quants_at = [&](int step, int p, int page) {
        return ((((size_t)page * a.pg.n_kv + head) << lg) + (tile_of(step, p) & ((1 << lg) - 1))) * (32 * HD) +
               (size_t)((p * C::kThreads + tid) % (2 * HD)) * 16;
    };
    const auto load_k = [&](int step) {
#pragma unroll
        for (int p = 0; p < C::kLoads; p++)
            kr[p] = *reinterpret_cast<const u4 *>(a.pg.kq + quants_at(step, p, page_k[p]));
    };
    const auto load_v = [&](int step) {
#pragma unroll
        for (int p = 0; p < C::kLoads; p++)
            vr[p] = *reinterpret_cast<const u4 *>(a.pg.vq + quants_at(step, p, page_v[p]));
    };
    // Piece i of the conversion: 8 quants of K(step + 1) or V(step) into LDS.
    const auto convert = [&](int step, int i) {
        const int p = i / 4, half = i & 1;
        const int at = p * C::kThreads + tid, tile = at / (2 * HD), u = at % (2 * HD);
        if ((i & 2) == 0) {
            const int key = u / (HD / 16), c = u % (HD / 16) * 2 + half;  // 16 dims of a key
            lds.k[(step + 1) & 1][tile][key][c ^ C::swizzle(key)] =
                half ? quants_f16(kr[p].z, kr[p].w) : quants_f16(kr[p].x, kr[p].y);
        } else {
            const int dim = u / 2, c = u % 2 * 2 + half;  // 16 keys of a dim
            lds.v[step & 1][tile][dim][c ^ C::swizzle_v(dim)] =
                half ? quants_f16(vr[p].z, vr[p].w) : quants_f16(vr[p].x, vr[p].y);
        }
    };
    h8 hi[KT][NT], lo[KT][C::F32 ? NT : 1];  // the last weighed step's weights
    f4 s[KT][NT][2];                         // the last multiplied step's scores
    // Fragment i of V(step): tile i / (HD/16), dims i % (HD/16).
    const auto read_v = [&](int step, int i) {
        return lds.v[step & 1][i / (HD / 16)][i % (HD / 16) * 16 + n][g ^ C::swizzle_v(n)];
    };
    const auto multiply_v = [&](int i, h8 f) {
        const int k = i / (HD / 16), d = i % (HD / 16);
#pragma unroll
        for (int j = 0; j < NT; j++) {
            w.acc[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, hi[k][j], w.acc[j][d], 0, 0, 0);
            if constexpr (C::F32)
                w.acc[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, lo[k][j], w.acc[j][d], 0, 0, 0);
        }
    };
    // Fragment i of K(step): half h of tile k against 32 dims, the dims outermost so that
    // products of one sum lie apart.
    const auto read_k = [&](int step, int i) {
        const int h = i % 2, k = i / 2 % KT, ce = i / 2 / KT;
        // swizzle(key) is n; the units it exchanges lie within 16
        const int key = (n >> 2) * 8 + h * 4 + (n & 3), in16 = ce / 2 % 2 * 8 + g * 2 + ce % 2;
        return lds.k[step & 1][k][key][ce / 4 * 16 + (in16 ^ n)];
    };
    const auto multiply_k = [&](int i, h8 f) {
        const int h = i % 2, k = i / 2 % KT, ce = i / 2 / KT;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const f4 sum = ce == 0 ? f4{0.f, 0.f, 0.f, 0.f} : s[k][j][h];
            s[k][j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, w.qa[j][ce / 2][ce % 2], sum, 0, 0, 0);
            if constexpr (C::F32)
                s[k][j][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, w.ql[j][ce / 2][ce % 2], s[k][j][h], 0, 0, 0);
        }
    };
    const auto load_next = [&](int t) {
        load_k(t + 3);
        load_v(t + 2);
#pragma unroll
        for (int p = 0; p < C::kLoads; p++) page_v[p] = page_k[p];
        look_up(t + 4, page_k);
    };
    // A phase of products: P(t)·V(t) when there is one, Q·K(t+1), with the pieces of the
    // conversion after it spread among them.  The order is as written (the
    // sched_barriers): left alone the compiler waits for each fragment at once, for
    // longer than its products take.
    const auto multiply = [&](int t, auto with_v) {
        constexpr int NV = decltype(with_v)::value ? C::kFrags : 0, N = NV + C::kFrags, A = C::kAhead;
        constexpr int kPieces = C::kLoads * 4, kEvery = C::kFrags / kPieces;
        const auto read = [&](int i) { return i < NV ? read_v(t, i) : read_k(t + 1, i - NV); };
        h8 f[A];
#pragma unroll
        for (int i = 0; i < A; i++) f[i] = read(i);
#pragma unroll
        for (int i = 0; i < N; i++) {
            __builtin_amdgcn_sched_barrier(0);
            if (i < NV) multiply_v(i, f[i % A]);
            else multiply_k(i - NV, f[i % A]);
            if (i + A < N) f[i % A] = read(i + A);
            // in the last products' shadow: the quants have had the longest time to come
            if (i >= N - C::kFrags && (i - (N - C::kFrags)) % kEvery == kEvery - 1)
                convert(t + 1, (i - (N - C::kFrags)) / kEvery);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_next(t);
    };
    const int steps = (t1 - t0 + KT - 1) / KT, group = wave / 4;
    if (steps > 0) {
        look_up(0, page_k);
        load_k(0);
#pragma unroll
        for (int p = 0; p < C::kLoads; p++) {
            convert(-1, p * 4);
            convert(-1, p * 4 + 1);
        }
#pragma unroll
        for (int p = 0; p < C::kLoads; p++) page_v[p] = page_k[p];
        look_up(1, page_k);
        load_k(1);
        load_v(0);
        // registers: K(1), V(0)
#pragma unroll
        for (int p = 0; p < C::kLoads; p++) page_v[p] = page_k[p];
        look_up(2, page_k);
        __syncthreads();
        if (group == 1) __syncthreads();
        multiply(-1, std::false_type{});
        __syncthreads();
    }
    if (idle) {  // no rows: only its share of the conversion, at the same barriers
        for (int t = 0; t < steps; t++) {
            const bool more = t + 1 < steps;
            if (group == 0 || more) __syncthreads();
#pragma unroll
            for (int i = 0; i < C::kLoads * 4; i++) convert(t + 1, i);
            load_next(t);
            if (more) __syncthreads();
        }
        return;
    }
    TilePages<false> tiles;
    // Steps that a wave's rows do not reach weigh nothing, like the copies past the end.
    for (int t = 0; t < steps; t++) {
        const int at = t0 + t * KT, turn = t * KT % 64;
        if (turn == 0) tiles.load(a, table, head, at, 1, t1);
        float sc[KT][3];
#pragma unroll
        for (int k = 0; k < KT; k++) tiles.scales(turn + k, sc[k]);
        w.template weigh<KT>(a, wt, at, at * 32 < all_lo || (at + KT) * 32 > all_hi, t1 * 32, sc, s, hi, lo, n, g);
        const bool more = t + 1 < steps;
        if (group == 0 || more) __syncthreads();
        multiply(t, std::true_type{});
        if (more) __syncthreads();
    }
    w.finish();
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int row = wt.row0 + j * 16 + n;
        if (j * 16 + n >= wt.rows) continue;
        const int tok = rt.tok0 + row / a.group, qh = head * a.group + row % a.group;
        if (ks.parts == 1) {
            const float inv = inverse(w.l[j]);
            T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD + g * 4;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) store4(dst + d * 16, scaled(w.acc[j][d], inv));
        } else {
            const size_t prow = ((size_t)unit * C::kRows + row - rt.row0) * plan.splits + split;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) store4(a.many_part + prow * HD + d * 16 + g * 4, scaled(w.acc[j][d], 1.f));
            if (g == 0) a.many_ml[prow] = make_float2(w.M[j], w.l[j]);
        }
    }
}

// Joins the parts of a row: its W waves take every W-th part, four of them in flight,
// and are summed in wave order.  The lanes share out the parts' references and
// sums, then the dims.
constexpr int kJoinWaves = 4;
template <typename T, int HD>
__device__ __forceinline__ void join_row(const AttnArgs &a, const RowTile &rt, int head, int i, int parts,
                                         const float *part, const float2 *part_ml, size_t prow) {
    constexpr int ND = HD / 64, W = kJoinWaves;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = rt.row0 + i, tok = rt.tok0 + r / a.group, qh = head * a.group + r % a.group;
    float m = kNoMax, l = 0.f, o[ND];
    for (int s = lane; s < parts; s += 64) m = fmaxf(m, part_ml[prow + s].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = 0.f;
    for (int b = wave; b < parts; b += 64 * W) {  // lane j: part b + j·W
        const int mine = b + lane * W;
        const float2 ml = mine < parts ? part_ml[prow + mine] : make_float2(kNoMax, 0.f);
        const float f = mine < parts ? __builtin_amdgcn_exp2f(ml.x - m) : 0.f, ls = ml.y * f;
        const int e = min((parts - b + W - 1) / W, 64);
        for (int s = 0; s < e; s += 4) {
            float v[4][ND];
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int d = 0; d < ND; d++) v[k][d] = part[(prow + b + min(s + k, e - 1) * W) * HD + d * 64 + lane];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (s + k >= e) break;
                const float fk = lane_f(f, s + k);
                l += lane_f(ls, s + k);
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] = fmaf(v[k][d], fk, o[d]);
            }
        }
    }
    T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD;
    static_assert(W == 4, "the sums below");
    __shared__ float o_s[W][HD], l_s[W];
#pragma unroll
    for (int d = 0; d < ND; d++) o_s[wave][d * 64 + lane] = o[d];
    if (lane == 0) l_s[wave] = l;
    __syncthreads();
    const float inv = inverse(l_s[0] + l_s[1] + l_s[2] + l_s[3]);
    for (int d = threadIdx.x; d < HD; d += W * 64)
        dst[d] = (T)((o_s[0][d] + o_s[1][d] + o_s[2][d] + o_s[3][d]) * inv);
}

// Row i0 + lane/L of a cut tile, L lanes a row (two rows a wave at 128 dims, in flight
// together): all parts, four at a time.
template <typename T, int HD>
struct ManyJoin {
    static constexpr int L = HD / 4 < 64 ? HD / 4 : 64, kRows = 64 / L, NV = HD / 4 / L;
    static __device__ __forceinline__ void rows(const AttnArgs &a, const RowTile &rt, int head, int i0, int parts,
                                                const float *part, const float2 *part_ml, size_t prow0, int splits) {
        const int lane = threadIdx.x & 63, c = lane % L, i = i0 + lane / L;
        const bool live = i < rt.rows;
        const size_t prow = prow0 + (size_t)(live ? lane / L : 0) * splits;
        float m = kNoMax, l = 0.f;
        for (int s = 0; s < parts; s += 4)
#pragma unroll
            for (int k = 0; k < 4; k++) m = fmaxf(m, part_ml[prow + min(s + k, parts - 1)].x);
        f4 o[NV] = {};
        for (int s = 0; s < parts; s += 4) {
            f4 v[4][NV];
            float2 ml[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const size_t p = prow + min(s + k, parts - 1);
                ml[k] = part_ml[p];
#pragma unroll
                for (int d = 0; d < NV; d++) v[k][d] = *reinterpret_cast<const f4 *>(part + p * HD + (d * L + c) * 4);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float f = s + k < parts ? __builtin_amdgcn_exp2f(ml[k].x - m) : 0.f;
                l = s + k < parts ? fmaf(ml[k].y, f, l) : l;
#pragma unroll
                for (int d = 0; d < NV; d++) o[d] = s + k < parts ? o[d] + v[k][d] * f : o[d];
            }
        }
        if (!live) return;
        const int r = rt.row0 + i, tok = rt.tok0 + r / a.group, qh = head * a.group + r % a.group;
        T *dst = static_cast<T *>(a.out) + (size_t)tok * a.out_stride + (size_t)qh * HD;
        const float inv = inverse(l);
#pragma unroll
        for (int d = 0; d < NV; d++) store4(dst + (d * L + c) * 4, scaled(o[d], inv));
    }
};

// Many rows have few parts: the waves of n_many workgroups take them in turn.  Few
// rows have many: a workgroup a row of a single token.
template <typename T, int HD, bool MANY>
__global__ __launch_bounds__(kJoinWaves * 64) void paged_attn_join_kernel(AttnArgs a, int n_many) {
    RowTile rt;
    if (!MANY || (int)blockIdx.x >= n_many) {
        const int each = MANY ? min(a.group, a.few_cap) : gridDim.z, id = blockIdx.x - n_many;
        const int head = MANY ? id / each % a.pg.n_kv : blockIdx.y, seq = MANY ? id / each / a.pg.n_kv : blockIdx.x;
        int i = MANY ? id % each : blockIdx.z;
        if (!few_rows(a, seq, &rt)) return;
        const KeySpan ks = key_span(a, rt, a.few_splits, a.few_per);
        if (ks.parts == 1 || i >= rt.rows) return;
        for (;;) {
            join_row<T, HD>(a, rt, head, i, ks.parts, a.few_part, a.few_ml,
                            few_row(a, rt, head, i) * a.few_splits);
            i += each;
            if (i >= rt.rows) break;
            __syncthreads();  // its LDS is read
        }
        return;
    }
    constexpr int BM = Many<T, HD>::kRows;
    ManyScan<BM> scan;
    const ManyPlan plan = many_plan<BM, HD>(a, scan);
    const int units = (plan.tiles - plan.whole) * a.pg.n_kv;
    using J = ManyJoin<T, HD>;
    const int first = (blockIdx.x * kJoinWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * J::kRows;
    for (int w = first; w < units * BM; w += n_many * kJoinWaves * J::kRows) {
        const int unit = w / BM, i = w % BM, head = unit % a.pg.n_kv;
        if (!many_rows(a, scan, plan.tiles - 1 - plan.whole - unit / a.pg.n_kv, &rt) || i >= rt.rows) continue;
        const KeySpan ks = key_span(a, rt, plan.splits, plan.per);
        if (ks.parts > 1)
            J::rows(a, rt, head, i, ks.parts, a.many_part, a.many_ml, (size_t)w * plan.splits, plan.splits);
    }
}

// How a call is laid out: which kernels run, and into how many parts at most
// they cut the keys of a row.
int few_cap(int max_new, int group) { return (int)std::min<long long>((long long)max_new * group, kFewRows); }
// Parts of many rows, together: two rounds (768 rows over 16384 keys, 96 workgroups
// uncut: 305 us with parts for one round, 282 for two, 283 for three).
constexpr int kManyParts = 2 * kCus;
constexpr int kJoinWgs = 8 * kCus;  // of many rows: as many as fit
struct Layout {
    bool few, many;
    int few_splits, many_tiles, many_parts;
    uint64_t few_rows;  // that may be cut
    int many_bm;        // rows of a tile
};

// Parts of 256 keys or more of a request with few rows.  One workgroup a CU when that
// comes out even: each then reads long runs, and one a CU draws the whole
// bandwidth (one request of 32768 keys, 16 heads of 128, fp32: 29 us with 256 of them, 33
// with 1024; 16 of 4096: 39 and 44).  Otherwise four a CU, as requests differ in
// length and what is left over weighs less (6 requests of 6000: 41 and 28);
// at 512 dims a CU has room for one, and more only queue (16 fp32 of 8192: 90 and 119).
int splits_for(int units, int head_dim, int max_kv) {
    const bool even = kCus % units == 0 || units % kCus == 0;
    const int by_fill = ((even || head_dim == 512 ? kCus : 4 * kCus) + units - 1) / units;
    const int by_keys = (int)(((long long)max_kv + 255) / 256);
    return std::clamp(by_fill, 1, std::max(by_keys, 1));
}

// Into how many parts `units` workgroups over `keys` 32-key tiles are best cut.
int best_parts(int units, int keys, int area) {
    int best = 1;
    float least = parts_cost(units, 1, keys, area);
    for (int p = 2; p <= 64 && keys / p >= 4 && units * p <= kManyParts; p++) {
        const float us = parts_cost(units, p, (keys + p - 1) / p, area);
        if (us < least) least = us, best = p;
    }
    return units ? best : 1;
}

Layout layout(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim, bool f16, int max_new, int max_kv) {
    const int group = n_q / n_kv;
    Layout y{};
    // requests with many rows exist only if max_new says so, with few only if a token's
    // heads are few; a lone request needs one kernel
    y.many = (long long)max_new * group > kFewRows;
    y.few = !y.many || (n_seqs > 1 && group <= kFewRows);
    y.few_splits = 1;
    y.many_bm = 1;
    if (y.few) {
        y.few_splits = splits_for(n_seqs * n_kv, head_dim, max_kv);
        y.few_rows = (uint64_t)n_seqs * n_kv * few_cap(max_new, group);
    }
    if (y.many) {
        y.many_bm = head_dim == 128   ? (f16 ? Many<_Float16, 128>::kRows : Many<float, 128>::kRows)
                    : head_dim == 256 ? (f16 ? Many<_Float16, 256>::kRows : Many<float, 256>::kRows)
                                      : (f16 ? Many<_Float16, 512>::kRows : Many<float, 512>::kRows);
        // a request with many rows has more than kFewRows (alone it has any number), and a
        // last tile that is not full
        const int last = n_seqs > 1 ? (int)std::min<long long>(n_seqs, (long long)n_tokens * group / (kFewRows + 1)) : 1;
        y.many_tiles = (int)((long long)n_tokens * group / y.many_bm) + std::max(last, 1);
        // The remainder of a lone request is known, and so are its parts.  Of several it
        // is n_kv at least: no room (and no join) where even that is not worth a cut.
        const int tiles = (int)(((long long)n_tokens * group + y.many_bm - 1) / y.many_bm);
        const int units = n_seqs == 1 ? (tiles - whole_tiles(tiles, n_kv)) * n_kv : n_kv;
        const int cut = best_parts(units, max_kv / 32 + 1, y.many_bm * head_dim);
        if (cut > 1) y.many_parts = n_seqs == 1 ? units * cut : (int)std::min<long long>(kManyParts, 64ll * y.many_tiles * n_kv);
    }
    return y;
}

template <typename T, int HD>
int launch(hipStream_t st, const AttnArgs &a, const Layout &y) {
    if (y.many) {
        const int wgs = a.many_tiles * a.pg.n_kv + a.many_room;
        hipLaunchKernelGGL((paged_attn_many_kernel<T, HD>), dim3(wgs), dim3(Many<T, HD>::kThreads), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    if (y.few) {
        hipLaunchKernelGGL((paged_attn_few_kernel<T, HD>), dim3(a.n_seqs * a.few_splits * a.pg.n_kv),
                           dim3(kFewWaves * 64), 0, st, a);
        SGQ_HIP(hipGetLastError());
    }
    const int each = std::min(a.group, a.few_cap), n_few = a.few_splits > 1 ? a.n_seqs * a.pg.n_kv * each : 0;
    if (a.many_room > 1) {
        const long long units = std::min<long long>(a.many_room / 2, (long long)a.many_tiles * a.pg.n_kv);
        const int n_many = (int)std::min<long long>(kJoinWgs, units * Many<T, HD>::kRows / (kJoinWaves * ManyJoin<T, HD>::kRows));
        hipLaunchKernelGGL((paged_attn_join_kernel<T, HD, true>), dim3(n_many + n_few), dim3(kJoinWaves * 64), 0, st, a,
                           n_many);
        SGQ_HIP(hipGetLastError());
    } else if (n_few) {
        hipLaunchKernelGGL((paged_attn_join_kernel<T, HD, false>), dim3(a.n_seqs, a.pg.n_kv, each), dim3(kJoinWaves * 64), 0, st, a, 0);
        SGQ_HIP(hipGetLastError());
    }
    return SGQ_OK;
}

}  // namespace

uint64_t paged_attn_workspace(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim, int max_new,
                              int max_kv) {
    uint64_t most = 0;  // of both row types
    for (int f16 = 0; f16 < 2; f16++) {
        const Layout y = layout(n_tokens, n_seqs, n_q, n_kv, head_dim, f16, max_new, max_kv);
        most = std::max(most, (y.few_splits > 1 ? y.few_rows * y.few_splits : 0) +
                                  (uint64_t)y.many_parts * y.many_bm);
    }
    return most * (head_dim + 2) * 4;
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
    // as many parts as fit into the workspace, the few rows' first
    const uint64_t part_bytes = (uint64_t)(p.pg.head_dim + 2) * 4;
    uint64_t room = p.workspace ? p.workspace_bytes / part_bytes : 0;
    if (y.few_splits > 1 && room >= 2 * y.few_rows) {
        a.few_splits = (int)std::min<uint64_t>(room / y.few_rows, y.few_splits);
        room -= y.few_rows * a.few_splits;
    } else {
        a.few_splits = 1;
    }
    const int tiles = std::max((int)(((long long)reach + 31) / 32), 1);
    a.few_per = std::max((tiles + a.few_splits - 1) / a.few_splits, 8);
    a.few = y.few, a.few_cap = few_cap(p.max_new, a.group);
    a.many_tiles = y.many_tiles;
    a.many_room = (int)std::min<uint64_t>(room / y.many_bm, y.many_parts);
    const uint64_t few_parts = a.few_splits > 1 ? y.few_rows * a.few_splits : 0;
    const uint64_t many_parts = (uint64_t)a.many_room * y.many_bm;
    a.few_part = static_cast<float *>(p.workspace);
    a.many_part = a.few_part + few_parts * p.pg.head_dim;
    a.few_ml = reinterpret_cast<float2 *>(a.many_part + many_parts * p.pg.head_dim);
    a.many_ml = a.few_ml + few_parts;
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
