// C entry points of the paged 8-bit KV cache: argument checks, then one launch
// each (paged_plan.hip, paged_kv.hip, paged_attn.hip).
#include <cmath>

#include "paged.h"

using namespace sgq;

namespace {

constexpr uint32_t kMaxRows = 1u << 22;  // packed rows of one step
constexpr uint64_t kMaxRowHeads = 1u << 26;  // rows x heads: every grid below 2^32 threads

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// log2 of a page size, -1 if it is none.
int page_log2(uint32_t page_size) {
    return page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

int check_table(const char *who, uint32_t n_seqs, uint32_t page_size, uint32_t max_pages,
                uint32_t n_pages) {
    SGQ_CHECK(n_seqs >= 1 && n_seqs <= kPagedMaxSeqs, "%s: n_seqs %u out of range (1..%u)", who,
              n_seqs, kPagedMaxSeqs);
    SGQ_CHECK(page_log2(page_size) >= 0, "%s: page_size %u unsupported (32, 64, 128)", who, page_size);
    SGQ_CHECK(max_pages >= 1 && (uint64_t)max_pages * page_size < (1u << 31) &&
                  (uint64_t)max_pages * n_seqs < (1u << 31),
              "%s: max_pages %u out of range", who, max_pages);
    SGQ_CHECK(n_pages >= 1 && (uint64_t)n_pages * page_size < (1u << 31), "%s: n_pages %u out of range",
              who, n_pages);
    return SGQ_OK;
}

int check_pages(const char *who, const sgq_kv_pages *p, PagedPages *pg) {
    if (!p || !p->k_quants || !p->v_quants || !p->k_scales || !p->v_scales)
        return fail(SGQ_ERR_VALIDATION, "%s: NULL pages", who);
    SGQ_CHECK(page_log2(p->page_size) >= 0, "%s: page_size %u unsupported (32, 64, 128)", who,
              p->page_size);
    SGQ_CHECK(p->n_pages >= 1 && (uint64_t)p->n_pages * p->page_size < (1u << 31),
              "%s: n_pages %u out of range", who, p->n_pages);
    SGQ_CHECK(p->n_kv_heads >= 1 && p->n_kv_heads <= 1024, "%s: n_kv_heads %u out of range (1..1024)",
              who, p->n_kv_heads);
    SGQ_CHECK(p->head_dim == 128 || p->head_dim == 256 || p->head_dim == 512,
              "%s: head_dim %u unsupported (128, 256, 512)", who, p->head_dim);
    SGQ_CHECK(aligned(p->k_quants, 16) && aligned(p->v_quants, 16) && aligned(p->k_scales, 4) &&
                  aligned(p->v_scales, 4),
              "%s: misaligned pages", who);
    *pg = PagedPages{p->k_quants, p->v_quants, p->k_scales, p->v_scales, (int)p->n_pages,
                     page_log2(p->page_size), (int)p->n_kv_heads, (int)p->head_dim};
    return SGQ_OK;
}

int check_rows(const char *who, const char *what, const void *p, uint64_t stride, uint64_t width,
               int act) {
    const uint64_t es = act == SGQ_ACT_F16 ? 2 : 4;
    SGQ_CHECK(stride >= width && stride < (1ull << 32), "%s: %s rows of %llu elements at stride %llu",
              who, what, (unsigned long long)width, (unsigned long long)stride);
    SGQ_CHECK(aligned(p, 16) && stride * es % 16 == 0, "%s: %s rows are not 16-byte aligned", who, what);
    return SGQ_OK;
}

int check_count(const char *who, uint32_t n_tokens, uint32_t n_heads) {
    SGQ_CHECK(n_tokens <= kMaxRows, "%s: n_tokens %u out of range", who, n_tokens);
    SGQ_CHECK((uint64_t)n_tokens * n_heads <= kMaxRowHeads, "%s: %u rows of %u heads in one step (at most %llu together)",
              who, n_tokens, n_heads, (unsigned long long)kMaxRowHeads);
    return SGQ_OK;
}

int check_act(const char *who, int act) {
    SGQ_CHECK(act == SGQ_ACT_F32 || act == SGQ_ACT_F16, "%s: activation type %d", who, act);
    return SGQ_OK;
}

}  // namespace

extern "C" {

int sgq_kv_pages_plan(sgq_ctx *ctx, const int32_t *cached_lens, const int32_t *new_lens,
                      uint32_t n_seqs, uint32_t page_size, int32_t *block_tables,
                      uint32_t max_pages, const int32_t *free_list, uint32_t n_pages,
                      const int32_t *n_free, int32_t *n_free_out, int32_t *kv_lens,
                      int32_t *cu_tokens, int32_t *slot_map, uint32_t n_tokens, int32_t *missing) {
    static const char who[] = "kv_pages_plan";
    if (!ctx || !cached_lens || !new_lens || !block_tables || !free_list || !n_free || !n_free_out ||
        !kv_lens || !cu_tokens || (n_tokens && !slot_map) || !missing)
        return fail(SGQ_ERR_VALIDATION, "%s: NULL argument", who);
    if (int rc = check_table(who, n_seqs, page_size, max_pages, n_pages)) return rc;
    SGQ_CHECK(n_tokens <= kMaxRows, "%s: n_tokens %u out of range", who, n_tokens);
    SGQ_CHECK(kv_lens != new_lens && free_list != block_tables, "%s: overlapping arguments", who);
    DeviceGuard dev(ctx_device(ctx));
    return launch_paged_plan(ctx_stream(ctx),
                             PagedPlan{cached_lens, new_lens, block_tables, free_list, n_free,
                                       n_free_out, kv_lens, cu_tokens, slot_map, missing, (int)n_seqs,
                                       page_log2(page_size), (int)max_pages, (int)n_pages,
                                       (int)n_tokens});
}

int sgq_kv_pages_release(sgq_ctx *ctx, const int32_t *done, uint32_t n_seqs, uint32_t page_size,
                         int32_t *kv_lens, int32_t *block_tables, uint32_t max_pages,
                         int32_t *free_list, uint32_t n_pages, int32_t *n_free) {
    static const char who[] = "kv_pages_release";
    if (!ctx || !done || !kv_lens || !block_tables || !free_list || !n_free)
        return fail(SGQ_ERR_VALIDATION, "%s: NULL argument", who);
    if (int rc = check_table(who, n_seqs, page_size, max_pages, n_pages)) return rc;
    SGQ_CHECK(done != kv_lens && free_list != block_tables, "%s: overlapping arguments", who);
    DeviceGuard dev(ctx_device(ctx));
    return launch_paged_release(ctx_stream(ctx),
                                PagedRelease{done, kv_lens, block_tables, free_list, n_free,
                                             (int)n_seqs, page_log2(page_size), (int)max_pages,
                                             (int)n_pages});
}

int sgq_kv_append_paged_q8(sgq_ctx *ctx, const sgq_kv_pages *pages, const void *k,
                           uint64_t k_stride, const void *v, uint64_t v_stride, int act,
                           const int32_t *slot_map, uint32_t n_tokens) {
    static const char who[] = "kv_append_paged_q8";
    PagedPages pg;
    if (!ctx || (n_tokens && (!k || !v || !slot_map)))
        return fail(SGQ_ERR_VALIDATION, "%s: NULL argument", who);
    if (int rc = check_pages(who, pages, &pg)) return rc;
    const bool headroom = act >= 0 && (act & SGQ_APPEND_HEADROOM);
    if (headroom) act &= ~SGQ_APPEND_HEADROOM;
    if (int rc = check_act(who, act)) return rc;
    if (int rc = check_count(who, n_tokens, pages->n_kv_heads)) return rc;
    const uint64_t width = (uint64_t)pg.n_kv * pg.head_dim;
    if (int rc = check_rows(who, "k", k, k_stride, width, act)) return rc;
    if (int rc = check_rows(who, "v", v, v_stride, width, act)) return rc;
    if (!n_tokens) return SGQ_OK;
    DeviceGuard dev(ctx_device(ctx));
    return launch_paged_append(ctx_stream(ctx), pg, k, k_stride, v, v_stride, act == SGQ_ACT_F16,
                               headroom ? 1.25f : 1.f, slot_map, n_tokens);
}

int sgq_kv_gather_paged_q8(sgq_ctx *ctx, const sgq_kv_pages *pages, const int32_t *slot_map,
                           uint32_t n_tokens, int act, void *k, uint64_t k_stride, void *v,
                           uint64_t v_stride) {
    static const char who[] = "kv_gather_paged_q8";
    PagedPages pg;
    if (!ctx || (n_tokens && (!k || !v || !slot_map)))
        return fail(SGQ_ERR_VALIDATION, "%s: NULL argument", who);
    if (int rc = check_pages(who, pages, &pg)) return rc;
    if (int rc = check_act(who, act)) return rc;
    if (int rc = check_count(who, n_tokens, pages->n_kv_heads)) return rc;
    const uint64_t width = (uint64_t)pg.n_kv * pg.head_dim;
    if (int rc = check_rows(who, "k", k, k_stride, width, act)) return rc;
    if (int rc = check_rows(who, "v", v, v_stride, width, act)) return rc;
    if (!n_tokens) return SGQ_OK;
    DeviceGuard dev(ctx_device(ctx));
    return launch_paged_gather(ctx_stream(ctx), pg, slot_map, n_tokens, act == SGQ_ACT_F16, k,
                               k_stride, v, v_stride);
}

uint64_t sgq_attn_paged_workspace(const sgq_kv_pages *pages, uint32_t n_seqs, uint32_t n_tokens,
                                  uint32_t n_q_heads, uint32_t max_new, uint32_t max_kv) {
    PagedPages pg;
    if (check_pages("attn_paged_workspace", pages, &pg) || !n_seqs || n_seqs > kPagedMaxSeqs ||
        !n_tokens || n_tokens > kMaxRows || !n_q_heads || n_q_heads % pg.n_kv ||
        n_q_heads / pg.n_kv > 64 || (uint64_t)n_tokens * n_q_heads > kMaxRowHeads)
        return 0;  // the call itself says what is wrong
    return paged_attn_workspace((int)n_tokens, (int)n_seqs, (int)n_q_heads, pg.n_kv, pg.head_dim,
                                (int)(max_new < kMaxRows ? max_new : kMaxRows),
                                (int)(max_kv < (1u << 31) ? max_kv : (1u << 31) - 1));
}

int sgq_attn_paged_q8(sgq_ctx *ctx, const sgq_kv_pages *pages, const void *q, uint64_t q_stride,
                      int act, const int32_t *block_tables, uint32_t max_pages,
                      const int32_t *kv_lens, const int32_t *cu_tokens, uint32_t n_seqs,
                      uint32_t n_tokens, uint32_t n_q_heads, uint32_t max_new, uint32_t max_kv,
                      uint32_t window, float scale, void *out, uint64_t out_stride,
                      void *workspace, uint64_t workspace_bytes) {
    static const char who[] = "attn_paged_q8";
    PagedAttn a;
    if (!ctx || (n_tokens && (!q || !out)) || !block_tables || !kv_lens || !cu_tokens)
        return fail(SGQ_ERR_VALIDATION, "%s: NULL argument", who);
    if (int rc = check_pages(who, pages, &a.pg)) return rc;
    if (int rc = check_act(who, act)) return rc;
    if (int rc = check_table(who, n_seqs, pages->page_size, max_pages, pages->n_pages)) return rc;
    SGQ_CHECK(n_q_heads >= 1 && n_q_heads % (uint32_t)a.pg.n_kv == 0 && n_q_heads / (uint32_t)a.pg.n_kv <= 64,
              "%s: %u query heads over %d kv heads", who, n_q_heads, a.pg.n_kv);
    if (int rc = check_count(who, n_tokens, n_q_heads)) return rc;
    SGQ_CHECK(window < (1u << 31), "%s: window %u out of range", who, window);
    SGQ_CHECK(std::isfinite(scale), "%s: scale is not finite", who);
    SGQ_CHECK(aligned(workspace, 16), "%s: workspace is not 16-byte aligned", who);
    const uint64_t width = (uint64_t)n_q_heads * pages->head_dim;
    if (int rc = check_rows(who, "q", q, q_stride, width, act)) return rc;
    if (int rc = check_rows(who, "out", out, out_stride, width, act)) return rc;
    if (!n_tokens || !max_new) return SGQ_OK;
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.tables = block_tables, a.kv_lens = kv_lens, a.cu = cu_tokens;
    a.max_pages = (int)max_pages, a.n_seqs = (int)n_seqs, a.n_tokens = (int)n_tokens;
    a.n_q = (int)n_q_heads;
    a.max_new = (int)(max_new < n_tokens ? max_new : n_tokens);
    a.max_kv = (int)(max_kv < (1u << 31) ? max_kv : (1u << 31) - 1);
    a.window = (int)window, a.f16 = act == SGQ_ACT_F16, a.scale = scale;
    a.workspace = workspace, a.workspace_bytes = workspace ? workspace_bytes : 0;
    DeviceGuard dev(ctx_device(ctx));
    return launch_paged_attn(ctx_stream(ctx), a);
}

}  // extern "C"
