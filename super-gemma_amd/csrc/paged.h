// The paged 8-bit KV cache of a batch of requests: what its translation units
// (paged_plan.hip, paged_kv.hip, paged_attn.hip, paged_api.hip) share.
//
// A page holds P = 32, 64 or 128 tokens of every kv head; slot = page·P + offset.
// Each (page, head) is one contiguous block of P·hd int8 quants for K and one
// for V, with one fp32 scale each:
//   K  [page][head][P][hd]           a token's row is contiguous: the lane of a
//                                    QK MFMA reads 16 bytes of its own key
//   V  [page][head][P/32][hd][32]    groups of 32 tokens transposed: the lane
//                                    of a PV MFMA reads 8 tokens of its own dim,
//                                    so neither operand passes through a shuffle
//   scales [page][head]
#pragma once
#include "sgq_internal.h"

namespace sgq {

// The calling thread's current device is the context's while one of these lives.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&prev_) != hipSuccess) prev_ = device;
        if (prev_ != device) (void)hipSetDevice(device);
        else prev_ = -1;
    }
    ~DeviceGuard() {
        if (prev_ >= 0) (void)hipSetDevice(prev_);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;

  private:
    int prev_ = -1;
};

// Requests in one step: their prefix sums stay in one workgroup's LDS.
constexpr uint32_t kPagedMaxSeqs = 4096;

struct PagedPlan {
    const int32_t *cached, *add;
    int32_t *tables;
    const int32_t *free_list, *n_free;
    int32_t *n_free_out, *kv_lens, *cu, *slots, *missing;
    int n_seqs, page_log2, max_pages, n_pages, n_tokens;
};
int launch_paged_plan(hipStream_t st, const PagedPlan &p);

struct PagedRelease {
    const int32_t *done;
    int32_t *kv_lens, *tables, *free_list, *n_free;
    int n_seqs, page_log2, max_pages, n_pages;
};
int launch_paged_release(hipStream_t st, const PagedRelease &p);

// Pages with their geometry; strides of token rows are in elements.
struct PagedPages {
    int8_t *kq, *vq;
    float *ks, *vs;
    int n_pages, page_log2, n_kv, head_dim;
};
int launch_paged_append(hipStream_t st, const PagedPages &pg, const void *k, uint64_t k_stride,
                        const void *v, uint64_t v_stride, bool f16, float growth,
                        const int32_t *slots, uint32_t n_tokens);
int launch_paged_gather(hipStream_t st, const PagedPages &pg, const int32_t *slots,
                        uint32_t n_tokens, bool f16, void *k, uint64_t k_stride, void *v,
                        uint64_t v_stride);

struct PagedAttn {
    PagedPages pg;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    const int32_t *tables, *kv_lens, *cu;
    int max_pages, n_seqs, n_tokens, n_q, max_new, max_kv, window;
    bool f16;
    float scale;
    void *workspace;
    uint64_t workspace_bytes;
};
int launch_paged_attn(hipStream_t st, const PagedAttn &a);
// Bytes with which launch_paged_attn splits the keys as far as it wants to.
uint64_t paged_attn_workspace(int n_tokens, int n_seqs, int n_q, int n_kv, int head_dim,
                              int max_new, int max_kv);

}  // namespace sgq
