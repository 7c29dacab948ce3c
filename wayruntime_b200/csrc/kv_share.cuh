// kv_share.cuh — pages that several sessions hold, and attention over them.
#pragma once

#include <atomic>

#include "wr_internal.cuh"

// The pages of 64 tokens, one per layer that has pages, that a session and its forks hold together (each has them in its
// table).  Sharing goes from a session's first page on (wr_cuda_kv_fork), so two sessions that hold the same column hold
// all columns before it too.  Nothing is written into a column while more than one session holds it.
struct wr_kv_column {
    std::atomic<uint32_t> holders{1};
};

// Leading pages that both hold.  (Caller holds ctx->lock, here and below: forking a session makes its list of columns longer.)
inline uint32_t wr_kv_common_pages(const wr_cuda_kv *a, const wr_cuda_kv *b)
{
    uint32_t lo = 0, hi = (uint32_t)std::min(a->columns.size(), b->columns.size());
    while (lo < hi) {                    // (the first hi columns agree from some place on no more)
        const uint32_t mid = (lo + hi + 1) / 2;
        if (a->columns[mid - 1] == b->columns[mid - 1]) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Rows [row0, row0 + n) are this session's alone to write.
inline bool wr_kv_writable(const wr_cuda_kv *kv, uint32_t row0, uint32_t n)
{
    for (size_t i = row0 / kPageTokens; i < kv->columns.size() && i * kPageTokens < (size_t)row0 + n; ++i)
        if (kv->columns[i]->holders.load(std::memory_order_relaxed) > 1) return false;
    return true;
}

// Whether two ranges of device memory have bytes in common.
inline bool wr_overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes)
{
    return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

int wr_shared_validate(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *seq_lens,
                       uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const void *q, const void *out,
                       uint32_t n_q, int mem);
// the rows that decode_step_shared appends on the way (device memory)
struct wr_shared_append {
    const float *k, *v;
    float theta_base;
    uint32_t n_rot_pairs, flags;
};
int wr_shared_launch(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *seq_lens,
                     uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const float *dq, float *dout,
                     uint32_t n_q, float scale_override, const wr_shared_append *append, bool dependent);
// wr_cuda_decode_step_shared; dependent: as wr_decode_step's.  Caller holds ctx->lock.
int wr_decode_step_shared(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *positions,
                          uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const float *q, const float *k_rows,
                          const float *v_rows, float *out, uint32_t n_q_heads, float theta_base, uint32_t n_rot_pairs, uint32_t flags,
                          float scale_override, int mem, bool dependent = true);

// kv_cache.cu: pages from the context's pool; everything a session holds back to it.  Caller holds ctx->lock.
int wr_pool_take(wr_cuda_ctx *ctx, uint64_t page_bytes, size_t n, size_t *pool_index, std::vector<void *> &out);
void wr_kv_give_back(wr_cuda_kv *kv);

// beam.cu: wr_cuda_beam_select on device memory; row r's logits at logits + (map ? map[r] : r) * ld.  Caller holds ctx->lock.
struct wr_beam_args {
    const float *logits;
    size_t ld;
    uint32_t groups, beams, vocab, n_out;
    const float *scores;                 // [groups][beams]
    float *out_scores;                   // [groups][n_out]
    uint32_t *out_beams, *out_tokens;
    bool mapped;
    uint8_t map[WR_CUDA_BATCH_MAX];
};
int wr_beam_validate(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t n_out);
int wr_beam_launch(wr_cuda_ctx *ctx, const wr_beam_args &a);
