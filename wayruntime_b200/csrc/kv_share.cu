// kv_share.cu — sessions that go on from one another: forks that hold the same pages, and the caches of a search's beams
// put into the order that the search has chosen.
//
// A fork holds its parent's full pages with it and copies the rows behind them.  Reordering n sessions by
// parents[i] needs no copy for a parent's first child, which takes over everything the parent holds: tables, pages and
// state change hands on the host.  Its further children copy the rows that are not shared into what sessions without
// children held.  What is read is never written in the same call, so all copies go at once.
#include <new>

#include "kv_share.cuh"
#include "rows_dev.cuh"

namespace {

// Copies of one launch: for every pair and layer, the rows of pages [page0, ceil(rows / 64)).
constexpr uint32_t kCopyThreads = 256, kCopyVecs = 4, kCopyBytes = kCopyThreads * kCopyVecs * 16, kCopyLayers = 256;
struct copy_pair {
    const uint64_t *from, *to;           // device page tables, [layer][n_pages]
    uint32_t page0, rows;
};
struct copy_params {
    copy_pair pair[WR_CUDA_BATCH_MAX];
    wr_kv_geom geom;
    uint64_t page_bytes;
    uint32_t n_pages, per_page;          // pages of a table; CTAs to a page
    uint16_t layer[kCopyLayers];
};

// HBM bounds it: every thread has four 16-byte loads under way (6 sessions' 700 own rows of 8 layers and 8 kv heads, 138 MB read and
// 138 written: 45 us with the host's part, 6.1 TB/s).  The last page's rows end inside a page, and a row's bytes do not lie together in
// it, so each vector asks which token it belongs to.
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const __grid_constant__ copy_params p)
{
    const copy_pair &c = p.pair[blockIdx.z];
    const uint32_t page = c.page0 + blockIdx.x / p.per_page;
    if (page * kPageTokens >= c.rows) return;
    const uint32_t tokens = min(c.rows - page * kPageTokens, kPageTokens);
    const size_t at = (size_t)p.layer[blockIdx.y] * p.n_pages + page;
    const char *from = reinterpret_cast<const char *>(c.from[at]);
    char *to = reinterpret_cast<char *>(c.to[at]);
    const uint64_t lo = (uint64_t)(blockIdx.x % p.per_page) * kCopyBytes + threadIdx.x * 16u;
    const uint32_t k_row = wr_hd_pad(p.geom.k_dim) * wr_geom_esize(p.geom), v_row = wr_hd_pad(p.geom.v_dim) * wr_geom_esize(p.geom);
    const bool tiled = p.geom.elem == WR_CUDA_F16 && wr_tiled(p.geom.k_dim) && (p.geom.v_dim == p.geom.k_dim || p.geom.v_dim == 0);
    uint4 v[kCopyVecs];
    bool mine[kCopyVecs];
#pragma unroll
    for (uint32_t i = 0; i < kCopyVecs; ++i) {
        const uint64_t off = lo + (uint64_t)i * kCopyThreads * 16u;
        mine[i] = off < p.page_bytes;
        if (mine[i] && tokens < kPageTokens) {
            const uint32_t in_head = (uint32_t)(off % (kPageTokens * (k_row + v_row)));
            mine[i] = (tiled ? in_head % (kPageTokens * 128u) / 128u
                             : in_head < kPageTokens * k_row ? in_head / k_row : (in_head - kPageTokens * k_row) / v_row) < tokens;
        }
        if (mine[i]) v[i] = *reinterpret_cast<const uint4 *>(from + off);
    }
#pragma unroll
    for (uint32_t i = 0; i < kCopyVecs; ++i)
        if (mine[i]) *reinterpret_cast<uint4 *>(to + lo + (uint64_t)i * kCopyThreads * 16u) = v[i];
}

struct state_params {
    const char *from[WR_CUDA_BATCH_MAX];
    char *to[WR_CUDA_BATCH_MAX];
    uint64_t bytes;
};
__global__ void __launch_bounds__(kCopyThreads) state_copy_kernel(const __grid_constant__ state_params p)
{
    for (uint64_t at = ((uint64_t)blockIdx.x * kCopyThreads + threadIdx.x) * 16u; at < p.bytes; at += (uint64_t)gridDim.x * kCopyThreads * 16u)
        *reinterpret_cast<uint4 *>(p.to[blockIdx.y] + at) = *reinterpret_cast<const uint4 *>(p.from[blockIdx.y] + at);
}

bool same_geom(const wr_kv_geom &a, const wr_kv_geom &b)
{
    return a.n_kv == b.n_kv && (!a.n_kv || (a.k_dim == b.k_dim && a.v_dim == b.v_dim && a.elem == b.elem));
}

// Enqueues the copies of all layers, layers with equal pages together.  (Ordinary launches: the rows have been written when
// they begin.  Who reads the copies waits for them: wr_pdl_rows.)
int copy_rows(wr_cuda_ctx *ctx, const wr_cuda_kv *of, const copy_pair *pairs, uint32_t n)
{
    copy_params p;
    uint32_t pages = 0;
    for (uint32_t i = 0; i < n; ++i) {
        p.pair[i] = pairs[i];
        const uint32_t end = (pairs[i].rows + kPageTokens - 1) / kPageTokens;
        if (end > pairs[i].page0) pages = std::max(pages, end - pairs[i].page0);
    }
    if (!pages) return WR_CUDA_OK;
    p.n_pages = of->n_pages;
    std::vector<uint8_t> done(of->n_layers, 0);
    for (uint32_t L = 0; L < of->n_layers; ++L) {
        if (done[L] || !of->layers[L].geom.n_kv) continue;
        p.geom = of->layers[L].geom;
        p.page_bytes = of->layers[L].page_bytes;
        p.per_page = (uint32_t)((p.page_bytes + kCopyBytes - 1) / kCopyBytes);
        uint32_t m = 0;
        for (uint32_t M = L; M < of->n_layers && m < kCopyLayers; ++M)
            if (!done[M] && of->layers[M].geom.n_kv && same_geom(of->layers[M].geom, p.geom)) {
                p.layer[m++] = (uint16_t)M;
                done[M] = 1;
            }
        kv_copy_kernel<<<dim3(pages * p.per_page, m, n), kCopyThreads, 0, ctx->stream>>>(p);
        const int rc = finish_launch(ctx);
        wr_pdl_rows(ctx);
        if (rc != WR_CUDA_OK) return rc;
    }
    return WR_CUDA_OK;
}
int copy_states(wr_cuda_ctx *ctx, const state_params &p, uint32_t n)
{
    if (!n) return WR_CUDA_OK;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((p.bytes / 16 + kCopyThreads - 1) / kCopyThreads, 4u * (uint32_t)ctx->sm_count);
    state_copy_kernel<<<dim3(blocks, n), kCopyThreads, 0, ctx->stream>>>(p);
    const int rc = finish_launch(ctx);
    wr_pdl_rows(ctx);                    // (the rows copied just before it may not be there either)
    return rc;
}

// Sessions change hands on the host, which a graph would not do again when it is launched.
bool capturing(wr_cuda_ctx *ctx) { return wr_ctx_capture(ctx) != 0; }

}  // namespace

extern "C" uint32_t wr_cuda_kv_shared_rows(const wr_cuda_kv *a, const wr_cuda_kv *b)
{
    if (!a || !b || a->ctx != b->ctx || a == b) return 0;
    std::lock_guard<std::mutex> g(a->ctx->lock);
    return wr_kv_common_pages(a, b) * kPageTokens;
}

extern "C" int wr_cuda_kv_fork(wr_cuda_ctx *ctx, wr_cuda_kv *kv, uint32_t n_rows, wr_cuda_kv **out)
{
    if (!ctx || !out) return WR_CUDA_ERR_INVAL;
    *out = nullptr;
    if (!kv || kv->ctx != ctx) return WR_CUDA_ERR_INVAL;
    if (n_rows > kv->max_ctx) return WR_CUDA_ERR_CTX_FULL;
    std::lock_guard<std::mutex> g(ctx->lock);
    WR_CUDA_TRY(cudaSetDevice(ctx->device));
    if (capturing(ctx)) return WR_CUDA_ERR_STATE;
    const int slot = kv->state_bytes && n_rows ? kv->state_slot(n_rows) : -1;
    if (kv->state_bytes && n_rows && slot < 0) return WR_CUDA_ERR_STATE;
    const uint32_t full = n_rows / kPageTokens, own = kv->n_pages - full;
    wr_cuda_kv *f = new (std::nothrow) wr_cuda_kv();
    if (!f) return WR_CUDA_ERR_NOMEM;
    f->ctx = ctx;
    f->n_layers = kv->n_layers;
    f->max_ctx = kv->max_ctx;
    f->n_pages = kv->n_pages;
    f->layers = kv->layers;
    f->state_bytes = kv->state_bytes;
    f->contig.assign(kv->n_layers, full ? 0 : 1);
    f->pages.assign(kv->pages.size(), nullptr);
    while (kv->columns.size() < full) kv->columns.push_back(new wr_kv_column());
    for (uint32_t i = 0; i < full; ++i) {
        kv->columns[i]->holders.fetch_add(1);
        f->columns.push_back(kv->columns[i]);
    }
    int rc = WR_CUDA_OK;
    for (uint32_t L = 0; L < kv->n_layers && rc == WR_CUDA_OK; ++L) {
        if (!kv->layers[L].geom.n_kv) continue;
        void *const *theirs = kv->pages.data() + (size_t)L * kv->n_pages;
        void **ours = f->pages.data() + (size_t)L * kv->n_pages;
        std::vector<void *> got;
        size_t pool = 0;
        rc = wr_pool_take(ctx, kv->layers[L].page_bytes, own, &pool, got);
        if (rc != WR_CUDA_OK) break;
        std::copy(theirs, theirs + full, ours);
        std::copy(got.begin(), got.end(), ours + full);
        for (uint32_t i = 1; i < own; ++i)
            if ((char *)got[i] != (char *)got[i - 1] + kv->layers[L].page_bytes) f->contig[L] = 0;
    }
    if (rc == WR_CUDA_OK && kv->state_bytes) {
        std::vector<void *> got;
        rc = wr_pool_take(ctx, kv->state_bytes, 2, &f->state_pool, got);
        if (rc == WR_CUDA_OK) {
            f->state[0] = got[0];
            f->state[1] = got[1];
        }
    }
    if (rc == WR_CUDA_OK) {
        const size_t bytes = f->pages.size() * sizeof(uint64_t);
        cudaError_t e = cudaMalloc((void **)&f->d_pages, bytes);
        if (e == cudaSuccess) e = cudaMemcpyAsync(f->d_pages, f->pages.data(), bytes, cudaMemcpyHostToDevice, ctx->stream);
        if (e != cudaSuccess) {
            (void)cudaGetLastError();
            rc = e == cudaErrorMemoryAllocation ? WR_CUDA_ERR_NOMEM : WR_CUDA_ERR_INTERNAL;
        }
    }
    if (rc == WR_CUDA_OK) {
        const copy_pair rest = {kv->d_pages, f->d_pages, full, n_rows};
        rc = copy_rows(ctx, kv, &rest, 1);
    }
    if (rc == WR_CUDA_OK && slot >= 0) {
        state_params s{};
        s.from[0] = (const char *)kv->state[slot];
        s.to[0] = (char *)f->state[slot];
        s.bytes = kv->state_bytes;
        rc = copy_states(ctx, s, 1);
        f->state_len[slot] = n_rows;
    }
    if (rc != WR_CUDA_OK) {
        (void)cudaStreamSynchronize(ctx->stream);
        wr_kv_give_back(f);
        delete f;
        return rc;
    }
    ctx->live_kv++;
    *out = f;
    // (rows that the last launch of shared attention may still be writing may be shared ones now)
    if (ctx->pdl_kind == WR_PDL_SHARED) ctx->pdl_kind = WR_PDL_ROWS;
    return WR_CUDA_OK;
}

extern "C" int wr_cuda_kv_reorder(wr_cuda_ctx *ctx, uint32_t n, wr_cuda_kv *const *kv, const uint32_t *parents, const uint32_t *rows)
{
    if (!ctx || !kv || !parents || !rows || n == 0) return WR_CUDA_ERR_INVAL;
    if (n > WR_CUDA_BATCH_MAX) return WR_CUDA_ERR_LIMIT;
    std::lock_guard<std::mutex> g(ctx->lock);
    for (uint32_t i = 0; i < n; ++i) {
        if (!kv[i] || kv[i]->ctx != ctx || parents[i] >= n) return WR_CUDA_ERR_INVAL;
        for (uint32_t j = 0; j < i; ++j)
            if (kv[j] == kv[i]) return WR_CUDA_ERR_INVAL;
        if (kv[i]->n_layers != kv[0]->n_layers || kv[i]->max_ctx != kv[0]->max_ctx || kv[i]->state_bytes != kv[0]->state_bytes)
            return WR_CUDA_ERR_INVAL;
        for (uint32_t L = 0; L < kv[0]->n_layers; ++L)
            if (!same_geom(kv[i]->layers[L].geom, kv[0]->layers[L].geom)) return WR_CUDA_ERR_INVAL;
        if (rows[i] > kv[i]->max_ctx) return WR_CUDA_ERR_CTX_FULL;
    }
    WR_CUDA_TRY(cudaSetDevice(ctx->device));
    if (capturing(ctx)) return WR_CUDA_ERR_STATE;
    // holds[i]: whose memory session i goes on with
    uint32_t holds[WR_CUDA_BATCH_MAX];
    bool taken[WR_CUDA_BATCH_MAX] = {}, first[WR_CUDA_BATCH_MAX] = {};
    for (uint32_t i = 0; i < n; ++i)
        if (parents[i] == i) first[i] = taken[i] = true, holds[i] = i;
    for (uint32_t i = 0; i < n; ++i)
        if (!first[i] && !taken[parents[i]]) first[i] = taken[parents[i]] = true, holds[i] = parents[i];
    copy_pair pairs[WR_CUDA_BATCH_MAX];
    state_params states{};
    int slots[WR_CUDA_BATCH_MAX];
    uint32_t copies = 0;
    for (uint32_t i = 0, to = 0; i < n; ++i) {
        const uint32_t from = parents[i];
        slots[i] = kv[from]->state_bytes && rows[from] ? kv[from]->state_slot(rows[from]) : -1;
        if (kv[from]->state_bytes && rows[from] && slots[i] < 0) return WR_CUDA_ERR_STATE;
        if (first[i]) continue;
        while (taken[to]) ++to;
        taken[to] = true;
        holds[i] = to;
        const uint32_t common = wr_kv_common_pages(kv[from], kv[to]);
        // (not only the rows to copy: the session goes on behind them)
        const uint32_t own = std::min(common * kPageTokens, rows[from]);
        if (!wr_kv_writable(kv[to], own, kv[to]->max_ctx - own)) return WR_CUDA_ERR_STATE;
        pairs[copies] = {kv[from]->d_pages, kv[to]->d_pages, common, rows[from]};
        if (slots[i] >= 0) {
            states.from[copies] = (const char *)kv[from]->state[slots[i]];
            states.to[copies] = (char *)kv[to]->state[slots[i]];
        }
        ++copies;
    }
    if (copies) {
        int rc = copy_rows(ctx, kv[0], pairs, copies);
        // (states of sessions without a row are not read: a step at position 0 starts them over)
        uint32_t m = 0;
        for (uint32_t c = 0; c < copies; ++c)
            if (states.from[c]) {
                states.from[m] = states.from[c];
                states.to[m++] = states.to[c];
            }
        states.bytes = kv[0]->state_bytes;
        if (rc == WR_CUDA_OK) rc = copy_states(ctx, states, m);
        if (rc != WR_CUDA_OK) return rc;
    }
    wr_cuda_kv was[WR_CUDA_BATCH_MAX];
    for (uint32_t i = 0; i < n; ++i) was[i] = std::move(*kv[i]);
    for (uint32_t i = 0; i < n; ++i) {
        *kv[i] = std::move(was[holds[i]]);
        if (first[i]) continue;
        kv[i]->state_len[0] = kv[i]->state_len[1] = -1;
        if (slots[i] >= 0) kv[i]->state_len[slots[i]] = rows[parents[i]];
    }
    return WR_CUDA_OK;
}
