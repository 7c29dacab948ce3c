// beam.cu — a beam search's choice: for every request the n_out best of beams x vocabulary by
//     total(b, v) = score_b + logit(b, v) - log sum_u exp(logit(b, u))
// The reference has no beam search; its sampler takes one row of logits (src/core/sample.c:239).
//
// One pass over the logits: a CTA takes a part of a row and leaves the part's sum of exponentials (against the part's
// maximum) and its n_out best logits; within a row totals are in the order of logits, so nothing else of the part can be
// among the row's best.  The CTA that is the last of its request puts the parts together: sums and totals in 64 bits,
// since candidates of two beams may lie closer than an F32 rounding.  HBM bounds it (4 bytes a logit) where there are many
// rows, round trips where there are few; a second kernel for the parts took 2 us more.
//
// Candidates are found with a threshold that is sure to keep n_out of them: of 32 lanes' maxima (distinct elements) the
// n_out-th largest.  What reaches it goes to a list, what still reaches the last threshold to another, and an entry's place in
// the result is the number of better ones there.  Where a list runs over (rows of few values) the best are taken one after the
// other instead.
// Ties go to the lower beam, then the lower token.  Logits of -inf are no candidates, nor is anything of a beam whose score is
// -inf or NaN (its row is not read) or whose sum is not finite (a NaN or +inf among its logits).
#include "kv_share.cuh"
#include "rows_dev.cuh"

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32, kVecs = 4, kBatch = kThreads * kVecs * 4;   // logits a CTA has in hand
constexpr uint32_t kList = 1024, kMaxLists = 1024;
constexpr uint32_t kNone = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
    wr_beam_args a;
    uint32_t parts, batches;             // parts of a row; batches of a part
    float2 *sums;                        // [row][part]: largest logit, sum of exponentials against it
    uint2 *best;                         // [row][part][n_out]: logit's bits, token; in order
    int *done;                           // [request]: parts that are there
};
// A CTA's shared memory: while it works on its part, and on a request's parts.
struct PartMemory {
    float v[kList], lane_top[kThreads], warp_m[kWarps], warp_s[kWarps], kept_v[kList];
    uint32_t i[kList], kept_i[kList], count, kept;
    int least;                           // the threshold, as a whole number in the order of floats
};
struct FinalMemory {
    double offset[WR_CUDA_BATCH_MAX], head[kMaxLists], t[kList], warp_t[kWarps];
    uint32_t b[kList], i[kList], count;
};
union Memory {
    PartMemory part;
    FinalMemory all;
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T> __device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
// The warp's values in descending order across its lanes.
template <typename T> __device__ __forceinline__ T warp_sort(T v, uint32_t lane)
{
#pragma unroll
    for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (uint32_t d = size >> 1; d >= 1; d >>= 1) {
            const T w = __shfl_xor_sync(0xffffffffu, v, d);
            const bool top = ((lane & d) == 0) == ((lane & size) == 0 || size == 32);     // this lane keeps the larger
            v = top == (w > v) ? w : v;
        }
    return v;
}
// the better of two candidates
__device__ __forceinline__ bool before(float v, uint32_t i, float w, uint32_t j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ const float *row_of(const wr_beam_args &a, uint32_t r) { return a.logits + (size_t)(a.mapped ? a.map[r] : r) * a.ld; }

// a < b in the order of results: the logit or total, then the beam, then the token
__device__ __forceinline__ bool before(double v, uint32_t b, uint32_t i, double w, uint32_t c, uint32_t j)
{
    return v > w || (v == w && (b < c || (b == c && i < j)));
}
__device__ __forceinline__ int order(float v) { const int i = __float_as_int(v); return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ float value(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
// sums of exponentials against two maxima as one
__device__ __forceinline__ void join(float &m, float &s, float m2, float s2)
{
    const float t = fmaxf(m, m2), base = t == -INFINITY ? 0.f : t;
    s = s * ex2((m - base) * kLog2e) + s2 * ex2((m2 - base) * kLog2e);
    m = t;
}

__device__ __forceinline__ void part_of_row(const BeamParams &p, PartMemory &sm, uint32_t part, uint32_t row)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = p.a.n_out;
    uint2 *const best = p.best + ((size_t)row * p.parts + part) * k;
    const float score = p.a.scores[row];
    if (!(score > -INFINITY)) {          // (NaN too)
        if (threadIdx.x == 0) p.sums[(size_t)row * p.parts + part] = make_float2(-INFINITY, 0.f);
        if (threadIdx.x < k) best[threadIdx.x] = make_uint2(__float_as_uint(-INFINITY), kNone);
        return;
    }
    // Vectors are aligned in memory: the row begins `lead` elements into the first one.
    const float *const x = row_of(p.a, row);
    const uint32_t lead = (uint32_t)((uintptr_t)x >> 2) & 3u;
    const uint64_t first = (uint64_t)part * p.batches * kBatch, end = (uint64_t)p.a.vocab + lead;
    auto load = [&](uint32_t b, float (&v)[4 * kVecs]) {
#pragma unroll
        for (uint32_t u = 0; u < kVecs; ++u) {
            const uint64_t at = first + (uint64_t)b * kBatch + (u * kThreads + threadIdx.x) * 4u;
            if (at >= lead && at + 4 <= end) {
                const float4 w = __ldcs(reinterpret_cast<const float4 *>(x + (at - lead)));
                v[4 * u] = w.x; v[4 * u + 1] = w.y; v[4 * u + 2] = w.z; v[4 * u + 3] = w.w;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[4 * u + e] = at + e >= lead && at + e < end ? __ldcs(x + (at + e - lead)) : -INFINITY;
            }
        }
    };
    auto token_of = [&](uint32_t b, uint32_t e) {
        return (uint32_t)(first + (uint64_t)b * kBatch + ((e / 4) * kThreads + threadIdx.x) * 4u + (e & 3) - lead);
    };
    float v[4 * kVecs], next[4 * kVecs], m = -INFINITY, s = 0.f;
    load(0, v);
    if (threadIdx.x == 0) {
        sm.count = sm.kept = 0;
        sm.least = order(-INFINITY);
    }
    __syncthreads();
    for (uint32_t b = 0; b < p.batches; ++b) {
        if (first + (uint64_t)b * kBatch >= end) break;
        if (b + 1 < p.batches) load(b + 1, next);
        float top = -INFINITY;
#pragma unroll
        for (uint32_t e = 0; e < 4 * kVecs; ++e) top = fmaxf(top, v[e]);
        const float was = m;
        m = fmaxf(m, top);
        const float base = m == -INFINITY ? 0.f : m;
        s *= ex2((was - base) * kLog2e);
#pragma unroll
        for (uint32_t e = 0; e < 4 * kVecs; ++e) s += ex2((v[e] - base) * kLog2e);
        // A threshold from what every lane has seen.  (Of more than 16, a warp's lanes alone let too many through: the first batch
        // asks all the CTA's.)
        float bound;
        if (k > 16 && b == 0) {
            sm.lane_top[threadIdx.x] = m;
            __syncthreads();
            uint32_t larger_ones = 0;
            for (uint32_t i = 0; i < kThreads; i += 4) {
                const float4 w = *reinterpret_cast<const float4 *>(sm.lane_top + i);
                larger_ones += (w.x > m || (w.x == m && i < threadIdx.x)) + (w.y > m || (w.y == m && i + 1 < threadIdx.x)) +
                               (w.z > m || (w.z == m && i + 2 < threadIdx.x)) + (w.w > m || (w.w == m && i + 3 < threadIdx.x));
            }
            if (larger_ones == k - 1) sm.least = order(m);
            __syncthreads();
            bound = value(sm.least);
        } else {
            // (a warp's threshold moves when one of its lanes' maxima does)
            if (__any_sync(0xffffffffu, m > was)) {
                const float kth = __shfl_sync(0xffffffffu, warp_sort(m, lane), k - 1);
                if (lane == 0) atomicMax(&sm.least, order(kth));
            }
            if (b == 0) __syncthreads();
            bound = value(*(volatile int *)&sm.least);           // (whichever warps have answered: any of their bounds is one)
        }
        if (top >= bound) {
#pragma unroll
            for (uint32_t e = 0; e < 4 * kVecs; ++e)
                if (v[e] >= bound && v[e] > -INFINITY) {
                    const uint32_t at = atomicAdd(&sm.count, 1);
                    if (at < kList) {
                        sm.v[at] = v[e];
                        sm.i[at] = token_of(b, e);
                    }
                }
        }
#pragma unroll
        for (uint32_t e = 0; e < 4 * kVecs; ++e) v[e] = next[e];
    }
    // the part's sum: lanes, then warps, in order
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        join(m, s, m2, s2);
    }
    if (lane == 0) {
        sm.warp_m[warp] = m;
        sm.warp_s[warp] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kWarps; ++w) join(m, s, sm.warp_m[w], sm.warp_s[w]);
        p.sums[(size_t)row * p.parts + part] = make_float2(m, s);
    }
    const uint32_t listed = sm.count;
    if (listed <= kList) {
        const float bound = value(sm.least);                     // (it has grown since most entries were listed)
        for (uint32_t i = threadIdx.x; i < listed; i += kThreads)
            if (sm.v[i] >= bound) {
                const uint32_t at = atomicAdd(&sm.kept, 1);
                sm.kept_v[at] = sm.v[i];
                sm.kept_i[at] = sm.i[i];
            }
        __syncthreads();
        const uint32_t n = sm.kept;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float w = sm.kept_v[i];
            const uint32_t at = sm.kept_i[i];
            uint32_t place = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < n; ++j) place += before(sm.kept_v[j], sm.kept_i[j], w, at);
            if (place < k) best[place] = make_uint2(__float_as_uint(w), at);
        }
        if (threadIdx.x >= n && threadIdx.x < k) best[threadIdx.x] = make_uint2(__float_as_uint(-INFINITY), kNone);
        return;
    }
    // too many for the list: the largest, then the largest behind it, and so on
    float last_v = INFINITY;
    uint32_t last_i = 0;
    bool started = false;
    for (uint32_t j = 0; j < k; ++j) {
        float top_v = -INFINITY;
        uint32_t top_i = kNone;
        for (uint32_t b = 0; b < p.batches; ++b) {
            load(b, v);
#pragma unroll
            for (uint32_t e = 0; e < 4 * kVecs; ++e) {
                const uint32_t at = token_of(b, e);
                if (v[e] > -INFINITY && (!started || before(last_v, last_i, v[e], at)) && before(v[e], at, top_v, top_i)) {
                    top_v = v[e];
                    top_i = at;
                }
            }
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, top_v, o);
            const uint32_t at = __shfl_xor_sync(0xffffffffu, top_i, o);
            if (before(w, at, top_v, top_i)) top_v = w, top_i = at;
        }
        __syncthreads();
        if (lane == 0) {
            sm.v[warp] = top_v;
            sm.i[warp] = top_i;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kWarps; ++w)
            if (before(sm.v[w], sm.i[w], top_v, top_i)) top_v = sm.v[w], top_i = sm.i[w];
        if (threadIdx.x == 0) best[j] = make_uint2(__float_as_uint(top_v), top_i);
        started = true;
        last_v = top_v;
        last_i = top_i;
    }
}

__device__ __forceinline__ void parts_of_request(const BeamParams &p, FinalMemory &sm, uint32_t group)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = p.a.n_out, beams = p.a.beams;
    const size_t row0 = (size_t)group * beams;
    const uint32_t lists = beams * p.parts;
    const uint2 *const best = p.best + row0 * p.parts * k;
    // every list's best, on its way while the sums are put together
    float mine[(kMaxLists + kThreads - 1) / kThreads];
#pragma unroll
    for (uint32_t u = 0; u < kMaxLists / kThreads; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads;
        if (i < lists) mine[u] = __uint_as_float(__ldcg(&best[(size_t)i * k].x));
    }
    if (threadIdx.x == 0) sm.count = 0;
    // score less the logarithm of the row's sum
    for (uint32_t b = warp; b < beams; b += kWarps) {
        const float2 *sums = p.sums + (row0 + b) * p.parts;
        float top = -INFINITY;
        for (uint32_t i = lane; i < p.parts; i += 32) top = fmaxf(top, __ldcg(sums + i).x);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        double s = 0.0;
        for (uint32_t i = lane; i < p.parts; i += 32) {
            const float2 ms = __ldcg(sums + i);
            if (ms.y != 0.f) s += (double)ms.y * exp((double)ms.x - (double)top);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const double t = (double)p.a.scores[row0 + b] - ((double)top + log(s));
        if (lane == 0) sm.offset[b] = t > -INFINITY && t < INFINITY ? t : -INFINITY;         // (no sum, or none that is finite)
    }
    __syncthreads();
    // a bound from 32 threads' best
    double top = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < kMaxLists / kThreads; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads;
        if (i >= lists) continue;
        sm.head[i] = sm.offset[i / p.parts] + (double)mine[u];
        top = larger(top, sm.head[i]);
    }
    const double kth = __shfl_sync(0xffffffffu, warp_sort(top, lane), k - 1);
    if (lane == 0) sm.warp_t[warp] = kth;
    __syncthreads();
    double bound = sm.warp_t[0];
    for (uint32_t w = 1; w < kWarps; ++w) bound = larger(bound, sm.warp_t[w]);
    // a warp to a list that reaches it
    for (uint32_t i = warp; i < lists; i += kWarps) {
        if (!(sm.head[i] >= bound && sm.head[i] > -INFINITY) || lane >= k) continue;
        const uint2 c = __ldcg(best + (size_t)i * k + lane);
        const double t = sm.offset[i / p.parts] + (double)__uint_as_float(c.x);
        if (!(t >= bound && t > -INFINITY)) continue;
        const uint32_t at = atomicAdd(&sm.count, 1);
        if (at < kList) {
            sm.t[at] = t;
            sm.b[at] = i / p.parts;
            sm.i[at] = c.y;
        }
    }
    __syncthreads();
    const uint32_t n = sm.count;
    float *const out_s = p.a.out_scores + (size_t)group * k;
    uint32_t *const out_b = p.a.out_beams + (size_t)group * k, *const out_t = p.a.out_tokens + (size_t)group * k;
    if (n <= kList) {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const double t = sm.t[i];
            const uint32_t b = sm.b[i], at = sm.i[i];
            uint32_t place = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < n; ++j) place += before(sm.t[j], sm.b[j], sm.i[j], t, b, at);
            if (place < k) {
                out_s[place] = (float)t;
                out_b[place] = b;
                out_t[place] = at;
            }
        }
        if (threadIdx.x >= n && threadIdx.x < k) {
            out_s[threadIdx.x] = -INFINITY;
            out_b[threadIdx.x] = out_t[threadIdx.x] = kNone;
        }
        return;
    }
    double last = INFINITY;
    uint32_t last_b = 0, last_i = 0;
    for (uint32_t place = 0; place < k; ++place) {
        double t = -INFINITY;
        uint32_t b = kNone, at = kNone;
        for (uint32_t i = threadIdx.x; i < lists * k; i += kThreads) {
            const uint2 e = __ldcg(best + i);
            const uint32_t of = i / k / p.parts;
            const double c = sm.offset[of] + (double)__uint_as_float(e.x);
            if (c > -INFINITY && (!place || before(last, last_b, last_i, c, of, e.y)) && before(c, of, e.y, t, b, at)) t = c, b = of, at = e.y;
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            const double c = __shfl_xor_sync(0xffffffffu, t, o);
            const uint32_t of = __shfl_xor_sync(0xffffffffu, b, o), token = __shfl_xor_sync(0xffffffffu, at, o);
            if (before(c, of, token, t, b, at)) t = c, b = of, at = token;
        }
        __syncthreads();
        if (lane == 0) {
            sm.t[warp] = t;
            sm.b[warp] = b;
            sm.i[warp] = at;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kWarps; ++w)
            if (before(sm.t[w], sm.b[w], sm.i[w], t, b, at)) t = sm.t[w], b = sm.b[w], at = sm.i[w];
        if (threadIdx.x == 0) {
            out_s[place] = (float)t;
            out_b[place] = b;
            out_t[place] = at;
        }
        last = t;
        last_b = b;
        last_i = at;
    }
}

__global__ void __launch_bounds__(kThreads) beam_select_kernel(const __grid_constant__ BeamParams p)
{
    __shared__ Memory sm;
    __shared__ bool last;
    pdl_wait();
    pdl_trigger();
    part_of_row(p, sm.part, blockIdx.x, blockIdx.y);
    // the request's last part to be there finds all the others
    const uint32_t group = blockIdx.y / p.a.beams, parts = p.a.beams * p.parts;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(p.done + group, 1) == (int)parts - 1;
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) p.done[group] = 0;
    parts_of_request(p, sm.all, group);
}

}  // namespace

int wr_beam_validate(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t n_out)
{
    if (groups == 0 || beams == 0 || vocab == 0 || n_out == 0) return WR_CUDA_ERR_INVAL;
    if (beams > WR_CUDA_BATCH_MAX || n_out > WR_CUDA_BEAM_MAX_OUT || (uint64_t)groups * beams > 65535u || vocab > 0x7fffffffu)
        return WR_CUDA_ERR_LIMIT;
    return WR_CUDA_OK;
}

int wr_beam_launch(wr_cuda_ctx *ctx, const wr_beam_args &a)
{
    BeamParams p{};
    p.a = a;
    const uint32_t rows = a.groups * a.beams, most = (uint32_t)(((uint64_t)a.vocab + 3 + kBatch - 1) / kBatch);
    // four CTAs to an SM are enough to keep its loads under way
    const uint32_t want = std::min(std::max(4u * (uint32_t)ctx->sm_count / rows, 1u), std::min(most, kMaxLists / a.beams));
    p.batches = (most + want - 1) / want;
    p.parts = (most + p.batches - 1) / p.batches;
    const size_t n = (size_t)rows * p.parts, sums = (n * sizeof(float2) + 255) & ~(size_t)255;
    char *ws = nullptr;
    int rc = wr_ctx_keep(ctx, WR_KEPT_HEAD + sums + n * a.n_out * sizeof(uint2), &ws);
    if (rc != WR_CUDA_OK) return rc;
    p.done = reinterpret_cast<int *>(ws + WR_KEPT_HEAD / 2);
    p.sums = reinterpret_cast<float2 *>(ws + WR_KEPT_HEAD);
    p.best = reinterpret_cast<uint2 *>(ws + WR_KEPT_HEAD + sums);
    WR_CUDA_TRY(wr_launch_pdl(beam_select_kernel, dim3(p.parts, rows), dim3(kThreads), (size_t)0, ctx->stream, p));
    return finish_launch(ctx);
}

extern "C" int wr_cuda_beam_select(wr_cuda_ctx *ctx, uint32_t n_groups, uint32_t beams, uint32_t vocab, const float *logits,
                                   const float *scores, uint32_t n_out, float *out_scores, uint32_t *out_beams, uint32_t *out_tokens,
                                   int mem)
{
    if (!ctx || !logits || !scores || !out_scores || !out_beams || !out_tokens) return WR_CUDA_ERR_INVAL;
    if (mem != WR_CUDA_MEM_HOST && mem != WR_CUDA_MEM_DEVICE) return WR_CUDA_ERR_INVAL;
    int rc = wr_beam_validate(n_groups, beams, vocab, n_out);
    if (rc != WR_CUDA_OK) return rc;
    std::lock_guard<std::mutex> g(ctx->lock);
    WR_CUDA_TRY(cudaSetDevice(ctx->device));
    wr_beam_args a{};
    a.groups = n_groups;
    a.beams = beams;
    a.vocab = vocab;
    a.n_out = n_out;
    a.ld = vocab;
    if (mem == WR_CUDA_MEM_DEVICE) {
        a.logits = logits;
        a.scores = scores;
        a.out_scores = out_scores;
        a.out_beams = out_beams;
        a.out_tokens = out_tokens;
        return wr_beam_launch(ctx, a);
    }
    const size_t rows = (size_t)n_groups * beams, outs = (size_t)n_groups * n_out, l = rows * vocab * 4, s = (rows * 4 + 255) & ~(size_t)255;
    rc = wr_ctx_reserve_stage(ctx, l + 2 * s + outs * 12, 0);
    if (rc != WR_CUDA_OK) return rc;
    char *d = (char *)ctx->stage_dev;
    WR_CUDA_TRY(cudaMemcpyAsync(d, logits, l, cudaMemcpyHostToDevice, ctx->stream));
    WR_CUDA_TRY(cudaMemcpyAsync(d + l, scores, rows * 4, cudaMemcpyHostToDevice, ctx->stream));
    a.logits = (const float *)d;
    a.scores = (const float *)(d + l);
    a.out_scores = (float *)(d + l + s);
    a.out_beams = (uint32_t *)(a.out_scores + outs);
    a.out_tokens = a.out_beams + outs;
    rc = wr_beam_launch(ctx, a);
    if (rc != WR_CUDA_OK) return rc;
    WR_CUDA_TRY(cudaMemcpyAsync(out_scores, a.out_scores, outs * 4, cudaMemcpyDeviceToHost, ctx->stream));
    WR_CUDA_TRY(cudaMemcpyAsync(out_beams, a.out_beams, outs * 4, cudaMemcpyDeviceToHost, ctx->stream));
    WR_CUDA_TRY(cudaMemcpyAsync(out_tokens, a.out_tokens, outs * 4, cudaMemcpyDeviceToHost, ctx->stream));
    return wr_ctx_sync_checked(ctx);
}
