// beam.cu — a beam search's choice: for every request the n_out best of beams x vocabulary by
//     total(b, v) = score_b + logit(b, v) - log sum_u exp(logit(b, u))
// The reference has no beam search; its sampler takes one row of logits (src/core/sample.c:239).
//
// One pass over the logits: a CTA takes a part of a row and leaves the part's sum of exponentials (against the part's
// maximum) and its n_out best logits; within a row totals are in the order of logits, so nothing else of the part can be
// among the row's best.  The CTA that is the last of its request puts the parts together.  Totals are 64-bit, since candidates of two
// beams may lie closer than an F32 rounding; a part's sum is F32 (a thread's terms, ex2.approx, then lanes and warps against the largest maximum),
// the parts' are added up in 64 bits: a row's logarithm is off by up to 4.3e-7 (16 rows of 1000 to 600000 logits of spread 0 to 6, in parts of one
// batch and of 37).  Rows of a call that are alike have sums alike, to the bit, so that their candidates tie.  Measured on a B200: one row of 32003 logits, 8 out, 7.0 us on
// the device, round trips one behind the other (a second kernel for the parts took 2 us more); 256 rows of 65536, 16 out, 18.8 us,
// 3.6 TB/s (67 MB, which stay in L2; 22.6 us from HBM), bound by instructions (comparing with the bound four logits at a time took 1.2 us off; more batches under way, two or three
// copies to shared memory a CTA, made it 24.7 and 26.0 us).
//
// Candidates are found with a threshold that is sure to keep n_out of them: of 32 threads' maxima (distinct elements) the
// n_out-th largest.  What reaches it goes to a list; where that are many, a higher threshold is looked for by halving; and an entry's
// place in the result is the number of better ones in the list.  Where a list runs over (rows of few values) the best are taken one
// after the other instead.
// Ties go to the lower beam, then the lower token.  Logits of -inf are no candidates, nor is anything of a beam whose score is
// -inf or NaN (its row is not read) or whose sum is not finite (a NaN or +inf among its logits).
#include <cfloat>

#include "kv_share.cuh"
#include "rows_dev.cuh"

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32, kVecs = 4, kBatch = kThreads * kVecs * 4;   // logits a CTA has in hand
constexpr uint32_t kList = 1024, kOwn = 6, kMaxLists = kOwn * kThreads;       // kOwn: a thread's entries of a request's
constexpr uint32_t kCtas = 4;             // to an SM (5, with 48 registers a thread: 256 rows 25.8 us; 16 rows 10.3 instead of 10.9)
constexpr uint32_t kNone = 0xffffffffu;
static_assert(kList / WR_CUDA_BEAM_MAX_OUT >= WR_CUDA_BEAM_MAX_OUT, "");
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
    wr_beam_args a;
    uint32_t parts, batches;             // parts of a row; batches of a part
    bool vectors;                        // all rows begin on 16 bytes
    float2 *sums;                        // [row][part]: largest logit, sum of exponentials against it
    uint2 *best;                         // [row][part][n_out]: logit's bits, token; in order
    int *done;                           // [request]: parts that are there
};
// A CTA's shared memory: while it works on its part, and on a request's parts.
struct PartMemory {
    uint64_t listed[kList], kept[kList]; // keys
    float top[2][32], warp_m[kWarps], warp_s[kWarps];
    uint32_t count[2][kWarps];
    uint32_t n_listed, n_kept;
};
struct FinalMemory {
    double offset[WR_CUDA_BATCH_MAX];
    float top[32];
    uint32_t count[2][kWarps], most[kWarps];
    uint64_t t[kList], at[kList];        // totals in the order of whole numbers; beam and token
    uint32_t n;
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
__device__ __forceinline__ const float *row_of(const wr_beam_args &a, uint32_t r) { return a.logits + (size_t)(a.mapped ? a.map[r] : r) * a.ld; }

__device__ __forceinline__ int order(float v) { const int i = __float_as_int(v); return i ^ ((i >> 31) & 0x7fffffff); }
__device__ __forceinline__ float value(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
// A row's candidate as one number, the better the larger: the logit, then the lower token.  (-0 and 0 are equal.)
__device__ __forceinline__ uint64_t key_of(float v, uint32_t token)
{
    return (uint64_t)((uint32_t)order(v + 0.f) ^ 0x80000000u) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint64_t key) { return value((int)((uint32_t)(key >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ uint64_t key_of(double t)
{
    const long long i = __double_as_longlong(t + 0.0);
    return (uint64_t)(i ^ ((i >> 63) & 0x7fffffffffffffffll)) ^ 0x8000000000000000ull;
}
__device__ __forceinline__ double total_of(uint64_t key)
{
    const long long i = (long long)(key ^ 0x8000000000000000ull);
    return __longlong_as_double(i ^ ((i >> 63) & 0x7fffffffffffffffll));
}
// The places of n entries in their order, by counting the better ones; eight threads to an entry.
template <typename Better, typename Place> __device__ __forceinline__ void rank(uint32_t n, Better better, Place place)
{
    const uint32_t sub = threadIdx.x & 7;
    for (uint32_t i0 = 0; i0 < n; i0 += kThreads / 8) {
        const uint32_t i = i0 + threadIdx.x / 8;
        uint32_t count = 0;
        if (i < n) {
#pragma unroll 4
            for (uint32_t j = sub; j < n; j += 8) count += better(j, i);
        }
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
        if (i < n && sub == 0) place(i, count);
    }
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// A number that k of all threads' values reach: of every warp's four largest, 32 together, the k-th.  (One that k of a warp's own reach
// lets eight times as many through.)  The CTA meets in it; `top` is not used again before it has met once more.
static_assert(kWarps * 4 == 32, "");
__device__ __forceinline__ float bound_of_all(float (&top)[32], float v, uint32_t k, uint32_t warp, uint32_t lane)
{
    const float sorted = warp_sort(v, lane);
    if (lane < 4) top[4 * warp + lane] = sorted;
    __syncthreads();
    return __shfl_sync(0xffffffffu, warp_sort(top[lane], lane), k - 1);
}
// The lanes' sums of exponentials, each against its own maximum, as one.
__device__ __forceinline__ float warp_max(float v) { return value(__reduce_max_sync(0xffffffffu, order(v))); }
__device__ __forceinline__ float shrunk(float from, float to) { return ex2((from - (to == -INFINITY ? 0.f : to)) * kLog2e); }
template <typename T> __device__ __forceinline__ void warp_join(float &m, T &s)
{
    const float top = warp_max(m);
    s *= (T)shrunk(m, top);
    m = top;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
}
// A bound, as the whole number in whose order it is, that k entries reach as well as the given one, but no more than `enough` where such a one
// is found: halving what lies between that and the largest.  reach(x): how many of the thread's own reach x.  The CTA meets in it.
template <typename Reach> __device__ __forceinline__ uint32_t higher_bound(uint32_t (&counts)[2][kWarps], Reach reach, uint32_t lo, uint32_t hi, uint32_t k,
                                                                           uint32_t enough, uint32_t warp, uint32_t lane)
{
    uint32_t mid = lo;
    for (uint32_t turn = 0;; ++turn) {
        uint32_t n = __reduce_add_sync(0xffffffffu, reach(mid));
        if (lane == 0) counts[turn & 1][warp] = n;
        __syncthreads();
        n = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) n += counts[turn & 1][w];
        if (turn && n < k) hi = mid;
        else lo = mid;
        if ((n <= enough && (n >= k || !turn)) || hi - lo <= 1 || hi < lo) return lo;
        mid = lo + (hi - lo) / 2;
    }
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
    // Which tokens a thread takes is the same in all rows of a call, so rows alike have sums alike, to the bit.  Four neighbours at a time where every
    // row is aligned (p.vectors), else every 256th: a warp's loads are neighbours then.  (32 x 8 rows of 65537: 19.9 us; four neighbours by single
    // loads 22.2.  Every 32nd leaves a part of few logits to one warp, whose four largest are a low bound: 4 x 151937 11.7 instead of 7.9.)
    const float *const x = row_of(p.a, row);
    const uint32_t first = part * p.batches * kBatch, end = p.a.vocab;       // (below 2^31; a batch more is below 2^32)
    auto load = [&](uint32_t b, float (&v)[4 * kVecs]) {
        const uint32_t lo = first + b * kBatch;
        const bool whole = lo + kBatch <= end;
        if (!p.vectors) {
            const float *const from = x + lo + threadIdx.x;
            if (whole) {
#pragma unroll
                for (uint32_t e = 0; e < 4 * kVecs; ++e) v[e] = __ldcs(from + kThreads * e);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4 * kVecs; ++e) v[e] = lo + threadIdx.x + kThreads * e < end ? __ldcs(from + kThreads * e) : -INFINITY;
            }
            return;
        }
        const float4 *const from = reinterpret_cast<const float4 *>(x + lo) + threadIdx.x;
        if (whole) {
#pragma unroll
            for (uint32_t u = 0; u < kVecs; ++u) {
                const float4 w = __ldcs(from + u * kThreads);
                v[4 * u] = w.x; v[4 * u + 1] = w.y; v[4 * u + 2] = w.z; v[4 * u + 3] = w.w;
            }
            return;
        }
#pragma unroll
        for (uint32_t u = 0; u < kVecs; ++u) {
            const uint32_t at = lo + (u * kThreads + threadIdx.x) * 4u;
            if (at + 4 <= end) {
                const float4 w = __ldcs(from + u * kThreads);
                v[4 * u] = w.x; v[4 * u + 1] = w.y; v[4 * u + 2] = w.z; v[4 * u + 3] = w.w;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[4 * u + e] = at + e < end ? __ldcs(x + at + e) : -INFINITY;
            }
        }
    };
    auto token_of = [&](uint32_t b, uint32_t e) {
        return first + b * kBatch + (p.vectors ? ((e / 4) * kThreads + threadIdx.x) * 4u + (e & 3) : e * kThreads + threadIdx.x);
    };
    float v[4 * kVecs], next[4 * kVecs], m = -INFINITY, bound = -FLT_MAX;
    uint64_t s2 = 0;                     // two sums of exponentials
    load(0, v);
    if (threadIdx.x == 0) {
        sm.n_listed = sm.n_kept = 0;
    }
    __syncthreads();
    const uint32_t batches = first < end ? min(p.batches, (end - first + kBatch - 1) / kBatch) : 0u;
    for (uint32_t b = 0; b < batches; ++b) {
        if (b + 1 < batches) load(b + 1, next);
        float tops[kVecs], top = -INFINITY;
#pragma unroll
        for (uint32_t u = 0; u < kVecs; ++u) tops[u] = max3(fmaxf(v[4 * u], v[4 * u + 1]), v[4 * u + 2], v[4 * u + 3]);
#pragma unroll
        for (uint32_t u = 0; u < kVecs; u += 2) top = max3(top, tops[u], tops[u + 1]);
        const float was = m;
        m = fmaxf(m, top);
        const float base = m == -INFINITY ? 0.f : m, shrink = ex2((was - base) * kLog2e);
        s2 = mul2(s2, pack2(shrink, shrink));
#pragma unroll
        for (uint32_t e = 0; e < 4 * kVecs; e += 2) {
            float d0, d1;
            unpack2(mul2(add2(pack2(v[e], v[e + 1]), pack2(-base, -base)), pack2(kLog2e, kLog2e)), d0, d1);
            s2 = add2(s2, pack2(ex2(d0), ex2(d1)));
        }
        // a threshold from what every thread has seen, looked for again whenever that has doubled
        // (not in the words of the last time: some may still be reading those)
        if ((b & (b + 1)) == 0) bound = fmaxf(bound_of_all(sm.top[__popc(b) & 1], m, k, warp, lane), -FLT_MAX);
        if (top >= bound) {
#pragma unroll
            for (uint32_t u = 0; u < kVecs; ++u) {
                if (tops[u] < bound) continue;
                uint32_t n = 0;
#pragma unroll
                for (uint32_t e = 4 * u; e < 4 * u + 4; ++e) n += v[e] >= bound;
                uint32_t at = atomicAdd(&sm.n_listed, n);
#pragma unroll
                for (uint32_t e = 4 * u; e < 4 * u + 4; ++e)
                    if (v[e] >= bound) {
                        if (at < kList) sm.listed[at] = key_of(v[e], token_of(b, e));
                        ++at;
                    }
            }
        }
#pragma unroll
        for (uint32_t e = 0; e < 4 * kVecs; ++e) v[e] = next[e];
    }
    // the part's sum: lanes, then warps, in order
    float s, half;
    unpack2(s2, s, half);
    s += half;
    warp_join(m, s);
    if (lane == 0) {
        sm.warp_m[warp] = m;
        sm.warp_s[warp] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
        for (uint32_t w = 1; w < kWarps; ++w) m = fmaxf(m, sm.warp_m[w]);
        for (uint32_t w = 0; w < kWarps; ++w) s = fmaf(sm.warp_s[w], shrunk(sm.warp_m[w], m), s);
        p.sums[(size_t)row * p.parts + part] = make_float2(m, s);
    }
    uint32_t n = sm.n_listed;
    if (n <= kList) {
        // As many comparisons to an entry as there are entries: fewer first, those that reach the last bound or, where these are many (a part
        // of which some warps have little; 16 beams of 5000 logits, 32 out: 53 us), a higher one.
        const uint64_t *list = sm.listed;
        const uint32_t enough = 5 * k;
        uint32_t least = (uint32_t)(key_of(bound, 0) >> 32);
        if (n > enough) {
            auto reach = [&](uint32_t x) {
                uint32_t c = 0;
                for (uint32_t i = threadIdx.x; i < n; i += kThreads) c += (uint32_t)(sm.listed[i] >> 32) >= x;
                return c;
            };
            float most = sm.warp_m[0];
#pragma unroll
            for (uint32_t w = 1; w < kWarps; ++w) most = fmaxf(most, sm.warp_m[w]);
            least = higher_bound(sm.count, reach, least, (uint32_t)(key_of(most, 0) >> 32), k, enough, warp, lane);
        }
        if (batches > 1 || n > enough) {
            for (uint32_t i = threadIdx.x; i < n; i += kThreads)
                if ((uint32_t)(sm.listed[i] >> 32) >= least) sm.kept[atomicAdd(&sm.n_kept, 1)] = sm.listed[i];
            __syncthreads();
            n = sm.n_kept;
            list = sm.kept;
        }
        rank(n, [&](uint32_t j, uint32_t i) { return list[j] > list[i]; },
             [&](uint32_t i, uint32_t place) { if (place < k) best[place] = make_uint2(__float_as_uint(logit_of(list[i])), ~(uint32_t)list[i]); });
        if (threadIdx.x >= n && threadIdx.x < k) best[threadIdx.x] = make_uint2(__float_as_uint(-INFINITY), kNone);
        return;
    }
    // too many for the list: the largest, then the largest behind it, and so on
    uint64_t last = ~0ull;
    for (uint32_t j = 0; j < k; ++j) {
        uint64_t most = 0;
        for (uint32_t b = 0; b < batches; ++b) {
            load(b, v);
#pragma unroll
            for (uint32_t e = 0; e < 4 * kVecs; ++e) {
                const uint64_t key = key_of(v[e], token_of(b, e));
                if (v[e] > -INFINITY && key < last && key > most) most = key;
            }
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) most = larger(most, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)most, o));
        __syncthreads();
        if (lane == 0) sm.listed[warp] = most;
        __syncthreads();
        for (uint32_t w = 0; w < kWarps; ++w) most = larger(most, sm.listed[w]);
        if (threadIdx.x == 0) best[j] = most ? make_uint2(__float_as_uint(logit_of(most)), ~(uint32_t)most) : make_uint2(__float_as_uint(-INFINITY), kNone);
        last = most;
    }
}

__device__ __forceinline__ void parts_of_request(const BeamParams &p, FinalMemory &sm, uint32_t group)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k = p.a.n_out, beams = p.a.beams;
    const size_t row0 = (size_t)group * beams;
    const uint32_t lists = beams * p.parts;
    const uint2 *const best = p.best + row0 * p.parts * k;
    // Few candidates: all of them are on their way while the sums are put together.  Many: the first of every list.
    const bool few = lists * k <= kOwn * kThreads;
    uint2 mine[kOwn];
#pragma unroll
    for (uint32_t u = 0; u < kOwn; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads;
        mine[u] = make_uint2(__float_as_uint(-INFINITY), kNone);
        if (i < (few ? lists * k : lists)) mine[u] = __ldcg(best + (few ? i : (size_t)i * k));
    }
    if (threadIdx.x == 0) sm.n = 0;
    // score less the logarithm of the row's sum
    for (uint32_t b = warp; b < beams; b += kWarps) {
        float m = -INFINITY;
        double s = 0.0;
        for (uint32_t i = lane; i < p.parts; i += 32) {
            const float2 ms = __ldcg(p.sums + (row0 + b) * p.parts + i);
            const float top = fmaxf(m, ms.x);
            s = s * (double)shrunk(m, top) + (double)ms.y * (double)shrunk(ms.x, top);
            m = top;
        }
        warp_join(m, s);
        const double t = (double)p.a.scores[row0 + b] - ((double)m + log(s));
        if (lane == 0) sm.offset[b] = t > -INFINITY && t < INFINITY ? t : -INFINITY;         // (no sum, or none that is finite)
    }
    __syncthreads();
    // a bound from the threads' best, rounded down
    const uint32_t per_beam = few ? p.parts * k : p.parts;
    double total[kOwn], top = -INFINITY;
#pragma unroll
    for (uint32_t u = 0; u < kOwn; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads;
        const double offset = i < beams * per_beam ? sm.offset[i / per_beam] : -INFINITY;
        total[u] = offset > -INFINITY ? offset + (double)__uint_as_float(mine[u].x) : -INFINITY;      // (no NaN from an infinite logit)
        top = larger(top, total[u]);
    }
    // (a few are ranked as quickly as a bound is found: 32 / 64 / 128 candidates 6.4 / 7.0 / 8.2 us without, 7.0 / 7.2 / 7.3 with it)
    float bound = -FLT_MAX;
    if (lists * k > 64) {
        // (No more lists than fill the list.  A warp's totals are one beam's or two: of a beam that is far behind, the four largest are a low bound.  16 beams of 32003 logits, 32
        // out: 1536 candidates reached it, more than the list holds, 115 instead of 15.6 us.)
        const float most = __double2float_rd(top);
        bound = fmaxf(bound_of_all(sm.top, most, k, warp, lane), -FLT_MAX);
        auto reach = [&](uint32_t x) {
            const float least = value((int)(x ^ 0x80000000u));
            uint32_t n = 0;
#pragma unroll
            for (uint32_t u = 0; u < kOwn; ++u) n += total[u] >= least;
            return n;
        };
        const uint32_t largest = __reduce_max_sync(0xffffffffu, (uint32_t)order(most) ^ 0x80000000u);
        if (lane == 0) sm.most[warp] = largest;
        __syncthreads();
        uint32_t hi = sm.most[0];
#pragma unroll
        for (uint32_t w = 1; w < kWarps; ++w) hi = max(hi, sm.most[w]);
        const uint32_t from = (uint32_t)order(bound) ^ 0x80000000u;
        bound = value((int)(higher_bound(sm.count, reach, from, hi, k, few ? 5 * k : kList / k, warp, lane) ^ 0x80000000u));
    }
    auto list = [&](double t, uint32_t b, uint32_t token) {
        if (!(t >= bound)) return;
        const uint32_t at = atomicAdd(&sm.n, 1);
        if (at >= kList) return;
        sm.t[at] = key_of(t);
        sm.at[at] = (uint64_t)b << 32 | token;
    };
#pragma unroll
    for (uint32_t u = 0; u < kOwn; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads, b = i / per_beam;
        if (few) {
            list(total[u], b, mine[u].y);
        } else if (total[u] >= bound) {                          // (whose list begins above it takes all of the list)
            const double offset = sm.offset[b];
#pragma unroll 8
            for (uint32_t j = 0; j < k; ++j) {
                const uint2 c = __ldcg(best + (size_t)i * k + j);
                list(offset + (double)__uint_as_float(c.x), b, c.y);
            }
        }
    }
    __syncthreads();
    const uint32_t n = sm.n;
    float *const out_s = p.a.out_scores + (size_t)group * k;
    uint32_t *const out_b = p.a.out_beams + (size_t)group * k, *const out_t = p.a.out_tokens + (size_t)group * k;
    auto put = [&](uint32_t place, uint64_t t, uint64_t at) {
        out_s[place] = at == ~0ull ? -INFINITY : (float)total_of(t);
        out_b[place] = (uint32_t)(at >> 32);
        out_t[place] = (uint32_t)at;
    };
    if (n <= kList) {
        rank(n, [&](uint32_t j, uint32_t i) { return (sm.t[j] > sm.t[i]) | ((sm.t[j] == sm.t[i]) & (sm.at[j] < sm.at[i])); },
             [&](uint32_t i, uint32_t place) { if (place < k) put(place, sm.t[i], sm.at[i]); });
        if (threadIdx.x >= n && threadIdx.x < k) put(threadIdx.x, 0, ~0ull);
        return;
    }
    // more equal ones than a list holds: one after the other
    uint64_t last = ~0ull, last_at = 0;
    for (uint32_t place = 0; place < k; ++place) {
        uint64_t most = 0, at = ~0ull;
        auto take = [&](uint64_t t, uint64_t of) {
            if (t > most || (t == most && of < at)) most = t, at = of;
        };
        for (uint32_t i = threadIdx.x; i < lists * k; i += kThreads) {
            const uint2 c = __ldcg(best + i);
            const double t = sm.offset[i / k / p.parts] + (double)__uint_as_float(c.x);
            const uint64_t key = key_of(t), of = (uint64_t)(i / k / p.parts) << 32 | c.y;
            if (t > -INFINITY && (!place || key < last || (key == last && of > last_at))) take(key, of);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
            const uint64_t t = __shfl_xor_sync(0xffffffffu, (unsigned long long)most, o), of = __shfl_xor_sync(0xffffffffu, (unsigned long long)at, o);
            take(t, of);
        }
        __syncthreads();
        if (lane == 0) {
            sm.t[warp] = most;
            sm.at[warp] = at;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kWarps; ++w) take(sm.t[w], sm.at[w]);
        if (threadIdx.x == 0) put(place, most, at);
        last = most;
        last_at = at;
    }
}

__global__ void __launch_bounds__(kThreads, kCtas) beam_select_kernel(const __grid_constant__ BeamParams p)
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
        int before;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.done + group) : "memory");
        last = before == (int)parts - 1;
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
    const uint32_t rows = a.groups * a.beams, most = (uint32_t)(((uint64_t)a.vocab + kBatch - 1) / kBatch);
    // As many CTAs as the SMs hold at once.  (Twice as many: 26.7 instead of 22.1 us for 256 rows, 11.7 instead of 11.3 for 16.)
    const uint32_t want = std::min(std::max(kCtas * (uint32_t)ctx->sm_count / rows, 1u), std::min(most, kMaxLists / a.beams));
    p.vectors = ((uintptr_t)a.logits & 15u) == 0 && a.ld % 4 == 0;
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
        // (a request's choice may be there before another's rows have been read; its own scores have been)
        const size_t rows = (size_t)n_groups * beams, outs = (size_t)n_groups * n_out * 4;
        for (const void *out : {(const void *)out_scores, (const void *)out_beams, (const void *)out_tokens})
            if (wr_overlap(out, outs, logits, rows * vocab * 4) ||
                (wr_overlap(out, outs, scores, rows * 4) && !(out == scores && out == out_scores && n_out == beams)))
                return WR_CUDA_ERR_INVAL;
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
