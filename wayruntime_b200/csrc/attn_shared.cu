// attn_shared.cu — decode attention for sessions whose first rows are the same pages (a batch behind one prompt, the beams
// of a search), on the tensor cores.
//
// A row of the result is softmax(scale q K^T) V over the session's keys, and the keys fall into two parts: those that the
// sessions of a group share, and the session's own behind them.  For any split of the keys
//     m = max of the parts' m_i,   l = sum of 2^(m_i - m) l_i,   o = sum of 2^(m_i - m) o_i / l
// (m_i the largest score of a part, in powers of two, l_i and o_i its sums against it), so the shared part is worked out once
// for all queries of the group: a page is fetched from HBM once for up to 64 of them.
//
// A BUNDLE is up to 64 queries of one kv head: some sessions of a group, with the query heads that share the kv head.  Its keys
// are a list of tiles of 128 (two pages): the group's shared rows, then each session's own.  The queries stay where they are for
// the whole list; in a session's own tiles the other sessions' columns get weights of zero.  (Work items of their own for own
// rows began and ended once more for a tile or two, 3 to 4 us each.)  A WORK ITEM is an even share of a bundle's tiles for one kv head.  Persistent CTAs, one per SM,
// draw items from a counter, longest first; when none is left they add the shares of a row up in order (add_up), so results do
// not hang on who worked what out.  Operands are swapped, as in attn_latent.cu: keys are the tensor core's M, queries
// its N, so a tile costs what its queries cost.  Per tile
//   * two loading warps bring K and V in with linear bulk copies (a page's blocks are the operand's layout);
//   * one warp issues S^T[key][query] = K . Q^T and O^T[dim][query] = V^T . P^T; the scores of the next tile are issued
//     before this tile's values, so both buffers of S are in use;
//   * four groups of four warps, each with a quarter of the queries, a thread per key: exponentials against a running reference,
//     P^T to shared memory (queries contiguous: the MN-major operand); then, a thread per value dimension, the tile's O^T is added
//     to sums in registers.  The reference moves when a score is more than 2^8 above the one that it was taken from: the threads vote, and only
//     then is the maximum over keys worked out (a segment's first tile always does).
// Queries and weights are split in two F16 numbers, two products each, the small one first: F32 rows come in and go out, and one F16
// rounding of either would leave 2^-12.  The two leave 2^-22 of a number, or 2^-25 where that is more: F16 ends there.  Queries are
// taken against a power of two of their row; weights against 2^-7 of the largest one, so what is lost of a weight is 2^-32 of that at most (a
// long flat tail behind one large score adds up what is lost of its weights).  Sums of
// one tile stay in the tensor core's accumulator (8 steps of 16 keys behind the small ones), longer ones are F32 additions in
// registers: the accumulator rounds towards zero, which over a long chunk would show.
// Every wait is bounded by the context's wait limit.
// Measured on a B200, F32 rows, 32 query and 8 kv heads, one launch behind another: 16 sessions behind 32768 rows, 145 MB, 33 us, of which
// the tiles take 23.3 at 6.4 TB/s (the copy bandwidth is 6.54; after 50 ms of nothing else the GPU is at its 1000 W, the SMs at 1690
// instead of 1965 MHz, and it is 39 us); 4 sessions behind 2011 rows 9.5 us, 2 behind 150 rows 6.5 us on the device.  What the tiles do not take, 10 us of a large launch, is its ends: queries 1.7, the last values 0.9, parts written
// and seen by the others 2, adding them up 2.5, the rest the launch itself.  Head dim 128 only: a tile's rings take the SM's shared memory.
#include <algorithm>
#include <type_traits>

#include "kv_share.cuh"
#include "mathx_dev.cuh"
#include "tcgen05_dev.cuh"
#include "warp_reduce.cuh"

namespace {

constexpr uint32_t kHd = 128, kTile = 128, kMaxQ = 64, kGroups = 4, kThreads = 96 + kGroups * 128;
constexpr uint32_t kPageBlock = kPageTokens * kHd * 2, kSlot = 2 * kPageBlock;   // K or V of a page, of a tile
constexpr uint32_t kBox = kTile * 128;                                           // 64 dims of a tile's keys
constexpr uint32_t kQBytes = 4 * kMaxQ * 128;                                    // high and low parts
constexpr uint32_t kKSlots = 2, kMaxVSlots = 3, kItemSlots = 8;
constexpr uint32_t kTmemCols = 512, kTmemO = 256;                                // two buffers of 128 columns each
constexpr uint32_t kMaxBundles = 64;
// Weights are held against a reference 2^kLift below the largest score; it moves when a score is 2^kGrow above that: 2^15 at most.
constexpr float kGrow = 8.0f, kLift = 7.0f, kLog2e = 1.4426950408889634f;

// A bundle's columns: its queries, rounded up to a size that the groups of threads are made for.  (High and low parts side by side are 32,
// 64 or 128 columns, 43, 50 or 64 cycles an instruction; fewer cost what 32 do.)
__host__ __device__ __forceinline__ uint32_t padded(uint32_t nq) { return nq <= 16 ? 16u : nq <= 32 ? 32u : 64u; }
struct Bundle {
    uint32_t group, row0, sessions;      // its group; its first session, how many
    uint32_t head0, heads;               // which of a kv head's query heads
    uint32_t shared, tiles, chunks, item0, part0;        // tiles: all of them, the shared ones first
    uint32_t nq, columns, inverse;       // sessions x heads; padded; 65536 / heads
};
// x / heads for a column's number, by 65536 / heads rounded up: 64 columns at most, so the remainder does not reach the next number
__device__ __forceinline__ uint32_t over_heads(const Bundle &b, uint32_t x) { return x * b.inverse >> 16; }
// Where share i of a bundle's tiles begins.  An own tile's work counts five quarters of a shared one's: where a share begins with own
// tiles, every session's first one sets its columns' references.  (16 sessions behind 32768 rows, 20 to 300 own ones: 35.4 us, 36.4 with even
// numbers; behind 6000, 50 to 1500 own ones: 25.5 and 25.1.)
__host__ __device__ __forceinline__ uint32_t weight_of(uint32_t shared, uint32_t tiles) { return 4 * shared + 5 * (tiles - shared); }
// (Shares of a weight of five at least have a tile each; or there are as many as tiles.)
__host__ __device__ __forceinline__ uint32_t shares_of(uint32_t shared, uint32_t tiles, uint32_t share)
{
    const uint32_t w = weight_of(shared, tiles), n = (w + share - 1) / share;
    return n >= tiles ? tiles : n < w / 5 ? n : w / 5;
}
__host__ __device__ __forceinline__ uint32_t share_at(const Bundle &b, uint32_t i)
{
    if (b.chunks == b.tiles) return i;
    const uint32_t w = weight_of(b.shared, b.tiles) * i / b.chunks;        // (2.7 million at most, times 592 at most)
    return w < 4 * b.shared ? (w + 2) / 4 : b.shared + (w - 4 * b.shared + 2) / 5;
}
struct SharedParams {
    Bundle bundle[kMaxBundles];
    const uint64_t *shared_pages[WR_CUDA_BATCH_MAX], *own_pages[WR_CUDA_BATCH_MAX];      // of a group; of a session, from its own rows on
    uint32_t shared_rows[WR_CUDA_BATCH_MAX], own_rows[WR_CUDA_BATCH_MAX];
    uint8_t first_bundle[WR_CUDA_BATCH_MAX];     // of a session; the next ones have its further heads
    uint32_t n_bundles, items, rows, n_q, n_kv, per;     // rows: of the result; per: query heads to a kv head
    const float *q, *k_new, *v_new;      // k_new: null where nothing is appended
    float theta;
    uint32_t n_rot;                      // pairs that new keys and the queries are rotated by; 0: none
    float *out;
    uint32_t parts;                      // of the bundles that have more than one; the others' rows are written at once
    float2 *ml;                          // [part]: reference (log2), sum
    float *o;                            // [part][128]
    int *sched;                          // next item, CTAs that have left
    int *done;                           // [bundle][kv head]: parts that are there, then rows that have been added up
    uint32_t team;                       // warps that add up a row
    uint32_t widest;                     // most queries of a bundle
    uint32_t early;                      // the shared rows have been written before the kernel in front of this one began
    float scale_log2;
    long long wait_limit;
    int *err;
};
struct Item {
    uint32_t tiles, tile0;               // tiles 0: no more work
    uint32_t bundle, kvh, part;
};
// Where a role is in a bundle's list: segment 0 is the shared rows, 1 + i the i-th session's own.
struct Place {
    uint32_t segment, tile;
};
__device__ __forceinline__ uint32_t rows_of(const SharedParams &p, const Bundle &b, uint32_t segment)
{
    return segment ? p.own_rows[b.row0 + segment - 1] : p.shared_rows[b.group];
}
__device__ __forceinline__ Place place_at(const SharedParams &p, const Bundle &b, uint32_t tile)
{
    Place at = {0, tile};
    for (uint32_t n; at.segment < b.sessions && at.tile >= (n = (rows_of(p, b, at.segment) + kTile - 1) / kTile); ++at.segment) at.tile -= n;
    return at;
}
__device__ __forceinline__ void step(const SharedParams &p, const Bundle &b, Place &at)
{
    ++at.tile;
    while (at.segment < b.sessions && at.tile * kTile >= rows_of(p, b, at.segment)) {
        at.tile = 0;
        ++at.segment;
    }
}
// a column's row of q and of the result
__device__ __forceinline__ uint32_t row_of(const SharedParams &p, const Bundle &b, uint32_t kvh, uint32_t column)
{
    const uint32_t session = over_heads(b, column);
    return (b.row0 + session) * p.n_q + kvh * p.per + b.head0 + column - session * b.heads;
}
// the tile's pages of one layer: the first one's address in the table, and whether there is a second
__device__ __forceinline__ const uint64_t *pages_of(const SharedParams &p, const Bundle &b, const Place &at, bool &two)
{
    two = rows_of(p, b, at.segment) > at.tile * kTile + kPageTokens;
    return (at.segment ? p.own_pages[b.row0 + at.segment - 1] : p.shared_pages[b.group]) + 2 * at.tile;
}
struct Bars {
    uint64_t k_full[kKSlots], k_free[kKSlots], v_full[kMaxVSlots], v_free[kMaxVSlots];
    uint64_t q_full, s_full[2], p_full[2], o_full[2], drained;
    uint64_t item_ready[kItemSlots];
    Item item[kItemSlots];
    uint32_t tmem;
    alignas(16) float up[2][kMaxQ];      // per query: what its scores still lack
    uint32_t large[2];                   // an item with an `up` that is not 1
    alignas(16) float nm[kMaxQ], a[kMaxQ];           // reference, negative; factor of its last change
    alignas(16) float red[kMaxQ][4];
};
// two buffers of P: high and low parts in one row of 128 bytes, or (more than 32 queries) in two
__host__ __device__ constexpr uint32_t p_bytes(uint32_t queries) { return queries > 32 ? 2 * kTile * 128 : kTile * 128; }
__host__ __device__ constexpr uint32_t v_slots(uint32_t queries) { return queries > 32 ? 2 : 3; }
constexpr uint32_t kSmem = kKSlots * kSlot + 2 * kSlot + kQBytes + 2 * p_bytes(64) + (uint32_t)sizeof(Bars);
static_assert(v_slots(32) * kSlot + 2 * p_bytes(32) == v_slots(64) * kSlot + 2 * p_bytes(64), "");
static_assert(kSmem <= 232448, "the CTA's shared memory is 227 KB at most");

// Whether the tile ends with the row that its session appends.
__device__ __forceinline__ bool appends(const SharedParams &p, const Bundle &b, const Place &at)
{
    return p.k_new && at.segment && (at.tile + 1) * kTile >= p.own_rows[b.row0 + at.segment - 1];
}
__device__ __forceinline__ uint32_t position_of(const SharedParams &p, const Bundle &b, uint32_t session)
{
    return p.shared_rows[b.group] + p.own_rows[session] - 1;
}
// What a new key is rotated by: a lane has dims 2 x lane and the next.  (Kept from row to row: the beams of a search are at one position,
// and the angles took 2 us where a work item appends two rows.)
struct Angles {
    uint32_t position;
    float sn[2], cs[2];
};
__device__ __noinline__ float4 angles_at(float theta, uint32_t position, uint32_t d)
{
    const float ln_theta = wrmath::log_ref(theta);
    float4 x;
    wrmath::rope_angle(position, d, kHd, ln_theta, x.x, x.z);
    wrmath::rope_angle(position, d + 1, kHd, ln_theta, x.y, x.w);
    return x;
}
__device__ __forceinline__ void turn_to(const SharedParams &p, Angles &a, uint32_t position, uint32_t lane)
{
    if (!p.n_rot || a.position == position) return;
    const float4 x = angles_at(p.theta, position, 2 * lane);
    a = {position, {x.x, x.y}, {x.z, x.w}};
}
// A session's new row of one kv head into its page, as wr_cuda_kv_append stores it (kernels.c:1406-1407, products rounded
// separately; quant.c:121-136): a warp, two pairs of dims to a lane.  Bulk copies that lane 0 issues afterwards see it.
__device__ __forceinline__ void append_row(const SharedParams &p, uint32_t session, uint32_t kvh, uint32_t which, const Angles &a, uint32_t lane)
{
    const uint32_t row = p.own_rows[session] - 1, d = 2 * lane;
    const float *const x = (which ? p.v_new : p.k_new) + ((size_t)session * p.n_kv + kvh) * kHd;
    float lo[2] = {x[d], x[d + 1]}, hi[2] = {x[d + kHd / 2], x[d + 1 + kHd / 2]};
    if (!which && p.n_rot) {
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
            if (d + e >= p.n_rot) continue;
            const float u = lo[e], v = hi[e];
            lo[e] = wrmath::sub(wrmath::mul(u, a.cs[e]), wrmath::mul(v, a.sn[e]));
            hi[e] = wrmath::add(wrmath::mul(u, a.sn[e]), wrmath::mul(v, a.cs[e]));
        }
    }
    char *const block = reinterpret_cast<char *>(p.own_pages[session][row / kPageTokens]) + wr_block_off(kvh, which, kHd);
    *reinterpret_cast<uint32_t *>(block + wr_elem_off(row % kPageTokens, d, kHd)) =
        wr_f32_to_f16_trunc(lo[0]) | (uint32_t)wr_f32_to_f16_trunc(lo[1]) << 16;
    *reinterpret_cast<uint32_t *>(block + wr_elem_off(row % kPageTokens, d + kHd / 2, kHd)) =
        wr_f32_to_f16_trunc(hi[0]) | (uint32_t)wr_f32_to_f16_trunc(hi[1]) << 16;
    asm volatile("fence.proxy.async.global;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ Item item_of(const SharedParams &p, uint32_t i)
{
    Item it{};
    if (i >= p.items) return it;
    while (it.bundle + 1 < p.n_bundles && i >= p.bundle[it.bundle + 1].item0) ++it.bundle;
    const Bundle &b = p.bundle[it.bundle];
    i -= b.item0;
    it.kvh = i % p.n_kv;
    i /= p.n_kv;
    it.tile0 = share_at(b, i);
    it.tiles = share_at(b, i + 1) - it.tile0;
    it.part = b.part0 + (i * p.n_kv + it.kvh) * b.nq;
    return it;
}
__device__ __forceinline__ void group_sync(uint32_t id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool group_or(uint32_t id, uint32_t threads, bool x)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(id), "r"(threads), "r"((uint32_t)x) : "memory");
    return r != 0;
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void all_sync() { asm volatile("bar.sync %0, %1;" ::"n"(1 + kGroups), "n"(128 * kGroups) : "memory"); }
__device__ __forceinline__ bool all_or(bool x) { return group_or(1 + kGroups, 128 * kGroups, x); }
// two F32 additions in one issue slot
__device__ __forceinline__ void add2(float &a, float &b, float x, float y)
{
    asm("{\n\t.reg .b64 s, t;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\tadd.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
// H consecutive columns of this thread's TMEM lane (no wait)
template <uint32_t H> __device__ __forceinline__ void tmem_ld(uint32_t at, float (&v)[H])
{
    if constexpr (H == 16) tc5::ld16(at, v);
    else if constexpr (H == 8) tc5::ld8(at, v);
    else tc5::ld4(at, v);
}
// Largest of the warp's 32 lanes for each of H values: v[0] holds that of the value whose index is returned.
template <uint32_t H> __device__ __forceinline__ uint32_t warp_max_many(float (&v)[H], uint32_t lane)
{
    uint32_t idx = 0;
#pragma unroll
    for (uint32_t o = 16, half = H / 2; o >= 1; o >>= 1, half >>= 1) {
        if (half) {
            const bool upper = (lane & o) != 0;
#pragma unroll
            for (uint32_t i = 0; i < H / 2; ++i)
                if (i < half) {
                    const float send = upper ? v[i] : v[i + half], keep = upper ? v[i + half] : v[i];
                    v[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, o));
                }
            if (upper) idx += half;
        } else {
            v[0] = fmaxf(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
        }
    }
    return idx;
}
// kind::f16, F16 x F16 -> F32: V^T (its dims contiguous) times P^T (its queries contiguous)
__device__ __forceinline__ uint32_t idesc_values(uint32_t n) { return tc5::idesc_f16(128, n) | tc5::kIdescAMnMajor | (1u << 16); }

// The parts of a row added up, in order.  The CTAs do this when there is
// no item left to draw; a team of warps takes a row, waits for its parts (bounded), and has up to 8 x team of them under way at once.
// (A kernel of its own behind this one was quicker on the device where there is little to do, 7.6 against 8.7 us for two short sessions,
// 21.0 against 22.1 for four groups behind 4096 rows, slower behind 32768, 38.4 against 37.8, and cost the host 2.2 us a call.)
constexpr uint32_t kMergeAhead = 8, kMergeWarps = 4 * kGroups;
__device__ __forceinline__ bool add_up(const SharedParams &p, float4 *sums, uint32_t warp, uint32_t lane)
{
    const uint32_t team = p.team, teams = kMergeWarps / team, sub = warp % team;
    bool ok = true;
    for (uint32_t j = blockIdx.x; j * teams < p.rows; j += gridDim.x) {
        const uint32_t row = j * teams + warp / team;
        const bool mine = row < p.rows;
        const uint32_t s = mine ? row / p.n_q : 0, head = mine ? row % p.n_q : 0, kvh = head / p.per;
        const uint32_t which = p.first_bundle[s] + head % p.per / kMaxQ;
        const Bundle &b = p.bundle[which];
        const uint32_t stride = p.n_kv * b.nq;
        const uint32_t first = b.part0 + kvh * b.nq + (s - b.row0) * b.heads + head % p.per - b.head0;
        int *const done = p.done + which * p.n_kv + kvh;
        uint32_t n = mine && ok && b.chunks > 1 ? b.chunks : 0;
        if (n && sub == 0) {                                     // (few ask: thousands of warps at these words held up what they wait for)
            long long t0 = 0;
            for (bool again = false;; again = true) {
                int there;
                asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(there) : "l"(done) : "memory");
                if (__all_sync(0xffffffffu, (uint32_t)there >= n)) break;
                if (!again) t0 = clock64();
                else if (__any_sync(0xffffffffu, clock64() - t0 > p.wait_limit)) {
                    ok = false;
                    break;
                }
            }
        }
        ok = !all_or(!ok);
        if (!ok) n = 0;
        auto part = [&](uint32_t i) { return first + i * stride; };
        float4 o[kMergeAhead], acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float m[kMergeAhead], top = WR_NEG_SENTINEL, l = 0.f;
        auto load = [&](uint32_t i0) {
#pragma unroll
            for (uint32_t u = 0; u < kMergeAhead; ++u) {
                const uint32_t i = i0 + u * team;
                if (i >= n) continue;
                o[u] = __ldcg(reinterpret_cast<const float4 *>(p.o + (size_t)part(i) * kHd) + lane);
                m[u] = __ldcg(&p.ml[part(i)].x);
            }
        };
        load(sub);
        for (uint32_t i = lane; i < n; i += 32) {
            const float2 ml = __ldcg(p.ml + part(i));
            const float t = fmaxf(top, ml.x);
            l = l * ex2(top - t) + ml.y * ex2(ml.x - t);
            top = t;
        }
        const float before = top;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        l *= ex2(before - top);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        for (uint32_t i0 = sub; i0 < n;) {
#pragma unroll
            for (uint32_t u = 0; u < kMergeAhead; ++u) {
                if (i0 + u * team >= n) continue;
                const float w = ex2(m[u] - top);
                acc.x = fmaf(w, o[u].x, acc.x); acc.y = fmaf(w, o[u].y, acc.y);
                acc.z = fmaf(w, o[u].z, acc.z); acc.w = fmaf(w, o[u].w, acc.w);
            }
            i0 += kMergeAhead * team;
            load(i0);
        }
        if (team > 1) {
            sums[warp * 32 + lane] = acc;
            all_sync();
            for (uint32_t w = 1; w < team && sub == 0; ++w) {
                const float4 x = sums[(warp + w) * 32 + lane];
                acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
            }
        }
        if (sub == 0 && n && ok) {
            // (a row of which no key counts, all scores -inf, is zeros)
            if (l == 0.f) acc = make_float4(0.f, 0.f, 0.f, 0.f);
            else acc = make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l);
            *(reinterpret_cast<float4 *>(p.out + (size_t)row * kHd) + lane) = acc;
            // the last row leaves the counter as it was (without a look at what it was: 0.5 us)
            if (lane == 0) atomicInc(reinterpret_cast<unsigned *>(done), n + b.nq - 1);
        }
        if (team > 1) all_sync();
    }
    return ok;
}

__global__ void __launch_bounds__(kThreads, 1) attn_shared_kernel(const __grid_constant__ SharedParams p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t v_ring = v_slots(p.widest), p_size = p_bytes(p.widest);
    uint8_t *const ks = smem_raw, *const qs = ks + kKSlots * kSlot, *const vs = qs + kQBytes, *const ps = vs + v_ring * kSlot;
    Bars &sm = *reinterpret_cast<Bars *>(ps + 2 * p_size);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Item first = item_of(p, blockIdx.x);                   // (1 us: the arguments' way into the constant cache)
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kKSlots; ++i) {
            mbar_init(&sm.k_full[i], 1);
            mbar_init(&sm.k_free[i], 1);
        }
        for (uint32_t i = 0; i < kMaxVSlots; ++i) {
            mbar_init(&sm.v_full[i], 1);
            mbar_init(&sm.v_free[i], 1);
        }
        for (uint32_t i = 0; i < kItemSlots; ++i) mbar_init(&sm.item_ready[i], 1);
        mbar_init(&sm.q_full, 4 * kGroups);
        mbar_init(&sm.s_full[0], 1);
        mbar_init(&sm.s_full[1], 1);
        mbar_init(&sm.p_full[0], 4 * kGroups);
        mbar_init(&sm.p_full[1], 4 * kGroups);
        mbar_init(&sm.o_full[0], 1);
        mbar_init(&sm.o_full[1], 1);
        mbar_init(&sm.drained, 1);
        fence_barrier_init();
    }
    if (warp == 1) tc5::alloc(&sm.tmem, kTmemCols);
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    // What the kernel before this one may still be writing waits for it, as late as can be.  With p.early that is not the shared rows.
    bool waited = false;
    auto wait_before = [&](bool need) {
        if (need && !waited) pdl_wait();
        waited |= need;
    };
    // The first queries are asked for before a whole ring of keys and values is: behind that they came 1 us later.  (The CTA's warps meet
    // once, in the first item, before any wait for a slot.)
    bool met = false;
    auto queries_first = [&](bool now) {
        if (now && !met) {
            __syncwarp();
            asm volatile("bar.sync 7, %0;" ::"n"(64 + 128 * kGroups) : "memory");
        }
        met |= now;
    };
    const uint32_t tmem = sm.tmem;
    const long long limit = p.wait_limit;
    // Item number `it` of this CTA (the first is its own number); the loading warp is at most four items ahead of the slowest reader.
    auto item_at = [&](uint32_t it, bool &ok) -> Item {
        if (it == 0) return first;
        uint64_t *bar = &sm.item_ready[it % kItemSlots];
        const uint32_t parity = (it / kItemSlots) & 1;
        ok = mbar_wait_warp(bar, parity, limit);
        return ok ? sm.item[it % kItemSlots] : Item{};
    };

    if (warp == 0) {                                             // work items and K
        uint32_t n = 0;
        bool ok = true;
        uint32_t next = 0;
        Angles angles = {~0u, {}, {}};
        for (uint32_t it = 0; ok; ++it) {
            const Item im = it ? item_of(p, next) : first;
            if (lane == 0) {
                sm.item[it % kItemSlots] = im;
                mbar_arrive(&sm.item_ready[it % kItemSlots]);    // (the first one's for the phases' sake)
            }
            if (!im.tiles) break;
            const Bundle &bd = p.bundle[im.bundle];
            Place at = place_at(p, bd, im.tile0);
            for (uint32_t t = 0; t < im.tiles; ++t, ++n, step(p, bd, at)) {
                bool two;
                const bool add = appends(p, bd, at);
                if (add) turn_to(p, angles, position_of(p, bd, bd.row0 + at.segment - 1), lane);
                const uint64_t *const table = pages_of(p, bd, at, two);
                asm volatile("" ::"l"(table));                   // (worked out before the wait)
                wait_before(at.segment != 0 || !p.early);
                queries_first(n == p.early);
                if (add) append_row(p, bd.row0 + at.segment - 1, im.kvh, 0, angles, lane);
                const uint32_t st = n % kKSlots;
                const uint64_t page[2] = {table[0], two ? table[1] : 0};      // (there when the slot is free)
                if (n >= kKSlots && !mbar_wait_warp(&sm.k_free[st], (n / kKSlots - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                if (lane) continue;
                mbar_expect_tx(&sm.k_full[st], (two ? 2 : 1) * kPageBlock);
                for (uint32_t g = 0; g < (two ? 2u : 1u); ++g) {
                    const char *src = reinterpret_cast<const char *>(page[g]) + wr_block_off(im.kvh, 0, kHd);
                    bulk_g2s(ks + st * kSlot + g * 8192, src, 8192, &sm.k_full[st]);
                    bulk_g2s(ks + st * kSlot + kBox + g * 8192, src + 8192, 8192, &sm.k_full[st]);
                }
            }
            queries_first(true);
            wait_before(true);                                   // (the counter is the earlier launch's until it has ended)
            if (ok && lane == 0) next = gridDim.x + (uint32_t)atomicAdd(p.sched, 1);
            next = __shfl_sync(0xffffffffu, next, 0);
        }
        wait_before(true);
        if (lane == 0) {
            if (!ok) atomicCAS(p.err, 0, 81);
            // the last CTA to leave makes the counters ready for the next launch
            __threadfence();
            if (atomicAdd(p.sched + 1, 1) == (int)gridDim.x - 1) {
                p.sched[0] = 0;
                p.sched[1] = 0;
            }
            for (uint32_t i = n - min(n, kKSlots); i < n; ++i) (void)mbar_wait(&sm.k_full[i % kKSlots], (i / kKSlots) & 1, limit);
        }
        __syncwarp();
    } else if (warp == 2) {                                      // V
        uint32_t n = 0;
        bool ok = true;
        for (uint32_t it = 0; ok; ++it) {
            const Item im = item_at(it, ok);
            if (!im.tiles) break;
            const Bundle &bd = p.bundle[im.bundle];
            Place at = place_at(p, bd, im.tile0);
            for (uint32_t t = 0; t < im.tiles; ++t, ++n, step(p, bd, at)) {
                bool two;
                const uint64_t *const table = pages_of(p, bd, at, two);
                asm volatile("" ::"l"(table));
                wait_before(at.segment != 0 || !p.early);
                queries_first(n == p.early);
                if (appends(p, bd, at)) append_row(p, bd.row0 + at.segment - 1, im.kvh, 1, Angles{}, lane);
                const uint32_t st = n % v_ring;
                const uint64_t page[2] = {table[0], two ? table[1] : 0};
                if (n >= v_ring && !mbar_wait_warp(&sm.v_free[st], (n / v_ring - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                if (lane) continue;
                mbar_expect_tx(&sm.v_full[st], (two ? 2 : 1) * kPageBlock);
                for (uint32_t g = 0; g < (two ? 2u : 1u); ++g)
                    bulk_g2s(vs + st * kSlot + g * kPageBlock, reinterpret_cast<const char *>(page[g]) + wr_block_off(im.kvh, 1, kHd),
                             kPageBlock, &sm.v_full[st]);
            }
            queries_first(true);
        }
        if (lane == 0) {
            if (!ok) atomicCAS(p.err, 0, 82);
            for (uint32_t i = n - min(n, v_ring); i < n; ++i) (void)mbar_wait(&sm.v_full[i % v_ring], (i / v_ring) & 1, limit);
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool lead = tc5::elect_one();
        const uint32_t q_addr = smem_u32(qs), p_addr = smem_u32(ps), k_addr = smem_u32(ks), v_addr = smem_u32(vs);
        uint32_t n_s = 0, n_o = 0;                               // tiles scored, multiplied
        bool ok = true;
        auto score = [&](uint32_t n) {
            const uint32_t st = n_s % kKSlots;
            if (!mbar_wait_warp(&sm.k_full[st], (n_s / kKSlots) & 1, limit)) return false;
            tc5::fence_after();
            const uint32_t d = tmem + (n_s & 1) * 2 * kMaxQ, idesc = tc5::idesc_f16(128, n);
            const uint64_t a = tc5::desc_kmajor(k_addr + st * kSlot), b = tc5::desc_kmajor(q_addr);
#pragma unroll
            for (uint32_t kk = 0; kk < 8; ++kk)                  // 16 dims a step
                if (lead) tc5::mma_ss(d, a + (kk >> 2) * (kBox >> 4) + 2 * (kk & 3), b + (kk >> 2) * (n * 128 >> 4) + 2 * (kk & 3), idesc, kk != 0);
            if (lead) {
                tc5::commit(&sm.k_free[st]);
                tc5::commit(&sm.s_full[n_s & 1]);
            }
            ++n_s;
            return true;
        };
        for (uint32_t it = 0; ok; ++it) {
            const Item im = item_at(it, ok);
            if (!im.tiles) break;
            const Bundle &bd = p.bundle[im.bundle];
            const uint32_t n = 2 * bd.columns;
            Place at = place_at(p, bd, im.tile0);
            ok = mbar_wait_warp(&sm.q_full, it & 1, limit) && score(n);
            for (uint32_t t = 0; t < im.tiles && ok; ++t, step(p, bd, at)) {
                // (the scores two tiles ago have been read: their P has been waited for.  Issued behind the values of the tile before:
                // whoever sees these scores knows those to be there.)
                if (t + 1 < im.tiles) ok = score(n);
                ok = ok && mbar_wait_warp(&sm.p_full[n_o & 1], (n_o >> 1) & 1, limit);
                const uint32_t st = n_o % v_ring;
                ok = ok && mbar_wait_warp(&sm.v_full[st], (n_o / v_ring) & 1, limit);
                if (!ok) break;
                tc5::fence_after();
                const uint32_t d = tmem + kTmemO + (n_o & 1) * 2 * kMaxQ, idesc = idesc_values(n), here = rows_of(p, bd, at.segment) - at.tile * kTile;
                const uint64_t a = tc5::desc_mnmajor(v_addr + st * kSlot, 8192), b = tc5::desc_mnmajor(p_addr + (n_o & 1) * p_size, kTile * 128);
#pragma unroll
                for (uint32_t kk = 0; kk < 8; ++kk)              // 16 keys a step, as far as there are any
                    if (lead && 16 * kk < here)
                        tc5::mma_ss(d, a + (kk >> 2) * (kPageBlock >> 4) + (kk & 3) * (2048 >> 4), b + kk * (2048 >> 4), idesc, kk != 0);
                if (lead) {
                    tc5::commit(&sm.v_free[st]);
                    tc5::commit(&sm.o_full[n_o & 1]);
                }
                ++n_o;
            }
        }
        if (!ok && lane == 0) atomicCAS(p.err, 0, 83);
        __syncwarp();
        if (lead) tc5::commit(&sm.drained);                      // no product is running when the TMEM is given back
        (void)mbar_wait_warp(&sm.drained, 0, limit);
    } else {
        // a thread per key (scores) and per value dimension (output): its TMEM lane either way; each group has a share of the queries
        const uint32_t quarter = warp & 3, group = (warp - 3) >> 2, key = quarter * 32 + lane, tid = (threadIdx.x - 96) & 127;
        const uint32_t bar = 1 + group, lanes = (quarter * 32) << 16;
        uint32_t n = 0;                                          // tiles so far
        bool ok = true;
        // The item's queries as operands: scaled so that scores are powers of two's exponents, in a high and a low F16 part.  Up to
        // 2^15 that leaves 2^-22 of an element or 2^-25, whichever is more; rows with larger ones are brought below it by a power of two.
        auto queries = [&](const Item &im, uint32_t it) {
            const Bundle &bd = p.bundle[im.bundle];
            const uint32_t rows = bd.columns;
            constexpr uint32_t kEach = kMaxQ / (4 * kGroups);
            const uint32_t each = rows / (4 * kGroups), r0 = (warp - 3) * each;     // rows of a warp: neighbours, mostly of one session
            float4 x[kEach];
            uint32_t from[kEach];                                // (row of q; ~0: none)
#pragma unroll
            for (uint32_t u = 0; u < kEach; ++u) {
                from[u] = u < each && r0 + u < bd.nq ? row_of(p, bd, im.kvh, r0 + u) : ~0u;
                asm volatile("" ::"r"(from[u]));
            }
            if (it == 0) {
                pdl_wait();
                pdl_trigger();
            }
#pragma unroll
            for (uint32_t u = 0; u < kEach; ++u) {
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (~from[u]) x[u] = __ldg(reinterpret_cast<const float4 *>(p.q + (size_t)from[u] * kHd) + lane);
            }
            if (it == 0) asm volatile("bar.arrive 7, %0;" ::"n"(64 + 128 * kGroups) : "memory");
            if (p.n_rot) {                                       // (as wr_cuda_kv_append rotates them)
                uint32_t of = ~0u;
                float cs[4], sn[4];                              // of dims 4 (lane % 16) .. + 3 and those 64 on
#pragma unroll
                for (uint32_t u = 0; u < kEach; ++u) {
                    const uint32_t session = over_heads(bd, r0 + u);
                    if (!~from[u]) break;
                    if (session != of) {
                        const float4 w = angles_at(p.theta, position_of(p, bd, bd.row0 + session), 2 * lane);
                        const float c[2] = {w.z, w.w}, d[2] = {w.x, w.y};
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            const uint32_t from = 2 * (lane & 15) + e / 2;
                            cs[e] = __shfl_sync(0xffffffffu, c[e & 1], from);
                            sn[e] = __shfl_sync(0xffffffffu, d[e & 1], from);
                        }
                        of = session;
                    }
                    float *const y = reinterpret_cast<float *>(&x[u]);
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        const float other = __shfl_xor_sync(0xffffffffu, y[e], 16);
                        if (4 * (lane & 15) + e >= p.n_rot) continue;
                        y[e] = lane < 16 ? wrmath::sub(wrmath::mul(y[e], cs[e]), wrmath::mul(other, sn[e]))
                                         : wrmath::add(wrmath::mul(other, sn[e]), wrmath::mul(y[e], cs[e]));
                    }
                }
            }
            if (threadIdx.x == 96) sm.large[it & 1] = 0;
            all_sync();
#pragma unroll
            for (uint32_t u = 0; u < kEach; ++u) {
                const uint32_t r = r0 + u;
                if (u >= each) continue;
                float y[4] = {x[u].x * p.scale_log2, x[u].y * p.scale_log2, x[u].z * p.scale_log2, x[u].w * p.scale_log2}, up = 1.f;
                const float top = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
                if (__any_sync(0xffffffffu, top >= 32768.f)) {
                    float most = top;
#pragma unroll
                    for (int o = 16; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    const int e = min((int)(__float_as_uint(most) >> 23) - 127, 126);
                    const float down = __int_as_float((127 - e) << 23);
                    up = __int_as_float((127 + e) << 23);
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) y[j] *= down;
                    if (lane == 0) sm.large[it & 1] = 1;
                }
                uint32_t hi[2], lo[2];
                split_half2(y[0], y[1], hi[0], lo[0]);
                split_half2(y[2], y[3], hi[1], lo[1]);
                // (rows and rows more: a multiple of 16, so the swizzle is the same)
                uint8_t *at = qs + (lane >> 4) * (2 * rows * 128) + r * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
                *reinterpret_cast<uint2 *>(at) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2 *>(at + rows * 128) = make_uint2(lo[0], lo[1]);
                if (lane == 0) sm.up[it & 1][r] = up;
            }
            fence_proxy_async();
            all_sync();                                          // (sm.up, sm.large)
            if (lane == 0) mbar_arrive(&sm.q_full);
        };
        Item im = item_at(0, ok);
        // (a warp whose wait ran out stays with the others: they leave together, and the groups' barriers count on all of them)
        ok = !all_or(!ok);
        auto work = [&](auto size, uint32_t it) {
            constexpr uint32_t NQ = decltype(size)::value, H = NQ / kGroups, V = H < 8 ? H : 8;     // V: queries to a store
            const uint32_t q0 = group * H;                       // this group's first query
            const float4 *const nm4 = reinterpret_cast<const float4 *>(sm.nm + q0), *const a4 = reinterpret_cast<const float4 *>(sm.a + q0);
            const bool large = sm.large[it & 1] != 0;
            const Bundle &bd = p.bundle[im.bundle];
            bool fresh = true, moved = false;                    // no tile of these queries yet; the last one moved the reference
            uint32_t zeros = 0;                                  // buffers of P that hold zeros for these queries
            float o[H], l[H];
#pragma unroll
            for (uint32_t j = 0; j < H; ++j) o[j] = l[j] = 0.f;
            // O^T of a finished tile, which columns [lo, hi) attended to (another session's values stay out of the others' sums even
            // where they are not numbers); then the change of reference that the tile behind it made.
            auto add_values = [&](uint32_t tile, int lo, int hi) {
                if (hi > 0 && lo < (int)H) {
                    const bool all = lo <= 0 && hi >= (int)H;
                    const uint32_t at = tmem + kTmemO + (tile & 1) * 2 * kMaxQ + lanes + q0;
#pragma unroll
                    for (uint32_t j0 = 0; j0 < H; j0 += V) {     // (eight at a time: more at once do not fit the registers)
                        float high[V], low[V];
                        tmem_ld(at + j0, high);
                        tmem_ld(at + NQ + j0, low);
                        tc5::wait_ld();
#pragma unroll
                        for (uint32_t j = 0; j < V; ++j)
                            if (fabsf(high[j]) != INFINITY) high[j] += low[j];   // (as in scores)
                        if (all) {
#pragma unroll
                            for (uint32_t j = 0; j < V; j += 2) add2(o[j0 + j], o[j0 + j + 1], high[j], high[j + 1]);
                        } else {
#pragma unroll
                            for (int j = 0; j < (int)V; ++j)
                                if ((int)j0 + j >= lo && (int)j0 + j < hi) o[j0 + j] += high[j];
                        }
                    }
                }
                if (moved) {
#pragma unroll
                    for (uint32_t j = 0; j < H; j += 4) {
                        const float4 a = a4[j / 4];
                        o[j] *= a.x; o[j + 1] *= a.y; o[j + 2] *= a.z; o[j + 3] *= a.w;
                    }
                }
            };
            // P of the tile is written: the tensor core may go on.
            auto hand_over = [&]() {
                fence_proxy_async();
                tc5::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_full[n & 1]);
            };
            auto put = [&](uint32_t at, const uint32_t (&x)[V / 2]) {
                // a key's row: the high parts of up to 64 queries, the low ones behind them or in rows of their own
                uint8_t *to = ps + (n & 1) * p_size + key * 128 + (at >> 7) * (kTile * 128) + ((((at >> 4) & 7) ^ (key & 7)) << 4) + (at & 15);
                if constexpr (V == 8) *reinterpret_cast<uint4 *>(to) = make_uint4(x[0], x[1], x[2], x[3]);
                else *reinterpret_cast<uint2 *>(to) = make_uint2(x[0], x[1]);
            };
            // Rows behind the last one may hold anything, and a weight of zero does not take a NaN out: those that the last step
            // multiplies are cleared.
            auto clear_rows = [&](uint32_t here) {
                const uint32_t st = n % v_ring;
                if (ok) ok = mbar_wait_warp(&sm.v_full[st], (n / v_ring) & 1, limit);
                if (key >= here && key < ((here + 15) & ~15u)) {
                    uint8_t *row = vs + st * kSlot + (key >> 6) * kPageBlock + (key & 63) * 128;
#pragma unroll
                    for (uint32_t e = 0; e < 16; ++e)
                        *reinterpret_cast<uint4 *>(row + (e >> 3) * 8192 + ((e ^ key) & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
            };
            // The scores of a tile are there, and with them O^T of the tile two before it; P's buffer is free.
            auto await_scores = [&]() {
                if (ok) ok = mbar_wait_warp(&sm.s_full[n & 1], (n >> 1) & 1, limit);
                tc5::fence_after();
            };
            // One tile of `here` keys or more, which columns [lo, hi) of this group attend to.
            auto tile = [&](uint32_t here, int lo, int hi) {
                const uint32_t at = tmem + (n & 1) * 2 * kMaxQ + lanes + q0;
                float s[H];
                auto mask = [&]() {
                    if (here >= kTile && lo <= 0 && hi >= (int)H) return;
                    const bool seen = key < here;
#pragma unroll
                    for (int j = 0; j < (int)H; ++j) s[j] = seen && j >= lo && j < hi ? s[j] : -INFINITY;
                };
                auto scores = [&](bool infinite) {
                    tmem_ld(at, s);
#pragma unroll
                    for (uint32_t j0 = 0; j0 < H; j0 += V) {
                        float low[V];
                        tmem_ld(at + NQ + j0, low);
                        tc5::wait_ld();
                        if (infinite) {
                            // (a row with an infinity: the high part has its product, the low one may have the other sign of it or a NaN)
#pragma unroll
                            for (uint32_t j = 0; j < V; ++j)
                                if (fabsf(s[j0 + j]) != INFINITY) s[j0 + j] += low[j];
                        } else {
#pragma unroll
                            for (uint32_t j = 0; j < V; j += 2) add2(s[j0 + j], s[j0 + j + 1], low[j], low[j + 1]);
                        }
                    }
                    if (large) {
#pragma unroll
                        for (uint32_t j = 0; j < H; ++j) s[j] *= sm.up[it & 1][q0 + j];
                    }
                };
                moved = fresh;
                if (!fresh) {
                    scores(false);
                    float top = -INFINITY;
#pragma unroll
                    for (uint32_t j = 0; j < H; j += 4) {
                        const float4 m = nm4[j / 4];
                        add2(s[j], s[j + 1], m.x, m.y);
                        add2(s[j + 2], s[j + 3], m.z, m.w);
                    }
                    mask();
#pragma unroll
                    for (uint32_t j = 0; j < H; j += 4) top = max3_nan(max3_nan(top, s[j], s[j + 1]), s[j + 2], s[j + 3]);
                    moved = group_or(bar, 128, !(top <= kGrow + kLift));     // (or not a number)
                }
                if (moved) {                                     // (the same in all threads of the group)
                    scores(true);
                    mask();
                    float v[H];
#pragma unroll
                    for (uint32_t j = 0; j < H; ++j) v[j] = s[j];
                    const uint32_t idx = warp_max_many<H>(v, lane);
                    sm.red[q0 + idx][quarter] = v[0];            // (lanes that share an index hold one value)
                    group_sync(bar);
                    if (tid < H) {
                        const float4 w = *reinterpret_cast<const float4 *>(sm.red[q0 + tid]);
                        const float ref = fmaxf(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)), WR_NEG_SENTINEL) - kLift;
                        const float old = fresh ? WR_NEG_SENTINEL : -sm.nm[q0 + tid];
                        const bool up = fresh || ref > old + kGrow;
                        sm.a[q0 + tid] = up ? ex2(old - ref) : 1.f;
                        if (up) sm.nm[q0 + tid] = -ref;
                    }
                    group_sync(bar);
#pragma unroll
                    for (uint32_t j = 0; j < H; j += 4) {
                        const float4 m = nm4[j / 4], a = a4[j / 4];
                        s[j] += m.x; s[j + 1] += m.y; s[j + 2] += m.z; s[j + 3] += m.w;
                        l[j] *= a.x; l[j + 1] *= a.y; l[j + 2] *= a.z; l[j + 3] *= a.w;
                    }
                    fresh = false;
                }
#pragma unroll
                for (uint32_t j = 0; j < H; j += V) {
                    uint32_t high[V / 2], low[V / 2];
#pragma unroll
                    for (uint32_t e = 0; e < V / 2; ++e) {
                        const float w0 = ex2(s[j + 2 * e]), w1 = ex2(s[j + 2 * e + 1]);
                        add2(l[j + 2 * e], l[j + 2 * e + 1], w0, w1);
                        split_half2(w0, w1, high[e], low[e]);
                    }
                    put(2 * (q0 + j), high);
                    put(2 * (q0 + j + NQ), low);
                }
                zeros &= ~(1u << (n & 1));
            };
            const uint32_t n0 = n, n_end = n + im.tiles;
            int lo1 = 0, hi1 = 0, lo2 = 0, hi2 = 0;              // columns of the last tile, of the one before it
            // (One loop for shared and own tiles, one copy of each of its steps: a kernel of twice the code took 1 to 2 us more.)
            // Segment after segment: what does not change within one is not looked up again for every tile.
            for (Place at = place_at(p, bd, im.tile0); n < n_end; at = {at.segment + 1, 0}) {
                const int lo = at.segment ? (int)((at.segment - 1) * bd.heads) - (int)q0 : 0, hi = at.segment ? lo + (int)bd.heads : (int)H;
                const bool mine = hi > 0 && lo < (int)H;
                for (int here = (int)(rows_of(p, bd, at.segment) - at.tile * kTile); here > 0 && n < n_end; here -= (int)kTile, ++n) {
                    await_scores();
                    if (n >= n0 + 2) add_values(n - 2, lo2, hi2);
                    moved = false;
                    if (mine) {
                        tile((uint32_t)here, lo, hi);
                    } else if (!(zeros >> (n & 1) & 1)) {
                        const uint32_t none[V / 2] = {};
#pragma unroll
                        for (uint32_t j = 0; j < H; j += V) {
                            put(2 * (q0 + j), none);
                            put(2 * (q0 + j + NQ), none);
                        }
                        zeros |= 1u << (n & 1);
                    }
                    if (here < (int)kTile && group == 0) clear_rows((uint32_t)here);
                    hand_over();
                    lo2 = lo1; hi2 = hi1;
                    lo1 = lo; hi1 = hi;
                }
            }
            const int idx = warp_reduce_many<(int)H>(l, (int)lane);      // (while the last product runs)
            sm.red[q0 + idx][quarter] = l[0];
            // (of either barrier the phase before is known to be over: the scores seen last came behind those values)
#pragma unroll 1
            for (uint32_t back = min(im.tiles, 2u); back; --back) {
                if (ok) ok = mbar_wait_warp(&sm.o_full[(n - back) & 1], ((n - back) >> 1) & 1, limit);
                tc5::fence_after();
                moved = moved && back == 2;
                add_values(n - back, back == 2 ? lo2 : lo1, back == 2 ? hi2 : hi1);
            }
            const uint32_t used = min(bd.nq - min(bd.nq, q0), H);        // this group's columns that are queries'
            const bool whole = bd.chunks == 1;
            if (!whole) {
                float *to = p.o + (size_t)(im.part + q0) * kHd + key;
#pragma unroll
                for (uint32_t j = 0; j < H; ++j)
                    if (j < used) to[(size_t)j * kHd] = o[j];
            }
            group_sync(bar);                                     // (sm.red)
            if (whole) {                                         // (the values that add_up gives one part)
#pragma unroll
                for (uint32_t j = 0; j < H; ++j) {
                    if (j >= used || !ok) break;
                    const float4 w = *reinterpret_cast<const float4 *>(sm.red[q0 + j]);
                    const float sum = (w.x + w.y) + (w.z + w.w);
                    p.out[(size_t)row_of(p, bd, im.kvh, q0 + j) * kHd + key] = sum == 0.f ? 0.f : o[j] / sum;
                }
            } else if (tid < used) {
                const float4 w = *reinterpret_cast<const float4 *>(sm.red[q0 + tid]);
                p.ml[im.part + q0 + tid] = make_float2(fresh ? WR_NEG_SENTINEL : -sm.nm[q0 + tid], (w.x + w.y) + (w.z + w.w));
            }
            ok = !all_or(!ok);
            if (!whole && ok && threadIdx.x == 96) {             // a part of these rows is there
                __threadfence();
                atomicAdd(p.done + im.bundle * p.n_kv + im.kvh, 1);
            }
        };
        for (uint32_t it = 0; ok && im.tiles; ++it) {
            queries(im, it);                                     // (the last item's scores have been read)
            switch (p.bundle[im.bundle].columns) {
            case 16: work(std::integral_constant<uint32_t, 16>{}, it); break;
            case 32: work(std::integral_constant<uint32_t, 32>{}, it); break;
            default: work(std::integral_constant<uint32_t, 64>{}, it);
            }
            im = item_at(it + 1, ok);
            ok = !all_or(!ok);
        }
        if (ok && p.parts) ok = add_up(p, reinterpret_cast<float4 *>(ps), warp - 3, lane);
        if (!ok && lane == 0) atomicCAS(p.err, 0, 84);
    }
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    if (warp == 1) tc5::dealloc(tmem, kTmemCols);
}

}  // namespace

// Groups: their sizes add up to the sessions, their rows are whole pages that all their sessions have, no more than the
// shortest of them attends.  Caller holds ctx->lock.
int wr_shared_validate(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *seq_lens,
                       uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const void *q, const void *out,
                       uint32_t n_q, int mem)
{
    int rc = wr_decode_validate(ctx, n_sess, kv, layer, seq_lens, q, out, n_q, mem, 0);
    if (rc != WR_CUDA_OK) return rc;
    if (kv[0]->hd_at(layer) != kHd) return WR_CUDA_ERR_UNSUPPORTED;
    if (!group_sess || !group_rows || n_groups == 0 || n_groups > n_sess) return WR_CUDA_ERR_INVAL;
    // (a row of the result may be there before another work item has read its query)
    const size_t bytes = (size_t)n_sess * n_q * kHd * sizeof(float);
    if (mem == WR_CUDA_MEM_DEVICE && wr_overlap(q, bytes, out, bytes)) return WR_CUDA_ERR_INVAL;
    uint32_t s = 0;
    for (uint32_t g = 0; g < n_groups; ++g) {
        if (group_sess[g] == 0 || group_sess[g] > n_sess - s || group_rows[g] % kPageTokens) return WR_CUDA_ERR_INVAL;
        for (uint32_t i = 0; i < group_sess[g]; ++i) {
            if (group_rows[g] > seq_lens[s + i]) return WR_CUDA_ERR_INVAL;
            if (i && wr_kv_common_pages(kv[s], kv[s + i]) < group_rows[g] / kPageTokens) return WR_CUDA_ERR_INVAL;
        }
        s += group_sess[g];
    }
    return s == n_sess ? WR_CUDA_OK : WR_CUDA_ERR_INVAL;
}

// What adding the parts up costs, in quarters of a tile.  One session's 1 / 2 / 3 / 5 tiles for eight kv heads: 6.0 / 6.9 / 6.9 / 8.9 us
// whole, - / 8.4 / 8.4 / 8.4 us in shares of a tile.
constexpr uint32_t kMergeCost = 13;
// Enqueue the kernel on device-resident q / out.  Caller holds ctx->lock and has validated the arguments.
int wr_shared_launch(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *seq_lens,
                     uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const float *dq, float *dout,
                     uint32_t n_q, float scale_override, const wr_shared_append *append, bool dependent)
{
    SharedParams p{};
    p.n_q = n_q;
    p.n_kv = kv[0]->n_kv_at(layer);
    p.per = n_q / p.n_kv;
    const uint32_t splits = (p.per + kMaxQ - 1) / kMaxQ, most = std::max(kMaxQ / p.per, 1u);     // bundles to a session, or sessions to a bundle
    uint32_t longest = 0;
    bool settled = true;                 // several hold the shared rows: no step has written them
    for (uint32_t g = 0, s = 0; g < n_groups; s += group_sess[g++]) {
        p.shared_pages[g] = kv[s]->d_pages + (size_t)layer * kv[s]->n_pages;
        p.shared_rows[g] = group_rows[g];
        settled = settled && (group_sess[g] > 1 || !group_rows[g]);
        for (uint32_t i = s; i < s + group_sess[g]; ++i) {
            p.own_pages[i] = kv[i]->d_pages + (size_t)layer * kv[i]->n_pages + group_rows[g] / kPageTokens;
            p.own_rows[i] = seq_lens[i] - group_rows[g];
        }
        for (uint32_t i = s; i < s + group_sess[g]; i += most) {
            const uint32_t n = std::min(most, s + group_sess[g] - i);
            if (p.n_bundles + splits > kMaxBundles) return WR_CUDA_ERR_LIMIT;
            const uint32_t shared = (group_rows[g] + kTile - 1) / kTile;
            uint32_t tiles = shared;
            for (uint32_t t = i; t < i + n; ++t) {
                tiles += (p.own_rows[t] + kTile - 1) / kTile;
                p.first_bundle[t] = (uint8_t)p.n_bundles;
            }
            for (uint32_t h = 0; h < splits; ++h) {
                const uint32_t heads = std::min(kMaxQ, p.per - h * kMaxQ);
                p.bundle[p.n_bundles++] = {g, i, n, h * kMaxQ, heads, shared, tiles, 0, 0, 0, n * heads, padded(n * heads), 65535 / heads + 1};
            }
            longest = std::max(longest, weight_of(shared, tiles));
        }
    }
    // Items are even shares of the bundles' lists, in one round of the SMs or a few, or whole lists: the less work one after the other,
    // an item's beginning and end counted as two tiles, the sooner.  No share is less than a tile.
    auto items_of = [&](uint32_t share) {
        uint64_t n = 0;
        for (uint32_t i = 0; i < p.n_bundles; ++i) {
            n += (uint64_t)shares_of(p.bundle[i].shared, p.bundle[i].tiles, share) * p.n_kv;
        }
        return n;
    };
    uint32_t share = longest, best = ~0u;
    for (uint32_t rounds = 1; rounds <= 5; ++rounds) {
        uint32_t lo = 4, hi = std::max(longest, 4u);             // the smallest share that makes no more items than that
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (items_of(mid) <= (uint64_t)rounds * ctx->sm_count) hi = mid;
            else lo = mid + 1;
        }
        if (rounds == 5) lo = longest;
        const uint32_t time = (uint32_t)((items_of(lo) + ctx->sm_count - 1) / ctx->sm_count) * (lo + 8) + (lo < longest ? kMergeCost : 0);
        if (time < best) {
            best = time;
            share = lo;
        }
    }
    uint64_t parts = 0;
    for (uint32_t i = 0; i < p.n_bundles; ++i) {
        Bundle &b = p.bundle[i];
        b.chunks = shares_of(b.shared, b.tiles, share);
        b.item0 = p.items;
        b.part0 = (uint32_t)parts;
        p.items += b.chunks * p.n_kv;
        if (b.chunks > 1) parts += (uint64_t)b.chunks * p.n_kv * b.nq;
    }
    if (parts > 0x7fffffffu) return WR_CUDA_ERR_LIMIT;
    // counters first: they are zeros between launches
    if ((size_t)p.n_bundles * p.n_kv * sizeof(int) + 256 > WR_KEPT_HEAD / 2) return WR_CUDA_ERR_LIMIT;
    const size_t head = WR_KEPT_HEAD, ml = ((size_t)parts * sizeof(float2) + 255) & ~(size_t)255;
    char *ws = nullptr;
    int rc = wr_ctx_keep(ctx, head + ml + (size_t)parts * kHd * sizeof(float), &ws);
    if (rc != WR_CUDA_OK) return rc;
    p.sched = reinterpret_cast<int *>(ws);
    p.done = reinterpret_cast<int *>(ws + 256);
    p.rows = n_sess * n_q;
    p.parts = (uint32_t)parts;
    p.ml = reinterpret_cast<float2 *>(ws + head);
    p.o = reinterpret_cast<float *>(ws + head + ml);
    p.q = dq;
    p.out = dout;
    if (append) {
        p.k_new = append->k;
        p.v_new = append->v;
        if (append->flags & WR_CUDA_APPEND_ROPE) {
            p.n_rot = append->n_rot_pairs >= 1 && append->n_rot_pairs < kHd / 2 ? append->n_rot_pairs : kHd / 2;     // kernels.c:1381-1383
            p.theta = append->theta_base < 1.0f ? 10000.0f : append->theta_base;                                    // kernels.c:1374
        }
    }
    p.scale_log2 = (scale_override > 0.0f ? scale_override : 1.0f / sqrtf((float)kHd)) * kLog2e;
    p.wait_limit = ctx->wait_limit;
    p.err = ctx->dev_err;
    if (!(ctx->attr_flags & 0x100u)) {
        WR_CUDA_TRY(cudaFuncSetAttribute(attn_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        ctx->attr_flags |= 0x100u;
    }
    const uint32_t grid = std::min<uint32_t>(p.items, (uint32_t)ctx->sm_count);
    // Behind another launch of this kernel, which writes rows that one session alone holds (a fork in between counts as another
    // kind of launch) and lets the next begin when all before it has ended.  Both run, or both are nodes of one graph.
    const unsigned long long capture = wr_ctx_capture(ctx);
    p.early = settled && dependent && ctx->pdl_index == ctx->launches && ctx->pdl_kind == WR_PDL_SHARED && ctx->pdl_capture == capture;
    for (uint32_t i = 0; i < p.n_bundles; ++i) p.widest = std::max(p.widest, p.bundle[i].columns);
    // a row's team: as many warps as there are for all rows at once
    for (p.team = kMergeWarps; p.team > 1 && (uint64_t)p.rows * p.team > (uint64_t)grid * kMergeWarps;) p.team /= 2;
    WR_CUDA_TRY(wr_launch(dependent, attn_shared_kernel, dim3(grid), dim3(kThreads), (size_t)kSmem, ctx->stream, p));
    ctx->launches++;
    ctx->pdl_kind = WR_PDL_SHARED;
    ctx->pdl_index = ctx->launches;
    ctx->pdl_capture = capture;
    WR_CUDA_TRY(cudaGetLastError());
    return WR_CUDA_OK;
}

// attn_decode_shared and, with `append`, decode_step_shared
static int shared_call(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *seq_lens, uint32_t n_groups,
                       const uint32_t *group_sess, const uint32_t *group_rows, const float *q, float *out, uint32_t n_q, float scale_override,
                       const wr_shared_append *append, int mem, bool dependent)
{
    const uint32_t n_kv = kv[0]->n_kv_at(layer);
    const size_t kv_bytes = append ? (size_t)n_sess * n_kv * kHd * sizeof(float) : 0, q_bytes = (size_t)n_sess * n_q * kHd * sizeof(float);
    if (mem == WR_CUDA_MEM_DEVICE)
        return wr_shared_launch(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, q, out, n_q, scale_override, append, dependent);
    int rc = wr_ctx_reserve_stage(ctx, 2 * kv_bytes + 2 * q_bytes, 0);
    if (rc != WR_CUDA_OK) return rc;
    char *d = (char *)ctx->stage_dev;
    float *const dq = (float *)(d + 2 * kv_bytes), *const dout = (float *)(d + 2 * kv_bytes + q_bytes);
    wr_shared_append staged;
    if (append) {
        staged = *append;
        staged.k = (const float *)d;
        staged.v = (const float *)(d + kv_bytes);
        WR_CUDA_TRY(cudaMemcpyAsync(d, append->k, kv_bytes, cudaMemcpyHostToDevice, ctx->stream));
        WR_CUDA_TRY(cudaMemcpyAsync(d + kv_bytes, append->v, kv_bytes, cudaMemcpyHostToDevice, ctx->stream));
    }
    WR_CUDA_TRY(cudaMemcpyAsync(dq, q, q_bytes, cudaMemcpyHostToDevice, ctx->stream));
    rc = wr_shared_launch(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, dq, dout, n_q, scale_override,
                          append ? &staged : nullptr, dependent);
    if (rc != WR_CUDA_OK) return rc;
    WR_CUDA_TRY(cudaMemcpyAsync(out, dout, q_bytes, cudaMemcpyDeviceToHost, ctx->stream));
    return wr_ctx_sync_checked(ctx);
}

extern "C" int wr_cuda_attn_decode_shared(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer,
                                          const uint32_t *seq_lens, uint32_t n_groups, const uint32_t *group_sess,
                                          const uint32_t *group_rows, const float *q, float *out, uint32_t n_q_heads,
                                          float scale_override, int mem)
{
    if (!ctx) return WR_CUDA_ERR_INVAL;
    std::lock_guard<std::mutex> g(ctx->lock);
    int rc = wr_shared_validate(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, q, out, n_q_heads, mem);
    if (rc != WR_CUDA_OK) return rc;
    WR_CUDA_TRY(cudaSetDevice(ctx->device));
    return shared_call(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, q, out, n_q_heads, scale_override, nullptr, mem, true);
}

int wr_decode_step_shared(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer, const uint32_t *positions,
                          uint32_t n_groups, const uint32_t *group_sess, const uint32_t *group_rows, const float *q, const float *k_rows,
                          const float *v_rows, float *out, uint32_t n_q_heads, float theta_base, uint32_t n_rot_pairs, uint32_t flags,
                          float scale_override, int mem, bool dependent)
{
    int rc = wr_append_validate(ctx, n_sess, kv, layer, positions, 1, k_rows, v_rows, q, n_q_heads, mem);
    if (rc != WR_CUDA_OK) return rc;
    uint32_t seq_lens[WR_CUDA_BATCH_MAX];
    for (uint32_t s = 0; s < n_sess; ++s) seq_lens[s] = positions[s] + 1;
    rc = wr_shared_validate(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, q, out, n_q_heads, mem);
    if (rc != WR_CUDA_OK) return rc;
    const size_t bytes = (size_t)n_sess * n_q_heads * kHd * sizeof(float), kv_bytes = (size_t)n_sess * kv[0]->n_kv_at(layer) * kHd * sizeof(float);
    if (mem == WR_CUDA_MEM_DEVICE && (wr_overlap(out, bytes, k_rows, kv_bytes) || wr_overlap(out, bytes, v_rows, kv_bytes))) return WR_CUDA_ERR_INVAL;
    // (a group's rows end before the row that is appended: what it shares is read only)
    for (uint32_t g = 0, s = 0; g < n_groups; s += group_sess[g++])
        for (uint32_t i = s; i < s + group_sess[g]; ++i)
            if (group_rows[g] > positions[i]) return WR_CUDA_ERR_INVAL;
    WR_CUDA_TRY(cudaSetDevice(ctx->device));
    const wr_shared_append append = {k_rows, v_rows, theta_base, n_rot_pairs, flags};
    return shared_call(ctx, n_sess, kv, layer, seq_lens, n_groups, group_sess, group_rows, q, out, n_q_heads, scale_override, &append, mem,
                       dependent);
}

extern "C" int wr_cuda_decode_step_shared(wr_cuda_ctx *ctx, uint32_t n_sess, wr_cuda_kv *const *kv, uint32_t layer,
                                          const uint32_t *positions, uint32_t n_groups, const uint32_t *group_sess,
                                          const uint32_t *group_rows, const float *q, const float *k_rows, const float *v_rows, float *out,
                                          uint32_t n_q_heads, float theta_base, uint32_t n_rot_pairs, uint32_t flags,
                                          float scale_override, int mem)
{
    if (!ctx) return WR_CUDA_ERR_INVAL;
    std::lock_guard<std::mutex> g(ctx->lock);
    return wr_decode_step_shared(ctx, n_sess, kv, layer, positions, n_groups, group_sess, group_rows, q, k_rows, v_rows, out, n_q_heads,
                                 theta_base, n_rot_pairs, flags, scale_override, mem);
}
