// PAGED_ATTENTION (parameter pack in include/zgml_cuda.h): softmax attention of the rows of a step over the 8-bit pages of their sequences.
//
// Both products run on the tensor cores in whole numbers, whose sums are exact: codes of 8 bits, which need no conversion, times digits of 8 bits.  A query is six digits of base 256 (45 bits
// of its largest element), a weight four (32 bits of the largest contribution); the digits of four queries are 24 and 16 columns of the instructions, codes their rows.  Stored codes are offset
// by 128: sum (c + 128) d - 128 sum d is exact too, and a bit of each code of a value is turned over.  Scales are powers of two: a key's joins its scores, a value's its weights.  A weight is 2^(s + e - n), with the score s in powers of
// two, e the exponent of its value's scale and n a whole number that no s + e passes by more than 3, so that the largest contributions keep their bits whatever the pages' scales
// are; the sum of the softmax has a frame m of its own, and the quotient is put right by the difference of the frames.  n falls again where weights have become small, before what they lose could add up to 2^-20 of
// sum w (127 scale) / sum w.  When n changes, products join those before in a frame of their own, in two parts, and the softmax's sum is kept in two: nothing grows with a sequence's length.
#include "pages.cuh"
#include "exp2.cuh"
#include "split_tc.cuh"

#include <algorithm>

namespace {

struct PgArgs {
    PagePool pool; PageShape s;
    float* dst; const float* q; const float* table; const void* sink;
    uint32_t* plan; float* part;     // what k_paged leaves for k_paged_join
    uint32_t B, H, rep, q_rs, dst_rs, window, sink_bf16, tokens, chunks;      // tokens of a sequence a warp takes together, chunks of a key head's query heads
    float scale, cap;
};
constexpr uint32_t kPgTile = 32, kPgShift = 29, kPgFlush = 512;      // tiles (512 of 32 products of two bytes: below 2^31)
constexpr float kPgCredit = 176.0f, kPgGrant = 3.0f;
constexpr uint32_t kPgPlan = 8;                                     // words of the plan before the rows' tiles: all tiles (64 bits), warps, -, warps / tiles (64 bits)
constexpr uint32_t kPgRows = 8, kPgLeast = 2;      // blocks of 32 rows that are read at once; tiles a warp at least where there are few (one sequence of 4096 tokens, us, with 1 / 2 / 4: 20.6 / 16.5 / 16.5)
constexpr float kPgSlack = 3.0f;                                     // weights reach 2^(29 + 3)
// Warps (CTAs) of an SM, by their registers: 16 of 128 a thread, 12 of 168, 8 of 255.
constexpr uint32_t pg_warps(int KC, int VC, int NT) { return NT == 1 && KC <= 2 && VC <= 4 ? 16 : NT == 1 && KC <= 4 && VC <= 8 ? 12 : 8; }
__device__ __forceinline__ float pg_sink(const PgArgs& a, uint32_t h) { return a.sink_bf16 ? __bfloat162float(reinterpret_cast<const bf16*>(a.sink)[h]) : reinterpret_cast<const float*>(a.sink)[h]; }
// 2^d of a whole number d, 0 below 2^-126
__device__ __forceinline__ float pg_pow2(float d) { return d < -126.0f ? 0.0f : __int_as_float(((int)fminf(d, 127.0f) + 127) << 23); }
// D = A B (+ D): 16 rows of 32 codes as they are stored and signed digits of a query; codes that have their sign and unsigned digits of weights
__device__ __forceinline__ void pg_scores(int (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], bool first) {
    if (first)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(0));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void pg_outputs(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pg_copy(uint32_t to, const uint8_t* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float pg_frame(float from, float to) { return from == to ? 1.0f : pg_pow2(from - to); }      // (also where both are infinite)
// 2^back x, in two steps: the scales of the values may lie anywhere
__device__ __forceinline__ float pg_scaled(float x, float back) {
    const float half = truncf(back * 0.5f);
    return x * exp2f(half) * exp2f(back - half);
}
// floats of a warp behind its tile: outputs in two parts, one of a lane for each four queries, statistics of queries (W = 8)
__host__ __device__ constexpr uint32_t pg_aside(uint32_t NT, uint32_t vp) { return NT * (8 * vp + 32 + 16); }
// What x brings joins f times a sum, f a power of two, kept as (sum, what its roundings added too much): W. Kahan, Communications of the ACM 8, 1965.  However many parts, two roundings of the sum of their magnitudes.
__device__ __forceinline__ float2 pg_add(float2 sum, float f, float x) {
    const float y = fmaf(-sum.y, f, x), t = fmaf(sum.x, f, y);
    return make_float2(t, fmaf(-sum.x, f, t) - y);
}
// sum of w x, by pairs
__device__ __forceinline__ float pg_tree(const float (&w)[8], const float (&x)[8]) {
    return (fmaf(w[0], x[0], w[1] * x[1]) + fmaf(w[2], x[2], w[3] * x[3])) + (fmaf(w[4], x[4], w[5] * x[5]) + fmaf(w[6], x[6], w[7] * x[7]));
}
// What a query's outputs are multiplied by as a power of two, and divided by, in the frames m of the sum and n of the outputs.
__device__ __forceinline__ float2 pg_finish(const PgArgs& a, uint32_t h, float m, float n, float sum) {
    float back = n - m - (float)kPgShift;
    if (a.sink) {
        const float sink = pg_sink(a, h) * kLog2e, to = fmaxf(m, ceilf(sink));      // (a sink far above the scores takes the frame with it)
        sum = sum * pg_frame(m, to) + (to == -INFINITY ? 0.0f : sa_ex2(sink - to));
        back += m - to;
    }
    return make_float2(back, sum);
}
// What a group of rows of one sequence, taken together, sees: its rows and its tiles of 32 positions.
struct PgGroup { uint32_t rows, first, tiles; };
__device__ __forceinline__ PgGroup pg_group(const PgArgs& a, uint32_t live, uint32_t r, int32_t slot) {
    PgGroup x = {0, 0, 0};
    uint32_t lo = 0xffffffffu, hi = 0;
    for (uint32_t i = 0; i < a.tokens && r + i < live; i++) {
        const BatchRow z = batch_row(a.table, r + i);
        if (z.slot != slot) break;
        x.rows++;
        if (page_row_ok(a.pool, a.s, z) && z.length > 0) { lo = min(lo, a.window && (uint32_t)z.length > a.window ? z.length - a.window : 0); hi = max(hi, (uint32_t)z.length); }
    }
    if (hi) { x.first = lo / kPgTile; x.tiles = (hi + kPgTile - 1) / kPgTile - x.first; }
    return x;
}
// 32 rows from `row` on, one a lane: tiles of those that begin a group, 0 of the others.  `run`: the row at which the run of one slot before them began.
__device__ __forceinline__ uint32_t pg_tiles(const PgArgs& a, uint32_t live, uint32_t row, uint32_t& run) {
    const uint32_t lane = threadIdx.x % 32, r = row + lane;
    const int32_t slot = r < live ? batch_row(a.table, r).slot : -1;
    if (a.tokens == 1) return slot < 0 ? 0 : pg_group(a, live, r, slot).tiles;
    const bool begins = r == 0 || r >= live || batch_row(a.table, r - 1).slot != slot;
    const uint32_t starts = __ballot_sync(0xffffffffu, begins), below = starts & (0xffffffffu >> (31 - lane)), start = below ? row + 31 - __clz(below) : run;
    run = starts ? row + 31 - __clz(starts) : run;
    return slot < 0 || (r - start) % a.tokens ? 0 : pg_group(a, live, r, slot).tiles;
}
// the first of the tiles that warp w of `warps` takes of all
__device__ __forceinline__ uint64_t pg_share(uint64_t all, uint32_t w, uint32_t warps) { return all * w / warps; }

// A warp of its own CTA takes a share of all tiles of the step - one group of rows after the other, one key head (and chunk of its query heads) after the other - so that
// warps have equal work whatever the sequences' lengths are, and none waits for another.  What it takes of a sequence begins or ends with it, or leaves a record for
// k_paged_join: (m, n, sum, outputs) of each query.  (W = 8: a CTA of eight warps for each group and key head, whose records are joined in shared memory: one launch, for few short sequences
// and where there is no workspace.)  A tile's next keys come while its weights and outputs are computed, its next values while the scores are.  4 NT queries at a time, query 4 t + lane % 4 a lane.
// Bound by HBM in long caches (32 / 8 heads of 128, 16 rows of up to 65536 tokens, 1307 MB: 202 us for the launch by itself, 6.5 TB/s).  64 rows of up to 4096, 305 MB, take 63 us, 4.9 TB/s: some 20 us of either are
// a warp's way to its first tile (table, page, copy, query, digits one after the other) and its changes of sequence and key head, with no copies under way.
template <int KC, int VC, int NT, bool FULL, int W>
__global__ void __launch_bounds__(32 * W, W == 1 ? pg_warps(KC, VC, NT) : 1) k_paged(const __grid_constant__ PgArgs a) {
    pdl_enter();
    extern __shared__ float4 pg_mem[];
    __shared__ uint64_t bars[W][2];                                  // of a warp's keys and values
    const PageShape& s = a.s;
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, row8 = lane / 4, j = lane % 4;
    const uint32_t heads = min(a.rep, 4u * NT), per_row = s.G * a.chunks;      // query heads of a chunk; products of a group of rows
    const uint32_t live = batch_head(a.table, a.B).rows;
    const uint32_t kp = FULL ? 32 * KC : s.kp, vp = FULL ? 16 * VC : s.vp, kc = kp / 32, vc = vp / 16, k_bytes = kPgTile * kp, buffer_bytes = k_bytes + kPgTile * vp + 32 + 4 * pg_aside(NT, vp);
    uint8_t* const buffer = reinterpret_cast<uint8_t*>(pg_mem) + warp * buffer_bytes;
    float2* const rec = reinterpret_cast<float2*>(buffer + k_bytes + kPgTile * vp + 32) + lane;      // a lane's outputs in two parts, 32 apart
    float* const aside = &rec[4 * NT * vp].x - lane;                 // what a lane seldom needs
    // rows that see nothing, or whose words are out of range
    auto settle = [&](uint32_t row) {
        const BatchRow z = batch_row(a.table, row);
        const bool ok = page_row_ok(a.pool, s, z);
        if (z.slot < 0 || (ok && z.length > 0)) return;
        for (uint32_t d = lane; d < a.H * s.dv; d += 32) a.dst[(size_t)row * a.dst_rs + d] = ok ? 0.0f : kBatchNaN;
    };
    uint32_t r, item, off;
    uint64_t left;                                                   // tiles that the warp takes
    PgGroup group;
    if constexpr (W == 1) {
        // Tiles before each row, of all, and the row in which the warp's share begins.  The rows of a step of at most 32 * kPgRows are read at once and kept.
        uint64_t* const before = reinterpret_cast<uint64_t*>(a.plan + kPgPlan);
        auto upto = [&](uint32_t mine) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, mine, o); if (lane >= (uint32_t)o) mine += t; }
            return mine;
        };
        const bool few = a.tokens == 1 && a.B <= 32 * kPgRows;
        uint32_t kept[kPgRows];
        uint64_t all = 0;
        if (few) {
            int2 z[kPgRows];                                         // slot, length
#pragma unroll
            for (uint32_t b = 0; b < kPgRows; b++)
                z[b] = 32 * b + lane < a.B ? *reinterpret_cast<const int2*>(a.table + ZG_BATCH_ROWS + (size_t)4 * (32 * b + lane)) : make_int2(-1, 0);
#pragma unroll
            for (uint32_t b = 0; b < kPgRows; b++) {
                if (32 * b >= live) break;
                BatchRow x;
                x.slot = 32 * b + lane < live ? z[b].x : -1; x.length = z[b].y; x.adapter = 0;
                const uint32_t hi = x.slot >= 0 && page_row_ok(a.pool, s, x) ? x.length : 0, lo = a.window && hi > a.window ? hi - a.window : 0;
                kept[b] = hi ? (hi + kPgTile - 1) / kPgTile - lo / kPgTile : 0;
                const uint32_t sum = upto(kept[b]);
                if (blockIdx.x == 0 && 32 * b + lane < live) before[32 * b + lane] = all + sum - kept[b];
                all += __shfl_sync(0xffffffffu, sum, 31);
            }
        } else {
            uint32_t run = 0;
            for (uint32_t row = 0; row < live; row += 32) {
                const uint32_t mine = pg_tiles(a, live, row, run), sum = upto(mine);
                if (blockIdx.x == 0 && row + lane < live) before[row + lane] = all + sum - mine;
                all += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        const uint64_t total = all * per_row;
        const uint32_t warps = (uint32_t)min((uint64_t)gridDim.x, max((uint64_t)1, total / kPgLeast));
        if (blockIdx.x == 0 && lane == 0) { before[live] = all; a.plan[0] = (uint32_t)total; a.plan[1] = (uint32_t)(total >> 32); a.plan[2] = warps; *reinterpret_cast<double*>(a.plan + 4) = total ? (double)warps / (double)total : 0.0; }
        const bool idle = blockIdx.x >= warps || !total;
        for (uint32_t row = gridDim.x - 1 - blockIdx.x; row < live; row += gridDim.x) settle(row);      // (from the last warp on, which may have nothing else to do)
        if (idle) return;
        const uint64_t begin = pg_share(total, blockIdx.x, warps), x = begin / per_row;
        left = pg_share(total, blockIdx.x + 1, warps) - begin;
        uint64_t seen = 0;
        uint32_t run = 0;
        r = item = off = 0;
        auto look = [&](uint32_t row, uint32_t mine) {
            const uint32_t sum = upto(mine), here = __ballot_sync(0xffffffffu, seen + sum > x);
            if (here) {
                const int l = __ffs(here) - 1;
                const uint32_t tiles = __shfl_sync(0xffffffffu, mine, l);
                const uint64_t in = begin - (seen + __shfl_sync(0xffffffffu, sum, l) - tiles) * per_row;
                r = row + l; item = (uint32_t)(in / tiles); off = (uint32_t)(in % tiles);
                return true;
            }
            seen += __shfl_sync(0xffffffffu, sum, 31);
            return false;
        };
        if (few) {
#pragma unroll
            for (uint32_t b = 0; b < kPgRows; b++) if (look(32 * b, kept[b])) break;
        } else for (uint32_t row = 0; row < live && !look(row, pg_tiles(a, live, row, run)); row += 32) {}
        group = pg_group(a, live, r, batch_row(a.table, r).slot);
    } else {
        r = blockIdx.x / per_row; item = blockIdx.x % per_row;
        if (r >= live) return;
        if (item == 0 && warp == 0) settle(r);
        const int32_t slot = batch_row(a.table, r).slot;
        if (slot < 0) return;
        if (a.tokens > 1) {
            uint32_t back = 0, same;                                 // rows of the same slot directly before r
            do {
                same = __ballot_sync(0xffffffffu, back + lane < r && batch_row(a.table, r - 1 - back - lane).slot == slot);
                back += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
            } while (same == 0xffffffffu);
            if (back % a.tokens) return;
        }
        group = pg_group(a, live, r, slot);
        if (!group.tiles) return;
        off = (uint32_t)pg_share(group.tiles, warp, W);
        left = (uint32_t)pg_share(group.tiles, warp + 1, W) - off;
    }
    const uint32_t k_bar = smem_u32(&bars[warp][0]), v_bar = k_bar + 8, at = smem_u32(buffer), heads_at = at + k_bytes + kPgTile * vp;
    if (lane == 0) {
        mbar_init(k_bar, 2);
        mbar_init(v_bar, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const size_t page_size = page_bytes(s);
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    uint32_t k_phase = 0, v_phase = 0;
    bool gave_up = false;                                            // a wait ran out: no more copies, and from there on no outputs are numbers
    for (;;) {
        const uint32_t g = item / a.chunks, chunk = item % a.chunks, slot = batch_row(a.table, r).slot, take = (uint32_t)min((uint64_t)(group.tiles - off), left);
        const uint32_t t0 = group.first + off, t1 = t0 + take, pages = ((group.first + group.tiles) * kPgTile + s.page - 1) >> s.shift;
        // the page of half `lane` of a tile: its id, -1 for one that does not exist, -2 behind the table's (the rest of a tile that no row sees)
        auto find = [&](uint32_t tile) {
            const uint32_t n = (tile * kPgTile + 16 * (lane & 1)) >> s.shift;
            return tile < t1 && n < pages && n < a.pool.most ? page_id(a.pool, slot, n) : -2;
        };
        const uint8_t* const parts = a.pool.pages + (size_t)g * s.head;
        // keys, with the scales, or values of a tile: a bulk copy for each half, by lanes 0 and 1.  What no page holds is left as it is, and gets scales alone
        auto fetch = [&](uint32_t tile, int32_t id, bool values) {
            if (lane >= 2) return;
            const uint8_t* part = parts + (size_t)max(id, 0) * page_size;
            const uint32_t in = (tile * kPgTile + 16 * lane) & (s.page - 1), bar = values ? v_bar : k_bar;
            mbar_expect_tx(bar, id < 0 ? 0 : values ? 16 * vp : 16 * kp + kPageHead);
            if (id < 0) {
                if (!values) {
                    *reinterpret_cast<float2*>(buffer + k_bytes + kPgTile * vp + kPageHead * lane) = id == -1 ? make_float2(kBatchNaN, kBatchNaN) : make_float2(1.0f, 1.0f);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
            } else if (values) pg_copy(at + k_bytes + 16 * vp * lane, part + kPageHead + s.page * kp + in * vp, 16 * vp, bar);
            else {
                pg_copy(at + 16 * kp * lane, part + kPageHead + in * kp, 16 * kp, bar);
                pg_copy(heads_at + kPageHead * lane, part, kPageHead, bar);
            }
        };
        int32_t id = find(t0);
        if (!gave_up && (W == 1 || take)) { fetch(t0, id, false); fetch(t0, id, true); }
        __syncwarp();
        id = find(t0 + 1);
        // what the lane's queries see, and its column of the first product: three of the six digits of a query, and 128 times their sums
        uint32_t len[NT], low[NT], all_in = 0xffffffffu, least = 0;      // (all_in, least: positions that every query sees)
        uint32_t qd[NT][KC][3][2];
        int offset[NT][3];
        float q_scale[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            len[t] = low[t] = 0;
            const uint32_t mine = 4 * t + j;
            if (mine / heads < group.rows && chunk * heads + mine % heads < a.rep) {
                const BatchRow x = batch_row(a.table, r + mine / heads);
                if (page_row_ok(a.pool, s, x)) { len[t] = x.length; low[t] = a.window && len[t] > a.window ? len[t] - a.window : 0; }
            }
            if (len[t]) { all_in = min(all_in, len[t]); least = max(least, low[t]); }
            const uint32_t i = 4 * t + row8 / 2, token = i / heads, h = chunk * heads + i % heads;
            const bool on = token < group.rows && h < a.rep;
            const float* q = a.q + (size_t)(r + (on ? token : 0)) * a.q_rs + (g * a.rep + (on ? h : 0)) * s.dk;
            float x[KC][8];
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t d = 32 * c + 8 * j + e;
                    x[c][e] = on && d < s.dk ? q[d] : 0.0f;
                    top = max(top, __float_as_uint(fabsf(x[c][e])));
                }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t e = max(top >> 23, 46u);                      // its exponent
            const float f = __uint_as_float((275u - e) << 23);           // 2^21 / 2^(e - 127): elements are below 2^22, so that their first digits are at most 64
            q_scale[t] = top >= 0x7f800000u ? kBatchNaN : __uint_as_float((e - 44u) << 23) * a.scale * (a.cap > 0.0f ? 1.0f : kLog2e);      // (1 / (f 2^23))
            q_scale[t] = __shfl_sync(0xffffffffu, q_scale[t], 8 * j);    // (of the lane's scores)
            // element = (hi + lo 2^-23) / f, hi and lo three digits each, of which an even row8's column takes 5, 3, 1 and an odd one's 4, 2, 0
            const bool odd = row8 & 1;
            int sums[3] = {0, 0, 0};
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint32_t hi[4], lo[4], word[3];
#pragma unroll
                    for (int i4 = 0; i4 < 4; i4++) {
                        const float y = x[c][4 * k + i4] * f, whole = rintf(y);
                        hi[i4] = (uint32_t)((int)whole + 0x8080);
                        lo[i4] = (uint32_t)((int)((y - whole) * 8388608.0f) + 0x8080);
                    }
#pragma unroll
                    for (int n3 = 0; n3 < 3; n3++) {
                        const bool high = n3 == 0 || (n3 == 1 && !odd);
                        const uint32_t at = n3 == 0 ? (odd ? 1 : 2) : n3 == 1 ? (odd ? 2 : 0) : (odd ? 0 : 1), pick = at | (at + 4) << 4;
                        uint32_t v[4];
#pragma unroll
                        for (int i4 = 0; i4 < 4; i4++) v[i4] = high ? hi[i4] : lo[i4];
                        word[n3] = __byte_perm(__byte_perm(v[0], v[1], pick), __byte_perm(v[2], v[3], pick), 0x5410) ^ (at == 2 ? 0u : 0x80808080u);
                        sums[n3] = __dp4a((int)word[n3], 0x01010101, sums[n3]);
                        qd[t][c][n3][k] = word[n3];
                    }
                }
#pragma unroll
            for (int n3 = 0; n3 < 3; n3++) {
                sums[n3] += __shfl_xor_sync(0xffffffffu, sums[n3], 1);
                sums[n3] += __shfl_xor_sync(0xffffffffu, sums[n3], 2);
                offset[t][n3] = -128 * ((n3 == 1 ? 128 : 256) * __shfl_sync(0xffffffffu, sums[n3], 8 * j) + __shfl_sync(0xffffffffu, sums[n3], 8 * j + 4));
            }
        }
        all_in = __reduce_min_sync(0xffffffffu, all_in);
        least = __reduce_max_sync(0xffffffffu, least);
        // Frames: m of the lane's sum of weights, n of the products' weights.  They stay while no score passes them by much, which one vote of the warp tells.  But weights far below n are rounded the
        // same way by the thousand (in one frame for a sequence, outputs of 1.3e-4 came out as 2.4e-4 behind 65536 keys some 2^29 below the first).  So lanes pay for n: for each tile, in which a lane's four weights may
        // lose 2^-28 of 2^n together, 2^n is taken from its credit, and kPgCredit times what they weigh is added.  Where nothing is left, n becomes what the present tile asks for, and lanes in debt get
        // kPgGrant times the new 2^n: eight lanes at most 48 times the largest contribution of this tile.  Their debts, of at most 2^n each, are 16 times that of the tile that set n, or less.  So all that is
        // taken is at most 176 + 48 + 16 times what all weights are, and what is lost 240 * 2^-28 of that, however many they are.  (64 rows of 64 / 8 heads of 128, up to 8192, us: 163, with one frame and plain
        // sums 153, with products put away every 8 tiles 170; of 32 / 8 heads, up to 4096, 64.3 with either.)
        float m[NT], n[NT], credit[NT];                              // credit in units of 2^n
        float2 sum[NT];
        auto kept = [&](int t) { return aside + 32 * t; };           // the frame of the products that were put away
        int o[NT][VC][2][4];                                         // even and odd digits: two of each
        uint32_t since = 0;                                          // tiles since the products were put away
        bool stored = false;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            m[t] = n[t] = *kept(t) = -INFINITY;
            credit[t] = 0.0f;
            sum[t] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < VC; c++)
#pragma unroll
                for (int k = 0; k < 8; k++) o[t][c][k / 4][k % 4] = 0;
        }
        auto output = [&](int t, int c, int k) {                     // in the frame n
            const int (&x)[2][4] = o[t][c];
            return fmaf(fmaf(fmaf((float)x[1][2 * k + 1], 256.0f, (float)x[0][2 * k + 1]), 256.0f, (float)x[1][2 * k]), 256.0f, (float)x[0][2 * k]);
        };
        auto place = [&](int t, int c, int k) { return 32 * (2 * (t * vc + c) + k); };
        for (uint32_t tile = t0; tile < t1 && !gave_up; tile++) {
            const bool more = tile + 1 < t1;
            if (!__all_sync(0xffffffffu, mbar_wait(k_bar, k_phase))) {
                gave_up = true;                                      // (what is under way lands before the memory is left)
                mbar_wait(k_bar, k_phase);
                mbar_wait(v_bar, v_phase);
                break;
            }
            k_phase ^= 1;
            const uint8_t* const mine = buffer + 8 * lane;
            const float2 s0 = *reinterpret_cast<const float2*>(buffer + k_bytes + kPgTile * vp), s1 = *reinterpret_cast<const float2*>(buffer + k_bytes + kPgTile * vp + kPageHead);
            const float4 scales = make_float4(s0.x, s0.y, s1.x, s1.y);      // of keys and values of each half
            // scores: sixteen positions a step, of which a lane gets two (row8 and row8 + 8) of its query
            float sc[NT][2][2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                int acc[NT][3][4];
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    if (!FULL && c >= kc) break;
                    const uint2 x = *reinterpret_cast<const uint2*>(mine + (2 * u * kc + c) * 256), y = *reinterpret_cast<const uint2*>(mine + ((2 * u + 1) * kc + c) * 256);
                    const uint32_t f[4] = {x.x, y.x, x.y, y.y};
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int n3 = 0; n3 < 3; n3++) pg_scores(acc[t][n3], f, qd[t][c][n3], c == 0);
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float scale = q_scale[t] * (u ? scales.z : scales.x);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float part[3];
#pragma unroll
                        for (int n3 = 0; n3 < 3; n3++) part[n3] = (float)(acc[t][n3][2 * k] * (n3 == 1 ? 128 : 256) + acc[t][n3][2 * k + 1] + offset[t][n3]);
                        sc[t][u][k] = fmaf(fmaf(part[0], 32768.0f, part[1]), 65536.0f, part[2]) * scale;
                    }
                }
            }
            __syncwarp();
            if (more) fetch(tile + 1, id, false);
            if (a.cap > 0.0f) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int k = 0; k < 4; k++) sc[t][k / 2][k % 2] = sa_capped(sc[t][k / 2][k % 2], a.cap, inv_cap) * kLog2e;
            }
            if (tile * kPgTile < least || tile * kPgTile + kPgTile > all_in) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t p = tile * kPgTile + 8 * k + row8;
                        if (p >= len[t] || p < low[t]) sc[t][k / 2][k % 2] = -INFINITY;
                    }
            }
            // weights
            const float e[2] = {scales.y == scales.y ? (float)((int)(__float_as_uint(scales.y) >> 23) - 127) : kBatchNaN, scales.w == scales.w ? (float)((int)(__float_as_uint(scales.w) >> 23) - 127) : kBatchNaN};
            bool over = false;
            float top[NT];                                           // the lane's largest contribution
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float top0 = fmaxf(sc[t][0][0], sc[t][0][1]), top1 = fmaxf(sc[t][1][0], sc[t][1][1]);
                top[t] = fmaxf(top0 + e[0], top1 + e[1]);
                over = over || top[t] > n[t] + kPgSlack || fmaxf(top0, top1) > m[t] + 64.0f || (credit[t] < 0.0f && n[t] > -INFINITY);
            }
            if (__any_sync(0xffffffffu, over) || since == kPgFlush) {
                if (since) {                                         // the products so far go to shared memory, in a frame of theirs
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        const float from = *kept(t), to = fmaxf(from, n[t]), before = pg_frame(from, to), now = pg_frame(n[t], to);
                        *kept(t) = to;
#pragma unroll
                        for (int c = 0; c < VC; c++) {
                            if (!FULL && c >= vc) break;
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const uint32_t at = place(t, c, k);
                                rec[at] = pg_add(stored ? rec[at] : make_float2(0.0f, 0.0f), before, output(t, c, k) * now);
                            }
#pragma unroll
                            for (int k = 0; k < 8; k++) o[t][c][k / 4][k % 4] = 0;
                        }
                    }
                    stored = true;
                    since = 0;
                }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float new_m = fmaxf(m[t], ceilf(fmaxf(fmaxf(sc[t][0][0], sc[t][0][1]), fmaxf(sc[t][1][0], sc[t][1][1])))), f = new_m == m[t] ? 1.0f : pg_pow2(m[t] - new_m);
                    float most = top[t], least_left = credit[t];
#pragma unroll
                    for (int k = 4; k < 32; k *= 2) { most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k)); least_left = fminf(least_left, __shfl_xor_sync(0xffffffffu, least_left, k)); }
                    const float new_n = least_left < 0.0f ? ceilf(most) : fmaxf(n[t], ceilf(most));
                    credit[t] = credit[t] >= 0.0f && n[t] > -INFINITY ? fminf(credit[t] * pg_pow2(fminf(n[t] - new_n, 60.0f)), 0x1p60f) : kPgGrant;
                    sum[t].x *= f; sum[t].y *= f;
                    m[t] = new_m; n[t] = new_n;
                }
            }
            since++;
            uint32_t low_digits[NT][2], high_digits[NT][2];              // of each half's weights: digits 0 and 2, and 1 and 3, of four positions
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float fm = m[t] == -INFINITY ? 0.0f : m[t], fn = (float)kPgShift - (n[t] == -INFINITY ? 0.0f : n[t]);
                float weights[2], mass = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t turned[2];
                    weights[u] = 0.0f;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const float x = sc[t][u][k], y = x == -INFINITY ? 0.0f : sa_ex2(x + (fn + e[u]));
                        mass += y;
                        weights[u] += sa_ex2(x - fm);
                        const uint32_t w = __float2uint_rn(y);
                        // a lane's weight is two columns of 16 bits, a position a row; turned around they are rows of positions
                        asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(turned[k]) : "r"(w));
                    }
                    low_digits[t][u] = __byte_perm(turned[0], turned[1], 0x6420);
                    high_digits[t][u] = __byte_perm(turned[0], turned[1], 0x7531);
                }
                sum[t] = pg_add(sum[t], 1.0f, (weights[0] + weights[1]) + (mass - mass));      // (a scale that is not a number is one of the sum's too)
                credit[t] = fmaf(mass, kPgCredit / (float)(1u << kPgShift), credit[t] - 1.0f);
            }
            __syncwarp();
            if (!__all_sync(0xffffffffu, mbar_wait(v_bar, v_phase))) {
                gave_up = true;
                if (more) mbar_wait(k_bar, k_phase);
                mbar_wait(v_bar, v_phase);
                break;
            }
            v_phase ^= 1;
#pragma unroll
            for (int c = 0; c < VC; c++) {
                if (!FULL && c >= vc) break;
                const uint2 x = *reinterpret_cast<const uint2*>(mine + k_bytes + c * 256), y = *reinterpret_cast<const uint2*>(mine + k_bytes + (vc + c) * 256);
                const uint32_t f[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, y.x ^ 0x80808080u, y.y ^ 0x80808080u};
#pragma unroll
                for (int t = 0; t < NT; t++) { pg_outputs(o[t][c][0], f, low_digits[t][0], low_digits[t][1]); pg_outputs(o[t][c][1], f, high_digits[t][0], high_digits[t][1]); }
            }
            __syncwarp();
            if (more) { fetch(tile + 1, id, true); id = find(tile + 2); }
            __syncwarp();
        }
        if (gave_up) {
#pragma unroll
            for (int t = 0; t < NT; t++) sum[t].x = kBatchNaN;
        }
        const bool whole = W == 1 && take == group.tiles;
        float* const record = whole || W > 1 ? nullptr : a.part + (size_t)(2 * blockIdx.x + (off ? 0 : 1)) * 4 * NT * (vp + 4);
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float top = m[t];
#pragma unroll
            for (int k = 4; k < 32; k *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            float total = sum[t].x * pg_frame(m[t], top);
#pragma unroll
            for (int k = 4; k < 32; k *= 2) total += __shfl_xor_sync(0xffffffffu, total, k);
            const uint32_t i = 4 * t + j, token = i / heads, h = chunk * heads + i % heads;
            const bool on = token < group.rows && h < a.rep;
            const float frame = fmaxf(*kept(t), n[t]), before = pg_frame(*kept(t), frame), now = pg_frame(n[t], frame);
            float* to;
            float2 f = make_float2(0.0f, 1.0f);
            if (whole) {
                const BatchRow z = batch_row(a.table, r + (on ? token : 0));
                if (!on || !page_row_ok(a.pool, s, z) || z.length == 0) continue;      // (the latter two: settle)
                f = pg_finish(a, g * a.rep + h, top, frame, total);
                to = a.dst + (size_t)(r + token) * a.dst_rs + (g * a.rep + h) * s.dv;
            } else {
                float* const stats = W > 1 ? aside - lane + 32 * NT + 4 * i : record + i * (vp + 4);
                to = stats + 4;
                if (row8 == 0) *reinterpret_cast<float4*>(stats) = make_float4(top, frame, total, 0.0f);
            }
#pragma unroll
            for (int c = 0; c < VC; c++) {
                if (!FULL && c >= vc) break;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t d = 16 * c + 8 * k + row8;
                    float v = output(t, c, k) * now;
                    const uint32_t at = place(t, c, k);
                    if (stored) v = pg_add(rec[at], before, v).x;
                    if (W > 1) rec[at].x = v;
                    else if (!whole) to[d] = v;
                    else if (d < s.dv) to[d] = pg_scaled(v / f.y, f.x);
                }
            }
        }
        __syncwarp();
        left -= take;
        if (W > 1 || !left) break;
        off = 0;
        if (++item == per_row) {
            item = 0;
            do {
                r += max(1u, group.rows);
                if (r >= live) return;
                group = pg_group(a, live, r, batch_row(a.table, r).slot);
            } while (batch_row(a.table, r).slot < 0 || !group.tiles);      // (there is one: the warp has tiles left)
        }
    }
    if (gave_up && lane == 0) count_timeout();
    if constexpr (W > 1) {
        static_assert(NT == 1 && W == 8);
        __syncthreads();
        const uint32_t g = item / a.chunks, h = item % a.chunks * heads + j % heads, row = r + j / heads;      // a lane's query and places are those that it had
        if (j / heads >= group.rows || h >= a.rep) return;
        const BatchRow z = batch_row(a.table, row);
        if (!page_row_ok(a.pool, s, z) || z.length == 0) return;
        const uint8_t* const records = reinterpret_cast<const uint8_t*>(pg_mem) + k_bytes + kPgTile * vp + 32;
        float4 st[W];
        float m = -INFINITY, n = -INFINITY, w[W], x[W];
#pragma unroll
        for (uint32_t k = 0; k < W; k++) {
            st[k] = reinterpret_cast<const float4*>(records + k * buffer_bytes)[2 * vp + 8 + j];
            m = fmaxf(m, st[k].x); n = fmaxf(n, st[k].y);
        }
#pragma unroll
        for (uint32_t k = 0; k < W; k++) { x[k] = st[k].z; w[k] = pg_frame(st[k].x, m); }
        const float2 f = pg_finish(a, g * a.rep + h, m, n, pg_tree(w, x));
#pragma unroll
        for (uint32_t k = 0; k < W; k++) w[k] = pg_frame(st[k].y, n);
        float* const to = a.dst + (size_t)row * a.dst_rs + (g * a.rep + h) * s.dv;
        for (uint32_t p = warp; p < 2 * vc; p += W) {
            const uint32_t d = 8 * p + row8;
#pragma unroll
            for (uint32_t k = 0; k < W; k++) x[k] = reinterpret_cast<const float2*>(records + k * buffer_bytes)[32 * p + lane].x;
            if (d < s.dv) to[d] = pg_scaled(pg_tree(w, x) / f.y, f.x);
        }
    }
}

// The records of a sequence that several warps took: a warp a query, or (SHARED) the four of a CTA, a quarter of the records each.  Bound by latency: eight records at a time, statistics
// and outputs at once.
template <bool SHARED>
__global__ void __launch_bounds__(128, 4) k_paged_join(const __grid_constant__ PgArgs a, const uint32_t queries) {
    pdl_enter();
    const PageShape& s = a.s;
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = blockIdx.y, query = SHARED ? blockIdx.x : 4 * blockIdx.x + warp, item = query / queries, i = query % queries, per_row = s.G * a.chunks;
    const uint32_t live = batch_head(a.table, a.B).rows;
    const uint64_t* const before = reinterpret_cast<const uint64_t*>(a.plan + kPgPlan);
    const uint4 plan = *reinterpret_cast<const uint4*>(a.plan);      // (asked for at once: what belongs to rows that are not live is not looked at)
    const double inv = *reinterpret_cast<const double*>(a.plan + 4);
    const uint64_t b0 = before[r], b1 = before[r + 1];
    const BatchRow begins = batch_row(a.table, r);
    if (r >= live || b1 == b0 || item >= per_row) return;
    const uint64_t all = plan.x | (uint64_t)plan.y << 32, tiles = b1 - b0, first = b0 * per_row + item * tiles;
    const uint32_t warps = plan.z;
    auto taker = [&](uint64_t tile) {                                // the last warp whose share begins at or before the tile
        const uint64_t n = (tile + 1) * warps - 1;
        uint32_t w = min((uint32_t)((double)tile * inv), warps - 1);
        while (w + 1 < warps && all * (w + 1) <= n) w++;
        while (w && all * w > n) w--;
        return w;
    };
    const uint32_t w0 = taker(first), w1 = taker(first + tiles - 1), count = w1 - w0 + 1;
    const uint32_t heads = min(a.rep, queries), token = i / heads, g = item / a.chunks, h = item % a.chunks * heads + i % heads;
    if (w0 == w1 || h >= a.rep || (token && token >= pg_group(a, live, r, begins.slot).rows)) return;
    const BatchRow z = token ? batch_row(a.table, r + token) : begins;
    if (!page_row_ok(a.pool, s, z) || z.length == 0) return;
    const uint32_t pitch = s.vp + 4;
    constexpr uint32_t kAtOnce = 8, kStep = SHARED ? 4 : 1;
    float m = -INFINITY, n = -INFINITY;
    float2 sum = make_float2(0.0f, 0.0f), v[8];                      // dims 128 (d / 4) + 4 lane + d % 4
#pragma unroll
    for (uint32_t d = 0; d < 8; d++) v[d] = make_float2(0.0f, 0.0f);
    for (uint32_t k0 = SHARED ? warp : 0; k0 < count; k0 += kAtOnce * kStep) {
        float4 st[kAtOnce], x[kAtOnce][2];
#pragma unroll
        for (uint32_t e = 0; e < kAtOnce; e++) {
            const uint32_t k = k0 + e * kStep;
            st[e] = make_float4(-INFINITY, -INFINITY, 0.0f, 0.0f); x[e][0] = x[e][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (k >= count) continue;
            const float* const from = a.part + ((size_t)(2 * (w0 + k) + (k ? 0 : 1)) * queries + i) * pitch;
            st[e] = *reinterpret_cast<const float4*>(from);
            if (4 * lane < s.vp) x[e][0] = *reinterpret_cast<const float4*>(from + 4 + 4 * lane);
            if (128 + 4 * lane < s.vp) x[e][1] = *reinterpret_cast<const float4*>(from + 132 + 4 * lane);
        }
        float new_m = m, new_n = n, w[kAtOnce], parts[kAtOnce];
#pragma unroll
        for (uint32_t e = 0; e < kAtOnce; e++) { new_m = fmaxf(new_m, st[e].x); new_n = fmaxf(new_n, st[e].y); }
#pragma unroll
        for (uint32_t e = 0; e < kAtOnce; e++) { w[e] = pg_frame(st[e].x, new_m); parts[e] = st[e].z; }
        sum = pg_add(sum, pg_frame(m, new_m), pg_tree(w, parts));
        const float f = pg_frame(n, new_n);
        m = new_m; n = new_n;
#pragma unroll
        for (uint32_t e = 0; e < kAtOnce; e++) w[e] = pg_frame(st[e].y, n);
#pragma unroll
        for (uint32_t d = 0; d < 8; d++) {
            if (d >= 4 && s.vp <= 128) break;
#pragma unroll
            for (uint32_t e = 0; e < kAtOnce; e++) { const float4 y = x[e][d / 4]; parts[e] = d % 4 == 0 ? y.x : d % 4 == 1 ? y.y : d % 4 == 2 ? y.z : y.w; }
            v[d] = pg_add(v[d], f, pg_tree(w, parts));
        }
    }
    if constexpr (SHARED) {
        __shared__ float stats[4][3];
        __shared__ float4 parts[4][64];
        if (lane == 0) { stats[warp][0] = m; stats[warp][1] = n; stats[warp][2] = sum.x; }
        parts[warp][lane] = make_float4(v[0].x, v[1].x, v[2].x, v[3].x); parts[warp][32 + lane] = make_float4(v[4].x, v[5].x, v[6].x, v[7].x);
        __syncthreads();
        if (warp) return;
        m = fmaxf(fmaxf(stats[0][0], stats[1][0]), fmaxf(stats[2][0], stats[3][0])); n = fmaxf(fmaxf(stats[0][1], stats[1][1]), fmaxf(stats[2][1], stats[3][1]));
        float w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        auto four = [&](float x0, float x1, float x2, float x3) { return fmaf(w[0], x0, w[1] * x1) + fmaf(w[2], x2, w[3] * x3); };
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) w[k] = pg_frame(stats[k][0], m);
        sum.x = four(stats[0][2], stats[1][2], stats[2][2], stats[3][2]);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) w[k] = pg_frame(stats[k][1], n);
#pragma unroll
        for (uint32_t q = 0; q < 2; q++) {
            const float4 x0 = parts[0][32 * q + lane], x1 = parts[1][32 * q + lane], x2 = parts[2][32 * q + lane], x3 = parts[3][32 * q + lane];
            v[4 * q].x = four(x0.x, x1.x, x2.x, x3.x); v[4 * q + 1].x = four(x0.y, x1.y, x2.y, x3.y);
            v[4 * q + 2].x = four(x0.z, x1.z, x2.z, x3.z); v[4 * q + 3].x = four(x0.w, x1.w, x2.w, x3.w);
        }
    }
    const float2 f = pg_finish(a, g * a.rep + h, m, n, sum.x);
    float* const to = a.dst + (size_t)(r + token) * a.dst_rs + (g * a.rep + h) * s.dv;
#pragma unroll
    for (uint32_t e = 0; e < 8; e++) {
        const uint32_t d = 128 * (e / 4) + 4 * lane + e % 4;
        if (d < s.dv) to[d] = pg_scaled(v[e].x / f.y, f.x);
    }
}

// floats before the records: the plan
size_t pg_plan_elems(uint32_t B) { return (kPgPlan + 2 * ((size_t)B + 1) + 3) / 4 * 4; }
template <int KC, int VC, int NT, bool FULL, int W>
bool pg_launch_as(const PgArgs& a, cudaStream_t st) {
    const size_t smem = W * (kPgTile * (a.s.kp + a.s.vp) + 32 + sizeof(float) * pg_aside(NT, a.s.vp));
    constexpr size_t most = W * (kPgTile * (32 * KC + 16 * VC) + 32 + sizeof(float) * pg_aside(NT, 16 * VC));
    if (!zg_smem_limit<k_paged<KC, VC, NT, FULL, W>>(most)) return false;
    launch_pdl(k_paged<KC, VC, NT, FULL, W>, dim3(W == 1 ? pg_warps(KC, VC, NT) * zg_sm_count() : a.B * a.s.G * a.chunks), dim3(32 * W), smem, st, a);
    return true;
}
// FULL: sizes that fill the kernel's, whose loops and addresses are then known when it is compiled
template <int KC, int VC, int NT, int W>
bool pg_launch(const PgArgs& a, cudaStream_t st) {
    return a.s.kp == 32 * KC && a.s.vp == 16 * VC ? pg_launch_as<KC, VC, NT, true, W>(a, st) : pg_launch_as<KC, VC, NT, false, W>(a, st);
}
// Queries that a warp takes together: four, of one row, or, where the step has more rows than the page table slots, of a slot's rows that follow one another; eight where a key head
// has more than four and the caches are large, whose pages then come through L2 once for them (64 / 8 heads of 128, us, with four and with eight: 16 rows of up to 65536 tokens
// 397 / 293, 32 of up to 16384 193 / 160, 64 of up to 8192 192 / 163, 64 of up to 4096 102 / 111; 64 rows of 32 / 2 heads of up to 4096 51 / 68, 9 x 7 rows of 16 / 2 heads of up to 2111 29 / 45).
struct PgForm { bool narrow, wide, one; uint32_t queries, tokens; };      // one: one launch
constexpr uint64_t kPgLarge = 1u << 22;
// One launch, a CTA of eight warps for each sequence and key head, where the longest sequence has, or its window shows, up to 1024 tokens and the CTAs make two waves at most (an SM holds one: its registers); else equal shares
// and a second launch that joins them. One launch / two, us: 3 products of 64-dim heads, 64 tokens 8.3 / 10.3, 576 10.3 / 12.4, 2048 16.5 / 13.3; 128 dims, 32 products, 1024 tokens 14.4 / 16.9, 2048
// 18.6 / 18.5; 128 products, 64 tokens 8.3 / 16.5, 4096 30.8 / 28.0; 256 products, 64 tokens 14.4 / 16.5, 1024 23.0 / 23.9, 2048 32.8 / 28.8; 512 products (four waves), 64 tokens 26.7 / 16.5.
bool pg_one(uint64_t products, uint64_t seen) { return products <= 2ull * zg_sm_count() && seen <= 1024; }
PgForm pg_form(const ZgSeqOp& op, uint32_t slots, bool scratch) {
    PgForm f;
    const PageShape s = page_shape(op.n[2], op.n[3], op.n[4], op.n[7]);
    const uint32_t rep = op.n[1] / op.n[2];
    f.narrow = s.kp <= 64 && s.vp <= 64;
    f.wide = s.kp > 128 || s.vp > 128;
    const uint64_t capacity = (uint64_t)op.n[8] << s.shift, seen = op.n[9] ? std::min(capacity, (uint64_t)op.n[9] + kPgTile) : capacity;      // positions of a row at most
    f.queries = scratch && rep > 4 && !f.wide && (uint64_t)op.n[0] * op.n[2] * seen >= kPgLarge ? 8 : 4;
    f.one = !scratch || pg_one(op.n[0] * op.n[2] * ((rep + 3) / 4), seen);
    f.tokens = op.n[0] > slots ? std::max(1u, f.queries / rep) : 1;
    return f;
}

}  // namespace

bool zg_paged_attention_valid(const ZgSeqOp& s, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    const size_t B = s.n[0], H = s.n[1], G = s.n[2], dk = s.n[3], dv = s.n[4], qrs = s.n[5], drs = s.n[6], page = s.n[7], most = s.n[8];
    if (!B || B > 65535 || !page_shape_ok(G, dk, dv, page) || !H || H > 1024 || H % G || !most || most >= (1u << 25)) return fail("paged_attention: shape");
    if ((B > 1 && qrs < s.off[0] + H * dk) || !fits(1, s.off[0], (B - 1) * qrs + H * dk) || (B > 1 && drs < s.off[1] + H * dv) || !fits(0, s.off[1], (B - 1) * drs + H * dv)) return fail("paged_attention: rows");
    if (!fits(2, 0, zg_page_words(G, dk, dv, page)) || !fits(3, 0, most) || !fits(4, 0, ZG_BATCH_ROWS + 4 * B)) return fail("paged_attention: pages or tables");
    if (s.buf[5] != ZG_NO_BUF && (s.n[10] > ZG_W_BF16 || !have(5) || (s.n[10] == ZG_W_BF16 ? (s.off[2] + H + 1) / 2 : s.off[2] + H) > elems[s.buf[5]])) return fail("paged_attention: sinks");
    if (!(s.f[0] - s.f[0] == 0.0f) || !(s.f[1] >= 0.0f) || !(s.f[1] - s.f[1] == 0.0f)) return fail("paged_attention: scale or cap");
    for (int i = 1; i < 6; i++) if (s.buf[0] == s.buf[i]) return fail("paged_attention: in place");
    return true;
}
size_t zg_paged_attention_scratch_elems(const ZgSeqOp& s) {
    const uint32_t vp = page_shape(s.n[2], s.n[3], s.n[4], s.n[7]).vp;
    return pg_plan_elems(s.n[0]) + (size_t)zg_sm_count() * 128 * (vp + 4);      // (two records of four queries for up to 16 warps an SM, of eight for up to 8)
}
unsigned int zg_paged_attention_timeouts() { return tc_timeouts(); }
bool zg_launch_paged_attention(const ZgOp& op, float* const* bufs, const size_t* elems, float* scratch, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    PgArgs a;
    a.s = page_shape(s.n[2], s.n[3], s.n[4], s.n[7]);
    a.pool = page_pool(bufs[s.buf[2]], elems[s.buf[2]], bufs[s.buf[3]], elems[s.buf[3]], s.n[8], a.s);
    a.B = s.n[0]; a.H = s.n[1]; a.rep = a.H / s.n[2]; a.q_rs = s.n[5]; a.dst_rs = s.n[6]; a.window = s.n[9]; a.sink_bf16 = s.n[10] == ZG_W_BF16;
    a.dst = bufs[s.buf[0]] + s.off[1]; a.q = bufs[s.buf[1]] + s.off[0]; a.table = bufs[s.buf[4]];
    a.sink = s.buf[5] == ZG_NO_BUF ? nullptr : a.sink_bf16 ? (const void*)wptr<bf16>(bufs, s.buf[5], s.off[2]) : (const void*)wptr<float>(bufs, s.buf[5], s.off[2]);
    a.scale = s.f[0]; a.cap = s.f[1];
    const PgForm f = pg_form(s, a.pool.slots, scratch != nullptr);
    a.chunks = (a.rep + f.queries - 1) / f.queries;
    a.tokens = f.tokens;
    a.plan = reinterpret_cast<uint32_t*>(scratch);
    a.part = f.one ? nullptr : scratch + pg_plan_elems(a.B);
    bool ok;
    if (f.one) ok = f.narrow ? pg_launch<2, 4, 1, 8>(a, st) : f.wide ? pg_launch<8, 16, 1, 8>(a, st) : pg_launch<4, 8, 1, 8>(a, st);
    else if (f.narrow) ok = f.queries == 4 ? pg_launch<2, 4, 1, 1>(a, st) : pg_launch<2, 4, 2, 1>(a, st);
    else if (!f.wide) ok = f.queries == 4 ? pg_launch<4, 8, 1, 1>(a, st) : pg_launch<4, 8, 2, 1>(a, st);
    else ok = pg_launch<8, 16, 1, 1>(a, st);
    if (!ok) return false;
    ZG_SEQ_CHECK();
    if (!f.one) {
        // Four warps a query where few sequences and heads are shared out over all warps, so that each has a dozen records or more (32 / 8 heads of 128, us, four / one: one sequence of 4096
        // tokens 16.5 / 24.7, of 65536 48.9 / 79.3, 16 of 4096 28.5 / 30.8; 64 of 4096 74.9 / 65.4, 256 of 1500 128 / 103).
        const uint32_t products = a.s.G * a.chunks * f.queries;
        if ((uint64_t)a.B * a.s.G * a.chunks <= zg_sm_count()) launch_pdl(k_paged_join<true>, dim3(products, a.B), dim3(128), 0, st, a, f.queries);
        else launch_pdl(k_paged_join<false>, dim3((products + 3) / 4, a.B), dim3(128), 0, st, a, f.queries);
        ZG_SEQ_CHECK();
    }
    return true;
}
