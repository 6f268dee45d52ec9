// PAGED_ATTENTION (parameter pack in include/zgml_cuda.h): softmax attention of the rows of a step over the 8-bit pages of their sequences.
//
// Both products run on the tensor cores in whole numbers, whose sums are exact: codes of 8 bits, which need no conversion, times digits of 8 bits.  A query is six digits of base 256 (45 bits
// of its largest element), a weight four (32 bits of the largest contribution); the digits of four queries are 24 and 16 columns of the instructions, codes their rows.  Stored codes are offset
// by 128: sum (c + 128) d - 128 sum d is exact too, and a bit of each code of a value is turned over.  Scales are powers of two: a key's joins its scores, a value's its weights.  A weight is 2^(s + e - n), with the score s in powers of
// two, e the exponent of its value's scale and n a whole number that no s + e so far passes by more than 3, so that the largest contributions keep their bits whatever the pages' scales
// are; the sum of the softmax has a frame m of its own, and the quotient is put right by 2^(n - m).
#include "pages.cuh"
#include "exp2.cuh"
#include "split_tc.cuh"

#include <algorithm>

namespace {

struct PgArgs {
    PagePool pool; PageShape s;
    float* dst; const float* q; const float* table; const void* sink;
    uint32_t B, H, rep, q_rs, dst_rs, window, sink_bf16, tokens, chunks;      // tokens of a sequence a CTA takes together, chunks of a key head's query heads
    float scale, cap;
};
constexpr uint32_t kPgWarps = 4, kPgTile = 32, kPgShift = 29, kPgFlush = 512;      // (512 tiles of 32 products of two bytes: below 2^31)
constexpr float kPgSlack = 3.0f;                                     // weights reach 2^(29 + 3)
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
__device__ __forceinline__ float pg_remote(const float* p, uint32_t rank) {
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void pg_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// CTA (share of the positions; key head and chunk of its query heads; row that begins a group of rows of one sequence).  A warp takes every kPgWarps-th tile of 32 positions of
// the share through a buffer of its own, so that warps wait for nothing but their own copies: the next tile's keys come while this one's weights and outputs are computed, its
// values while the scores are.  4 NT queries a CTA, query 4 t + lane % 4 a lane.
template <int KC, int VC, int NT, bool FULL>
__global__ void __launch_bounds__(32 * kPgWarps, NT == 1 && KC <= 4 ? 3 : 1) k_paged(const __grid_constant__ PgArgs a) {
    pdl_enter();
    extern __shared__ float4 pg_mem[];
    __shared__ uint64_t bars[kPgWarps][2];                           // of a warp's keys and values
    __shared__ float stats[kPgWarps][4 * NT][3], joined[4 * NT][3], factor[4 * NT][2];      // m, n, sum
    const PageShape& s = a.s;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, row8 = lane / 4, j = lane % 4;
    const uint32_t r = blockIdx.z, g = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks, splits = gridDim.x, split = blockIdx.x;
    const BatchHead head = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    uint32_t group = 1;                                              // rows from r on that this CTA takes
    if (a.tokens > 1) {
        uint32_t back = 0;                                           // rows of the same slot directly before r
        for (bool more = true; more;) {
            const uint32_t i = back + lane;
            const bool same = i < r && batch_row(a.table, r - 1 - i).slot == w.slot;
            const uint32_t other = ~__ballot_sync(0xffffffffu, same);
            back += other ? __ffs(other) - 1 : 32;
            more = !other;
        }
        if (back % a.tokens) return;
        const bool same = lane > 0 && lane < a.tokens && r + lane < head.rows && batch_row(a.table, r + lane).slot == w.slot;
        group = min(a.tokens, (uint32_t)__ffs(~(__ballot_sync(0xffffffffu, same) | 1u)) - 1);
    }
    const uint32_t heads = min(a.rep, 4u * NT);                      // of a chunk
    // what the lane's queries see, and its column of the first product: two of the six digits of a query, and 128 times their sums
    uint32_t len[NT], low[NT], all_lo = 0xffffffffu, all_hi = 0;
    uint32_t qd[NT][KC][3][2];
    int offset[NT][3];
    float q_scale[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        len[t] = low[t] = 0;
        const uint32_t mine = 4 * t + j;
        if (mine / heads < group && chunk * heads + mine % heads < a.rep) {
            const BatchRow x = batch_row(a.table, r + mine / heads);
            if (page_row_ok(a.pool, s, x)) { len[t] = x.length; low[t] = a.window && len[t] > a.window ? len[t] - a.window : 0; }
        }
        if (len[t]) { all_lo = min(all_lo, low[t]); all_hi = max(all_hi, len[t]); }
        const uint32_t i = 4 * t + row8 / 2, token = i / heads, h = chunk * heads + i % heads;
        const bool on = token < group && h < a.rep;
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
    all_lo = __reduce_min_sync(0xffffffffu, all_lo);
    all_hi = __reduce_max_sync(0xffffffffu, all_hi);
    // this CTA's tiles
    const uint32_t first = all_hi ? all_lo / kPgTile : 0, tiles = all_hi ? (all_hi + kPgTile - 1) / kPgTile - first : 0;
    const uint32_t t0 = first + (uint32_t)((uint64_t)tiles * split / splits), t1 = first + (uint32_t)((uint64_t)tiles * (split + 1) / splits);
    const uint32_t kp = FULL ? 32 * KC : s.kp, vp = FULL ? 16 * VC : s.vp, kc = kp / 32, vc = vp / 16, k_bytes = kPgTile * kp;
    const uint32_t buffer_bytes = k_bytes + kPgTile * vp + 32, pitch = vp + 4;
    uint8_t* const buffer = reinterpret_cast<uint8_t*>(pg_mem) + warp * buffer_bytes;
    float* const rec = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(pg_mem) + kPgWarps * buffer_bytes);      // [warps][4 NT][pitch]
    const uint32_t pages = (all_hi + s.page - 1) >> s.shift;
    // the page of half `lane & 1` of a tile: its id, -1 for one that does not exist, -2 behind the last one that a row sees
    auto find = [&](uint32_t tile) {
        if (tile >= t1) return -2;
        const uint32_t n = (tile * kPgTile + 16 * (lane & 1)) >> s.shift;
        return n < pages ? page_id(a.pool, w.slot, n) : -2;
    };
    const size_t page_size = page_bytes(s);
    const uint8_t* const parts = a.pool.pages + (size_t)g * s.head;
    // Keys, with the scales, or values of a tile: a bulk copy for each half, by lanes 0 and 1.  What no page holds is left as it is, and gets scales alone.
    const uint32_t k_bar = smem_u32(&bars[warp][0]), v_bar = k_bar + 8, at = smem_u32(buffer), heads_at = at + k_bytes + kPgTile * vp;
    if (lane == 0) {
        mbar_init(k_bar, 2);
        mbar_init(v_bar, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
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
    // Frames: m of the lane's sum of weights, n of the products' weights.  They stay while no score passes them by much, which one vote of the warp tells.
    float m[NT], n[NT], sum[NT];
    int o[NT][VC][2][4];                                             // even and odd digits: two of each
    uint32_t all_in = 0xffffffffu, least = 0, since = 0;             // positions that every query sees; tiles since the sums were put away
    bool stored = false;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m[t] = n[t] = -INFINITY; sum[t] = 0.0f;
        if (len[t]) { all_in = min(all_in, len[t]); least = max(least, low[t]); }
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) o[t][c][k / 4][k % 4] = 0;
    }
    // The sums so far, times alpha, go to the warp's record, where a lane has places of its own.
    auto flush = [&](const float (&alpha)[NT]) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float* const to = rec + (size_t)(warp * 4 * NT + 4 * t + j) * pitch;
#pragma unroll
            for (int c = 0; c < VC; c++) {
                if (!FULL && c >= vc) break;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int (&x)[2][4] = o[t][c];
                    const float v = fmaf(fmaf(fmaf((float)x[1][2 * k + 1], 256.0f, (float)x[0][2 * k + 1]), 256.0f, (float)x[1][2 * k]), 256.0f, (float)x[0][2 * k]);
                    float* const at = to + 16 * c + 8 * k + row8;
                    *at = ((stored ? *at : 0.0f) + v) * alpha[t];
                }
#pragma unroll
                for (int k = 0; k < 8; k++) o[t][c][k / 4][k % 4] = 0;
            }
        }
        stored = true;
        since = 0;
    };
    all_in = __reduce_min_sync(0xffffffffu, all_in);
    least = __reduce_max_sync(0xffffffffu, least);
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    {
        const int32_t id = find(t0 + warp);
        if (t0 + warp < t1) { fetch(t0 + warp, id, false); fetch(t0 + warp, id, true); }
        __syncwarp();
    }
    int32_t id = find(t0 + warp + kPgWarps);
    bool gave_up = false;
    uint32_t k_phase = 0, v_phase = 0;
    for (uint32_t tile = t0 + warp; tile < t1; tile += kPgWarps) {
        const bool more = tile + kPgWarps < t1;
        if (!__all_sync(0xffffffffu, mbar_wait(k_bar, k_phase))) { gave_up = true; break; }
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
        if (more) { fetch(tile + kPgWarps, id, false); k_phase ^= 1; }
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
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float top0 = fmaxf(sc[t][0][0], sc[t][0][1]), top1 = fmaxf(sc[t][1][0], sc[t][1][1]);
            over = over || fmaxf(top0 + e[0], top1 + e[1]) > n[t] + kPgSlack || fmaxf(top0, top1) > m[t] + 64.0f;
        }
        if (__any_sync(0xffffffffu, over) || since == kPgFlush) {
            float alpha[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float top0 = fmaxf(sc[t][0][0], sc[t][0][1]), top1 = fmaxf(sc[t][1][0], sc[t][1][1]), new_m = fmaxf(m[t], ceilf(fmaxf(top0, top1)));
                float new_n = fmaxf(n[t], ceilf(fmaxf(top0 + e[0], top1 + e[1])));
#pragma unroll
                for (int k = 4; k < 32; k *= 2) new_n = fmaxf(new_n, __shfl_xor_sync(0xffffffffu, new_n, k));
                alpha[t] = new_n == n[t] ? 1.0f : pg_pow2(n[t] - new_n);
                sum[t] *= new_m == m[t] ? 1.0f : pg_pow2(m[t] - new_m);
                m[t] = new_m; n[t] = new_n;
            }
            if (stored || since) flush(alpha);
        }
        since++;
        uint32_t low_digits[NT][2], high_digits[NT][2];              // of each half's weights: digits 0 and 2, and 1 and 3, of four positions
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float fm = m[t] == -INFINITY ? 0.0f : m[t], fn = (float)kPgShift - (n[t] == -INFINITY ? 0.0f : n[t]);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t turned[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float x = sc[t][u][k], y = x == -INFINITY ? 0.0f : sa_ex2(x + (fn + e[u]));
                    sum[t] += sa_ex2(x - fm) + (y - y);              // (a scale that is not a number is one of the sum's too)
                    const uint32_t w = __float2uint_rn(y);
                    // a lane's weight is two columns of 16 bits, a position a row; turned around they are rows of positions
                    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(turned[k]) : "r"(w));
                }
                low_digits[t][u] = __byte_perm(turned[0], turned[1], 0x6420);
                high_digits[t][u] = __byte_perm(turned[0], turned[1], 0x7531);
            }
        }
        __syncwarp();
        if (!__all_sync(0xffffffffu, mbar_wait(v_bar, v_phase))) { gave_up = true; break; }
#pragma unroll
        for (int c = 0; c < VC; c++) {
            if (!FULL && c >= vc) break;
            const uint2 x = *reinterpret_cast<const uint2*>(mine + k_bytes + c * 256), y = *reinterpret_cast<const uint2*>(mine + k_bytes + (vc + c) * 256);
            const uint32_t f[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, y.x ^ 0x80808080u, y.y ^ 0x80808080u};
#pragma unroll
            for (int t = 0; t < NT; t++) { pg_outputs(o[t][c][0], f, low_digits[t][0], low_digits[t][1]); pg_outputs(o[t][c][1], f, high_digits[t][0], high_digits[t][1]); }
        }
        __syncwarp();
        if (more) { fetch(tile + kPgWarps, id, true); v_phase ^= 1; id = find(tile + 2 * kPgWarps); }
        __syncwarp();
    }
    if (gave_up) {                                                   // what is under way lands before the memory is used for other things; outputs are not numbers
        mbar_wait(k_bar, k_phase);
        mbar_wait(v_bar, v_phase);
        if (lane == 0) count_timeout();
#pragma unroll
        for (int t = 0; t < NT; t++) sum[t] = kBatchNaN;
    }
    // the warps' records join in shared memory, then those of the cluster's CTAs
    {
        float one[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) one[t] = 1.0f;
        flush(one);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        float top = m[t];
#pragma unroll
        for (int k = 4; k < 32; k *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        sum[t] *= m[t] == top ? 1.0f : pg_pow2(m[t] - top);
#pragma unroll
        for (int k = 4; k < 32; k *= 2) sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], k);
        if (row8 == 0) { stats[warp][4 * t + j][0] = top; stats[warp][4 * t + j][1] = n[t]; stats[warp][4 * t + j][2] = sum[t]; }
    }
    __syncthreads();
    auto frame = [](float from, float to) { return from == to ? 1.0f : pg_pow2(from - to); };      // (also where both are infinite)
    float* const mine = reinterpret_cast<float*>(pg_mem);             // [4 NT][pitch], where tiles were
    const uint32_t queries = group * heads;
    for (uint32_t x = threadIdx.x; x < queries * vp; x += 32 * kPgWarps) {
        const uint32_t i = x / vp, d = x - i * vp;
        float top_m = -INFINITY, top_n = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < kPgWarps; k++) { top_m = fmaxf(top_m, stats[k][i][0]); top_n = fmaxf(top_n, stats[k][i][1]); }
#pragma unroll
        for (uint32_t k = 0; k < kPgWarps; k++) {
            l = fmaf(stats[k][i][2], frame(stats[k][i][0], top_m), l);
            v = fmaf(rec[(k * 4 * NT + i) * pitch + d], frame(stats[k][i][1], top_n), v);
        }
        mine[i * pitch + d] = v;
        if (d == 0) { joined[i][0] = top_m; joined[i][1] = top_n; joined[i][2] = l; }
    }
    if (splits > 1) pg_cluster_sync(); else __syncthreads();
    if (threadIdx.x < queries) {                                     // a query's frame over all CTAs, and what its outputs are multiplied by
        const uint32_t i = threadIdx.x, h = chunk * heads + i % heads;
        float top_m = -INFINITY, top_n = -INFINITY, l = 0.0f;
        for (uint32_t k = 0; k < splits; k++) { top_m = fmaxf(top_m, pg_remote(&joined[i][0], k)); top_n = fmaxf(top_n, pg_remote(&joined[i][1], k)); }
        for (uint32_t k = 0; k < splits; k++) l = fmaf(pg_remote(&joined[i][2], k), frame(pg_remote(&joined[i][0], k), top_m), l);
        float back = top_n - top_m - (float)kPgShift;
        if (a.sink && h < a.rep) {
            const float sink = pg_sink(a, g * a.rep + h) * kLog2e;
            const float to = fmaxf(top_m, ceilf(sink));              // (a sink far above the scores takes the frame with it)
            l = l * frame(top_m, to) + (to == -INFINITY ? 0.0f : sa_ex2(sink - to));
            back += top_m - to;
        }
        factor[i][0] = back; factor[i][1] = l;
    }
    __syncthreads();
    const uint32_t share = (s.dv + splits - 1) / splits, d0 = split * share, d1 = min(d0 + share, s.dv);
    for (uint32_t x = threadIdx.x; d0 < d1 && x < queries * (d1 - d0); x += 32 * kPgWarps) {
        const uint32_t i = x / (d1 - d0), d = d0 + x - i * (d1 - d0), h = chunk * heads + i % heads, row = r + i / heads;
        if (h >= a.rep) continue;
        float top_n = -INFINITY, v = 0.0f;
        for (uint32_t k = 0; k < splits; k++) top_n = fmaxf(top_n, pg_remote(&joined[i][1], k));
        for (uint32_t k = 0; k < splits; k++) v = fmaf(pg_remote(mine + i * pitch + d, k), frame(pg_remote(&joined[i][1], k), top_n), v);
        const BatchRow z = batch_row(a.table, row);
        const float back = factor[i][0], half = truncf(back * 0.5f);      // (in two steps: the scales of the values may lie anywhere)
        float out = v / factor[i][1] * exp2f(half) * exp2f(back - half);
        if (z.length == 0) out = 0.0f;
        if (!page_row_ok(a.pool, s, z)) out = kBatchNaN;
        a.dst[(size_t)row * a.dst_rs + (g * a.rep + h) * s.dv + d] = out;
    }
    if (splits > 1) pg_cluster_sync();                               // no CTA leaves while its record is read
}

template <int KC, int VC, int NT, bool FULL>
bool pg_launch_as(const PgArgs& a, uint32_t splits, cudaStream_t st) {
    const size_t buffers = (size_t)kPgWarps * (kPgTile * (a.s.kp + a.s.vp) + 32), records = sizeof(float) * kPgWarps * 4 * NT * (a.s.vp + 4);
    constexpr size_t most = (size_t)kPgWarps * (kPgTile * (32 * KC + 16 * VC) + 32) + sizeof(float) * kPgWarps * 4 * NT * (16 * VC + 4);
    if (!zg_smem_limit<k_paged<KC, VC, NT, FULL>>(most)) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.s.G * a.chunks, a.B); cfg.blockDim = dim3(32 * kPgWarps); cfg.dynamicSmemBytes = buffers + records; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_zg_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_paged<KC, VC, NT, FULL>, a);
    return true;
}
// FULL: sizes that fill the kernel's, whose loops and addresses are then known when it is compiled
template <int KC, int VC, int NT>
bool pg_launch(const PgArgs& a, uint32_t splits, cudaStream_t st) {
    return a.s.kp == 32 * KC && a.s.vp == 16 * VC ? pg_launch_as<KC, VC, NT, true>(a, splits, st) : pg_launch_as<KC, VC, NT, false>(a, splits, st);
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
size_t zg_paged_attention_scratch_elems(const ZgSeqOp&) { return 0; }
unsigned int zg_paged_attention_timeouts() { return tc_timeouts(); }
bool zg_launch_paged_attention(const ZgOp& op, float* const* bufs, const size_t* elems, float*, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    PgArgs a;
    a.s = page_shape(s.n[2], s.n[3], s.n[4], s.n[7]);
    a.pool = page_pool(bufs[s.buf[2]], elems[s.buf[2]], bufs[s.buf[3]], elems[s.buf[3]], s.n[8], a.s);
    a.B = s.n[0]; a.H = s.n[1]; a.rep = a.H / s.n[2]; a.q_rs = s.n[5]; a.dst_rs = s.n[6]; a.window = s.n[9]; a.sink_bf16 = s.n[10] == ZG_W_BF16;
    a.dst = bufs[s.buf[0]] + s.off[1]; a.q = bufs[s.buf[1]] + s.off[0]; a.table = bufs[s.buf[4]];
    a.sink = s.buf[5] == ZG_NO_BUF ? nullptr : a.sink_bf16 ? (const void*)wptr<bf16>(bufs, s.buf[5], s.off[2]) : (const void*)wptr<float>(bufs, s.buf[5], s.off[2]);
    a.scale = s.f[0]; a.cap = s.f[1];
    // Queries that a CTA takes together: of one row, or, where the step has more rows than the page table slots, of the rows that a slot has then.
    const bool narrow = a.s.kp <= 64 && a.s.vp <= 64, wide = a.s.kp > 128 || a.s.vp > 128;
    const uint64_t together = (uint64_t)a.rep * std::max<uint32_t>(1, a.B / std::max(1u, a.pool.slots));
    const uint32_t queries = together <= 4 || wide ? 4 : 8;
    a.chunks = (a.rep + queries - 1) / queries;
    a.tokens = std::max(1u, queries / a.rep);
    const uint32_t ctas = a.B * a.s.G * a.chunks, most = std::max<uint32_t>(1, (uint32_t)std::min<uint64_t>(8, ((uint64_t)s.n[8] << a.s.shift) / 256));
    uint32_t splits = 1;
    while (splits < most && ctas * splits < 4 * zg_sm_count()) splits *= 2;
    if (splits > most) splits = most;
    bool ok;
    if (narrow) ok = queries == 4 ? pg_launch<2, 4, 1>(a, splits, st) : pg_launch<2, 4, 2>(a, splits, st);
    else if (!wide) ok = queries == 4 ? pg_launch<4, 8, 1>(a, splits, st) : pg_launch<4, 8, 2>(a, splits, st);
    else ok = pg_launch<8, 16, 1>(a, splits, st);
    if (!ok) return false;
    ZG_SEQ_CHECK();
    return true;
}
