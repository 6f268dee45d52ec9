// SHARED_ATTENTION (parameter pack in include/zgml_cuda.h): every row of a batch attends over the keys of one prefix that all rows share and over the
// keys of its own sequence, with one softmax over both.
//
// Softmax attention over a set of keys that falls into shares needs a record (m, l, o) per share: the largest score, the sum of exp(s - m) and the sum of
// exp(s - m) v.  Records of any shares merge into the whole: m = max m_i, l = sum l_i e^(m_i - m), o = sum o_i e^(m_i - m) / l.
#include "batch_table.cuh"
#include "split_tc.cuh"

#include <algorithm>

namespace {

struct SaArgs {
    float* dst; const float* q; const float* kc; const float* vc; const float* kp; const float* vp; const float* table;
    const void* sink;
    float* part;                     // records [B, H, shares + splits, 4 + dv]: m, l, -, -, o; null: a row's keys are one share
    uint32_t B, H, G, rep, dk, dv, q_rs, kw, vw, R, pkw, pvw, Rp, dst_rs, slots, pslots, sink_bf16;
    uint32_t shares, splits;         // shares of the prefix, which k_shared_prefix walks (0: k_shared_rows walks all keys), and of what is left to k_shared_rows
    float scale, cap;
};
// What a row sees: `prefix` keys of the shared prefix, then `own` of its slot.
struct SaKeys { const float* kp; const float* vp; const float* kc; const float* vc; uint32_t prefix, own; bool live, bad; };
__device__ __forceinline__ SaKeys sa_keys(const SaArgs& a, uint32_t r, uint32_t g) {
    SaKeys k;
    const BatchHead h = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    k.live = r < h.rows && w.slot >= 0;
    const bool no_prefix = h.prefix == 0;
    k.bad = (uint32_t)w.slot >= a.slots || (uint32_t)w.length > a.R || (!no_prefix && ((uint32_t)h.prefix > a.Rp || (uint32_t)h.prefix_slot >= a.pslots));
    const bool ok = k.live && !k.bad;
    k.prefix = ok ? (uint32_t)h.prefix : 0u;
    k.own = ok ? (uint32_t)w.length : 0u;
    const size_t p0 = ok && !no_prefix ? (size_t)h.prefix_slot * a.Rp : 0, c0 = ok ? (size_t)w.slot * a.R : 0;
    k.kp = a.kp + p0 * a.pkw + g * a.dk; k.vp = a.vp + p0 * a.pvw + g * a.dv;
    k.kc = a.kc + c0 * a.kw + g * a.dk; k.vc = a.vc + c0 * a.vw + g * a.dv;
    return k;
}
__device__ __forceinline__ float sa_sink(const SaArgs& a, uint32_t h) {
    return a.sink_bf16 ? __bfloat162float(reinterpret_cast<const bf16*>(a.sink)[h]) : reinterpret_cast<const float*>(a.sink)[h];
}
// record of share i of a row's head
__device__ __forceinline__ float* sa_record(const SaArgs& a, uint32_t r, uint32_t h, uint32_t i) { return a.part + ((size_t)(r * a.H + h) * (a.shares + a.splits) + i) * (4 + a.dv); }
// keys of a share when n keys fall into at most `shares` of them
__device__ __forceinline__ uint32_t sa_share(uint32_t n, uint32_t shares, uint32_t least) { return max(least, ((n + shares - 1) / shares + 15) & ~15u); }
constexpr uint32_t kSaShare = 64;    // the least
// weight of a share whose largest score is m, in the frame of the largest of all; a share that saw nothing weighs nothing
__device__ __forceinline__ float sa_weight(float m, float top) { return m == -INFINITY ? 0.0f : expf(m - top); }

template <bool VEC>
__device__ __forceinline__ float4 sa_load(const float* p, uint32_t d, uint32_t n, bool on) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!on) return v;
    if constexpr (VEC) { if (d < n) v = *reinterpret_cast<const float4*>(p + d); }
    else {
        if (d < n) v.x = p[d];
        if (d + 1 < n) v.y = p[d + 1];
        if (d + 2 < n) v.z = p[d + 2];
        if (d + 3 < n) v.w = p[d + 3];
    }
    return v;
}

// CTA (row, key head, chunk of RQ of its query heads; share of the keys).  LK lanes share a key: each holds NV float4 of it, of the queries and of the outputs; a warp
// takes 32 / LK keys at a time, the warps' keys are interleaved.  Every lane group keeps its own running maximum and sum, merged once at the end.
constexpr uint32_t kSaWarps = 4;
template <int RQ, int NV, bool VEC>
__global__ void __launch_bounds__(32 * kSaWarps) k_shared_rows(SaArgs a, uint32_t chunks, uint32_t LK) {
    pdl_enter();
    extern __shared__ float sh[];                                   // [warps][RQ][2 + dv]
    const uint32_t c = blockIdx.x % chunks, g = blockIdx.x / chunks % a.G, r = blockIdx.x / chunks / a.G, split = blockIdx.y;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LK - 1), group = lane / LK, per_warp = 32 / LK;
    const uint32_t h0 = g * a.rep + c * RQ, nq = min((uint32_t)RQ, a.rep - c * RQ);
    const SaKeys k = sa_keys(a, r, g);
    if (!k.live) return;
    const uint32_t first = a.shares ? k.prefix : 0u, n = k.prefix + k.own, share = sa_share(n - first, a.splits, kSaShare), k0 = first + split * share, k1 = min(n, k0 + share);
    if (split && k0 >= n) return;                                   // (share 0 leaves a record however few the keys are)
    float4 q[RQ][NV], o[RQ][NV];
    float m[RQ], l[RQ];
#pragma unroll
    for (int i = 0; i < RQ; i++) {
        m[i] = -INFINITY; l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            q[i][j] = sa_load<VEC>(a.q + (size_t)r * a.q_rs + (size_t)(h0 + i) * a.dk, 4 * (sub + LK * j), a.dk, i < (int)nq);
            o[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    for (uint32_t base = k0 + warp * per_warp; base < k1; base += kSaWarps * per_warp) {
        const uint32_t u = base + group;
        const bool on = u < k1, own = u >= k.prefix;
        const float* kr = own ? k.kc + (size_t)(u - k.prefix) * a.kw : k.kp + (size_t)u * a.pkw;
        const float* vr = own ? k.vc + (size_t)(u - k.prefix) * a.vw : k.vp + (size_t)u * a.pvw;
        float4 x[NV], v[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            x[j] = sa_load<VEC>(kr, 4 * (sub + LK * j), a.dk, on);
            v[j] = sa_load<VEC>(vr, 4 * (sub + LK * j), a.dv, on);
        }
        float s[RQ];
#pragma unroll
        for (int i = 0; i < RQ; i++) {
            s[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; j++) s[i] = fmaf(q[i][j].x, x[j].x, fmaf(q[i][j].y, x[j].y, fmaf(q[i][j].z, x[j].z, fmaf(q[i][j].w, x[j].w, s[i]))));
        }
        for (uint32_t w = LK >> 1; w > 0; w >>= 1)
#pragma unroll
            for (int i = 0; i < RQ; i++) s[i] += __shfl_xor_sync(0xffffffffu, s[i], w);
#pragma unroll
        for (int i = 0; i < RQ; i++) {
            s[i] *= a.scale;
            if (a.cap > 0.0f) s[i] = a.cap * tanhf(s[i] / a.cap);
            if (!on) s[i] = -INFINITY;
            if (s[i] > m[i]) {
                const float f = sa_weight(m[i], s[i]);
                m[i] = s[i];
                l[i] *= f;
#pragma unroll
                for (int j = 0; j < NV; j++) { o[i][j].x *= f; o[i][j].y *= f; o[i][j].z *= f; o[i][j].w *= f; }
            }
            const float p = s[i] == -INFINITY ? 0.0f : expf(s[i] - m[i]);
            l[i] += p;
#pragma unroll
            for (int j = 0; j < NV; j++) { o[i][j].x = fmaf(p, v[j].x, o[i][j].x); o[i][j].y = fmaf(p, v[j].y, o[i][j].y); o[i][j].z = fmaf(p, v[j].z, o[i][j].z); o[i][j].w = fmaf(p, v[j].w, o[i][j].w); }
        }
    }
    // the lane groups of a warp, then the warps
    const uint32_t rec = 2 + a.dv;
#pragma unroll
    for (int i = 0; i < RQ; i++) {
        float top = m[i];
        for (uint32_t w = LK; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float f = sa_weight(m[i], top);
        l[i] *= f;
        for (uint32_t w = LK; w < 32; w <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float4 v = make_float4(o[i][j].x * f, o[i][j].y * f, o[i][j].z * f, o[i][j].w * f);
            for (uint32_t w = LK; w < 32; w <<= 1) {
                v.x += __shfl_xor_sync(0xffffffffu, v.x, w); v.y += __shfl_xor_sync(0xffffffffu, v.y, w);
                v.z += __shfl_xor_sync(0xffffffffu, v.z, w); v.w += __shfl_xor_sync(0xffffffffu, v.w, w);
            }
            const uint32_t d = 4 * (sub + LK * j);
            float* out = sh + (warp * RQ + i) * rec + 2 + d;
            if (group == 0) {
                if (d < a.dv) out[0] = v.x;
                if (d + 1 < a.dv) out[1] = v.y;
                if (d + 2 < a.dv) out[2] = v.z;
                if (d + 3 < a.dv) out[3] = v.w;
            }
        }
        if (lane == 0) { sh[(warp * RQ + i) * rec] = top; sh[(warp * RQ + i) * rec + 1] = l[i]; }
    }
    __syncthreads();
    for (uint32_t i = 0; i < nq; i++) {
        float top = -INFINITY, sum = 0.0f, f[kSaWarps];
#pragma unroll
        for (uint32_t w = 0; w < kSaWarps; w++) top = fmaxf(top, sh[(w * RQ + i) * rec]);
#pragma unroll
        for (uint32_t w = 0; w < kSaWarps; w++) { f[w] = sa_weight(sh[(w * RQ + i) * rec], top); sum = fmaf(sh[(w * RQ + i) * rec + 1], f[w], sum); }
        const uint32_t h = h0 + i;
        float* out;
        float inv = 1.0f;
        if (a.shares + a.splits > 1) {
            float* mine = sa_record(a, r, h, a.shares + split);
            if (threadIdx.x == 0) { mine[0] = top; mine[1] = sum; }
            out = mine + 4;
        } else {
            out = a.dst + (size_t)r * a.dst_rs + (size_t)h * a.dv;
            if (a.sink && top != -INFINITY) sum += expf(sa_sink(a, h) - top);
            inv = k.bad ? kBatchNaN : top == -INFINITY ? 0.0f : 1.0f / sum;          // nothing seen: zeros
        }
        for (uint32_t d = threadIdx.x; d < a.dv; d += 32 * kSaWarps) {
            float v = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kSaWarps; w++) v = fmaf(sh[(w * RQ + i) * rec + 2 + d], f[w], v);
            out[d] = v * inv;
        }
    }
}
// CTA (row, head): the records of its shares become the result
__global__ void __launch_bounds__(128) k_shared_merge(SaArgs a) {
    pdl_enter();
    const uint32_t h = blockIdx.x % a.H, r = blockIdx.x / a.H;
    const SaKeys k = sa_keys(a, r, 0);
    if (!k.live) return;
    const uint32_t of_prefix = a.shares ? k.prefix : 0u, left = k.prefix + k.own - of_prefix, per = sa_share(of_prefix, max(1u, a.shares), kSaShare), per_left = sa_share(left, a.splits, kSaShare);
    const uint32_t n0 = (of_prefix + per - 1) / per, n = n0 + max(1u, (left + per_left - 1) / per_left);
    const float* rec = sa_record(a, r, h, 0);
    auto at = [&](uint32_t s) { return rec + (size_t)(s < n0 ? s : a.shares + s - n0) * (4 + a.dv); };
    float top = -INFINITY;
    for (uint32_t s = 0; s < n; s++) top = fmaxf(top, at(s)[0]);
    float sum = 0.0f;
    for (uint32_t s = 0; s < n; s++) sum = fmaf(at(s)[1], sa_weight(at(s)[0], top), sum);
    if (a.sink && top != -INFINITY) sum += expf(sa_sink(a, h) - top);
    const float inv = k.bad ? kBatchNaN : top == -INFINITY ? 0.0f : 1.0f / sum;
    float* out = a.dst + (size_t)r * a.dst_rs + (size_t)h * a.dv;
    for (uint32_t d = threadIdx.x; d < a.dv; d += 128) {
        float v = 0.0f;
        for (uint32_t s = 0; s < n; s++) v = fmaf(at(s)[4 + d], sa_weight(at(s)[0], top), v);
        out[d] = v * inv;
    }
}

// ── the prefix on the tensor cores ───────────────────────────────────────────────────────────────────────────────────
// All query rows of a key head meet the same keys of the prefix, so its part of the attention is two matrix products.  CTA (key head, share of the prefix, tile of 128 query
// rows): 64 keys and values at a time are read from the cache once, split into half-precision pairs on their way to shared memory (a scale per key, one per tile of
// values; split_tc.cuh) and multiplied by tcgen05.mma, three MMAs a product.  Warps 0 - 15 do everything but issue: they load tile t + 2 while they split tile
// t + 1 and take the softmax of tile t; four threads share a query row, each with a quarter of the keys and of the output columns.  Warp 16 issues.
//   TMEM: scores of two tiles, which become the probabilities in place (A operand), outputs of two tiles, the queries' pairs (A operand).
//   What pairs cannot hold - something not finite, magnitudes too far apart for one scale - is found as it is split; the CTA then walks its share again in plain f32.
// Every wait is bounded; a CTA whose wait ran out counts it and makes NaN of its rows.
constexpr uint32_t kSpWorkers = 512, kSpThreads = kSpWorkers + 32, kSpStages = 3, kSpKeys = 64;
template <int NC, int DV> struct SpLayout {
    static constexpr uint32_t k_part = NC * kSpKeys * 128, v_part = DV * 128, stage = 2 * (k_part + v_part);      // bytes; a part: hi or lo
    static constexpr uint32_t share = kSpStages * stage, kf = share + 2 * 4 * 128 * 4, vf = kf + kSpStages * kSpKeys * 4, red = vf + 16, bars = red + 2 * 16 * 4, size = bars + 128 + 1024;
};
__device__ __forceinline__ float sp_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// Not zero, but below 2^-18 of the magnitude its scale is made for: a pair keeps fewer than 22 bits of it.  More than a few of them in a patch of 512 values (normally
// distributed ones have 0.006) mean that something is small as a whole.
__device__ __forceinline__ uint32_t sp_small(float x) { const float a = fabsf(x); return a < 0.0625f && a > 0.0f ? 1u : 0u; }
constexpr uint32_t kSpSmall = 4;
struct SpCta { uint32_t g, split, tile, k0, k1; const float* kp; const float* vp; };
// query row i of the CTA's tile
struct SpRow { bool on; uint32_t r, h; };
__device__ __forceinline__ SpRow sp_row(const SaArgs& a, const SpCta& c, const BatchHead& head, uint32_t i) {
    SpRow w;
    const uint32_t at = c.tile * 128 + i;
    w.r = at / a.rep; w.h = c.g * a.rep + at % a.rep;
    w.on = w.r < head.rows;
    if (w.on) { const BatchRow b = batch_row(a.table, w.r); w.on = (uint32_t)b.slot < a.slots && (uint32_t)b.length <= a.R; }
    if (!w.on) w.r = 0;
    return w;
}
// The CTA's share in plain f32: a warp takes four of its eight rows at a time, a lane four dims of a key and four columns of a value.
__device__ __noinline__ void sp_plain(const SaArgs& a, const SpCta& c, const BatchHead& head) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t i0 = warp * 8; i0 < warp * 8 + 8; i0 += 4) {
        float4 q[4], o[4];
        float m[4], l[4];
        SpRow w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w[i] = sp_row(a, c, head, i0 + i);
            q[i] = sa_load<true>(a.q + (size_t)w[i].r * a.q_rs + (size_t)w[i].h * a.dk, 4 * lane, a.dk, w[i].on);
            o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); m[i] = -INFINITY; l[i] = 0.0f;
        }
        for (uint32_t u = c.k0; u < c.k1; u++) {
            const float4 x = sa_load<true>(c.kp + (size_t)u * a.pkw, 4 * lane, a.dk, true), v = sa_load<true>(c.vp + (size_t)u * a.pvw, 4 * lane, a.dv, true);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float s = warp_sum(fmaf(q[i].x, x.x, fmaf(q[i].y, x.y, fmaf(q[i].z, x.z, q[i].w * x.w)))) * a.scale;
                if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
                const float top = fmaxf(m[i], s), f = sa_weight(m[i], top), p = s == -INFINITY ? 0.0f : expf(s - top);
                m[i] = top; l[i] = fmaf(l[i], f, p);
                o[i].x = fmaf(o[i].x, f, p * v.x); o[i].y = fmaf(o[i].y, f, p * v.y); o[i].z = fmaf(o[i].z, f, p * v.z); o[i].w = fmaf(o[i].w, f, p * v.w);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (!w[i].on) continue;
            float* rec = sa_record(a, w[i].r, w[i].h, c.split);
            if (lane == 0) { rec[0] = m[i]; rec[1] = l[i]; }
            if (4 * lane < a.dv) { rec[4 + 4 * lane] = o[i].x; rec[5 + 4 * lane] = o[i].y; rec[6 + 4 * lane] = o[i].z; rec[7 + 4 * lane] = o[i].w; }
        }
    }
}
template <int NC, int DV>
__global__ void __launch_bounds__(kSpThreads, 1) k_shared_prefix(const SaArgs a, const uint32_t row_tiles) {
    typedef SpLayout<NC, DV> L;
    constexpr uint32_t kS = 0, kO = 2 * kSpKeys, kQ = kO + 2 * DV;         // TMEM columns
    static_assert(kQ + 64 * NC <= 512, "TMEM columns");
    extern __shared__ uint8_t dsm_raw[];
    const uint32_t base = (smem_u32(dsm_raw) + 1023u) & ~1023u;
    uint8_t* const mem = dsm_raw + (base - smem_u32(dsm_raw));
    const uint32_t full = base + L::bars, empty = full + 8 * kSpStages, s_full = empty + 8 * kSpStages, o_full = s_full + 16, p_full = o_full + 16, q_full = p_full + 8, tmem_slot = q_full + 8;
    uint32_t* const trouble = reinterpret_cast<uint32_t*>(mem + (tmem_slot + 4 - base));          // 1: something that pairs cannot hold, 2: a wait that ran out
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kSpStages; i++) { mbar_init(full + 8 * i, 16); mbar_init(empty + 8 * i, 1); }
        for (uint32_t i = 0; i < 2; i++) { mbar_init(s_full + 8 * i, 1); mbar_init(o_full + 8 * i, 1); }
        mbar_init(p_full, 16); mbar_init(q_full, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *trouble = 0;
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const BatchHead head = batch_head(a.table, a.B);
    SpCta c;
    c.tile = blockIdx.x % row_tiles; c.split = blockIdx.x / row_tiles % a.shares; c.g = blockIdx.x / row_tiles / a.shares;      // CTAs of the same keys are neighbours
    const bool sound = head.prefix > 0 && (uint32_t)head.prefix <= a.Rp && (uint32_t)head.prefix_slot < a.pslots && c.tile * 128 < head.rows * a.rep;
    const uint32_t P = sound ? (uint32_t)head.prefix : 0u, per = sa_share(P, a.shares, kSaShare);
    c.k0 = min(P, c.split * per); c.k1 = min(P, c.k0 + per);
    const size_t p0 = sound ? (size_t)head.prefix_slot * a.Rp : 0;
    c.kp = a.kp + p0 * a.pkw + c.g * a.dk; c.vp = a.vp + p0 * a.pvw + c.g * a.dv;
    const uint32_t n_tiles = (c.k1 - c.k0 + kSpKeys - 1) / kSpKeys;
    fence_before();
    __syncthreads();
    fence_after();

    if (n_tiles && warp == 16) {
        constexpr uint32_t idesc_s = (1u << 4) | ((kSpKeys >> 3) << 17) | ((128u >> 4) << 24), idesc_o = (1u << 4) | ((DV >> 3) << 17) | ((128u >> 4) << 24);      // f16 x f16 -> f32
        const bool leader = elect_one();
        bool ok = mbar_wait(q_full, 0);
        fence_after();
        // three products, the small ones first: hi lo, lo hi, hi hi.  B parts of `part` bytes at b (hi, then lo), chunks of 64 along the summed dimension 8 KB apart
        auto scores = [&](uint32_t t) {
            if (ok) ok = mbar_wait(full + 8 * (t % kSpStages), (t / kSpStages) & 1);
            fence_after();
            if (!(leader && ok)) return;
            const uint32_t d = kS + (t & 1) * kSpKeys, b = desc_low(base + (t % kSpStages) * L::stage);
#pragma unroll
            for (uint32_t x = 0; x < 3; x++) {
                const uint32_t qa = kQ + (x == 1 ? 32 * NC : 0), kb = b + (x == 0 ? L::k_part >> 4 : 0);
#pragma unroll
                for (uint32_t k = 0; k < 4 * NC; k++) {
                    if (x == 0 && k == 0) mma_ts<false>(d, qa, kb, idesc_s);
                    else mma_ts<true>(d, qa + 8 * k, kb + (k / 4) * (kSpKeys * 128 >> 4) + 2 * (k % 4), idesc_s);
                }
            }
            mma_commit(s_full + 8 * (t & 1));
        };
        // probabilities of 16 keys lie in 16 columns: 8 with their hi pairs, 8 with their lo pairs
        auto values = [&](uint32_t t) {
            if (ok) ok = mbar_wait(p_full, t & 1);
            fence_after();
            if (!(leader && ok)) return;
            const uint32_t d = kO + (t & 1) * DV, pa = kS + (t & 1) * kSpKeys, b = desc_low(base + (t % kSpStages) * L::stage + 2 * L::k_part);
#pragma unroll
            for (uint32_t x = 0; x < 3; x++) {
#pragma unroll
                for (uint32_t k = 0; k < kSpKeys / 16; k++) {
                    if (x == 0 && k == 0) mma_ts<false>(d, pa, b + (L::v_part >> 4), idesc_o);
                    else mma_ts<true>(d, pa + 16 * k + (x == 1 ? 8 : 0), b + (x == 0 ? L::v_part >> 4 : 0) + 2 * k, idesc_o);
                }
            }
            mma_commit(o_full + 8 * (t & 1));
            mma_commit(empty + 8 * (t % kSpStages));
        };
        for (uint32_t t = 0; t < n_tiles && ok; t++) {
            scores(t);
            if (t) values(t - 1);
        }
        if (ok) values(n_tiles - 1);
        if (!ok && lane == 0) { count_timeout(); atomicOr(trouble, 2u); }
        __syncwarp();
    } else if (n_tiles) {
        constexpr int OW = DV / 4, KT = DV == 128 ? 8 : 4;               // output columns and value rows of a thread
        const uint32_t part = warp >> 2, row = (warp & 3) * 32 + lane, lanes = ((warp & 3) * 32) << 16, half = lane >> 4, hl = lane & 15;
        const uint32_t v_key = DV == 128 ? 16 * (warp & 3) + 8 * half : 8 * (warp & 7) + 4 * half, v_col = 32 * (DV == 128 ? warp >> 2 : warp >> 3) + 2 * hl;
        float* const share = reinterpret_cast<float*>(mem + L::share);
        float* const kf = reinterpret_cast<float*>(mem + L::kf);
        float* const vf = reinterpret_cast<float*>(mem + L::vf);
        uint32_t* const red = reinterpret_cast<uint32_t*>(mem + L::red);
        bool ok = true, slow = false;
        float4 kr[2][NC];                                                // keys 2 warp + half and 32 more, 4 dims of every chunk of 64
        float2 vr[KT];                                                   // KT values, two columns
        auto load = [&](uint32_t t) {
            const uint32_t u0 = c.k0 + t * kSpKeys;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t u = u0 + 32 * j + 2 * warp + half;
#pragma unroll
                for (int i = 0; i < NC; i++) kr[j][i] = sa_load<true>(c.kp + (size_t)u * a.pkw, 64 * i + 4 * hl, a.dk, u < c.k1);
            }
#pragma unroll
            for (int j = 0; j < KT; j++) {
                const uint32_t u = u0 + v_key + j;
                vr[j] = u < c.k1 && v_col < a.dv ? *reinterpret_cast<const float2*>(c.vp + (size_t)u * a.pvw + v_col) : make_float2(0.0f, 0.0f);
            }
        };
        auto convert = [&](uint32_t t) {
            const uint32_t s = t % kSpStages;
            uint8_t* const stage = mem + s * L::stage;
            float vm = 0.0f;
#pragma unroll
            for (int j = 0; j < KT; j++) vm = abs_or_inf(abs_or_inf(vm, vr[j].x), vr[j].y);
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(vm));           // magnitudes order as their bits do
            if (lane == 0) red[(t & 1) * 16 + warp] = top;
            bar_sync(5, kSpWorkers);
            vm = __uint_as_float(__reduce_max_sync(0xffffffffu, red[(t & 1) * 16 + (lane & 15)]));
            float vs, v_inv;
            split_scale(vm, vs, v_inv);
            if (t >= kSpStages && ok) ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * s, (t / kSpStages - 1) & 1));
            uint32_t small = 0, n_small = 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t key = 32 * j + 2 * warp + half;
                float km = 0.0f, ks, k_inv;
#pragma unroll
                for (int i = 0; i < NC; i++) km = abs_or_inf(abs_or_inf(abs_or_inf(abs_or_inf(km, kr[j][i].x), kr[j][i].y), kr[j][i].z), kr[j][i].w);
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, x));
                split_scale(km, ks, k_inv);
                slow = slow || !(k_inv == k_inv);
                if (hl == 0) kf[s * kSpKeys + key] = k_inv;
#pragma unroll
                for (int i = 0; i < NC; i++) {
                    const float4 x = make_float4(kr[j][i].x * ks, kr[j][i].y * ks, kr[j][i].z * ks, kr[j][i].w * ks);
                    small += sp_small(x.x) + sp_small(x.y) + sp_small(x.z) + sp_small(x.w);
                    uint2 hi, lo;
                    split2(x.x, x.y, hi.x, lo.x); split2(x.z, x.w, hi.y, lo.y);
                    uint8_t* const out = stage + i * kSpKeys * 128 + key * 128 + (((hl >> 1) ^ (key & 7)) << 4) + 8 * (hl & 1);
                    *reinterpret_cast<uint2*>(out) = hi;
                    *reinterpret_cast<uint2*>(out + L::k_part) = lo;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                uint32_t hi[KT / 2], lo[KT / 2];
#pragma unroll
                for (int j = 0; j < KT; j += 2) {
                    const float x = (e ? vr[j].y : vr[j].x) * vs, y = (e ? vr[j + 1].y : vr[j + 1].x) * vs;
                    n_small += sp_small(x) + sp_small(y);
                    split2(x, y, hi[j / 2], lo[j / 2]);
                }
                const uint32_t col = v_col + e;
                uint8_t* const out = stage + 2 * L::k_part + col * 128 + (((v_key >> 3) ^ (col & 7)) << 4) + 2 * (v_key & 7);
                if constexpr (KT == 8) {
                    *reinterpret_cast<uint4*>(out) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(out + L::v_part) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                } else {
                    *reinterpret_cast<uint2*>(out) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(out + L::v_part) = make_uint2(lo[0], lo[1]);
                }
            }
            small = __reduce_add_sync(0xffffffffu, small); n_small = __reduce_add_sync(0xffffffffu, n_small);
            slow = slow || !(v_inv == v_inv) || small >= kSpSmall || n_small >= kSpSmall;
            if (threadIdx.x == 0) vf[s] = v_inv;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * s);
        };
        load(0);
        // The queries come by whole rows into the later stages, and a thread takes its quarter row from there.
        const SpRow w = sp_row(a, c, head, row);
        uint32_t n_share = 0;
        auto row_max = [&](float x) {                                    // over the row's four threads; two buffers in turns, so one barrier is enough
            float* s = share + (n_share++ & 1) * 512;
            s[part * 128 + row] = x;
            bar_sync(1 + (warp & 3), 128);
            return fmaxf(fmaxf(s[row], s[128 + row]), fmaxf(s[256 + row], s[384 + row]));
        };
        float f;                                                         // a score in units of log2 is f times the key's factor times the product
        {
            float* const stage = reinterpret_cast<float*>(mem + L::stage);
            constexpr uint32_t Q4 = 16 * NC;                             // float4s of a row; float4 j of row r lies at place j ^ (r & 7)
            for (uint32_t i = threadIdx.x; i < 128 * Q4; i += kSpWorkers) {
                const uint32_t r = i / Q4, j = i % Q4;
                const SpRow x = sp_row(a, c, head, r);
                const bool on = x.on && 4 * j < a.dk;
                const float* from = a.q + (size_t)x.r * a.q_rs + (size_t)x.h * a.dk;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(stage + 4 * (r * Q4 + (j ^ (r & 7))))), "l"(on ? from + 4 * j : from), "r"(on ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            bar_sync(5, kSpWorkers);
            float4 x[4 * NC];                                            // 16 NC dims from 16 NC part on
            float mx = 0.0f, qs, q_inv;
#pragma unroll
            for (int i = 0; i < 4 * NC; i++) x[i] = *reinterpret_cast<const float4*>(stage + 4 * (row * Q4 + ((4 * NC * part + i) ^ (row & 7))));
#pragma unroll
            for (int i = 0; i < 4 * NC; i++) mx = abs_or_inf(abs_or_inf(abs_or_inf(abs_or_inf(mx, x[i].x), x[i].y), x[i].z), x[i].w);
            split_scale(row_max(mx), qs, q_inv);
            uint32_t small = 0;
#pragma unroll
            for (int i = 0; i < NC; i++) {                               // 16 dims: 8 columns of pairs
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 y = make_float4(x[4 * i + j].x * qs, x[4 * i + j].y * qs, x[4 * i + j].z * qs, x[4 * i + j].w * qs);
                    small += sp_small(y.x) + sp_small(y.y) + sp_small(y.z) + sp_small(y.w);
                    split2(y.x, y.y, hi[2 * j], lo[2 * j]);
                    split2(y.z, y.w, hi[2 * j + 1], lo[2 * j + 1]);
                }
                tmem_st(lanes + kQ + 8 * (NC * part + i), hi);
                tmem_st(lanes + kQ + 32 * NC + 8 * (NC * part + i), lo);
            }
            slow = small >= kSpSmall || !(q_inv == q_inv);
            f = q_inv * a.scale * 1.4426950408889634f;
            tmem_wait_st();
            fence_before();
            bar_sync(5, kSpWorkers);                                     // the stages are free
            if (lane == 0) mbar_arrive(q_full);
        }
        float o[OW];
#pragma unroll
        for (int i = 0; i < OW; i++) o[i] = 0.0f;
        float m = -INFINITY, l = 0.0f, alpha_prev = 1.0f, f_prev = 0.0f;
        auto add_output = [&](uint32_t t) {                              // outputs of tile t join the running ones
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * (t & 1), (t >> 1) & 1));
            fence_after();
            uint32_t v[OW];
            tmem_ld(lanes + kO + (t & 1) * DV + OW * part, v);
            tmem_wait_ld(v);
#pragma unroll
            for (int j = 0; j < OW; j += 2) {
                const float2 r = __ffma2_rn(make_float2(o[j], o[j + 1]), make_float2(alpha_prev, alpha_prev),
                                            __fmul2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), make_float2(f_prev, f_prev)));
                o[j] = r.x; o[j + 1] = r.y;
            }
        };
        convert(0);
        if (n_tiles > 1) load(1);
#pragma unroll 1
        for (uint32_t t = 0; t < n_tiles; t++) {
            if (t + 1 < n_tiles) {
                convert(t + 1);
                if (t + 2 < n_tiles) load(t + 2);
            } else bar_sync(5, kSpWorkers);                              // factors of tile t are there (inside the loop the barrier of the next tile says so)
            const uint32_t s = lanes + kS + (t & 1) * kSpKeys + 16 * part, u0 = c.k0 + t * kSpKeys + 16 * part;
            const float4* const key_f = reinterpret_cast<const float4*>(kf + (t % kSpStages) * kSpKeys + 16 * part);
            const float v_inv = vf[t % kSpStages];
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * (t & 1), (t >> 1) & 1));
            fence_after();
            uint32_t v[16];
            tmem_ld(s, v);
            tmem_wait_ld(v);
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const float4 y = key_f[j / 4];
                x[j] = __uint_as_float(v[j]) * (y.x * f); x[j + 1] = __uint_as_float(v[j + 1]) * (y.y * f); x[j + 2] = __uint_as_float(v[j + 2]) * (y.z * f); x[j + 3] = __uint_as_float(v[j + 3]) * (y.w * f);
            }
            if (a.cap > 0.0f) {
#pragma unroll
                for (int j = 0; j < 16; j++) x[j] = a.cap * tanhf(x[j] * 0.6931471805599453f / a.cap) * 1.4426950408889634f;
            }
            if (u0 + 16 > c.k1) {
#pragma unroll
                for (int j = 0; j < 16; j++) if (u0 + j >= c.k1) x[j] = -INFINITY;
            }
            float m0 = x[0], m1 = x[1];
#pragma unroll
            for (int j = 2; j < 16; j += 2) { m0 = fmaxf(m0, x[j]); m1 = fmaxf(m1, x[j + 1]); }
            const float mx = row_max(fmaxf(m0, m1)), m_new = fmaxf(m, mx);
            slow = slow || mx == INFINITY;
            const float alpha = m == -INFINITY ? 0.0f : sp_ex2(m - m_new), shift = m_new == -INFINITY ? 14.0f : 14.0f - m_new;      // probabilities times 2^14
            m = m_new;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                x[j] = sp_ex2(x[j] + shift); x[j + 1] = sp_ex2(x[j + 1] + shift);
                l0 += x[j]; l1 += x[j + 1];
                split2(x[j], x[j + 1], v[j / 2], v[8 + j / 2]);
            }
            tmem_st(s, v);
            l = fmaf(l, alpha, l0 + l1);
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
            if (t) add_output(t - 1);
            alpha_prev = alpha; f_prev = v_inv;
        }
        add_output(n_tiles - 1);
        {
            float* s = share + (n_share & 1) * 512;                      // the row's sum
            s[part * 128 + row] = l;
            bar_sync(1 + (warp & 3), 128);
            l = (s[row] + s[128 + row]) + (s[256 + row] + s[384 + row]);
        }
        constexpr float unit = 1.0f / 16384.0f;
        // Outputs leave by whole rows, through the idle stages.
        float4* const out = reinterpret_cast<float4*>(mem);
#pragma unroll
        for (int j = 0; j < OW; j += 4) out[row * (DV / 4) + (((OW * part + j) / 4) ^ (row & 7))] = make_float4(o[j] * unit, o[j + 1] * unit, o[j + 2] * unit, o[j + 3] * unit);
        if (slow || (w.on && m < -1e36f)) atomicOr(trouble, 1u);
        if (!ok) { atomicOr(trouble, 2u); if (lane == 0) count_timeout(); }
        bar_sync(5, kSpWorkers);
        const uint32_t what = *reinterpret_cast<volatile uint32_t*>(trouble);
        if (what == 1) sp_plain(a, c, head);
        else {
            const bool lost = what & 2u;
            if (w.on && part == 0) { float* rec = sa_record(a, w.r, w.h, c.split); rec[0] = lost ? kBatchNaN : m * 0.6931471805599453f; rec[1] = lost ? kBatchNaN : l * unit; }
            for (uint32_t i = threadIdx.x; i < 128 * (DV / 4); i += kSpWorkers) {
                const uint32_t r = i / (DV / 4), j = i % (DV / 4);
                const SpRow x = sp_row(a, c, head, r);
                if (!x.on || 4 * j >= a.dv) continue;
                *reinterpret_cast<float4*>(sa_record(a, x.r, x.h, c.split) + 4 + 4 * j) = lost ? make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN) : out[r * (DV / 4) + (j ^ (r & 7))];
            }
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(0u) : "memory");
}

// What decides a launch: queries a CTA of k_shared_rows holds (RQ), float4 a lane holds (NV), lanes that share a key (LK), shares of its keys; shares of the prefix
// on the tensor cores (0: k_shared_rows walks the prefix too).
struct SaShape { uint32_t RQ, NV, LK, chunks, splits, shares, row_tiles; };
SaShape sa_shape(const ZgSeqOp& s, bool wide) {
    const uint32_t B = s.n[0], G = s.n[2], rep = s.n[1] / G, dk = s.n[3], dv = s.n[4], dim = std::max(dk, dv), R = s.n[8], Rp = s.n[11], sms = zg_sm_count();
    SaShape p = {};
    p.NV = dim <= 512 ? 4 : dim <= 640 ? 5 : 8;
    p.LK = 1;
    while (p.LK * 4 * p.NV < dim) p.LK <<= 1;
    p.RQ = std::min(rep, p.NV == 8 ? 2u : 4u);
    p.chunks = (rep + p.RQ - 1) / p.RQ;
    if (wide && Rp && dk <= 128 && dv <= 128 && B * rep >= 32) {
        // The number of shares that keeps the GPU busy with the fewest tiles of 64 keys one after the other, and six tiles' time for each start and end.
        p.row_tiles = (B * rep + 127) / 128;
        const uint32_t items = p.row_tiles * G, tiles = (Rp + 63) / 64;
        uint64_t best = ~0ull;
        for (uint32_t n = 1; n <= std::min(tiles, 64u); n++) {
            const uint64_t cost = (uint64_t)((items * n + sms - 1) / sms) * (((Rp + n - 1) / n + 15) / 16 + 24);
            if (cost < best) { best = cost; p.shares = n; }
        }
    }
    const uint32_t ctas = B * G * p.chunks, keys = R + (p.shares ? 0 : Rp);
    p.splits = std::max(1u, std::min({(8 * sms + ctas - 1) / ctas, (keys + kSaShare - 1) / kSaShare, 128u}));
    return p;
}
// 16-byte loads of every operand, as far as sizes and offsets say so (buffers begin at 16 bytes at least)
bool sa_vec(const ZgSeqOp& s) {
    for (uint32_t x : {s.n[3], s.n[4], s.n[5], s.n[6], s.n[7], s.off[0], s.off[1], s.off[2]}) if (x % 4) return false;
    return s.buf[4] == ZG_NO_BUF || !(s.n[9] % 4 || s.n[10] % 4 || s.off[3] % 4 || s.off[4] % 4);
}
template <int NC, int DV>
bool sa_launch_prefix(const SaArgs& a, const SaShape& p, cudaStream_t st) {
    typedef SpLayout<NC, DV> L;
    if (!zg_smem_limit<k_shared_prefix<NC, DV>>(L::size)) return false;
    launch_pdl(k_shared_prefix<NC, DV>, dim3(p.row_tiles * a.shares * a.G), dim3(kSpThreads), L::size, st, a, p.row_tiles);
    return true;
}
template <int RQ, int NV>
bool sa_launch_rows(const SaArgs& a, const SaShape& p, bool vec, cudaStream_t st) {
    const dim3 grid(a.B * a.G * p.chunks, a.splits);
    const size_t smem = sizeof(float) * kSaWarps * RQ * (2 + a.dv);
    if (smem > 48 * 1024) {
        if (!(vec ? zg_smem_limit<k_shared_rows<RQ, NV, true>>(sizeof(float) * kSaWarps * RQ * 1026) : zg_smem_limit<k_shared_rows<RQ, NV, false>>(sizeof(float) * kSaWarps * RQ * 1026))) return false;
    }
    if (vec) launch_pdl(k_shared_rows<RQ, NV, true>, grid, dim3(32 * kSaWarps), smem, st, a, p.chunks, p.LK);
    else launch_pdl(k_shared_rows<RQ, NV, false>, grid, dim3(32 * kSaWarps), smem, st, a, p.chunks, p.LK);
    return true;
}

}  // namespace

bool zg_shared_attention_valid(const ZgSeqOp& s, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    const size_t B = s.n[0], H = s.n[1], G = s.n[2], dk = s.n[3], dv = s.n[4], qrs = s.n[5], kw = s.n[6], vw = s.n[7], R = s.n[8], pkw = s.n[9], pvw = s.n[10], Rp = s.n[11], drs = s.n[12];
    if (!B || !H || !G || H % G || !dk || !dv || dk > 1024 || dv > 1024 || !R || B > 65536 || H > 1024 || R >= (1u << 31) || Rp >= (1u << 31)) return fail("shared_attention: shape");
    if ((B > 1 && qrs < s.off[0] + H * dk) || !fits(1, s.off[0], (B - 1) * qrs + H * dk) || (B > 1 && drs < s.off[6] + H * dv) || !fits(0, s.off[6], (B - 1) * drs + H * dv)) return fail("shared_attention: rows");
    if (kw < s.off[1] + G * dk || vw < s.off[2] + G * dv || !fits(2, 0, R * kw) || !fits(3, 0, R * vw)) return fail("shared_attention: caches");
    const bool prefix = s.buf[4] != ZG_NO_BUF || s.buf[5] != ZG_NO_BUF;
    if (prefix && (!Rp || pkw < s.off[3] + G * dk || pvw < s.off[4] + G * dv || !fits(4, 0, Rp * pkw) || !fits(5, 0, Rp * pvw))) return fail("shared_attention: prefix");
    if (!prefix && Rp) return fail("shared_attention: prefix rows without a prefix");
    if (!fits(6, 0, ZG_BATCH_ROWS + 4 * B)) return fail("shared_attention: table");
    if (s.buf[7] != ZG_NO_BUF && (s.n[13] > ZG_W_BF16 || !have(7) || (s.n[13] == ZG_W_BF16 ? (s.off[5] + H + 1) / 2 : s.off[5] + H) > elems[s.buf[7]])) return fail("shared_attention: sinks");
    if (!(s.f[0] - s.f[0] == 0.0f) || !(s.f[1] >= 0.0f) || !(s.f[1] - s.f[1] == 0.0f)) return fail("shared_attention: scale or cap");
    for (int i = 1; i < 8; i++) if (s.buf[0] == s.buf[i]) return fail("shared_attention: in place");
    return true;
}
size_t zg_shared_attention_scratch_elems(const ZgSeqOp& s) {
    const SaShape p = sa_shape(s, sa_vec(s));
    return p.shares + p.splits > 1 ? (size_t)s.n[0] * s.n[1] * (p.shares + p.splits) * (4 + s.n[4]) : 0;
}
bool zg_launch_shared_attention(const ZgOp& op, float* const* bufs, const size_t* elems, float* scratch, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    SaArgs a;
    a.B = s.n[0]; a.H = s.n[1]; a.G = s.n[2]; a.rep = a.H / a.G; a.dk = s.n[3]; a.dv = s.n[4]; a.q_rs = s.n[5]; a.kw = s.n[6]; a.vw = s.n[7]; a.R = s.n[8]; a.pkw = s.n[9]; a.pvw = s.n[10]; a.Rp = s.n[11];
    a.dst_rs = s.n[12]; a.sink_bf16 = s.n[13] == ZG_W_BF16;
    a.dst = bufs[s.buf[0]] + s.off[6]; a.q = bufs[s.buf[1]] + s.off[0]; a.kc = bufs[s.buf[2]] + s.off[1]; a.vc = bufs[s.buf[3]] + s.off[2];
    const bool prefix = s.buf[4] != ZG_NO_BUF;
    a.kp = prefix ? bufs[s.buf[4]] + s.off[3] : a.kc; a.vp = prefix ? bufs[s.buf[5]] + s.off[4] : a.vc;
    if (!prefix) { a.pkw = a.kw; a.pvw = a.vw; }
    auto slots = [&](int k, int v, size_t kn, size_t vn) { return (uint32_t)std::min<size_t>({elems[s.buf[k]] / kn, elems[s.buf[v]] / vn, (size_t)1 << 31}); };
    a.slots = slots(2, 3, (size_t)a.R * a.kw, (size_t)a.R * a.vw);
    a.pslots = prefix ? slots(4, 5, (size_t)a.Rp * a.pkw, (size_t)a.Rp * a.pvw) : 0;
    a.table = bufs[s.buf[6]];
    a.sink = s.buf[7] == ZG_NO_BUF ? nullptr : a.sink_bf16 ? (const void*)wptr<bf16>(bufs, s.buf[7], s.off[5]) : (const void*)wptr<float>(bufs, s.buf[7], s.off[5]);
    a.scale = s.f[0]; a.cap = s.f[1];
    const bool vec = sa_vec(s);
    SaShape p = sa_shape(s, vec && scratch);
    if (!scratch) p.splits = 1;                       // no room for records: a row's keys are one share
    a.shares = p.shares; a.splits = p.splits;
    a.part = scratch;
    if (a.shares) {
        const bool k1 = a.dk <= 64, v1 = a.dv <= 64;
        if (!(k1 ? v1 ? sa_launch_prefix<1, 64>(a, p, st) : sa_launch_prefix<1, 128>(a, p, st) : v1 ? sa_launch_prefix<2, 64>(a, p, st) : sa_launch_prefix<2, 128>(a, p, st))) return false;
        ZG_SEQ_CHECK();
    }
    bool ok = false;
#define ZG_SA(NV_)                                                                       \
    switch (p.RQ) {                                                                      \
        case 1: ok = sa_launch_rows<1, NV_>(a, p, vec, st); break;                       \
        case 2: ok = sa_launch_rows<2, NV_>(a, p, vec, st); break;                       \
        case 3: ok = sa_launch_rows<3, NV_>(a, p, vec, st); break;                       \
        default: ok = sa_launch_rows<4, NV_>(a, p, vec, st); break;                      \
    }
    if (p.NV == 4) { ZG_SA(4); }
    else if (p.NV == 5) { ZG_SA(5); }
    else if (p.RQ == 1) ok = sa_launch_rows<1, 8>(a, p, vec, st);
    else ok = sa_launch_rows<2, 8>(a, p, vec, st);
#undef ZG_SA
    if (!ok) return false;
    ZG_SEQ_CHECK();
    if (a.shares + a.splits > 1) {
        launch_pdl(k_shared_merge, dim3(a.B * a.H), dim3(128), 0, st, a);
        ZG_SEQ_CHECK();
    }
    return true;
}
unsigned int zg_shared_attention_timeouts() { return tc_timeouts(); }
