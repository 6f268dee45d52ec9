// SHARED_ATTENTION (parameter pack in include/zgml_cuda.h): every row of a batch attends over the keys of one prefix that all rows share and over the
// keys of its own sequence, with one softmax over both.
//
// Softmax attention over a set of keys that falls into shares needs a record (m, l, o) per share: the largest score, the sum of exp(s - m) and the sum of
// exp(s - m) v.  Records of any shares merge into the whole: m = max m_i, l = sum l_i e^(m_i - m), o = sum o_i e^(m_i - m) / l.
#include "batch_table.cuh"
#include "exp2.cuh"
#include "split_tc.cuh"

#include <algorithm>

namespace {

struct SaArgs {
    float* dst; const float* q; const float* kc; const float* vc; const float* kp; const float* vp; const float* table;
    const void* sink;
    float* part;                     // records [B, H, shares (0: splits), 4 + dv]: m, l, -, -, o
    uint32_t B, H, G, rep, dk, dv, q_rs, kw, vw, R, pkw, pvw, Rp, dst_rs, slots, pslots, sink_bf16;
    uint32_t shares, splits;         // shares of the prefix, which k_shared_prefix walks (0: k_shared_rows walks all keys), and of what is left to k_shared_rows
    float scale, cap;
    uint32_t k_x, v_x;               // first columns of the prefix's key and value heads, for copies by tensor maps over whole rows
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
__device__ __forceinline__ float* sa_record(const SaArgs& a, uint32_t r, uint32_t h, uint32_t i) { return a.part + ((size_t)(r * a.H + h) * (a.shares ? a.shares : a.splits) + i) * (4 + a.dv); }
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

// CTA (share of the keys; row, key head, chunk of RQ of its query heads).  LK lanes share a key: each holds NV float4 of it, of the queries and of the outputs; a warp
// takes two keys per lane group at a time, the warps' keys are interleaved.  Keys and values come through a ring of kSaRing stages a warp, and a lane reads only what it
// copied itself, so nothing but its own copies is waited for.  Every lane group keeps its own running maximum and sum and leaves a record in shared memory.
// The shares of a row are a cluster (of at most 8) whose CTAs take a slice of the output columns each.  The records that k_shared_prefix has left join there, or in the
// one CTA of a row.  Where eight shares are too few (a.part with a.shares = 0) CTAs leave records for k_shared_merge.
// What bounds it is instruction latency beside the reads: 32 rows with 257 keys of their own on average took 53 us with one key per lane group and turn and the lane groups
// merged by shuffles (600 instructions a turn of 4 keys), 27 us now; 47 us with a bulk copy per row, 35 us with the copies in pieces between the products.
constexpr uint32_t kSaRing = 2, kSaMaxWarps = 8, kSaCluster = 8, kSaMost = 256 + 64;      // most records that meet: of 8 warps' lane groups and of the prefix
__device__ __forceinline__ float2 sa_remote2(const float* p, uint32_t rank) {
    uint32_t at;
    float2 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 sa_remote4(const float* p, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sa_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
template <bool VEC>
__device__ __forceinline__ void sa_copy(uint32_t at, const float* p, uint32_t d, uint32_t n, bool on) {
    if constexpr (VEC) {
        const bool in = on && d < n;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(in ? p + d : p), "r"(in ? 16 : 0) : "memory");
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const bool in = on && d + i < n;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at + 4 * i), "l"(in ? p + d + i : p), "r"(in ? 4 : 0) : "memory");
        }
    }
}
// weights of `count` records in the frame of the largest maximum, by one warp: at(e) is the maximum and sum of record e.  Returns the maximum; *sum: of all.
template <class At>
__device__ __forceinline__ float sa_weights(float* weight, uint32_t count, const At& at, float* sum) {
    const uint32_t lane = threadIdx.x & 31;
    float top = -INFINITY, total = 0.0f;
    for (uint32_t e = lane; e < count; e += 32) top = fmaxf(top, at(e).x);
    top = warp_max(top);
    for (uint32_t e = lane; e < count; e += 32) {
        const float2 y = at(e);
        const float f = sa_weight(y.x, top);
        weight[e] = f;
        total = fmaf(y.y, f, total);
    }
    *sum = warp_sum(total);
    return top;
}
template <int RQ, int NV, bool VEC>
__global__ void __launch_bounds__(32 * kSaMaxWarps) k_shared_rows(const SaArgs a, uint32_t chunks, uint32_t LK) {
    pdl_enter();
    extern __shared__ float4 ring[];                                // [warps][kSaRing][2][2 NV][32]; then the records [warps][lane groups][RQ][4 + padded dv], and the CTA's own
    __shared__ float weight[RQ][kSaMost], sum_of[RQ], top_of[RQ];
    float* const sh = reinterpret_cast<float*>(ring);
    const uint32_t split = blockIdx.x % a.splits, item = blockIdx.x / a.splits, c = item % chunks, g = item / chunks % a.G, r = item / chunks / a.G, warps = blockDim.x >> 5;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LK - 1), group = lane / LK, groups = 32 / LK;
    const uint32_t h0 = g * a.rep + c * RQ, nq = min((uint32_t)RQ, a.rep - c * RQ);
    const bool records = a.part && !a.shares;                       // for k_shared_merge
    const SaKeys k = sa_keys(a, r, g);
    if (!k.live) return;                                            // (the whole cluster)
    const uint32_t first = a.shares ? k.prefix : 0u, n = k.prefix + k.own, share = sa_share(n - first, a.splits, kSaShare), k0 = min(n, first + split * share), k1 = min(n, k0 + share);
    if (records && split && k0 >= n) return;                        // (share 0 leaves a record however few the keys are)
    const uint32_t step = 2 * warps * groups, turns = (k1 - k0 + step - 1) / step;
    float4* const mine = ring + (size_t)warp * kSaRing * 4 * NV * 32 + lane;
    auto fetch = [&](uint32_t t) {
        if (t < turns) {
            const uint32_t to = smem_u32(mine + (t % kSaRing) * 4 * NV * 32);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t u = k0 + t * step + (2 * warp + x) * groups + group;
                const bool on = u < k1, own = u >= k.prefix;
                const uint32_t at = own ? u - k.prefix : u;
                const float* kr = on ? (own ? k.kc : k.kp) + (size_t)at * (own ? a.kw : a.pkw) : k.kc;
                const float* vr = on ? (own ? k.vc : k.vp) + (size_t)at * (own ? a.vw : a.pvw) : k.vc;
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    sa_copy<VEC>(to + (x * 2 * NV + j) * 512, kr, 4 * (sub + LK * j), a.dk, on);
                    sa_copy<VEC>(to + (x * 2 * NV + NV + j) * 512, vr, 4 * (sub + LK * j), a.dv, on);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (uint32_t t = 0; t < kSaRing - 1; t++) fetch(t);
    // Scores in units of log2: the scale and log2(e) are folded into the queries.
    const float unit = a.cap > 0.0f ? a.scale : a.scale * kLog2e;
    const float inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    float2 q[RQ][2 * NV], o[RQ][2 * NV];
    float m[RQ], l[RQ];
#pragma unroll
    for (int i = 0; i < RQ; i++) {
        m[i] = -INFINITY; l[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const float4 x = sa_load<VEC>(a.q + (size_t)r * a.q_rs + (size_t)(h0 + i) * a.dk, 4 * (sub + LK * j), a.dk, i < (int)nq);
            q[i][2 * j] = make_float2(x.x * unit, x.y * unit); q[i][2 * j + 1] = make_float2(x.z * unit, x.w * unit);
            o[i][2 * j] = o[i][2 * j + 1] = make_float2(0.0f, 0.0f);
        }
    }
#pragma unroll 1
    for (uint32_t t = 0; t < turns; t++) {
        fetch(t + kSaRing - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kSaRing - 1) : "memory");
        const uint32_t u = k0 + t * step + 2 * warp * groups + group;
        const float4* from = mine + (t % kSaRing) * 4 * NV * 32;
        float s[2][RQ];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            float2 d[RQ];
#pragma unroll
            for (int i = 0; i < RQ; i++) d[i] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float4 y = from[32 * (x * 2 * NV + j)];
#pragma unroll
                for (int i = 0; i < RQ; i++) d[i] = __ffma2_rn(q[i][2 * j + 1], make_float2(y.z, y.w), __ffma2_rn(q[i][2 * j], make_float2(y.x, y.y), d[i]));
            }
#pragma unroll
            for (int i = 0; i < RQ; i++) s[x][i] = d[i].x + d[i].y;
        }
        for (uint32_t w = LK >> 1; w > 0; w >>= 1)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int i = 0; i < RQ; i++) s[x][i] += __shfl_xor_sync(0xffffffffu, s[x][i], w);
        float up = -INFINITY;                                       // by how much any maximum grows
#pragma unroll
        for (int i = 0; i < RQ; i++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                if (a.cap > 0.0f) s[x][i] = kLog2e * sa_capped(s[x][i], a.cap, inv_cap);
                if (u + x * groups >= k1) s[x][i] = -INFINITY;
            }
            up = fmaxf(up, fmaxf(s[0][i], s[1][i]) > m[i] ? 1.0f : -1.0f);
        }
        if (__any_sync(0xffffffffu, up > 0.0f)) {
#pragma unroll
            for (int i = 0; i < RQ; i++) {
                const float top = fmaxf(m[i], fmaxf(s[0][i], s[1][i])), f = m[i] == -INFINITY ? 0.0f : sa_ex2(m[i] - top);
                m[i] = top;
                l[i] *= f;
#pragma unroll
                for (int j = 0; j < 2 * NV; j++) o[i][j] = __fmul2_rn(o[i][j], make_float2(f, f));
            }
        }
#pragma unroll
        for (int i = 0; i < RQ; i++) {
#pragma unroll
            for (int x = 0; x < 2; x++) s[x][i] = s[x][i] == -INFINITY ? 0.0f : sa_ex2(s[x][i] - m[i]);
            l[i] += s[0][i] + s[1][i];
        }
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const float4 v = from[32 * (x * 2 * NV + NV + j)];
#pragma unroll
                for (int i = 0; i < RQ; i++) {
                    const float2 p = make_float2(s[x][i], s[x][i]);
                    o[i][2 * j] = __ffma2_rn(p, make_float2(v.x, v.y), o[i][2 * j]);
                    o[i][2 * j + 1] = __ffma2_rn(p, make_float2(v.z, v.w), o[i][2 * j + 1]);
                }
            }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                                // the ring is idle
    const uint32_t dvp = (a.dv + 3) & ~3u, rec = 4 + dvp, local = warps * groups;      // record e, head i: at (e RQ + i) rec
#pragma unroll
    for (int i = 0; i < RQ; i++) {
        float* out = sh + ((size_t)(warp * groups + group) * RQ + i) * rec;
        if (sub == 0) { out[0] = m[i] * kLn2; out[1] = l[i]; }      // (infinite where no key was seen)
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const uint32_t d = 4 * (sub + LK * j);
            if (d < dvp) *reinterpret_cast<float4*>(out + 4 + d) = make_float4(o[i][2 * j].x, o[i][2 * j].y, o[i][2 * j + 1].x, o[i][2 * j + 1].y);
        }
    }
    __syncthreads();
    const uint32_t per = sa_share(k.prefix, max(1u, a.shares), kSaShare), n_prefix = a.shares ? (k.prefix + per - 1) / per : 0u;
    const bool alone = a.splits == 1;                               // the prefix's records join here; in a cluster later
    for (uint32_t i = warp; i < nq; i += warps) {
        const float* prefix = a.shares ? sa_record(a, r, h0 + i, 0) : nullptr;
        const float* here = sh + i * rec;
        float sum;
        const float top = sa_weights(weight[i], local + (alone ? n_prefix : 0u), [&](uint32_t e) { return *reinterpret_cast<const float2*>(e < local ? here + (size_t)e * RQ * rec : prefix + (size_t)(e - local) * (4 + a.dv)); }, &sum);
        if (lane == 0) { top_of[i] = top; sum_of[i] = sum; }
    }
    __syncthreads();
    // what the CTA's sums and weights make of the row: the factor of its outputs
    auto closing = [&](uint32_t i) {
        float sum = sum_of[i];
        if (a.sink && top_of[i] != -INFINITY) sum += expf(sa_sink(a, h0 + i) - top_of[i]);
        return k.bad ? kBatchNaN : top_of[i] == -INFINITY ? 0.0f : 1.0f / sum;          // nothing seen: zeros
    };
    auto store = [&](uint32_t i, uint32_t d, float4 v) {
        float* out = a.dst + (size_t)r * a.dst_rs + (size_t)(h0 + i) * a.dv + d;
        if (d + 3 < a.dv && (reinterpret_cast<uintptr_t>(out) & 15) == 0) { *reinterpret_cast<float4*>(out) = v; return; }
        out[0] = v.x;
        if (d + 1 < a.dv) out[1] = v.y;
        if (d + 2 < a.dv) out[2] = v.z;
        if (d + 3 < a.dv) out[3] = v.w;
    };
    auto add = [](float4& v, const float4 x, float f) { v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w); };
    auto add_prefix = [&](float4& v, uint32_t i, uint32_t d, uint32_t e0) {      // (dv is a multiple of four there)
        const float* prefix = sa_record(a, r, h0 + i, 0) + 4 + d;
#pragma unroll 6
        for (uint32_t e = 0; e < n_prefix; e++) add(v, *reinterpret_cast<const float4*>(prefix + (size_t)e * (4 + a.dv)), weight[i][e0 + e]);
    };
    float* const sums = sh + (size_t)local * RQ * rec;              // in a cluster: the CTA's own record per head, behind the others
    const uint32_t quads = dvp / 4;
    for (uint32_t x = threadIdx.x; x < nq * quads; x += blockDim.x) {
        const uint32_t i = x / quads, d = 4 * (x % quads);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t e = 0; e < local; e++) add(v, *reinterpret_cast<const float4*>(sh + ((size_t)e * RQ + i) * rec + 4 + d), weight[i][e]);
        if (records) {
            float* out = sa_record(a, r, h0 + i, split);
            if (d == 0) { out[0] = top_of[i]; out[1] = sum_of[i]; }
            for (uint32_t e = 0; e < 4; e++) if (d + e < a.dv) out[4 + d + e] = (&v.x)[e];
        } else if (alone) {
            if (n_prefix) add_prefix(v, i, d, local);
            const float f = closing(i);
            store(i, d, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
        } else {
            if (d == 0) { sums[i * rec] = top_of[i]; sums[i * rec + 1] = sum_of[i]; }
            *reinterpret_cast<float4*>(sums + i * rec + 4 + d) = v;
        }
    }
    if (records || alone) return;
    sa_cluster_sync();
    for (uint32_t i = warp; i < nq; i += warps) {
        const float* prefix = a.shares ? sa_record(a, r, h0 + i, 0) : nullptr;
        float sum;
        const float top = sa_weights(weight[i], a.splits + n_prefix, [&](uint32_t e) {
            return e < a.splits ? sa_remote2(sums + i * rec, e) : *reinterpret_cast<const float2*>(prefix + (size_t)(e - a.splits) * (4 + a.dv)); }, &sum);
        if (lane == 0) { top_of[i] = top; sum_of[i] = sum; }
    }
    __syncthreads();
    const uint32_t slice = (quads + a.splits - 1) / a.splits, q0 = min(quads, split * slice), width = min(quads, q0 + slice) - q0;
    for (uint32_t x = threadIdx.x; x < nq * width; x += blockDim.x) {
        const uint32_t i = x / width, d = 4 * (q0 + x % width);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float4 y[kSaCluster];                                       // all on their way before the first is added
#pragma unroll
        for (uint32_t e = 0; e < kSaCluster; e++) if (e < a.splits) y[e] = sa_remote4(sums + i * rec + 4 + d, e);
#pragma unroll
        for (uint32_t e = 0; e < kSaCluster; e++) if (e < a.splits) add(v, y[e], weight[i][e]);
        if (n_prefix) add_prefix(v, i, d, a.splits);
        const float f = closing(i);
        store(i, d, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
    sa_cluster_sync();                                              // no CTA leaves while its sums are read
}
// CTA (row, head): the records of its shares become the result.  Warp 0 finds the weights; then the warps take every fourth record each.
__global__ void __launch_bounds__(256) k_shared_merge(const SaArgs a) {
    pdl_enter();
    __shared__ float weight[128], total, part[7][1024 / 4 * 4];
    const uint32_t h = blockIdx.x % a.H, r = blockIdx.x / a.H, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SaKeys k = sa_keys(a, r, 0);
    if (!k.live) return;
    const uint32_t left = k.prefix + k.own, per = sa_share(left, a.splits, kSaShare), n = max(1u, (left + per - 1) / per);
    const float* rec = sa_record(a, r, h, 0);
    if (warp == 0) {
        float mm[4], ll[4], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const uint32_t e = lane + 32 * x;
            mm[x] = -INFINITY; ll[x] = 0.0f;
            if (e < n) { mm[x] = rec[(size_t)e * (4 + a.dv)]; ll[x] = rec[(size_t)e * (4 + a.dv) + 1]; }
            top = fmaxf(top, mm[x]);
        }
        top = warp_max(top);
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const float f = sa_weight(mm[x], top);
            sum = fmaf(ll[x], f, sum);
            if (lane + 32 * x < n) weight[lane + 32 * x] = f;
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            if (a.sink && top != -INFINITY) sum += expf(sa_sink(a, h) - top);
            total = k.bad ? kBatchNaN : top == -INFINITY ? 0.0f : 1.0f / sum;
        }
    }
    __syncthreads();
    float* out = a.dst + (size_t)r * a.dst_rs + (size_t)h * a.dv;
    for (uint32_t d = lane; d < a.dv; d += 32) {
        float v = 0.0f;
        for (uint32_t e = warp; e < n; e += 8) v = fmaf(rec[(size_t)e * (4 + a.dv) + 4 + d], weight[e], v);
        if (warp) part[warp - 1][d] = v; else out[d] = v;
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.dv; d += 256) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 7; w++) v += part[w][d];
        out[d] = (out[d] + v) * total;
    }
}

// ── the prefix on the tensor cores ───────────────────────────────────────────────────────────────────────────────────
// All query rows of a key head meet the same keys of the prefix, so its part of the attention is two matrix products.  CTA (key head, share of the prefix, tile of 128 query
// rows): 64 keys and values at a time are read from the cache once, split into half-precision pairs on their way to shared memory (one scale per tile;
// split_tc.cuh) and multiplied by tcgen05.mma, three MMAs a product.  Warp 25 copies (TMA), warps 16 - 23 split, warp 24 issues, warps 0 - 15 are the softmax: four threads share a query
// row, each with a quarter of the keys and of the output columns.  (With all of it in the same 16 warps, one phase after the other, a tile took 7700 clocks.)
//   TMEM: scores of two tiles, which become the probabilities in place (A operand), outputs of two tiles, the queries' pairs (A operand).
//   Elements of a pair are off by at most 2^-25 where the largest of a row or tile is below 2^15 (split_tc.cuh), so a score by at most 2 dk 2^-10 times its scales'
//   inverses; with those times log2(e) below kSpLoud = 2^-17 that is less than 2^-18 for 128 dims.  Louder scores (beyond 2^20), values that are small as a whole beside others of their tile
//   and what is not finite are found on the way; the CTA then walks its share again in plain f32.
// Every wait is bounded; a CTA whose wait ran out counts it and makes NaN of its rows.
constexpr uint32_t kSpRows = 512, kSpSplit = 256, kSpThreads = kSpRows + kSpSplit + 128, kSpStages = 2, kSpKeys = 64;      // threads: softmax, splitting, issue and copies (two warps of four)
template <int NC, int DV> struct SpLayout {
    static constexpr uint32_t k_part = NC * kSpKeys * 128, v_part = DV * 128, stage = 2 * (k_part + v_part);      // bytes; a part: hi or lo
    // the queries pass through the second stage on their way to TMEM; keys and values as they come lie behind
    static constexpr uint32_t k_raw = kSpStages * stage > stage + NC * 32768 ? kSpStages * stage : stage + NC * 32768, v_raw = k_raw + kSpKeys * 64 * NC * 4, share = v_raw + kSpKeys * DV * 4;
    static constexpr uint32_t factors = share + 2 * 4 * 128 * 4, red = factors + kSpStages * 16, rows = red + 4 * 8 * 4, bars = rows + 128 * 4, size = bars + 192 + 1024;
};
constexpr float kSpLoud = 1.0f / 131072.0f;
// Eight values of one column, or two of one key, that are not zero but below these parts of the tile's largest: a pair keeps 22 bits of a value above 2^-18, 19 above 2^-21.
constexpr float kSpColumn = 1.0f / 262144.0f, kSpKey = 1.0f / 2097152.0f;
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
__device__ __noinline__ void sp_plain(const SaArgs& a, const float* kp, const float* vp, uint32_t k0, uint32_t k1, uint32_t split, const uint32_t* rows) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t i0 = warp * 8; i0 < warp * 8 + 8; i0 += 4) {
        float4 q[4], o[4];
        float m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = rows[i0 + i];
            q[i] = sa_load<true>(a.q + (size_t)(w >> 10) * a.q_rs + (size_t)(w & 1023) * a.dk, 4 * lane, a.dk, w != 0xffffffffu);
            o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); m[i] = -INFINITY; l[i] = 0.0f;
        }
        for (uint32_t u = k0; u < k1; u++) {
            const float4 x = sa_load<true>(kp + (size_t)u * a.pkw, 4 * lane, a.dk, true), v = sa_load<true>(vp + (size_t)u * a.pvw, 4 * lane, a.dv, true);
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
            const uint32_t w = rows[i0 + i];
            if (w == 0xffffffffu) continue;
            float* rec = sa_record(a, w >> 10, w & 1023, split);
            if (lane == 0) { rec[0] = m[i]; rec[1] = l[i]; }
            if (4 * lane < a.dv) { rec[4 + 4 * lane] = o[i].x; rec[5 + 4 * lane] = o[i].y; rec[6 + 4 * lane] = o[i].z; rec[7 + 4 * lane] = o[i].w; }
        }
    }
}
template <int NC, int DV>
__global__ void __launch_bounds__(kSpThreads, 1) k_shared_prefix(const __grid_constant__ SaArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const uint32_t row_tiles) {
    typedef SpLayout<NC, DV> L;
    constexpr uint32_t kS = 0, kO = 2 * kSpKeys, kQ = kO + 2 * DV;         // TMEM columns
    static_assert(kQ + 64 * NC <= 512, "TMEM columns");
    extern __shared__ uint8_t dsm_raw[];
    const uint32_t base = (smem_u32(dsm_raw) + 1023u) & ~1023u;
    uint8_t* const mem = dsm_raw + (base - smem_u32(dsm_raw));
    const uint32_t full = base + L::bars, empty = full + 8 * kSpStages, s_full = empty + 8 * kSpStages, o_full = s_full + 16, p_full = o_full + 16, q_full = p_full + 16, tmem_slot = q_full + 8, raw_full = tmem_slot + 8, raw_empty = raw_full + 16;      // (the latter: keys, values)
    uint32_t* const trouble = reinterpret_cast<uint32_t*>(mem + (tmem_slot + 4 - base));          // 1: something that pairs cannot hold, 2: a wait that ran out
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (in a form that the compiler knows to be the same in all lanes)
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kSpStages; i++) { mbar_init(full + 8 * i, 8); mbar_init(empty + 8 * i, 1); }
        for (uint32_t i = 0; i < 2; i++) { mbar_init(s_full + 8 * i, 1); mbar_init(o_full + 8 * i, 1); mbar_init(p_full + 8 * i, 16); mbar_init(raw_full + 8 * i, 1); mbar_init(raw_empty + 8 * i, 8); }
        mbar_init(q_full, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *trouble = 0;
    }
    if (warp == 24) {
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
    const uint32_t n_tiles = __shfl_sync(0xffffffffu, (c.k1 - c.k0 + kSpKeys - 1) / kSpKeys, 0);
    uint32_t* const rows = reinterpret_cast<uint32_t*>(mem + L::rows);     // row << 10 | head of the tile's query rows, all bits set where there is none
    if (threadIdx.x < 128) {
        const SpRow w = sp_row(a, c, head, threadIdx.x);
        rows[threadIdx.x] = w.on ? w.r << 10 | w.h : 0xffffffffu;
    }
    fence_before();
    __syncthreads();
    fence_after();

    // Registers: 896 threads of 72 at launch, 64512 in all = 512 x 72 + 256 x 96 + 128 x 24.
    if (warp >= 24) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
        if (n_tiles && warp == 24) {
            // Issue.  Three products, the small ones first: hi lo, lo hi, hi hi.  B parts: hi, then lo; chunks of 64 along the summed dimension are 8 KB apart.  The whole warp
            // does all but the issue itself, so that addresses stay warp-uniform.
            constexpr uint32_t idesc_s = (1u << 4) | ((kSpKeys >> 3) << 17) | ((128u >> 4) << 24), idesc_o = (1u << 4) | ((DV >> 3) << 17) | ((128u >> 4) << 24);      // f16 x f16 -> f32
            uint32_t in = 0, in_phase = 0, out = 0;                      // stages of the next scores and values
            bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0));
            auto scores = [&](uint32_t t) {
                const uint32_t d = kS + (t & 1) * kSpKeys, b = desc_low(base) + in * (L::stage >> 4);
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (uint32_t x = 0; x < 3; x++)
#pragma unroll
                        for (uint32_t k = 0; k < 4 * NC; k++) {
                            const uint32_t qa = kQ + (x == 1 ? 32 * NC : 0) + 8 * k, kb = b + (x == 0 ? L::k_part >> 4 : 0) + (k / 4) * (kSpKeys * 128 >> 4) + 2 * (k % 4);
                            if (x == 0 && k == 0) mma_ts<false>(d, qa, kb, idesc_s); else mma_ts<true>(d, qa, kb, idesc_s);
                        }
                    mma_commit(s_full + 8 * (t & 1));
                }
                __syncwarp();
                if (++in == kSpStages) { in = 0; in_phase ^= 1; }
            };
            // probabilities of 16 keys lie in 16 columns: 8 with their hi pairs, 8 with their lo pairs
            auto values = [&](uint32_t t) {
                const uint32_t d = kO + (t & 1) * DV, pa = kS + (t & 1) * kSpKeys, b = desc_low(base) + out * (L::stage >> 4) + (2 * L::k_part >> 4), freed = empty + 8 * out;
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (uint32_t x = 0; x < 3; x++)
#pragma unroll
                        for (uint32_t k = 0; k < kSpKeys / 16; k++) {
                            const uint32_t p = pa + 16 * k + (x == 1 ? 8 : 0), vb = b + (x == 0 ? L::v_part >> 4 : 0) + 2 * k;
                            if (x == 0 && k == 0) mma_ts<false>(d, p, vb, idesc_o); else mma_ts<true>(d, p, vb, idesc_o);
                        }
                    mma_commit(o_full + 8 * (t & 1));
                    mma_commit(freed);
                }
                __syncwarp();
                if (++out == kSpStages) out = 0;
            };
            // Whichever is ready comes next.  (Scores before values in turns cost 1500 clocks a tile: the values waited for keys that waited for their stage.)  Scores of tile t
            // overwrite the probabilities of tile t - 2, whose values have been issued: products execute in order.
            uint32_t next_s = 0, next_v = 0, spins = 0;
            while (ok && next_v < n_tiles) {
                if (next_v < next_s && __all_sync(0xffffffffu, mbar_test(p_full + 8 * (next_v & 1), (next_v >> 1) & 1))) { values(next_v++); spins = 0; }
                else if (next_s < n_tiles && next_s <= next_v + 1 && __all_sync(0xffffffffu, mbar_test(full + 8 * in, in_phase))) { scores(next_s++); spins = 0; }
                else ok = ++spins < kTcSpin;
            }
            if (!ok && lane == 0) { count_timeout(); atomicOr(trouble, 2u); }
            __syncwarp();
        } else if (n_tiles && warp == 25) {
            // copies: 64 rows of the prefix at a time, what lies behind the share among them
            if (elect_one()) {
                const uint32_t y0 = (uint32_t)head.prefix_slot * a.Rp + c.k0;
                bool ok = true;
                for (uint32_t t = 0; t < n_tiles && ok; t++) {
                    ok = mbar_wait(raw_empty, (t & 1) ^ 1);
                    if (ok) { mbar_expect_tx(raw_full, kSpKeys * a.dk * 4); tma_2d(base + L::k_raw, &map_k, a.k_x + c.g * a.dk, y0 + t * kSpKeys, raw_full); ok = mbar_wait(raw_empty + 8, (t & 1) ^ 1); }
                    if (ok) { mbar_expect_tx(raw_full + 8, kSpKeys * a.dv * 4); tma_2d(base + L::v_raw, &map_v, a.v_x + c.g * a.dv, y0 + t * kSpKeys, raw_full + 8); }
                }
                if (!ok) { count_timeout(); atomicOr(trouble, 2u); }
            }
            __syncwarp();
        }
    } else if (warp >= 16) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        if (n_tiles) {
            // ── keys and values: global memory, registers, pairs in shared memory ──
            constexpr int KT = DV == 128 ? 8 : 4;                        // value rows of a thread, of two blocks of 32 columns
            const uint32_t sw = warp - 16, half = lane >> 4, hl = lane & 15;
            const uint32_t v_key = DV == 128 ? 16 * (sw & 3) + 8 * half : 8 * sw + 4 * half, v_col = (DV == 128 ? 64 * (sw >> 2) : 0) + 2 * hl;
            float2* const factors = reinterpret_cast<float2*>(mem + L::factors);
            uint32_t* const red = reinterpret_cast<uint32_t*>(mem + L::red);
            bool ok = true, slow = false;
            float4 kr[4][NC];                                            // keys 16 j + 2 sw + half, 4 dims of every chunk of 64
            float2 vr[2][KT];                                            // KT values, two columns of each block
            // what TMA has brought -> registers; the place is free for the next tile then.  Keys behind the share count as zeros: what lies there is not looked at
            const float* const k_raw = reinterpret_cast<const float*>(mem + L::k_raw);
            const float* const v_raw = reinterpret_cast<const float*>(mem + L::v_raw);
            auto load_keys = [&](uint32_t t) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(raw_full, t & 1));
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t key = 16 * j + 2 * sw + half;
#pragma unroll
                    for (int i = 0; i < NC; i++) kr[j][i] = sa_load<true>(k_raw + key * a.dk, 64 * i + 4 * hl, a.dk, c.k0 + t * kSpKeys + key < c.k1);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty);
            };
            auto load_values = [&](uint32_t t) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(raw_full + 8, t & 1));
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (uint32_t j = 0; j < KT; j++) {
                        const uint32_t key = v_key + j;
                        vr[b][j] = c.k0 + t * kSpKeys + key < c.k1 && v_col + 32 * b < a.dv ? *reinterpret_cast<const float2*>(v_raw + key * a.dv + v_col + 32 * b) : make_float2(0.0f, 0.0f);
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(raw_empty + 8);
            };
            // the largest magnitude over the warps, from a warp's; magnitudes order as their bits do
            auto over_warps = [&](float x, uint32_t at) {
                const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(x));
                if (lane == 0) red[at * 8 + sw] = top;
                bar_sync(5, kSpSplit);
                return __uint_as_float(__reduce_max_sync(0xffffffffu, red[at * 8 + (lane & 7)]));
            };
            uint32_t fill = 0, fill_phase = 1;                           // the stage that is filled next
#pragma unroll 1
            for (uint32_t t = 0; t < n_tiles; t++) {
                uint8_t* const stage = mem + fill * L::stage;
                float km = 0.0f;
                load_keys(t);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < NC; i++) km = fmaxf(fmaxf(fmaxf(km, fabsf(kr[j][i].x)), fmaxf(fabsf(kr[j][i].y), fabsf(kr[j][i].z))), fabsf(kr[j][i].w));
                km = over_warps(km, t & 1);                              // (two places in turns: one barrier is enough)
                float ks, k_inv, vs, v_inv;
                split_scale(km, ks, k_inv);
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * fill, fill_phase));
                if (t == 1 && ok) ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0));      // the queries pass through the later stages
                uint8_t* const k_out = stage + (2 * sw + half) * 128 + (((hl >> 1) ^ ((2 * sw + half) & 7)) << 4) + 8 * (hl & 1);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < NC; i++) {
                        uint2 hi, lo;
                        split2(kr[j][i].x * ks, kr[j][i].y * ks, hi.x, lo.x); split2(kr[j][i].z * ks, kr[j][i].w * ks, hi.y, lo.y);
                        uint8_t* const out = k_out + i * kSpKeys * 128 + j * 16 * 128;
                        *reinterpret_cast<uint2*>(out) = hi;
                        *reinterpret_cast<uint2*>(out + L::k_part) = lo;
                    }
                load_values(t);
                float vm = 0.0f, cm[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                uint32_t least = 0xffffffffu;                            // the smallest of the keys' two values, zeros left out
#pragma unroll
                for (int b = 0; b < 2; b++) {
#pragma unroll
                    for (int j = 0; j < KT; j++) {
                        cm[b][0] = fmaxf(cm[b][0], fabsf(vr[b][j].x)); cm[b][1] = fmaxf(cm[b][1], fabsf(vr[b][j].y));
                        least = min(least, __float_as_uint(fmaxf(fabsf(vr[b][j].x), fabsf(vr[b][j].y))) - 1u);
                    }
                    vm = fmaxf(vm, fmaxf(cm[b][0], cm[b][1]));
                }
                vm = over_warps(vm, 2 + (t & 1));
                split_scale(vm, vs, v_inv);
                slow = slow || !(k_inv == k_inv) || !(v_inv == v_inv) || least < __float_as_uint(vm * kSpKey);
#pragma unroll
                for (int b = 0; b < 2; b++) slow = slow || (cm[b][0] > 0.0f && cm[b][0] < vm * kSpColumn) || (cm[b][1] > 0.0f && cm[b][1] < vm * kSpColumn);
                if (sw == 0 && lane == 0) factors[fill] = make_float2(k_inv, v_inv);
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        uint32_t hi[KT / 2], lo[KT / 2];
#pragma unroll
                        for (int j = 0; j < KT; j += 2) split2((e ? vr[b][j].y : vr[b][j].x) * vs, (e ? vr[b][j + 1].y : vr[b][j + 1].x) * vs, hi[j / 2], lo[j / 2]);
                        const uint32_t col = v_col + 32 * b + e;
                        uint8_t* const out = stage + 2 * L::k_part + col * 128 + (((v_key >> 3) ^ (col & 7)) << 4) + 2 * (v_key & 7);
                        if constexpr (KT == 8) {
                            *reinterpret_cast<uint4*>(out) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4*>(out + L::v_part) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        } else {
                            *reinterpret_cast<uint2*>(out) = make_uint2(hi[0], hi[1]);
                            *reinterpret_cast<uint2*>(out + L::v_part) = make_uint2(lo[0], lo[1]);
                        }
                    }
                if (slow) atomicOr(trouble, 1u);
                if (!ok && lane == 0) atomicOr(trouble, 2u);             // before the pairs are handed over: whoever takes them reads it afterwards
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * fill);
                if (++fill == kSpStages) { fill = 0; fill_phase ^= 1; }
            }
            if (!ok && lane == 0) count_timeout();
        }
    } else if (n_tiles) {
        // ── softmax: four threads per query row ──
        constexpr int OW = DV / 4;                                       // output columns of a thread
        const uint32_t part = warp >> 2, row = (warp & 3) * 32 + lane, lanes = ((warp & 3) * 32) << 16;
        float* const share = reinterpret_cast<float*>(mem + L::share);
        const float2* const factors = reinterpret_cast<const float2*>(mem + L::factors);      // of a stage's keys and values
        bool ok = true, slow = false;
        uint32_t n_share = 0;
        auto row_max = [&](float x) {                                    // over the row's four threads; two buffers in turns, so one barrier is enough
            float* s = share + (n_share++ & 1) * 512;
            s[part * 128 + row] = x;
            bar_sync(1 + (warp & 3), 128);
            return fmaxf(fmaxf(s[row], s[128 + row]), fmaxf(s[256 + row], s[384 + row]));
        };
        float f;                                                         // a score in units of log2 is f times the keys' factor times the product
        // The queries come by whole rows into the later stages, and a thread takes its quarter row from there.
        {
            float* const stage = reinterpret_cast<float*>(mem + L::stage);
            constexpr uint32_t Q4 = 16 * NC;                             // float4s of a row; float4 j of row r lies at place j ^ (r & 7)
            for (uint32_t i = threadIdx.x; i < 128 * Q4; i += kSpRows) {
                const uint32_t r = i / Q4, j = i % Q4;
                const uint32_t w = rows[r];
                const bool on = w != 0xffffffffu && 4 * j < a.dk;
                const float* from = on ? a.q + (size_t)(w >> 10) * a.q_rs + (size_t)(w & 1023) * a.dk : a.q;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(stage + 4 * (r * Q4 + (j ^ (r & 7))))), "l"(on ? from + 4 * j : from), "r"(on ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            bar_sync(6, kSpRows);
            float4 x[4 * NC];                                            // 16 NC dims from 16 NC part on
            float mx = 0.0f, qs, q_inv;
#pragma unroll
            for (int i = 0; i < 4 * NC; i++) x[i] = *reinterpret_cast<const float4*>(stage + 4 * (row * Q4 + ((4 * NC * part + i) ^ (row & 7))));
#pragma unroll
            for (int i = 0; i < 4 * NC; i++) mx = abs_or_inf(abs_or_inf(abs_or_inf(abs_or_inf(mx, x[i].x), x[i].y), x[i].z), x[i].w);
            split_scale(row_max(mx), qs, q_inv);
            if (a.scale < 0.0f) qs = -qs;                                // f is not negative
#pragma unroll
            for (int i = 0; i < NC; i++) {                               // 16 dims: 8 columns of pairs
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 y = make_float4(x[4 * i + j].x * qs, x[4 * i + j].y * qs, x[4 * i + j].z * qs, x[4 * i + j].w * qs);
                    split2(y.x, y.y, hi[2 * j], lo[2 * j]);
                    split2(y.z, y.w, hi[2 * j + 1], lo[2 * j + 1]);
                }
                tmem_st(lanes + kQ + 8 * (NC * part + i), hi);
                tmem_st(lanes + kQ + 32 * NC + 8 * (NC * part + i), lo);
            }
            f = q_inv * fabsf(a.scale) * kLog2e;
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);                          // the queries are there, and the stages are free
        }
        float o[OW];
#pragma unroll
        for (int i = 0; i < OW; i++) o[i] = 0.0f;
        // Probabilities are held times 2^14.  The outputs lose that factor as they join the running ones: what was kept with it would overflow 2^14 times too early.
        constexpr float p_unit = 1.0f / 16384.0f;
        float m = -INFINITY, l = 0.0f, alpha_prev = 1.0f, f_prev = 0.0f;
        auto add_output = [&](uint32_t t) {                              // outputs of tile t join the running ones
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * (t & 1), (t >> 1) & 1));
            fence_after();
#pragma unroll
            for (int h = 0; h < OW; h += 16) {                           // sixteen at a time: registers
                uint32_t v[16];
                tmem_ld(lanes + kO + (t & 1) * DV + OW * part + h, v);
                tmem_wait_ld(v);
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 r = __ffma2_rn(make_float2(o[h + j], o[h + j + 1]), make_float2(alpha_prev, alpha_prev),
                                                __fmul2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), make_float2(f_prev, f_prev)));
                    o[h + j] = r.x; o[h + j + 1] = r.y;
                }
            }
        };
        uint32_t at = 0, at_phase = 0;                                   // stage of tile t
#pragma unroll 1
        for (uint32_t t = 0; t < n_tiles; t++) {
            const uint32_t s = lanes + kS + (t & 1) * kSpKeys + 16 * part, u0 = c.k0 + t * kSpKeys + 16 * part;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * at, at_phase) && mbar_wait(s_full + 8 * (t & 1), (t >> 1) & 1));      // (the former for the factors)
            fence_after();
            const float2 inv = factors[at];
            if (++at == kSpStages) { at = 0; at_phase ^= 1; }
            uint32_t v[16];
            tmem_ld(s, v);
            tmem_wait_ld(v);
            float x[16], unit = fmaxf(f * inv.x, 1e-37f);
            slow = slow || !(fabsf(f * inv.x) <= kSpLoud);
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = __uint_as_float(v[j]);
            if (a.cap > 0.0f) {                                          // here in units of log2
                const float inv_cap = 1.0f / a.cap;
#pragma unroll
                for (int j = 0; j < 16; j++) x[j] = sa_capped(x[j] * (unit * kLn2), a.cap, inv_cap) * kLog2e;
                unit = 1.0f;
            }
            if (u0 + 16 > c.k1) {
#pragma unroll
                for (int j = 0; j < 16; j++) if (u0 + j >= c.k1) x[j] = -INFINITY;
            }
            float m0 = x[0], m1 = x[1];
#pragma unroll
            for (int j = 2; j < 16; j += 2) { m0 = fmaxf(m0, x[j]); m1 = fmaxf(m1, x[j + 1]); }
            const float mx = fmaxf(m0, m1), m_new = fmaxf(m, row_max(mx * unit));
            slow = slow || m_new == INFINITY;
            const float alpha = m == -INFINITY ? 0.0f : sa_ex2(m - m_new), shift = m_new == -INFINITY ? 14.0f : 14.0f - m_new;      // probabilities times 2^14
            m = m_new;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float2 y = __ffma2_rn(make_float2(x[j], x[j + 1]), make_float2(unit, unit), make_float2(shift, shift));
                const float p0 = sa_ex2(y.x), p1 = sa_ex2(y.y);
                l0 += p0; l1 += p1;
                split2(p0, p1, v[j / 2], v[8 + j / 2]);
            }
            tmem_st(s, v);
            l = fmaf(l, alpha, l0 + l1);
            tmem_wait_st();
            fence_before();
            __syncwarp();
            // (a barrier for even and one for odd tiles: warps may be a tile apart)
            if (lane == 0) mbar_arrive(p_full + 8 * (t & 1));
            if (t) add_output(t - 1);
            alpha_prev = alpha; f_prev = inv.y * p_unit;
        }
        add_output(n_tiles - 1);
        {
            float* s = share + (n_share & 1) * 512;                      // the row's sum
            s[part * 128 + row] = l;
            bar_sync(1 + (warp & 3), 128);
            l = (s[row] + s[128 + row]) + (s[256 + row] + s[384 + row]);
        }
        // Outputs leave by whole rows, through the idle stages.
        float4* const out = reinterpret_cast<float4*>(mem);
#pragma unroll
        for (int j = 0; j < OW; j += 4) out[row * (DV / 4) + (((OW * part + j) / 4) ^ (row & 7))] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        const uint32_t mine = rows[row];
        if (slow || (mine != 0xffffffffu && m < -1e36f)) atomicOr(trouble, 1u);
        if (!ok) { atomicOr(trouble, 2u); if (lane == 0) count_timeout(); }
        bar_sync(6, kSpRows);
        const uint32_t what = *reinterpret_cast<volatile uint32_t*>(trouble);
        if (what == 1) sp_plain(a, c.kp, c.vp, c.k0, c.k1, c.split, rows);
        else {
            const bool lost = what & 2u;
            if (mine != 0xffffffffu && part == 0) { float* rec = sa_record(a, mine >> 10, mine & 1023, c.split); rec[0] = lost ? kBatchNaN : m * kLn2; rec[1] = lost ? kBatchNaN : l * p_unit; }
            for (uint32_t i = threadIdx.x; i < 128 * (DV / 4); i += kSpRows) {
                const uint32_t r = i / (DV / 4), j = i % (DV / 4);
                const uint32_t w = rows[r];
                if (w == 0xffffffffu || 4 * j >= a.dv) continue;
                *reinterpret_cast<float4*>(sa_record(a, w >> 10, w & 1023, c.split) + 4 + 4 * j) = lost ? make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN) : out[r * (DV / 4) + (j ^ (r & 7))];
            }
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 24) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(0u) : "memory");
}

// ── the prefix on the tensor cores, heads wider than 128 ─────────────────────────────────────────────────────────────
// A head of 576 dims has no room for 128 queries beside its keys, and 512 columns of outputs none beside the scores.  So everything streams: a first kernel leaves the
// queries, keys and values as half-precision pairs in the workspace (a scale per row; values inside the key rows of a latent are the same pairs), and CTA (key head, share
// of the prefix, up to 256 output columns, tile of 128 query rows) multiplies tiles of 128 keys from there, 64 dims at a time, through three stages that TMA fills:
//   scores[128 rows x 128 keys] += queries[64 dims] keys[64 dims]^T, three MMAs a product;  outputs[128 x 64 columns] += probabilities[128 keys] values[128 keys x 64 columns].
// Values come as the keys do, by rows, and are read as a transposed operand.  Warps 0 - 7 are the softmax (two threads a query row, each with half of the keys and of the output
// columns), warp 8 issues, warp 9 copies.
// A tensor core's f32 sum is cut, not rounded, at every product that joins it, always towards zero.  So the small products (hi lo, lo hi) of the scores have sums of their own, which
// are added as the scores are read, and a tile's outputs join running ones in registers.  (With all three in one sum, and outputs that stayed in TMEM from tile to tile: 16 rows, 16
// heads of 576 / 512 were off by 1.9e-6 behind 4096 keys and 4.3e-6 behind 32768, instead of 7.7e-7 and 8.7e-7; twenty tiles of positive values came out 1.8e-5 too small.)
// TMEM: large sums of two tiles (which become scores and then probabilities in place), outputs of one.  Small sums borrow half of the outputs' columns.  The products go scores of
// tile t + 1, values of tile t, scores of t + 2; values of t fill the half first that has no small sums of t + 1 in it, and the other one when those have been read, so nothing waits.
// What bounds it: 64 KB of operands for every 64 dims of a tile, which an SM takes 1030 clocks to read and 770 to multiply.  256 query rows, 4096 keys of 576 dims, 512 columns:
// pairs 8.5 us, this kernel 21.4 us (a tile a CTA: about 7500 clocks until the first copy, 11500 scores, 4000 outputs), k_shared_rows 27 us.
// What pairs cannot hold is known before the first product (the first kernel's scales and flags): the CTA then walks its share in plain f32.
constexpr uint32_t kSwKeys = 128, kSwCols = 256, kSwStages = 3, kSwPart = 128 * 128, kSwStage = 4 * kSwPart, kSwSoft = 256, kSwThreads = kSwSoft + 128;
constexpr uint32_t kSwFactors = kSwStages * kSwStage, kSwRows = kSwFactors + 2 * 128 * 8, kSwShare = kSwRows + 512, kSwRed = kSwShare + 2 * 256 * 4, kSwBars = kSwRed + 128, kSwSmem = kSwBars + 128 + 1024;
struct SwArgs {
    __half* q; __half* k; __half* v;             // pairs: [hi, lo][G][rows][dims, padded to 64]
    float* qf; float* kf; float* vf;             // what a row's pairs were divided by: [G][rows]; of a row of zeros 0, of a query that is not finite NaN
    uint32_t* flags;                             // [keys, values][G][blocks of eight rows]: something that pairs cannot hold
    uint32_t KR, QR, dkp, dvp, v0, latent, halves, row_tiles;      // rows of keys and queries; first column of the values in their plane; values are the keys' pairs
};
// Block of eight rows -> pairs.  Blocks: keys, values (unless they are the keys'), queries.  A thread holds four dims of the eight rows, and there are no more threads than that takes.
__global__ void __launch_bounds__(256) k_shared_pairs(const SaArgs a, const SwArgs w) {
    pdl_enter();
    __shared__ uint32_t red[8][8], bad_rows;
    const uint32_t kb = w.KR / 8, kinds = w.latent ? 1 : 2, keys = kinds * kb * a.G;
    const uint32_t kind = blockIdx.x >= keys ? 2 : blockIdx.x / (kb * a.G), in = kind == 2 ? blockIdx.x - keys : blockIdx.x % (kb * a.G), per = kind == 2 ? w.QR / 8 : kb, g = in / per, b = in % per;
    const BatchHead head = batch_head(a.table, a.B);
    const bool sound = head.prefix > 0 && (uint32_t)head.prefix <= a.Rp && (uint32_t)head.prefix_slot < a.pslots;
    const uint32_t P = sound ? (uint32_t)head.prefix : 0u, r0 = 8 * b, dim = kind == 1 ? a.dv : a.dk, dimp = kind == 1 ? w.dvp : w.dkp, t4 = 4 * threadIdx.x;
    if (!sound || (kind == 2 ? r0 >= head.rows * a.rep : r0 >= P + kSwKeys)) return;      // (a tile may reach so far behind the prefix: zeros there)
    float4 x[8];
    float mx[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float* from = nullptr;
        if (kind == 2) {
            SpCta c; c.g = g; c.tile = 0;
            const SpRow q = sp_row(a, c, head, r0 + i);
            if (q.on) from = a.q + (size_t)q.r * a.q_rs + (size_t)q.h * a.dk;
        } else if (r0 + i < P) {
            const size_t row = (size_t)head.prefix_slot * a.Rp + r0 + i;
            from = kind ? a.vp + row * a.pvw + g * a.dv : a.kp + row * a.pkw + g * a.dk;
        }
        x[i] = sa_load<true>(from, t4, dim, from != nullptr);
        mx[i] = abs_or_inf(abs_or_inf(abs_or_inf(abs_or_inf(0.0f, x[i].x), x[i].y), x[i].z), x[i].w);
    }
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) bad_rows = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx[i]));
        if (lane == 0) red[i][warp] = top;
    }
    __syncthreads();
    bool bad = false;
    float4 cm = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint32_t rows = kind == 2 ? w.QR : w.KR;
    __half* const plane = kind == 2 ? w.q : kind ? w.v : w.k;
    float* const factor = kind == 2 ? w.qf : kind ? w.vf : w.kf;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < blockDim.x / 32 ? red[i][lane] : 0u));
        float s, inv;
        split_scale(top, s, inv);
        const bool wrong = !(inv == inv);
        if (wrong) { x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); bad = true; }
        if (threadIdx.x == 0) factor[(size_t)g * rows + r0 + i] = wrong && kind == 2 ? kBatchNaN : wrong || top == 0.0f ? 0.0f : kind == 2 ? inv * fabsf(a.scale) * kLog2e : inv;
        if (kind == 2 && a.scale < 0.0f) s = -s;
        x[i] = make_float4(x[i].x * s, x[i].y * s, x[i].z * s, x[i].w * s);
        cm = make_float4(fmaxf(cm.x, fabsf(x[i].x)), fmaxf(cm.y, fabsf(x[i].y)), fmaxf(cm.z, fabsf(x[i].z)), fmaxf(cm.w, fabsf(x[i].w)));
        if (t4 < dimp) {
            uint2 hi, lo;
            split2(x[i].x, x[i].y, hi.x, lo.x); split2(x[i].z, x[i].w, hi.y, lo.y);
            *reinterpret_cast<uint2*>(plane + ((size_t)g * rows + r0 + i) * dimp + t4) = hi;
            *reinterpret_cast<uint2*>(plane + ((size_t)(a.G + g) * rows + r0 + i) * dimp + t4) = lo;
        }
    }
    if (kind == 2) return;
    // a column of values that is small as a whole beside its rows: pairs keep 22 bits above 2^-18 of a row's largest, which is scaled to 2^14 at least
    if (kind == 1 || (w.latent && t4 >= w.v0 && t4 < w.v0 + a.dv)) {
        constexpr float least = 32768.0f * kSpColumn;
        bad = bad || (cm.x > 0.0f && cm.x < least) || (cm.y > 0.0f && cm.y < least) || (cm.z > 0.0f && cm.z < least) || (cm.w > 0.0f && cm.w < least);
    }
    if (__syncthreads_or(bad) && threadIdx.x == 0) bad_rows = 1;
    if (threadIdx.x == 0) w.flags[((size_t)kind * a.G + g) * kb + b] = bad_rows;
}
// The CTA's share in plain f32, a warp a row at a time
__device__ __noinline__ void sw_plain(const SaArgs& a, const float* kp, const float* vp, uint32_t k0, uint32_t k1, uint32_t split, uint32_t c0, const uint32_t* rows) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t i = warp; i < 128; i += kSwThreads / 32) {
        const uint32_t w = rows[i];
        if (w == 0xffffffffu) continue;
        float4 q[8], o[2] = {};
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) q[j] = sa_load<true>(a.q + (size_t)(w >> 10) * a.q_rs + (size_t)(w & 1023) * a.dk, 4 * lane + 128 * j, a.dk, true);
        for (uint32_t u = k0; u < k1; u++) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float4 x = sa_load<true>(kp + (size_t)u * a.pkw, 4 * lane + 128 * j, a.dk, true);
                s = fmaf(q[j].x, x.x, fmaf(q[j].y, x.y, fmaf(q[j].z, x.z, fmaf(q[j].w, x.w, s))));
            }
            s = warp_sum(s) * a.scale;
            if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
            const float top = fmaxf(m, s), f = sa_weight(m, top), p = s == -INFINITY ? 0.0f : expf(s - top);
            m = top; l = fmaf(l, f, p);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float4 v = sa_load<true>(vp + (size_t)u * a.pvw, c0 + 4 * lane + 128 * j, a.dv, true);
                o[j].x = fmaf(o[j].x, f, p * v.x); o[j].y = fmaf(o[j].y, f, p * v.y); o[j].z = fmaf(o[j].z, f, p * v.z); o[j].w = fmaf(o[j].w, f, p * v.w);
            }
        }
        float* rec = sa_record(a, w >> 10, w & 1023, split);
        if (lane == 0 && c0 == 0) { rec[0] = m; rec[1] = l; }
#pragma unroll
        for (int j = 0; j < 2; j++) if (c0 + 4 * lane + 128 * j < a.dv) *reinterpret_cast<float4*>(rec + 4 + c0 + 4 * lane + 128 * j) = o[j];
    }
}
__global__ void __launch_bounds__(kSwThreads, 1) k_shared_wide(const __grid_constant__ SaArgs a, const __grid_constant__ SwArgs w, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                              const __grid_constant__ CUtensorMap map_v) {
    constexpr uint32_t kS = 0, kO = 2 * kSwKeys, kHalf = kSwCols / 2;       // TMEM columns; a half of the outputs
    static_assert(kHalf >= kSwKeys, "small sums in a half of the outputs");
    extern __shared__ uint8_t dsm_raw[];
    const uint32_t base = (smem_u32(dsm_raw) + 1023u) & ~1023u;
    uint8_t* const mem = dsm_raw + (base - smem_u32(dsm_raw));
    const uint32_t full = base + kSwBars, empty = full + 8 * kSwStages, s_full = empty + 8 * kSwStages, p_full = s_full + 16, o_full = p_full + 16, o_read = o_full + 16, small_read = o_read + 16, tmem_slot = small_read + 8;
    uint32_t* const lost = reinterpret_cast<uint32_t*>(mem + (tmem_slot + 4 - base));      // a wait ran out
    uint32_t* const red = reinterpret_cast<uint32_t*>(mem + kSwRed);        // largest and smallest factor of the values, largest of the keys
    uint32_t* const rows = reinterpret_cast<uint32_t*>(mem + kSwRows);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kSwStages; i++) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
        for (uint32_t i = 0; i < 2; i++) { mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, kSwSoft / 32); mbar_init(o_full + 8 * i, 1); mbar_init(o_read + 8 * i, kSwSoft / 64); }
        mbar_init(small_read, kSwSoft / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *lost = 0;
        red[0] = 0; red[1] = 0x7f800000u; red[2] = 0;
    }
    if (warp == kSwSoft / 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const BatchHead head = batch_head(a.table, a.B);
    SpCta c;
    const uint32_t half = blockIdx.x / w.row_tiles % w.halves, c0 = half * kSwCols, cols = min(kSwCols, a.dv - c0);
    c.tile = blockIdx.x % w.row_tiles; c.split = blockIdx.x / w.row_tiles / w.halves % a.shares; c.g = blockIdx.x / w.row_tiles / w.halves / a.shares;      // CTAs of the same keys are neighbours
    const bool sound = head.prefix > 0 && (uint32_t)head.prefix <= a.Rp && (uint32_t)head.prefix_slot < a.pslots && c.tile * 128 < head.rows * a.rep;
    const uint32_t P = sound ? (uint32_t)head.prefix : 0u, per = sa_share(P, a.shares, kSaShare);
    c.k0 = min(P, c.split * per); c.k1 = min(P, c.k0 + per);
    const size_t p0 = sound ? (size_t)head.prefix_slot * a.Rp : 0;
    c.kp = a.kp + p0 * a.pkw + c.g * a.dk; c.vp = a.vp + p0 * a.pvw + c.g * a.dv;
    const uint32_t n_tiles = __shfl_sync(0xffffffffu, (c.k1 - c.k0 + kSwKeys - 1) / kSwKeys, 0), nc = w.dkp / 64, nv = (cols + 63) / 64;
    const float* const kf = w.kf + (size_t)c.g * w.KR;
    const float* const vf = (w.latent ? w.kf : w.vf) + (size_t)c.g * w.KR;
    __syncthreads();
    // The largest and smallest factors of the share, and flags of all rows that its tiles touch
    bool slow = false;
    float f = 0.0f;                                                         // of the thread's query row
    if (n_tiles) {
        uint32_t v_top = 0, v_low = 0x7f800000u, k_top = 0;                 // (factors order as their bits do)
        for (uint32_t u = c.k0 + threadIdx.x; u < c.k1; u += kSwThreads) {
            const uint32_t y = __float_as_uint(vf[u]);
            v_top = max(v_top, y);
            if (y) v_low = min(v_low, y);
            k_top = max(k_top, __float_as_uint(kf[u]));
        }
        const uint32_t kb = w.KR / 8, b1 = (c.k0 + n_tiles * kSwKeys) / 8;
        for (uint32_t b = c.k0 / 8 + threadIdx.x; b < b1; b += kSwThreads) {
            slow = slow || w.flags[(size_t)c.g * kb + b] != 0;
            if (!w.latent) slow = slow || w.flags[(size_t)(a.G + c.g) * kb + b] != 0;
        }
        v_top = __reduce_max_sync(0xffffffffu, v_top); v_low = __reduce_min_sync(0xffffffffu, v_low); k_top = __reduce_max_sync(0xffffffffu, k_top);
        if (lane == 0) { atomicMax(red, v_top); atomicMin(red + 1, v_low); atomicMax(red + 2, k_top); }
        if (threadIdx.x < kSwSoft) {
            const uint32_t row = threadIdx.x & 127, at = c.tile * 128 + row;
            const SpRow q = sp_row(a, c, head, row);
            rows[row] = q.on ? q.r << 10 | q.h : 0xffffffffu;
            if (at < head.rows * a.rep) f = w.qf[(size_t)c.g * w.QR + at];
        }
    }
    __syncthreads();
    const float v_ref = __uint_as_float(red[0]), k_ref = __uint_as_float(red[2]);
    slow = slow || !(f * k_ref <= kSpLoud * 128.0f / (float)max(128u, a.dk)) || (red[0] && __uint_as_float(red[1]) < v_ref * (1.0f / 32768.0f));
    fence_before();
    const bool plain = __syncthreads_or(slow);
    fence_after();
    // Registers: 384 threads of 168 at launch, 64512 in all = 256 x 232 + 128 x 40.
    if (plain) {
        sw_plain(a, c.kp, c.vp, c.k0, c.k1, c.split, c0, rows);
    } else if (!n_tiles) {
    } else if (warp >= kSwSoft / 32) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == kSwSoft / 32 + 1) {
            if (elect_one()) {
                const uint32_t yq = c.g * w.QR + c.tile * 128, yk = c.g * w.KR + c.k0, q_lo = a.G * w.QR, k_lo = a.G * w.KR;
                uint32_t s = 0, phase = 1;
                bool ok = true;
                auto place = [&](uint32_t bytes) {
                    ok = ok && mbar_wait(empty + 8 * s, phase);
                    if (ok) mbar_expect_tx(full + 8 * s, bytes);
                    return ok;
                };
                auto next = [&] { if (++s == kSwStages) { s = 0; phase ^= 1; } };
                for (uint32_t t = 0; t <= n_tiles && ok; t++) {
                    if (t < n_tiles)
                        for (uint32_t i = 0; i < nc && place(kSwStage); i++) {
                            const uint32_t to = base + s * kSwStage, bar = full + 8 * s;
                            tma_2d(to, &map_q, 64 * i, yq, bar); tma_2d(to + kSwPart, &map_q, 64 * i, yq + q_lo, bar);
                            tma_2d(to + 2 * kSwPart, &map_k, 64 * i, yk + t * kSwKeys, bar); tma_2d(to + 3 * kSwPart, &map_k, 64 * i, yk + t * kSwKeys + k_lo, bar);
                            next();
                        }
                    if (t)
                        for (uint32_t z = 0; z < 2; z++) {
                            const uint32_t i = 2 * ((t & 1) ^ 1 ^ z), n = i < nv ? min(2u, nv - i) : 0u;
                            if (!n || !place(n * 2 * kSwPart)) continue;
                            for (uint32_t e = 0; e < n; e++) {
                                const uint32_t to = base + s * kSwStage + 2 * e * kSwPart, bar = full + 8 * s, x = w.v0 + c0 + 64 * (i + e);
                                tma_2d(to, &map_v, x, yk + (t - 1) * kSwKeys, bar); tma_2d(to + kSwPart, &map_v, x, yk + (t - 1) * kSwKeys + k_lo, bar);
                            }
                            next();
                        }
                }
                if (!ok) { count_timeout(); atomicOr(lost, 1u); }
            }
            __syncwarp();
        } else if (warp == kSwSoft / 32) {
            // Issue.  Three products: hi lo and lo hi into the small sums, hi hi into the large ones; of a tile's values the small ones first.
            constexpr uint32_t idesc_s = (1u << 4) | ((kSwKeys >> 3) << 17) | ((128u >> 4) << 24), idesc_o = (1u << 4) | (1u << 16) | ((64u >> 3) << 17) | ((128u >> 4) << 24);      // f16 x f16 -> f32; B transposed
            uint32_t s = 0, phase = 0;
            bool ok = true;
            auto take = [&] { ok = ok && __all_sync(0xffffffffu, mbar_wait(full + 8 * s, phase)); fence_after(); return ok; };
            auto next = [&] { if (++s == kSwStages) { s = 0; phase ^= 1; } };
            for (uint32_t t = 0; t <= n_tiles && ok; t++) {
                const uint32_t small = kO + (t & 1) * kHalf;                // the half where this tile's small sums go
                if (t < n_tiles) {
                    // (the large ones overwrite the probabilities of tile t - 2, whose values have been issued: products execute in order)
                    if (t >= 2) ok = __all_sync(0xffffffffu, mbar_wait(o_read + 8 * (t & 1), t & 1));
                    const uint32_t d = kS + (t & 1) * kSwKeys;
                    for (uint32_t i = 0; i < nc && take(); i++) {
                        const uint32_t q = desc_low(base + s * kSwStage), k = q + (2 * kSwPart >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t x = 0; x < 3; x++)
#pragma unroll
                                for (uint32_t j = 0; j < 4; j++) {
                                    const uint32_t qa = q + (x == 1 ? kSwPart >> 4 : 0) + 2 * j, ka = k + (x == 0 ? kSwPart >> 4 : 0) + 2 * j;
                                    if (x != 1 && j == 0 && i == 0) mma_ss<false>(x < 2 ? small : d, qa, ka, idesc_s); else mma_ss<true>(x < 2 ? small : d, qa, ka, idesc_s);
                                }
                            mma_commit(empty + 8 * s);
                            if (i + 1 == nc) mma_commit(s_full + 8 * (t & 1));
                        }
                        __syncwarp();
                        next();
                    }
                }
                if (t && ok) {
                    const uint32_t u = t - 1, p = kS + (u & 1) * kSwKeys;
                    ok = __all_sync(0xffffffffu, mbar_wait(p_full + 8 * (u & 1), (u >> 1) & 1));
                    for (uint32_t z = 0; z < 2 && ok; z++) {                // the half with the small sums of tile t comes last
                        const uint32_t h = (t & 1) ^ 1 ^ z, i = 2 * h, n = i < nv ? min(2u, nv - i) : 0u;
                        if (u) ok = __all_sync(0xffffffffu, mbar_wait(o_read + 8 * h, (u - 1) & 1));
                        if (ok && z && t < n_tiles) ok = __all_sync(0xffffffffu, mbar_wait(small_read, t & 1));
                        fence_after();
                        if (!ok || (n && !take())) break;
                        if (elect_one()) {
                            for (uint32_t e = 0; e < n; e++) {
                                const uint32_t d = kO + 64 * (i + e), v = (((base + s * kSwStage + 2 * e * kSwPart) & 0x3FFFF) >> 4) | (64u << 16);      // groups of eight keys are 1024 B apart
#pragma unroll
                                for (uint32_t x = 0; x < 3; x++)
#pragma unroll
                                    for (uint32_t j = 0; j < kSwKeys / 16; j++) {
                                        const uint32_t pa = p + 16 * j + (x == 1 ? 8 : 0), va = v + (x == 0 ? kSwPart >> 4 : 0) + 128 * j;
                                        if (x == 0 && j == 0) mma_ts<false>(d, pa, va, idesc_o); else mma_ts<true>(d, pa, va, idesc_o);
                                    }
                            }
                            if (n) mma_commit(empty + 8 * s);
                            mma_commit(o_full + 8 * h);
                        }
                        __syncwarp();
                        if (n) next();
                    }
                }
            }
            if (!ok && lane == 0) { count_timeout(); atomicOr(lost, 1u); }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // softmax: two threads a query row, each with half of the keys and of the output columns
        constexpr int OW = kHalf;
        const uint32_t part = warp >> 2, row = threadIdx.x & 127, lanes = ((warp & 3) * 32) << 16;
        float2* const factors = reinterpret_cast<float2*>(mem + kSwFactors);
        float* const share = reinterpret_cast<float*>(mem + kSwShare);
        const float v_inv = v_ref > 0.0f ? 1.0f / v_ref : 0.0f, inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;      // (a power of two)
        uint32_t n_share = 0;
        auto other = [&](float x) {                                         // what the row's other thread has; two buffers in turns, so one barrier is enough
            float* s = share + (n_share++ & 1) * 256;
            s[part * 128 + row] = x;
            bar_sync(2 + (warp & 3), 64);
            return s[(part ^ 1) * 128 + row];
        };
        float m = -INFINITY, l = 0.0f, alpha_prev = 0.0f;
        float2 o[OW / 2];
#pragma unroll
        for (int i = 0; i < OW / 2; i++) o[i] = make_float2(0.0f, 0.0f);
        bool ok = true;
        auto add_output = [&](uint32_t t) {                                 // outputs of tile t, the thread's half of them, join the running ones
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * part, t & 1));
            fence_after();
#pragma unroll
            for (int h = 0; h < OW; h += 16) {
                if (OW * part + h >= 64 * nv) break;
                uint32_t v[16];
                tmem_ld(lanes + kO + OW * part + h, v);
                tmem_wait_ld(v);
#pragma unroll
                for (int j = 0; j < 16; j += 2) o[(h + j) / 2] = __ffma2_rn(o[(h + j) / 2], make_float2(alpha_prev, alpha_prev), make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])));
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_read + 8 * part);
        };
#pragma unroll 1
        for (uint32_t t = 0; t < n_tiles; t++) {
            float2* const fs = factors + (t & 1) * 128;
            if (part == 0) {
                const uint32_t u = c.k0 + t * kSwKeys + row;
                fs[row] = u < c.k1 ? make_float2(kf[u], vf[u] * v_inv * 16384.0f) : make_float2(0.0f, 0.0f);      // probabilities times 2^14, in the frame of the share's largest values
            }
            bar_sync(1, kSwSoft);
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * (t & 1), (t >> 1) & 1));
            fence_after();
            const uint32_t s = lanes + kS + (t & 1) * kSwKeys, small = lanes + kO + (t & 1) * kHalf, h0 = 64 * part, left = c.k1 - c.k0 - t * kSwKeys;
            // Loops of 16 keys, whose scores go back to TMEM in between: a tile is often the only one, and code that runs once costs its fetching (all 128 unrolled took
            // 18000 clocks).
            float top = -INFINITY;
#pragma unroll 1
            for (uint32_t h = h0; h < h0 + 64; h += 16) {
                uint32_t v[16], u[16];
                tmem_ld(s + h, v);
                tmem_ld(small + h, u);
                tmem_wait_ld(v);
                tmem_wait_ld(u);
#pragma unroll
                for (int j = 0; j < 16; j++) v[j] = __float_as_uint((__uint_as_float(v[j]) + __uint_as_float(u[j])) * (f * fs[h + j].x));
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = __float_as_uint(sa_capped(__uint_as_float(v[j]) * kLn2, a.cap, inv_cap) * kLog2e);
                }
                if (h + 16 > left) {
#pragma unroll
                    for (int j = 0; j < 16; j++) if (h + j >= left) v[j] = 0xff800000u;
                }
#pragma unroll
                for (int j = 0; j < 16; j++) top = fmaxf(top, __uint_as_float(v[j]));
                tmem_st(s + h, v);
            }
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(small_read);
            top = fmaxf(top, other(top));
            const float m_new = fmaxf(m, top), alpha = m == -INFINITY ? 0.0f : sa_ex2(m - m_new);
            m = m_new;
            float l0 = 0.0f, l1 = 0.0f;
#pragma unroll 1
            for (uint32_t h = h0; h < h0 + 64; h += 16) {
                uint32_t x[16], v[16];
                tmem_ld(s + h, x);
                tmem_wait_ld(x);
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float p0 = sa_ex2(__uint_as_float(x[j]) - m), p1 = sa_ex2(__uint_as_float(x[j + 1]) - m);
                    l0 += p0; l1 += p1;
                    split2(p0 * fs[h + j].y, p1 * fs[h + j + 1].y, v[j / 2], v[8 + j / 2]);
                }
                tmem_st(s + h, v);
            }
            l = fmaf(l, alpha, l0 + l1);
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * (t & 1));
            if (t) add_output(t - 1);
            alpha_prev = alpha;
        }
        add_output(n_tiles - 1);
        l += other(l);
        if (!ok && lane == 0) { count_timeout(); atomicOr(lost, 1u); }
        // Outputs leave by whole rows, through the idle stages.
        const float unit = v_ref * (1.0f / 16384.0f);
        float4* const out = reinterpret_cast<float4*>(mem);
#pragma unroll
        for (int j = 0; j < OW; j += 4)
            out[row * (kSwCols / 4) + (((OW * part + j) / 4) ^ (row & 7))] = make_float4(o[j / 2].x * unit, o[j / 2].y * unit, o[j / 2 + 1].x * unit, o[j / 2 + 1].y * unit);
        bar_sync(1, kSwSoft);
        const bool gone = *reinterpret_cast<volatile uint32_t*>(lost);
        const uint32_t mine = rows[row];
        if (mine != 0xffffffffu && half == 0 && part == 0) { float* rec = sa_record(a, mine >> 10, mine & 1023, c.split); rec[0] = gone ? kBatchNaN : m * kLn2; rec[1] = gone ? kBatchNaN : l; }
        const uint32_t e = threadIdx.x % (kSwCols / 4);
        constexpr uint32_t kStep = kSwSoft / (kSwCols / 4);                 // rows at a time
#pragma unroll 1
        for (uint32_t r0 = threadIdx.x / (kSwCols / 4); r0 < 128; r0 += 8 * kStep) {
            uint32_t to[8];
            float4 y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) { to[i] = rows[r0 + kStep * i]; y[i] = out[(r0 + kStep * i) * (kSwCols / 4) + (e ^ ((r0 + kStep * i) & 7))]; }
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (to[i] != 0xffffffffu && 4 * e < cols)
                    *reinterpret_cast<float4*>(sa_record(a, to[i] >> 10, to[i] & 1023, c.split) + 4 + c0 + 4 * e) = gone ? make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN) : y[i];
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kSwSoft / 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(0u) : "memory");
}

// What decides a launch: queries a CTA of k_shared_rows holds (RQ), float4 a lane holds (NV), lanes that share a key (LK), shares of its keys; shares of the prefix
// on the tensor cores (0: k_shared_rows walks the prefix too).
// Rows x heads x prefix from which the two launches of k_shared_wide pay (16 heads of 576 and 512 dims, up to 256 keys of their own; us, on the tensor cores and in
// k_shared_rows alone): 16 rows, 256 keys 45.1 / 43.1, 512 keys 45.2 / 55.5, 4096 keys 53 / 230; 6 rows, 1024 keys 41.1 / 36.9; 2 rows, 8192 keys 57.4 / 69.7; 64 rows, 256 keys 74.0 / 88.1.
constexpr uint64_t kSwLeast = 1u << 17;
// The same for k_shared_prefix (32 heads over 8 key heads of 128, up to 512 keys of their own; us, with it and without): 8 rows, 512 keys 33 / 26, 1024 34.6 / 32, 2048 37 / 43,
// 8192 49 / 108; 32 rows, 64 keys 35 / 25, 256 36.8 / 32.8, 512 36 / 41, 1024 39 / 59; 128 rows, 64 keys 77 / 69, 256 84 / 94.  And from 32 query rows a key head on, since a quarter of
// a tile is still full then: 4 rows (16 query rows), 4096 keys 37 / 29, 8192 45 / 47; 2 rows, 4096 keys 36.6 / 36.9, 8192 45 / 57; 1 row, 8192 keys 37 / 29.  (So few rows over
// more keys would gain: the plain walk grows with rows and keys, this form with keys alone, and the rule does not weigh them against each other.)
constexpr uint64_t kSpLeast = 3u << 17;
struct SaShape { uint32_t RQ, NV, LK, chunks, splits, warps, shares, row_tiles, halves; bool records; };      // halves: of the output columns, of a head wider than 128 (0: k_shared_prefix)
SaShape sa_shape(const ZgSeqOp& s, bool wide) {
    const uint32_t B = s.n[0], G = s.n[2], rep = s.n[1] / G, dk = s.n[3], dv = s.n[4], dim = std::max(dk, dv), R = s.n[8], Rp = s.n[11], sms = zg_sm_count();
    SaShape p = {};
    p.NV = dim <= 512 ? 4 : dim <= 640 ? 5 : 8;
    p.LK = 1;
    while (p.LK * 4 * p.NV < dim) p.LK <<= 1;
    p.RQ = std::min(rep, p.NV == 8 ? 2u : 4u);
    p.chunks = (rep + p.RQ - 1) / p.RQ;
    const bool narrow = dim <= 128;
    if (wide && Rp && B * rep >= 32 && (uint64_t)B * s.n[1] * Rp >= (narrow ? kSpLeast : kSwLeast) && (narrow || (2ull * G * (Rp + 2 * kSwKeys) < 1u << 31))) {      // (rows of pairs are counted in 31 bits)
        // The number of shares that keeps the GPU busy with the fewest tiles of 64 (128) keys one after the other, and six tiles' (one tile's) time for each start and end.
        p.row_tiles = (B * rep + 127) / 128;
        p.halves = narrow ? 0 : (dv + kSwCols - 1) / kSwCols;
        const uint32_t items = p.row_tiles * G * std::max(1u, p.halves), tile = narrow ? 64 : kSwKeys, tiles = (Rp + tile - 1) / tile;
        uint64_t best = ~0ull;
        for (uint32_t n = 1; n <= std::min(tiles, 64u); n++) {
            const uint32_t keys = ((Rp + n - 1) / n + 15) / 16;
            const uint64_t cost = (uint64_t)((items * n + sms - 1) / sms) * (narrow ? keys + 24 : (keys + 7) / 8 + 1);
            if (cost < best) { best = cost; p.shares = n; }
        }
    }
    // Shares of at least 64 keys while the SMs are not covered several times over.  Up to eight of a row merge inside a cluster; beyond that, which only few rows over many
    // keys ask for, through records and a second launch.
    const uint32_t ctas = B * G * p.chunks, keys = R + (p.shares ? 0 : Rp), most = (keys + kSaShare - 1) / kSaShare;
    p.splits = std::max(1u, std::min({3 * sms / ctas, most, kSaCluster}));
    p.warps = ctas * p.splits >= sms || p.NV > 4 ? 4 : kSaMaxWarps;      // (eight warps' rings of the widest rows do not fit)
    if (!p.shares && 2 * ctas * kSaCluster < sms && most >= 4 * kSaCluster) { p.splits = std::min({(2 * sms + ctas - 1) / ctas, most / 2, 128u}); p.records = true; }
    return p;
}
// 16-byte loads of every operand, as far as sizes and offsets say so (buffers begin at 16 bytes at least)
bool sa_vec(const ZgSeqOp& s) {
    for (uint32_t x : {s.n[3], s.n[4], s.n[5], s.n[6], s.n[7], s.off[0], s.off[1], s.off[2]}) if (x % 4) return false;
    return s.buf[4] == ZG_NO_BUF || !(s.n[9] % 4 || s.n[10] % 4 || s.off[3] % 4 || s.off[4] % 4);
}
// rows of a prefix cache, boxes of 64 rows of one head
bool sa_encode(CUtensorMap* map, const float* base, uint64_t width, uint64_t rows, uint32_t dim) {
    const cuuint64_t dims[2] = {width, rows}, stride[1] = {width * 4};
    const cuuint32_t box[2] = {dim, kSpKeys}, one[2] = {1, 1};
    EncodeTiledFn fn = encode_tiled();
    if (!fn) { zg_set_error("cuTensorMapEncodeTiled entry point not available"); return false; }
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(base), dims, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { zg_set_error("cuTensorMapEncodeTiled(prefix) failed (%d)", (int)r); return false; }
    return true;
}
template <int NC, int DV>
bool sa_launch_prefix(const SaArgs& a, const SaShape& p, cudaStream_t st) {
    typedef SpLayout<NC, DV> L;
    CUtensorMap mk, mv;
    const uint64_t rows = (uint64_t)a.pslots * a.Rp;
    if (!sa_encode(&mk, a.kp - a.k_x, a.pkw, rows, a.dk) || !sa_encode(&mv, a.vp - a.v_x, a.pvw, rows, a.dv)) return false;
    if (!zg_smem_limit<k_shared_prefix<NC, DV>>(L::size)) return false;
    launch_pdl(k_shared_prefix<NC, DV>, dim3(p.row_tiles * a.shares * a.G), dim3(kSpThreads), L::size, st, a, mk, mv, p.row_tiles);
    return true;
}
// Where the pairs of k_shared_wide lie in the workspace, behind the records; `base` null: how many floats all of it takes
size_t sw_layout(const ZgSeqOp& s, const SaShape& p, float* base, uint32_t k_x, uint32_t v_x, SwArgs* w) {
    const uint32_t G = s.n[2], dk = s.n[3], dv = s.n[4];
    w->KR = (s.n[11] + 7) / 8 * 8 + kSwKeys; w->QR = p.row_tiles * 128;
    w->dkp = (dk + 63) / 64 * 64; w->dvp = (dv + 63) / 64 * 64;
    // the values of a latent: columns of the same rows, from a multiple of 16 bytes of pairs on
    w->latent = s.buf[4] == s.buf[5] && s.n[9] == s.n[10] && G == 1 && v_x >= k_x && v_x - k_x + dv <= dk && (v_x - k_x) % 8 == 0;
    w->v0 = w->latent ? v_x - k_x : 0;
    w->halves = p.halves; w->row_tiles = p.row_tiles;
    size_t at = ((size_t)s.n[0] * s.n[1] * p.shares * (4 + dv) + 255) & ~(size_t)255;
    auto place = [&](auto*& ptr, size_t floats) { ptr = base ? reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + at) : nullptr; at = (at + floats + 255) & ~(size_t)255; };
    place(w->q, (size_t)G * w->QR * w->dkp);                        // (two halves of 16 bits a value)
    place(w->k, (size_t)G * w->KR * w->dkp);
    place(w->v, w->latent ? 0 : (size_t)G * w->KR * w->dvp);
    place(w->qf, (size_t)G * w->QR); place(w->kf, (size_t)G * w->KR); place(w->vf, w->latent ? 0 : (size_t)G * w->KR);
    place(w->flags, (size_t)2 * G * w->KR / 8);
    return at;
}
bool sw_encode(CUtensorMap* map, const __half* base, uint64_t dims_, uint64_t rows) {
    const cuuint64_t dims[2] = {dims_, rows}, stride[1] = {dims_ * 2};
    const cuuint32_t box[2] = {64, 128}, one[2] = {1, 1};
    EncodeTiledFn fn = encode_tiled();
    if (!fn) { zg_set_error("cuTensorMapEncodeTiled entry point not available"); return false; }
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(base), dims, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { zg_set_error("cuTensorMapEncodeTiled(pairs) failed (%d)", (int)r); return false; }
    return true;
}
bool sa_launch_wide(const ZgOp& op, const SaArgs& a, const SwArgs& w, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    if (!sw_encode(&mq, w.q, w.dkp, 2ull * a.G * w.QR) || !sw_encode(&mk, w.k, w.dkp, 2ull * a.G * w.KR)) return false;
    if (!sw_encode(&mv, w.latent ? w.k : w.v, w.latent ? w.dkp : w.dvp, 2ull * a.G * w.KR)) return false;
    if (!zg_smem_limit<k_shared_wide>(kSwSmem)) return false;
    launch_pdl(k_shared_pairs, dim3(a.G * ((w.latent ? 1 : 2) * (w.KR / 8) + w.QR / 8)), dim3((std::max(w.dkp, w.dvp) / 4 + 31) / 32 * 32), 0, st, a, w);
    ZG_SEQ_CHECK();
    launch_pdl(k_shared_wide, dim3(w.row_tiles * w.halves * a.shares * a.G), dim3(kSwThreads), kSwSmem, st, a, w, mq, mk, mv);
    return true;
}
template <int RQ, int NV, bool VEC>
bool sa_launch_rows(const SaArgs& a, const SaShape& p, cudaStream_t st) {
    constexpr size_t limit = 200 * 1024;
    const uint32_t dvp = (a.dv + 3) / 4 * 4;
    const size_t smem = std::max<size_t>((size_t)p.warps * kSaRing * 4 * NV * 512, sizeof(float) * (p.warps * (32 / p.LK) + 1) * RQ * (4 + dvp));
    if (smem > limit) { zg_set_error("shared_attention: %zu bytes of shared memory", smem); return false; }
    if (!zg_smem_limit<k_shared_rows<RQ, NV, VEC>>(limit)) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits * a.B * a.G * p.chunks); cfg.blockDim = dim3(32 * p.warps); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_zg_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.records ? 1 : p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_shared_rows<RQ, NV, VEC>, a, p.chunks, p.LK);
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
    SwArgs w;
    if (p.halves) return sw_layout(s, p, nullptr, s.off[3], s.off[4], &w);
    return (size_t)s.n[0] * s.n[1] * (p.shares + (p.records ? p.splits : 0)) * (4 + s.n[4]);
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
    a.pslots = prefix ? std::min(slots(4, 5, (size_t)a.Rp * a.pkw, (size_t)a.Rp * a.pvw), 0x7fffffffu / a.Rp) : 0;      // (rows are counted in 31 bits)
    a.k_x = s.off[3]; a.v_x = s.off[4];
    a.table = bufs[s.buf[6]];
    a.sink = s.buf[7] == ZG_NO_BUF ? nullptr : a.sink_bf16 ? (const void*)wptr<bf16>(bufs, s.buf[7], s.off[5]) : (const void*)wptr<float>(bufs, s.buf[7], s.off[5]);
    a.scale = s.f[0]; a.cap = s.f[1];
    const bool vec = sa_vec(s);
    SaShape p = sa_shape(s, vec && scratch);
    if (p.records && !scratch) { p.records = false; p.splits = kSaCluster; }      // no room for records
    a.shares = p.shares; a.splits = p.splits;
    a.part = p.shares || p.records ? scratch : nullptr;
    if (a.shares && p.halves) {
        SwArgs w;
        sw_layout(s, p, scratch, a.k_x, a.v_x, &w);
        if (!sa_launch_wide(op, a, w, st)) return false;
        ZG_SEQ_CHECK();
    } else if (a.shares) {
        const bool k1 = a.dk <= 64, v1 = a.dv <= 64;
        if (!(k1 ? v1 ? sa_launch_prefix<1, 64>(a, p, st) : sa_launch_prefix<1, 128>(a, p, st) : v1 ? sa_launch_prefix<2, 64>(a, p, st) : sa_launch_prefix<2, 128>(a, p, st))) return false;
        ZG_SEQ_CHECK();
    }
    bool ok = false;
#define ZG_SA(NV_)                                                                       \
    switch (p.RQ) {                                                                      \
        case 1: ok = vec ? sa_launch_rows<1, NV_, true>(a, p, st) : sa_launch_rows<1, NV_, false>(a, p, st); break;                       \
        case 2: ok = vec ? sa_launch_rows<2, NV_, true>(a, p, st) : sa_launch_rows<2, NV_, false>(a, p, st); break;                       \
        case 3: ok = vec ? sa_launch_rows<3, NV_, true>(a, p, st) : sa_launch_rows<3, NV_, false>(a, p, st); break;                       \
        default: ok = vec ? sa_launch_rows<4, NV_, true>(a, p, st) : sa_launch_rows<4, NV_, false>(a, p, st); break;                      \
    }
    if (p.NV == 4) { ZG_SA(4); }
    else if (p.NV == 5) { ZG_SA(5); }
    else if (p.RQ == 1) ok = vec ? sa_launch_rows<1, 8, true>(a, p, st) : sa_launch_rows<1, 8, false>(a, p, st);
    else ok = vec ? sa_launch_rows<2, 8, true>(a, p, st) : sa_launch_rows<2, 8, false>(a, p, st);
#undef ZG_SA
    if (!ok) return false;
    ZG_SEQ_CHECK();
    if (p.records) {
        launch_pdl(k_shared_merge, dim3(a.B * a.H), dim3(256), 0, st, a);
        ZG_SEQ_CHECK();
    }
    return true;
}
unsigned int zg_shared_attention_timeouts() { return tc_timeouts(); }
