// SHARED_ATTENTION (parameter pack in include/zgml_cuda.h): every row of a batch attends over the keys of one prefix that all rows share and over the
// keys of its own sequence, with one softmax over both.
//
// Softmax attention over a set of keys that falls into shares needs a record (m, l, o) per share: the largest score, the sum of exp(s - m) and the sum of
// exp(s - m) v.  Records of any shares merge into the whole: m = max m_i, l = sum l_i e^(m_i - m), o = sum o_i e^(m_i - m) / l.
#include "batch_table.cuh"

#include <algorithm>

namespace {

struct SaArgs {
    float* dst; const float* q; const float* kc; const float* vc; const float* kp; const float* vp; const float* table;
    const void* sink;
    float* part;                     // records [B, H, splits, 4 + dv]: m, l, -, -, o; null: a row's keys are one share
    uint32_t B, H, G, rep, dk, dv, q_rs, kw, vw, R, pkw, pvw, Rp, dst_rs, slots, pslots, sink_bf16, splits;
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
    const uint32_t n = k.prefix + k.own, share = (n + a.splits - 1) / a.splits, k0 = min(n, split * share), k1 = min(n, k0 + share);
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
        if (a.splits > 1) {
            float* mine = a.part + ((size_t)(r * a.H + h) * a.splits + split) * (4 + a.dv);
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
    const float* rec = a.part + (size_t)blockIdx.x * a.splits * (4 + a.dv);
    float top = -INFINITY;
    for (uint32_t s = 0; s < a.splits; s++) top = fmaxf(top, rec[(size_t)s * (4 + a.dv)]);
    float sum = 0.0f;
    for (uint32_t s = 0; s < a.splits; s++) sum = fmaf(rec[(size_t)s * (4 + a.dv) + 1], sa_weight(rec[(size_t)s * (4 + a.dv)], top), sum);
    if (a.sink && top != -INFINITY) sum += expf(sa_sink(a, h) - top);
    const float inv = k.bad ? kBatchNaN : top == -INFINITY ? 0.0f : 1.0f / sum;
    float* out = a.dst + (size_t)r * a.dst_rs + (size_t)h * a.dv;
    for (uint32_t d = threadIdx.x; d < a.dv; d += 128) {
        float v = 0.0f;
        for (uint32_t s = 0; s < a.splits; s++) v = fmaf(rec[(size_t)s * (4 + a.dv) + 4 + d], sa_weight(rec[(size_t)s * (4 + a.dv)], top), v);
        out[d] = v * inv;
    }
}

// What decides a launch: queries a CTA holds (RQ), float4 a lane holds (NV), lanes that share a key (LK), shares of the keys.
struct SaShape { uint32_t RQ, NV, LK, chunks, splits; };
SaShape sa_shape(const ZgSeqOp& s) {
    const uint32_t B = s.n[0], G = s.n[2], rep = s.n[1] / G, dim = std::max(s.n[3], s.n[4]), keys = s.n[8] + s.n[11];
    SaShape p;
    p.NV = dim <= 512 ? 4 : dim <= 640 ? 5 : 8;
    p.LK = 1;
    while (p.LK * 4 * p.NV < dim) p.LK <<= 1;
    p.RQ = std::min(rep, p.NV == 8 ? 2u : 4u);
    p.chunks = (rep + p.RQ - 1) / p.RQ;
    const uint32_t ctas = B * G * p.chunks;
    p.splits = std::max(1u, std::min({(8 * zg_sm_count() + ctas - 1) / ctas, (keys + 63) / 64, 128u}));
    return p;
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
    const SaShape p = sa_shape(s);
    return p.splits > 1 ? (size_t)s.n[0] * s.n[1] * p.splits * (4 + s.n[4]) : 0;
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
    const SaShape p = sa_shape(s);
    a.splits = scratch ? p.splits : 1;
    a.part = scratch;
    auto aligned = [](const float* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const bool vec = a.dk % 4 == 0 && a.dv % 4 == 0 && a.q_rs % 4 == 0 && a.kw % 4 == 0 && a.vw % 4 == 0 && a.pkw % 4 == 0 && a.pvw % 4 == 0 && aligned(a.q) && aligned(a.kc) && aligned(a.vc) &&
                     aligned(a.kp) && aligned(a.vp);
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
    if (a.splits > 1) {
        launch_pdl(k_shared_merge, dim3(a.B * a.H), dim3(128), 0, st, a);
        ZG_SEQ_CHECK();
    }
    return true;
}
