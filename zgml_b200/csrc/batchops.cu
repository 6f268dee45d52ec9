// Sequence-model DeviceOps of a step that advances many requests at once (parameter packs in include/zgml_cuda.h): BATCH_APPEND and LOGIT_RULES;
// SHARED_ATTENTION and ADAPTER_LINEAR have files of their own.  What distinguishes the rows - slot, length, adapter, rules - lies in a table that the host rewrites between
// executions of one captured program.
#include "batch_table.cuh"

#include <algorithm>
#include <cmath>

namespace {

// ── BATCH_APPEND ─────────────────────────────────────────────────────────────────────────────────────────────────────
struct BaArgs {
    float* cache; const float* src; const float* table; const float* freqs; float* turned;
    uint32_t B, cols, src_rs, src_col, width, cache_col, R, slots, key_heads, dim, turn_at, rot, halves, q_heads, q_col, dst_rs, dst_col;
    double ratio;                                                    // base^(-2 / rot)
};
// CTA (row, share of its values).  The angle of a far position needs more bits than f32 has (position 100000 times a frequency near 1 is off by 4e-3 there): it is formed
// and reduced to a turn in 64 bits, once per pair for all heads of the share, and only the remainder goes through f32 sine and cosine.  A frequency base^(-2i / rot) is
// the i-th power of a number from the host, by squaring: its rounding comes i times, so off by i 2^-53 of itself, and an angle by that much of itself (largest where i times
// the frequency is: behind 100000 positions 3e-11 for 128 values and base 10000).
// One row is bound by latency: with all of its 6144 values in one CTA and exp in 64 bits it took 4 us longer.
constexpr uint32_t kBaThreads = 256, kBaValues = 4;                  // values a thread
__global__ void __launch_bounds__(kBaThreads) k_batch_append(BaArgs a) {
    pdl_enter();
    extern __shared__ float2 turn[];                                 // [rot / 2]: cosine, sine
    const uint32_t r = blockIdx.x;
    const BatchHead head = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    const bool ok = (uint32_t)w.slot < a.slots && (uint32_t)w.length <= a.R && head.prefix >= 0;
    const uint32_t keys = a.key_heads * a.dim, all = a.cols + a.q_heads * a.dim, first = blockIdx.y * (kBaThreads * kBaValues) + threadIdx.x;
    const float* src = a.src + (size_t)r * a.src_rs;
    // values: first the appended columns, then the query heads.  What a value of a turned head becomes: x cos - y sin or y cos + x sin, with its partner
    float x[kBaValues], y[kBaValues];
    uint32_t pair[kBaValues];                                        // bit 31: the second of its pair; all bits: copied
#pragma unroll
    for (uint32_t i = 0; i < kBaValues; i++) {
        const uint32_t c = first + i * kBaThreads;
        x[i] = y[i] = 0.0f; pair[i] = 0xffffffffu;
        if (c >= all) continue;
        const uint32_t at = c < a.cols ? c : c - a.cols, in = at % a.dim - a.turn_at, half = a.rot / 2;
        const float* p = src + (c < a.cols ? a.src_col : a.q_col) + at;
        x[i] = *p;
        if ((c < a.cols && at >= keys) || in >= a.rot) continue;
        const bool second = a.halves ? in >= half : in & 1;
        const int partner = a.halves ? (second ? -(int)half : (int)half) : second ? -1 : 1;
        y[i] = p[partner];
        pair[i] = (a.halves ? (second ? in - half : in) : in >> 1) | (second ? 0x80000000u : 0u);
    }
    for (uint32_t i = threadIdx.x; i < a.rot / 2; i += kBaThreads) {
        double f = 1.0;
        if (a.freqs) f = (double)a.freqs[i];
        else {
            double power = a.ratio;
            for (uint32_t e = i; e; e >>= 1) { if (e & 1) f *= power; power *= power; }
        }
        const double angle = ((double)head.prefix + w.length - 1) * f, two_pi = 6.283185307179586476925;
        float s, c;
        sincosf((float)(angle - two_pi * rint(angle / two_pi)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    // Of rows that name the same place the last one stays, whatever order the CTAs run in.
    bool later = false;
    for (uint32_t i = r + 1 + threadIdx.x; i < head.rows; i += kBaThreads) {
        const BatchRow z = batch_row(a.table, i);
        later = later || (z.slot == w.slot && z.length == w.length);
    }
    later = __syncthreads_or(later);
    const bool append = ok && w.length > 0 && !later;
    float* const cache = a.cache + (append ? ((size_t)w.slot * a.R + (w.length - 1)) * a.width : 0) + a.cache_col;
    float* const turned = a.turned + (size_t)r * a.dst_rs + a.dst_col;
#pragma unroll
    for (uint32_t i = 0; i < kBaValues; i++) {
        const uint32_t c = first + i * kBaThreads;
        if (c >= all) continue;
        float v = x[i];
        if (pair[i] != 0xffffffffu) {
            const float2 t = turn[pair[i] & 0x7fffffffu];
            v = pair[i] >> 31 ? v * t.x + y[i] * t.y : v * t.x - y[i] * t.y;
        }
        if (c >= a.cols) turned[c - a.cols] = ok ? v : kBatchNaN;
        else if (append) cache[c] = v;
    }
}

// ── LOGIT_RULES ──────────────────────────────────────────────────────────────────────────────────────────────────────
struct LrArgs {
    float* dst; const float* src; const float* table; const int32_t* history; const int2* bias; const uint32_t* masks;
    uint32_t B, V, src_rs, dst_rs, history_rows, slots, entries, mask_rows;
};
struct LrRow { int32_t slot, length, first, mask, bias_first, bias_count; float repetition, presence, frequency; };
__device__ __forceinline__ LrRow lr_row(const float* table, uint32_t r) {
    const int4* p = reinterpret_cast<const int4*>(table + ZG_BATCH_ROWS + (size_t)ZG_RULE_WORDS * r);
    const int4 x = p[0], y = p[1], z = p[2];
    LrRow w;
    w.slot = x.x; w.length = x.y; w.first = x.z; w.mask = x.w; w.bias_first = y.x; w.bias_count = y.y;
    w.repetition = __int_as_float(y.z); w.presence = __int_as_float(y.w); w.frequency = __int_as_float(z.x);
    return w;
}
constexpr uint32_t kLrThreads = 256;
// CTA (row, slice of the vocabulary): counts of the slice's tokens in the row's history (a half word for those before `first`, one for those from there on; LONG: bit 31 for
// the former, where a history may hold more than 65535 words) and biases of the slice in shared memory, then the
// logits, which were asked for at the start: a thread holds NV times four neighbours.  A history is read once per slice (from L2), which costs less than counts of a whole
// vocabulary in memory: 64 rows over 128256 tokens with 4096 words each read 33 MB for it beside the 66 MB of logits.
template <int NV, bool VEC, bool LONG>
__global__ void __launch_bounds__(kLrThreads, 6) k_logit_rules(LrArgs a) {
    pdl_enter();
    extern __shared__ uint4 lr_mem[];                                // [slice] counts, [slice] biases
    constexpr uint32_t slice = kLrThreads * 4 * NV;
    uint32_t* const counts = reinterpret_cast<uint32_t*>(lr_mem);
    float* const bias = reinterpret_cast<float*>(counts + slice);
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * slice, n = min(slice, a.V - v0);
    const BatchHead head = batch_head(a.table, a.B);
    const LrRow w = lr_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    const float* src = a.src + (size_t)r * a.src_rs + v0;
    float* dst = a.dst + (size_t)r * a.dst_rs + v0;
    float4 z[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t t = 4 * (threadIdx.x + kLrThreads * i);
        z[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (VEC && t + 4 <= n) z[i] = *reinterpret_cast<const float4*>(src + t);
        else { if (t < n) z[i].x = src[t]; if (t + 1 < n) z[i].y = src[t + 1]; if (t + 2 < n) z[i].z = src[t + 2]; if (t + 3 < n) z[i].w = src[t + 3]; }
    }
    const bool ok = (w.length == 0 || ((uint32_t)w.slot < a.slots && (uint32_t)w.length <= a.history_rows)) && w.first >= 0 && (w.mask < 0 || (uint32_t)w.mask < a.mask_rows) &&
                    (w.bias_count == 0 || (w.bias_count > 0 && w.bias_first >= 0 && (uint32_t)w.bias_first + (uint32_t)w.bias_count <= a.entries));
    const bool counted = ok && w.length > 0, biased = ok && w.bias_count > 0;
    // (a mask word serves 8 threads' tokens; a row of words begins anywhere)
    const uint32_t* mask = ok && w.mask >= 0 ? a.masks + (size_t)w.mask * ((a.V + 31) / 32) + v0 / 32 : nullptr;
    uint32_t allowed[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t t = 4 * (threadIdx.x + kLrThreads * i);
        allowed[i] = mask && t < n ? mask[t / 32] >> (t & 31) : 0xfu;
    }
    if (counted || biased) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            lr_mem[threadIdx.x + kLrThreads * i] = make_uint4(0, 0, 0, 0);
            if (biased) lr_mem[slice / 4 + threadIdx.x + kLrThreads * i] = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        if (counted) {
            const int32_t* past = a.history + (size_t)w.slot * a.history_rows;
            auto count = [&](int32_t token, uint32_t i) {
                const uint32_t t = (uint32_t)token - v0;             // tokens outside the vocabulary belong to no slice
                if (t >= n) return;
                if constexpr (LONG) { if (i >= (uint32_t)w.first) atomicAdd(counts + t, 1u); else atomicOr(counts + t, 0x80000000u); }
                else atomicAdd(counts + t, i >= (uint32_t)w.first ? 1u : 0x10000u);
            };
            const uint32_t length = w.length, lead = min(length, (4u - ((uint32_t)(reinterpret_cast<uintptr_t>(past) >> 2) & 3u)) & 3u), body = (length - lead) / 4;
            if (threadIdx.x < lead) count(past[threadIdx.x], threadIdx.x);
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < body; i += kLrThreads) {
                const int4 x = *reinterpret_cast<const int4*>(past + lead + 4 * i);
                const uint32_t at = lead + 4 * i;
                count(x.x, at); count(x.y, at + 1); count(x.z, at + 2); count(x.w, at + 3);
            }
            if (lead + 4 * body + threadIdx.x < length) count(past[lead + 4 * body + threadIdx.x], lead + 4 * body + threadIdx.x);
        }
        // Entries in order, 32 at a time by one warp; where a token is named twice among them its first lane adds them up, so that every run gives the same sum.
        if (biased && threadIdx.x >= kLrThreads - 32) {
            const uint32_t lane = threadIdx.x & 31;
            for (uint32_t i = 0; i < (uint32_t)w.bias_count; i += 32) {
                const bool on = i + lane < (uint32_t)w.bias_count;
                const int2 e = on ? a.bias[(size_t)w.bias_first + i + lane] : make_int2(-1, 0);
                const uint32_t t = (uint32_t)e.x - v0, mine = on && t < n ? t : 0xffffffffu;
                if (!__any_sync(0xffffffffu, mine != 0xffffffffu)) continue;
                const uint32_t same = __match_any_sync(0xffffffffu, mine);
                float sum = __int_as_float(e.y);
                if (__any_sync(0xffffffffu, mine != 0xffffffffu && (same & (same - 1)))) {
                    sum = 0.0f;
                    for (uint32_t l = 0; l < 32; l++) {
                        const float x = __shfl_sync(0xffffffffu, __int_as_float(e.y), l);
                        if (same >> l & 1) sum += x;
                    }
                }
                if (mine != 0xffffffffu && __ffs(same) - 1 == (int)lane) bias[t] += sum;
                __syncwarp();
            }
        }
        __syncthreads();
    }
    auto rule = [&](float v, uint32_t c) {
        if (!c) return v;
        const uint32_t made = c & (LONG ? 0x7fffffffu : 0xffffu);
        v = v > 0.0f ? v / w.repetition : v * w.repetition;
        return made ? v - w.presence - w.frequency * (float)made : v;
    };
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const uint32_t t = 4 * (threadIdx.x + kLrThreads * i);
        if (t >= n) break;
        float4 v = z[i];
        if (counted) {
            const uint4 c = lr_mem[threadIdx.x + kLrThreads * i];
            v.x = rule(v.x, c.x); v.y = rule(v.y, c.y); v.z = rule(v.z, c.z); v.w = rule(v.w, c.w);
        }
        if (biased) {
            const float4 b = reinterpret_cast<const float4*>(lr_mem)[slice / 4 + threadIdx.x + kLrThreads * i];
            v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
        }
        if (!(allowed[i] & 1)) v.x = -INFINITY;
        if (!(allowed[i] & 2)) v.y = -INFINITY;
        if (!(allowed[i] & 4)) v.z = -INFINITY;
        if (!(allowed[i] & 8)) v.w = -INFINITY;
        if (!ok) v = make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN);
        if (VEC && t + 4 <= n) *reinterpret_cast<float4*>(dst + t) = v;
        else { dst[t] = v.x; if (t + 1 < n) dst[t + 1] = v.y; if (t + 2 < n) dst[t + 2] = v.z; if (t + 3 < n) dst[t + 3] = v.w; }
    }
}

}  // namespace

// As much shared memory as an SM has: six CTAs of 32 KB, once per kernel and device.
template <auto KERNEL>
static bool lr_carveout() {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && (done.load() >> dev & 1)) return true;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e != cudaSuccess) { zg_set_error("cudaFuncSetAttribute(shared memory carveout) failed: %s", cudaGetErrorString(e)); return false; }
    if (dev < 64) done.fetch_or(1ull << dev);
    return true;
}
bool zg_batch_op_valid(const ZgOp& op, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    const ZgSeqOp& s = op.u.seq;
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    switch (op.tag) {
        case ZG_OP_BATCH_APPEND: {
            const size_t B = s.n[0], cols = s.n[1], srs = s.n[2], width = s.n[3], R = s.n[4], heads = s.n[5], dim = s.n[6], rot = s.n[8], q_heads = s.n[10];
            if (!B || !cols || B > 65536 || width < s.off[1] + cols || !R || R >= (1u << 31) || s.n[9] > 1) return fail("batch_append: shape");
            if (cols > (1u << 24) || q_heads > 65536 || dim > 65536 || q_heads * dim > (1u << 24)) return fail("batch_append: width");
            if ((heads || q_heads) && !dim) return fail("batch_append: head size");
            if (heads * dim > cols || rot % 2 || rot > 2048 || (rot && (s.n[7] + rot > dim || (s.buf[3] == ZG_NO_BUF && !(s.f[0] > 0.0f && s.f[0] - s.f[0] == 0.0f))))) return fail("batch_append: turned heads");
            if (rot && s.buf[3] != ZG_NO_BUF && !fits(3, s.off[4], rot / 2)) return fail("batch_append: frequency table");
            if ((B > 1 && srs < s.off[0] + cols) || !fits(1, s.off[0], (B - 1) * srs + cols) || !fits(0, 0, R * width) || !fits(2, 0, ZG_BATCH_ROWS + 4 * B)) return fail("batch_append: extent");
            if (q_heads) {
                const size_t n = q_heads * dim;
                if ((B > 1 && srs < s.off[2] + n) || !fits(1, s.off[2], (B - 1) * srs + n) || (B > 1 && s.n[11] < s.off[3] + n) || !fits(4, s.off[3], (B - 1) * (size_t)s.n[11] + n)) return fail("batch_append: query heads");
                if (s.buf[4] == s.buf[0] || s.buf[4] == s.buf[1] || s.buf[4] == s.buf[2] || s.buf[4] == s.buf[3]) return fail("batch_append: in place");
            }
            if (s.buf[0] == s.buf[1] || s.buf[0] == s.buf[2] || s.buf[0] == s.buf[3]) return fail("batch_append: in place");
            return true;
        }
        case ZG_OP_SHARED_ATTENTION: return zg_shared_attention_valid(s, elems, n_bufs, why, why_n);
        case ZG_OP_ADAPTER_LINEAR: return zg_adapter_linear_valid(s, elems, n_bufs, why, why_n);
        case ZG_OP_LOGIT_RULES: {
            const size_t B = s.n[0], V = s.n[1], srs = s.n[2], drs = s.n[3], Rh = s.n[4];
            if (!B || !V || B > 65535 || V >= (1u << 31) || Rh >= (1u << 31)) return fail("logit_rules: shape");
            if ((B > 1 && (srs < V || drs < V)) || !fits(0, s.off[0], (B - 1) * drs + V) || !fits(1, s.off[1], (B - 1) * srs + V)) return fail("logit_rules: rows");
            if (!fits(2, 0, ZG_BATCH_ROWS + ZG_RULE_WORDS * B)) return fail("logit_rules: table");
            if ((s.buf[3] != ZG_NO_BUF) != (Rh > 0) || (Rh && !fits(3, 0, Rh))) return fail("logit_rules: history");
            if (s.buf[4] != ZG_NO_BUF && !fits(4, 0, 2)) return fail("logit_rules: biases");
            if (s.buf[5] != ZG_NO_BUF && !fits(5, 0, (V + 31) / 32)) return fail("logit_rules: masks");
            for (int i = 2; i < 6; i++) if (s.buf[0] == s.buf[i]) return fail("logit_rules: in place");
            if (s.buf[0] == s.buf[1] && (s.off[0] != s.off[1] || srs != drs)) return fail("logit_rules: logits that overlap the destination have to be the destination");
            return true;
        }
        default: return fail("not a sequence op");
    }
}
uint32_t zg_batch_op_writes(uint32_t tag) { return tag == ZG_OP_BATCH_APPEND ? 1u | (1u << 4) : 1u; }      // the cache and the turned query heads
size_t zg_batch_op_scratch_elems(const ZgOp& op) {
    return op.tag == ZG_OP_SHARED_ATTENTION ? zg_shared_attention_scratch_elems(op.u.seq) : op.tag == ZG_OP_ADAPTER_LINEAR ? zg_adapter_linear_scratch_elems(op.u.seq) : 0;
}

bool zg_launch_batch_op(const ZgOp& op, float* const* bufs, const size_t* elems, float* scratch, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    switch (op.tag) {
        case ZG_OP_BATCH_APPEND: {
            BaArgs a;
            a.cache = bufs[s.buf[0]]; a.src = bufs[s.buf[1]]; a.table = bufs[s.buf[2]];
            a.B = s.n[0]; a.cols = s.n[1]; a.src_rs = s.n[2]; a.src_col = s.off[0]; a.width = s.n[3]; a.cache_col = s.off[1]; a.R = s.n[4];
            a.rot = s.n[8]; a.key_heads = a.rot ? s.n[5] : 0; a.dim = s.n[6] ? s.n[6] : 1; a.turn_at = s.n[7]; a.halves = s.n[9];
            a.q_heads = s.n[10]; a.q_col = s.off[2]; a.dst_rs = s.n[11]; a.dst_col = s.off[3];
            a.freqs = a.rot && s.buf[3] != ZG_NO_BUF ? bufs[s.buf[3]] + s.off[4] : nullptr;
            a.turned = a.q_heads ? bufs[s.buf[4]] : nullptr;
            a.ratio = a.rot && !a.freqs ? std::pow((double)s.f[0], -2.0 / a.rot) : 1.0;
            a.slots = (uint32_t)std::min<size_t>(elems[s.buf[0]] / ((size_t)a.R * a.width), (size_t)1 << 31);
            const uint32_t share = kBaThreads * kBaValues;
            launch_pdl(k_batch_append, dim3(a.B, (a.cols + a.q_heads * a.dim + share - 1) / share), dim3(kBaThreads), (a.rot / 2) * sizeof(float2), st, a);
            ZG_SEQ_CHECK();
            return true;
        }
        case ZG_OP_SHARED_ATTENTION: return zg_launch_shared_attention(op, bufs, elems, scratch, st);
        case ZG_OP_ADAPTER_LINEAR: return zg_launch_adapter_linear(op, bufs, scratch, st);
        case ZG_OP_LOGIT_RULES: {
            LrArgs a;
            a.dst = bufs[s.buf[0]] + s.off[0]; a.src = bufs[s.buf[1]] + s.off[1]; a.table = bufs[s.buf[2]];
            a.B = s.n[0]; a.V = s.n[1]; a.src_rs = s.n[2]; a.dst_rs = s.n[3]; a.history_rows = s.n[4];
            auto given = [&](int i) { return s.buf[i] != ZG_NO_BUF; };
            a.history = given(3) ? reinterpret_cast<const int32_t*>(bufs[s.buf[3]]) : nullptr;
            a.bias = given(4) ? reinterpret_cast<const int2*>(bufs[s.buf[4]]) : nullptr;
            a.masks = given(5) ? reinterpret_cast<const uint32_t*>(bufs[s.buf[5]]) : nullptr;
            a.slots = given(3) ? (uint32_t)std::min<size_t>(elems[s.buf[3]] / a.history_rows, (size_t)1 << 31) : 0;
            a.entries = given(4) ? (uint32_t)std::min<size_t>(elems[s.buf[4]] / 2, (size_t)1 << 31) : 0;
            a.mask_rows = given(5) ? (uint32_t)std::min<size_t>(elems[s.buf[5]] / ((a.V + 31) / 32), (size_t)1 << 31) : 0;
            // Slices of 4096 tokens where they fill the GPU, of 1024 where they do not.  128256 tokens, 4096 words of history, us with either: 4 rows 8.3 / 6.2, 8 rows 9.1 / 8.3,
            // 12 rows 10.3 / 10.3, 24 rows 10.3 / 14.8, 64 rows 20.6 / 32.8.  (Of 8192 tokens: 64 rows 22.6.)
            const bool vec = a.src_rs % 4 == 0 && a.dst_rs % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst)) & 15) == 0;
            const bool large = a.history_rows >= 65536 || (uint64_t)a.B * ((a.V + 4095) / 4096) >= 2 * zg_sm_count();
            const uint32_t slice = large ? 4096 : 1024;
            const dim3 grid((a.V + slice - 1) / slice, a.B);
            const size_t smem = slice * (a.bias ? 8 : 4);
#define ZG_RULES(NV_, VEC_, LONG_)                                                                                                     \
    do {                                                                                                                               \
        if (!lr_carveout<k_logit_rules<NV_, VEC_, LONG_>>()) return false;                                                             \
        launch_pdl(k_logit_rules<NV_, VEC_, LONG_>, grid, dim3(kLrThreads), smem, st, a);                                              \
    } while (0)
            if (a.history_rows >= 65536) { if (vec) ZG_RULES(4, true, true); else ZG_RULES(4, false, true); }
            else if (large) { if (vec) ZG_RULES(4, true, false); else ZG_RULES(4, false, false); }
            else if (vec) ZG_RULES(1, true, false);
            else ZG_RULES(1, false, false);
#undef ZG_RULES
            ZG_SEQ_CHECK();
            return true;
        }
        default: zg_set_error("not a sequence op"); return false;
    }
}
