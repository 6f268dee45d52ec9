// Sequence-model DeviceOps of a step that advances many requests at once (parameter packs in include/zgml_cuda.h): BATCH_APPEND and LOGIT_RULES;
// SHARED_ATTENTION and ADAPTER_LINEAR have files of their own.  What distinguishes the rows - slot, length, adapter, rules - lies in a table that the host rewrites between
// executions of one captured program.
#include "batch_table.cuh"

#include <algorithm>

namespace {

// ── BATCH_APPEND ─────────────────────────────────────────────────────────────────────────────────────────────────────
struct BaArgs {
    float* cache; const float* src; const float* table; const float* freqs; float* turned;
    uint32_t B, cols, src_rs, src_col, width, cache_col, R, slots, key_heads, dim, turn_at, rot, halves, q_heads, q_col, dst_rs, dst_col;
    double base;
};
// CTA: one row.  The angle of a far position needs more bits than f32 has (position 100000 times a frequency near 1 is off by 4e-3 there): it is formed
// and reduced to a turn in 64 bits, once per pair for all heads, and only the remainder goes through f32 sine and cosine.
__global__ void __launch_bounds__(256) k_batch_append(BaArgs a) {
    pdl_enter();
    extern __shared__ float2 turn[];                                 // [rot / 2]: cosine, sine
    const uint32_t r = blockIdx.x;
    const BatchHead head = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    const bool ok = (uint32_t)w.slot < a.slots && (uint32_t)w.length <= a.R && head.prefix >= 0;
    for (uint32_t i = threadIdx.x; i < a.rot / 2; i += blockDim.x) {
        const double f = a.freqs ? (double)a.freqs[i] : exp(-2.0 * i / a.rot * log(a.base));
        const double x = ((double)head.prefix + w.length - 1) * f, two_pi = 6.283185307179586476925;
        float s, c;
        sincosf((float)(x - two_pi * rint(x / two_pi)), &s, &c);
        turn[i] = make_float2(c, s);
    }
    // Of rows that name the same place the last one stays, whatever order the CTAs run in.
    bool later = false;
    for (uint32_t i = r + 1 + threadIdx.x; i < head.rows; i += blockDim.x) {
        const BatchRow x = batch_row(a.table, i);
        later = later || (x.slot == w.slot && x.length == w.length);
    }
    later = __syncthreads_or(later);
    const float* src = a.src + (size_t)r * a.src_rs;
    // value j of a head that begins at p
    auto value = [&](const float* p, uint32_t j) {
        const uint32_t at = j - a.turn_at;
        if (at >= a.rot) return p[j];
        const uint32_t half = a.rot / 2, pair = a.halves ? (at < half ? at : at - half) : at >> 1, first = a.halves ? pair : 2 * pair, second = a.halves ? pair + half : 2 * pair + 1;
        const float x = p[a.turn_at + first], y = p[a.turn_at + second];
        const float2 t = turn[pair];
        return at == first ? x * t.x - y * t.y : x * t.y + y * t.x;
    };
    const uint32_t heads = a.key_heads * a.dim;
    if (ok && w.length > 0 && !later) {
        float* out = a.cache + ((size_t)w.slot * a.R + (w.length - 1)) * a.width + a.cache_col;
        const float* p = src + a.src_col;
        for (uint32_t c = threadIdx.x; c < a.cols; c += blockDim.x) out[c] = c < heads ? value(p + c / a.dim * a.dim, c % a.dim) : p[c];
    }
    if (a.q_heads) {
        float* out = a.turned + (size_t)r * a.dst_rs + a.dst_col;
        const float* p = src + a.q_col;
        for (uint32_t c = threadIdx.x; c < a.q_heads * a.dim; c += blockDim.x) out[c] = ok ? value(p + c / a.dim * a.dim, c % a.dim) : kBatchNaN;
    }
}

// ── LOGIT_RULES ──────────────────────────────────────────────────────────────────────────────────────────────────────
struct LrArgs {
    float* dst; const float* src; const float* table; const int32_t* history; const int2* bias; const uint32_t* masks;
    uint32_t B, V, src_rs, dst_rs, history_rows, slots, entries, mask_rows, slice;
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
constexpr uint32_t kLrSeen = 0x80000000u;
// CTA (slice of the vocabulary, row): counts of the slice's tokens in the row's history (bit 31: the token occurs at all), biases of the slice, then one pass over the logits
__global__ void __launch_bounds__(256) k_logit_rules(LrArgs a) {
    pdl_enter();
    extern __shared__ uint32_t counts[];                             // [slice] counts, [slice] biases
    float* const bias = reinterpret_cast<float*>(counts + a.slice);
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * a.slice, n = min(a.slice, a.V - v0);
    const BatchHead head = batch_head(a.table, a.B);
    const LrRow w = lr_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    const float* src = a.src + (size_t)r * a.src_rs + v0;
    float* dst = a.dst + (size_t)r * a.dst_rs + v0;
    const bool ok = (w.length == 0 || ((uint32_t)w.slot < a.slots && (uint32_t)w.length <= a.history_rows)) && w.first >= 0 && (w.mask < 0 || (uint32_t)w.mask < a.mask_rows) &&
                    (w.bias_count == 0 || (w.bias_count > 0 && w.bias_first >= 0 && (uint32_t)w.bias_first + (uint32_t)w.bias_count <= a.entries));
    if (!ok) {
        for (uint32_t i = threadIdx.x; i < n; i += 256) dst[i] = kBatchNaN;
        return;
    }
    for (uint32_t i = threadIdx.x; i < n; i += 256) { counts[i] = 0; bias[i] = 0.0f; }
    __syncthreads();
    const int32_t* past = a.history + (size_t)(w.length ? w.slot : 0) * a.history_rows;
    for (uint32_t i = threadIdx.x; i < (uint32_t)w.length; i += 256) {
        const uint32_t t = (uint32_t)past[i] - v0;                   // tokens outside the vocabulary belong to no slice
        if (t < n) { if (i >= (uint32_t)w.first) atomicAdd(counts + t, 1u); else atomicOr(counts + t, kLrSeen); }
    }
    // Entries in order, 32 at a time by one warp; those of one token are added by its first lane, so that a token named twice gets the same sum in every run.
    if (threadIdx.x < 32) {
        for (uint32_t i = 0; i < (uint32_t)w.bias_count; i += 32) {
            const bool on = i + threadIdx.x < (uint32_t)w.bias_count;
            const int2 e = on ? a.bias[(size_t)w.bias_first + i + threadIdx.x] : make_int2(-1, 0);
            const uint32_t t = (uint32_t)e.x - v0, mine = on && t < n ? t : 0xffffffffu;
            const uint32_t same = __match_any_sync(0xffffffffu, mine);
            float sum = 0.0f;
            for (uint32_t l = 0; l < 32; l++) {
                const float x = __shfl_sync(0xffffffffu, __int_as_float(e.y), l);
                if (same >> l & 1) sum += x;
            }
            if (mine != 0xffffffffu && __ffs(same) - 1 == (int)threadIdx.x) bias[t] += sum;
            __syncwarp();
        }
    }
    __syncthreads();
    const uint32_t* mask = w.mask >= 0 ? a.masks + (size_t)w.mask * ((a.V + 31) / 32) : nullptr;
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        float z = src[i];
        const uint32_t c = counts[i], made = c & ~kLrSeen;
        if (c) {
            z = z > 0.0f ? z / w.repetition : z * w.repetition;
            if (made) z = z - w.presence - w.frequency * (float)made;
        }
        z += bias[i];
        if (mask && !(mask[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1)) z = -INFINITY;
        dst[i] = z;
    }
}

}  // namespace

bool zg_batch_op_valid(const ZgOp& op, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    const ZgSeqOp& s = op.u.seq;
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    switch (op.tag) {
        case ZG_OP_BATCH_APPEND: {
            const size_t B = s.n[0], cols = s.n[1], srs = s.n[2], width = s.n[3], R = s.n[4], heads = s.n[5], dim = s.n[6], rot = s.n[8], q_heads = s.n[10];
            if (!B || !cols || B > 65536 || width < s.off[1] + cols || !R || R >= (1u << 31) || s.n[9] > 1) return fail("batch_append: shape");
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
            a.base = s.f[0];
            a.slots = (uint32_t)std::min<size_t>(elems[s.buf[0]] / ((size_t)a.R * a.width), (size_t)1 << 31);
            launch_pdl(k_batch_append, dim3(a.B), dim3(256), (a.rot / 2) * sizeof(float2), st, a);
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
            a.slice = 4096;
            launch_pdl(k_logit_rules, dim3((a.V + a.slice - 1) / a.slice, a.B), dim3(256), a.slice * 8, st, a);
            ZG_SEQ_CHECK();
            return true;
        }
        default: zg_set_error("not a sequence op"); return false;
    }
}
