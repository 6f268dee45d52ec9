// Sequence-model DeviceOps over paged caches in 8 bits (parameter packs in include/zgml_cuda.h): PAGE_APPEND, PAGE_READ and PAGE_COPY; PAGED_ATTENTION has a file of its own.
#include "pages.cuh"

#include <algorithm>
#include <cmath>

namespace {

// ── PAGE_APPEND ──────────────────────────────────────────────────────────────────────────────────────────────────────
constexpr uint32_t kPaThreads = 256, kPaQueries = 1024, kPaPairs = 128;      // query values a CTA; pairs of a head
struct PaArgs {
    PagePool pool; PageShape s;
    uint8_t* pages; const float* src; const float* table; float* turned; const float* freqs;
    uint32_t B, src_rs, k_col, v_col, q_col, q_heads, dst_rs, turn_at, rot, halves;
    double freq[kPaPairs];                                           // base^(-2i / rot), where no table of frequencies is given
};
// Cosine and sine of a position's turn.  Everything up to the turned value is in 64 bits, and that is rounded once: a code is a turned value over its scale, rounded, and an
// error of f32's size would now and then make it its neighbour, an error of a hundredth of a head's largest value.
__device__ __forceinline__ void pa_turn(const PaArgs& a, double position, uint32_t i, double* sin_, double* cos_) {
    const double angle = position * (a.freqs ? (double)a.freqs[i] : a.freq[i]), turns = rint(angle * 0.15915494309189533577);
    sincos(fma(-turns, 2.449293598294706e-16, fma(-turns, 6.283185307179586232, angle)), sin_, cos_);      // (two parts of 2 pi: 106 bits)
}
// what a scale has to be at least: the smallest power of two (2^-126 at least) of which 127 times reach the value whose bits are given; NaN where that is not finite
__device__ __forceinline__ float pa_scale(uint32_t bits) {
    if (bits >= 0x7f800000u) return kBatchNaN;
    int e = (int)(bits >> 23) - 127;                                 // (what is below 2^-119 has the smallest scale in any case)
    e = (bits & 0x7fffffu) > 0x7e0000u ? e - 5 : e - 6;              // 127 / 64 = 1.984375
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}
__device__ __forceinline__ uint32_t pa_code(float x, float inv) { return (uint32_t)(int)(rintf(x * inv) + 128.0f); }

// CTA (row, key head | share of the query heads).  The first of a step's rows that join a page owns it: it finds the others in the table (the last of several at one place
// counts), and no other CTA touches the page's part of its head, so no order of CTAs changes anything.
__global__ void __launch_bounds__(kPaThreads) k_page_append(const __grid_constant__ PaArgs a) {
    pdl_enter();
    extern __shared__ float4 pa_mem[];
    __shared__ int32_t joined[64];                                   // row that brings token t of the page, or -1
    __shared__ uint32_t list[64];                                    // tokens that come, in order
    __shared__ uint32_t most[2];
    __shared__ double2 turn[kPaPairs];
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const PageShape& s = a.s;
    const BatchHead head = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    bool ok = page_row_ok(a.pool, s, w) && head.prefix >= 0;
    const uint32_t place = ok && w.length > 0 ? (uint32_t)w.length - 1 : 0;
    const int32_t id = ok && w.length > 0 ? page_id(a.pool, w.slot, place >> s.shift) : 0;
    ok = ok && id >= 0;
    if (blockIdx.y >= s.G) {                                         // query heads
        const uint32_t first = (blockIdx.y - s.G) * kPaQueries, n = a.q_heads * s.dk, half = a.rot / 2;
        const float* src = a.src + (size_t)r * a.src_rs + a.q_col;
        float* dst = a.turned + (size_t)r * a.dst_rs;
        if (ok)
            for (uint32_t i = tid; i < half; i += kPaThreads) pa_turn(a, (double)head.prefix + w.length - 1, i, &turn[i].y, &turn[i].x);
        __syncthreads();
        for (uint32_t c = first + tid; c < min(first + kPaQueries, n); c += kPaThreads) {
            const uint32_t in = c % s.dk - a.turn_at;
            float v = src[c];
            if (in < a.rot) {
                const bool second = a.halves ? in >= half : in & 1;
                const float other = src[(int)c + (a.halves ? (second ? -(int)half : (int)half) : second ? -1 : 1)];
                const double2 t = turn[a.halves ? (second ? in - half : in) : in >> 1];
                v = (float)(second ? (double)v * t.x + (double)other * t.y : (double)v * t.x - (double)other * t.y);
            }
            dst[c] = ok ? v : kBatchNaN;
        }
        return;
    }
    if (!ok || w.length == 0) return;
    // the rows that join this page
    if (tid < 64) joined[tid] = -1;
    if (tid < 2) most[tid] = 0;
    __syncthreads();
    bool earlier = false;
    for (uint32_t i = tid; i < head.rows; i += kPaThreads) {
        const BatchRow z = batch_row(a.table, i);
        if (z.slot != w.slot || z.length <= 0 || (uint32_t)(z.length - 1) >> s.shift != place >> s.shift) continue;
        if (i < r) earlier = true;
        else atomicMax(&joined[(z.length - 1) & (s.page - 1)], (int)i);
    }
    if (__syncthreads_or(earlier)) return;
    if (tid < 32) {
        uint32_t n = 0;
        for (uint32_t t = 0; t < s.page; t += 32) {
            const bool here = t + tid < s.page && joined[t + tid] >= 0;
            const uint32_t all = __ballot_sync(0xffffffffu, here);
            if (here) list[n + __popc(all & ((1u << tid) - 1))] = t + tid;
            n += __popc(all);
        }
        if (tid == 0) most[0] = n;
    }
    __syncthreads();
    const uint32_t n = most[0], g = blockIdx.y, width = s.dk + s.dv, half = a.rot / 2;
    __syncthreads();
    if (tid == 0) most[0] = 0;
    __syncthreads();
    float* const tile = reinterpret_cast<float*>(pa_mem);             // [tokens that come][keys | values]
    uint32_t top[2] = {0, 0};
    // turned pairs, the other keys, and values
    for (uint32_t x = tid; x < n * half; x += kPaThreads) {
        const uint32_t m = x / half, i = x - m * half, t = list[m], p = a.turn_at + (a.halves ? i : 2 * i), q = p + (a.halves ? half : 1);
        const float* src = a.src + (size_t)joined[t] * a.src_rs + a.k_col + g * s.dk;
        double sin_, cos_;
        pa_turn(a, (double)head.prefix + ((place & ~(s.page - 1)) + t), i, &sin_, &cos_);
        const double u = src[p], v = src[q];
        const float y0 = (float)(u * cos_ - v * sin_), y1 = (float)(u * sin_ + v * cos_);
        tile[m * width + p] = y0; tile[m * width + q] = y1;
        top[0] = max(top[0], max(__float_as_uint(fabsf(y0)), __float_as_uint(fabsf(y1))));
    }
    for (uint32_t x = tid; x < n * width; x += kPaThreads) {
        const uint32_t m = x / width, c = x - m * width;
        if (c < s.dk && c - a.turn_at < a.rot) continue;
        const float v = a.src[(size_t)joined[list[m]] * a.src_rs + (c < s.dk ? a.k_col + g * s.dk + c : a.v_col + g * s.dv + c - s.dk)];
        tile[x] = v;
        top[c >= s.dk] = max(top[c >= s.dk], __float_as_uint(fabsf(v)));
    }
    for (int i = 0; i < 2; i++) {
        top[i] = __reduce_max_sync(0xffffffffu, top[i]);
        if ((tid & 31) == 0) atomicMax(&most[i], top[i]);
    }
    __syncthreads();
    uint8_t* const part = a.pages + (size_t)id * page_bytes(s) + (size_t)g * s.head;
    const bool fresh = joined[0] >= 0;
    float inv[2];
    float2 before = *reinterpret_cast<const float2*>(part), after;
    if (fresh) before = make_float2(0.0f, 0.0f);
    after.x = pa_scale(most[0]); after.y = pa_scale(most[1]);
    after.x = before.x != before.x ? before.x : after.x < before.x ? before.x : after.x;      // (a scale that is not a number stays until the page begins anew)
    after.y = before.y != before.y ? before.y : after.y < before.y ? before.y : after.y;
    inv[0] = 1.0f / after.x; inv[1] = 1.0f / after.y;
    // codes that the page has, in multiples of a larger scale
    for (int i = 0; i < 2; i++) {
        const float ratio = (i ? before.y : before.x) * inv[i];
        if (fresh || !(ratio < 1.0f)) continue;
        uint32_t* codes = reinterpret_cast<uint32_t*>(part + kPageHead + (i ? s.page * s.kp : 0));
        for (uint32_t x = tid; x < s.page * (i ? s.vp : s.kp) / 4; x += kPaThreads) {
            const uint32_t c = codes[x];
            uint32_t o = 0;
#pragma unroll
            for (int b = 0; b < 32; b += 8) o |= pa_code((float)(c >> b & 255) - 128.0f, ratio) << b;
            codes[x] = o;
        }
    }
    __syncthreads();
    if (tid == 0) *reinterpret_cast<float2*>(part) = after;
    if (after.x == after.x)
        for (uint32_t x = tid; x < n * s.dk; x += kPaThreads) {
            const uint32_t m = x / s.dk, c = x - m * s.dk;
            part[key_byte(s, list[m], c)] = (uint8_t)pa_code(tile[m * width + c], inv[0]);
        }
    if (after.y == after.y)
        for (uint32_t x = tid; x < n * s.dv; x += kPaThreads) {
            const uint32_t m = x / s.dv, c = x - m * s.dv;
            part[value_byte(s, list[m], c)] = (uint8_t)pa_code(tile[m * width + s.dk + c], inv[1]);
        }
}

// ── PAGE_READ ────────────────────────────────────────────────────────────────────────────────────────────────────────
struct PrArgs {
    PagePool pool; PageShape s;
    const float* table; float* dst;
    uint32_t B, dst_rs, k_col, v_col;
};
constexpr uint32_t kPrThreads = 256, kPrRows = 16;
// CTA (16 rows, key head)
__global__ void __launch_bounds__(kPrThreads) k_page_read(const PrArgs a) {
    pdl_enter();
    const PageShape& s = a.s;
    const BatchHead head = batch_head(a.table, a.B);
    const uint32_t first = blockIdx.x * kPrRows, g = blockIdx.y, width = s.dk + s.dv;
    for (uint32_t x = threadIdx.x; x < kPrRows * width; x += kPrThreads) {
        const uint32_t m = x / width, c = x - m * width, r = first + m;
        if (r >= head.rows) return;
        const BatchRow w = batch_row(a.table, r);
        if (w.slot < 0) continue;
        float v = kBatchNaN;
        if (page_row_ok(a.pool, s, w)) {
            v = 0.0f;
            if (w.length > 0) {
                const uint32_t place = w.length - 1, t = place & (s.page - 1);
                const int32_t id = page_id(a.pool, w.slot, place >> s.shift);
                const uint8_t* part = a.pool.pages + (size_t)max(id, 0) * page_bytes(s) + (size_t)g * s.head;
                const float2 scale = *reinterpret_cast<const float2*>(part);
                const uint8_t code = part[c < s.dk ? key_byte(s, t, c) : value_byte(s, t, c - s.dk)];
                v = id < 0 ? kBatchNaN : ((float)code - 128.0f) * (c < s.dk ? scale.x : scale.y);
            }
        }
        a.dst[(size_t)r * a.dst_rs + (c < s.dk ? a.k_col + g * s.dk + c : a.v_col + g * s.dv + c - s.dk)] = v;
    }
}

// ── PAGE_COPY ────────────────────────────────────────────────────────────────────────────────────────────────────────
constexpr uint32_t kPcThreads = 256, kPcVectors = 4;                 // vectors of 16 bytes a thread
// CTA (move, share of the page): bound by the reads and writes.  VEC: pages of whole vectors
template <typename V>
__global__ void __launch_bounds__(kPcThreads) k_page_copy(V* pages, const float* table, uint32_t B, uint32_t count, uint32_t vectors) {
    pdl_enter();
    const uint32_t m = blockIdx.x, first = blockIdx.y * (kPcThreads * kPcVectors) + threadIdx.x;
    const BatchHead head = batch_head(table, B);
    const int4 w = *reinterpret_cast<const int4*>(table + ZG_BATCH_ROWS + (size_t)4 * m);
    if (m >= head.rows || (uint32_t)w.x >= count || (uint32_t)w.y >= count || w.x == w.y) return;
    const V* from = pages + (size_t)w.x * vectors;
    V* to = pages + (size_t)w.y * vectors;
    V v[kPcVectors];
#pragma unroll
    for (uint32_t i = 0; i < kPcVectors; i++) if (first + i * kPcThreads < vectors) v[i] = from[first + i * kPcThreads];
#pragma unroll
    for (uint32_t i = 0; i < kPcVectors; i++) if (first + i * kPcThreads < vectors) to[first + i * kPcThreads] = v[i];
}

}  // namespace

bool zg_page_op_valid(const ZgOp& op, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    const ZgSeqOp& s = op.u.seq;
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    switch (op.tag) {
        case ZG_OP_PAGE_APPEND: {
            const size_t B = s.n[0], G = s.n[1], dk = s.n[2], dv = s.n[3], srs = s.n[4], page = s.n[5], most = s.n[6], at = s.n[7], rot = s.n[8], qh = s.n[10], trs = s.n[11];
            if (!B || B > 65536 || !page_shape_ok(G, dk, dv, page) || !most || most >= (1u << 25) || s.n[9] > 1 || qh > 65536) return fail("page_append: shape");
            if (rot % 2 || at + rot > dk || (rot && s.buf[4] == ZG_NO_BUF && !(s.f[0] > 0.0f && s.f[0] - s.f[0] == 0.0f))) return fail("page_append: turned values");
            if (rot && s.buf[4] != ZG_NO_BUF && !fits(4, s.off[4], rot / 2)) return fail("page_append: frequency table");
            const size_t end = std::max<size_t>(std::max<size_t>(s.off[0] + G * dk, s.off[1] + G * dv), qh ? s.off[2] + qh * dk : 0);
            if ((B > 1 && srs < end) || !fits(1, 0, (B - 1) * srs + end)) return fail("page_append: rows");
            if (!fits(0, 0, zg_page_words(G, dk, dv, page)) || !fits(2, 0, most) || !fits(3, 0, ZG_BATCH_ROWS + 4 * B)) return fail("page_append: pages or tables");
            if (qh && ((B > 1 && trs < s.off[3] + qh * dk) || !fits(5, s.off[3], (B - 1) * trs + qh * dk))) return fail("page_append: query heads");
            for (int i = 1; i < 6; i++) if (s.buf[i] == s.buf[0] || (qh && i < 5 && s.buf[i] == s.buf[5])) return fail("page_append: in place");
            return true;
        }
        case ZG_OP_PAGE_READ: {
            const size_t B = s.n[0], G = s.n[1], dk = s.n[2], dv = s.n[3], drs = s.n[4], page = s.n[5], most = s.n[6];
            if (!B || B > (1u << 24) || !page_shape_ok(G, dk, dv, page) || !most || most >= (1u << 25)) return fail("page_read: shape");
            const size_t k0 = s.off[0], k1 = k0 + G * dk, v0 = s.off[1], v1 = v0 + G * dv, end = std::max(k1, v1);
            if ((k0 < v1 && v0 < k1) || (B > 1 && drs < end) || !fits(0, 0, (B - 1) * drs + end)) return fail("page_read: rows");
            if (!fits(1, 0, zg_page_words(G, dk, dv, page)) || !fits(2, 0, most) || !fits(3, 0, ZG_BATCH_ROWS + 4 * B)) return fail("page_read: pages or tables");
            for (int i = 1; i < 4; i++) if (s.buf[i] == s.buf[0]) return fail("page_read: in place");
            return true;
        }
        case ZG_OP_PAGE_COPY: {
            const size_t B = s.n[0], words = s.n[1];
            if (!B || B > (1u << 24) || !words || words > (1u << 24)) return fail("page_copy: shape");
            if (!fits(0, 0, words) || !fits(1, 0, ZG_BATCH_ROWS + 4 * B)) return fail("page_copy: pages or table");
            if (s.buf[0] == s.buf[1]) return fail("page_copy: in place");
            return true;
        }
        default: return fail("not a sequence op");
    }
}

bool zg_launch_page_op(const ZgOp& op, float* const* bufs, const size_t* elems, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    auto pool = [&](int pages, int table, const PageShape& shape) { return page_pool(bufs[s.buf[pages]], elems[s.buf[pages]], bufs[s.buf[table]], elems[s.buf[table]], s.n[6], shape); };
    switch (op.tag) {
        case ZG_OP_PAGE_APPEND: {
            PaArgs a = {};
            a.s = page_shape(s.n[1], s.n[2], s.n[3], s.n[5]);
            a.pool = pool(0, 2, a.s);
            a.pages = reinterpret_cast<uint8_t*>(bufs[s.buf[0]]); a.src = bufs[s.buf[1]]; a.table = bufs[s.buf[3]];
            a.B = s.n[0]; a.src_rs = s.n[4]; a.k_col = s.off[0]; a.v_col = s.off[1]; a.q_col = s.off[2]; a.q_heads = s.n[10]; a.dst_rs = s.n[11];
            a.turn_at = s.n[7]; a.rot = s.n[8]; a.halves = s.n[9];
            a.turned = a.q_heads ? bufs[s.buf[5]] + s.off[3] : nullptr;
            a.freqs = a.rot && s.buf[4] != ZG_NO_BUF ? bufs[s.buf[4]] + s.off[4] : nullptr;
            if (!a.freqs) for (uint32_t i = 0; i < a.rot / 2; i++) a.freq[i] = std::pow((double)s.f[0], -2.0 * i / a.rot);
            const size_t smem = sizeof(float) * std::min(a.s.page, a.B) * (a.s.dk + a.s.dv);
            if (!zg_smem_limit<k_page_append>(sizeof(float) * 64 * 512)) return false;
            launch_pdl(k_page_append, dim3(a.B, a.s.G + (a.q_heads * a.s.dk + kPaQueries - 1) / kPaQueries), dim3(kPaThreads), smem, st, a);
            ZG_SEQ_CHECK();
            return true;
        }
        case ZG_OP_PAGE_READ: {
            PrArgs a;
            a.s = page_shape(s.n[1], s.n[2], s.n[3], s.n[5]);
            a.pool = pool(1, 2, a.s);
            a.table = bufs[s.buf[3]]; a.dst = bufs[s.buf[0]]; a.B = s.n[0]; a.dst_rs = s.n[4]; a.k_col = s.off[0]; a.v_col = s.off[1];
            launch_pdl(k_page_read, dim3((a.B + kPrRows - 1) / kPrRows, a.s.G), dim3(kPrThreads), 0, st, a);
            ZG_SEQ_CHECK();
            return true;
        }
        case ZG_OP_PAGE_COPY: {
            const uint32_t B = s.n[0], words = s.n[1], count = (uint32_t)std::min<size_t>(elems[s.buf[0]] / words, 0x7fffffffu), share = kPcThreads * kPcVectors;
            if (words % 4 == 0) launch_pdl(k_page_copy<uint4>, dim3(B, (words / 4 + share - 1) / share), dim3(kPcThreads), 0, st, reinterpret_cast<uint4*>(bufs[s.buf[0]]), bufs[s.buf[1]], B, count, words / 4);
            else launch_pdl(k_page_copy<uint32_t>, dim3(B, (words + share - 1) / share), dim3(kPcThreads), 0, st, reinterpret_cast<uint32_t*>(bufs[s.buf[0]]), bufs[s.buf[1]], B, count, words);
            ZG_SEQ_CHECK();
            return true;
        }
        default: zg_set_error("not a sequence op"); return false;
    }
}
