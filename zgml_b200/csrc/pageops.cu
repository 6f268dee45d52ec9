// Sequence-model DeviceOps over paged caches in 8 bits (parameter packs in include/zgml_cuda.h): PAGE_APPEND, PAGE_READ and PAGE_COPY; PAGED_ATTENTION has a file of its own.
#include "pages.cuh"

#include <algorithm>
#include <cmath>

namespace {

// ── PAGE_APPEND ──────────────────────────────────────────────────────────────────────────────────────────────────────
constexpr uint32_t kPaThreads = 256, kPaPairs = 128, kPaRows = 16, kPaTurns = 4;      // pairs of a head; rows a CTA at most; tokens of a page whose turns are kept, and rows behind its first that make it many
struct PaArgs {
    PagePool pool; PageShape s;
    uint8_t* pages; const float* src; const float* table; float* turned; const float* freqs;
    uint32_t B, src_rs, k_col, v_col, q_col, q_heads, dst_rs, turn_at, rot, halves, rows, part, vec, key_rows, key_ctas, shares;      // rows of a CTA of queries, values of a row in it; rows of keys' CTAs, CTAs of those rows
    double freq[kPaPairs];                                           // base^(-2i / rot), where no table of frequencies is given
};
// Cosine and sine of a position's turn.  Everything up to the turned value is in 64 bits, and that is rounded once: a code is a turned value over its scale, rounded, and an
// error of f32's size would now and then make it its neighbour, an error of a hundredth of a head's largest value.  The angle over pi, less an even whole number, comes from a product
// with both parts of 1 / pi.
__device__ __forceinline__ double2 pa_turn(const PaArgs& a, double position, uint32_t i) {
    constexpr double inv_pi = 0.31830988618379069122, inv_pi_low = -1.9678676675182485832e-17;
    const double angle = position * (a.freqs ? (double)a.freqs[i] : a.freq[i]), even = 2.0 * rint(angle * (0.5 * inv_pi));
    double2 t;
    sincospi(fma(angle, inv_pi_low, fma(angle, inv_pi, -even)), &t.y, &t.x);
    return t;
}
__device__ __forceinline__ float2 pa_turned(float x, float y, double2 t) { return make_float2((float)((double)x * t.x - (double)y * t.y), (float)((double)x * t.y + (double)y * t.x)); }
// what a scale has to be at least: the smallest power of two (2^-126 at least) of which 127 times reach the value whose bits are given; NaN where that is not finite
__device__ __forceinline__ float pa_scale(uint32_t bits) {
    if (bits >= 0x7f800000u) return kBatchNaN;
    int e = (int)(bits >> 23) - 127;                                 // (what is below 2^-119 has the smallest scale in any case)
    e = (bits & 0x7fffffu) > 0x7e0000u ? e - 5 : e - 6;              // 127 / 64 = 1.984375
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}
__device__ __forceinline__ uint32_t pa_code(float x, float inv) { return (uint32_t)(int)(rintf(x * inv) + 128.0f); }

// Query heads of the CTA's rows: a part of their values.  Bound by reading and writing them; what is asked for of the rows comes for all at once.
__device__ void pa_queries(const PaArgs& a, const BatchHead& head, uint32_t r0, uint32_t first, double2* turn) {
    __shared__ int8_t states[kPaRows];                               // of a row: -1 idle, 0 out of range
    const PageShape& s = a.s;
    const uint32_t rows = min(a.rows, head.rows - r0), n = min(a.part, a.q_heads * s.dk - first), half = a.rot / 2;
    if (threadIdx.x < rows) {
        const BatchRow w = batch_row(a.table, r0 + threadIdx.x);
        bool ok = page_row_ok(a.pool, s, w) && head.prefix >= 0;
        ok = ok && (w.length == 0 || page_id(a.pool, w.slot, (w.length - 1) >> s.shift) >= 0);
        states[threadIdx.x] = w.slot < 0 ? -1 : ok;
    }
    for (uint32_t x = threadIdx.x; x < rows * half; x += kPaThreads) {
        const uint32_t m = x / half;
        const BatchRow w = batch_row(a.table, r0 + m);
        if (w.slot >= 0 && w.length >= 0 && head.prefix >= 0) turn[x] = pa_turn(a, (double)head.prefix + w.length - 1, x - m * half);
    }
    __syncthreads();
    const float4 lost = make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN);
    if (a.vec) {                                                     // four pairs, or four values that stay
        const uint32_t quads = a.rot / 8, each = quads + (s.dk - a.rot) / 4, items = n / s.dk * each;
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < rows * items; i += kPaThreads) {
            const uint32_t m = i / items, x = i - m * items, h = x / each, k = x - h * each;
            const int state = states[m];
            if (state < 0) continue;
            const float* src = a.src + (size_t)(r0 + m) * a.src_rs + a.q_col + first;
            float* dst = a.turned + (size_t)(r0 + m) * a.dst_rs + first;
            uint32_t p = h * s.dk, q = p;
            if (k < quads) { p += a.turn_at + (a.halves ? 4 * k : 8 * k); q = p + (a.halves ? half : 4); }
            else { const uint32_t d = 4 * (k - quads); p += d < a.turn_at ? d : d + a.rot; }
            float4 u = *reinterpret_cast<const float4*>(src + p);
            if (k < quads) {
                float4 v = *reinterpret_cast<const float4*>(src + q);
                const double2* y = turn + m * half + 4 * k;
                float2 z[4];
                if (a.halves) { z[0] = pa_turned(u.x, v.x, y[0]); z[1] = pa_turned(u.y, v.y, y[1]); z[2] = pa_turned(u.z, v.z, y[2]); z[3] = pa_turned(u.w, v.w, y[3]); }
                else { z[0] = pa_turned(u.x, u.y, y[0]); z[1] = pa_turned(u.z, u.w, y[1]); z[2] = pa_turned(v.x, v.y, y[2]); z[3] = pa_turned(v.z, v.w, y[3]); }
                if (a.halves) { u = make_float4(z[0].x, z[1].x, z[2].x, z[3].x); v = make_float4(z[0].y, z[1].y, z[2].y, z[3].y); }
                else { u = make_float4(z[0].x, z[0].y, z[1].x, z[1].y); v = make_float4(z[2].x, z[2].y, z[3].x, z[3].y); }
                *reinterpret_cast<float4*>(dst + q) = state ? v : lost;
            }
            *reinterpret_cast<float4*>(dst + p) = state ? u : lost;
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < rows * n; i += kPaThreads) {
        const uint32_t m = i / n, c = i - m * n, in = c % s.dk - a.turn_at;
        const int state = states[m];
        if (state < 0) continue;
        const float* src = a.src + (size_t)(r0 + m) * a.src_rs + a.q_col + first;
        float v = src[c];
        if (in < a.rot) {
            const bool second = a.halves ? in >= half : in & 1;
            const float other = src[(int)c + (a.halves ? (second ? -(int)half : (int)half) : second ? -1 : 1)];
            const float2 z = pa_turned(second ? other : v, second ? v : other, turn[m * half + (a.halves ? (second ? in - half : in) : in >> 1)]);
            v = second ? z.y : z.x;
        }
        a.turned[(size_t)(r0 + m) * a.dst_rs + first + c] = state ? v : kBatchNaN;
    }
}

// what a scale becomes when values up to `most` (their bits) join it (one that is not a number stays until the page begins anew)
__device__ __forceinline__ float pa_after(float before, uint32_t most) {
    const float x = pa_scale(most);
    return before != before || x < before ? before : x;
}
// codes of a part's keys or values in multiples of a larger scale
__device__ __forceinline__ void pa_rescale(const PageShape& s, uint8_t* part, bool values, float before, float after, uint32_t first, uint32_t step) {
    const float ratio = before / after;
    if (!(ratio < 1.0f)) return;
    uint32_t* codes = reinterpret_cast<uint32_t*>(part + kPageHead + (values ? s.page * s.kp : 0));
#pragma unroll 4
    for (uint32_t x = first; x < s.page * (values ? s.vp : s.kp) / 4; x += step) {
        const uint32_t c = codes[x];
        uint32_t o = 0;
#pragma unroll
        for (int b = 0; b < 32; b += 8) o |= pa_code((float)(c >> b & 255) - 128.0f, ratio) << b;
        codes[x] = o;
    }
}
// The tokens of one page that a step brings, for all heads: a warp a head, which reads them twice (for the scales, for the codes); turns are made once.
__device__ void pa_few(const PaArgs& a, const BatchHead& head, uint8_t* page, const int32_t* joined, const uint32_t* list, uint32_t n, uint32_t begin, double2* turn) {
    const PageShape& s = a.s;
    const uint32_t lane = threadIdx.x & 31, half = a.rot / 2, turns = min(n, kPaTurns);
    for (uint32_t x = threadIdx.x; x < turns * half; x += kPaThreads) turn[x] = pa_turn(a, (double)head.prefix + (begin + list[x / half]), x % half);
    __syncthreads();
    for (uint32_t g = threadIdx.x >> 5; g < s.G; g += kPaThreads / 32) {
        uint8_t* const part = page + (size_t)g * s.head;
        float2 before = *reinterpret_cast<const float2*>(part);
        uint32_t most_k = 0, most_v = 0;
        float inv_k = 0.0f, inv_v = 0.0f;
        auto pass = [&](bool codes) {
            for (uint32_t m = 0; m < n; m++) {
                const uint32_t t = list[m];
                const float* const row = a.src + (size_t)joined[t] * a.src_rs;
                const float* const keys = row + a.k_col + g * s.dk;
                const float* const values = row + a.v_col + g * s.dv;
#pragma unroll 4
                for (uint32_t c = lane; c < s.dv; c += 32) {
                    const float v = values[c];
                    if (!codes) most_v = max(most_v, __float_as_uint(fabsf(v)));
                    else if (inv_v == inv_v) part[value_byte(s, t, c)] = (uint8_t)pa_code(v, inv_v);
                }
#pragma unroll 2
                for (uint32_t i = lane; i < half; i += 32) {
                    const uint32_t p = a.turn_at + (a.halves ? i : 2 * i), q = p + (a.halves ? half : 1);
                    const float2 y = pa_turned(keys[p], keys[q], m < turns ? turn[m * half + i] : pa_turn(a, (double)head.prefix + (begin + t), i));
                    if (!codes) most_k = max(most_k, max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y))));
                    else if (inv_k == inv_k) { part[key_byte(s, t, p)] = (uint8_t)pa_code(y.x, inv_k); part[key_byte(s, t, q)] = (uint8_t)pa_code(y.y, inv_k); }
                }
                for (uint32_t c = lane; c < s.dk - a.rot; c += 32) {
                    const uint32_t d = c < a.turn_at ? c : c + a.rot;
                    const float v = keys[d];
                    if (!codes) most_k = max(most_k, __float_as_uint(fabsf(v)));
                    else if (inv_k == inv_k) part[key_byte(s, t, d)] = (uint8_t)pa_code(v, inv_k);
                }
            }
        };
        pass(false);
        if (joined[0] >= 0) before = make_float2(0.0f, 0.0f);
        const float2 after = make_float2(pa_after(before.x, __reduce_max_sync(0xffffffffu, most_k)), pa_after(before.y, __reduce_max_sync(0xffffffffu, most_v)));
        if (joined[0] < 0) { pa_rescale(s, part, false, before.x, after.x, lane, 32); pa_rescale(s, part, true, before.y, after.y, lane, 32); }
        __syncwarp();
        if (lane == 0) *reinterpret_cast<float2*>(part) = after;
        inv_k = 1.0f / after.x; inv_v = 1.0f / after.y;
        pass(true);
    }
}
// The same of many, for a head's keys or its values and a whole CTA.  Keys go to shared memory as they are turned; values are read again when their scale is known (with both in shared memory
// fewer CTAs are resident: 1.5 times the time for 2048 tokens of 8 heads of 128).
__device__ void pa_many(const PaArgs& a, const BatchHead& head, uint8_t* part, uint32_t g, bool values, const int32_t* joined, const uint32_t* list, uint32_t n, uint32_t begin, float* tile) {
    __shared__ uint32_t most;
    const PageShape& s = a.s;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, half = a.rot / 2;
    float* const scale = reinterpret_cast<float*>(part) + values;
    float before = *scale;
    uint32_t top = 0;
    __syncthreads();                                                 // (another head's, or its keys, are done)
    if (tid == 0) most = 0;
    for (uint32_t m = warp; m < n; m += kPaThreads / 32) {
        const uint32_t t = list[m];
        const float* const row = a.src + (size_t)joined[t] * a.src_rs;
        if (values) {
#pragma unroll 4
            for (uint32_t c = lane; c < s.dv; c += 32) top = max(top, __float_as_uint(fabsf(row[a.v_col + g * s.dv + c])));
            continue;
        }
        const double position = (double)head.prefix + (begin + t);
        const float* const keys = row + a.k_col + g * s.dk;
#pragma unroll 2
        for (uint32_t i = lane; i < half; i += 32) {
            const uint32_t p = a.turn_at + (a.halves ? i : 2 * i), q = p + (a.halves ? half : 1);
            const float2 y = pa_turned(keys[p], keys[q], pa_turn(a, position, i));
            tile[m * s.dk + p] = y.x; tile[m * s.dk + q] = y.y;
            top = max(top, max(__float_as_uint(fabsf(y.x)), __float_as_uint(fabsf(y.y))));
        }
        for (uint32_t c = lane; c < s.dk - a.rot; c += 32) {
            const uint32_t d = c < a.turn_at ? c : c + a.rot;
            const float v = keys[d];
            tile[m * s.dk + d] = v;
            top = max(top, __float_as_uint(fabsf(v)));
        }
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&most, top);
    __syncthreads();
    if (joined[0] >= 0) before = 0.0f;
    const float after = pa_after(before, most), inv = 1.0f / after;
    if (joined[0] < 0) pa_rescale(s, part, values, before, after, tid, kPaThreads);
    __syncthreads();
    if (tid == 0) *scale = after;
    if (after != after) return;
    if (!values) {                                                   // four values of a key at a time
        for (uint32_t m = warp; m < n; m += kPaThreads / 32)
            for (uint32_t c = 4 * lane; c < s.dk; c += 128) {
                const float* from = tile + m * s.dk + c;
                uint8_t* to = part + key_byte(s, list[m], c);
                if (c + 4 <= s.dk) *reinterpret_cast<uint32_t*>(to) = pa_code(from[0], inv) | pa_code(from[1], inv) << 8 | pa_code(from[2], inv) << 16 | pa_code(from[3], inv) << 24;
                else for (uint32_t k = 0; c + k < s.dk; k++) to[k] = (uint8_t)pa_code(from[k], inv);
            }
        return;
    }
    // one value of tokens t, t + 1, t + 8, t + 9 where all of them come, else byte by byte
    for (uint32_t unit = 0; unit < s.page / 16; unit++)
#pragma unroll 2
        for (uint32_t y = tid; y < 4 * s.vp; y += kPaThreads) {
            const uint32_t c = 16 * (y / 64) + 8 * (y & 1) + (y % 64) / 8, t = 16 * unit + 2 * ((y / 2) & 3);
            const int32_t r0 = joined[t], r1 = joined[t + 1], r8 = joined[t + 8], r9 = joined[t + 9];
            if (c >= s.dv || (r0 & r1 & r8 & r9) < 0) continue;      // (none of them)
            uint8_t* to = part + value_byte(s, t, c);
            auto code = [&](int32_t r) { return pa_code(a.src[(size_t)r * a.src_rs + a.v_col + g * s.dv + c], inv); };
            if ((r0 | r1 | r8 | r9) >= 0) *reinterpret_cast<uint32_t*>(to) = code(r0) | code(r1) << 8 | code(r8) << 16 | code(r9) << 24;
            else {
                if (r0 >= 0) to[0] = (uint8_t)code(r0);
                if (r1 >= 0) to[1] = (uint8_t)code(r1);
                if (r8 >= 0) to[2] = (uint8_t)code(r8);
                if (r9 >= 0) to[3] = (uint8_t)code(r9);
            }
        }
}
// Row r's page, where r is the first of the step's rows that join it: it finds the others in the table (the last of several at one place counts), and no other CTA touches the
// page's part of a head, so no order of CTAs changes anything.
__device__ void pa_keys(const PaArgs& a, const BatchHead& head, uint32_t r, bool many, uint32_t y, float* mem) {
    __shared__ int32_t joined[64];                                   // row that brings token t of the page, or -1
    __shared__ uint32_t list[64];                                    // tokens that come, in order
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x;
    const PageShape& s = a.s;
    const BatchRow w = batch_row(a.table, r);
    const uint32_t place = (uint32_t)w.length - 1;
    const int32_t id = page_id(a.pool, w.slot, place >> s.shift);
    if (id < 0) return;
    __syncthreads();
    if (tid < 64) joined[tid] = -1;
    __syncthreads();
    bool earlier = false;
#pragma unroll 8
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
            const uint32_t all = __ballot_sync(0xffffffffu, here), mine = n + __popc(all & ((1u << tid) - 1));
            if (here) list[mine] = t + tid;
            n += __popc(all);
        }
        if (tid == 0) count = n;
    }
    __syncthreads();
    uint8_t* const page = a.pages + (size_t)id * page_bytes(s);
    if (!many) pa_few(a, head, page, joined, list, count, place & ~(s.page - 1), reinterpret_cast<double2*>(mem));
    else for (uint32_t u = y; u < 2 * s.G; u += a.shares) pa_many(a, head, page + (size_t)(u % s.G) * s.head, u % s.G, u >= s.G, joined, list, count, place & ~(s.page - 1), mem);
}
// CTAs (rows; share of their work), then (rows; part of the query heads).  Where the four rows behind the one that begins a page join it too, as a prompt's do, its heads' keys and values are shared out;
// else one CTA, another for each of the rows' pages, takes all heads, a warp each, and makes each turn once (8 heads of 128, us, shared out from two tokens on / from five / from sixteen: 128 sequences of 2
// tokens 35.5 / 20.5 / 20.7, 64 of 8 28.3 / 28.5 / 34.9, 4 of 512 50.0 / 43.1 / 67.6).  Bound by latency: 256 single rows 11 us, 2048 rows of four prompts 36 us, 2.4 TB/s.
__global__ void __launch_bounds__(kPaThreads) k_page_append(const __grid_constant__ PaArgs a) {
    pdl_enter();
    extern __shared__ float4 pa_mem[];
    const PageShape& s = a.s;
    const uint32_t lane = threadIdx.x & 31;
    const BatchHead head = batch_head(a.table, a.B);
    if (blockIdx.x >= a.key_ctas) {
        const uint32_t b = blockIdx.x - a.key_ctas, blocks = (a.B + a.rows - 1) / a.rows, r0 = b % blocks * a.rows;
        if (r0 < head.rows) pa_queries(a, head, r0, b / blocks * a.part, reinterpret_cast<double2*>(pa_mem));
        return;
    }
    const uint32_t y = blockIdx.x % a.shares, r0 = blockIdx.x / a.shares * a.key_rows, r = min(r0 + lane, a.B - 1);
    const BatchRow w = batch_row(a.table, r), z = batch_row(a.table, r ? r - 1 : 0);
    if (r0 >= head.rows) return;
    // rows that append something, and not to the page that the row before them appends to (as most rows of a prompt do); those whose page the next four join
    const bool live = r0 + lane < head.rows && w.length > 0;
    const uint32_t nth = (uint32_t)(w.length - 1) >> s.shift;
    const bool begins = live && lane < a.key_rows && w.slot >= 0 && page_row_ok(a.pool, s, w) && head.prefix >= 0 &&
                        !(r && z.slot == w.slot && z.length > 0 && (uint32_t)(z.length - 1) >> s.shift == nth);
    bool many = true;
#pragma unroll
    for (uint32_t d = 1; d <= kPaTurns; d++) {
        const int32_t slot = __shfl_down_sync(0xffffffffu, w.slot, d);
        const uint32_t page = __shfl_down_sync(0xffffffffu, nth, d);
        const int follows = __shfl_down_sync(0xffffffffu, (int)live, d);      // (every lane takes part in all three)
        many &= follows && slot == w.slot && page == nth;
    }
    const uint32_t few = __ballot_sync(0xffffffffu, begins && !many);
    for (uint32_t todo = __ballot_sync(0xffffffffu, begins && (many || __popc(few & ((1u << lane) - 1)) % a.shares == y)); todo; todo &= todo - 1) {
        const uint32_t first = __ffs(todo) - 1;
        pa_keys(a, head, r0 + first, !(few >> first & 1), y, reinterpret_cast<float*>(pa_mem));
    }
}

// ── PAGE_READ ────────────────────────────────────────────────────────────────────────────────────────────────────────
struct PrArgs {
    PagePool pool; PageShape s;
    const float* table; float* dst;
    uint32_t B, dst_rs, k_col, v_col, vec;
};
constexpr uint32_t kPrThreads = 256, kPrRows = 16;
// CTA (16 rows, key head): bound by latency, of the table, the page's id, its scale and its codes, one after the other for 16 KB of writes (2186 rows of 8 heads of 128: 12 us for the launch by itself, of which its
// 18 MB of writes need 2.7).  The rows' pages are found once.  Keys are read four codes at a time; values, of which a tile holds sixteen tokens side by side, a tile at a
// time for all rows whose tokens it holds (byte by byte for each row a step of append and read took 1.5 us more: every byte came from a line of its own).
__global__ void __launch_bounds__(kPrThreads) k_page_read(const PrArgs a) {
    pdl_enter();
    __shared__ const uint8_t* parts[kPrRows];                        // null: zeros, or nothing (tokens: -1), or no numbers (-2)
    __shared__ int32_t tokens[kPrRows];
    __shared__ alignas(16) int8_t rows[kPrRows][16];                 // of a tile that row m reads for all: the row of each of its tokens, or -1
    __shared__ uint32_t leaders;
    const PageShape& s = a.s;
    const uint32_t first = blockIdx.x * kPrRows, g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == 0) {
        const BatchHead head = batch_head(a.table, a.B);
        const uint32_t r = first + lane;
        const BatchRow w = batch_row(a.table, min(r, a.B - 1));
        const uint8_t* part = nullptr;
        int32_t token = -1;
        if (lane < kPrRows && r < head.rows && w.slot >= 0) {
            token = -2;
            if (page_row_ok(a.pool, s, w)) {
                const int32_t id = w.length > 0 ? page_id(a.pool, w.slot, (uint32_t)(w.length - 1) >> s.shift) : -1;
                if (w.length == 0) token = 0;
                else if (id >= 0) { token = (w.length - 1) & (int)(s.page - 1); part = a.pool.pages + (size_t)id * page_bytes(s) + (size_t)g * s.head; }
            }
        }
        // rows of one tile go together, unless a token is asked for twice: the second time it belongs to another tile's turn
        const unsigned long long at = part ? (unsigned long long)(part - a.pool.pages) << 2 | (uint32_t)token >> 4 : ~0ull - lane;
        const uint32_t tile = __match_any_sync(0xffffffffu, at), same = tile & __match_any_sync(0xffffffffu, token), turn = __popc(same & ((1u << lane) - 1));
        const uint32_t together = tile & __match_any_sync(0xffffffffu, turn), leader = __ffs(together) - 1;
        if (lane < kPrRows) {
            parts[lane] = part; tokens[lane] = token;
            *reinterpret_cast<int4*>(rows[lane]) = make_int4(-1, -1, -1, -1);
        }
        __syncwarp();
        if (part) rows[leader][token & 15] = (int8_t)lane;
        const uint32_t all = __ballot_sync(0xffffffffu, part && leader == lane);
        if (lane == 0) leaders = all;
    }
    __syncthreads();
    auto row_at = [&](uint32_t m) { return a.dst + (size_t)(first + m) * a.dst_rs; };
    // keys, and rows without a page
    const uint32_t words = (s.dk + 3) / 4;
    for (uint32_t m = warp; m < kPrRows; m += kPrThreads / 32) {
        const int32_t t = tokens[m];
        if (t == -1) continue;
        const uint8_t* part = parts[m];
        float* to = row_at(m) + a.k_col + g * s.dk;
        if (!part) {
            const float v = t == -2 ? kBatchNaN : 0.0f;
            for (uint32_t d = lane; d < s.dk; d += 32) to[d] = v;
            for (uint32_t d = lane; d < s.dv; d += 32) row_at(m)[a.v_col + g * s.dv + d] = v;
            continue;
        }
        const float scale = reinterpret_cast<const float*>(part)[0];
        for (uint32_t k = lane; k < words; k += 32) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(part + key_byte(s, t, 4 * k));
            const float v[4] = {((float)(word & 255) - 128.0f) * scale, ((float)(word >> 8 & 255) - 128.0f) * scale, ((float)(word >> 16 & 255) - 128.0f) * scale, ((float)(word >> 24) - 128.0f) * scale};
            if (a.vec) *reinterpret_cast<float4*>(to + 4 * k) = make_float4(v[0], v[1], v[2], v[3]);
            else for (uint32_t e = 0; 4 * k + e < s.dk && e < 4; e++) to[4 * k + e] = v[e];
        }
    }
    // values
    const uint32_t tiles = s.vp / 16;
    uint32_t turn = 0;
    for (uint32_t todo = leaders; todo; todo &= todo - 1) {
        const uint32_t m = __ffs(todo) - 1, unit = tokens[m] & ~15;
        const float scale = reinterpret_cast<const float*>(parts[m])[1];
        for (uint32_t c = (warp + kPrThreads / 32 - turn) % (kPrThreads / 32); c < tiles; c += kPrThreads / 32) {
            const uint2 x = *reinterpret_cast<const uint2*>(parts[m] + value_byte(s, unit, 16 * c) + 8 * lane);
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) {
                const uint32_t d = 16 * c + 8 * (e / 4) + lane / 4, token = 2 * (lane & 3) + 8 * ((e / 2) & 1) + (e & 1);
                const int row = rows[m][token];
                if (row >= 0 && d < s.dv) row_at(row)[a.v_col + g * s.dv + d] = ((float)((e < 4 ? x.x : x.y) >> (8 * (e & 3)) & 255) - 128.0f) * scale;
            }
        }
        turn = (turn + tiles) % (kPrThreads / 32);
    }
}

// ── PAGE_COPY ────────────────────────────────────────────────────────────────────────────────────────────────────────
constexpr uint32_t kPcThreads = 256, kPcVectors = 4;                 // vectors of 16 bytes a thread
// CTA (move, share of the page): bound by the reads and writes: 268 MB, 4079 pages of 33 KB, in 40 us for the launch by itself, 6.7 TB/s (replays, us: one vector a thread 53.3, four 47.1, eight 49.2).  V: vectors of 16
// bytes, or words where a page is no whole number of vectors.
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
            // Keys and values of each head in a CTA of their own (one prompt of 512 tokens, us, together / apart: 28.9 / 22.6, four 48.4 / 43.7), fewer where there are many rows, which each of a page's
            // CTAs looks through (8192 rows with 16 CTAs / with four: 173 / 143).  As many rows as such CTAs, so that each row's page may have one.  More rows of queries where there are many; query heads in smaller parts where there are few rows
            // (with 1024 / 4096 values, us: 64 rows of 32 / 8 heads of 128 14.4 / 16.4, 128 17.1 / 18.3, 256 of pairs 20.7 / 22.1; 512 26.7 / 24.6, 2048 51.0 / 44.7).
            a.rows = std::min(kPaRows, (a.B + 511) / 512);
            a.shares = std::min(2 * a.s.G, std::max(1u, 32768 / a.B));
            a.key_rows = std::min(kPaRows, 2 * a.s.G);
            a.key_ctas = (a.B + a.key_rows - 1) / a.key_rows * a.shares;
            const uint32_t heads = std::max(1u, a.B <= 256 ? 1024 / a.s.dk : 4096 / a.s.dk), parts = (a.q_heads + heads - 1) / heads;
            a.part = heads * a.s.dk;
            a.vec = a.q_heads && a.s.dk % 4 == 0 && a.turn_at % 4 == 0 && a.rot % 8 == 0 && a.src_rs % 4 == 0 && a.q_col % 4 == 0 && a.dst_rs % 4 == 0 && s.off[3] % 4 == 0;
            const size_t smem = std::max<size_t>({sizeof(float) * std::min(a.s.page, a.B) * a.s.dk, sizeof(double2) * std::max(a.rows, std::min(kPaTurns, a.B)) * (a.rot / 2)});
            if (!zg_smem_limit<k_page_append>(sizeof(float) * 64 * 256)) return false;
            launch_pdl(k_page_append, dim3(a.key_ctas + (a.B + a.rows - 1) / a.rows * parts), dim3(kPaThreads), smem, st, a);
            ZG_SEQ_CHECK();
            return true;
        }
        case ZG_OP_PAGE_READ: {
            PrArgs a;
            a.s = page_shape(s.n[1], s.n[2], s.n[3], s.n[5]);
            a.pool = pool(1, 2, a.s);
            a.table = bufs[s.buf[3]]; a.dst = bufs[s.buf[0]]; a.B = s.n[0]; a.dst_rs = s.n[4]; a.k_col = s.off[0]; a.v_col = s.off[1];
            a.vec = a.s.dk % 4 == 0 && a.dst_rs % 4 == 0 && a.k_col % 4 == 0;
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
