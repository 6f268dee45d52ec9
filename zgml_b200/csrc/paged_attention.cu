// PAGED_ATTENTION (parameter pack in include/zgml_cuda.h): softmax attention of the rows of a step over the 8-bit pages of their sequences.
#include "pages.cuh"

#include <algorithm>

namespace {

struct PgArgs {
    PagePool pool; PageShape s;
    float* dst; const float* q; const float* table; const void* sink;
    uint32_t B, H, rep, q_rs, dst_rs, window, sink_bf16;
    float scale, cap;
};
constexpr uint32_t kPgWarps = 8;
__device__ __forceinline__ float pg_sink(const PgArgs& a, uint32_t h) { return a.sink_bf16 ? __bfloat162float(reinterpret_cast<const bf16*>(a.sink)[h]) : reinterpret_cast<const float*>(a.sink)[h]; }

// CTA (query head, row): a warp per token, the warps' tokens interleaved, one running maximum and sum a warp.
__global__ void __launch_bounds__(32 * kPgWarps) k_paged_rows(const PgArgs a) {
    pdl_enter();
    __shared__ float q[256], acc[kPgWarps][256], m_[kPgWarps], l_[kPgWarps];
    const uint32_t h = blockIdx.x, r = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = h / a.rep;
    const PageShape& s = a.s;
    const BatchHead head = batch_head(a.table, a.B);
    const BatchRow w = batch_row(a.table, r);
    if (r >= head.rows || w.slot < 0) return;
    const bool ok = page_row_ok(a.pool, s, w);
    for (uint32_t d = threadIdx.x; d < s.dk; d += blockDim.x) q[d] = a.q[(size_t)r * a.q_rs + h * s.dk + d] * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[8] = {};
    bool bad = !ok;
    const uint32_t length = ok ? w.length : 0, lo = a.window && length > a.window ? length - a.window : 0;
    for (uint32_t j = lo + warp; j < length; j += kPgWarps) {
        const uint32_t t = j & (s.page - 1);
        const int32_t id = page_id(a.pool, w.slot, j >> s.shift);
        if (id < 0) { bad = true; break; }
        const uint8_t* part = a.pool.pages + (size_t)id * page_bytes(s) + (size_t)g * s.head;
        const float2 scale = *reinterpret_cast<const float2*>(part);
        float dot = 0.0f;
        for (uint32_t d = lane; d < s.dk; d += 32) dot = fmaf(q[d], ((float)part[key_byte(s, t, d)] - 128.0f) * scale.x, dot);
        dot = warp_sum(dot);
        if (a.cap > 0.0f) dot = a.cap * tanhf(dot / a.cap);
        const float top = fmaxf(m, dot), f = m == -INFINITY ? 0.0f : expf(m - top), p = expf(dot - top);
        m = top; l = l * f + p;
        for (uint32_t i = 0, d = lane; d < s.dv; i++, d += 32) o[i] = o[i] * f + p * ((float)part[value_byte(s, t, d)] - 128.0f) * scale.y;
    }
    for (uint32_t i = 0, d = lane; d < s.dv; i++, d += 32) acc[warp][d] = o[i];
    if (lane == 0) { m_[warp] = m; l_[warp] = l; }
    bad = __syncthreads_or(bad);
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t i = 0; i < kPgWarps; i++) top = fmaxf(top, m_[i]);
    const bool none = top == -INFINITY && length <= lo;
    if (a.sink) top = fmaxf(top, pg_sink(a, h));
    for (uint32_t i = 0; i < kPgWarps; i++) sum += m_[i] == -INFINITY ? l_[i] : l_[i] * expf(m_[i] - top);
    if (a.sink) sum += expf(pg_sink(a, h) - top);
    for (uint32_t d = threadIdx.x; d < s.dv; d += blockDim.x) {
        float v = 0.0f;
        for (uint32_t i = 0; i < kPgWarps; i++) v += m_[i] == -INFINITY ? acc[i][d] : acc[i][d] * expf(m_[i] - top);
        a.dst[(size_t)r * a.dst_rs + h * s.dv + d] = bad ? kBatchNaN : none ? 0.0f : v / sum;
    }
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
bool zg_launch_paged_attention(const ZgOp& op, float* const* bufs, const size_t* elems, float*, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    PgArgs a;
    a.s = page_shape(s.n[2], s.n[3], s.n[4], s.n[7]);
    a.pool = page_pool(bufs[s.buf[2]], elems[s.buf[2]], bufs[s.buf[3]], elems[s.buf[3]], s.n[8], a.s);
    a.B = s.n[0]; a.H = s.n[1]; a.rep = a.H / s.n[2]; a.q_rs = s.n[5]; a.dst_rs = s.n[6]; a.window = s.n[9]; a.sink_bf16 = s.n[10] == ZG_W_BF16;
    a.dst = bufs[s.buf[0]] + s.off[1]; a.q = bufs[s.buf[1]] + s.off[0]; a.table = bufs[s.buf[4]];
    a.sink = s.buf[5] == ZG_NO_BUF ? nullptr : a.sink_bf16 ? (const void*)wptr<bf16>(bufs, s.buf[5], s.off[2]) : (const void*)wptr<float>(bufs, s.buf[5], s.off[2]);
    a.scale = s.f[0]; a.cap = s.f[1];
    launch_pdl(k_paged_rows, dim3(a.H, a.B), dim3(32 * kPgWarps), 0, st, a);
    ZG_SEQ_CHECK();
    return true;
}
