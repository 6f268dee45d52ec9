// ADAPTER_LINEAR (parameter pack in include/zgml_cuda.h): dst[r] = base[r] + s_a B_a (A_a src[r]), a the adapter of row r.  Two chained products through `rank` values a
// row; a run of rows with one adapter shares its weights.
//
//   * k_adapter_few: a cluster of 8 CTAs per run of at most 8 rows.  Each CTA sums its eighth of the inputs, the eighths meet over distributed shared memory, and each CTA
//     makes its eighth of the outputs: one launch, and the second product's weights are on their way while the first one is summed.
//   * k_adapter_shrink, k_adapter_expand: blocks of 128 rows on tcgen05, for prompts.
#include "batch_table.cuh"
#include "split_tc.cuh"

#include <algorithm>

namespace {

struct AdArgs {
    float* dst; const float* src; const float* base; const float* scales; const float* table;
    uint32_t B, N, K, rank, adapters, src_rs, dst_rs, base_rs;
};
// what a row asks for: an adapter, or ...
constexpr int kAdNone = -1, kAdIdle = -2, kAdBad = -3;
__device__ __forceinline__ int ad_of(const AdArgs& a, const BatchHead& head, uint32_t r) {
    if (r >= head.rows) return kAdIdle;
    const BatchRow w = batch_row(a.table, r);
    return w.slot < 0 ? kAdIdle : w.adapter < 0 ? kAdNone : (uint32_t)w.adapter >= a.adapters ? kAdBad : w.adapter;
}

// ── few rows ─────────────────────────────────────────────────────────────────────────────────────────────────────────
constexpr uint32_t kAfRows = 8, kAfCluster = 8, kAfThreads = 256, kAfStage = 96 * 1024;      // bytes of the second product's weights that are fetched ahead
__device__ __forceinline__ float af_remote(uint32_t at, uint32_t rank) {
    uint32_t there;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}
__device__ __forceinline__ float4 af_remote4(uint32_t at, uint32_t rank) {
    uint32_t there;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
    return v;
}
// R: rows of the run at most; J: rank values at a time.  x and the weights in vectors of WVec<WT>::n where VEC
template <typename WT, int R, int J, bool VEC>
__device__ __forceinline__ void af_shrink(const AdArgs& a, const WT* __restrict__ wa, const float* __restrict__ x, uint32_t rows, uint32_t k0, uint32_t k1, float* part) {
    constexpr uint32_t V = VEC ? WVec<WT>::n : 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t j0 = warp * J; j0 < a.rank; j0 += 8 * J) {
        float acc[J][R];
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int r = 0; r < R; r++) acc[j][r] = 0.0f;
#pragma unroll 2
        for (uint32_t k = k0 + V * lane; k < k1; k += 32 * V) {
            float w[J][V];
#pragma unroll
            for (int j = 0; j < J; j++) {
                const WT* from = wa + (size_t)min(j0 + j, a.rank - 1) * a.K + k;
                if constexpr (VEC) wld_vec<WT>(from, w[j]); else w[j][0] = wld(from, 0);
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (R > 1 && r >= (int)rows) break;
                float y[V];
                if constexpr (VEC) {
#pragma unroll
                    for (int v = 0; v < (int)V; v += 4) wld_vec<float>(x + (size_t)r * a.src_rs + k + v, y + v);
                } else y[0] = x[(size_t)r * a.src_rs + k];
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int v = 0; v < (int)V; v++) acc[j][r] = fmaf(w[j][v], y[v], acc[j][r]);
            }
        }
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (R > 1 && r >= (int)rows) break;
                const float s = warp_sum(acc[j][r]);
                if (lane == 0 && j0 + j < a.rank) part[r * a.rank + j0 + j] = s;
            }
    }
}
template <typename WT, int R, bool VEC>
__device__ __forceinline__ void af_expand(const AdArgs& a, const WT* wb, const float* base, float* dst, uint32_t rows, uint32_t n0, uint32_t n1, const float* h) {
    for (uint32_t n = n0 + threadIdx.x; n < n1; n += kAfThreads) {
        const WT* row = wb + (size_t)(n - n0) * a.rank;
        float acc[R];
#pragma unroll
        for (int r = 0; r < R; r++) acc[r] = 0.0f;
        if constexpr (VEC) {
            for (uint32_t j = 0; j < a.rank; j += 4) {
                float w[4];
                if constexpr (sizeof(WT) == 2) {
                    const uint2 u = *reinterpret_cast<const uint2*>(row + j);
                    w[0] = __uint_as_float(u.x << 16); w[1] = __uint_as_float(u.x & 0xFFFF0000u); w[2] = __uint_as_float(u.y << 16); w[3] = __uint_as_float(u.y & 0xFFFF0000u);
                } else wld_vec<float>(row + j, w);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float4 y = *reinterpret_cast<const float4*>(h + r * a.rank + j);
                    acc[r] = fmaf(w[0], y.x, fmaf(w[1], y.y, fmaf(w[2], y.z, fmaf(w[3], y.w, acc[r]))));
                }
            }
        } else {
            for (uint32_t j = 0; j < a.rank; j++) {
                const float w = wld(row, j);
#pragma unroll
                for (int r = 0; r < R; r++) acc[r] = fmaf(w, h[r * a.rank + j], acc[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++)
            if (R == 1 || r < (int)rows) dst[(size_t)r * a.dst_rs + n] = base[(size_t)r * a.base_rs + n] + acc[r];
    }
}
// The same with LJ lanes to an output, 16 bytes of its weights each, so that a warp reads whole rows side by side: of rank 64 a lane per output met one bank, or
// 32 lines a load (14336 outputs, 8 rows: 51 us).  U outputs (of one row) or R rows (of one output) at a time make C sums a lane, which meet by halves: a lane ends with
// C / LJ of them, or one.  Loads of the next outputs, and the base, are under way meanwhile.
template <typename WT, int R, int LJ>
__device__ __forceinline__ void af_expand_wide(const AdArgs& a, const WT* wb, const float* base, float* dst, uint32_t rows, uint32_t n0, uint32_t n1, const float* h) {
    constexpr uint32_t E = 16 / sizeof(WT), G = 32 / LJ, U = R == 1 ? 8 : 1, C = R * U, kept = C > LJ ? C / LJ : 1, step = kAfThreads / 32 * G * U;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (LJ - 1);
    const bool on = sub * E < a.rank;
    uint32_t c0 = 0;                                                 // the first sum that the lane ends with
    bool mine = true;                                                // it stores
    {
        uint32_t count = C;
#pragma unroll
        for (int d = LJ / 2; d > 0; d >>= 1) {
            if (count > 1) { count /= 2; c0 += lane & d ? count : 0; }
            else mine = mine && !(lane & d);
        }
    }
    float2 y[R][E / 2];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int e = 0; e < (int)E / 2; e++) y[r][e] = on ? make_float2(h[r * a.rank + sub * E + 2 * e], h[r * a.rank + sub * E + 2 * e + 1]) : make_float2(0.0f, 0.0f);
    uint4 next[U];
    auto load = [&](uint32_t first) {
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t n = first + u * G + lane / LJ;
            next[u] = on && n < n1 ? *reinterpret_cast<const uint4*>(wb + (size_t)(n - n0) * a.rank + sub * E) : make_uint4(0, 0, 0, 0);
        }
    };
    uint32_t first = n0 + warp * G * U;
    load(first);
    for (; first < n1; first += step) {
        uint4 now[U];
        float b[kept], v[C];
        bool to[kept];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) now[u] = next[u];
        load(first + step);
#pragma unroll
        for (uint32_t i = 0; i < kept; i++) {
            const uint32_t c = c0 + i, r = R == 1 ? 0 : c, n = first + (R == 1 ? c * G : 0) + lane / LJ;
            to[i] = mine && n < n1 && r < rows;
            b[i] = to[i] ? base[(size_t)r * a.base_rs + n] : 0.0f;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t x[4] = {now[u].x, now[u].y, now[u].z, now[u].w};
            float2 w[E / 2];
#pragma unroll
            for (int e = 0; e < (int)E / 2; e++)
                w[e] = sizeof(WT) == 2 ? make_float2(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xFFFF0000u)) : make_float2(__uint_as_float(x[2 * e & 3]), __uint_as_float(x[(2 * e + 1) & 3]));
#pragma unroll
            for (int r = 0; r < R; r++) {
                float2 z = __fmul2_rn(w[0], y[r][0]);
#pragma unroll
                for (int e = 1; e < (int)E / 2; e++) z = __ffma2_rn(w[e], y[r][e], z);
                v[R == 1 ? u : r] = z.x + z.y;
            }
        }
        int count = C;
#pragma unroll
        for (int d = LJ / 2; d > 0; d >>= 1) {
            const bool up = lane & d;
            if (count > 1) {
                count /= 2;
#pragma unroll
                for (int i = 0; i < count; i++) {
                    const float there = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + count], d);
                    v[i] = (up ? v[i + count] : v[i]) + there;
                }
            } else v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
        }
#pragma unroll
        for (uint32_t i = 0; i < kept; i++) {
            const uint32_t c = c0 + i, r = R == 1 ? 0 : c, n = first + (R == 1 ? c * G : 0) + lane / LJ;
            if (to[i]) dst[(size_t)r * a.dst_rs + n] = b[i] + v[i];
        }
    }
}
template <typename WT, int R>
__device__ __forceinline__ void af_expand_by(uint32_t lanes, const AdArgs& a, const WT* wb, const float* base, float* dst, uint32_t rows, uint32_t n0, uint32_t n1, const float* h) {
    switch (lanes) {
        case 1: af_expand_wide<WT, R, 1>(a, wb, base, dst, rows, n0, n1, h); break;
        case 2: af_expand_wide<WT, R, 2>(a, wb, base, dst, rows, n0, n1, h); break;
        case 4: af_expand_wide<WT, R, 4>(a, wb, base, dst, rows, n0, n1, h); break;
        case 8: af_expand_wide<WT, R, 8>(a, wb, base, dst, rows, n0, n1, h); break;
        default: af_expand_wide<WT, R, 16>(a, wb, base, dst, rows, n0, n1, h);
    }
}
// vec_k: x and A in vectors; vec_j: rows of B in vectors of four; WIDE: `lanes` lanes share an output; stage: bytes of B fetched
// ahead (0: not)
// (64 registers: 64 rows are 512 CTAs, four an SM; at 80 they took 12.4 us instead of 8.3)
template <typename WT, bool WIDE>
__global__ void __launch_bounds__(kAfThreads, WIDE ? 2 : 4) __cluster_dims__(kAfCluster, 1, 1) k_adapter_few(AdArgs a, const WT* __restrict__ wa, const WT* __restrict__ wb, uint32_t k_slice, uint32_t n_slice,
                                                                                             uint32_t vec_k, uint32_t vec_j, uint32_t lanes, uint32_t stage) {
    pdl_enter();
    extern __shared__ float4 af_mem[];                               // [stage] weights of the CTA's outputs; [8][rank] the CTA's sums; [8][rank] all sums
    const uint32_t rank_id = blockIdx.x % kAfCluster, r = blockIdx.x / kAfCluster;
    const BatchHead head = batch_head(a.table, a.B);
    const int mine = ad_of(a, head, r);
    if (mine == kAdIdle) return;
    const uint32_t n0 = min(a.N, rank_id * n_slice), n1 = min(a.N, n0 + n_slice);
    const float* base = a.base + (size_t)r * a.base_rs;
    float* dst = a.dst + (size_t)r * a.dst_rs;
    if (mine < 0) {
        if (mine == kAdBad || base != dst)
            for (uint32_t n = n0 + threadIdx.x; n < n1; n += kAfThreads) dst[n] = mine == kAdNone ? base[n] : kBatchNaN;
        return;
    }
    // the run of rows with this adapter, inside a block of eight rows: its first row's cluster takes all of it
    if (r % kAfRows && ad_of(a, head, r - 1) == mine) return;
    uint32_t rows = 1;
    {
        bool on = true;
#pragma unroll
        for (uint32_t i = 1; i < kAfRows; i++) {
            on = on && r % kAfRows + i < kAfRows && ad_of(a, head, min(r + i, a.B - 1)) == mine && r + i < a.B;
            rows += on ? 1u : 0u;
        }
    }
    wa += (size_t)mine * a.rank * a.K;
    wb += (size_t)mine * a.N * a.rank + (size_t)n0 * a.rank;
    float* const part = reinterpret_cast<float*>(af_mem) + stage / 4;
    float* const h = part + kAfRows * ((a.rank + 3) & ~3u);
    if (stage && n1 > n0) {
        const uint32_t bytes = (n1 - n0) * a.rank * (uint32_t)sizeof(WT), at = (uint32_t)__cvta_generic_to_shared(af_mem);
        for (uint32_t i = 16 * threadIdx.x; i < bytes; i += 16 * kAfThreads)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + i), "l"(reinterpret_cast<const char*>(wb) + i), "r"(min(16u, bytes - i)) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float scale = a.scales ? a.scales[mine] : 1.0f;
    const float* x = a.src + (size_t)r * a.src_rs;
    const uint32_t k0 = min(a.K, rank_id * k_slice), k1 = min(a.K, k0 + k_slice);
    if (rows == 1) {
        if (vec_k) af_shrink<WT, 1, 2, true>(a, wa, x, rows, k0, k1, part); else af_shrink<WT, 1, 2, false>(a, wa, x, rows, k0, k1, part);
    } else {
        if (vec_k) af_shrink<WT, kAfRows, 2, true>(a, wa, x, rows, k0, k1, part); else af_shrink<WT, kAfRows, 2, false>(a, wa, x, rows, k0, k1, part);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (uint32_t i = threadIdx.x; i < kAfRows * a.rank; i += kAfThreads) {
        float s = 0.0f;
        if (i < rows * a.rank) {
            const uint32_t at = (uint32_t)__cvta_generic_to_shared(part + i);
            float v[kAfCluster];                                     // all on their way before the first is added
#pragma unroll
            for (uint32_t c = 0; c < kAfCluster; c++) v[c] = af_remote(at, c);
#pragma unroll
            for (uint32_t c = 0; c < kAfCluster; c++) s += v[c];
        }
        h[i] = s * scale;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // its wait is at the end: no CTA leaves while its sums are read
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    const WT* const from = stage ? reinterpret_cast<const WT*>(af_mem) : wb;
    if constexpr (WIDE) {
        if (rows == 1) af_expand_by<WT, 1>(lanes, a, from, base, dst, rows, n0, n1, h); else af_expand_by<WT, kAfRows>(lanes, a, from, base, dst, rows, n0, n1, h);
    } else if (rows == 1) {
        if (vec_j) af_expand<WT, 1, true>(a, from, base, dst, rows, n0, n1, h); else af_expand<WT, 1, false>(a, from, base, dst, rows, n0, n1, h);
    } else {
        if (vec_j) af_expand<WT, kAfRows, true>(a, from, base, dst, rows, n0, n1, h); else af_expand<WT, kAfRows, false>(a, from, base, dst, rows, n0, n1, h);
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ── many rows ────────────────────────────────────────────────────────────────────────────────────────────────────────
// Blocks of 128 rows on tcgen05.  Activations (and f32 weights) go in as three bfloat16 parts, all 24 bits of them: three products over bfloat16 weights, six over f32 ones.
// Rows of a block that have another adapter than the product at hand are computed and left out.
//   k_adapter_shrink: the 8 CTAs of a cluster share a block's inputs.  x is split on its way to shared memory; up to kAmRuns adapters accumulate side by side in TMEM; the
//   partial sums meet over distributed shared memory and leave as the parts that the second product wants: x is read once.
//   k_adapter_expand: a CTA keeps the block's rank values and walks tiles of 128 outputs: four warps bring weights and issue, eight add the base and write.  Base and dst
//   are what bounds it.
// (The same on mma.sync took 124 us for 2048 rows of 4096 inputs, 14336 outputs, rank 64, with its issue rate as the bound: 11.3 T operations of products at 130 T/s.)
// Every wait is bounded; a CTA whose wait ran out counts it and makes NaN of its rows.
constexpr uint32_t kAmRows = 128, kAmRank = 64, kAmPart = kAmRows * 128;      // rows of a block, rank values, bytes of a part of 128 rows of 64 values
// Chunks of 64 inputs that a sum on the tensor cores holds before it joins those before it, rounded: the cores cut their sums, always towards zero.  2048 rows, rank 64, error
// against 64 bits and us with all of a CTA's inputs in one sum and in sums of four chunks: 4096 inputs 8.2e-7, 84.2 / 4.0e-7, 85.2; 14336 inputs 3.0e-6, 109 / 4.0e-7, 113; 32768
// inputs 9.2e-6, 196 / 5.2e-7, 204; 512 rows of f32 weights, 14336 inputs 8.1e-6, 65.7 / 1.0e-6, 67.7.  (Plain f32: 5.9e-7, 1.1e-6, 2.2e-6, 6.0e-7.)
constexpr uint32_t kAmJoin = 4;
template <typename WT> struct AmParts { static constexpr uint32_t n = sizeof(WT) == 2 ? 1 : 3; };      // of the weights: bfloat16 ones are one part themselves
template <typename WT> constexpr uint32_t kAmRuns = sizeof(WT) == 2 ? 4 : 2;
// products, small ones first: {part of x, part of w}
template <typename WT> struct AmProducts { static constexpr uint32_t n = sizeof(WT) == 2 ? 3 : 6; };
template <typename WT> __device__ constexpr uint32_t am_x(uint32_t i) { return sizeof(WT) == 2 ? 2 - i : i == 0 ? 2 : i == 1 || i == 3 ? 1 : 0; }
template <typename WT> __device__ constexpr uint32_t am_w(uint32_t i) { return sizeof(WT) == 2 ? 0 : i == 0 || i == 3 || i == 5 ? 0 : i == 1 || i == 4 ? 1 : 2; }
// byte of piece c (16 bytes) of a row of 128 bytes in a K-major, 128-byte swizzled operand
__device__ __forceinline__ uint32_t am_at(uint32_t row, uint32_t c) { return row * 128 + ((c ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t am_idesc(uint32_t n) { return (1u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((128u >> 4) << 24); }      // bf16 x bf16 -> f32, 128 rows
// eight f32 values as 16 bytes of each of three parts
__device__ __forceinline__ void am_split(const float4 x, const float4 y, uint4 (&p)[3]) {
    split3(x.x, x.y, p[0].x, p[1].x, p[2].x); split3(x.z, x.w, p[0].y, p[1].y, p[2].y);
    split3(y.x, y.y, p[0].z, p[1].z, p[2].z); split3(y.z, y.w, p[0].w, p[1].w, p[2].w);
}
__device__ __forceinline__ void am_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Runs of a block's rows: {first row, end, adapter or what else}.  Found by warp 0; `skip` of a run leaves it out.  Everybody waits for it.
struct AmRun { int first, end, which; };
template <class Skip>
__device__ __forceinline__ void am_find_runs(const AdArgs& a, const BatchHead& head, uint32_t r0, int* which, AmRun* runs, uint32_t* count, const Skip& skip) {
    if (threadIdx.x < kAmRows) which[threadIdx.x] = r0 + threadIdx.x < a.B ? ad_of(a, head, r0 + threadIdx.x) : kAdIdle;
    __syncthreads();
    if (threadIdx.x < 32) {
        uint32_t n = 0;
        int open = -1;                                               // where the run that is not closed yet starts
        for (uint32_t w = 0; w < kAmRows; w += 32) {
            const uint32_t i = w + threadIdx.x;
            uint32_t starts = __ballot_sync(0xffffffffu, i == 0 || which[i] != which[i - 1]);
            for (; starts; starts &= starts - 1) {
                const int at = (int)w + __ffs(starts) - 1;
                if (open >= 0 && !skip(which[open])) { if (threadIdx.x == 0) runs[n] = {open, at, which[open]}; n++; }
                open = at;
            }
        }
        if (!skip(which[open])) { if (threadIdx.x == 0) runs[n] = {open, (int)kAmRows, which[open]}; n++; }
        if (threadIdx.x == 0) *count = n;
    }
    __syncthreads();
}
template <typename WT> struct AsLayout {
    // weights of bfloat16 sessions come a chunk ahead, through three slots; f32 ones are split as they come, into two
    static constexpr uint32_t weights = kAmRank * 128, w_run = AmParts<WT>::n * weights, w_slots = sizeof(WT) == 2 ? 3 : 2, w_slot = kAmRuns<WT> * w_run, x_stage = 3 * kAmPart;
    static constexpr uint32_t w = 2 * x_stage, which = w + w_slots * w_slot, runs = which + kAmRows * 4, bars = runs + kAmRows * 12, size = bars + 64 + 1024;
    static constexpr uint32_t width = kAmRank + 4;                   // of the partial sums, which take the first stage's place in the end
    static_assert(kAmRows * width * 4 <= x_stage, "partial sums");
};
template <typename WT>
__global__ void __launch_bounds__(256, 1) __cluster_dims__(kAfCluster, 1, 1) k_adapter_shrink(AdArgs a, const WT* __restrict__ wa, uint4* __restrict__ parts) {
    typedef AsLayout<WT> L;
    constexpr uint32_t kJoined = 256;                                // TMEM column of the joined sums, behind those under way
    static_assert(kAmJoin % 2 == 0 && kAmJoin >= 4 && kJoined >= kAmRuns<WT> * kAmRank, "pairs of chunks, TMEM columns");
    extern __shared__ uint8_t am_raw[];
    const uint32_t base = (smem_u32(am_raw) + 1023u) & ~1023u;
    uint8_t* const mem = am_raw + (base - smem_u32(am_raw));
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, share = blockIdx.x % kAfCluster, r0 = blockIdx.x / kAfCluster * kAmRows;
    int* const which = reinterpret_cast<int*>(mem + L::which);
    AmRun* const all = reinterpret_cast<AmRun*>(mem + L::runs);
    const uint32_t done = base + L::bars, tmem_slot = done + 16;
    uint32_t* const count = reinterpret_cast<uint32_t*>(mem + L::bars + 24);
    volatile uint32_t* const lost = count + 1;
    if (threadIdx.x == 0) {
        *lost = 0;
        mbar_init(done, 1); mbar_init(done + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const BatchHead head = batch_head(a.table, a.B);
    fence_before();
    am_find_runs(a, head, r0, which, all, count, [](int w) { return w < 0; });
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(mem + (tmem_slot - base)), n_runs = *count;
    const uint32_t chunks = (a.K + 63) / 64, per = (chunks + kAfCluster - 1) / kAfCluster, c0 = min(chunks, share * per), n = min(chunks, c0 + per) - c0;
    // thread: piece c (8 inputs) of rows p, p + 32, p + 64, p + 96 of x; of row p (and p + 32) of the weights
    const uint32_t c = threadIdx.x & 7, p = threadIdx.x >> 3;
    uint32_t uses = 0;                                               // chunks that have gone through the stages: use u takes stage u & 1
    bool ok = true;
    bool x_on[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x_on[i] = which[p + 32 * i] >= 0;
    // as many adapters at a time as accumulate side by side
    for (uint32_t e0 = 0; e0 < n_runs; e0 += kAmRuns<WT>) {
        const uint32_t runs = min(kAmRuns<WT>, n_runs - e0);
        const AmRun* const run = all + e0;
        const WT* w_from[kAmRuns<WT>];
#pragma unroll
        for (uint32_t i = 0; i < kAmRuns<WT>; i++) w_from[i] = wa + (size_t)run[min(i, runs - 1)].which * a.rank * a.K;
        float4 xa[4][2], xb[4][2];                                   // of the next even and odd chunk
        auto load = [&](uint32_t t, float4 (&x)[4][2]) {
            const uint32_t k = (c0 + t) * 64 + 8 * c;                // K is a multiple of eight here
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool on = t < n && k < a.K && x_on[i];
                const float* from = a.src + (size_t)(r0 + p + 32 * i) * a.src_rs + k;
                x[i][0] = on ? *reinterpret_cast<const float4*>(from) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                x[i][1] = on ? *reinterpret_cast<const float4*>(from + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        };
        auto weights = [&](uint32_t t, uint32_t slot) {
            const uint32_t k = (c0 + t) * 64 + 8 * c;
            if (t < n) {
#pragma unroll
                for (uint32_t i = 0; i < kAmRuns<WT>; i++) {
                    if (i >= runs) break;
#pragma unroll
                    for (uint32_t j = p; j < kAmRank; j += 32) {
                        const bool on = j < a.rank && k < a.K;
                        const uint32_t to = L::w + slot * L::w_slot + i * L::w_run + am_at(j, c);
                        const WT* from = on ? w_from[i] + (size_t)j * a.K + k : wa;
                        if constexpr (sizeof(WT) == 2) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + to), "l"(from), "r"(on ? 16 : 0) : "memory");
                        else {
                            uint4 w[3];
                            const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            am_split(on ? *reinterpret_cast<const float4*>(from) : zero, on ? *reinterpret_cast<const float4*>(from + 4) : zero, w);
#pragma unroll
                            for (int y = 0; y < 3; y++) *reinterpret_cast<uint4*>(mem + to + y * L::weights) = w[y];
                        }
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // Where the sums of kAmJoin chunks are under way, number g of them.  Up to two runs have room for two of them, so that one is joined to those before while the next one is
        // made; more runs wait for it.
        const bool twice = runs <= 2;
        auto at = [&](uint32_t g) { return tmem + (twice && (g & 1) ? 2 * kAmRank : 0u); };
        uint32_t slot = 0;                                           // of the weights of chunk t
        auto chunk = [&](uint32_t t, float4 (&x)[4][2]) {
            const uint32_t s = uses & 1;
            uint8_t* const out = mem + s * L::x_stage;
            if (uses >= 2 && ok) ok = __all_sync(0xffffffffu, mbar_wait(done + 8 * s, ((uses >> 1) - 1) & 1));
            const uint32_t after = slot + 1 == L::w_slots ? 0 : slot + 1;
            if constexpr (sizeof(WT) == 2) weights(t + 1, after); else weights(t, slot);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint4 w[3];
                am_split(x[i][0], x[i][1], w);
#pragma unroll
                for (int y = 0; y < 3; y++) *reinterpret_cast<uint4*>(out + y * kAmPart + am_at(p + 32 * i, c)) = w[y];
            }
            load(t + 2, x);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            am_proxy_fence();
            __syncthreads();
            if (warp == 0) {
                const uint32_t xs = desc_low(base) + s * (L::x_stage >> 4), w0 = desc_low(base + L::w) + slot * (L::w_slot >> 4), idesc = am_idesc(kAmRank), freed = done + 8 * s, to = at(t / kAmJoin);
                fence_after();
                if (elect_one() && ok) {
#pragma unroll
                    for (uint32_t i = 0; i < kAmRuns<WT>; i++) {
                        if (i >= runs) break;
#pragma unroll
                        for (uint32_t y = 0; y < AmProducts<WT>::n; y++)
#pragma unroll
                            for (uint32_t z = 0; z < 4; z++) {
                                const uint32_t xd = xs + am_x<WT>(y) * (kAmPart >> 4) + 2 * z, wd = w0 + (i * L::w_run + am_w<WT>(y) * L::weights) / 16 + 2 * z;
                                if (y == 0 && z == 0) { if (t % kAmJoin == 0) mma_ss<false>(to + i * kAmRank, xd, wd, idesc); else mma_ss<true>(to + i * kAmRank, xd, wd, idesc); }
                                else mma_ss<true>(to + i * kAmRank, xd, wd, idesc);
                            }
                    }
                    mma_commit(freed);
                }
                __syncwarp();
            }
            slot = after;
            uses++;
        };
        const uint32_t row = (warp & 3) * 32 + lane, col = 32 * (warp >> 2), lanes = ((warp & 3) * 32) << 16;
        // Sums of kAmJoin chunks (number g of them) join those of the chunks before
        auto join = [&](uint32_t g) {
            fence_after();
#pragma unroll 1
            for (uint32_t i = 0; i < runs; i++) {
                uint32_t v[32], w[32];
                tmem_ld(at(g) + lanes + i * kAmRank + col, v);
                if (g) tmem_ld(tmem + lanes + kJoined + i * kAmRank + col, w);
                tmem_wait_ld(v);
                if (g) {
                    tmem_wait_ld(w);
#pragma unroll
                    for (int y = 0; y < 32; y++) v[y] = __float_as_uint(__uint_as_float(v[y]) + __uint_as_float(w[y]));
                }
                tmem_st(tmem + lanes + kJoined + i * kAmRank + col, v);
            }
            tmem_wait_st();
            fence_before();
        };
        // products of the last chunk (1) or the one before (2)
        auto wait_for = [&](uint32_t back) { if (ok) ok = __all_sync(0xffffffffu, mbar_wait(done + 8 * ((uses - back) & 1), ((uses - back) >> 1) & 1)); };
        load(0, xa);
        load(1, xb);
        if constexpr (sizeof(WT) == 2) weights(0, 0);
#pragma unroll 1
        for (uint32_t t = 0; t < n; t += 2) {
            chunk(t, xa);
            if (t + 1 < n) chunk(t + 1, xb);
            if (!twice && (t + 2) % kAmJoin == 0 && t + 2 < n) { wait_for(1); join(t / kAmJoin); }
            if (twice && t && t % kAmJoin == 0) {                    // (chunk t + 1 has waited for the last of the sums before)
                if (t + 1 == n) wait_for(2);
                join(t / kAmJoin - 1);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // all products of these runs are there; their sums take the first stage's place
        if (n) wait_for(1);
        if (n > 1) wait_for(2);
        fence_after();
        if (!ok) *lost = 1;                                          // a warp whose wait ran out has written over operands that others read
        __syncthreads();
        ok = !*lost;
        float* const sums = reinterpret_cast<float*>(mem);           // [128][width]
#pragma unroll 1
        for (uint32_t i = 0; i < runs; i++) {
            uint32_t v[32];
            tmem_ld(at((n - 1) / kAmJoin) + lanes + i * kAmRank + col, v);
            tmem_wait_ld(v);
            if (n > kAmJoin) {
                uint32_t w[32];
                tmem_ld(tmem + lanes + kJoined + i * kAmRank + col, w);
                tmem_wait_ld(w);
#pragma unroll
                for (int y = 0; y < 32; y++) v[y] = __float_as_uint(__uint_as_float(v[y]) + __uint_as_float(w[y]));
            }
            if (row >= (uint32_t)run[i].first && row < (uint32_t)run[i].end) {
#pragma unroll
                for (int y = 0; y < 32; y += 4)
                    *reinterpret_cast<float4*>(sums + row * L::width + col + y) = !ok ? make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN) : !n ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                        : make_float4(__uint_as_float(v[y]), __uint_as_float(v[y + 1]), __uint_as_float(v[y + 2]), __uint_as_float(v[y + 3]));
            }
        }
        fence_before();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        // this CTA's sixteen rows: four rank values a thread
        {
            const uint32_t mine = share * (kAmRows / kAfCluster) + (threadIdx.x >> 4), j = 4 * (threadIdx.x & 15);
            if (mine >= (uint32_t)run[0].first && mine < (uint32_t)run[runs - 1].end && which[mine] >= 0) {
                float4 e[kAfCluster], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);      // all on their way before the first is added
#pragma unroll
                for (uint32_t x = 0; x < kAfCluster; x++) e[x] = af_remote4(smem_u32(sums + mine * L::width + j), x);
#pragma unroll
                for (uint32_t x = 0; x < kAfCluster; x++) { v.x += e[x].x; v.y += e[x].y; v.z += e[x].z; v.w += e[x].w; }
                const float f = a.scales ? a.scales[which[mine]] : 1.0f;
                uint2 w[3];
                split3(v.x * f, v.y * f, w[0].x, w[1].x, w[2].x);
                split3(v.z * f, v.w * f, w[0].y, w[1].y, w[2].y);
#pragma unroll
                for (int y = 0; y < 3; y++) reinterpret_cast<uint2*>(parts)[((size_t)y * a.B + r0 + mine) * (kAmRank / 4) + j / 4] = w[y];
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (!ok && threadIdx.x == 0) count_timeout();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

constexpr uint32_t kAxWriters = 256, kAxThreads = kAxWriters + 128;
template <typename WT> struct AxLayout {
    // turns: 32 rows of 64 outputs (68 floats a row: rows and columns of them meet different banks), two for each of 8 writing warps
    static constexpr uint32_t stages = sizeof(WT) == 2 ? 3 : 1, stage = AmParts<WT>::n * kAmPart, width = 68, turn = 32 * width * 4, ring = stages * stage;
    static constexpr uint32_t which = ring + 8 * 2 * turn, runs = which + kAmRows * 4, bars = runs + kAmRows * 12, size = bars + 128 + 1024;
};
// CTA (share of the outputs, block of 128 rows).  TMEM: sums of two tiles, the rows' rank values (A operand).
template <typename WT>
__global__ void __launch_bounds__(kAxThreads, 1) k_adapter_expand(AdArgs a, const WT* __restrict__ wb, const uint4* __restrict__ parts, uint32_t quads) {
    typedef AxLayout<WT> L;
    constexpr uint32_t kH = 256;                                     // TMEM column of the rank values: 32 a part
    extern __shared__ uint8_t am_raw[];
    const uint32_t base = (smem_u32(am_raw) + 1023u) & ~1023u;
    uint8_t* const mem = am_raw + (base - smem_u32(am_raw));
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, r0 = blockIdx.y * kAmRows;
    AmRun* const runs = reinterpret_cast<AmRun*>(mem + L::runs);
    const uint32_t full = base + L::bars, empty = full + 8 * L::stages, sum_full = empty + 8 * L::stages, sum_empty = sum_full + 16, tmem_slot = sum_empty + 16;
    uint32_t* const count = reinterpret_cast<uint32_t*>(mem + (tmem_slot + 8 - base));
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < L::stages; i++) { mbar_init(full + 8 * i, 4); mbar_init(empty + 8 * i, 1); }
        for (uint32_t i = 0; i < 2; i++) { mbar_init(sum_full + 8 * i, 1); mbar_init(sum_empty + 8 * i, 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const BatchHead head = batch_head(a.table, a.B);
    const bool in_place = a.base == a.dst;
    int* const which = reinterpret_cast<int*>(mem + L::which);
    fence_before();
    am_find_runs(a, head, r0, which, runs, count, [](int w) { return w < 0; });
    fence_after();
    const uint32_t tiles = (a.N + 127) / 128, per = (tiles + gridDim.x - 1) / gridDim.x, t0 = min(tiles, blockIdx.x * per), n = min(tiles, t0 + per) - t0, n_runs = *count;
    bool ok = true;
    // The rows' rank values, a row a lane.  Those of rows without any are whatever was there: their outputs are left out.
    if (warp < 4) {
        const uint32_t row = r0 + 32 * warp + lane;
#pragma unroll
        for (uint32_t y = 0; y < 3; y++) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint4 u = row < a.B ? parts[((size_t)y * a.B + row) * 8 + i] : make_uint4(0, 0, 0, 0);
                v[4 * i] = u.x; v[4 * i + 1] = u.y; v[4 * i + 2] = u.z; v[4 * i + 3] = u.w;
            }
            tmem_st((32 * warp << 16) + kH + 32 * y, v);
        }
        tmem_wait_st();
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp >= 8) {
        // bring weights, issue: of a tile one run of rows after the other
        const uint32_t id = threadIdx.x - kAxWriters, c = id & 7, items = n * n_runs;      // piece c of rows id / 8 + 16 i
        uint32_t slot = 0, phase = 1, at_slot = 0, at_phase = 0, f_tile = 0, f_run = 0;
        auto fill = [&]() {                                          // the next stage
            const int adapter = runs[f_run].which;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, phase));
            if (ok) {                                                // otherwise the stage may still be read
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    const uint32_t row = (id >> 3) + 16 * i, o = (t0 + f_tile) * 128 + row, to = slot * L::stage + am_at(row, c);
                    const bool on = o < a.N && 8 * c < a.rank;       // the rank is a multiple of eight here
                    const WT* from = on ? wb + ((size_t)adapter * a.N + o) * a.rank + 8 * c : wb;
                    if constexpr (sizeof(WT) == 2) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + to), "l"(from), "r"(on ? 16 : 0) : "memory");
                    else {
                        uint4 w[3];
                        const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        am_split(on ? *reinterpret_cast<const float4*>(from) : zero, on ? *reinterpret_cast<const float4*>(from + 4) : zero, w);
#pragma unroll
                        for (int y = 0; y < 3; y++) *reinterpret_cast<uint4*>(mem + to + y * kAmPart) = w[y];
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++slot == L::stages) { slot = 0; phase ^= 1; }
            if (++f_run == n_runs) { f_run = 0; f_tile++; }
        };
        constexpr uint32_t kAhead = L::stages - 1;                   // stages that are on their way while one is used
        // (a group for every stage ahead, empty where there are fewer items: the waits below count groups)
        for (uint32_t i = 0; i + 1 < L::stages; i++) { if (i < items) fill(); else asm volatile("cp.async.commit_group;" ::: "memory"); }
        for (uint32_t item = 0; item < items; item++) {
            if (item + kAhead < items) fill(); else asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
            am_proxy_fence();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(full + 8 * at_slot);     // (otherwise the waits for this stage run out too, and its sums are never there)
            if (warp == 8) {
                const uint32_t d = (item & 1) * 128, w0 = desc_low(base) + at_slot * (L::stage >> 4), freed = empty + 8 * at_slot, idesc = am_idesc(128);
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * at_slot, at_phase));
                if (ok && item >= 2) ok = __all_sync(0xffffffffu, mbar_wait(sum_empty + 8 * (item & 1), ((item >> 1) - 1) & 1));
                fence_after();
                if (elect_one() && ok) {
#pragma unroll
                    for (uint32_t y = 0; y < AmProducts<WT>::n; y++)
#pragma unroll
                        for (uint32_t z = 0; z < 4; z++) {
                            const uint32_t h = kH + 32 * am_x<WT>(y) + 8 * z, ws = w0 + am_w<WT>(y) * (kAmPart >> 4) + 2 * z;
                            if (y == 0 && z == 0) mma_ts<false>(d, h, ws, idesc); else mma_ts<true>(d, h, ws, idesc);
                        }
                    mma_commit(sum_full + 8 * (item & 1));
                    mma_commit(freed);
                }
                __syncwarp();
            }
            if (++at_slot == L::stages) { at_slot = 0; at_phase ^= 1; }
        }
    } else {
        // Add the base, write: 32 rows and 64 outputs of a tile a warp.  The base comes by whole rows, a tile ahead; a lane adds the sums of its row, and whole rows leave.
        const uint32_t row0 = (warp & 3) * 32, col0 = 64 * (warp >> 2), lr = lane >> 4, lc = 4 * (lane & 15), lane_row = row0 + lane;
        float* const ring = reinterpret_cast<float*>(mem + L::ring + warp * 2 * L::turn);
        const uint32_t ring_at = smem_u32(ring);
        uint32_t live = 0, bad = 0, none = 0;                        // rows of the warp: with a result, a result that is not a number, the base alone
        {
            const int w = which[lane_row];
            live = __ballot_sync(0xffffffffu, w != kAdIdle && !(w == kAdNone && in_place)); bad = __ballot_sync(0xffffffffu, w == kAdBad); none = __ballot_sync(0xffffffffu, w < 0);
        }
        auto fetch = [&](uint32_t t) {
            const uint32_t o = (t0 + t) * 128 + col0 + lc;
            if (t < n && quads) {
                const bool in = o + 4 <= a.N;                        // zeros otherwise
#pragma unroll 4
                for (uint32_t x = 0; x < 16; x++) {
                    const uint32_t r = 2 * x + lr;
                    if ((live & ~bad) >> r & 1)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring_at + (t & 1) * L::turn + r * (4 * L::width) + 4 * lc), "l"(in ? a.base + (size_t)(r0 + row0 + r) * a.base_rs + o : a.base), "r"(in ? 16 : 0) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        fetch(0);
        uint32_t item = 0;
        for (uint32_t t = 0; t < n; t++) {
            fetch(t + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            float* const turn = ring + (t & 1) * (L::turn / 4);
            if (!quads) {
                for (uint32_t x = 0; x < 64; x++) turn[lane * L::width + x] = 0.0f;
            }
            for (uint32_t e = 0; e < n_runs; e++, item++) {
                const bool here = runs[e].first < (int)row0 + 32 && runs[e].end > (int)row0, mine = runs[e].first <= (int)lane_row && runs[e].end > (int)lane_row;
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(sum_full + 8 * (item & 1), (item >> 1) & 1));
                fence_after();
                if (here) {
#pragma unroll
                    for (uint32_t h = 0; h < 64; h += 32) {
                        uint32_t v[32];
                        tmem_ld((row0 << 16) + (item & 1) * 128 + col0 + h, v);
                        tmem_wait_ld(v);
                        if (mine) {
#pragma unroll
                            for (int x = 0; x < 32; x += 4) {
                                float4* const to = reinterpret_cast<float4*>(turn + lane * L::width + h + x);
                                float4 b = *to;
                                b.x += __uint_as_float(v[x]); b.y += __uint_as_float(v[x + 1]); b.z += __uint_as_float(v[x + 2]); b.w += __uint_as_float(v[x + 3]);
                                *to = ok ? b : make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN);
                            }
                        }
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(sum_empty + 8 * (item & 1));
            }
            const uint32_t o = (t0 + t) * 128 + col0 + lc;
            const bool all = quads && o + 4 <= a.N;
#pragma unroll 4
            for (uint32_t x = 0; x < 16; x++) {
                const uint32_t r = 2 * x + lr;
                if (!(live >> r & 1)) continue;
                float4 v = *reinterpret_cast<const float4*>(turn + r * L::width + lc);
                if (bad >> r & 1) v = make_float4(kBatchNaN, kBatchNaN, kBatchNaN, kBatchNaN);
                float* const to = a.dst + (size_t)(r0 + row0 + r) * a.dst_rs + o;
                if (all) *reinterpret_cast<float4*>(to) = v;
                else {
                    const float* from = a.base + (size_t)(r0 + row0 + r) * a.base_rs + o;      // not copied: `v` is the sum alone
#pragma unroll
                    for (uint32_t z = 0; z < 4; z++) if (o + z < a.N) to[z] = bad >> r & 1 ? kBatchNaN : none >> r & 1 ? from[z] : from[z] + (&v.x)[z];
                }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    if (!ok && lane == 0) count_timeout();
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(0u) : "memory");
}

// More rows than kAmLeast go in blocks, where rank and strides allow their 16-byte pieces, unless the op says which way to take: a block walks its runs one after the other, and only the
// host knows how long they are.  us in blocks and by runs of eight: 4096 inputs and outputs, rank 16: 256 rows in runs of 64 26.7 / 20.4, 512 in runs of 128 24.6 / 30.4, of 8 102 / 27, of one 712 / 45;
// 14336 outputs, rank 64: 64 rows of one run 27 / 42, 256 in runs of 128 26.5 / 57.7.  (The length of runs decides, which no size says: the number of rows is right where many rows are
// prompts and few rows are decoded, and `form` is for the rest.)
constexpr uint32_t kAmLeast = 256;
bool many_rows(const ZgSeqOp& s) {
    const uint32_t B = s.n[0], K = s.n[2], rank = s.n[3], form = s.n[9];
    return (form == 2 || (form == 0 && B > kAmLeast)) && K % 8 == 0 && rank % 8 == 0 && rank <= kAmRank && s.n[5] % 4 == 0 && s.off[2] % 4 == 0 && s.off[0] % 8 == 0 && s.off[1] % 8 == 0;
}
template <typename WT>
bool launch_few(const AdArgs& a, const WT* wa, const WT* wb, cudaStream_t st) {
    auto aligned = [](const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    const uint32_t V = WVec<WT>::n, k_slice = ((a.K + kAfCluster - 1) / kAfCluster + V - 1) / V * V, n_slice = ((a.N + kAfCluster - 1) / kAfCluster + 7) / 8 * 8;
    const uint32_t vec_k = a.K % V == 0 && a.src_rs % 4 == 0 && aligned(wa, 16) && aligned(a.src, 16);
    const uint32_t vec_j = a.rank % 4 == 0 && aligned(wb, 4 * sizeof(WT));
    // Several lanes an output for long weights or many outputs; a lane an output, in a kernel of half the registers, otherwise.  64 rows of 4096 inputs, a run each, us by several
    // lanes and by one: rank 8, 2048 outputs 10.3 / 6.3; rank 16, 4096 outputs 10.3 / 8.4, 8192 12.4 / 10.3, 14336 14.4 / 19.7; rank 32, 4096 12.4 / 14.4; rank 64, 4096 18.5 / 42.8
    constexpr uint32_t E = 16 / sizeof(WT);
    uint32_t lanes = 1;
    while (lanes * E < a.rank) lanes *= 2;
    const bool wide = a.rank % E == 0 && lanes <= 16 && aligned(wb, 16) && (a.rank * sizeof(WT) >= 64 || n_slice > 1024);
    // A slice begins at n_slice rank weights from the adapter's, which is N rank from the next one's
    const size_t bytes = (size_t)n_slice * a.rank * sizeof(WT);
    const uint32_t stage = bytes <= kAfStage && aligned(wb, 16) && (size_t)a.N * a.rank * sizeof(WT) % 16 == 0 ? (uint32_t)((bytes + 15) & ~(size_t)15) : 0;
    const size_t smem = stage + 2 * kAfRows * sizeof(float) * ((a.rank + 3) / 4 * 4);
    constexpr size_t limit = kAfStage + 2 * kAfRows * sizeof(float) * 1024;
    if (wide) {
        if (!zg_smem_limit<k_adapter_few<WT, true>>(limit)) return false;
        launch_pdl(k_adapter_few<WT, true>, dim3(a.B * kAfCluster), dim3(kAfThreads), smem, st, a, wa, wb, k_slice, n_slice, vec_k, vec_j, lanes, stage);
    } else {
        if (!zg_smem_limit<k_adapter_few<WT, false>>(limit)) return false;
        launch_pdl(k_adapter_few<WT, false>, dim3(a.B * kAfCluster), dim3(kAfThreads), smem, st, a, wa, wb, k_slice, n_slice, vec_k, vec_j, lanes, stage);
    }
    return true;
}
template <typename WT>
bool launch_many(const AdArgs& a, const WT* wa, const WT* wb, float* parts, cudaStream_t st) {
    if (!zg_smem_limit<k_adapter_shrink<WT>>(AsLayout<WT>::size) || !zg_smem_limit<k_adapter_expand<WT>>(AxLayout<WT>::size)) return false;
    const uint32_t blocks = (a.B + kAmRows - 1) / kAmRows, tiles = (a.N + 127) / 128;
    launch_pdl(k_adapter_shrink<WT>, dim3(blocks * kAfCluster), dim3(256), AsLayout<WT>::size, st, a, wa, reinterpret_cast<uint4*>(parts));
    ZG_COUNT_LAUNCH();
    const uint32_t quads = a.dst_rs % 4 == 0 && a.base_rs % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.dst) | reinterpret_cast<uintptr_t>(a.base)) & 15) == 0;
    launch_pdl(k_adapter_expand<WT>, dim3(std::max(1u, std::min(tiles, zg_sm_count() / blocks)), blocks), dim3(kAxThreads), AxLayout<WT>::size, st, a, wb, reinterpret_cast<const uint4*>(parts), quads);
    return true;
}

}  // namespace

bool zg_adapter_linear_valid(const ZgSeqOp& s, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto have = [&](int i) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs; };
    auto fits = [&](int i, size_t off, size_t n) { return have(i) && off + n <= elems[s.buf[i]]; };
    auto wfits = [&](int i, uint32_t wdt, size_t off, size_t n) { return wdt <= ZG_W_BF16 && have(i) && (wdt == ZG_W_BF16 ? (off + n + 1) / 2 : off + n) <= elems[s.buf[i]]; };
    if (s.n[9] > 2) return fail("adapter_linear: form");
    const size_t B = s.n[0], N = s.n[1], K = s.n[2], rank = s.n[3], A = s.n[4], srs = s.n[5], drs = s.n[6], brs = s.n[8];
    if (!B || !N || !K || !rank || !A || B > 65536 || rank > 1024 || A > ((size_t)1 << 48) / (rank * std::max(N, K))) return fail("adapter_linear: shape");      // (no product below passes 64 bits)
    if ((B > 1 && (srs < K || drs < N || brs < N)) || !fits(0, s.off[3], (B - 1) * drs + N) || !fits(1, s.off[2], (B - 1) * srs + K) || !fits(5, s.off[5], (B - 1) * brs + N)) return fail("adapter_linear: rows");
    if (!wfits(2, s.n[7], s.off[0], A * rank * K) || !wfits(2, s.n[7], s.off[1], A * rank * N)) return fail("adapter_linear: weights");
    if (s.buf[3] != ZG_NO_BUF && !fits(3, s.off[4], A)) return fail("adapter_linear: scales");
    if (!fits(4, 0, ZG_BATCH_ROWS + 4 * B)) return fail("adapter_linear: table");
    if (s.buf[0] == s.buf[1] || s.buf[0] == s.buf[2] || s.buf[0] == s.buf[3] || s.buf[0] == s.buf[4]) return fail("adapter_linear: in place");
    if (s.buf[0] == s.buf[5] && (s.off[3] != s.off[5] || drs != brs)) return fail("adapter_linear: a base that overlaps the destination has to be the destination");
    return true;
}
size_t zg_adapter_linear_scratch_elems(const ZgSeqOp& s) { return many_rows(s) ? (size_t)3 * s.n[0] * kAmRank / 2 : 0; }      // rank values in three bfloat16 parts
bool zg_launch_adapter_linear(const ZgOp& op, float* const* bufs, float* scratch, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    AdArgs a;
    a.dst = bufs[s.buf[0]] + s.off[3]; a.src = bufs[s.buf[1]] + s.off[2]; a.base = bufs[s.buf[5]] + s.off[5]; a.scales = s.buf[3] != ZG_NO_BUF ? bufs[s.buf[3]] + s.off[4] : nullptr; a.table = bufs[s.buf[4]];
    a.B = s.n[0]; a.N = s.n[1]; a.K = s.n[2]; a.rank = s.n[3]; a.adapters = s.n[4]; a.src_rs = s.n[5]; a.dst_rs = s.n[6]; a.base_rs = s.n[8];
    bool ok = false;
    const bool many = scratch && many_rows(s);
    ZG_SEQ_WDT(s.n[7], ok = many ? launch_many<WT>(a, wptr<WT>(bufs, s.buf[2], s.off[0]), wptr<WT>(bufs, s.buf[2], s.off[1]), scratch, st)
                                 : launch_few<WT>(a, wptr<WT>(bufs, s.buf[2], s.off[0]), wptr<WT>(bufs, s.buf[2], s.off[1]), st));
    if (!ok) return false;
    ZG_SEQ_CHECK();
    return true;
}
unsigned int zg_adapter_timeouts() { return tc_timeouts(); }
