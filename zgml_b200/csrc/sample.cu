// SAMPLE (parameter pack in include/zgml_cuda.h): the next token of each row of logits.
#include "batch_table.cuh"

#include <algorithm>

namespace {

struct SmArgs {
    int32_t* dst; const float* logits; const float* table; float* probability;
    uint32_t B, V, rs, slice;
};
constexpr uint32_t kSmThreads = 512, kSmWarps = kSmThreads / 32, kSmBins = 1024, kSmList = 512, kSmCluster = 8, kSmSlice = 40960;
constexpr uint32_t kSmIndexBits = 20;
typedef unsigned long long u64;

struct SmShared {
    u64 mass[kSmBins]; uint32_t count[kSmBins];
    ulonglong2 list[kSmList], all_list[kSmList];                     // {order, weight} of candidates, own and of the cluster
    u64 best, total, warp_mass[kSmWarps], found_mass, threshold;
    uint32_t nan, n_list, found_count, found_bin, warp_count[kSmWarps];
};
__device__ __forceinline__ uint32_t sm_at(const void* p, uint32_t rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ uint32_t sm_peer(const uint32_t* p, uint32_t rank) { uint32_t v; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sm_at(p, rank)) : "memory"); return v; }
__device__ __forceinline__ u64 sm_peer(const u64* p, uint32_t rank) { u64 v; asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sm_at(p, rank)) : "memory"); return v; }
__device__ __forceinline__ ulonglong2 sm_peer(const ulonglong2* p, uint32_t rank) {
    ulonglong2 v;
    asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "r"(sm_at(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void sm_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// numbers that are ordered as the floats are (no NaN; -0 has become 0)
__device__ __forceinline__ uint32_t sm_key(float z) { const uint32_t b = __float_as_uint(z); return b & 0x80000000u ? ~b : b | 0x80000000u; }
__device__ __forceinline__ float sm_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// what decides who comes first: the logit, then the lower index
__device__ __forceinline__ u64 sm_order(float z, uint32_t index) { return ((u64)sm_key(z) << kSmIndexBits) | ((1u << kSmIndexBits) - 1 - index); }
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A cluster per row, its CTAs each a slice of the vocabulary in shared memory.  What top_k and top_p cut at is found by counts (sums of weights) of the tokens by bins of
// logits, the bin where the target is passed looked at more closely until at most kSmList candidates are left, which are ranked one against the other.  Weights are whole
// multiples of 2^-43 of the largest, their sums exact in 64 bits, so that no order of additions changes a choice.
__global__ void __launch_bounds__(kSmThreads) k_sample(const SmArgs a) {
    pdl_enter();
    extern __shared__ float4 sm_mem[];
    __shared__ SmShared sh;
    float* const z = reinterpret_cast<float*>(sm_mem);
    const uint32_t r = blockIdx.y, rank = blockIdx.x, C = gridDim.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const BatchHead head = batch_head(a.table, a.B);
    const int4 w0 = *reinterpret_cast<const int4*>(a.table + ZG_BATCH_ROWS + (size_t)ZG_SAMPLE_WORDS * r);
    const float u = a.table[ZG_BATCH_ROWS + (size_t)ZG_SAMPLE_WORDS * r + 4], T = __int_as_float(w0.x), top_p = __int_as_float(w0.z), min_p = __int_as_float(w0.w);
    const int32_t top_k = w0.y;
    if (r >= head.rows || top_k < 0) return;                         // (the whole cluster)
    const bool ok = T >= 0.0f && T < INFINITY && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    const uint32_t v0 = min(rank * a.slice, a.V), n = min(a.slice, a.V - v0);
    const float* src = a.logits + (size_t)r * a.rs + v0;
    if (tid == 0) { sh.best = 0; sh.nan = 0; }
    __syncthreads();
    {
        u64 best = 0;
        bool nan = false;
        for (uint32_t i = tid; i < n; i += kSmThreads) {
            const float x = src[i] + 0.0f;
            z[i] = x;
            nan = nan || x != x;
            best = max(best, sm_order(x, v0 + i));
        }
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        nan = __any_sync(0xffffffffu, nan);
        if (lane == 0) { atomicMax(&sh.best, best); if (nan) sh.nan = 1; }
    }
    __syncthreads();
    if (C > 1) sm_cluster_sync();
    u64 best = 0;
    bool bad = !ok;
    for (uint32_t c = 0; c < C; c++) { best = max(best, sm_peer(&sh.best, c)); bad = bad || sm_peer(&sh.nan, c); }
    const float M = sm_value((uint32_t)(best >> kSmIndexBits));
    bad = bad || M == -INFINITY;
    const bool greedy = T == 0.0f;
    if (bad || greedy) {
        if (rank == 0 && tid == 0) {
            a.dst[r] = bad ? -1 : (int32_t)((1u << kSmIndexBits) - 1 - (uint32_t)(best & ((1u << kSmIndexBits) - 1)));
            if (a.probability) a.probability[r] = bad ? kBatchNaN : 1.0f;
        }
        if (C > 1) sm_cluster_sync();                                // no CTA leaves while it is read
        return;
    }
    const double inv_t = 1.0 / (double)T;
    const float bins_at = 32.0f / T;                                 // bins of 1 / 32 of an exponent; what is below e^-32 has no weight
    const double least = log((double)min_p);                         // (compared as exponents: those of tokens just below the largest logit round to 1)
    auto exponent = [&](float x) { return x == M ? 0.0 : ((double)x - (double)M) * inv_t; };
    auto share = [&](float x) { return exp(exponent(x)); };
    auto weight = [&](float x) { return __double2ull_rn(share(x) * 8796093022208.0); };      // 2^43
    auto bin_of = [&](float x) { const float d = (M - x) * bins_at; return d < (float)kSmBins ? (uint32_t)d : x == M ? 0u : kSmBins - 1; };
    u64 threshold = 0;
    for (int by_mass = 0; by_mass < 2; by_mass++) {
        if (by_mass ? top_p >= 1.0f : top_k == 0 || (uint32_t)top_k >= a.V) continue;
        u64 lo = threshold, hi = best, above = 0, target = top_k;
        uint32_t shift = 0;
        bool linear = true;
        for (;;) {
            for (uint32_t i = tid; i < kSmBins; i += kSmThreads) { sh.count[i] = 0; sh.mass[i] = 0; }
            if (tid == 0) sh.n_list = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += kSmThreads) {
                const float x = z[i];
                const u64 o = sm_order(x, v0 + i);
                if (o < lo || o > hi) continue;
                const uint32_t b = linear ? bin_of(x) : (uint32_t)((hi - o) >> shift);
                atomicAdd(&sh.count[b], 1u);
                if (by_mass) { const u64 w = weight(x); if (w) atomicAdd(&sh.mass[b], w); }
            }
            __syncthreads();
            if (C > 1) sm_cluster_sync();
            // a thread adds up two neighbours of the cluster's bins, and the block finds the one in which the target is reached
            u64 mine[2];
            uint32_t here[2];
            for (int j = 0; j < 2; j++) {
                const uint32_t b = 2 * tid + j;
                u64 m = 0;
                uint32_t k = 0;
                for (uint32_t c = 0; c < C; c++) { k += sm_peer(&sh.count[b], c); if (by_mass) m += sm_peer(&sh.mass[b], c); }
                here[j] = k;
                mine[j] = by_mass ? m : k;
            }
            u64 before = mine[0] + mine[1];
            for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, before, o); if (lane >= (uint32_t)o) before += t; }
            if (lane == 31) sh.warp_mass[warp] = before;
            __syncthreads();
            u64 all = 0;
            for (uint32_t i = 0; i < kSmWarps; i++) { if (i < warp) before += sh.warp_mass[i]; all += sh.warp_mass[i]; }
            if (by_mass && linear) target = max((u64)1, (u64)ceil((double)top_p * (double)all));
            before += above - mine[0] - mine[1];
            for (int j = 0; j < 2; j++) {
                if (before < target && before + mine[j] >= target) { sh.found_bin = 2 * tid + j; sh.found_count = here[j]; sh.found_mass = before; }
                before += mine[j];
            }
            __syncthreads();
            const uint32_t bin = sh.found_bin, count = sh.found_count;
            above = sh.found_mass;
            // where the bin lies in the order
            if (linear) {
                auto bound = [&](bool upper) {                       // largest key whose bin is >= bin (upper), or smallest one whose bin is <= bin
                    uint32_t l = 0x007fffffu, h = (uint32_t)(best >> kSmIndexBits);      // keys from -inf to the largest logit's
                    while (l < h) {
                        const uint32_t m = l + (h - l + (upper ? 1 : 0)) / 2, b = bin_of(sm_value(m));
                        if (upper) { if (b >= bin) l = m; else h = m - 1; }
                        else { if (b <= bin) h = m; else l = m + 1; }
                    }
                    return l;
                };
                hi = min(hi, ((u64)bound(true) << kSmIndexBits) | ((1u << kSmIndexBits) - 1));
                lo = max(lo, (u64)bound(false) << kSmIndexBits);
                linear = false;
            } else {
                hi -= (u64)bin << shift;
                lo = max(lo, hi >= (1ull << shift) - 1 ? hi - ((1ull << shift) - 1) : 0);
            }
            if (C > 1) sm_cluster_sync();                            // (peers have read the bins)
            if (count > kSmList) {
                shift = 0;
                while ((hi - lo) >> shift >= kSmBins) shift++;
                continue;
            }
            for (uint32_t i = tid; i < n; i += kSmThreads) {
                const float x = z[i];
                const u64 o = sm_order(x, v0 + i);
                if (o < lo || o > hi) continue;
                sh.list[atomicAdd(&sh.n_list, 1u)] = make_ulonglong2(o, by_mass ? weight(x) : 1);
            }
            __syncthreads();
            if (C > 1) sm_cluster_sync();
            for (uint32_t c = 0, at = 0; c < C; c++) {
                const uint32_t k = sm_peer(&sh.n_list, c);
                for (uint32_t i = tid; i < k; i += kSmThreads) sh.all_list[at + i] = sm_peer(&sh.list[i], c);
                at += k;
            }
            __syncthreads();
            if (tid < count) {
                const ulonglong2 me = sh.all_list[tid];
                u64 ahead = above;
                for (uint32_t i = 0; i < count; i++) { const ulonglong2 x = sh.all_list[i]; if (x.x > me.x) ahead += x.y; }
                if (ahead < target && ahead + me.y >= target) sh.threshold = me.x;
            }
            __syncthreads();
            threshold = sh.threshold;
            if (C > 1) sm_cluster_sync();                            // (peers have read the list)
            break;
        }
    }
    // the draw: sums of what stays by warps' parts, then the part in which u of all is passed
    const uint32_t part = ((n + kSmWarps - 1) / kSmWarps + 31) / 32 * 32, from = min(warp * part, n), to = min(from + part, n);
    auto stays = [&](uint32_t i) {
        const float x = z[i];
        if (sm_order(x, v0 + i) < threshold) return (u64)0;
        return exponent(x) >= least ? (u64)weight(x) : (u64)0;
    };
    u64 sum = 0;
    for (uint32_t i = from + lane; i < to; i += 32) sum += stays(i);
    sum = warp_sum64(sum);
    if (lane == 0) sh.warp_mass[warp] = sum;
    __syncthreads();
    if (tid == 0) { u64 t = 0; for (uint32_t i = 0; i < kSmWarps; i++) t += sh.warp_mass[i]; sh.total = t; }
    __syncthreads();
    if (C > 1) sm_cluster_sync();
    u64 all = 0, base = 0;
    for (uint32_t c = 0; c < C; c++) { const u64 t = sm_peer(&sh.total, c); all += t; if (c < rank) base += t; }
    const double drawn = (double)u * (double)all;
    for (uint32_t i = 0; i < warp; i++) base += sh.warp_mass[i];
    if (!((double)base > drawn) && (double)(base + sum) > drawn) {
        for (uint32_t i = from; i < to; i += 32) {
            const u64 w = i + lane < to ? stays(i + lane) : 0;
            u64 upto = w;
            for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += t; }
            const uint32_t passed = __ballot_sync(0xffffffffu, (double)(base + upto) > drawn);
            if (passed) {
                if ((int)lane == __ffs(passed) - 1) {
                    a.dst[r] = (int32_t)(v0 + i + lane);
                    if (a.probability) a.probability[r] = (float)(share(z[i + lane]) * 8796093022208.0 / (double)all);
                }
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (C > 1) sm_cluster_sync();                                    // no CTA leaves while its sums are read
}

}  // namespace

bool zg_sample_valid(const ZgSeqOp& s, const size_t* elems, size_t n_bufs, char* why, size_t why_n) {
    auto fail = [&](const char* m) { snprintf(why, why_n, "%s", m); return false; };
    auto fits = [&](int i, size_t off, size_t n) { return s.buf[i] != ZG_NO_BUF && s.buf[i] < n_bufs && off + n <= elems[s.buf[i]]; };
    const size_t B = s.n[0], V = s.n[1], rs = s.n[2];
    if (!B || B > 65535 || !V || V > kSmCluster * kSmSlice) return fail("sample: shape");
    if ((B > 1 && rs < V) || !fits(1, s.off[1], (B - 1) * rs + V) || !fits(0, s.off[0], B) || !fits(2, 0, ZG_BATCH_ROWS + ZG_SAMPLE_WORDS * B)) return fail("sample: rows or table");
    if (s.buf[3] != ZG_NO_BUF && !fits(3, s.off[2], B)) return fail("sample: probabilities");
    for (int i = 1; i < 4; i++) if (s.buf[i] == s.buf[0] || (i < 3 && s.buf[3] == s.buf[i])) return fail("sample: in place");
    return true;
}
bool zg_launch_sample(const ZgOp& op, float* const* bufs, cudaStream_t st) {
    const ZgSeqOp& s = op.u.seq;
    SmArgs a;
    a.dst = reinterpret_cast<int32_t*>(bufs[s.buf[0]]) + s.off[0]; a.logits = bufs[s.buf[1]] + s.off[1]; a.table = bufs[s.buf[2]];
    a.probability = s.buf[3] == ZG_NO_BUF ? nullptr : bufs[s.buf[3]] + s.off[2];
    a.B = s.n[0]; a.V = s.n[1]; a.rs = s.n[2];
    const uint32_t C = a.V <= 1024 ? 1 : kSmCluster;
    a.slice = ((a.V + C - 1) / C + 3) / 4 * 4;
    if (!zg_smem_limit<k_sample>(sizeof(float) * kSmSlice)) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C, a.B); cfg.blockDim = dim3(kSmThreads); cfg.dynamicSmemBytes = sizeof(float) * a.slice; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_zg_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_sample, a);
    ZG_SEQ_CHECK();
    return true;
}
