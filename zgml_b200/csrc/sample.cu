// SAMPLE (parameter pack in include/zgml_cuda.h): the next token of each row of logits.
#include "batch_table.cuh"

#include <algorithm>
#include <type_traits>

namespace {

struct SmArgs {
    int32_t* dst; const float* logits; const float* table; float* probability;
    uint32_t B, V, rs, slice, vec;
};
constexpr uint32_t kSmBins = 1024, kSmList = 1024, kSmCluster = 8, kSmSlice = 40960, kSmHalf = 16384;      // tokens of a slice at most; those that leave room for another CTA
constexpr uint32_t kSmIndexBits = 20, kSmIndexMask = (1u << kSmIndexBits) - 1;
constexpr double kSmOne = 8796093022208.0;                           // 2^43: the largest weight
typedef unsigned long long u64;

struct SmShared {
    alignas(16) uint32_t mass_low[kSmBins], mass_high[kSmBins], count[kSmBins];      // (sums of 64 bits by words: additions of 64 bits to shared memory are loops)
    ulonglong2 list[kSmList], all_list[kSmList];                     // {order, weight} of candidates, own and of the cluster
    double table[32];                                                // 2^(43 + i / 32)
    u64 best, total, warp_mass[32], group_mass[32], found_mass, threshold, found_target;
    uint32_t n_list[2], n_all, n_picked, span[2], found_count, found_bin, found_upto, warp_count[32], group_count[32];      // groups of 32 bins
};
__device__ __forceinline__ uint32_t sm_at(const void* p, uint32_t rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
// the same place of another CTA of the cluster, as an address of ordinary loads, of which many are under way at once
template <class X>
__device__ __forceinline__ const X* sm_peer(const X* p, uint32_t rank) {
    const X* at;
    asm("mapa.u64 %0, %1, %2;" : "=l"(at) : "l"(p), "r"(rank));
    return at;
}
__device__ __forceinline__ void sm_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void sm_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// numbers that are ordered as the floats are (no NaN; -0 has become 0)
__device__ __forceinline__ uint32_t sm_key(float z) { const uint32_t b = __float_as_uint(z); return b & 0x80000000u ? ~b : b | 0x80000000u; }
__device__ __forceinline__ float sm_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// what decides who comes first: the logit, then the lower index
__device__ __forceinline__ u64 sm_order(float z, uint32_t index) { return ((u64)sm_key(z) << kSmIndexBits) | (kSmIndexMask - index); }
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Weights round(2^43 e^x) of exponents x <= 0: 2^(k / 32) of a table times the exponential's series up to r^5, |r| <= ln 2 / 64, whose next term is below 2^-48 (reduction by a table:
// P. Tang, ACM Transactions on Mathematical Software 15, 1989).  Whole numbers are taken from the mantissa of sums with 2^52 and 1.5 * 2^52.
constexpr double kSmShift = 6755399441055744.0, kSmSteps = 46.166241308446828384;      // 1.5 * 2^52; 32 / ln 2
// t: the exponent in 32nds of a power of two, -3000 at least; *k: t rounded.  table: 2^(43 + i / 32)
__device__ __forceinline__ u64 sm_weight(double t, const double* table, int* k) {
    const double shifted = t + kSmShift, r = t - (shifted - kSmShift);
    const int n = __double2loint(shifted);
    *k = n;
    constexpr double l = 0.021660849392498290;                       // ln 2 / 32
    const double p = fma(fma(fma(fma(fma(l * l * l * l * l / 120.0, r, l * l * l * l / 24.0), r, l * l * l / 6.0), r, l * l / 2.0), r, l), r, 1.0);
    const double power = table[n & 31];
    const double w = fma(p, __hiloint2double(__double2hiint(power) + ((n & ~31) << 15), __double2loint(power)), 4503599627370496.0);
    return (u64)__double_as_longlong(w) & 0xfffffffffffffull;
}

// A cluster of C CTAs per row, each a slice of the vocabulary: kept in shared memory (KEEP), or, where the rows fill the GPU several times, read again from L2 by smaller CTAs of which more are
// resident.  Tokens are counted by bins of logits below the largest, 1 / 32 of a power of two wide; what top_k or top_p cuts off begins in the bin in which
// the counts (sums of weights) reach their target.  Where at most kSmList tokens lie in the bins up to there, one CTA gets them all and puts them in order; otherwise the bin is looked at more closely
// until at most kSmList candidates are left in it, which every CTA gets and looks through.  Weights are whole multiples of 2^-43 of the largest, their sums exact in 64 bits, so that no order of additions
// changes a choice.  Bound by instructions (some 70 a logit and pass, 11 of them of 64 bits) where rows fill the SMs, by phases that wait for one another where they do not: 64 rows of 128256 tokens 58 us,
// 32 flat ones with top_p 43 (three passes with weights or bins behind the first), one of 49152 14.
template <int C, bool KEEP>
__global__ void __launch_bounds__(KEEP ? 512 : 256, KEEP ? 2 : 4) k_sample(const SmArgs a) {
    pdl_enter();
    constexpr uint32_t T_ = KEEP ? 512 : 256, kWarps = T_ / 32, kBinsEach = kSmBins / T_;
    extern __shared__ float4 sm_mem[];
    __shared__ SmShared sh;
    float* const z = reinterpret_cast<float*>(sm_mem);
    const uint32_t r = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const BatchHead head = batch_head(a.table, a.B);
    const int4 w0 = *reinterpret_cast<const int4*>(a.table + ZG_BATCH_ROWS + (size_t)ZG_SAMPLE_WORDS * r);
    const float u = a.table[ZG_BATCH_ROWS + (size_t)ZG_SAMPLE_WORDS * r + 4], T = __int_as_float(w0.x), top_p = __int_as_float(w0.z), min_p = __int_as_float(w0.w);
    const int32_t top_k = w0.y;
    if (r >= head.rows || top_k < 0) return;                         // (the whole cluster)
    const bool ok = T >= 0.0f && T < INFINITY && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    const uint32_t v0 = min(rank * a.slice, a.V), n = min(a.slice, a.V - v0);
    const float* src = a.logits + (size_t)r * a.rs + v0;
    auto four = [&](uint32_t i, bool again) {                        // tokens i .. i + 3 of the slice, i a multiple of 4; what is behind its end counts nothing
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i >= n) return x;
        if (KEEP && again) return *reinterpret_cast<const float4*>(z + i);
        if (a.vec && i + 4 <= n) x = *reinterpret_cast<const float4*>(src + i);
        else { x.x = src[i]; if (i + 1 < n) x.y = src[i + 1]; if (i + 2 < n) x.z = src[i + 2]; if (i + 3 < n) x.w = src[i + 3]; }
        x.x += 0.0f; x.y += 0.0f; x.z += 0.0f; x.w += 0.0f;          // (-0 becomes 0)
        return x;
    };
    // f(four logits, place of the first in the slice, how many of them count) for all tokens of places [from, to), the next ones asked for before.  Work on the four goes side by side where f
    // has no branches between them: an exponential is a dozen operations of 64 bits, each of which waits for the one before it.
    auto fours = [&](uint32_t from, uint32_t to, uint32_t first, uint32_t step, auto&& f) {
        uint32_t i = from + 4 * first;
        float4 x = four(i, true), y = four(i + 4 * step, true);
#pragma unroll 1
        for (; i < to; i += 4 * step) {
            const float4 next = four(i + 8 * step, true);
            const float v[4] = {x.x, x.y, x.z, x.w};
            f(v, i, min(4u, to - i));
            x = y; y = next;
        }
    };
    // f(logit, place) one after the other
    auto each = [&](uint32_t from, uint32_t to, uint32_t first, uint32_t step, auto&& f) {
        fours(from, to, first, step, [&](const float (&v)[4], uint32_t i, uint32_t count) {
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) if (k < count) f(v[k], i + k);
        });
    };
    auto cluster_sync = [&] { if (C > 1) { sm_cluster_arrive(); sm_cluster_wait(); } else __syncthreads(); };
    if (tid < 32) sh.table[tid] = exp2(43.0 + tid / 32.0);
    if (tid == 0) { sh.best = 0; sh.n_all = 0; sh.n_list[0] = sh.n_list[1] = 0; }
    for (uint32_t i = tid; i < kSmBins; i += T_) sh.count[i] = sh.mass_low[i] = sh.mass_high[i] = 0;
    __syncthreads();
    {
        float top = -INFINITY;
        uint32_t where = 0;
        bool nan = false;
#pragma unroll 4
        for (uint32_t i = 4 * tid; i < n; i += 4 * T_) {
            const float4 x = four(i, false);
            if (KEEP) *reinterpret_cast<float4*>(z + i) = x;
            const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) if (i + k < n) { nan = nan || v[k] != v[k]; if (v[k] > top) { top = v[k]; where = i + k; } }
        }
        u64 best = n ? sm_order(top, v0 + where) : 0;                // (a thread's places ascend: its first largest one)
        if (top == -INFINITY) best = 0;
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (__any_sync(0xffffffffu, nan)) best = ~0ull;
        if (lane == 0) atomicMax(&sh.best, best);
    }
    __syncthreads();
    cluster_sync();
    u64 best = 0;
#pragma unroll
    for (uint32_t c = 0; c < C; c++) best = max(best, *sm_peer(&sh.best, c));
    const float M = sm_value((uint32_t)(best >> kSmIndexBits));
    const bool bad = !ok || best == 0 || best == ~0ull;              // (nothing above -inf; something that is no number)
    if (bad || T == 0.0f) {
        if (rank == 0 && tid == 0) {
            a.dst[r] = bad ? -1 : (int32_t)(kSmIndexMask - (uint32_t)(best & kSmIndexMask));
            if (a.probability) a.probability[r] = bad ? kBatchNaN : 1.0f;
        }
        cluster_sync();                                              // no CTA leaves while it is read
        return;
    }
    // Exponents: (x - M) / T, in 32nds of a power of two as one product with x where that loses nothing (near), what is far below the largest as if it were at 45.
    const double inv_t = 1.0 / (double)T, steps = inv_t * kSmSteps, top_steps = -(double)M * steps;
    const bool near = fabs(top_steps) < 65536.0 && T < 1e30f;
    const float lowest = near ? M - 45.0f * T : 0.0f;
    auto exponent = [&](float x) { return x == M ? 0.0 : ((double)x - (double)M) * inv_t; };
    auto in_steps = [&](float x) { return near ? fma((double)fmaxf(x, lowest), steps, top_steps) : fmax(exponent(x) * kSmSteps, -2100.0); };
    auto weight = [&](float x) { int k; return sm_weight(in_steps(x), sh.table, &k); };
    // bins of a 32nd of a power of two below the largest logit (the last one: all below 2^-32 of it), as the weight's rounding has them
    auto bin_of = [&](float x) { return min((uint32_t)-__double2loint(in_steps(x) + kSmShift), kSmBins - 1); };
    // the smallest logit that min_p lets through (compared as exponents: powers of what is just below the largest logit round to 1)
    float least_x = -INFINITY;
    if (min_p > 0.0f) {
        const double least = log((double)min_p);
        uint32_t key = sm_key((float)((double)M + least * (double)T));
        const uint32_t most = (uint32_t)(best >> kSmIndexBits);
        // from there in growing steps to one on the other side, then by halves between them
        auto through = [&](uint32_t k) { return exponent(sm_value(k)) >= least; };
        uint32_t in = most, out = 0x007fffffu;                       // the largest logit is let through, -inf is not
        key = min(max(key, out + 1), most);
        const bool down = through(key);
        (down ? in : out) = key;
        for (uint32_t step = 1; in - out > step; step *= 2) {
            const uint32_t k = down ? in - step : out + step;
            const bool t = through(k);
            (t ? in : out) = k;
            if (t != down) break;
        }
        while (in - out > 1) { const uint32_t k = out + (in - out) / 2; if (through(k)) in = k; else out = k; }
        least_x = sm_value(in);
    }
    auto draw = [&](float x, uint32_t index, u64 all) {
        a.dst[r] = (int32_t)index;
        if (a.probability) a.probability[r] = (float)(exp(exponent(x)) * kSmOne / (double)all);
    };
    const bool by_k = top_k != 0 && (uint32_t)top_k < a.V, by_p = top_p < 1.0f;
    u64 threshold = 0;
    // counts (and sums of weights) of the tokens in [lo, hi] by their bins: of equal width below the largest logit, or of the order's numbers
    auto add_mass = [&](uint32_t b, u64 w) {
        const uint32_t low = (uint32_t)w;
        if (w) {
            const uint32_t old = atomicAdd(&sh.mass_low[b], low), high = (uint32_t)(w >> 32) + (old + low < old);
            if (high) atomicAdd(&sh.mass_high[b], high);
        }
        atomicAdd(&sh.count[b], 1u);
    };
    // sums of groups of 32 bins, the masses' by 16 bits and 32
    auto group_sums = [&](bool masses) {
#pragma unroll
        for (uint32_t g = warp; g < kSmBins / 32; g += kWarps) {
            const uint32_t tokens = __reduce_add_sync(0xffffffffu, sh.count[32 * g + lane]);
            u64 mass = 0;
            if (masses) {
                const uint32_t low = sh.mass_low[32 * g + lane];
                mass = ((u64)__reduce_add_sync(0xffffffffu, sh.mass_high[32 * g + lane]) << 32) + ((u64)__reduce_add_sync(0xffffffffu, low >> 16) << 16) + __reduce_add_sync(0xffffffffu, low & 0xffffu);
            }
            if (lane == 0) { sh.group_count[g] = tokens; sh.group_mass[g] = mass; }
        }
    };
    auto within = [&](float x, u64 lo, u64 hi) { return x >= sm_value(max((uint32_t)(lo >> kSmIndexBits), 0x007fffffu)) && x <= sm_value((uint32_t)(hi >> kSmIndexBits)); };
    auto count_bins = [&](u64 lo, u64 hi, bool linear, uint32_t shift, bool masses) {
        if (masses && lo == 0 && linear)                             // (of all tokens: those with weights go four at a time)
            fours(0, n, tid, T_, [&](const float (&x)[4], uint32_t, uint32_t valid) {
                int k[4];
                u64 w[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) w[e] = sm_weight(in_steps(x[e]), sh.table, &k[e]);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    if (e >= valid) break;
                    add_mass(min((uint32_t)-k[e], kSmBins - 1), w[e]);
                }
            });
        else if (lo == 0 && linear)
            fours(0, n, tid, T_, [&](const float (&x)[4], uint32_t, uint32_t valid) {
                uint32_t b[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) b[e] = bin_of(x[e]);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (e < valid) atomicAdd(&sh.count[b[e]], 1u);
            });
        else
            each(0, n, tid, T_, [&](float x, uint32_t i) {
                if (!within(x, lo, hi)) return;
                const u64 o = sm_order(x, v0 + i);
                if (o < lo || o > hi) return;
                int k = 0;
                const u64 w = masses ? sm_weight(in_steps(x), sh.table, &k) : 0;
                add_mass(linear ? bin_of(x) : (uint32_t)((hi - o) >> shift), w);
            });
        __syncthreads();
        group_sums(masses);
        cluster_sync();
    };
    // Of the bins of N CTAs: the one in which `target` is reached (with `share_of` >= 0: target = share_of of the sum), how many tokens it has, what comes before it and the tokens up to its end.  One
    // warp looks for the group, then in the group (with all bins of eight CTAs read by all threads 4 us instead of 1.5).
    auto find_bin = [&](auto ctas, bool masses, u64 target, double share_of, u64 above) {
        constexpr uint32_t N = decltype(ctas)::value;
        if (warp == 0) {
            auto peer = [&](const auto* p, uint32_t c) { return N == 1 ? p : sm_peer(p, c); };
            uint32_t tokens[2] = {0, 0}, tokens_before = 0;
            u64 mass[2] = {0, 0}, before = above;
            uint32_t at = lane;                                      // group, then bin
#pragma unroll
            for (int level = 0; level < 2; level++) {
                uint32_t t[N], low[N], high[N];
#pragma unroll
                for (uint32_t c = 0; c < N; c++) {
                    t[c] = *(level ? peer(&sh.count[at], c) : peer(&sh.group_count[at], c));
                    if (!masses) low[c] = high[c] = 0;
                    else if (level) { low[c] = *peer(&sh.mass_low[at], c); high[c] = *peer(&sh.mass_high[at], c); }
                    else { const u64 m = *peer(&sh.group_mass[at], c); low[c] = (uint32_t)m; high[c] = (uint32_t)(m >> 32); }
                }
#pragma unroll
                for (uint32_t c = 0; c < N; c++) { tokens[level] += t[c]; mass[level] += masses ? (u64)high[c] << 32 | low[c] : t[c]; }
                uint32_t upto = tokens[level];
                u64 sum = mass[level];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 m = __shfl_up_sync(0xffffffffu, sum, o);
                    const uint32_t q = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) { sum += m; upto += q; }
                }
                if (level == 0 && share_of >= 0.0) target = max((u64)1, (u64)ceil(share_of * (double)__shfl_sync(0xffffffffu, sum, 31)));
                before += sum - mass[level];
                tokens_before += upto - tokens[level];
                const bool here = before < target && before + mass[level] >= target;
                if (level) {
                    if (here) { sh.found_bin = at; sh.found_count = tokens[1]; sh.found_mass = before; sh.found_upto = tokens_before + tokens[1]; sh.found_target = target; }
                } else {
                    const int group = max(__ffs(__ballot_sync(0xffffffffu, here)) - 1, 0);
                    before = __shfl_sync(0xffffffffu, before, group);
                    tokens_before = __shfl_sync(0xffffffffu, tokens_before, group);
                    at = 32 * group + lane;
                }
            }
        }
        __syncthreads();
        return sh.found_target;
    };
    const std::integral_constant<uint32_t, C> cluster;
    if (by_k || by_p) {
        count_bins(0, best, true, 0, !by_k);
        u64 target = find_bin(cluster, !by_k, top_k, by_k ? -1.0 : (double)top_p, 0);
        const uint32_t first_bin = sh.found_bin;
        if (sh.found_upto <= kSmList) {
            // few: they go to the first CTA
            uint32_t* const n_list = &sh.n_list[1];
            fours(0, n, tid, T_, [&](const float (&x)[4], uint32_t i, uint32_t valid) {
                uint32_t b[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) b[e] = bin_of(x[e]);
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (e < valid && b[e] <= first_bin) sh.list[atomicAdd(n_list, 1u)].x = sm_order(x[e], v0 + i + e);
            });
            __syncthreads();
            // one addition to the first CTA's number for a CTA's candidates
            if (tid == 0) {
                uint32_t begin;
                asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(begin) : "r"(sm_at(&sh.n_all, 0)), "r"(*n_list) : "memory");
                sh.n_list[0] = begin;
            }
            __syncthreads();
            for (uint32_t t = tid; t < *n_list; t += T_) {
                const u64 x = sh.list[t].x;
                asm volatile("st.shared::cluster.v2.u64 [%0], {%1, %2};" ::"r"(sm_at(&sh.all_list[sh.n_list[0] + t], 0)), "l"(x), "l"(weight(sm_value((uint32_t)(x >> kSmIndexBits)))) : "memory");
            }
            cluster_sync();                                          // (before that no CTA leaves: its bins are read)
            if (rank != 0) return;
            const uint32_t count = sh.n_all;
            // In falling order of x (the order of the logits; then that of falling numbers, in which indices rise): placed by buckets, which rise as x falls, then ranked in their bucket (64 rows
            // with a thousand candidates: 54 us, each ranked among all of them 129).
            auto sort = [&](auto&& bucket) {
                for (uint32_t i = tid; i < kSmBins; i += T_) sh.count[i] = 0;
                __syncthreads();
                for (uint32_t t = tid; t < count; t += T_) atomicAdd(&sh.count[bucket(sh.all_list[t])], 1u);
                __syncthreads();
                uint32_t begin[kBinsEach], sum = 0;
#pragma unroll
                for (uint32_t k = 0; k < kBinsEach; k++) { begin[k] = sum; sum += sh.count[kBinsEach * tid + k]; }
                uint32_t before = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, before, o); if (lane >= (uint32_t)o) before += t; }
                if (lane == 31) sh.warp_count[warp] = before;
                __syncthreads();
#pragma unroll
                for (uint32_t i = 0; i < kWarps; i++) if (i < warp) before += sh.warp_count[i];
#pragma unroll
                for (uint32_t k = 0; k < kBinsEach; k++) sh.count[kBinsEach * tid + k] = sh.mass_low[kBinsEach * tid + k] = before - sum + begin[k];
                __syncthreads();
                for (uint32_t t = tid; t < count; t += T_) { const ulonglong2 x = sh.all_list[t]; sh.list[atomicAdd(&sh.count[bucket(x)], 1u)] = x; }
                __syncthreads();
                for (uint32_t t = tid; t < count; t += T_) {
                    const ulonglong2 x = sh.list[t];
                    const uint32_t b = bucket(x), first = sh.mass_low[b], end = sh.count[b];
                    uint32_t at = first;
                    for (uint32_t i = first; i < end; i++) at += sh.list[i].x > x.x;
                    sh.all_list[at] = x;
                }
                __syncthreads();
            };
            // sums of y up to each place; the sum of all
            constexpr uint32_t kEach = kSmList / T_;
            u64 upto_[kEach];
            auto scan = [&] {
                u64 sum = 0;
#pragma unroll
                for (uint32_t k = 0; k < kEach; k++) { const uint32_t t = kEach * tid + k; sum += t < count ? sh.all_list[t].y : 0; upto_[k] = sum; }
                u64 before = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, before, o); if (lane >= (uint32_t)o) before += t; }
                __syncthreads();
                if (lane == 31) sh.warp_mass[warp] = before;
                __syncthreads();
                u64 all = 0;
#pragma unroll
                for (uint32_t i = 0; i < kWarps; i++) { if (i < warp) before += sh.warp_mass[i]; all += sh.warp_mass[i]; }
#pragma unroll
                for (uint32_t k = 0; k < kEach; k++) upto_[k] += before - sum;
                return all;
            };
            sort([&](const ulonglong2& x) { return bin_of(sm_value((uint32_t)(x.x >> kSmIndexBits))); });
            if (by_k) {
                for (uint32_t t = top_k + tid; t < count; t += T_) sh.all_list[t].y = 0;
                __syncthreads();
            }
            if (by_p) {
                const u64 sum = scan();
                if (by_k) target = max((u64)1, (u64)ceil((double)top_p * (double)sum));
#pragma unroll
                for (uint32_t k = 0; k < kEach; k++) { const uint32_t t = kEach * tid + k; if (t < count && upto_[k] - sh.all_list[t].y >= target) sh.all_list[t].y = 0; }
                __syncthreads();
            }
            // in order of their indices
            for (uint32_t t = tid; t < count; t += T_) {
                const ulonglong2 x = sh.all_list[t];
                const float v = sm_value((uint32_t)(x.x >> kSmIndexBits));
                const bool on = x.y && v >= least_x;
                sh.all_list[t] = make_ulonglong2((x.x & kSmIndexMask) << 32 | __float_as_uint(v), on ? x.y : 0);
            }
            const uint32_t width = (a.V + kSmBins - 1) / kSmBins;
            sort([&](const ulonglong2& x) { return (kSmIndexMask - (uint32_t)(x.x >> 32)) / width; });
            const u64 all = scan();
            const double drawn = (double)u * (double)all;
#pragma unroll
            for (uint32_t k = 0; k < kEach; k++) {
                const uint32_t t = kEach * tid + k;
                if (t >= count) break;
                const ulonglong2 x = sh.all_list[t];
                if (x.y && !((double)(upto_[k] - x.y) > drawn) && (double)upto_[k] > drawn) draw(__uint_as_float((uint32_t)x.x), kSmIndexMask - (uint32_t)(x.x >> 32), all);
            }
            return;
        }
        for (int by_mass = by_k ? 0 : 1; by_mass <= (by_p ? 1 : 0); by_mass++) {
            u64 lo = threshold, hi = best, above = 0;
            uint32_t shift = 0;
            bool linear = true, counted = by_mass == !by_k;          // (the bins above are this one's first)
            for (;;) {
                if (!counted) {
                    __syncthreads();
                    for (uint32_t i = tid; i < kSmBins; i += T_) sh.count[i] = sh.mass_low[i] = sh.mass_high[i] = 0;
                    __syncthreads();
                    count_bins(lo, hi, linear, shift, by_mass);
                    target = find_bin(cluster, by_mass, by_mass ? target : (u64)top_k, by_mass && linear ? (double)top_p : -1.0, above);
                }
                counted = false;
                const uint32_t bin = sh.found_bin, count = sh.found_count;
                above = sh.found_mass;
                if (count > kSmList) {
                    // where the bin lies in the order, and bins of that
                    if (linear) {
                        auto bound = [&](bool upper) {               // largest key whose bin is >= bin (upper), or smallest one whose bin is <= bin
                            uint32_t l = 0x007fffffu, h = (uint32_t)(best >> kSmIndexBits);      // keys from -inf to the largest logit's
                            while (l < h) {
                                const uint32_t m = l + (h - l + (upper ? 1 : 0)) / 2, b = bin_of(sm_value(m));
                                if (upper) { if (b >= bin) l = m; else h = m - 1; }
                                else { if (b <= bin) h = m; else l = m + 1; }
                            }
                            return l;
                        };
                        hi = min(hi, ((u64)bound(true) << kSmIndexBits) | kSmIndexMask);
                        lo = max(lo, (u64)bound(false) << kSmIndexBits);
                        linear = false;
                    } else {
                        hi -= (u64)bin << shift;
                        lo = max(lo, hi >= (1ull << shift) - 1 ? hi - ((1ull << shift) - 1) : 0);
                    }
                    shift = 0;
                    while ((hi - lo) >> shift >= kSmBins) shift++;
                    cluster_sync();                                  // (peers have read the bins)
                    continue;
                }
                uint32_t* const n_list = &sh.n_list[1];
                if (tid == 0) *n_list = 0;
                __syncthreads();
                fours(0, n, tid, T_, [&](const float (&x)[4], uint32_t i, uint32_t valid) {
                    uint32_t in = 0;
                    if (linear) {
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) in |= (bin_of(x[e]) == bin) << e;
                    } else {
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) in |= within(x[e], lo, hi) << e;
                    }
                    if (!in) return;
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) {
                        if (e >= valid || !(in >> e & 1)) continue;
                        const u64 o = sm_order(x[e], v0 + i + e);
                        if (o >= lo && o <= hi && (linear || (uint32_t)((hi - o) >> shift) == bin)) sh.list[atomicAdd(n_list, 1u)].x = o;
                    }
                });
                __syncthreads();
                for (uint32_t t = tid; t < *n_list; t += T_) sh.list[t].y = by_mass ? weight(sm_value((uint32_t)(sh.list[t].x >> kSmIndexBits))) : 1;      // (side by side: few lanes of a warp find one)
                __syncthreads();
                cluster_sync();                                      // (and peers have read the bins)
                uint32_t ends[C];
#pragma unroll
                for (uint32_t c = 0; c < C; c++) ends[c] = *sm_peer(n_list, c);
#pragma unroll
                for (uint32_t c = 1; c < C; c++) ends[c] += ends[c - 1];
                // Every CTA gets them all, and looks for the one in which the target is reached by bins of their own range, then among the few of one bin.
                uint32_t top = 0, least = 0xffffffffu;
                if (tid == 0) { sh.n_picked = 0; sh.span[0] = 0; sh.span[1] = 0xffffffffu; }
                for (uint32_t i = tid; i < kSmBins; i += T_) sh.count[i] = sh.mass_low[i] = sh.mass_high[i] = 0;
                for (uint32_t t = tid; t < count; t += T_) {
                    uint32_t c = 0, begin = 0;
#pragma unroll
                    for (uint32_t k = 0; k + 1 < C; k++) if (t >= ends[k]) { c = k + 1; begin = ends[k]; }
                    const ulonglong2 x = *sm_peer(&sh.list[t - begin], c);
                    sh.all_list[t] = x;
                    top = max(top, (uint32_t)(x.x >> kSmIndexBits)); least = min(least, (uint32_t)(x.x >> kSmIndexBits));
                }
                __syncthreads();
                top = __reduce_max_sync(0xffffffffu, top); least = __reduce_min_sync(0xffffffffu, least);
                if (lane == 0) { atomicMax(&sh.span[0], top); atomicMin(&sh.span[1], least); }
                __syncthreads();
                const u64 last = (u64)sh.span[0] << kSmIndexBits | kSmIndexMask, first = (u64)sh.span[1] << kSmIndexBits;
                uint32_t apart = 0;
                while ((last - first) >> apart >= kSmBins) apart++;
                for (uint32_t t = tid; t < count; t += T_) { const ulonglong2 x = sh.all_list[t]; add_mass((uint32_t)((last - x.x) >> apart), x.y); }
                __syncthreads();
                group_sums(true);
                __syncthreads();
                find_bin(std::integral_constant<uint32_t, 1>(), true, target, -1.0, above);
                const uint32_t inner = sh.found_bin;
                const u64 ahead_of = sh.found_mass;
                for (uint32_t t = tid; t < count; t += T_) if ((uint32_t)((last - sh.all_list[t].x) >> apart) == inner) sh.count[atomicAdd(&sh.n_picked, 1u)] = t;
                __syncthreads();
                for (uint32_t t = warp; t < sh.n_picked; t += kWarps) {
                    const ulonglong2 me = sh.all_list[sh.count[t]];
                    u64 ahead = 0;
                    for (uint32_t i = lane; i < sh.n_picked; i += 32) { const ulonglong2 x = sh.all_list[sh.count[i]]; if (x.x > me.x) ahead += x.y; }
                    ahead = ahead_of + warp_sum64(ahead);
                    if (ahead < target && ahead + me.y >= target && lane == 0) sh.threshold = me.x;
                }
                __syncthreads();
                threshold = sh.threshold;
                break;
            }
        }
    }
    // the draw: sums of what stays by warps' parts, then the part in which u of all is passed
    const uint32_t part = ((n + kWarps - 1) / kWarps + 127) / 128 * 128, from = min(warp * part, n), to = min(from + part, n);
    const float cut = threshold ? sm_value((uint32_t)(threshold >> kSmIndexBits)) : -INFINITY, last = fmaxf(cut, least_x);      // what stays: larger logits, and this one up to an index
    const uint32_t last_index = threshold && cut >= least_x ? kSmIndexMask - (uint32_t)(threshold & kSmIndexMask) : 0xffffffffu;
    auto stays = [&](const float (&x)[4], uint32_t i, uint32_t valid, u64 (&w)[4]) {
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) w[e] = weight(x[e]);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) if (!(e < valid && (x[e] > last || (x[e] == last && v0 + i + e <= last_index)))) w[e] = 0;
    };
    u64 sum = 0;
    fours(from, to, lane, 32, [&](const float (&x)[4], uint32_t i, uint32_t valid) {
        u64 w[4];
        stays(x, i, valid, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
    });
    sum = warp_sum64(sum);
    __syncthreads();
    if (lane == 0) sh.warp_mass[warp] = sum;
    __syncthreads();
    if (tid == 0) { u64 t = 0; for (uint32_t i = 0; i < kWarps; i++) t += sh.warp_mass[i]; sh.total = t; }
    __syncthreads();
    cluster_sync();
    u64 all = 0, base = 0;
#pragma unroll
    for (uint32_t c = 0; c < C; c++) { const u64 t = *sm_peer(&sh.total, c); all += t; if (c < rank) base += t; }
    const double drawn = (double)u * (double)all;
    for (uint32_t i = 0; i < warp; i++) base += sh.warp_mass[i];
    if (!((double)base > drawn) && (double)(base + sum) > drawn) {
        for (uint32_t i = from; i < to; i += 128) {                  // a lane's four neighbours at a time
            const uint32_t place = i + 4 * lane;
            const float4 y = four(place, true);
            const float x[4] = {y.x, y.y, y.z, y.w};
            u64 w[4];
            stays(x, place, place < to ? to - place : 0, w);
            const u64 mine = (w[0] + w[1]) + (w[2] + w[3]);
            u64 upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= (uint32_t)o) upto += t; }
            const uint32_t passed = __ballot_sync(0xffffffffu, (double)(base + upto) > drawn);
            if (passed) {
                if ((int)lane == __ffs(passed) - 1) {
                    u64 at = base + upto - mine;
                    bool found = false;
#pragma unroll
                    for (uint32_t q = 0; q < 4; q++) {
                        at += w[q];
                        if (!found && (double)at > drawn) { found = true; draw(x[q], v0 + i + 4 * lane + q, all); }
                    }
                }
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    cluster_sync();                                                  // no CTA leaves while its sums are read
}

template <int C, bool KEEP>
bool sm_launch(const SmArgs& a, cudaStream_t st) {
    if (KEEP && !zg_smem_limit<k_sample<C, KEEP>>(sizeof(float) * kSmSlice)) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C, a.B); cfg.blockDim = dim3(KEEP ? 512 : 256); cfg.dynamicSmemBytes = KEEP ? sizeof(float) * a.slice : 0; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_zg_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_sample<C, KEEP>, a);
    return true;
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
    a.vec = a.rs % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
    // CTAs of a row: eight, fewer where a slice would be small (one row of 4096 tokens, us, by 1 / 8 CTAs: 10.3 / 12.3), or where the rows fill the SMs, two CTAs each, without, and their slices
    // leave room for two (256 rows of 32000 tokens by 2 / 4 / 8 CTAs: 51.5 / 61.4 / 86.1; 64 rows: 30.8 / 24.6 / 30.8; 64 rows of 65536: 47.1 / 34.9 / 39.5).
    const uint32_t sms = zg_sm_count();
    auto slice = [&](uint32_t C) { return ((a.V + C - 1) / C + 3) / 4 * 4; };
    uint32_t C = kSmCluster;
    while (C > 1 && (slice(C) <= 2048 || ((uint64_t)a.B * C > 2 * sms && slice(C / 2) <= kSmHalf))) C /= 2;
    a.slice = slice(C);
    // Slices are kept up to three waves of CTAs (128256 tokens, us, kept / read again: 1 row 18.5 / 28.7, 32 rows 43.7 / 75.8, 64 58.8 / 79.9, 96 76.5 / 92.3, 128 95.8 / 99.5,
    // 192 149 / 145, 512 364 / 340; 200000 tokens: 32 rows 63.5 / 77.8, 64 104 / 98).
    const bool keep = C < kSmCluster || (uint64_t)a.B * C <= 3 * sms * (a.slice <= kSmHalf ? 2 : 1);
    if (!(C == 1 ? sm_launch<1, true>(a, st) : C == 2 ? sm_launch<2, true>(a, st) : C == 4 ? sm_launch<4, true>(a, st) : keep ? sm_launch<kSmCluster, true>(a, st) : sm_launch<kSmCluster, false>(a, st))) return false;
    ZG_SEQ_CHECK();
    return true;
}
