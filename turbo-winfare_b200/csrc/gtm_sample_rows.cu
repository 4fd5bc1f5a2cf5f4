// Sampling a batch's rows (gtm_sample_rows, include/gtmoe_sampling.h).
//
// One cluster of CTAs per row: each keeps its share of the row's logits in shared memory (larger
// vocabularies are read from L2 again), so HBM is read once and every later pass runs on chip, with no
// workspace and one launch.
//   1 the largest logit, and its lowest id;
//   2 the cuts. Ranked by logit, every cut keeps a run from the top, so the kept set is the ids whose
//     key (logit, then lower id) is at least a border's. Ids are counted per level of max - logit,
//     1/64 wide; a level's weights agree within 1.6%, so the counts alone bracket the nucleus' border
//     to a few levels. One pass then sums the exact weights (all, above the bracket, per level in
//     it), and the ids of the level that holds the border are gathered and ranked. More ids than the
//     gather holds (equal or nearly equal logits) are narrowed by the logit's ordered bits instead;
//   3 the draw: sums of the kept weights per warp's run of ids, CTA and cluster, then one warp finds
//     the id in the run that the target falls in.
// Weights exp(l - max) are formed in 64 bits, rounded to multiples of 2^-(62 - bits of the vocabulary)
// and summed as 64-bit integers: the sums cannot overflow, do not depend on their order (so the token
// is reproducible, atomics and all) and are within 2^-44 of the weights' at a vocabulary of 2^18. The
// 64-bit weights bound a large batch: ~11 double-precision operations each, on units that do 64 a cycle.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>

#include "gtm_internal.h"
#include "gtmoe_sampling.h"

namespace cg = cooperative_groups;

namespace gtm {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kLevels = 2048;
constexpr int kGather = 1024;          // ids of the border's level that are ranked at once
constexpr uint32_t kSmemIds = 40960;   // ids of a share that stay in shared memory
constexpr uint64_t kMantissa = (1ull << 52) - 1;

struct Rows {
    GtmSamplingRow v[GTM_SAMPLE_MAX_ROWS];
};

struct SampleArgs {
    const float* logits;
    uint64_t row_stride;
    const double* uniform;
    uint32_t *token, *kept;
    float* logprob;
    uint32_t vocab, slice;   // ids per CTA, a multiple of 1024
    int shift;               // weights are multiples of 2^-shift
    bool vec, resident;      // 16-byte loads; the share stays in shared memory
};

__device__ __forceinline__ float as_logit(float x) { return x != x ? -INFINITY : (x == 0.0f ? 0.0f : x); }
// Larger logit, larger bits.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t id) {
    return (static_cast<unsigned long long>(ordered(x)) << 32) | static_cast<uint32_t>(~id);
}

struct Shared {
    double power[256];                  // 2^(j / 256)
    unsigned long long mass[kLevels];   // also the gathered keys
    uint32_t count[kLevels];
    unsigned long long warp_mass[kWarps], warp_mass2[kWarps];
    double warp_lo[kWarps], warp_hi[kWarps];
    uint32_t warp_count[kWarps];
    unsigned long long cta_key, cta_mass, cta_mass2, draw_mass, border_key;   // each read by the peers: none is reused
    uint32_t tie_count, draw_count, gathered;
    uint32_t first, last, by_count;     // the bracket's levels; the level that holds the top_k-th id
    uint32_t pick;                      // the level that holds the border
    unsigned long long pick_mass;       // mass and count of the levels above it
    uint32_t pick_count;
};

// exp(d * ln 2 / rate') as a multiple of 2^-shift, rate = 256 log2(e) / temperature: 2^(y / 256) with y =
// k + r, |r| <= 1/2, from a table of 2^(j / 256) and the exponential series to the fourth power of
// r ln 2 / 256 (the next term is below 2^-54).
__device__ __forceinline__ unsigned long long fixed_exp(const double* power, double d, double rate, int shift) {
    constexpr double kLn = 0.69314718055994530942 / 256.0;
    const double y = d * rate;
    if (!(y > -16000.0)) return 0;   // below 2^-62
    const double t = y + 6755399441055744.0;   // 1.5 * 2^52: the nearest integer in the low word
    const int k = __double2loint(t);
    const double r = y - (t - 6755399441055744.0);
    double p = fma(r, kLn * kLn * kLn * kLn / 24.0, kLn * kLn * kLn / 6.0);
    p = fma(p, r, kLn * kLn / 2.0);
    p = fma(p, r, kLn);
    p = fma(p, r, 1.0);
    const unsigned long long m = (static_cast<unsigned long long>(__double_as_longlong(p * power[k & 255])) & kMantissa) | (1ull << 52);
    // p * power is within [1, 2) except for a rounding to just below 1 or to 2, where the exponent moves by one
    const int e = static_cast<int>(static_cast<unsigned>(__double2hiint(p * power[k & 255])) >> 20) - 1023;
    const int s = 52 - shift - (k >> 8) - e;
    if (s > 60) return 0;
    return s > 0 ? (m + (1ull << (s - 1))) >> s : m << -s;
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <int CL>
__global__ void __launch_bounds__(kThreads, 1) smp_rows(const __grid_constant__ SampleArgs a, const __grid_constant__ Rows rows) {
    extern __shared__ __align__(16) float slice_s[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), row = blockIdx.x / CL;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const GtmSamplingRow rule = rows.v[row];
    const float* src = a.logits + row * a.row_stride;
    const uint32_t base = min(a.vocab, rank * a.slice), n = min(a.slice, a.vocab - base), n4 = (n + 3) & ~3u;
    // four logits from a multiple of 4 on; -infinity past the share
    auto four = [&](uint32_t i) -> float4 {
        if (a.resident) return *reinterpret_cast<const float4*>(slice_s + i);
        float4 x;
        x.x = as_logit(__ldg(src + base + i));
        x.y = i + 1 < n ? as_logit(__ldg(src + base + i + 1)) : -INFINITY;
        x.z = i + 2 < n ? as_logit(__ldg(src + base + i + 2)) : -INFINITY;
        x.w = i + 3 < n ? as_logit(__ldg(src + base + i + 3)) : -INFINITY;
        return x;
    };
    auto logit = [&](uint32_t i) { return a.resident ? slice_s[i] : as_logit(__ldg(src + base + i)); };

    // ---- 1: the largest logit and its lowest id
    unsigned long long best = 0;
    auto look = [&](uint32_t i, float x) {
        x = i < n ? as_logit(x) : -INFINITY;
        const unsigned long long key = i < n ? key_of(x, base + i) : 0;
        best = key > best ? key : best;
        return x;
    };
    if (a.resident && a.vec) {
        constexpr int U = 4;   // loads in flight per thread
        for (uint32_t i0 = tid * 4; i0 < n4; i0 += kThreads * 4 * U) {
            float4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = i0 + u * kThreads * 4;
                if (i + 3 < n) {
                    x[u] = __ldg(reinterpret_cast<const float4*>(src + base + i));
                } else if (i < n) {
                    x[u].x = __ldg(src + base + i);
                    x[u].y = i + 1 < n ? __ldg(src + base + i + 1) : 0.0f;
                    x[u].z = i + 2 < n ? __ldg(src + base + i + 2) : 0.0f;
                    x[u].w = 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = i0 + u * kThreads * 4;
                if (i < n) *reinterpret_cast<float4*>(slice_s + i) = make_float4(look(i, x[u].x), look(i + 1, x[u].y), look(i + 2, x[u].z), look(i + 3, x[u].w));
            }
        }
    } else {
        for (uint32_t i = tid; i < n4; i += kThreads) {
            const float x = look(i, i < n ? __ldg(src + base + i) : 0.0f);
            if (a.resident) slice_s[i] = x;
        }
    }
    if (tid < 256) sh.power[tid] = exp2(tid * (1.0 / 256.0));
    for (int i = tid; i < kLevels; i += kThreads) sh.count[i] = 0;
    if (tid == 0) sh.first = kLevels, sh.last = kLevels, sh.by_count = kLevels, sh.gathered = 0, sh.pick = kLevels;
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (lane == 0) sh.warp_mass[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = sh.warp_mass[lane];
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) sh.cta_key = best;
    }
    cluster.sync();
    best = 0;
#pragma unroll
    for (int r = 0; r < CL; ++r) {
        const unsigned long long other = *cluster.map_shared_rank(&sh.cta_key, r);
        best = other > best ? other : best;
    }
    const float top = from_ordered(static_cast<uint32_t>(best >> 32));
    const uint32_t top_id = ~static_cast<uint32_t>(best);
    if (isinf(top)) {   // the same for every CTA of the cluster
        if (rank == 0 && tid == 0) {
            a.token[row] = 0xFFFFFFFFu;
            if (a.kept) a.kept[row] = 0;
            if (a.logprob) a.logprob[row] = __int_as_float(0x7FC00000);
        }
        cluster.sync();   // no CTA leaves while another may read its shared memory
        return;
    }
    constexpr double kRate = 256.0 * 1.4426950408889634074;
    const double top_d = top;
    auto weight = [&](float x) { return fixed_exp(sh.power, static_cast<double>(x) - top_d, kRate, a.shift); };
    auto level = [&](float x) { return static_cast<uint32_t>(fminf((top - x) * 64.0f, kLevels - 1.0f)); };
    const bool greedy = !(rule.temperature > 0.0f);
    const bool cut_p = !greedy && rule.top_p < 1.0f, cut_k = !greedy && rule.top_k > 0 && static_cast<uint32_t>(rule.top_k) < a.vocab;
    // ids with p below min_p of the largest are out of the draw
    const double floor_d = !greedy && rule.min_p > 0.0f ? log(static_cast<double>(rule.min_p)) : -INFINITY;

    // ---- 2a: counts per level, and the bracket
    uint32_t first = kLevels, last = kLevels;
    constexpr int kPart = kLevels / CL;   // levels that a CTA sums over the cluster
    if (cut_p || cut_k) {
        for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
            const float4 x = four(i);
            if (x.x > -INFINITY) atomicAdd(&sh.count[level(x.x)], 1u);
            if (x.y > -INFINITY) atomicAdd(&sh.count[level(x.y)], 1u);
            if (x.z > -INFINITY) atomicAdd(&sh.count[level(x.z)], 1u);
            if (x.w > -INFINITY) atomicAdd(&sh.count[level(x.w)], 1u);
        }
        cluster.sync();
        uint32_t c = 0;
        const int mine = rank * kPart + tid;
        if (tid < kPart)
            for (int r = 0; r < CL; ++r) c += *cluster.map_shared_rank(&sh.count[mine], r);
        cluster.sync();
        if (tid < kPart)
            for (int r = 0; r < CL; ++r) *cluster.map_shared_rank(&sh.count[mine], r) = c;
        cluster.sync();
        // two levels per thread: counts and bounds of the mass down to and including each
        static_assert(kLevels == 2 * kThreads, "");
        const uint32_t c0 = sh.count[2 * tid], c1 = sh.count[2 * tid + 1];
        // a level's edges are off by the rounding of (max - l) * 64 and by the weights' own: 2^-12 covers both
        const double q0 = exp(-(2 * tid) / 64.0) * (1 + 0x1p-12), q1 = exp(-(2 * tid + 1) / 64.0), q2 = exp(-(2 * tid + 2) / 64.0) * (1 - 0x1p-12);
        double lo0 = c0 * q1 * (1 - 0x1p-12), hi0 = c0 * q0, lo1 = tid == kThreads - 1 ? 0.0 : c1 * q2, hi1 = c1 * q1 * (1 + 0x1p-12);
        uint32_t pc = c0 + c1;
        double pl = lo0 + lo1, ph = hi0 + hi1;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
            const double ul = __shfl_up_sync(0xffffffffu, pl, o), uh = __shfl_up_sync(0xffffffffu, ph, o);
            if (lane >= o) pc += uc, pl += ul, ph += uh;
        }
        if (lane == 31) sh.warp_count[warp] = pc, sh.warp_lo[warp] = pl, sh.warp_hi[warp] = ph;
        __syncthreads();
        uint32_t bc = 0;
        double bl = 0.0, bh = 0.0, all_lo = 0.0, all_hi = 0.0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) bc += sh.warp_count[w], bl += sh.warp_lo[w], bh += sh.warp_hi[w];
            all_lo += sh.warp_lo[w], all_hi += sh.warp_hi[w];
        }
        const double p = rule.top_p;
        const uint32_t cum1 = bc + pc, cum0 = cum1 - c1;
        const double l1 = bl + pl, l0 = l1 - lo1, h1 = bh + ph, h0 = h1 - hi1;
        if (cut_p) {   // sums of doubles are off by far less than 2^-20
            const double low = p * all_lo * (1 - 0x1p-20), high = p * all_hi * (1 + 0x1p-20);
            if (c0 && h0 >= low) atomicMin(&sh.first, 2 * tid);
            if (c1 && h1 >= low) atomicMin(&sh.first, 2 * tid + 1);
            if (c0 && l0 >= high) atomicMin(&sh.last, 2 * tid);
            if (c1 && l1 >= high) atomicMin(&sh.last, 2 * tid + 1);
        }
        if (cut_k) {
            if (c0 && cum0 >= static_cast<uint32_t>(rule.top_k)) atomicMin(&sh.by_count, 2 * tid);
            if (c1 && cum1 >= static_cast<uint32_t>(rule.top_k)) atomicMin(&sh.by_count, 2 * tid + 1);
        }
        __syncthreads();
        first = cut_p ? min(sh.first, sh.by_count) : sh.by_count;
        last = cut_p ? min(min(sh.last, sh.by_count), kLevels - 1u) : sh.by_count;
        // counts of the levels above the bracket
        if (2 * tid == first) sh.pick_count = cum0 - c0;
        if (2 * tid + 1 == first) sh.pick_count = cum1 - c1;
        for (int i = tid; i < kLevels; i += kThreads) sh.mass[i] = 0;
        __syncthreads();
    }
    const bool bracket = first < kLevels;   // else every id is kept

    // ---- 2b: exact sums: the whole distribution, the levels above the bracket, each level in it
    unsigned long long whole = 0, above_mass = 0;
    {
        unsigned long long sum = 0, up = 0;
        for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
            const float4 x4 = four(i);
            const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned long long w = x[j] > -INFINITY ? weight(x[j]) : 0ull;
                sum += w;
                if (cut_p && w) {
                    const uint32_t lev = level(x[j]);
                    if (lev < first)
                        up += w;
                    else if (lev <= last)
                        atomicAdd(&sh.mass[lev - first], w);
                }
            }
        }
        sum = warp_sum(sum), up = warp_sum(up);
        if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_mass2[warp] = up;
        __syncthreads();
        if (warp == 0) {
            sum = warp_sum(sh.warp_mass[lane]), up = warp_sum(sh.warp_mass2[lane]);
            if (lane == 0) sh.cta_mass = sum, sh.cta_mass2 = up;
        }
        cluster.sync();
        for (int r = 0; r < CL; ++r) {
            whole += *cluster.map_shared_rank(&sh.cta_mass, r);
            above_mass += *cluster.map_shared_rank(&sh.cta_mass2, r);
        }
    }
    uint32_t above = 0, border_level = kLevels, ties = 0xFFFFFFFFu;
    unsigned long long need = 0, border = 0;   // ids with a key below `border` are out
    bool tied = false;                         // and of those with the border's logit only the first `ties` stay
    if (bracket) {
        need = cut_p ? static_cast<unsigned long long>(ceil(static_cast<double>(rule.top_p) * static_cast<double>(whole))) : ~0ull;
        above = sh.pick_count;
        if (warp == 0) {   // walk the bracket's levels, 32 at a time; masses of the whole cluster
            unsigned long long run = above_mass;
            uint32_t run_c = above;
            for (uint32_t i = first; i <= last; i += 32) {
                const uint32_t lev = i + lane;
                unsigned long long own = 0;
                if (cut_p && lev <= last)
                    for (int r = 0; r < CL; ++r) own += *cluster.map_shared_rank(&sh.mass[lev - first], r);
                uint32_t own_c = lev <= last ? sh.count[lev] : 0, pc = own_c;
                unsigned long long pm = own;
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long um = __shfl_up_sync(0xffffffffu, pm, o);
                    const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
                    if (lane >= o) pm += um, pc += uc;
                }
                const bool here = lev <= last && ((cut_p && run + pm >= need) || (cut_k && run_c + pc >= static_cast<uint32_t>(rule.top_k)));
                const uint32_t vote = __ballot_sync(0xffffffffu, here);
                if (vote) {
                    if (lane == __ffs(vote) - 1) sh.pick = lev, sh.pick_mass = run + pm - own, sh.pick_count = run_c + pc - own_c;
                    break;
                }
                run += __shfl_sync(0xffffffffu, pm, 31);
                run_c += __shfl_sync(0xffffffffu, pc, 31);
            }
        }
        cluster.sync();   // also: no peer reads this CTA's masses any more
        border_level = sh.pick;
        above = sh.pick_count, above_mass = sh.pick_mass;
    }
    if (border_level < kLevels) {
        // ---- 2c: the border within its level
        const uint32_t members = sh.count[border_level];
        if (members <= kGather) {
            unsigned long long* list = cluster.map_shared_rank(sh.mass, 0);
            uint32_t* next = cluster.map_shared_rank(&sh.gathered, 0);
            for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
                const float4 x4 = four(i);
                const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (x[j] > -INFINITY && level(x[j]) == border_level) list[atomicAdd(next, 1u)] = key_of(x[j], base + i + j);
            }
            cluster.sync();
            if (rank == 0) {   // each member's rank and the mass above it; the border is the first that reaches a cut
                if (tid == 0) sh.border_key = 0;
                unsigned long long* weights = sh.mass + kGather;
                const unsigned long long key = tid < members ? sh.mass[tid] : 0;
                if (tid < members) weights[tid] = weight(from_ordered(static_cast<uint32_t>(key >> 32)));
                __syncthreads();
                if (tid < members) {
                    unsigned long long m = above_mass + weights[tid];
                    uint32_t c = above + 1;
                    for (uint32_t j = 0; j < members; ++j)
                        if (sh.mass[j] > key) m += weights[j], ++c;
                    if ((cut_p && m >= need) || (cut_k && c >= static_cast<uint32_t>(rule.top_k))) atomicMax(&sh.border_key, key);
                }
                __syncthreads();
            }
            cluster.sync();
            border = *cluster.map_shared_rank(&sh.border_key, 0);
        } else {
            uint32_t lo = 0, bits = 32;   // the border's logit has these high bits
            for (int pass = 0; pass < 3; ++pass) {
                for (int i = tid; i < kLevels; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
                __syncthreads();
                const uint32_t take = pass == 2 ? 10 : 11;
                for (uint32_t i = tid; i < n; i += kThreads) {
                    const float x = logit(i);
                    if (!(x > -INFINITY) || level(x) != border_level || (pass > 0 && (ordered(x) >> bits) != lo)) continue;
                    const uint32_t at = kLevels - 1 - ((ordered(x) >> (bits - take)) & ((1u << take) - 1));   // larger logits first
                    if (cut_p) {
                        const unsigned long long w = weight(x);
                        if (w) atomicAdd(&sh.mass[at], w);
                    }
                    atomicAdd(&sh.count[at], 1u);
                }
                cluster.sync();
                unsigned long long m = 0;
                uint32_t c = 0;
                const int mine = rank * kPart + tid;
                if (tid < kPart)
                    for (int r = 0; r < CL; ++r) {
                        m += *cluster.map_shared_rank(&sh.mass[mine], r);
                        c += *cluster.map_shared_rank(&sh.count[mine], r);
                    }
                cluster.sync();
                if (tid < kPart)
                    for (int r = 0; r < CL; ++r) {
                        *cluster.map_shared_rank(&sh.mass[mine], r) = m;
                        *cluster.map_shared_rank(&sh.count[mine], r) = c;
                    }
                cluster.sync();
                if (warp == 0) {
                    unsigned long long run = above_mass;
                    uint32_t run_c = above;
                    for (int i = 0; i < kLevels; i += 32) {
                        const unsigned long long own = sh.mass[i + lane];
                        const uint32_t own_c = sh.count[i + lane];
                        unsigned long long pm = own;
                        uint32_t pc = own_c;
                        for (int o = 1; o < 32; o <<= 1) {
                            const unsigned long long um = __shfl_up_sync(0xffffffffu, pm, o);
                            const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
                            if (lane >= o) pm += um, pc += uc;
                        }
                        const bool here = (cut_p && run + pm >= need) || (cut_k && run_c + pc >= static_cast<uint32_t>(rule.top_k));
                        const uint32_t vote = __ballot_sync(0xffffffffu, here);
                        if (vote) {
                            if (lane == __ffs(vote) - 1) sh.pick = i + lane, sh.pick_mass = run + pm - own, sh.pick_count = run_c + pc - own_c;
                            break;
                        }
                        run += __shfl_sync(0xffffffffu, pm, 31);
                        run_c += __shfl_sync(0xffffffffu, pc, 31);
                    }
                }
                __syncthreads();
                above = sh.pick_count, above_mass = sh.pick_mass;
                lo = (lo << take) | (kLevels - 1 - sh.pick);
                bits -= take;
                if (pass == 2) {
                    const unsigned long long w = weight(from_ordered(lo));
                    ties = sh.count[sh.pick];
                    if (cut_k) ties = min(ties, static_cast<uint32_t>(rule.top_k) - above);
                    if (cut_p && w) {
                        const unsigned long long t = (need - above_mass + w - 1) / w;
                        ties = t < ties ? static_cast<uint32_t>(t) : ties;
                    }
                    border = static_cast<unsigned long long>(lo) << 32;
                    tied = true;
                }
                __syncthreads();
            }
        }
    }

    // ---- 3: the draw
    if (!greedy) {
        const double rate = kRate / static_cast<double>(rule.temperature);
        const uint32_t edge = static_cast<uint32_t>(border >> 32);
        const uint32_t run = a.slice / kWarps;   // a warp's run of ids, a multiple of 32
        const uint32_t r0 = min(n, warp * run), r1 = min(n, r0 + run);
        uint32_t ties_before = 0;   // ids at the border's logit before this CTA's warp
        if (tied) {
            uint32_t c = 0;
            for (uint32_t i = r0 + lane; i < r1; i += 32) c += ordered(logit(i)) == edge;
            for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (lane == 0) sh.warp_count[warp] = c;
            __syncthreads();
            if (tid == 0) {
                uint32_t s = 0;
                for (int w = 0; w < kWarps; ++w) s += sh.warp_count[w];
                sh.tie_count = s;
            }
            cluster.sync();
            for (uint32_t r = 0; r < rank; ++r) ties_before += *cluster.map_shared_rank(&sh.tie_count, r);
            for (int w = 0; w < warp; ++w) ties_before += sh.warp_count[w];
            cluster.sync();
        }
        auto in_cuts = [&](float x, uint32_t i) {
            return x > -INFINITY && key_of(x, base + i) >= border && static_cast<double>(x) - top_d >= floor_d;
        };
        auto mass = [&](float x) { return fixed_exp(sh.power, static_cast<double>(x) - top_d, rate, a.shift); };
        // lane's id of the 32 from i0 on: whether it is kept; `seen` counts the ties so far (the whole warp calls it)
        auto keep_tied = [&](uint32_t i0, uint32_t& seen) {
            const uint32_t i = i0 + lane;
            const float x = i < r1 ? logit(i) : -INFINITY;
            const bool at = ordered(x) == edge;
            const uint32_t vote = __ballot_sync(0xffffffffu, at);
            const bool keep = in_cuts(x, i) && (!at || seen + __popc(vote & ((1u << lane) - 1)) < ties);
            seen += __popc(vote);
            return keep;
        };
        unsigned long long sum = 0;
        uint32_t count = 0, seen = ties_before;
        for (uint32_t i0 = r0; i0 < r1; i0 += 32) {
            const uint32_t i = i0 + lane;
            const float x = i < r1 ? logit(i) : -INFINITY;
            const bool keep = tied ? keep_tied(i0, seen) : in_cuts(x, i);
            if (keep) sum += mass(x), ++count;
        }
        sum = warp_sum(sum);
        for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
        if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_count[warp] = count;
        __syncthreads();
        if (warp == 0) {
            const unsigned long long s = warp_sum(sh.warp_mass[lane]);
            uint32_t c = sh.warp_count[lane];
            for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (lane == 0) sh.draw_mass = s, sh.draw_count = c;
        }
        cluster.sync();
        unsigned long long all = 0, before = 0;
        uint32_t kept = 0;
        for (uint32_t r = 0; r < CL; ++r) {
            const unsigned long long s = *cluster.map_shared_rank(&sh.draw_mass, r);
            if (r < rank) before += s;
            all += s;
            kept += *cluster.map_shared_rank(&sh.draw_count, r);
        }
        double u = a.uniform[row];
        u = u >= 0.0 ? fmin(u, 1.0) : 0.0;   // NaN and negative values to 0
        unsigned long long target = static_cast<unsigned long long>(u * static_cast<double>(all));
        if (target >= all) target = all - 1;
        for (int w = 0; w < warp; ++w) before += sh.warp_mass[w];
        if (target >= before && target < before + sum) {   // this warp's run holds the token
            // the 32 ids that hold it: sums of 32 groups at a time, a group per lane (its ids taken in turn from
            // a place of its own: 32 different banks), or group after group where ties need their order
            unsigned long long at = before;
            uint32_t group = r0, seen_at = ties_before;
            if (tied) {
                for (uint32_t i0 = r0; i0 < r1; i0 += 32) {
                    uint32_t seen_now = seen_at;
                    const bool keep = keep_tied(i0, seen_now);
                    const unsigned long long s = warp_sum(keep ? mass(logit(i0 + lane)) : 0ull);
                    group = i0;
                    if (at + s > target) break;
                    at += s;
                    seen_at = seen_now;
                }
            } else {
                for (uint32_t g0 = r0; g0 < r1; g0 += 1024) {
                    unsigned long long s = 0;
                    for (int j = 0; j < 32; ++j) {
                        const uint32_t i = g0 + lane * 32 + ((j + lane) & 31);
                        const float x = i < r1 ? logit(i) : -INFINITY;
                        if (in_cuts(x, i)) s += mass(x);
                    }
                    unsigned long long p = s;
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long up = __shfl_up_sync(0xffffffffu, p, o);
                        if (lane >= o) p += up;
                    }
                    const uint32_t vote = __ballot_sync(0xffffffffu, at + p > target);
                    if (vote) {
                        const int f = __ffs(vote) - 1;
                        group = g0 + f * 32;
                        at += __shfl_sync(0xffffffffu, p - s, f);
                        break;
                    }
                    at += __shfl_sync(0xffffffffu, p, 31);
                }
            }
            const uint32_t i = group + lane;
            const float x = i < r1 ? logit(i) : -INFINITY;
            const bool keep = tied ? keep_tied(group, seen_at) : in_cuts(x, i);
            unsigned long long p = keep ? mass(x) : 0ull;
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long up = __shfl_up_sync(0xffffffffu, p, o);
                if (lane >= o) p += up;
            }
            const uint32_t vote = __ballot_sync(0xffffffffu, at + p > target);
            if (vote && lane == __ffs(vote) - 1) {
                a.token[row] = base + i;
                if (a.kept) a.kept[row] = kept;
                if (a.logprob) {
                    const double unit = __hiloint2double((1023 + a.shift) << 20, 0);
                    a.logprob[row] = static_cast<float>(static_cast<double>(x) - top_d - log(static_cast<double>(whole) / unit));
                }
            }
        }
    } else if (rank == 0 && tid == 0) {
        a.token[row] = top_id;
        if (a.kept) a.kept[row] = 1;
        if (a.logprob) {
            const double unit = __hiloint2double((1023 + a.shift) << 20, 0);
            a.logprob[row] = static_cast<float>(-log(static_cast<double>(whole) / unit));
        }
    }
    cluster.sync();   // no CTA leaves while another may read its shared memory
}

template <int CL>
cudaError_t launch(SampleArgs& a, const Rows& r, uint32_t n, cudaStream_t st) {
    const uint32_t per = (a.vocab + CL - 1) / CL;
    a.slice = (per + 1023) / 1024 * 1024;
    a.resident = a.slice <= kSmemIds;
    cudaError_t e = cudaFuncSetAttribute(smp_rows<CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemIds * sizeof(float));
    if (e == cudaSuccess && CL > 8) e = cudaFuncSetAttribute(smp_rows<CL>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n * CL);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = a.resident ? a.slice * sizeof(float) : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CL, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, smp_rows<CL>, a, r);
}

}  // namespace
}  // namespace gtm

using namespace gtm;

extern "C" GTM_API int gtm_sample_rows(const float* logits, uint32_t n, uint32_t vocab, uint64_t row_stride,
                                       const GtmSamplingRow* rows, const double* uniform, uint32_t* token, uint32_t* kept,
                                       float* logprob, void* stream) {
    const char* fn = "gtm_sample_rows";
    if (n == 0) {
        clear_error();
        return GTM_OK;
    }
    if (n > GTM_SAMPLE_MAX_ROWS) return set_error(GTM_ERR_INVALID, "%s: n=%u rows (at most %u)", fn, n, GTM_SAMPLE_MAX_ROWS);
    if (!logits || !rows || !token) return set_error(GTM_ERR_INVALID, "%s: null pointer", fn);
    if (vocab == 0 || vocab > GTM_SAMPLE_MAX_VOCAB)
        return set_error(GTM_ERR_INVALID, "%s: vocab=%u (1..%u)", fn, vocab, GTM_SAMPLE_MAX_VOCAB);
    if (n > 1 && row_stride < vocab)
        return set_error(GTM_ERR_INVALID, "%s: row_stride %llu below the vocabulary %u", fn, (unsigned long long)row_stride, vocab);
    auto aligned = [](const void* p, size_t m) { return reinterpret_cast<uintptr_t>(p) % m == 0; };
    if (!aligned(logits, 4) || !aligned(uniform, 8) || !aligned(token, 4) || !aligned(kept, 4) || !aligned(logprob, 4))
        return set_error(GTM_ERR_MISALIGNED, "%s: uniforms need 8-byte alignment, the others 4", fn);
    Rows r;
    for (uint32_t i = 0; i < n; ++i) {
        const GtmSamplingRow& p = rows[i];
        if (!(p.temperature >= 0.0f) || !std::isfinite(p.temperature))
            return set_error(GTM_ERR_INVALID, "%s: row %u: temperature must be finite and >= 0", fn, i);
        if (!(p.top_p > 0.0f && p.top_p <= 1.0f)) return set_error(GTM_ERR_INVALID, "%s: row %u: top_p must be in (0, 1]", fn, i);
        if (!(p.min_p >= 0.0f && p.min_p <= 1.0f)) return set_error(GTM_ERR_INVALID, "%s: row %u: min_p must be in [0, 1]", fn, i);
        if (p.top_k < 0) return set_error(GTM_ERR_INVALID, "%s: row %u: top_k must be >= 0", fn, i);
        if (p.temperature > 0.0f && !uniform) return set_error(GTM_ERR_INVALID, "%s: row %u needs a uniform", fn, i);
        r.v[i] = p;
    }
    SampleArgs a;
    a.logits = logits, a.row_stride = row_stride, a.uniform = uniform;
    a.token = token, a.kept = kept, a.logprob = logprob;
    a.vocab = vocab;
    int bits = 0;
    while ((1u << bits) < vocab) ++bits;
    a.shift = std::min(52, 62 - bits);
    a.vec = aligned(logits, 16) && (n == 1 || row_stride % 4 == 0);
    const cudaError_t e = getenv("CL16") ? launch<16>(a, r, n, static_cast<cudaStream_t>(stream)) : launch<8>(a, r, n, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_cuda_error(fn, e);
    }
    clear_error();
    return GTM_OK;
}
