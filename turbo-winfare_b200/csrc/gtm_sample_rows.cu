// Sampling a batch's rows (gtm_sample_rows, include/gtmoe_sampling.h).
//
// One cluster of CTAs per row: each keeps its share of the row's logits in shared memory (larger
// vocabularies are read from L2 again), so HBM is read once and every later pass runs on chip, with no
// workspace and one launch.
//   1 the largest logit, and its lowest id;
//   2 the cuts. Ranked by logit, every cut keeps a run from the top, so the kept set is the ids whose
//     key (logit, then lower id) is at least a border's. Ids are counted per level of max - logit,
//     1/128 wide; a level's weights agree within 0.8%, so the counts alone bracket the nucleus' border
//     to a few levels. One pass then sums the exact weights (all, above the bracket, per level in
//     it), and the ids of the level that holds the border are gathered and ranked. More ids than the
//     gather holds (equal or nearly equal logits) are narrowed by the logit's ordered bits instead;
//   3 the draw: sums of the kept weights per warp's run of ids, CTA and cluster, then one warp finds
//     the id in the run that the target falls in.
// Weights exp(l - max) are rounded to multiples of 2^-40 and summed as 64-bit integers: the sums cannot
// overflow, and do not depend on their order, so a token is reproducible, atomics and all.
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
constexpr float kPerNat = 128.0f;      // levels of max - logit: 16 and more is the last
constexpr int kGather = 1024;          // ids of the border's level that are ranked at once
constexpr uint32_t kSmemIds = 40960;   // ids of a share that stay in shared memory
constexpr uint64_t kMantissa = (1ull << 52) - 1;
constexpr int kShift = 40;             // weights are multiples of 2^-40: 2^22 of them stay below 2^63

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
    int power10[1024];                  // 2^(j / 1024) in units of 2^-30
    unsigned long long mass[kLevels];   // also the gathered keys
    uint32_t count[kLevels];
    unsigned long long warp_mass[kWarps], warp_mass2[kWarps];
    float warp_lo[kWarps], warp_hi[kWarps];
    uint32_t warp_count[kWarps];
    unsigned long long cta_key, cta_mass, cta_mass2, draw_mass, border_key;   // each read by the peers: none is reused
    uint32_t tie_count, draw_count, gathered;
    uint32_t first, last, by_count;     // the bracket's levels; the level that holds the top_k-th id
    uint32_t pick;                      // the level that holds the border
    unsigned long long pick_mass;       // mass and count of the levels above it
    uint32_t pick_count;
};

// exp((x - top) / temperature) as a multiple of 2^-40. Two forms:
//   exact: 2^(y / 256) with y = 256 log2(e) (x - top) / temperature = k + r, |r| <= 1/2, from a table of
//     2^(j / 256) and the exponential series to the fourth power of r ln 2 / 256 (the next term is below 2^-54);
//   short, for weights below 2^-10, i.e. most ids, in ~25 instructions: 2^(y / 1024) with y = c x - c top,
//     c = 1024 log2(e) / temperature as a sum of two floats and c top as an integer and a float; r is an fma of
//     an exact product (|r| <= 1, off by 2^-23), the series goes to its square in fp32 and is multiplied with
//     the table's 30 bits in integers: off by about 2^-31 of the weight, so by 2^-41.
// Which form an id takes depends on its logit alone, so equal logits weigh the same.
struct Scale {
    double rate;         // 256 log2(e) / temperature
    float hi, lo;        // 1,024 log2(e) / temperature as a sum of two floats; hi NaN: no short form
    float top_f;         // c top - top_i
    int top_i;
};
__device__ __forceinline__ Scale scale_of(double temperature, float top) {
    constexpr double kLog2e = 1.4426950408889634074;
    Scale c;
    c.rate = 256.0 * kLog2e / temperature;
    const double ten = 4.0 * c.rate, at = ten * top;
    c.hi = static_cast<float>(ten);
    c.lo = static_cast<float>(ten - static_cast<double>(c.hi));
    if (fabs(at) < 2097152.0) {   // 2^21: products c x that matter stay below 2^22, where their integers are exact
        c.top_i = __double2int_rn(at);
        c.top_f = static_cast<float>(at - c.top_i);
    } else {
        c.hi = __int_as_float(0x7FC00000);
        c.lo = c.top_f = 0.0f;
        c.top_i = 0;
    }
    return c;
}
__device__ __noinline__ unsigned long long exact_exp(const double* power, double d, double rate) {
    constexpr double kLn = 0.69314718055994530942 / 256.0;
    const double y = d * rate;
    if (!(y > -256.0 * 42)) return 0;   // below half of 2^-41; also x = -infinity
    const double t = y + 6755399441055744.0;   // 1.5 * 2^52: the nearest integer in the low word
    const int k = __double2loint(t);
    const double r = y - (t - 6755399441055744.0);
    double p = fma(r, kLn * kLn * kLn * kLn / 24.0, kLn * kLn * kLn / 6.0);
    p = fma(p, r, kLn * kLn / 2.0);
    p = fma(p, r, kLn);
    p = fma(p, r, 1.0) * power[k & 255];   // [1, 2), or just beside it by a rounding
    const unsigned long long m = (static_cast<unsigned long long>(__double_as_longlong(p)) & kMantissa) | (1ull << 52);
    const int s = 52 - kShift - (k >> 8) - (static_cast<int>(static_cast<unsigned>(__double2hiint(p)) >> 20) - 1023);
    return (m + (1ull << (s - 1))) >> s;   // 11 <= s <= 55
}
// The short form where it holds; else `big` is set (x = -infinity, and whatever is below 2^-42, among them).
__device__ __forceinline__ uint32_t short_exp(const Shared& sh, float x, const Scale& c, bool& big) {
    const float t = __fmaf_rn(x, c.hi, 12582912.0f);   // 1.5 * 2^23: the nearest integer in the low bits
    const int k = __float_as_int(t) - 0x4B400000 - c.top_i;
    big = static_cast<uint32_t>(k + 42 * 1024) >= 32u * 1024;   // a t beyond its range gives a k beyond this one
    float r = __fmaf_rn(x, c.hi, -__fsub_rn(t, 12582912.0f));
    r = __fsub_rn(__fmaf_rn(x, c.lo, r), c.top_f);
    constexpr float kLn = 0.69314718055994530942f / 1024.0f;
    // (z + z^2 / 2) * 2^32 with z = r kLn, to the nearest integer (below 2^22 in magnitude)
    const float g = __fmaf_rn(r, 0.5f * kLn * kLn * 4294967296.0f, kLn * 4294967296.0f);
    const int p = __float_as_int(__fmaf_rn(r, g, 12582912.0f)) - 0x4B400000;
    const int m = sh.power10[k & 1023];
    const uint32_t w = static_cast<uint32_t>(m + __mulhi(m, p)) >> ((-11 - (k >> 10)) & 31);   // twice the weight
    return big ? 0u : (w + 1) >> 1;
}
__device__ __forceinline__ unsigned long long fixed_exp(const Shared& sh, float x, float top, const Scale& c) {
    bool big;
    const uint32_t w = short_exp(sh, x, c, big);
    return big ? exact_exp(sh.power, static_cast<double>(x) - static_cast<double>(top), c.rate) : w;
}
// Sums weights with the exact forms put off: they are few, and a warp that stops for each holds up the others.
struct Summer {
    unsigned long long sum = 0;
    float put_off = -INFINITY;
    __device__ __forceinline__ void add(const Shared& sh, float x, float top, const Scale& c) {
        bool big;
        sum += short_exp(sh, x, c, big);
        if (big && x > -INFINITY) {
            if (put_off > -INFINITY) sum += exact_exp(sh.power, static_cast<double>(put_off) - static_cast<double>(top), c.rate);
            put_off = x;
        }
    }
    __device__ __forceinline__ unsigned long long total(const Shared& sh, float top, const Scale& c) {
        if (put_off > -INFINITY) sum += exact_exp(sh.power, static_cast<double>(put_off) - static_cast<double>(top), c.rate);
        put_off = -INFINITY;
        return sum;
    }
};

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
    if (tid < 256) sh.power[tid] = exp2(tid * (1.0 / 256.0));
    sh.power10[tid] = __double2int_rn(exp2(tid * (1.0 / 1024.0)) * 1073741824.0);
    unsigned long long best = 0;
    auto look = [&](uint32_t i, float x) {
        x = i < n ? as_logit(x) : -INFINITY;
        const unsigned long long key = i < n ? key_of(x, base + i) : 0;
        best = key > best ? key : best;
        return x;
    };
    if (a.resident && a.vec) {
        constexpr int U = 8;   // loads in flight per thread
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
    const Scale one = scale_of(1.0, top);
    const double top_d = top;
    auto weight = [&](float x) { return fixed_exp(sh, x, top, one); };
    // the nearest level, in the low bits of a float of 2^23 or more
    auto level = [&](float x) { return __float_as_uint(fminf(fmaf(top - x, kPerNat, 8388608.0f), 8388607.0f + kLevels)) - 0x4B000000u; };
    const bool greedy = !(rule.temperature > 0.0f);
    const bool cut_p = !greedy && rule.top_p < 1.0f, cut_k = !greedy && rule.top_k > 0 && static_cast<uint32_t>(rule.top_k) < a.vocab;
    // ids with a key below `border` are out: at first those without a finite logit, and those with p below
    // min_p of the largest, by the least logit that is not
    unsigned long long border = static_cast<unsigned long long>(ordered(-3.402823466e38f)) << 32;
    if (!greedy && rule.min_p > 0.0f) {
        const double floor_d = log(static_cast<double>(rule.min_p));
        uint32_t o = ordered(static_cast<float>(top_d + floor_d));
        while (o < ordered(top) && !(static_cast<double>(from_ordered(o)) - top_d >= floor_d)) ++o;
        while (o > ordered(-3.402823466e38f) && static_cast<double>(from_ordered(o - 1)) - top_d >= floor_d) --o;
        border = static_cast<unsigned long long>(o) << 32;
    }

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
        // a level's edges are off by the rounding of (max - l) * 128, its mass by fp32 sums and exponentials: 2^-12
        // covers them all
        constexpr float kMore = 1.0f + 0x1p-12f, kLess = 1.0f - 0x1p-12f;
        const float q0 = expf((0.5f - 2.0f * tid) / kPerNat), q1 = expf((-0.5f - 2.0f * tid) / kPerNat), q2 = expf((-1.5f - 2.0f * tid) / kPerNat);
        const float lo0 = c0 * q1 * kLess, hi0 = c0 * q0 * kMore, lo1 = tid == kThreads - 1 ? 0.0f : c1 * q2 * kLess, hi1 = c1 * q1 * kMore;
        uint32_t pc = c0 + c1;
        float pl = lo0 + lo1, ph = hi0 + hi1;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
            const float ul = __shfl_up_sync(0xffffffffu, pl, o), uh = __shfl_up_sync(0xffffffffu, ph, o);
            if (lane >= o) pc += uc, pl += ul, ph += uh;
        }
        if (lane == 31) sh.warp_count[warp] = pc, sh.warp_lo[warp] = pl, sh.warp_hi[warp] = ph;
        __syncthreads();
        uint32_t bc = 0;
        float bl = 0.0f, bh = 0.0f, all_lo = 0.0f, all_hi = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) bc += sh.warp_count[w], bl += sh.warp_lo[w], bh += sh.warp_hi[w];
            all_lo += sh.warp_lo[w], all_hi += sh.warp_hi[w];
        }
        const uint32_t cum1 = bc + pc, cum0 = cum1 - c1;
        const float l1 = bl + pl, l0 = bl + (pl - lo1), h1 = bh + ph, h0 = bh + (ph - hi1);
        if (cut_p) {
            const float low = rule.top_p * all_lo * kLess, high = rule.top_p * all_hi * kMore;
            if (c0 && h0 * kMore >= low) atomicMin(&sh.first, 2 * tid);
            if (c1 && h1 * kMore >= low) atomicMin(&sh.first, 2 * tid + 1);
            if (c0 && l0 * kLess >= high) atomicMin(&sh.last, 2 * tid);
            if (c1 && l1 * kLess >= high) atomicMin(&sh.last, 2 * tid + 1);
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
        Summer every, over;
        // below every id of the bracket
        const float low = !(bracket && cut_p) ? INFINITY : last == kLevels - 1u ? -3.402823466e38f : top - (static_cast<float>(last) + 1.0f) / kPerNat;
        for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
            const float4 x4 = four(i);
            const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) every.add(sh, x[j], top, one);
            const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (most >= low) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t lev = level(x[j]);
                    if (x[j] >= low && lev <= last) {
                        if (lev < first)
                            over.add(sh, x[j], top, one);
                        else
                            atomicAdd(&sh.mass[lev - first], weight(x[j]));
                    }
                }
            }
        }
        unsigned long long sum = every.total(sh, top, one), up = over.total(sh, top, one);
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
    unsigned long long need = 0;
    bool tied = false;   // of the ids with the border's logit only the first `ties` stay
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
            border = max(border, *cluster.map_shared_rank(&sh.border_key, 0));
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
                    tied = static_cast<unsigned long long>(lo) << 32 >= border;   // else min_p leaves fewer
                    border = max(border, static_cast<unsigned long long>(lo) << 32);
                }
                __syncthreads();
            }
        }
    }

    // ---- 3: the draw
    if (!greedy) {
        const Scale heat = scale_of(rule.temperature, top);
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
        const float edge_x = from_ordered(edge);
        const uint32_t least = static_cast<uint32_t>(border);
        auto in_cuts = [&](float x, uint32_t i) {   // key_of(x, base + i) >= border
            return x > edge_x || (x == edge_x && ~(base + i) >= least);
        };
        auto mass = [&](float x) { return fixed_exp(sh, x, top, heat); };
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
        Summer draw;
        uint32_t count = 0, seen = ties_before;
        if (tied) {
            for (uint32_t i0 = r0; i0 < r1; i0 += 32) {
                const uint32_t i = i0 + lane;
                if (keep_tied(i0, seen)) draw.add(sh, logit(i), top, heat), ++count;
            }
        } else {
            for (uint32_t i0 = r0; i0 < r1; i0 += 128) {
                const uint32_t i = i0 + 4 * lane;
                const float4 x4 = i < r1 ? four(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                const float x[4] = {x4.x, x4.y, x4.z, x4.w};
                const float most = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                if (!__any_sync(0xffffffffu, most >= edge_x)) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (in_cuts(x[j], i + j)) draw.add(sh, x[j], top, heat), ++count;
            }
        }
        const unsigned long long sum = warp_sum(draw.total(sh, top, heat));
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
                    Summer part;
                    for (int j = 0; j < 32; ++j) {
                        const uint32_t i = g0 + lane * 32 + ((j + lane) & 31);
                        const float x = i < r1 ? logit(i) : -INFINITY;
                        if (in_cuts(x, i)) part.add(sh, x, top, heat);
                    }
                    const unsigned long long s = part.total(sh, top, heat);
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
                    a.logprob[row] = static_cast<float>(static_cast<double>(x) - top_d - log(static_cast<double>(whole) * 0x1p-40));
                }
            }
        }
    } else if (rank == 0 && tid == 0) {
        a.token[row] = top_id;
        if (a.kept) a.kept[row] = 1;
        if (a.logprob) {
            a.logprob[row] = static_cast<float>(-log(static_cast<double>(whole) * 0x1p-40));
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
    a.vec = aligned(logits, 16) && (n == 1 || row_stride % 4 == 0);
    const cudaError_t e = getenv("CL16") ? launch<16>(a, r, n, static_cast<cudaStream_t>(stream)) : launch<8>(a, r, n, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_cuda_error(fn, e);
    }
    clear_error();
    return GTM_OK;
}
