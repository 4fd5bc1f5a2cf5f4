// Sampling a batch's rows (gtm_sample_rows, include/gtmoe_sampling.h).
//
// One cluster of CTAs per row: each keeps its share of the row's logits in shared memory (larger
// shares are read from L2 again), so HBM is read once and every later pass runs on chip, with no
// workspace and one launch. Two things take its time: instructions, ~25 for an id's weight, as many for the counts
// and the bracket's test (half of the issue slots at 64 rows), and ten cluster barriers a row (its largest stall):
// one row of 262,144 ids takes 47 us, 64 rows under mixed rules 170-181, 512 rows 871 (1.7 each); the bytes of 64 are
// 10.4 us.
//   1 the largest logit, and its lowest id;
//   2 the cuts. Ranked by logit, every cut keeps a run from the top, so the kept set is the ids whose
//     key (logit, then lower id) is at least a border's. Ids are counted per level of max - logit,
//     1/128 wide where it counts; a level's weights agree within 0.8%, so the counts alone bracket the
//     nucleus' border to a few levels. One pass sums the exact weights (all of them, and those above the bracket) and
//     gathers the bracket's ids, among which one CTA finds the border by halves. A bracket of more than 3,200 ids (nearly equal
//     logits) is narrowed by its levels' masses and then by the logit's ordered bits instead;
//   3 the draw: sums of the kept weights per warp's run of ids, CTA and cluster, then one warp finds
//     the id in the run that the target falls in.
// Weights exp(l - max) are rounded to multiples of 2^-40 and summed as 64-bit integers: the sums cannot
// overflow, and do not depend on their order, so a token is reproducible, atomics and all.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "gtm_internal.h"
#include "gtmoe_sampling.h"

namespace cg = cooperative_groups;

namespace gtm {
namespace {

constexpr int kLevels = 2048;
// Levels of max - logit: 1/128 wide up to 8 (1,024 of them), then three times as wide; 32 and more is the last.
constexpr float kFine = 128.0f, kCoarse = 128.0f / 3.0f, kOne = 8388608.0f;   // 2^23: a float's integers from here on
// The nearest level, in the low bits of a float; monotone in d.
__device__ __forceinline__ float near_level(float d) {
    return fminf(fmaf(d, kFine, kOne), fmaf(d, kCoarse, kOne + 683.0f));
}
__device__ __forceinline__ float level_middle(int level) { return level <= 1024 ? level / kFine : (level - 683) / kCoarse; }
constexpr uint32_t kGather = 3200;     // ids of a bracket that are gathered
constexpr uint32_t kHalfIds = 16384;   // or of one that leaves room for a second CTA
constexpr uint32_t kSmemIds = 40960;   // ids of a share that stay in shared memory
constexpr int kGroups = 10;            // parts of a warp's run of ids in the draw (128 ids of a share in shared memory)

// 2^(j / 1024) in units of 2^-62, from the exponential series in 64-bit arithmetic at compile time.
struct PowerTable {
    unsigned long long v[1024];
    constexpr PowerTable() : v() {
        for (int j = 0; j < 1024; ++j) {
            // 2^(j / 1024) = e^z, z < 0.7, as 1 + z (1 + z / 2 (1 + z / 3 (...))) in units of 2^-62
            constexpr unsigned long long kLn2 = 3196577161300663914ull;   // ln 2 in units of 2^-62
            const unsigned long long z = kLn2 / 1024 * j + kLn2 % 1024 * j / 1024;
            unsigned long long sum = 1ull << 62;
            for (int i = 24; i > 0; --i) sum = (1ull << 62) + mul62(z, sum) / i;
            v[j] = sum;
        }
    }
    static constexpr unsigned long long mul62(unsigned long long a, unsigned long long b) {   // a b / 2^62
        const unsigned long long ah = a >> 32, al = a & 0xFFFFFFFFu, bh = b >> 32, bl = b & 0xFFFFFFFFu;
        const unsigned long long mid = (al * bl >> 32) + (ah * bl & 0xFFFFFFFFu) + (al * bh & 0xFFFFFFFFu);
        const unsigned long long hi = ah * bh + (ah * bl >> 32) + (al * bh >> 32) + (mid >> 32);
        return (hi << 2) | (mid >> 30 & 3u);
    }
};
__device__ const PowerTable kPowers;

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

template <int kWarps>
struct __align__(16) Shared {
    unsigned long long power62[1024];   // 2^(j / 1024) in units of 2^-62
    int power30[1024];                  // and of 2^-30
    unsigned long long mass[kGather];   // masses of levels, or the gathered ids' keys
    uint32_t count[kLevels];
    unsigned long long key_lo, key_hi;  // of the gathered ids
    uint3 half[2][kWarps];
    unsigned long long warp_mass[kWarps], warp_mass2[kWarps], group_mass[kWarps][kGroups];
    float warp_near[kWarps], warp_var[kWarps];
    uint32_t warp_count[kWarps];
    unsigned long long cta_key, cta_mass, cta_mass2, draw_mass, border_key;   // each read by the peers: none is reused
    double floor_d;                     // log(min_p)
    float scale[3];                     // 1,024 log2(e) / temperature as a sum
    uint32_t tie_count, draw_count, gathered, members, border_at;
    uint32_t first, last, by_count;     // the bracket's levels; the level that holds the top_k-th id
    uint32_t pick;                      // the level that holds the border
    unsigned long long pick_mass;       // mass and count of the levels above it
    uint32_t pick_count;
};

// exp((x - top) / temperature) as a multiple of 2^-40, without double precision, of which this GPU does little.
// With c = 1024 log2(e) / temperature as a sum of three floats it is 2^(y / 1024), y = c (x - top), in two forms:
//   short, for weights below 2^-10, i.e. most ids, in ~25 instructions: y = c x - c top, c top as an integer and a
//     float; y = k + r with r an fma of an exact product (|r| <= 1, off by 2^-23); the series of 2^(r / 1024)
//     goes to its square in fp32 and is multiplied with 30 bits of a table of 2^(j / 1024): off by about 2^-31
//     of the weight, so by 2^-41;
//   exact: x - top as a sum of two floats, the products as sums of two floats each, added as 64-bit integers in
//     units of 2^-40; the series to its cube (the next term is below 2^-46) and the table's 62 bits in integers.
// Which form an id takes depends on its logit alone, so equal logits weigh the same.
struct Scale {
    float hi, lo, lo2;   // c
    float top_f;         // c top - top_i
    int top_i;
    bool brief;          // the short form may be used
};
__device__ __forceinline__ Scale scale_of(float hi, float lo, float lo2, float top) {
    Scale c;
    c.hi = hi, c.lo = lo, c.lo2 = lo2;
    const float p = __fmul_rn(hi, top);
    c.brief = fabsf(p) < 2097152.0f;   // 2^21: products c x that matter stay below 2^22, where their integers are exact
    const float n = rintf(p);
    c.top_i = c.brief ? static_cast<int>(n) : 0;
    c.top_f = __fadd_rn(__fsub_rn(p, n), __fmaf_rn(lo, top, __fmaf_rn(hi, top, -p)));
    return c;
}
template <class Sh>
__device__ __noinline__ unsigned long long exact_exp(const Sh& sh, float x, float top, float hi, float lo, float lo2) {
    const float d = __fsub_rn(x, top), b = __fsub_rn(d, x);
    if (d == 0.0f) return 1ull << 40;
    const float y = __fmul_rn(d, hi);
    if (!(y > -42.0f * 1024.0f)) return 0;   // far below: v is not formed
    const float e = __fsub_rn(__fsub_rn(x, __fsub_rn(d, b)), __fadd_rn(top, b));   // what the difference was rounded by
    const float q = __fmul_rn(d, lo);
    constexpr float kUnit = 1099511627776.0f;   // 2^40
    long long v = __float2ll_rn(y * kUnit) + __float2ll_rn(__fmaf_rn(d, hi, -y) * kUnit);
    v += __float2ll_rn(q * kUnit) + __float2ll_rn(__fmaf_rn(d, lo, -q) * kUnit);
    v += __float2ll_rn(__fmaf_rn(d, lo2, __fmaf_rn(e, hi, e * lo)) * kUnit);
    v = v > 0 ? 0 : v;
    const int k = static_cast<int>(v >> 40);
    if (k < -41 * 1024) return 0;   // below half of 2^-40; the shift below stays under 64
    const unsigned long long r = static_cast<unsigned long long>(v) << 24;              // in units of 2^-64
    const unsigned long long z = __umul64hi(r, 12486629536330718ull);                   // times ln 2 / 1024
    const unsigned long long z2 = __umul64hi(z, z) >> 1, z3 = __umul64hi(__umul64hi(z2, z), 6148914691236517205ull);   // / 3
    const unsigned long long m = sh.power62[k & 1023];
    const unsigned long long w = m + __umul64hi(m, z + z2 + z3);
    const int s = 22 - (k >> 10);
    return (w + (1ull << (s - 1))) >> s;
}
// The short form where it holds; else `big` is set (x = -infinity, and whatever is below 2^-42, among them).
template <class Sh>
__device__ __forceinline__ uint32_t short_exp(const Sh& sh, float x, const Scale& c, bool& big) {
    const float t = __fmaf_rn(x, c.hi, 12582912.0f);   // 1.5 * 2^23: the nearest integer in the low bits
    // unsigned, as what a t beyond its range gives wraps around; it gives a k beyond this one
    const uint32_t ku = __float_as_uint(t) - 0x4B400000u - static_cast<uint32_t>(c.top_i);
    const int k = static_cast<int>(ku);
    big = ku + 42u * 1024 >= 32u * 1024 || !c.brief;
    float r = __fmaf_rn(x, c.hi, -__fsub_rn(t, 12582912.0f));
    r = __fsub_rn(__fmaf_rn(x, c.lo, r), c.top_f);
    constexpr float kLn = 0.69314718055994530942f / 1024.0f;
    // (z + z^2 / 2) * 2^32 with z = r kLn, to the nearest integer (below 2^22 in magnitude)
    const float g = __fmaf_rn(r, 0.5f * kLn * kLn * 4294967296.0f, kLn * 4294967296.0f);
    const int p = static_cast<int>(__float_as_uint(__fmaf_rn(r, g, 12582912.0f)) - 0x4B400000u);
    const int m = sh.power30[k & 1023];
    const uint32_t w = (static_cast<uint32_t>(m) + static_cast<uint32_t>(__mulhi(m, p))) >> ((-11 - (k >> 10)) & 31);   // twice the weight
    return big ? 0u : (w + 1) >> 1;
}
template <class Sh>
__device__ __forceinline__ unsigned long long fixed_exp(const Sh& sh, float x, float top, const Scale& c) {
    bool big;
    const uint32_t w = short_exp(sh, x, c, big);
    return big ? exact_exp(sh, x, top, c.hi, c.lo, c.lo2) : w;
}
// The weights of four ids, those of `in`: short forms in one straight run (below 2^-10, so four fit 32 bits); the
// exact ones, which are few, stay behind in `big`.
template <class Sh>
__device__ __forceinline__ uint32_t short_four(const Sh& sh, const float (&x)[4], const bool (&in)[4], const Scale& c, uint32_t (&w)[4], uint32_t& big) {
    uint32_t sum = 0;
    big = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bool b;
        w[j] = short_exp(sh, x[j], c, b);
        w[j] = in[j] ? w[j] : 0u;
        big |= b && in[j] ? 1u << j : 0u;
        sum += w[j];
    }
    return sum;
}
__device__ __forceinline__ float pick(const float (&x)[4], int j) { return j & 2 ? (j & 1 ? x[3] : x[2]) : (j & 1 ? x[1] : x[0]); }

// ceil(p x) for 0 < p < 1, in integers.
__device__ __forceinline__ unsigned long long product_up(float p, unsigned long long x) {
    const uint32_t bits = __float_as_uint(p), e = bits >> 23;
    const unsigned long long m = e ? (bits & 0x7FFFFFu) | 0x800000u : bits & 0x7FFFFFu;   // p = m 2^-q
    const int q = 150 - static_cast<int>(e ? e : 1);                                       // 24 or more
    unsigned long long lo = m * x, hi = __umul64hi(m, x);
    if (q >= 88) return 1;
    if (q >= 64) return (hi >> (q - 64)) + ((lo | (hi & ((1ull << (q - 64)) - 1))) ? 1 : 0);
    return (hi << (64 - q)) + (lo >> q) + ((lo & ((1ull << q) - 1)) ? 1 : 0);
}
// floor(u x) for 0 <= u < 1, in integers (u to 64 bits).
__device__ __forceinline__ unsigned long long product_down(double u, unsigned long long x) {
    const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(u));
    const int e = static_cast<int>(bits >> 52);   // u = m 2^(e - 1075)
    const int s = 1011 + 0 - e;                   // to units of 2^-64: m 2^(e - 1011)
    if (e == 0 || s >= 53) return 0;
    const unsigned long long m = (bits & ((1ull << 52) - 1)) | (1ull << 52);
    return __umul64hi(s >= 0 ? m >> s : m << -s, x);
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <int CL, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) smp_rows(const __grid_constant__ SampleArgs a, const __grid_constant__ Rows rows) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int kWarps = kThreads / 32;
    Shared<kWarps>& sh = *reinterpret_cast<Shared<kWarps>*>(smem);
    float* slice_s = reinterpret_cast<float*>(smem + sizeof(sh));
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
        if (a.vec && i + 3 < n) {
            x = __ldg(reinterpret_cast<const float4*>(src + base + i));
            return make_float4(as_logit(x.x), as_logit(x.y), as_logit(x.z), as_logit(x.w));
        }
        x.x = as_logit(__ldg(src + base + i));
        x.y = i + 1 < n ? as_logit(__ldg(src + base + i + 1)) : -INFINITY;
        x.z = i + 2 < n ? as_logit(__ldg(src + base + i + 2)) : -INFINITY;
        x.w = i + 3 < n ? as_logit(__ldg(src + base + i + 3)) : -INFINITY;
        return x;
    };
    auto logit = [&](uint32_t i) { return a.resident ? slice_s[i] : as_logit(__ldg(src + base + i)); };

    // ---- 1: the largest logit and its lowest id
    for (int i = tid; i < 1024; i += kThreads) {
        sh.power62[i] = kPowers.v[i];
        sh.power30[i] = static_cast<int>((kPowers.v[i] + (1ull << 31)) >> 32);
    }
    if (tid == kThreads - 1) {   // what takes double precision, on one thread beside the loads
        const double c = 1477.3197218702985291 / static_cast<double>(rule.temperature);   // 1024 log2(e)
        const float hi = static_cast<float>(c), lo = static_cast<float>(c - hi);
        sh.scale[0] = hi;
        sh.scale[1] = isinf(hi) ? 0.0f : lo;
        sh.scale[2] = isinf(hi) ? 0.0f : static_cast<float>(c - hi - lo);
    } else if (tid == kThreads - 33 && rule.min_p > 0.0f) {
        sh.floor_d = log(static_cast<double>(rule.min_p));
    }
    float most = -INFINITY;
    uint32_t most_id = base;
    auto look = [&](uint32_t i, float x) {   // a thread's ids come in rising order
        x = i < n ? as_logit(x) : -INFINITY;
        if (x > most) most = x, most_id = base + i;
        return x;
    };
    if (a.vec) {
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
                if (i >= n) continue;
                const float4 y = make_float4(look(i, x[u].x), look(i + 1, x[u].y), look(i + 2, x[u].z), look(i + 3, x[u].w));
                if (a.resident) *reinterpret_cast<float4*>(slice_s + i) = y;
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
    unsigned long long best = key_of(most, most_id);
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (lane == 0) sh.warp_mass[warp] = best;
    __syncthreads();
    if (warp == 0) {
        best = lane < kWarps ? sh.warp_mass[lane] : 0;
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) sh.cta_key = best;
    }
    cluster.sync();
    best = lane < CL ? *cluster.map_shared_rank(&sh.cta_key, lane) : 0;   // a CTA's value per lane, here and below
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
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
    // 1,024 log2(e) as a sum of three floats
    constexpr double kC = 1477.3197218702985291;
    constexpr float kHi = static_cast<float>(kC), kLo = static_cast<float>(kC - kHi), kLo2 = static_cast<float>(kC - kHi - kLo);
    const Scale one = scale_of(kHi, kLo, kLo2, top);
    auto weight = [&](float x) { return fixed_exp(sh, x, top, one); };
    auto level = [&](float x) { return __float_as_uint(fminf(near_level(top - x), kOne - 1.0f + kLevels)) - 0x4B000000u; };
    const bool greedy = !(rule.temperature > 0.0f);
    const bool cut_p = !greedy && rule.top_p < 1.0f, cut_k = !greedy && rule.top_k > 0 && static_cast<uint32_t>(rule.top_k) < a.vocab;
    // ids with a key below `border` are out: at first those without a finite logit, and those with p below
    // min_p of the largest, by the least logit that is not
    unsigned long long border = static_cast<unsigned long long>(ordered(-3.402823466e38f)) << 32;
    if (!greedy && rule.min_p > 0.0f) {
        if (tid == 0) {
            const double floor_d = sh.floor_d, top_d = top;
            uint32_t o = ordered(static_cast<float>(top_d + floor_d));
            while (o < ordered(top) && !(static_cast<double>(from_ordered(o)) - top_d >= floor_d)) ++o;
            while (o > ordered(-3.402823466e38f) && static_cast<double>(from_ordered(o - 1)) - top_d >= floor_d) --o;
            sh.border_key = static_cast<unsigned long long>(o) << 32;
        }
        __syncthreads();
        border = sh.border_key;
        __syncthreads();
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
#pragma unroll 8
            for (int r = 0; r < CL; ++r) c += *cluster.map_shared_rank(&sh.count[mine], r);
        cluster.sync();
        if (tid < kPart)
#pragma unroll 8
            for (int r = 0; r < CL; ++r) *cluster.map_shared_rank(&sh.count[mine], r) = c;
        cluster.sync();
        // a few levels per thread: counts, and the mass down to and including each, near enough
        constexpr int kEach = kLevels / kThreads;
        uint32_t cnt[kEach], pc = 0;
        float near_mass[kEach], pe = 0.0f, var = 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = kEach * tid + j;
            const uint32_t k = sh.count[i];
            const float e = k * expf(-level_middle(i)), wide = i > 1024 ? 9.0f : 1.0f;
            if (k && !(i == 0 && k == 1)) var += wide * e * e / k;   // a lone largest id weighs 1
            pc += k, pe += e;
            cnt[j] = pc, near_mass[j] = pe;   // from the thread's first level on
        }
        const uint32_t own_c = pc;
        const float own_e = pe;
        for (int o = 16; o > 0; o >>= 1) var += __shfl_xor_sync(0xffffffffu, var, o);
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
            const float ue = __shfl_up_sync(0xffffffffu, pe, o);
            if (lane >= o) pc += uc, pe += ue;
        }
        if (lane == 31) sh.warp_count[warp] = pc, sh.warp_near[warp] = pe, sh.warp_var[warp] = var;
        __syncthreads();
        uint32_t bc = pc - own_c;
        float be = pe - own_e, all = 0.0f;
        var = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) bc += sh.warp_count[w], be += sh.warp_near[w];
            all += sh.warp_near[w], var += sh.warp_var[w];
        }
        // an id's weight is off by up to 1/256 of itself, evenly spread in a level: 3.5 standard deviations of the
        // sum (and 2^-13 of it for the rest) to either side, mostly a level or two
        const float slack = 3.5f * (1.0f / 256.0f) * 0.57735f * sqrtf(var) + all * 0x1p-13f;
        const float low = rule.top_p * all - slack, high = rule.top_p * all + slack;
#pragma unroll
        for (int j = kEach - 1; j >= 0; --j) {
            if (cnt[j] == (j ? cnt[j - 1] : 0u)) continue;   // no ids
            const int i = kEach * tid + j;
            const float m = be + near_mass[j];
            if (cut_p && m >= low) atomicMin(&sh.first, i);
            if (cut_p && m >= high) atomicMin(&sh.last, i);
            if (cut_k && bc + cnt[j] >= static_cast<uint32_t>(rule.top_k)) atomicMin(&sh.by_count, i);
        }
        __syncthreads();
        first = cut_p ? min(min(sh.first, sh.by_count), kLevels - 1u) : sh.by_count;
        last = cut_p ? min(min(sh.last, sh.by_count), kLevels - 1u) : sh.by_count;
        // ids above the bracket, and ids down to its end
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const uint32_t i = kEach * tid + j;
            if (i == first) sh.pick_count = bc + (j ? cnt[j - 1] : 0u);
            if (i == last) sh.members = bc + cnt[j];
        }
        __syncthreads();
    }
    const bool bracket = first < kLevels;   // else every id is kept
    uint32_t above = bracket ? sh.pick_count : 0;
    const uint32_t members = bracket ? sh.members - above : 0;
    const bool gather = members <= kGather;

    // ---- 2b: exact sums: the whole distribution, the levels above the bracket, each level in it
    unsigned long long whole = 0, above_mass = 0;
    {
        unsigned long long sum = 0, up = 0;
        float put_off = -INFINITY;   // an id whose exact form waits, so that no warp stops for each
        auto exact = [&](float x) {
            const unsigned long long w = exact_exp(sh, x, top, one.hi, one.lo, one.lo2);
            sum += w;
            if (level(x) < first) up += w;
        };
        // level(x) < first is near < before_first, level(x) <= last near <= to_last
        const bool collect = bracket && gather;
        const float before_first = kOne + (bracket ? first : 0);
        const float to_last = collect ? (last == kLevels - 1u ? INFINITY : kOne + last) : -1.0f;
        for (uint32_t i = tid * 4; i < n; i += kThreads * 4) {
            const float4 x4 = four(i);
            const float x[4] = {x4.x, x4.y, x4.z, x4.w};
            constexpr bool kAll[4] = {true, true, true, true};
            uint32_t w[4], big;
            sum += short_four(sh, x, kAll, one, w, big);
            uint32_t above4 = 0, inside = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float near = near_level(top - x[j]);
                above4 += near < before_first ? w[j] : 0u;
                inside |= near >= before_first && near <= to_last ? 1u << j : 0u;
            }
            up += above4;
            for (uint32_t left = inside | big; left; left &= left - 1) {
                const int j = __ffs(left) - 1;
                const float y = pick(x, j);
                if (!(y > -INFINITY)) continue;
                if (inside >> j & 1) sh.mass[atomicAdd(&sh.gathered, 1u)] = key_of(y, base + i + j);
                if (big >> j & 1) {
                    if (put_off > -INFINITY) exact(put_off);
                    put_off = y;
                }
            }
        }
        if (put_off > -INFINITY) exact(put_off);
        sum = warp_sum(sum), up = warp_sum(up);
        if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_mass2[warp] = up;
        __syncthreads();
        if (warp == 0) {
            sum = warp_sum(lane < kWarps ? sh.warp_mass[lane] : 0ull), up = warp_sum(lane < kWarps ? sh.warp_mass2[lane] : 0ull);
            if (lane == 0) sh.cta_mass = sum, sh.cta_mass2 = up;
        }
        cluster.sync();
        whole = warp_sum(lane < CL ? *cluster.map_shared_rank(&sh.cta_mass, lane) : 0ull);
        above_mass = warp_sum(lane < CL ? *cluster.map_shared_rank(&sh.cta_mass2, lane) : 0ull);
    }
    uint32_t border_level = kLevels, ties = 0xFFFFFFFFu;
    unsigned long long need = 0;
    bool tied = false;   // of the ids with the border's logit only the first `ties` stay
    if (bracket) need = cut_p ? product_up(rule.top_p, whole) : ~0ull;
    bool sought = bracket;
    if (bracket && gather && above_mass < need) {   // else the bracket begins too low
        // ---- 2c: the bracket's ids, to the cluster's first CTA, sorted; the border is the first that reaches a cut
        if (rank != 0) {
            if (tid == 0) sh.border_at = atomicAdd(cluster.map_shared_rank(&sh.gathered, 0), sh.gathered);
            __syncthreads();
            unsigned long long* list = cluster.map_shared_rank(sh.mass, 0) + sh.border_at;
            for (uint32_t i = tid; i < sh.gathered; i += kThreads) list[i] = sh.mass[i];
        }
        cluster.sync();
        if (rank == 0) {
            // a few ids per thread; the border is the largest key with which those from it on reach a cut: halves of
            // the range [lo, hi) that holds it, until one id is left
            if (tid == 0) sh.border_key = 0, sh.key_lo = ~0ull, sh.key_hi = 0;
            __syncthreads();
            constexpr int kMine = (kGather + kThreads - 1) / kThreads;
            static_assert(kMine < 8, "a warp's sums of 24-bit parts stay within 32 bits");
            unsigned long long key[kMine], w[kMine];
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                const uint32_t i = tid + j * kThreads;
                key[j] = i < members ? sh.mass[i] : 0;
                w[j] = key[j] ? weight(from_ordered(static_cast<uint32_t>(key[j] >> 32))) : 0;
                if (key[j]) {
                    atomicMin(&sh.key_lo, key[j]);
                    atomicMax(&sh.key_hi, key[j]);
                }
            }
            __syncthreads();
            unsigned long long lo = sh.key_lo, hi = sh.key_hi + 1;
            // ids from `from` on, and their mass (24 and 17 bits apart: 3,200 weights of 2^40 at most)
            int turn = 0;
            auto down_to = [&](unsigned long long from, uint32_t& count) {
                uint32_t c = 0, wl = 0, wh = 0;
#pragma unroll
                for (int j = 0; j < kMine; ++j)
                    if (key[j] >= from) ++c, wl += static_cast<uint32_t>(w[j]) & 0xFFFFFFu, wh += static_cast<uint32_t>(w[j] >> 24);
                c = __reduce_add_sync(0xffffffffu, c), wl = __reduce_add_sync(0xffffffffu, wl), wh = __reduce_add_sync(0xffffffffu, wh);
                if (lane == 0) sh.half[turn][warp] = make_uint3(c, wl, wh);
                __syncthreads();
                const uint3 v = lane < kWarps ? sh.half[turn][lane] : make_uint3(0, 0, 0);
                turn ^= 1;
                count = __reduce_add_sync(0xffffffffu, v.x);
                const unsigned long long l = __reduce_add_sync(0xffffffffu, v.y & 0xFFFFu), h = __reduce_add_sync(0xffffffffu, v.y >> 16);
                return l + (h << 16) + (static_cast<unsigned long long>(__reduce_add_sync(0xffffffffu, v.z)) << 24);
            };
            const auto reached = [&](unsigned long long mass, uint32_t count) {
                return (cut_p && above_mass + mass >= need) || (cut_k && above + count >= static_cast<uint32_t>(rule.top_k));
            };
            uint32_t at_lo, at_hi = 0, c;
            const bool any = reached(down_to(lo, at_lo), at_lo);
            while (any && at_lo - at_hi > 1) {
                const unsigned long long mid = lo + (hi - lo) / 2;
                if (reached(down_to(mid, c), c))
                    lo = mid, at_lo = c;
                else
                    hi = mid, at_hi = c;
            }
#pragma unroll
            for (int j = 0; j < kMine; ++j)
                if (any && key[j] >= lo && key[j] < hi) sh.border_key = key[j];
            __syncthreads();
        }
        cluster.sync();
        const unsigned long long key = *cluster.map_shared_rank(&sh.border_key, 0);
        sought = key == 0;   // the bracket ends too high
        border = max(border, key);
        cluster.sync();      // the peers have read the key
    }
    if (sought) {
        // ---- 2c otherwise (many nearly equal logits, or a border that the counts misjudged): the exact masses of all
        // levels, and then of the parts of the border's by the bits of the logit
        first = 0, last = kLevels - 1, above = 0, above_mass = 0;
        for (int i = tid; i < kLevels; i += kThreads) sh.mass[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n && cut_p; i += kThreads) {
            const float x = logit(i);
            if (x > -INFINITY) atomicAdd(&sh.mass[level(x)], weight(x));
        }
        cluster.sync();
        if (warp == 0) {   // walk the levels, 32 at a time; masses of the whole cluster
            unsigned long long run = above_mass;
            uint32_t run_c = above;
            for (uint32_t i = first; i <= last; i += 32) {
                const uint32_t lev = i + lane;
                unsigned long long own = 0;
                if (cut_p && lev <= last)
#pragma unroll 2
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
        {
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
#pragma unroll 2
                    for (int r = 0; r < CL; ++r) {
                        m += *cluster.map_shared_rank(&sh.mass[mine], r);
                        c += *cluster.map_shared_rank(&sh.count[mine], r);
                    }
                cluster.sync();
                if (tid < kPart)
#pragma unroll 2
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
        const Scale heat = scale_of(sh.scale[0], sh.scale[1], sh.scale[2], top);
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
        unsigned long long sum = 0;
        uint32_t count = 0, seen = ties_before;
        // ids of a group: 128 at a time
        const uint32_t per_group = (run + kGroups * 128 - 1) / (kGroups * 128) * 128;
        // this lane's share of the 128 ids from i0 on (its four, in id order)
        auto of_four = [&](uint32_t i0, float (&x)[4], bool (&in)[4]) {
            const uint32_t i = i0 + 4 * lane;
            const float4 x4 = i < r1 ? four(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            x[0] = x4.x, x[1] = x4.y, x[2] = x4.z, x[3] = x4.w;
#pragma unroll
            for (int j = 0; j < 4; ++j) in[j] = in_cuts(x[j], i + j);
        };
        auto exact_mass = [&](float x) { return exact_exp(sh, x, top, heat.hi, heat.lo, heat.lo2); };
        auto mass_of_four = [&](const float (&x)[4], const bool (&in)[4]) {
            uint32_t w[4], big;
            unsigned long long m = short_four(sh, x, in, heat, w, big);
            for (; big; big &= big - 1) m += exact_mass(pick(x, __ffs(big) - 1));
            return m;
        };
        if (tied) {
            for (uint32_t i0 = r0; i0 < r1; i0 += 32) {
                const uint32_t i = i0 + lane;
                if (keep_tied(i0, seen)) sum += mass(logit(i)), ++count;
            }
        } else {
            float put_off = -INFINITY;   // as above
            int put_off_group = 0;
            for (int g = 0; g < kGroups; ++g) {
                unsigned long long m = 0;
                for (uint32_t i0 = r0 + g * per_group; i0 < min(r1, r0 + (g + 1) * per_group); i0 += 128) {
                    float x[4];
                    bool in[4];
                    of_four(i0, x, in);
                    if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) continue;
                    uint32_t w[4], big;
                    m += short_four(sh, x, in, heat, w, big);
#pragma unroll
                    for (int j = 0; j < 4; ++j) count += in[j];
                    for (; big; big &= big - 1) {
                        if (put_off > -INFINITY) m += exact_mass(pick(x, __ffs(big) - 1));
                        else put_off = pick(x, __ffs(big) - 1), put_off_group = g;
                    }
                }
                m = warp_sum(m);
                if (lane == 0) sh.group_mass[warp][g] = m;
                sum += lane == 0 ? m : 0ull;
            }
            __syncwarp();
            if (put_off > -INFINITY) {
                const unsigned long long m = exact_mass(put_off);
                sum += m;
                atomicAdd(&sh.group_mass[warp][put_off_group], m);
            }
        }
        sum = warp_sum(sum);
        for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
        if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_count[warp] = count;
        __syncthreads();
        if (warp == 0) {
            const unsigned long long s = warp_sum(lane < kWarps ? sh.warp_mass[lane] : 0ull);
            uint32_t c = lane < kWarps ? sh.warp_count[lane] : 0u;
            for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (lane == 0) sh.draw_mass = s, sh.draw_count = c;
        }
        cluster.sync();
        const unsigned long long of_lane = lane < CL ? *cluster.map_shared_rank(&sh.draw_mass, lane) : 0ull;
        const unsigned long long all = warp_sum(of_lane);
        unsigned long long before = warp_sum(lane < rank ? of_lane : 0ull);
        const uint32_t kept = __reduce_add_sync(0xffffffffu, lane < CL ? *cluster.map_shared_rank(&sh.draw_count, lane) : 0u);
        const double u = a.uniform[row];   // NaN and negative values stand for 0
        const unsigned long long target = !(u > 0.0) ? 0 : u < 1.0 ? min(product_down(u, all), all - 1) : all - 1;
        for (int w = 0; w < warp; ++w) before += sh.warp_mass[w];
        if (target >= before && target < before + sum) {   // this warp's run holds the token
            // the group that holds it, the 128 ids in that, and the id; where ties need their order, 32 ids at a time
            unsigned long long at = before;
            uint32_t group = r0, seen_at = ties_before;
            uint32_t id = 0;
            float x = -INFINITY;
            bool mine = false;
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
                const uint32_t i = group + lane;
                x = i < r1 ? logit(i) : -INFINITY;
                const bool keep = keep_tied(group, seen_at);
                unsigned long long p = keep ? mass(x) : 0ull;
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long up = __shfl_up_sync(0xffffffffu, p, o);
                    if (lane >= o) p += up;
                }
                const uint32_t vote = __ballot_sync(0xffffffffu, at + p > target);
                mine = vote && lane == __ffs(vote) - 1;
                id = base + i;
            } else {
                __syncwarp();   // lane 0's group sums
                int g = 0;
                for (; g < kGroups - 1 && at + sh.group_mass[warp][g] <= target; ++g) at += sh.group_mass[warp][g];
                for (uint32_t i0 = r0 + g * per_group; i0 < r1; i0 += 128) {
                    float y[4];
                    bool in[4];
                    of_four(i0, y, in);
                    const unsigned long long m = mass_of_four(y, in);
                    unsigned long long p = m;
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long up = __shfl_up_sync(0xffffffffu, p, o);
                        if (lane >= o) p += up;
                    }
                    const uint32_t vote = __ballot_sync(0xffffffffu, at + p > target);
                    if (vote) {
                        mine = lane == __ffs(vote) - 1;
                        if (mine) {
                            unsigned long long run_m = at + p - m;
                            for (int j = 0; j < 4; ++j) {
                                const float z = pick(y, j);
                                const bool keep = j & 2 ? (j & 1 ? in[3] : in[2]) : (j & 1 ? in[1] : in[0]);
                                if (!keep) continue;
                                run_m += mass(z);
                                if (run_m > target) {
                                    x = z;
                                    id = base + i0 + 4 * lane + j;
                                    break;
                                }
                            }
                        }
                        break;
                    }
                    at += __shfl_sync(0xffffffffu, p, 31);
                }
            }
            if (mine) {
                a.token[row] = id;
                if (a.kept) a.kept[row] = kept;
                if (a.logprob) {
                    a.logprob[row] = static_cast<float>(static_cast<double>(x) - static_cast<double>(top) - log(static_cast<double>(whole) * 0x1p-40));
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

template <int CL, int T>
cudaError_t launch(SampleArgs& a, const Rows& r, uint32_t n, cudaStream_t st) {
    using Sh = Shared<T / 32>;
    constexpr uint32_t kMost = T == 1024 ? kSmemIds : kHalfIds;
    static_assert(T == 1024 || 2 * (sizeof(Sh) + kMost * sizeof(float) + 1024) <= 228 * 1024, "two CTAs on an SM");
    const uint32_t per = (a.vocab + CL - 1) / CL;
    a.slice = (per + 1023) / 1024 * 1024;
    a.resident = a.slice <= kMost;
    cudaError_t e = cudaFuncSetAttribute(smp_rows<CL, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Sh) + kMost * sizeof(float));
    if (e == cudaSuccess && CL > 8) e = cudaFuncSetAttribute(smp_rows<CL, T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n * CL);
    cfg.blockDim = dim3(T);
    cfg.dynamicSmemBytes = sizeof(Sh) + (a.resident ? a.slice * sizeof(float) : 0);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CL, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, smp_rows<CL, T>, a, r);
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
    // Few rows are a matter of latency: sixteen CTAs a row, or eight, keep every SM at work (262,144 ids: 8 rows
    // 75 us, 12 rows 69 with eight of 1,024 threads against 90 of 512). Many rows are one of throughput: CTAs of
    // 512 threads, two on an SM, so that one's barriers pass behind the other's work, and as few a row as take
    // their share into shared memory (four against eight: 64 rows of 32,000 ids 54 against 68 us, of 262,144 198
    // against 195), or fewer still where the rows alone fill the GPU (512 of 262,144 ids: 871 against 1,027).
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = n <= 8                                ? launch<16, 1024>(a, r, n, st)
                          : vocab <= 4 * kHalfIds || n > 128 ? launch<4, 512>(a, r, n, st)
                          : n <= 32                             ? launch<8, 1024>(a, r, n, st)
                                                                : launch<8, 512>(a, r, n, st);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_cuda_error(fn, e);
    }
    clear_error();
    return GTM_OK;
}
