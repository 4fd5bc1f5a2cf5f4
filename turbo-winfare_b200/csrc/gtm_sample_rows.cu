// Sampling a batch's rows (gtm_sample_rows, include/gtmoe_sampling.h).
//
// One cluster of eight CTAs per row: each keeps an eighth of the row's logits in shared memory
// (larger vocabularies are read from L2 again), so HBM is read once and every later pass runs on
// chip, with no workspace and one launch.
//   1 the largest logit, and its lowest id;
//   2 the cuts. Ranked by logit, every cut keeps a run from the top, so the kept set is "logit
//     above a threshold, and the lowest r ids at it". A histogram of 2,048 levels (first of
//     max - logit in steps of 1/64, then of the logit's ordered bits inside the level that holds
//     the border, 11 + 11 + 10 of them) narrows the border to equal logits in at most four passes;
//   3 the draw: sums of the kept weights per warp's run of ids, CTA and cluster, then one warp
//     walks the run that the target falls in.
// Weights exp(l - max) are 64-bit, rounded to multiples of 2^-(62 - bits of the vocabulary), and
// summed as 64-bit integers: the sums cannot overflow, do not depend on their order (so the token
// is reproducible, atomics and all) and are within 2^-44 of the weights' at a vocabulary of 2^18.
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

constexpr int kCluster = 8;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kLevels = 2048;
constexpr uint32_t kSmemIds = 40960;   // ids of a slice that stay in shared memory

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
    bool vec, resident;      // 16-byte loads; the slice stays in shared memory
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

struct Shared {
    unsigned long long mass[kLevels];
    uint32_t count[kLevels];
    unsigned long long warp_mass[kWarps];
    uint32_t warp_count[kWarps];
    unsigned long long cta_key;
    unsigned long long cta_mass;
    uint32_t cta_count;
    uint32_t pick;            // the level that holds the border
    unsigned long long pick_mass;
    uint32_t pick_count;
};

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1)
    smp_rows(const __grid_constant__ SampleArgs a, const __grid_constant__ Rows rows) {
    extern __shared__ __align__(16) float slice_s[];
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), row = blockIdx.x / kCluster;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const GtmSamplingRow rule = rows.v[row];
    const float* src = a.logits + row * a.row_stride;
    const uint32_t base = min(a.vocab, rank * a.slice), n = min(a.slice, a.vocab - base);
    auto logit = [&](uint32_t i) { return a.resident ? slice_s[i] : as_logit(__ldg(src + base + i)); };

    // ---- 1: the largest logit and its lowest id
    unsigned long long best = 0;
    auto look = [&](uint32_t i, float x) {
        x = as_logit(x);
        const unsigned long long key = (static_cast<unsigned long long>(ordered(x)) << 32) | static_cast<uint32_t>(~(base + i));
        best = key > best ? key : best;
        return x;
    };
    if (a.resident && a.vec) {
        for (uint32_t i = threadIdx.x * 4; i < n; i += kThreads * 4) {
            if (i + 3 < n) {
                const float4 x = __ldg(reinterpret_cast<const float4*>(src + base + i));
                *reinterpret_cast<float4*>(slice_s + i) = make_float4(look(i, x.x), look(i + 1, x.y), look(i + 2, x.z), look(i + 3, x.w));
            } else {
                for (uint32_t j = i; j < n; ++j) slice_s[j] = look(j, __ldg(src + base + j));
            }
        }
    } else {
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const float x = look(i, __ldg(src + base + i));
            if (a.resident) slice_s[i] = x;
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if (lane == 0) sh.warp_mass[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) best = sh.warp_mass[w] > best ? sh.warp_mass[w] : best;
        sh.cta_key = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < kCluster; ++r) {
        const unsigned long long other = *cluster.map_shared_rank(&sh.cta_key, r);
        best = other > best ? other : best;
    }
    const float top = from_ordered(static_cast<uint32_t>(best >> 32));
    const uint32_t top_id = ~static_cast<uint32_t>(best);
    if (isinf(top)) {   // the same for every CTA of the cluster
        if (rank == 0 && threadIdx.x == 0) {
            a.token[row] = 0xFFFFFFFFu;
            if (a.kept) a.kept[row] = 0;
            if (a.logprob) a.logprob[row] = __int_as_float(0x7FC00000);
        }
        cluster.sync();   // no CTA leaves while another may read its shared memory
        return;
    }
    const double unit = __hiloint2double((1023 + a.shift) << 20, 0);
    auto weight = [&](float x) {   // exp(x - top) in units of 2^-shift
        return static_cast<unsigned long long>(__double2ll_rn(exp(static_cast<double>(x) - static_cast<double>(top)) * unit));
    };
    const bool greedy = !(rule.temperature > 0.0f);
    const bool cut_p = !greedy && rule.top_p < 1.0f, cut_k = !greedy && rule.top_k > 0;
    // ids with p below min_p of the largest are out from the start
    const double floor_d = !greedy && rule.min_p > 0.0f ? log(static_cast<double>(rule.min_p)) : -INFINITY;
    auto alive = [&](float x) { return static_cast<double>(x) - static_cast<double>(top) >= floor_d; };

    // ---- 2: the border: ids of a logit above `edge` are kept, and the first `ties` ids at it
    uint32_t edge = 0, ties = 0xFFFFFFFFu, above = 0;   // edge 0 is below every finite logit's bits
    unsigned long long whole = 0;                       // the whole distribution's mass
    {
        unsigned long long need_mass = 0, above_mass = 0;
        uint32_t lo = 0, bits = 32;   // the border's logit has these high bits once pass > 0
        uint32_t level0 = 0;
        const int passes = (cut_p || cut_k) ? 4 : 1;
        for (int pass = 0; pass < passes; ++pass) {
            for (int i = threadIdx.x; i < kLevels; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
            __syncthreads();
            const uint32_t take = pass == 3 ? 10 : 11;
            auto near_level = [&](float x) { return static_cast<uint32_t>(fminf((top - x) * 64.0f, kLevels - 1.0f)); };
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                const float x = logit(i);
                uint32_t lev;
                if (pass == 0) {
                    lev = near_level(x);
                } else {
                    if (near_level(x) != level0 || (pass > 1 && (ordered(x) >> bits) != lo)) continue;
                    lev = kLevels - 1 - ((ordered(x) >> (bits - take)) & ((1u << take) - 1));   // larger logits first
                }
                if (!(x > -INFINITY)) continue;
                const unsigned long long w = weight(x);
                if (w) atomicAdd(&sh.mass[lev], w);
                if (alive(x)) atomicAdd(&sh.count[lev], 1u);
            }
            cluster.sync();
            // every CTA sums its eighth of the levels over the cluster, then all gather the sums
            constexpr int kPart = kLevels / kCluster;
            unsigned long long m = 0;
            uint32_t c = 0;
            const int mine = rank * kPart + threadIdx.x;
            if (threadIdx.x < kPart)
                for (int r = 0; r < kCluster; ++r) {
                    m += *cluster.map_shared_rank(&sh.mass[mine], r);
                    c += *cluster.map_shared_rank(&sh.count[mine], r);
                }
            cluster.sync();
            if (threadIdx.x < kPart)
                for (int r = 0; r < kCluster; ++r) {
                    *cluster.map_shared_rank(&sh.mass[mine], r) = m;
                    *cluster.map_shared_rank(&sh.count[mine], r) = c;
                }
            cluster.sync();
            if (warp == 0) {   // walk the levels from the top, 32 at a time
                unsigned long long sum = 0;
                if (pass == 0) {
                    for (int i = lane; i < kLevels; i += 32) sum += sh.mass[i];
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    whole = sum;
                    if (cut_p) {
                        const double t = static_cast<double>(rule.top_p) * static_cast<double>(sum);
                        need_mass = static_cast<unsigned long long>(ceil(t));
                    }
                }
                uint32_t found = kLevels;
                unsigned long long run_m = above_mass;
                uint32_t run_c = above;
                for (int i = 0; i < kLevels && passes > 1; i += 32) {
                    unsigned long long pm = sh.mass[i + lane];
                    uint32_t pc = sh.count[i + lane];
                    const unsigned long long own_m = pm;
                    const uint32_t own_c = pc;
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long um = __shfl_up_sync(0xffffffffu, pm, o);
                        const uint32_t uc = __shfl_up_sync(0xffffffffu, pc, o);
                        if (lane >= o) pm += um, pc += uc;
                    }
                    const bool here = (cut_p && run_m + pm >= need_mass) || (cut_k && run_c + pc >= static_cast<uint32_t>(rule.top_k));
                    const uint32_t vote = __ballot_sync(0xffffffffu, here);
                    if (vote) {
                        const int f = __ffs(vote) - 1;
                        found = i + f;
                        run_m += __shfl_sync(0xffffffffu, pm - own_m, f);
                        run_c += __shfl_sync(0xffffffffu, pc - own_c, f);
                        break;
                    }
                    run_m += __shfl_sync(0xffffffffu, pm, 31);
                    run_c += __shfl_sync(0xffffffffu, pc, 31);
                }
                if (lane == 0) sh.pick = found, sh.pick_mass = run_m, sh.pick_count = run_c, sh.cta_mass = whole, sh.cta_key = need_mass;
            }
            __syncthreads();
            if (pass == 0) whole = sh.cta_mass, need_mass = sh.cta_key;
            const uint32_t found = sh.pick;
            if (passes == 1 || found == kLevels) {   // no border: everything alive is kept
                above = sh.pick_count;
                break;
            }
            above = sh.pick_count, above_mass = sh.pick_mass;
            if (pass == 0) {
                level0 = found;
            } else {
                lo = (lo << take) | (kLevels - 1 - found);
                if (pass == 3) lo &= 0xFFFFFFFFu;
                bits -= take;
            }
            if (pass == 3) {
                edge = lo;
                const unsigned long long w = weight(from_ordered(edge));
                ties = sh.count[found];
                if (cut_k) ties = min(ties, static_cast<uint32_t>(rule.top_k) - above);
                if (cut_p && w) {
                    const unsigned long long short_of = need_mass > above_mass ? need_mass - above_mass : 1;
                    const unsigned long long t = (short_of + w - 1) / w;
                    ties = t < ties ? static_cast<uint32_t>(t) : ties;
                }
                if (above == 0 && ties == 0) ties = 1;
            }
            __syncthreads();
        }
    }
    const bool border = edge != 0;

    // ---- 3: the draw
    uint32_t token = top_id, kept = 1;
    if (!greedy) {
        const double scale = 1.0 / static_cast<double>(rule.temperature);
        auto mass = [&](float x) {
            return static_cast<unsigned long long>(
                __double2ll_rn(exp((static_cast<double>(x) - static_cast<double>(top)) * scale) * unit));
        };
        const uint32_t run = a.slice / kWarps;   // a warp's run of ids
        const uint32_t r0 = warp * run, r1 = min(n, r0 + run);
        // ids at the border's logit before this CTA and warp
        uint32_t ties_before = 0;
        if (border) {
            uint32_t c = 0;
            for (uint32_t i = r0 + lane; i < r1; i += 32) c += ordered(logit(i)) == edge;
            for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
            if (lane == 0) sh.warp_count[warp] = c;
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t s = 0;
                for (int w = 0; w < kWarps; ++w) s += sh.warp_count[w];
                sh.cta_count = s;
            }
            cluster.sync();
            for (uint32_t r = 0; r < rank; ++r) ties_before += *cluster.map_shared_rank(&sh.cta_count, r);
            for (int w = 0; w < warp; ++w) ties_before += sh.warp_count[w];
            cluster.sync();
        }
        // walks the run, calling f(id, weight) with lanes in id order; every lane calls it
        auto walk = [&](auto&& f) {
            uint32_t seen = ties_before;
            for (uint32_t i0 = r0; i0 < r1; i0 += 32) {
                const uint32_t i = i0 + lane;
                const float x = i < r1 ? logit(i) : -INFINITY;
                const uint32_t o = ordered(x);
                bool keep = x > -INFINITY && alive(x);
                if (border) {
                    const uint32_t at = __ballot_sync(0xffffffffu, o == edge);
                    if (o == edge)
                        keep = keep && seen + __popc(at & ((1u << lane) - 1)) < ties;
                    else
                        keep = keep && o > edge;
                    seen += __popc(at);
                }
                if (f(base + i, keep ? mass(x) : 0ull, keep)) break;
            }
        };
        unsigned long long sum = 0;
        uint32_t count = 0;
        walk([&](uint32_t, unsigned long long w, bool keep) {
            sum += w;
            count += keep;
            return false;
        });
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            count += __shfl_xor_sync(0xffffffffu, count, o);
        }
        if (lane == 0) sh.warp_mass[warp] = sum, sh.warp_count[warp] = count;
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long s = 0;
            uint32_t c = 0;
            for (int w = 0; w < kWarps; ++w) s += sh.warp_mass[w], c += sh.warp_count[w];
            sh.cta_mass = s, sh.cta_count = c;
        }
        cluster.sync();
        unsigned long long all = 0, before = 0;
        kept = 0;
        for (uint32_t r = 0; r < kCluster; ++r) {
            const unsigned long long s = *cluster.map_shared_rank(&sh.cta_mass, r);
            if (r < rank) before += s;
            all += s;
            kept += *cluster.map_shared_rank(&sh.cta_count, r);
        }
        double u = a.uniform[row];
        u = u >= 0.0 ? fmin(u, 1.0) : 0.0;   // NaN and negative values to 0
        unsigned long long target = static_cast<unsigned long long>(u * static_cast<double>(all));
        if (target >= all) target = all - 1;
        for (int w = 0; w < warp; ++w) before += sh.warp_mass[w];
        if (target >= before && target < before + sum) {   // this warp's run holds the token
            unsigned long long run_m = before;
            walk([&](uint32_t id, unsigned long long w, bool) {
                unsigned long long p = w;
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long up = __shfl_up_sync(0xffffffffu, p, o);
                    if (lane >= o) p += up;
                }
                const uint32_t vote = __ballot_sync(0xffffffffu, run_m + p > target);
                if (vote) {
                    if (lane == __ffs(vote) - 1) {
                        a.token[row] = id;
                        if (a.kept) a.kept[row] = kept;
                        if (a.logprob) {
                            const double d = static_cast<double>(as_logit(__ldg(src + id))) - static_cast<double>(top);
                            a.logprob[row] = static_cast<float>(d - log(static_cast<double>(whole) / unit));
                        }
                    }
                    return true;
                }
                run_m += __shfl_sync(0xffffffffu, p, 31);
                return false;
            });
        }
    } else if (rank == 0 && threadIdx.x == 0) {
        a.token[row] = token;
        if (a.kept) a.kept[row] = kept;
        if (a.logprob) a.logprob[row] = static_cast<float>(-log(static_cast<double>(whole) / unit));
    }
    cluster.sync();   // no CTA leaves while another may read its shared memory
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
    const uint32_t per = (vocab + kCluster - 1) / kCluster;
    a.slice = (per + 1023) / 1024 * 1024;
    int bits = 0;
    while ((1u << bits) < vocab) ++bits;
    a.shift = 62 - bits;
    a.resident = a.slice <= kSmemIds;
    a.vec = aligned(logits, 16) && (n == 1 || row_stride % 4 == 0);
    const size_t smem = a.resident ? a.slice * sizeof(float) : 0;
    const cudaError_t set = cudaFuncSetAttribute(smp_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemIds * sizeof(float));
    if (set != cudaSuccess) return set_cuda_error(fn, set);
    smp_rows<<<n * kCluster, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(a, r);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    clear_error();
    return GTM_OK;
}
