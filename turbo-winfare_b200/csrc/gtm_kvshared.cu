// The shared prefix of a step's rows (include/gtmoe_attention.h), computed once for all of them on
// the tcgen05 tensor cores.
//
// A unit is a kv head and 64 query rows (row, query head of the group). Per tile of 128 ring rows:
//   S^T [128 positions x 64 rows] = K q^T: K's codes become fp16 in tensor memory (operand A, a
//     position per lane), q's high and low limbs wait in shared memory (operand B);
//   softmax weights, a position per thread: p = exp2(s2 - m) * vs, its limbs into shared memory;
//   O^T [dims x 64 rows] += V^T p: V's codes become fp16 in shared memory (operand A, dims
//     contiguous), p is operand B. O stays in tensor memory.
// Rows on the N side make a unit of any number of rows cost what its 64 columns cost, and a
// position per lane lets a thread apply its own scales. m only moves when a score passes it by 8 (a
// factor of 256 that fp16 has room for): a tile mostly takes one vote, and neither the maxima over its
// positions (across lanes) nor a rescaled O. Tiles follow ring slots, not positions: softmax does not mind the
// order, no tile wraps, and each row's span is a mask on the slot's position.
//
// A tensor core's addition to its accumulator is cut to fp32, not rounded, which biases a long sum by
// up to 2^-24 of it per instruction. So a score's limbs are summed apart (HD / 16 instructions each),
// and O goes to memory after kLongest tiles (16 instructions each), where results are added in fp32.
//
// S and O are issued by two warps, so that neither waits behind the other's barriers: while the
// softmax works on tile i + 1, O of tile i and S of tile i + 2 are formed side by side, and K and V
// are converted at an even pace. O takes a tile's positions in two halves, so that one half of p is
// written while the other is read.
//
// The work is the flat list of (kv head, unit, tile), cut into equal runs, one per CTA; a CTA leaves a
// partial result for each unit it touches.
//
// The tensor pipe is the floor: a 128 x 128 x 16 instruction takes ~62 cycles whatever of its 128 columns
// is used, so two limbs of 64 rows cost (HD / 16) x 62 for S and, where the limbs do not fit side by side
// (512 dims), twice that for O: ~6,000 cycles a tile of 512 dims. A tile takes ~10,000: the hand-overs of
// K, V, S and p each add a wait, and no role is busy throughout (without any one of conversions, softmax or
// half the products it took 5 to 20% less). 512 rows (16 / 2 heads of 512) over 32,768 positions: 1.49-1.52 ms;
// 32 rows over 16,384: 72 us; 61 windowed rows (8 heads of 256): 20 us.
// kLongest, that prompt's time and error against 64 bits: 8 tiles 1.74 ms and 3.6e-6, 12 1.63 and 4.4e-6 (as the
// plain fp32 form), 16 1.55 and 5.3e-6, 20 1.52 and 6.2e-6. 20 is taken: still within fp32 sums of that length. Runs
// of up to 20 tiles (32 rows over 16,384 positions: 3.4e-6 against the plain form's 3.7e-6) do not notice.
//
// Roles: warps 0-7 softmax and O (32 of the 64 columns each half of them); 8-11 K; 12-15 V; 16 issues
// S, 17 O; 18 and 19 load the codes of K and V. Every wait is bounded (1 s); one that runs out stops the
// CTA, marks its results NaN and is recorded in the workspace's error word.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "gtm_frag.cuh"
#include "gtm_kvattn.cuh"
#include "gtm_tcgen05.cuh"

namespace gtm {
namespace {

constexpr int N = kSharedRows;
constexpr int TP = 128;              // positions of a tile
constexpr int kThreads = 640;
constexpr uint64_t kWaitNs = 1000000000ull, kTestWaitNs = 2000000ull;
constexpr int KA = 4;                // K chunks (64 dims) in tensor memory
// log2 of how far a weight may grow before m moves. Smaller would hold small weights better and move m more often:
// 512 rows over 32,768 positions 1.51 ms with 8, 1.53 with 6, 1.59 with 4; 32 rows over 16,384 72, 74 and 76 us.
constexpr float kSlack = 8.0f;
constexpr uint32_t kLongest = 20;    // tiles summed in tensor memory before the result goes to memory

template <int HD>
struct Shape {
    static constexpr int kChunks = HD / 64;      // K chunks of a tile
    static constexpr int kVStages = HD / 64;     // V stages of a tile: 128 dims x 64 positions
    static constexpr int RK = HD == 512 ? 2 : 4, RV = HD == 512 ? 2 : 4, VST = HD == 512 ? 2 : 4;
    static constexpr int kQ = 2 * kChunks * 8192, kP = 2 * 16384, kV = VST * 16384, kRawK = RK * 8192, kRawV = RV * 8192;
    static constexpr int kBars = 2 * RK + 2 * RV + 2 * KA + 2 * VST + 2 + 4 + 1;
    static constexpr int kSmall = (4 * N + 4 * N + 2 * N) * 4 + kBars * 8 + 16;
    static constexpr int kSmem = kQ + kP + kV + kRawK + kRawV + kSmall;
    // tensor memory columns. An MMA of N <= 128 takes the time of N = 128, so a limb pair goes in one
    // where there is room for two results: always for S, for O up to 256 dims.
    static constexpr bool kPairO = HD <= 256;
    static constexpr uint32_t kOWidth = kPairO ? 2 * N : N;
    static constexpr uint32_t kOCol = 0, kSCol = HD / 128 * kOWidth, kACol = kSCol + 2 * N;
    static_assert(kACol + KA * 32 <= 512, "tensor memory");
    static_assert(kSmem <= 232448, "shared memory");
};

struct SharedArgs {
    CUtensorMap k_map, v_map;      // the prefix's codes [capacity][kv_heads * head_dim]
    const float *ks, *vs;          // [kv_heads][capacity]
    const float* q;
    uint32_t q_heads, kv_heads, n, grp, capacity, ring_tiles, window, prefix_len, total;
    uint32_t lo[kMaxUnitsPerHead], first[kMaxUnitsPerHead], tiles[kMaxUnitsPerHead];   // a unit's first position, its ring tile, and its tiles
    SharedPlan plan;
    int* err;
    int test_wait;   // warp 16's first wait is for an arrival that never comes, under kTestWaitNs
};

// Whether any of a softmax group's 128 threads says so (hardware barrier 1 or 2).
__device__ __forceinline__ bool any_of_128(uint32_t bar, bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(x ? 1u : 0u), "r"(bar) : "memory");
    return r != 0;
}
// One arrival for the warp: 32 lanes' arrivals on one barrier are taken one by one.
__device__ __forceinline__ void arrive_warp(uint64_t* a, uint64_t* b = nullptr) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
        tc::mbar_arrive(a);
        if (b) tc::mbar_arrive(b);
    }
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                    "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
// Operand whose M or N side is contiguous: rows (K) of 64 fp16, 8-row atoms of 1,024 bytes in the
// 128-byte swizzle; `block` bytes to the next 64 of M or N.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t addr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)((block >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

// 16 codes to 8 + 8 fp16
template <int FMT>
__device__ __forceinline__ void widen(const uint4& w, uint32_t (&o)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t b = bias_codes<FMT>(x[i]);
        o[2 * i] = pair_in_word<FMT, 0>(b);
        o[2 * i + 1] = pair_in_word<FMT, 1>(b);
    }
}

struct Segment {
    uint32_t kvh, unit, tile, tiles, slot;
    uint32_t left;   // places of the list until the next one
};
__device__ __forceinline__ Segment segment_at(const SharedArgs& a, uint32_t g, uint32_t end) {
    Segment s;
    const uint32_t per_head = a.plan.start[a.plan.units];
    s.kvh = g / per_head;
    const uint32_t r = g - s.kvh * per_head;
    uint32_t u = 0;
    for (uint32_t step = kMaxUnitsPerHead / 2; step; step >>= 1)
        if (u + step < a.plan.units && a.plan.start[u + step] <= r) u += step;
    s.unit = u;
    s.tile = r - a.plan.start[u];
    s.left = min(a.plan.start[u + 1] - r, end - g);
    s.tiles = min(min(s.left, a.tiles[u] - s.tile), kLongest);
    if (s.tile + s.tiles < a.tiles[u]) s.left = s.tiles;   // else what fills up the unit's last run goes, too
    s.slot = blockIdx.x + s.kvh * a.plan.units + u;
    return s;
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kThreads, 1)
    kv_shared(const __grid_constant__ SharedArgs a, const __grid_constant__ RowU32 pos) {
    using S = Shape<HD>;
    constexpr int RK = S::RK, RV = S::RV, VST = S::VST, C = S::kChunks, MT = HD / 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;                    // [chunk][limb][64 rows][128 B]
    uint8_t* sP = sQ + S::kQ;              // [limb][128 positions][128 B]
    uint8_t* sV = sP + S::kP;              // [stage][dims 0-63, 64-127][64 positions][128 B]
    uint8_t* sRawK = sV + S::kV;           // [stage][128 positions][64 B], 64-byte swizzle
    uint8_t* sRawV = sRawK + S::kRawK;     // [stage][64 positions][128 B], 128-byte swizzle
    float* wtop = reinterpret_cast<float*>(sRawV + S::kRawV);   // [4 warps][64]
    float* m_s = wtop + 4 * N;             // running maxima
    float* f_s = m_s + N;                  // factors of a rescale
    float* qf_s = f_s + N;                 // q's power of two and log2(e)
    float* g_s = qf_s + N;                 // a second factor, when results merge
    uint32_t* rlo = reinterpret_cast<uint32_t*>(g_s + N);   // rows' spans, from the unit's first position
    uint32_t* rhi = rlo + N;
    uint64_t* bars = reinterpret_cast<uint64_t*>(rhi + N);
    uint64_t *rk_full = bars, *rk_empty = rk_full + RK, *rv_full = rk_empty + RK, *rv_empty = rv_full + RV,
             *ka_full = rv_empty + RV, *ka_empty = ka_full + KA, *v_full = ka_empty + KA, *v_empty = v_full + VST,
             *s_full = v_empty + VST, *s_empty = s_full + 1, *p_full = s_empty + 1, *p_empty = p_full + 2;
    uint64_t* never_bar = p_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(never_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < RK; ++i) tc::mbar_init(&rk_full[i], 1), tc::mbar_init(&rk_empty[i], 4);
        for (int i = 0; i < RV; ++i) tc::mbar_init(&rv_full[i], 1), tc::mbar_init(&rv_empty[i], 4);
        for (int i = 0; i < KA; ++i) tc::mbar_init(&ka_full[i], 4), tc::mbar_init(&ka_empty[i], 1);
        for (int i = 0; i < VST; ++i) tc::mbar_init(&v_full[i], 4), tc::mbar_init(&v_empty[i], 1);
        tc::mbar_init(s_full, 1), tc::mbar_init(s_empty, 8);
        for (int i = 0; i < 2; ++i) tc::mbar_init(&p_full[i], 4), tc::mbar_init(&p_empty[i], 1);   // a half of the positions
        tc::mbar_init(never_bar, 1);
        *abort_flag = (tc::smem_u32(smem) & 1023u) ? 1 : 0;   // the swizzled layouts need it
        tc::mbar_fence_init();
    }
    if (warp == 17) tc::tmem_alloc(tmem_slot, 512);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = __reduce_or_sync(0xffffffffu, *tmem_slot);   // in a uniform register, as MMA operands are

    const uint32_t g0 = min(a.total, blockIdx.x * a.plan.per), g1 = min(a.total, g0 + a.plan.per);
    // K chunks (as many V stages) and tiles so far, the same for every role; the slot that already holds
    // this CTA's result
    uint32_t kc = 0, ti = 0, done_slot = 0xFFFFFFFFu;
    // Brings a segment's q into shared memory; false once the CTA has given up.
    auto begin = [&](const Segment& sg) -> bool {
        if (__syncthreads_or(*abort_flag)) {
            if (tid < N) a.plan.ml[static_cast<size_t>(sg.slot) * N + tid] = make_float2(0.0f, __int_as_float(0x7FC00000));
            return false;
        }
        if (sg.slot == done_slot) return true;   // the same unit goes on: its q, spans and maxima stay
        // ---- q's limbs and the rows' spans
        for (int r = warp; r < N; r += kThreads / 32) {
            const uint32_t qr = sg.unit * N + r, row = qr / a.grp, h = qr - row * a.grp;
            const bool live = row < a.n;
            const float* src = a.q + (static_cast<size_t>(row) * a.q_heads + sg.kvh * a.grp + h) * HD;
            float x[HD / 32], top = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 128; ++i) {
                const float4 v = live ? __ldg(reinterpret_cast<const float4*>(src) + lane + 32 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) top = fmaxf(top, fabsf(x[i]));
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = query_exponent(top);
            const float down = query_down(e);
#pragma unroll
            for (int i = 0; i < HD / 128; ++i) {
                const int d = 4 * lane + 128 * i;
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float u = x[4 * i + 2 * j] * down, v = x[4 * i + 2 * j + 1] * down;
                    hi[j] = cvt2(u, v);
                    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
                    lo[j] = cvt2(u - b.x, v - b.y);
                }
                const int c = d >> 6, unit16 = (d & 63) >> 3;
                const int off = c * 16384 + r * 128 + ((unit16 ^ (r & 7)) << 4) + (d & 4) * 2;
                *reinterpret_cast<uint2*>(sQ + off) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(sQ + 8192 + off) = make_uint2(lo[0], lo[1]);
            }
            if (lane == 0) {
                qf_s[r] = query_up(e) * kLog2e * (FMT == GTM_KV_E4M3 ? 256.0f : 1.0f);
                m_s[r] = -INFINITY;
                const Span sp = live ? row_span(pos.v[row], a.window, a.prefix_len) : Span{0, 0, 0, 0};
                // columns without a row are never read: they need no mask
                rlo[r] = !live ? 0u : sp.pn ? sp.pa - a.lo[sg.unit] : 1u;
                rhi[r] = !live ? 0xFFFFFFFFu : sp.pn ? sp.pa - a.lo[sg.unit] + sp.pn : 0u;
            }
        }
        tc::fence_proxy_async_smem();
        __syncthreads();
        return true;
    };
    auto ring_tile = [&](const Segment& sg, uint32_t t) {
        const uint32_t b = a.first[sg.unit] + sg.tile + t;
        return b >= a.ring_tiles ? b - a.ring_tiles : b;
    };
    // 640 threads x 96 registers at launch >= 256 x 128 + 384 x 72: the softmax keeps 32 scores and 32 sums
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        // ---- softmax: a position and 32 columns per thread
        constexpr int H = N / 2;
        const int p = tid & 127, grp = warp >> 2, half = p >> 6;
        const int col0 = grp * H;   // the group's columns
        const uint32_t bar = 1 + grp;
        const uint32_t lane_addr = (tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16)) + col0;
        float *tops = wtop + (warp & 3) * N + col0, *m_c = m_s + col0, *f_c = f_s + col0;
        const float* qf_c = qf_s + col0;
        const uint32_t *rlo_c = rlo + col0, *rhi_c = rhi + col0;
        for (uint32_t g = g0; g < g1;) {
            const Segment sg = segment_at(a, g, g1);
            g += sg.left;
            if (!begin(sg)) {
                done_slot = sg.slot;
                continue;
            }
            const uint32_t s0 = a.lo[sg.unit] % a.capacity;
            const float *ksp = a.ks + static_cast<size_t>(sg.kvh) * a.capacity, *vsp = a.vs + static_cast<size_t>(sg.kvh) * a.capacity;
            const uint32_t max_lo = __reduce_max_sync(0xffffffffu, rlo_c[lane]);
            const uint32_t min_hi = __reduce_min_sync(0xffffffffu, rhi_c[lane]);
            float l[H];
#pragma unroll
            for (int i = 0; i < H; ++i) l[i] = 0.0f;
            uint32_t slot = ring_tile(sg, 0) * TP + p;
            float ks_next = slot < a.capacity ? __ldg(ksp + slot) : 1.0f, vs_next = slot < a.capacity ? __ldg(vsp + slot) : 1.0f;
            bool ok = true;
            for (uint32_t t = 0; t < sg.tiles; ++t) {
                const uint32_t x = ti + t;
                const float ks = ks_next, vs = vs_next, lg = log2_vs(vs) - (kWeightTop - kSlack);
                const bool in_ring = slot < a.capacity;
                const uint32_t at = slot - s0 + (slot < s0 ? a.capacity : 0u);   // from the unit's first position
                if (t + 1 < sg.tiles) {
                    slot = ring_tile(sg, t + 1) * TP + p;
                    ks_next = slot < a.capacity ? __ldg(ksp + slot) : 1.0f;
                    vs_next = slot < a.capacity ? __ldg(vsp + slot) : 1.0f;
                }
                const bool all_in = __all_sync(0xffffffffu, in_ring && at >= max_lo && at < min_hi);
                ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(s_full, x & 1, abort_flag, kWaitNs));
                // the group's warps meet in barriers below, so they leave together or not at all
                if (any_of_128(bar, !ok)) { ok = false; break; }
                tc::tc_fence_after();
                float s[H], over = -INFINITY;   // s2, -infinity where masked; whether a weight would pass the top
#pragma unroll
                for (int c0 = 0; c0 < H; c0 += 16) {
                    uint32_t v[16], w[16];
                    tc::tmem_ld16_sync(lane_addr + S::kSCol + c0, v);
                    tc::tmem_ld16_sync(lane_addr + S::kSCol + N + c0, w);
#pragma unroll
                    for (int c = 0; c < 16; ++c) s[c0 + c] = __uint_as_float(v[c]) + __uint_as_float(w[c]);
                }
                tc::tc_fence_before();
                arrive_warp(s_empty);   // the next tile's S may be formed
#pragma unroll
                for (int c = 0; c < H; c += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(qf_c + c);
                    s[c] *= ks * f.x, s[c + 1] *= ks * f.y, s[c + 2] *= ks * f.z, s[c + 3] *= ks * f.w;
                }
                if (!all_in) {
#pragma unroll
                    for (int c = 0; c < H; ++c) s[c] = in_ring && at >= rlo_c[c] && at < rhi_c[c] ? s[c] : -INFINITY;
                }
#pragma unroll
                for (int c = 0; c < H; c += 4) {   // (-infinity) - (-infinity) is NaN, which fmaxf passes over
                    const float4 m4 = *reinterpret_cast<const float4*>(m_c + c);
                    over = fmaxf(over, fmaxf(fmaxf(s[c] - m4.x, s[c + 1] - m4.y), fmaxf(s[c + 2] - m4.z, s[c + 3] - m4.w)));
                }
                const bool raise = any_of_128(bar, over + lg > kSlack);
                if (raise) {
                    // new maxima: 15 exchanges and one more leave a column's maximum over the warp's positions
                    // with two lanes
                    for (int c0 = 0; c0 < H; c0 += 16) {
                        float y[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) y[c] = (c0 ? s[c + 16] : s[c]) + lg;
#pragma unroll
                        for (int w = 8; w > 0; w >>= 1)
#pragma unroll
                            for (int c = 0; c < w; ++c) {
                                const float keep = (lane & w) ? y[c + w] : y[c], send = (lane & w) ? y[c] : y[c + w];
                                y[c] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, w));
                            }
                        y[0] = fmaxf(y[0], __shfl_xor_sync(0xffffffffu, y[0], 16));
                        if (lane < 16) tops[c0 + lane] = y[0];
                    }
                    tc::named_bar_sync(bar, 128);
                    if (p < H) {
                        const float* w = wtop + col0 + p;
                        const float old = m_c[p], now = fmaxf(fmaxf(fmaxf(w[0], w[N]), fmaxf(w[2 * N], w[3 * N])), old);
                        f_c[p] = old == now ? 1.0f : ex2(old - now);
                        m_c[p] = now;
                    }
                    tc::named_bar_sync(bar, 128);
#pragma unroll
                    for (int i = 0; i < H; ++i) l[i] *= f_c[i];
                    if (t > 0) {
                        ok = __all_sync(0xffffffffu, tc::mbar_wait(&p_empty[1], (x & 1) ^ 1, abort_flag, kWaitNs));
                        tc::tc_fence_after();
                        for (int c0 = 0; c0 < static_cast<int>(S::kSCol / N) * 2; ++c0) {
                            uint32_t v[16];
                            const uint32_t addr = lane_addr + S::kOCol + (c0 >> 1) * N + (c0 & 1) * 16;
                            tc::tmem_ld16_sync(addr, v);
#pragma unroll
                            for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * f_c[(c0 & 1) * 16 + c]);
                            tmem_st16(addr, v);
                        }
                        tc::tmem_st_wait();
                        tc::tc_fence_before();
                        // Each warp has rescaled its own 32 of O's 128 lanes, but p_full[0], which lets a product
                        // into all of them, is the arrival of two of the group's warps only: none goes on before
                        // all four are done.
                        tc::named_bar_sync(bar, 128);
                    }
                }
                ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&p_empty[half], (x & 1) ^ 1, abort_flag, kWaitNs));
                uint8_t* prow = sP + p * 128;
#pragma unroll
                for (int c0 = 0; c0 < H; c0 += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        const float2 m2 = *reinterpret_cast<const float2*>(m_c + c0 + c);
                        float e[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {   // 0 where masked, whatever m and vs are; a NaN goes through
                            const bool out = s[c0 + c + j] == -INFINITY;
                            e[j] = out ? 0.0f : ex2(s[c0 + c + j] - (j ? m2.y : m2.x));
                            l[c0 + c + j] += e[j];
                            e[j] = out ? 0.0f : e[j] * vs;
                        }
                        hi[c >> 1] = cvt2(e[0], e[1]);
                        const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&hi[c >> 1]));
                        lo[c >> 1] = cvt2(e[0] - w.x, e[1] - w.y);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int off = (((col0 + c0) / 8 + u) ^ (p & 7)) << 4;
                        *reinterpret_cast<uint4*>(prow + off) = make_uint4(hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
                        *reinterpret_cast<uint4*>(prow + 16384 + off) = make_uint4(lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
                    }
                }
                tc::fence_proxy_async_smem();
                arrive_warp(&p_full[half]);
            }
            const uint32_t last = ti + sg.tiles - 1;
            ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&p_empty[1], last & 1, abort_flag, kWaitNs));
            ok = !any_of_128(bar, !ok);
            // ---- the segment's result, merged into what this CTA left in the slot before
            float2* ml = a.plan.ml + static_cast<size_t>(sg.slot) * N + col0;
            float* part = a.plan.part + (static_cast<size_t>(sg.slot) * N + col0) * HD;
            const bool merge = sg.slot == done_slot;
            if (ok) {
                tc::tc_fence_after();
#pragma unroll
                for (int i = 0; i < H; ++i) {
                    float sum = l[i];
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == i) tops[i] = sum;
                }
                tc::named_bar_sync(bar, 128);
                if (p < H) {
                    const float* w = wtop + col0 + p;
                    float sum = (w[0] + w[N]) + (w[2 * N] + w[3 * N]), m = m_c[p], f = 1.0f, gold = 0.0f;
                    if (merge) {
                        const float2 old = ml[p];
                        const float now = fmaxf(m, old.x);
                        f = m == now ? 1.0f : ex2(m - now);
                        gold = old.x == now ? 1.0f : ex2(old.x - now);
                        sum = sum * f + old.y * gold;
                        m = now;
                    }
                    ml[p] = make_float2(m, sum);
                    f_c[p] = f * (FMT == GTM_KV_E4M3 ? 256.0f : 1.0f);
                    g_s[col0 + p] = gold;
                }
                // scales as they were (mostly): what is there only has to be added to, which needs no answer
                const bool rescale = any_of_128(bar, merge && p < H && g_s[col0 + p] != 1.0f);
                for (int c0 = 0; c0 < MT * 2; ++c0) {
                    uint32_t v[16];
                    const int r0 = (c0 & 1) * 16;
                    tc::tmem_ld16_sync(lane_addr + S::kOCol + (c0 >> 1) * S::kOWidth + r0, v);
                    if (S::kPairO) {
                        uint32_t w[16];
                        tc::tmem_ld16_sync(lane_addr + S::kOCol + (c0 >> 1) * S::kOWidth + N + r0, w);
#pragma unroll
                        for (int c = 0; c < 16; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) + __uint_as_float(w[c]));
                    }
                    float* dst = part + static_cast<size_t>(r0) * HD + (c0 >> 1) * 128 + p;
                    float old[16];
                    if (rescale) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) old[c] = dst[c * HD];
                    }
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const float o = __uint_as_float(v[c]) * f_c[r0 + c];
                        if (merge && !rescale)
                            asm volatile("red.global.add.f32 [%0], %1;" :: "l"(dst + c * HD), "f"(o) : "memory");
                        else
                            dst[c * HD] = rescale ? fmaf(old[c], g_s[col0 + r0 + c], o) : o;
                    }
                }
                tc::tc_fence_before();
            } else if (p < H) {
                ml[p] = make_float2(0.0f, __int_as_float(0x7FC00000));
            }
            ti += sg.tiles;
            done_slot = sg.slot;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    for (uint32_t g = g0; g < g1;) {
        const Segment sg = segment_at(a, g, g1);
        g += sg.left;
        const bool good = begin(sg);
        done_slot = sg.slot;
        if (!good) continue;
        const uint32_t vc = kc;
        if (warp >= 8 && warp < 12) {   // ---- K: codes to fp16 in tensor memory, a position per lane
            const int p = 32 * (warp & 3) + lane;
            const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + S::kACol;
            uint32_t it = kc;
            const uint32_t end = kc + sg.tiles * C;
            for (; it < end; ++it) {
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&rk_full[it % RK], (it / RK) & 1, abort_flag, kWaitNs))) break;
                const uint8_t* raw = sRawK + (it % RK) * 8192 + p * 64;
                uint32_t o[32];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 w = *reinterpret_cast<const uint4*>(raw + ((j ^ ((p >> 1) & 3)) << 4));
                    uint32_t h[8];
                    widen<FMT>(w, h);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[8 * j + i] = h[i];
                }
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&ka_empty[it % KA], ((it / KA) & 1) ^ 1, abort_flag, kWaitNs))) break;
                tc::tc_fence_after();
                tc::tmem_st32(lane_addr + (it % KA) * 32, o);
                tc::tmem_st_wait();
                tc::tc_fence_before();
                arrive_warp(&ka_full[it % KA], &rk_empty[it % RK]);   // the raw slot only after its words were used
            }
        } else if (warp >= 12 && warp < 16) {   // ---- V: codes to fp16 in shared memory, dims contiguous
            const int p = (tid - 384) & 63, half = (tid - 384) >> 6;
            uint32_t it = vc;
            const uint32_t end = vc + sg.tiles * S::kVStages;
            for (; it < end; ++it) {
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&rv_full[it % RV], (it / RV) & 1, abort_flag, kWaitNs))) break;
                const uint8_t* raw = sRawV + (it % RV) * 8192 + p * 128;
                uint32_t h[4][8];   // converted while the stage is still being multiplied
#pragma unroll
                for (int j = 0; j < 4; ++j) widen<FMT>(*reinterpret_cast<const uint4*>(raw + (((half * 4 + j) ^ (p & 7)) << 4)), h[j]);
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&v_empty[it % VST], ((it / VST) & 1) ^ 1, abort_flag, kWaitNs))) break;
                uint8_t* dst = sV + (it % VST) * 16384 + half * 8192 + p * 128;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    *reinterpret_cast<uint4*>(dst + (((2 * j) ^ (p & 7)) << 4)) = make_uint4(h[j][0], h[j][1], h[j][2], h[j][3]);
                    *reinterpret_cast<uint4*>(dst + (((2 * j + 1) ^ (p & 7)) << 4)) = make_uint4(h[j][4], h[j][5], h[j][6], h[j][7]);
                }
                tc::fence_proxy_async_smem();
                arrive_warp(&v_full[it % VST], &rv_empty[it % RV]);
            }
        } else if (warp == 18 || warp == 19) {   // ---- codes of K and of V
            if (lane == 0) {
                const bool is_v = warp == 19;
                const uint32_t R = is_v ? RV : RK, first = is_v ? vc : kc, end = first + sg.tiles * C;
                uint64_t *full = is_v ? rv_full : rk_full, *empty = is_v ? rv_empty : rk_empty;
                uint8_t* dst = is_v ? sRawV : sRawK;
                uint32_t it = first;
                for (; it < end; ++it) {
                    const uint32_t c = (it - first) % C;
                    const int y = static_cast<int>(ring_tile(sg, (it - first) / C) * TP), x = static_cast<int>(sg.kvh * HD);
                    if (!tc::mbar_wait(&empty[it % R], ((it / R) & 1) ^ 1, abort_flag, kWaitNs)) break;
                    tc::mbar_arrive_expect_tx(&full[it % R], 8192);
                    if (is_v)
                        tc::tma_load_2d(dst + (it % R) * 8192, &a.v_map, x + static_cast<int>(c % MT * 128), y + static_cast<int>(c / MT * 64), &full[it % R]);
                    else
                        tc::tma_load_2d(dst + (it % R) * 8192, &a.k_map, x + static_cast<int>(c * 64), y, &full[it % R]);
                }
                if (*abort_flag) {   // no exit while copies into this CTA's shared memory are in flight
                    volatile int never = 0;
                    for (uint32_t j = it > R ? it - R : 0; j < it; ++j) tc::mbar_wait(&full[j % R], (j / R) & 1, &never, kWaitNs);
                }
            }
        } else if (warp == 16) {   // ---- S: the whole warp, one elected lane issues
            constexpr uint32_t kQk = tc::idesc_f16(128, 2 * N);
            const uint32_t qa = tc::smem_u32(sQ), d = tmem + S::kSCol;
            uint32_t ik = kc;
            bool ok = !a.test_wait || kc || __all_sync(0xffffffffu, tc::mbar_wait(never_bar, 0, abort_flag, kTestWaitNs));
            for (uint32_t t = 0; t < sg.tiles && ok; ++t) {
                if (!__all_sync(0xffffffffu, tc::mbar_wait(s_empty, ((ti + t) & 1) ^ 1, abort_flag, kWaitNs))) break;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&ka_full[ik % KA], (ik / KA) & 1, abort_flag, kWaitNs));
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t ka = tmem + S::kACol + (ik % KA) * 32;
                    const uint64_t qd = tc::sdesc_sw128(qa + c * 16384);   // 64 high rows, then 64 low rows
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_f16_ts(d, ka + 8 * k, qd + 2 * k, kQk, (c > 0 || k > 0) ? 1u : 0u);
                    tc::mma_commit(&ka_empty[ik % KA]);
                    ++ik;
                }
                if (ok) tc::mma_commit(s_full);
            }
            if (*abort_flag && ik > 0) {   // issued MMAs end before tensor memory is released
                volatile int never = 0;
                tc::mbar_wait(&ka_empty[(ik - 1) % KA], ((ik - 1) / KA) & 1, &never, kWaitNs);
            }
        } else if (warp == 17) {   // ---- O, likewise
            constexpr uint32_t kPv = tc::idesc_f16(128, S::kOWidth) | (1u << 15) | (1u << 16);   // both operands M/N-contiguous
            const uint32_t va = tc::smem_u32(sV), pa = tc::smem_u32(sP);
            uint32_t iv = vc;
            bool ok = true;
            for (uint32_t t = 0; t < sg.tiles && ok; ++t) {
#pragma unroll
                for (int c = 0; c < C; ++c) {   // 128 dims c % MT, positions' half c / MT
                    const int half = c / MT, mt = c % MT;
                    if (mt == 0) ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&p_full[half], (ti + t) & 1, abort_flag, kWaitNs));
                    ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&v_full[iv % VST], (iv / VST) & 1, abort_flag, kWaitNs));
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t d = tmem + S::kOCol + mt * S::kOWidth;
                    const uint64_t vd = sdesc_mn(va + (iv % VST) * 16384, 8192), pd = sdesc_mn(pa + half * 64 * 128, 16384);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {   // 16 positions: 2,048 bytes
                        tc::mma_f16(d, vd + 128 * k, pd + 128 * k, kPv, (t > 0 || half || k > 0) ? 1u : 0u);
                        if (!S::kPairO) tc::mma_f16(d, vd + 128 * k, pd + (16384 >> 4) + 128 * k, kPv, 1u);
                    }
                    tc::mma_commit(&v_empty[iv % VST]);
                    ++iv;
                    if (mt == MT - 1) tc::mma_commit(&p_empty[half]);
                }
            }
            if (*abort_flag && iv > 0) {
                volatile int never = 0;
                tc::mbar_wait(&v_empty[(iv - 1) % VST], ((iv - 1) / VST) & 1, &never, kWaitNs);
            }
        }
        kc += sg.tiles * C;
        ti += sg.tiles;
    }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_flag) atomicExch(a.err, 2);
    if (warp == 17) {
        tc::tmem_relinquish();
        tc::tmem_dealloc(tmem, 512);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int map_codes(CUtensorMap* m, const void* codes, uint64_t width, uint64_t rows, uint32_t box_w, uint32_t box_rows,
              CUtensorMapSwizzle swizzle) {
    static std::atomic<EncodeTiledFn> found{nullptr};   // two threads' first calls may look it up at once
    EncodeTiledFn encode = found.load(std::memory_order_relaxed);
    if (!encode) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return set_error(GTM_ERR_CUDA, "cuTensorMapEncodeTiled not available");
        encode = reinterpret_cast<EncodeTiledFn>(f);
        found.store(encode, std::memory_order_relaxed);
    }
    const cuuint64_t dims[2] = {width, rows}, strides[1] = {width};
    const cuuint32_t box[2] = {box_w, box_rows}, estr[2] = {1, 1};
    const CUresult r = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(GTM_ERR_CUDA, "cuTensorMapEncodeTiled (prefix codes) failed (%d)", (int)r);
    return GTM_OK;
}

// A unit's first attended position, its ring tile, and its number of tiles.
struct UnitSpan {
    uint32_t lo, first, tiles;
};
UnitSpan unit_span(const SharedCall& c, const RowU32& pos, uint32_t unit) {
    const uint32_t grp = c.q_heads / c.kv_heads, cap = c.prefix->capacity;
    const uint32_t r0 = unit * N / grp, r1 = std::min(c.n, (unit * N + N + grp - 1) / grp);
    uint32_t lo = 0xFFFFFFFFu, hi = 0;
    for (uint32_t i = r0; i < r1; ++i) {
        const Span s = row_span(pos.v[i], c.window, c.prefix_len);
        if (s.pn) lo = std::min(lo, s.pa), hi = std::max(hi, s.pa + s.pn);
    }
    if (hi == 0) return {0, 0, 0};
    const uint32_t ring = (cap + TP - 1) / TP, s0 = lo % cap, len = hi - lo;   // len <= capacity
    const uint64_t end = static_cast<uint64_t>(s0) + len;
    uint64_t tiles;
    if (end <= cap)
        tiles = (end - 1) / TP - s0 / TP + 1;
    else   // wrapped: to the ring's end, then from its start, no tile twice
        tiles = std::min<uint64_t>(ring, (ring - s0 / TP) + (end - cap - 1) / TP + 1);
    return {lo, s0 / TP, static_cast<uint32_t>(tiles)};
}

template <int HD>
int launch(const SharedArgs& a, const RowU32& pos, uint32_t fmt, uint32_t ctas, cudaStream_t st) {
    const auto kernel = fmt == GTM_KV_INT8 ? kv_shared<HD, GTM_KV_INT8> : kv_shared<HD, GTM_KV_E4M3>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<HD>::kSmem);
    if (e != cudaSuccess) return set_cuda_error("gtm_attention_kv_rows", e);
    kernel<<<ctas, kThreads, Shape<HD>::kSmem, st>>>(a, pos);
    return GTM_OK;
}

}  // namespace

size_t shared_slots(uint32_t q_heads, uint32_t kv_heads, uint32_t n, int num_sms) {
    const uint64_t units = (static_cast<uint64_t>(n) * (q_heads / kv_heads) + N - 1) / N * kv_heads;
    return units + num_sms;
}

// The list of tiles is cut into runs of `per`, one for each CTA. A run that touches two units pays for it: q, the
// first tile's way through every role, the drain and the result, ~20 us together at 512 dims, as much as three or
// four tiles. So each unit's tiles are filled up to whole runs where that makes runs at most three tiles longer
// (32 rows over 16,384 positions, 2 heads of 512: 7 tiles a run and 88 us, or 8 and 71).
void plan_shared(const SharedCall& c, const RowU32& pos, int num_sms, SharedPlan& plan) {
    plan.units = (c.n * (c.q_heads / c.kv_heads) + N - 1) / N;
    uint32_t tiles[kMaxUnitsPerHead];
    uint64_t total = 0;
    for (uint32_t u = 0; u < plan.units; ++u) total += tiles[u] = unit_span(c, pos, u).tiles;
    total *= c.kv_heads;
    const uint32_t flat = static_cast<uint32_t>(std::max<uint64_t>(1, (total + num_sms - 1) / num_sms));
    uint32_t fill = 1;
    plan.per = flat;
    for (uint32_t per = flat; per <= flat + 3; ++per) {
        uint64_t runs = 0;
        for (uint32_t u = 0; u < plan.units; ++u) runs += (tiles[u] + per - 1) / per;
        if (runs * c.kv_heads <= static_cast<uint64_t>(num_sms)) {
            plan.per = fill = per;
            break;
        }
    }
    plan.start[0] = 0;
    for (uint32_t u = 0; u < plan.units; ++u) plan.start[u + 1] = plan.start[u] + (tiles[u] + fill - 1) / fill * fill;
}

int launch_shared(const SharedCall& c, const RowU32& pos, const SharedPlan& plan, int num_sms, cudaStream_t st) {
    SharedArgs a;
    const GtmKvCache* p = c.prefix;
    const uint64_t width = static_cast<uint64_t>(c.kv_heads) * c.head_dim;
    const size_t vec = static_cast<size_t>(c.prefix_seq) * p->capacity * c.kv_heads;
    int rc = map_codes(&a.k_map, static_cast<const uint8_t*>(p->k_dev) + vec * c.head_dim, width, p->capacity, 64, TP,
                       CU_TENSOR_MAP_SWIZZLE_64B);
    if (!rc) rc = map_codes(&a.v_map, static_cast<const uint8_t*>(p->v_dev) + vec * c.head_dim, width, p->capacity, 128, 64,
                            CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    a.ks = p->k_scale_dev + vec, a.vs = p->v_scale_dev + vec;
    a.q = c.q;
    a.q_heads = c.q_heads, a.kv_heads = c.kv_heads, a.n = c.n, a.grp = c.q_heads / c.kv_heads;
    a.capacity = p->capacity, a.ring_tiles = (p->capacity + TP - 1) / TP;
    a.window = c.window, a.prefix_len = c.prefix_len;
    a.total = plan.start[plan.units] * c.kv_heads;
    for (uint32_t u = 0; u < plan.units; ++u) {
        const UnitSpan s = unit_span(c, pos, u);
        a.lo[u] = s.lo, a.first[u] = s.first, a.tiles[u] = s.tiles;
    }
    a.plan = plan;
    a.err = c.err, a.test_wait = c.test_wait ? 1 : 0;
    const uint32_t ctas = (a.total + plan.per - 1) / plan.per;
    if (c.head_dim == 128) return launch<128>(a, pos, p->format, ctas, st);
    if (c.head_dim == 256) return launch<256>(a, pos, p->format, ctas, st);
    return launch<512>(a, pos, p->format, ctas, st);
}

}  // namespace gtm
