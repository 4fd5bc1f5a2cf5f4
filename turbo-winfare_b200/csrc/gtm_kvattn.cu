// Attention over the one-byte KV caches (include/gtmoe_attention.h).
//
// softmax(q K^T) V with K = codes * ks and V = codes * vs, one scale per position. Codes are exact
// in fp16 (int8 directly, e4m3 with its exponent bias moved: the value times 2^-8), so the tensor
// cores multiply them as they are and only the other operand is split: q and the weights p are
// carried as an fp16 high and low part (22 bits), two products each, accumulated in fp32. The
// scales stay outside: a score is multiplied by its position's ks, a weight by its vs.
//
// Running softmax in base 2 per query head: with s2 = log2(e) * q.k the stabiliser is m >= max(s2 +
// log2 vs) - 15.9, so a carried weight p = exp2(s2 - m) * vs fits fp16 whatever the scales are
// (its limbs are off by up to 2^-40.9 of the largest one), while l = sum of exp2(s2 - m) and the weighted sum O stay
// in fp32. Masked positions take a weight of exactly 0 by selection, so nothing that a ring row
// outside a row's span holds reaches a sum. A partial result (m, l, O) is merged by kv_combine.
//
// kv_rows: a CTA per (row, kv head, run of positions), for positions that one row attends.
// kv_shared (gtm_kvshared.cu): the prefix, for all rows at once.
#include <algorithm>
#include <cmath>

#include "gtm_frag.cuh"
#include "gtm_kvattn.cuh"

namespace gtm {
namespace {

// ---- rows over their own positions ----------------------------------------------------------------

struct RowsArgs {
    Side own, pre;
    const float* q;
    float* ctx;
    float* part;     // [item][kv_heads][group][head_dim]
    float2* ml;      // [item][kv_heads][group]: m (base 2), l
    uint32_t q_heads, kv_heads, n, window, prefix_len, chunk;
    bool list_prefix;   // prefix positions are in the rows' lists, not in kv_shared
};

// A row of one item with nothing elsewhere is written to ctx at once.
__device__ __forceinline__ bool is_whole(const RowsArgs& a, uint32_t items, const Span& sp) {
    return items == 1 && (a.list_prefix || sp.pn == 0);
}
struct Starts {
    uint32_t v[kMaxBatchRows + 1];   // first item of each row, then the number of items
};

template <int HD>
struct RowsShape {
    static constexpr int kWarps = HD == 512 ? 8 : 4;   // of each kind
    static constexpr int kTile = 16 * kWarps;
    static constexpr int kDims = HD / kWarps;   // V dims of a warp
    static constexpr int kD = kDims / 8;        // contiguous V codes of a thread: 8 or 4
    static constexpr int kChunks = HD / 64;
    static constexpr int kThreads = 2 * kWarps * 32;
};

// Barriers among part of the CTA's warps: a full wait, and an arrival that does not wait.
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" :: "r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" :: "r"(id), "r"(threads) : "memory"); }

// The second and third kernel of a call are set up while the one before ends (1.5 to 3 us less each), and start
// here, with all its results in sight. None is let in earlier: kv_combine's CTAs took room from kv_rows' last ones
// (32 own rows 105.5 -> 107.6 us), and kv_rows beside kv_shared gained on one shape (107.7 -> 101.4) and lost on
// another (93.2 -> 96.3).
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... Q>
cudaError_t launch_after(bool early, void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, const Q&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr, cfg.numAttrs = early ? 1 : 0;   // only behind a kernel of the same call
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A tile's two products are made by two kinds of warps, so that both run at once: the first half of the
// CTA scores 16 positions a warp (A = K: 16 positions x 16 dims; B = q: 16 dims x 8 heads), agrees on
// the heads' maxima and leaves the weights in one of two buffers; the second half adds all of the tile's
// positions to a warp's share of the dims (A = V^T: 16 dims x 16 positions; B = p). The order of dims and
// positions inside a product is free, so threads read contiguous codes: 16 of a K vector, kD of a V
// vector. Codes of the next tile are loaded into the registers that the products have just emptied.
//
// Bytes are the floor (a code is read once per row and kv head, for at most 8 heads' products), but the
// chain of a tile bounds it: load, widening and products, a barrier among the scorers, exponentials, the
// hand-over, the sums. 32 rows of 77-8,192 positions, 2 heads of 512 (275 MB): 84 us, 3.3 TB/s, with one CTA
// of 16 warps per SM; 61 windowed rows, 8 heads of 256, two of 8 warps: 55 us; one row of 1,024: 4.3. All warps
// scoring and then summing took 99 and 64 us (91 and 55 since, with the same runs); then neither leaving out the products nor codes that stay in L2
// made it faster.
template <int HD, int FMT>
__global__ void __launch_bounds__(RowsShape<HD>::kThreads, HD == 512 ? 1 : 2)
    kv_rows(const __grid_constant__ RowsArgs a, const __grid_constant__ Starts starts, const __grid_constant__ RowU32 pos,
            const __grid_constant__ RowU32 seq) {
    using S = RowsShape<HD>;
    constexpr int T = S::kTile, W = S::kWarps, D = S::kD, C = S::kChunks, kHalf = W * 32, kAll = S::kThreads;
    constexpr int kPad = T + 8;   // halves per head row of P
    constexpr int kScorers = 1, kFull = 2, kEmpty = 4;   // barriers; a buffer's number is added to the last two
    __shared__ uint4 qf_s[C][2][2][32];                  // [64-dim chunk][limb][half][lane]: B fragments of q
    __shared__ __align__(16) __half p_s[2][2][8][kPad];  // [buffer][limb][head][position]
    __shared__ float f_s[2][8];                          // what the sums so far are multiplied by
    // addresses of the codes of four tiles: the scorers are two tiles ahead at most, and each looks one further
    __shared__ __align__(16) uint64_t kaddr[4][T], vaddr[4][T];
    __shared__ float2 sc_s[2][T];                        // ks, vs
    __shared__ float wmax[2][W][8], qscale[8], lsum[W][8], m_s[8];

    const uint32_t item = blockIdx.x, kvh = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3, oct = lane >> 2;
    const bool scorer = warp < W;
    const int part = scorer ? warp : warp - W;   // the warp among its kind
    uint32_t row = 0;
    for (uint32_t step = 256; step; step >>= 1)
        if (row + step < a.n && starts.v[row + step] <= item) row += step;
    // rows without positions share their start with the next row: the last row with start <= item is meant
    const uint32_t items = starts.v[row + 1] - starts.v[row];
    const int grp = static_cast<int>(a.q_heads / a.kv_heads);
    Span sp = row_span(pos.v[row], a.window, a.prefix_len);
    const bool direct = is_whole(a, items, sp);
    if (!a.list_prefix) sp.pn = 0;
    const uint32_t total = sp.pn + sp.on;
    const uint32_t j0 = (item - starts.v[row]) * a.chunk, j1 = min(total, j0 + a.chunk);
    const uint32_t tiles = (j1 - j0 + T - 1) / T;
    const uint32_t pslot = sp.pn ? sp.pa % a.pre.capacity : 0, oslot = sp.oa % a.own.capacity;
    const uint64_t own_vec = static_cast<uint64_t>(seq.v[row]) * a.own.capacity * a.kv_heads + kvh;
    const uint64_t own_sc = (static_cast<uint64_t>(seq.v[row]) * a.kv_heads + kvh) * a.own.capacity;

    // Entry tid of tile t: addresses of its K and V codes, and its scales. The last position stands in for those
    // past the run (their weight is 0).
    auto write_places = [&](uint32_t t, float2& sc) {
        if (tid >= T) return;
        const uint32_t j = min(j0 + t * T + tid, j1 - 1);
        const bool p = j < sp.pn;
        const uint32_t cap = p ? a.pre.capacity : a.own.capacity;
        uint64_t slot = p ? static_cast<uint64_t>(pslot) + j : static_cast<uint64_t>(oslot) + (j - sp.pn);
        if (slot >= cap) slot -= cap;
        const uint64_t vec = ((p ? kvh : own_vec) + slot * a.kv_heads) * HD;
        const uint64_t at = (p ? static_cast<uint64_t>(kvh) * cap : own_sc) + slot;
        kaddr[t & 3][tid] = reinterpret_cast<uint64_t>((p ? a.pre.k : a.own.k) + vec);
        vaddr[t & 3][tid] = reinterpret_cast<uint64_t>((p ? a.pre.v : a.own.v) + vec);
        sc = make_float2(__ldg((p ? a.pre.ks : a.own.ks) + at), __ldg((p ? a.pre.vs : a.own.vs) + at));
    };

    wait_for_kernel_before();
    float2 sc_next = make_float2(0.0f, 0.0f);
    write_places(0, sc_next);
    if (tid < T) sc_s[0][tid] = sc_next;
    // q of head h: scaled by a power of two, then high and low fp16 parts
    for (int h = warp; h < 8; h += 2 * W) {
        const float* src = a.q + (static_cast<size_t>(row) * a.q_heads + static_cast<size_t>(kvh) * grp + h) * HD;
        float x[HD / 32], top = 0.0f;
#pragma unroll
        for (int i = 0; i < HD / 128; ++i) {
            // a plain load: ctx may be q's own buffer
            const float4 v = h < grp ? reinterpret_cast<const float4*>(src)[lane + 32 * i] : make_float4(0.f, 0.f, 0.f, 0.f);
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) top = fmaxf(top, fabsf(x[i]));
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = query_exponent(top);
        const float down = query_down(e);
        if (lane == 0) qscale[h] = query_up(e) * kLog2e * (FMT == GTM_KV_E4M3 ? 256.0f : 1.0f);
#pragma unroll
        for (int i = 0; i < HD / 128; ++i) {
            const int d = 4 * lane + 128 * i;   // four dims of one 16-dim run
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float u = x[4 * i + 2 * j] * down, v = x[4 * i + 2 * j + 1] * down;
                hi[j] = cvt2(u, v);
                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi[j]));
                lo[j] = cvt2(u - b.x, v - b.y);
            }
            const int c = d >> 6, t = (d >> 4) & 3, half = (d >> 3) & 1, at = (d >> 2) & 1;
            reinterpret_cast<uint2*>(&qf_s[c][0][half][h * 4 + t])[at] = make_uint2(hi[0], hi[1]);
            reinterpret_cast<uint2*>(&qf_s[c][1][half][h * 4 + t])[at] = make_uint2(lo[0], lo[1]);
        }
    }
    __syncthreads();

    if (scorer) {
        uint4 kr[2][C];
        auto load_k = [&](uint32_t t) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint4* p = reinterpret_cast<const uint4*>(kaddr[t & 3][part * 16 + oct + 8 * r]) + quad;
#pragma unroll
                for (int c = 0; c < C; ++c) kr[r][c] = __ldg(p + 4 * c);
            }
        };
        load_k(0);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        const float qs[2] = {qscale[2 * quad], qscale[2 * quad + 1]};
        for (uint32_t t = 0; t < tiles; ++t) {
            const bool more = t + 1 < tiles;
            const int buf = t & 1;
            if (more) write_places(t + 1, sc_next);
            // four sums per score (limb, half of the dims' runs): short chains, as each product's addition
            // to the accumulator is cut to fp32 rather than rounded, and four products in flight
            float part4[4][4] = {};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t w0[4] = {kr[0][c].x, kr[0][c].y, kr[0][c].z, kr[0][c].w};
                const uint32_t w1[4] = {kr[1][c].x, kr[1][c].y, kr[1][c].z, kr[1][c].w};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 hi = qf_s[c][0][half][lane], lo = qf_s[c][1][half][lane];
                    const uint32_t bh[4] = {hi.x, hi.y, hi.z, hi.w}, bl[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t b0 = bias_codes<FMT>(w0[2 * half + j]), b1 = bias_codes<FMT>(w1[2 * half + j]);
                        const uint32_t a0 = pair_in_word<FMT, 0>(b0), a2 = pair_in_word<FMT, 1>(b0);
                        const uint32_t a1 = pair_in_word<FMT, 0>(b1), a3 = pair_in_word<FMT, 1>(b1);
                        mma16816(part4[j], a0, a1, a2, a3, bh[2 * j], bh[2 * j + 1]);
                        mma16816(part4[2 + j], a0, a1, a2, a3, bl[2 * j], bl[2 * j + 1]);
                    }
                }
            }
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = (part4[0][i] + part4[1][i]) + (part4[2][i] + part4[3][i]);
            // s: positions oct and oct + 8 of the warp's 16, heads 2 quad and 2 quad + 1
            float vs[2], top[2] = {-INFINITY, -INFINITY};
            bool valid[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int p = part * 16 + oct + 8 * r;
                const float2 sc = sc_s[buf][p];
                valid[r] = j0 + t * T + p < j1;
                vs[r] = sc.y;
                const float lg = log2_vs(sc.y) - kWeightTop;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[2 * r + h] = valid[r] ? s[2 * r + h] * sc.x * qs[h] : -INFINITY;
                    top[h] = fmaxf(top[h], s[2 * r + h] + (valid[r] ? lg : 0.0f));
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                for (int x = 4; x < 32; x <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
            }
            if (oct == 0) *reinterpret_cast<float2*>(&wmax[buf][part][2 * quad]) = make_float2(top[0], top[1]);
            if (more && tid < T) sc_s[buf ^ 1][tid] = sc_next;
            bar_sync(kScorers, kHalf);
            if (more) load_k(t + 1);
            float mn[2] = {m[0], m[1]};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float2 x = *reinterpret_cast<const float2*>(&wmax[buf][w][2 * quad]);
                mn[0] = fmaxf(mn[0], x.x), mn[1] = fmaxf(mn[1], x.y);
            }
            if (t >= 2) bar_sync(kEmpty + buf, kAll);   // the sums of tile t - 2 have used the buffer
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = m[h] == mn[h] ? 1.0f : ex2(m[h] - mn[h]);
                m[h] = mn[h];
                l[h] *= f;
                if (part == 0 && oct == 0) f_s[buf][2 * quad + h] = f;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float e = valid[r] ? ex2(s[2 * r + h] - mn[h]) : 0.0f;
                    l[h] += e;
                    const float p = valid[r] ? e * vs[r] : 0.0f;
                    const __half hi = __float2half_rn(p);
                    const int at = part * 16 + oct + 8 * r;
                    p_s[buf][0][2 * quad + h][at] = hi;
                    p_s[buf][1][2 * quad + h][at] = __float2half_rn(p - __half2float(hi));
                }
            }
            bar_arrive(kFull + buf, kAll);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            for (int x = 4; x < 32; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
        }
        if (oct == 0) {
            lsum[part][2 * quad] = l[0], lsum[part][2 * quad + 1] = l[1];
            if (part == 0) m_s[2 * quad] = m[0], m_s[2 * quad + 1] = m[1];
        }
        __syncthreads();
        return;
    }

    uint32_t vr[T / 16][4][D / 4];
    const uint64_t vdim = static_cast<uint64_t>(part * S::kDims + oct * D);
    auto load_v = [&](uint32_t t, int ks) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint64_t p = vaddr[t & 3][16 * ks + 4 * quad + r] + vdim;
            if constexpr (D == 8) {
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
                vr[ks][r][0] = w.x, vr[ks][r][1] = w.y;
            } else {
                vr[ks][r][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
            }
        }
    };
#pragma unroll
    for (int ks = 0; ks < T / 16; ++ks) load_v(0, ks);
    float o[D / 2][4];
#pragma unroll
    for (int i = 0; i < D / 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    for (uint32_t t = 0; t < tiles; ++t) {
        const bool more = t + 1 < tiles;
        const int buf = t & 1;
        bar_sync(kFull + buf, kAll);   // the weights, and the addresses of the next tile
        const float fs[2] = {f_s[buf][2 * quad], f_s[buf][2 * quad + 1]};
        float add[D / 2][4] = {};   // this tile's share, added to o in fp32 (see above)
#pragma unroll
        for (int ks = 0; ks < T / 16; ++ks) {
            const uint2 bh = *reinterpret_cast<const uint2*>(&p_s[buf][0][oct][16 * ks + 4 * quad]);
            const uint2 bl = *reinterpret_cast<const uint2*>(&p_s[buf][1][oct][16 * ks + 4 * quad]);
#pragma unroll
            for (int wd = 0; wd < D / 4; ++wd) {
                uint32_t w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = bias_codes<FMT>(vr[ks][r][wd]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t a0 = pair_of_words<FMT>(w[0], w[1], 2 * i), a1 = pair_of_words<FMT>(w[0], w[1], 2 * i + 1);
                    const uint32_t a2 = pair_of_words<FMT>(w[2], w[3], 2 * i), a3 = pair_of_words<FMT>(w[2], w[3], 2 * i + 1);
                    mma16816(add[2 * wd + i], a0, a1, a2, a3, bh.x, bh.y);
                    mma16816(add[2 * wd + i], a0, a1, a2, a3, bl.x, bl.y);
                }
            }
            if (more) load_v(t + 1, ks);
        }
        if (t + 2 < tiles) bar_arrive(kEmpty + buf, kAll);
#pragma unroll
        for (int i = 0; i < D / 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = o[i][j] * fs[j & 1] + add[i][j];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int head = 2 * quad + h;
        if (head >= grp) continue;
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) l += lsum[w][head];
        const float f = (FMT == GTM_KV_E4M3 ? 256.0f : 1.0f) / (direct ? l : 1.0f);
        const size_t at = (static_cast<size_t>(item) * a.kv_heads + kvh) * grp + head;
        float* dst = direct ? a.ctx + (static_cast<size_t>(row) * a.q_heads + static_cast<size_t>(kvh) * grp + head) * HD : a.part + at * HD;
#pragma unroll
        for (int i = 0; i < D / 4; ++i)
            *reinterpret_cast<float4*>(dst + vdim + 4 * i) =
                make_float4(o[2 * i][h] * f, o[2 * i][h + 2] * f, o[2 * i + 1][h] * f, o[2 * i + 1][h + 2] * f);
        if (!direct && part == 0 && oct == 0) a.ml[at] = make_float2(m_s[head], l);
    }
}

// One CTA per (query head, row): the row's partial results merged, its own items' and the shared part's. Latency
// is all: two dependent rounds of loads, 5 to 9 us behind the other kernels. A factor per thread and eight
// results in flight, for long lists, gained nothing (6.6 against 5.9 us for one row, 10.3 against 9 for 32).
template <int HD>
__global__ void __launch_bounds__(HD / 4) kv_combine(const __grid_constant__ RowsArgs a, const __grid_constant__ Starts starts,
                                                     const __grid_constant__ RowU32 pos, const __grid_constant__ SharedPlan sh) {
    wait_for_kernel_before();
    const uint32_t head = blockIdx.x, row = blockIdx.y;
    const uint32_t first = starts.v[row], items = starts.v[row + 1] - first;
    const Span sp = row_span(pos.v[row], a.window, a.prefix_len);
    if (is_whole(a, items, sp)) return;
    // result s < items: [item][kv head][group]; then slots c + u of the CTAs that took the unit's tiles
    const size_t at = static_cast<size_t>(first) * a.q_heads + head;
    const uint32_t grp = a.q_heads / a.kv_heads, kvh = head / grp, qr = row * grp + head % grp;
    uint32_t parts = items;
    size_t slot = 0;
    if (!a.list_prefix && sp.pn) {
        const uint32_t u = qr / kSharedRows, g = kvh * sh.start[sh.units] + sh.start[u], tiles = sh.start[u + 1] - sh.start[u];
        const uint32_t c0 = g / sh.per, c1 = (g + tiles - 1) / sh.per;
        slot = (static_cast<size_t>(c0) + kvh * sh.units + u) * kSharedRows + qr % kSharedRows;
        parts += c1 - c0 + 1;
    }
    auto ml = [&](uint32_t s) { return s < items ? a.ml[at + static_cast<size_t>(s) * a.q_heads] : sh.ml[slot + static_cast<size_t>(s - items) * kSharedRows]; };
    float m = -INFINITY, l = 0.0f;
    for (uint32_t s = 0; s < parts; ++s) m = fmaxf(m, ml(s).x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s = 0; s < parts; ++s) {
        const float2 x = ml(s);
        const float f = ex2(x.x - m);
        const float* src = s < items ? a.part + (at + static_cast<size_t>(s) * a.q_heads) * HD : sh.part + (slot + static_cast<size_t>(s - items) * kSharedRows) * HD;
        const float4 p = reinterpret_cast<const float4*>(src)[threadIdx.x];
        l += x.y * f;
        o.x += p.x * f, o.y += p.y * f, o.z += p.z * f, o.w += p.w * f;
    }
    const float r = 1.0f / l;
    reinterpret_cast<float4*>(a.ctx + (static_cast<size_t>(row) * a.q_heads + head) * HD)[threadIdx.x] =
        make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
}

// Prefix positions x kv heads over all rows from which the prefix is computed once for all (two rows or more).
// kv_shared costs 10 (128 dims) to 25 us (512) however little it does; kv_rows reads the prefix again for every
// row at 3.3-4.3 TB/s. Calls replayed from a graph, us, once for all against row by row, int8 (e4m3 takes 1-2 us
// more on both sides): 2 heads of 512, 16 rows x 2,048 positions (65,536) 38 against 29, 32 rows (131,072) 39 against
// 53, but 2 rows x 32,768 (131,072) 75 against 60; 8 heads of 256, 4 rows x 2,048 (65,536) 25 against 15, 8 rows
// (131,072) 25 against 25, 32 rows x 512 (131,072) 24 against 25, 2 rows x 16,384 (262,144) 48 against 47; 8 heads
// of 128, 8 rows x 2,048 (131,072) 21 against 18, 16 rows 22 against 29; 4 heads of 128 under 32, 16 rows x 2,048
// (131,072) 23 against 19. The rule knows neither the heads' width nor how full a unit's 64 columns are.
constexpr uint64_t kSharedFrom = 98304;

// Items of all rows are at most n plus this (a run is at least the total / target).
constexpr uint32_t kTargetCtas = 592;
uint32_t target_items(uint32_t kv_heads) { return std::max(1u, kTargetCtas / kv_heads); }

template <int HD>
int launch_rows(RowsArgs& a, Starts& starts, const RowU32& pos, const RowU32& seq, const SharedPlan& sh, uint32_t fmt, int num_sms, cudaStream_t st) {
    using S = RowsShape<HD>;
    uint64_t sum = 0;
    uint32_t len[kMaxBatchRows];
    bool merge = false;
    for (uint32_t i = 0; i < a.n; ++i) {
        const Span s = row_span(pos.v[i], a.window, a.prefix_len);
        len[i] = s.on + (a.list_prefix ? s.pn : 0);
        merge = merge || (!a.list_prefix && s.pn);
        sum += len[i];
    }
    const uint64_t want = (sum + target_items(a.kv_heads) - 1) / target_items(a.kv_heads);
    const uint64_t least = std::max<uint64_t>(1, (want + S::kTile - 1) / S::kTile);   // tiles of a run, for the workspace
    if (least * S::kTile > 0x7FFFFFFFull) return set_error(GTM_ERR_UNSUPPORTED, "gtm_attention_kv_rows: %llu positions", (unsigned long long)sum);
    // Runs up to twice as long, or four tiles longer, where that makes the rounds of CTAs x (tiles + 1 for a run's
    // start) fewer by a sixteenth: 32 rows of 77-8,192 positions, 2 heads of 512: 4 tiles, four rounds 106 us, 5
    // tiles, three rounds 99; 3 rows of 1,000-8,000 36 -> 25. Below that short runs even out better (up to 3%). For
    // many rows the search would cost the host more than it gives.
    uint64_t tiles = least;
    if (a.n <= 128) {
        const uint64_t slots = static_cast<uint64_t>(num_sms) * (HD == 512 ? 1 : 2);
        uint64_t best = 0;
        for (uint64_t t = least; t <= least + std::min<uint64_t>(std::max<uint64_t>(least, 4), 8); ++t) {
            const uint32_t run = static_cast<uint32_t>(t * S::kTile);
            uint64_t runs = 0;
            for (uint32_t i = 0; i < a.n; ++i) runs += (len[i] + run - 1) / run;
            const uint64_t cost = (runs * a.kv_heads + slots - 1) / slots * (t + 1);
            if (t == least) best = cost * 15 / 16 + 1;   // what another has to stay below
            else if (cost < best) best = cost, tiles = t;
        }
    }
    a.chunk = static_cast<uint32_t>(tiles * S::kTile);
    starts.v[0] = 0;
    for (uint32_t i = 0; i < a.n; ++i) {
        const uint32_t items = (len[i] + a.chunk - 1) / a.chunk;
        starts.v[i + 1] = starts.v[i] + items;
        merge = merge || items > 1;
    }
    const uint32_t items = starts.v[a.n];
    a.ml = reinterpret_cast<float2*>(a.part + static_cast<size_t>(items) * a.q_heads * HD);
    const dim3 grid(items, a.kv_heads);
    const bool shared = !a.list_prefix && sh.start[sh.units];
    cudaError_t e = cudaSuccess;
    if (items)
        e = launch_after(shared, fmt == GTM_KV_INT8 ? kv_rows<HD, GTM_KV_INT8> : kv_rows<HD, GTM_KV_E4M3>, grid, S::kThreads, st, a, starts, pos, seq);
    if (e == cudaSuccess && merge)
        e = launch_after(items || shared, kv_combine<HD>, dim3(a.q_heads, a.n), HD / 4, st, a, starts, pos, sh);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_cuda_error("gtm_attention_kv_rows", e);
    }
    return GTM_OK;
}

bool heads_ok(uint32_t q_heads, uint32_t kv_heads) {
    return kv_heads > 0 && q_heads > 0 && q_heads <= 65535u && q_heads % kv_heads == 0 && q_heads / kv_heads <= kKvMaxGroup;
}

// The workspace: the error word, the rows' partial results, the shared part's.
constexpr size_t kErrBytes = 256;
thread_local bool t_test_wait = false;   // gtm_attention_kv_test_wait

size_t up256(size_t x) { return (x + 255) / 256 * 256; }
// rows' items: sum of ceil(len / chunk) <= n + sum / chunk <= n + target
size_t rows_bytes(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n) {
    return up256((static_cast<size_t>(n) + target_items(kv_heads)) * q_heads * (head_dim + 2) * sizeof(float));
}
size_t shared_bytes(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n, int sms) {
    return up256(shared_slots(q_heads, kv_heads, n, sms) * kSharedRows * (head_dim + 2) * sizeof(float));
}

// The SM count of the current device; 148 (a B200's) where there is no device to ask, so that a
// workspace can be planned on a host without one.
cudaError_t num_sms(int* sms) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        *sms = 148;
        return cudaSuccess;
    }
    return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

}  // namespace
}  // namespace gtm

using namespace gtm;

extern "C" {

GTM_API size_t gtm_attention_kv_workspace_bytes(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n) {
    if (!heads_ok(q_heads, kv_heads) || (head_dim != 128 && head_dim != 256 && head_dim != 512) || n == 0 || n > kMaxBatchRows)
        return 0;
    int sms = 0;
    if (num_sms(&sms) != cudaSuccess) return 0;
    return kErrBytes + rows_bytes(q_heads, kv_heads, head_dim, n) + shared_bytes(q_heads, kv_heads, head_dim, n, sms);
}

GTM_API int gtm_attention_kv_rows(const GtmKvCache* c, const GtmKvCache* prefix, uint32_t prefix_seq, uint32_t prefix_len,
                                  uint32_t q_heads, uint32_t n, uint32_t window, const float* q, const uint32_t* seqs,
                                  const uint32_t* positions, float* ctx, void* ws, size_t ws_bytes, void* stream) {
    const char* fn = "gtm_attention_kv_rows";
    int rc = check_kv(fn, "cache", c);
    if (rc) return rc;
    if (prefix_len) {
        rc = check_kv(fn, "prefix", prefix);
        if (rc) return rc;
        if (prefix->format != c->format || prefix->kv_heads != c->kv_heads || prefix->head_dim != c->head_dim)
            return set_error(GTM_ERR_INVALID, "%s: the prefix's format or heads are not the cache's", fn);
        if (prefix_seq >= prefix->num_seqs)
            return set_error(GTM_ERR_INVALID, "%s: prefix sequence %u of %u", fn, prefix_seq, prefix->num_seqs);
    }
    if (!heads_ok(q_heads, c->kv_heads))
        return set_error(GTM_ERR_UNSUPPORTED, "%s: q_heads %u / kv_heads %u (a group of 1..%u)", fn, q_heads, c->kv_heads,
                         kKvMaxGroup);
    if (n == 0) {
        clear_error();
        return GTM_OK;
    }
    if (n > kMaxBatchRows) return set_error(GTM_ERR_INVALID, "%s: n=%u rows (at most %u)", fn, n, kMaxBatchRows);
    if (!q || !ctx || !seqs || !positions) return set_error(GTM_ERR_INVALID, "%s: null pointer", fn);
    if (!ptr_aligned(q, 16) || !ptr_aligned(ctx, 16) || !ptr_aligned(ws, 16))
        return set_error(GTM_ERR_MISALIGNED, "%s: q, ctx and workspace need 16-byte alignment", fn);
    RowU32 pos, seq;
    uint64_t in_prefix = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const Span s = row_span(positions[i], window, prefix_len);
        in_prefix += s.pn;
        if (positions[i] == 0xFFFFFFFFu || seqs[i] >= c->num_seqs || s.on > c->capacity ||
            (s.pn && prefix_len - s.pa > prefix->capacity))
            return set_error(GTM_ERR_INVALID, "%s: row %u (sequence %u of %u, position %u, prefix %u) does not fit the rings", fn,
                             i, seqs[i], c->num_seqs, positions[i], prefix_len);
        pos.v[i] = positions[i];
        seq.v[i] = seqs[i];
    }
    const size_t need = gtm_attention_kv_workspace_bytes(q_heads, c->kv_heads, c->head_dim, n);
    if (!ws || ws_bytes < need) return set_error(GTM_ERR_WORKSPACE, "%s: workspace needs %zu bytes", fn, need);
    const size_t row_bytes = static_cast<size_t>(n) * q_heads * c->head_dim * sizeof(float);
    if ((ctx != q && overlap(q, row_bytes, ctx, row_bytes)) || overlap(ws, need, q, row_bytes) || overlap(ws, need, ctx, row_bytes))
        return set_error(GTM_ERR_INVALID, "%s: q, ctx and workspace overlap", fn);
    const auto side = [](const GtmKvCache* x, size_t s) {
        const size_t vec = s * x->capacity * x->kv_heads;
        return Side{static_cast<const uint8_t*>(x->k_dev) + vec * x->head_dim, static_cast<const uint8_t*>(x->v_dev) + vec * x->head_dim,
                    x->k_scale_dev + vec, x->v_scale_dev + vec, x->capacity};
    };
    RowsArgs a;
    a.own = side(c, 0);
    a.pre = prefix_len ? side(prefix, prefix_seq) : a.own;
    a.q = q;
    a.ctx = ctx;
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kErrBytes);
    a.q_heads = q_heads, a.kv_heads = c->kv_heads, a.n = n;
    a.window = window, a.prefix_len = prefix_len;
    int sms = 0;
    const cudaError_t de = num_sms(&sms);
    if (de != cudaSuccess) return set_cuda_error(fn, de);
    SharedPlan plan;
    plan.units = 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool test_wait = t_test_wait;
    t_test_wait = false;
    a.list_prefix = n < 2 || in_prefix * c->kv_heads < kSharedFrom;
    if (!a.list_prefix) {
        const SharedCall call{prefix, prefix_seq, prefix_len, q_heads, c->kv_heads, c->head_dim, n, window, q, static_cast<int*>(ws), test_wait};
        plan_shared(call, pos, sms, plan);
        plan.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kErrBytes + rows_bytes(q_heads, c->kv_heads, c->head_dim, n));
        plan.ml = reinterpret_cast<float2*>(plan.part + shared_slots(q_heads, c->kv_heads, n, sms) * kSharedRows * c->head_dim);
        if (plan.start[plan.units]) rc = launch_shared(call, pos, plan, sms, st);
        if (rc) return rc;
    }
    Starts starts;
    if (c->head_dim == 128)
        rc = launch_rows<128>(a, starts, pos, seq, plan, c->format, sms, st);
    else if (c->head_dim == 256)
        rc = launch_rows<256>(a, starts, pos, seq, plan, c->format, sms, st);
    else
        rc = launch_rows<512>(a, starts, pos, seq, plan, c->format, sms, st);
    if (rc) return rc;
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    clear_error();
    return GTM_OK;
}

GTM_API int gtm_attention_kv_check(void* ws, void* stream) {
    const char* fn = "gtm_attention_kv_check";
    if (!ws) return set_error(GTM_ERR_INVALID, "%s: null workspace", fn);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int flag = 0;
    cudaError_t e = cudaMemcpyAsync(&flag, ws, sizeof(int), cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess && flag) {
        e = cudaMemsetAsync(ws, 0, sizeof(int), st);
        if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    }
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    if (flag) return set_error(GTM_ERR_TIMEOUT, "gtm_attention_kv_rows: a pipeline wait over the prefix timed out (flag %d)", flag);
    clear_error();
    return GTM_OK;
}

GTM_API int gtm_attention_kv_test_wait(void) {
    t_test_wait = true;
    clear_error();
    return GTM_OK;
}

}  // extern "C"
