// Attention over the one-byte KV caches (include/gtmoe_attention.h).
//
// kv_partial: one CTA per (kv head, chunk of positions, row), the row's prefix and own positions
// taken as one list; online softmax over tiles of 64 positions in fp32; kv_combine merges a row's
// chunks.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "gtm_kvcache.cuh"

namespace gtm {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;
constexpr uint32_t kMaxGroup = 8;

// One side (prefix or own cache) as the kernels address it.
struct Side {
    const uint8_t *k, *v;
    const float *ks, *vs;
    uint32_t capacity;
};

struct AttnArgs {
    Side own, pre;
    const float* q;
    float* part;     // [n][q_heads][splits][head_dim]
    float2* ml;      // [n][q_heads][splits]: largest score, sum of exp(score - largest)
    float* ctx;
    uint32_t q_heads, kv_heads, splits, window, prefix_len;
};

struct Span {
    uint32_t pa, pn, oa, on;   // prefix: first and count; own: first and count
};
__host__ __device__ __forceinline__ Span row_span(uint32_t pos, uint32_t window, uint32_t prefix_len) {
    const uint64_t end = static_cast<uint64_t>(pos) + 1;
    const uint64_t first = window && end > window ? end - window : 0;
    const uint64_t P = prefix_len;
    Span s;
    const uint64_t pe = end < P ? end : P;
    s.pa = static_cast<uint32_t>(first < P ? first : P);
    s.pn = static_cast<uint32_t>(pe > first ? pe - first : 0);
    s.oa = static_cast<uint32_t>(first > P ? first : P);
    s.on = static_cast<uint32_t>(end > s.oa ? end - s.oa : 0);
    return s;
}

template <int FMT>
__device__ __forceinline__ float2 two_codes(uint32_t two) {
    if constexpr (FMT == GTM_KV_INT8) {
        return make_float2(static_cast<float>(static_cast<int8_t>(two & 0xFFu)),
                           static_cast<float>(static_cast<int8_t>((two >> 8) & 0xFFu)));
    } else {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
        return __half22float2(__half2(h));
    }
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kThreads) kv_partial(const __grid_constant__ AttnArgs a, const __grid_constant__ RowU32 pos,
                                                       const __grid_constant__ RowU32 seq) {
    constexpr int L = HD / 32;   // codes of a vector per lane
    __shared__ float qs[kMaxGroup * HD];
    __shared__ float sc[kMaxGroup][kTile];
    __shared__ float vs_s[kTile], m_s[kMaxGroup], f_s[kMaxGroup], l_s[kMaxGroup];
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, row = blockIdx.z;
    const int grp = static_cast<int>(a.q_heads / a.kv_heads);
    const Span sp = row_span(pos.v[row], a.window, a.prefix_len);
    const uint32_t total = sp.pn + sp.on;
    const uint32_t chunk = (total + a.splits - 1) / a.splits;
    const uint64_t b0 = static_cast<uint64_t>(split) * chunk;
    const uint32_t j0 = static_cast<uint32_t>(b0 < total ? b0 : total), j1 = min(total, j0 + chunk);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* q = a.q + (static_cast<size_t>(row) * a.q_heads + static_cast<size_t>(kvh) * grp) * HD;
    for (int i = threadIdx.x; i < grp * HD; i += kThreads) qs[i] = q[i];
    if (threadIdx.x < kMaxGroup) m_s[threadIdx.x] = -INFINITY, l_s[threadIdx.x] = 0.0f;
    float acc[kMaxGroup][2] = {};
    // list position j -> the vector's index in its side's codes, and its scale's index
    auto place = [&](uint32_t j, const Side*& s, size_t& vec, size_t& sca) {
        const bool pre = j < sp.pn;
        s = pre ? &a.pre : &a.own;
        const uint32_t t = pre ? sp.pa + j : sp.oa + (j - sp.pn);
        const uint32_t slot = t % s->capacity;
        const size_t sq = pre ? 0 : seq.v[row];
        vec = ((sq * s->capacity + slot) * a.kv_heads + kvh) * HD;
        sca = (sq * a.kv_heads + kvh) * s->capacity + slot;
    };
    for (uint32_t t0 = j0; t0 < j1; t0 += kTile) {
        const int n = static_cast<int>(min(j1 - t0, static_cast<uint32_t>(kTile)));
        __syncthreads();
        for (int j = warp; j < n; j += kThreads / 32) {
            const Side* s;
            size_t vec, sca;
            place(t0 + j, s, vec, sca);
            const float ks = s->ks[sca];
            if (lane == 0) vs_s[j] = s->vs[sca];
            for (int g = 0; g < grp; ++g) {
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < L / 2; ++i) {
                    const int c = 2 * lane + 64 * i;
                    const float2 k = two_codes<FMT>(*reinterpret_cast<const uint16_t*>(s->k + vec + c));
                    d += qs[g * HD + c] * k.x + qs[g * HD + c + 1] * k.y;
                }
                for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
                if (lane == 0) sc[g][j] = d * ks;
            }
        }
        __syncthreads();
        if (warp < grp) {
            float m = m_s[warp];
            const float old = m;
            for (int j = lane; j < n; j += 32) m = fmaxf(m, sc[warp][j]);
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            float l = 0.0f;
            for (int j = lane; j < n; j += 32) {
                const float e = expf(sc[warp][j] - m);
                l += e;
                sc[warp][j] = e * vs_s[j];
            }
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane == 0) {
                const float f = expf(old - m);
                f_s[warp] = f;
                l_s[warp] = l_s[warp] * f + l;
                m_s[warp] = m;
            }
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < static_cast<int>(kMaxGroup); ++g)
            if (g < grp) acc[g][0] *= f_s[g], acc[g][1] *= f_s[g];
        for (int j = 0; j < n; ++j) {
            const Side* s;
            size_t vec, sca;
            place(t0 + j, s, vec, sca);
            if (2 * threadIdx.x < HD) {
                const float2 v = two_codes<FMT>(*reinterpret_cast<const uint16_t*>(s->v + vec + 2 * threadIdx.x));
#pragma unroll
                for (int g = 0; g < static_cast<int>(kMaxGroup); ++g)
                    if (g < grp) acc[g][0] += sc[g][j] * v.x, acc[g][1] += sc[g][j] * v.y;
            }
        }
    }
    __syncthreads();
    for (int g = 0; g < grp; ++g) {
        const size_t at = (static_cast<size_t>(row) * a.q_heads + static_cast<size_t>(kvh) * grp + g) * a.splits + split;
        if (threadIdx.x == 0) a.ml[at] = make_float2(m_s[g], l_s[g]);
        if (2 * threadIdx.x < HD)
            *reinterpret_cast<float2*>(a.part + at * HD + 2 * threadIdx.x) = make_float2(acc[g][0], acc[g][1]);
    }
}

// One CTA per (query head, row): the chunks' (largest, sum, weighted V) merged.
__global__ void __launch_bounds__(512) kv_combine(const __grid_constant__ AttnArgs a, uint32_t hd) {
    const size_t at = static_cast<size_t>(blockIdx.y) * a.q_heads + blockIdx.x;
    const float2* ml = a.ml + at * a.splits;
    const float* p = a.part + at * a.splits * hd;
    float m = -INFINITY;
    for (uint32_t s = 0; s < a.splits; ++s) m = fmaxf(m, ml[s].x);
    float l = 0.0f, o = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s) {
        if (ml[s].x == -INFINITY && ml[s].y == 0.0f) continue;   // an empty chunk
        const float f = expf(ml[s].x - m);
        l += ml[s].y * f;
        o += p[static_cast<size_t>(s) * hd + threadIdx.x] * f;
    }
    a.ctx[at * hd + threadIdx.x] = o / l;
}

uint32_t splits_for(uint32_t kv_heads, uint32_t n) {
    const uint32_t want = (592 + n * kv_heads - 1) / (n * kv_heads);
    return std::max(1u, want);
}

template <int HD>
void launch(const AttnArgs& a, const RowU32& pos, const RowU32& seq, uint32_t n, uint32_t fmt, cudaStream_t st) {
    const dim3 grid(a.kv_heads, a.splits, n);
    if (fmt == GTM_KV_INT8)
        kv_partial<HD, GTM_KV_INT8><<<grid, kThreads, 0, st>>>(a, pos, seq);
    else
        kv_partial<HD, GTM_KV_E4M3><<<grid, kThreads, 0, st>>>(a, pos, seq);
    kv_combine<<<dim3(a.q_heads, n), HD, 0, st>>>(a, HD);
}

bool heads_ok(uint32_t q_heads, uint32_t kv_heads) {
    return kv_heads > 0 && q_heads > 0 && q_heads <= 65535u && q_heads % kv_heads == 0 && q_heads / kv_heads <= kMaxGroup;
}

}  // namespace
}  // namespace gtm

using namespace gtm;

extern "C" {

GTM_API size_t gtm_attention_kv_workspace_bytes(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n) {
    if (!heads_ok(q_heads, kv_heads) || (head_dim != 128 && head_dim != 256 && head_dim != 512) || n == 0 || n > kMaxBatchRows)
        return 0;
    // n' * splits(n') over n' <= n rows is at most this many partials per query head
    const size_t rows = static_cast<size_t>(n) + 592 / kv_heads + 1;
    return rows * q_heads * (head_dim + 2) * sizeof(float) + 256;
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
                         kMaxGroup);
    if (n == 0) {
        clear_error();
        return GTM_OK;
    }
    if (n > kMaxBatchRows) return set_error(GTM_ERR_INVALID, "%s: n=%u rows (at most %u)", fn, n, kMaxBatchRows);
    if (!q || !ctx || !seqs || !positions) return set_error(GTM_ERR_INVALID, "%s: null pointer", fn);
    if (!ptr_aligned(q, 16) || !ptr_aligned(ctx, 16) || !ptr_aligned(ws, 16))
        return set_error(GTM_ERR_MISALIGNED, "%s: q, ctx and workspace need 16-byte alignment", fn);
    RowU32 pos, seq;
    for (uint32_t i = 0; i < n; ++i) {
        const Span s = row_span(positions[i], window, prefix_len);
        if (positions[i] == 0xFFFFFFFFu || seqs[i] >= c->num_seqs || s.on > c->capacity ||
            (s.pn && prefix_len - s.pa > prefix->capacity))
            return set_error(GTM_ERR_INVALID, "%s: row %u (sequence %u of %u, position %u, prefix %u) does not fit the rings", fn,
                             i, seqs[i], c->num_seqs, positions[i], prefix_len);
        pos.v[i] = positions[i];
        seq.v[i] = seqs[i];
    }
    const size_t need = gtm_attention_kv_workspace_bytes(q_heads, c->kv_heads, c->head_dim, n);
    if (!ws || ws_bytes < need) return set_error(GTM_ERR_WORKSPACE, "%s: workspace needs %zu bytes", fn, need);
    AttnArgs a;
    const auto side = [](const GtmKvCache* x, size_t s) {
        const size_t vec = s * x->capacity * x->kv_heads;
        return Side{static_cast<const uint8_t*>(x->k_dev) + vec * x->head_dim, static_cast<const uint8_t*>(x->v_dev) + vec * x->head_dim,
                    x->k_scale_dev + vec, x->v_scale_dev + vec, x->capacity};
    };
    a.own = side(c, 0);
    a.pre = prefix_len ? side(prefix, prefix_seq) : a.own;
    a.q = q;
    a.q_heads = q_heads, a.kv_heads = c->kv_heads;
    a.window = window, a.prefix_len = prefix_len;
    a.splits = splits_for(c->kv_heads, n);
    a.part = static_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(a.part + static_cast<size_t>(n) * q_heads * a.splits * c->head_dim);
    a.ctx = ctx;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->head_dim == 128)
        launch<128>(a, pos, seq, n, c->format, st);
    else if (c->head_dim == 256)
        launch<256>(a, pos, seq, n, c->format, st);
    else
        launch<512>(a, pos, seq, n, c->format, st);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    clear_error();
    return GTM_OK;
}

}  // extern "C"
