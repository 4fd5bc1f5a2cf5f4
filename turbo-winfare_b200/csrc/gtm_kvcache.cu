// Writing and reading the one-byte ring KV caches (include/gtmoe_attention.h).
//
// kv_write: one warp per (row, head). y = x / sqrt(mean x^2 + eps) * w, rotated, is formed in 64
// bits and rounded once: to fp32 for a query, to a one-byte code for a key or value. In 64 bits a
// sum's order moves y by ~1e-16, so a code (an integer near y / scale) is the definition's except
// for a chance of ~1e-14 per value; in 32 bits about one code in 10^5 would follow the reduction
// tree. The angles position * theta^(-2i/head_dim) are the same for every head of a row: the
// CTA's threads form one cosine and sine each, and all its heads take them from shared memory.
// Per value the pass moves 4 bytes in and 4 (query) or 1 (key, value) out; the 64-bit work is ~12
// operations a value plus ~150 a pair and CTA, long chains of which bound large calls:
// 512 rows of 16 + 2 x 8 heads of 256 take 12.4 us against 4.2 for the bytes. 32 rows take 3.8 us and
// one 3.2, nearly all launch, a row's loads and the angles' chain of operations.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>

#include "gtm_kvcache.cuh"

namespace gtm {
namespace {

constexpr int kWriteWarps = 8;

struct WriteArgs {
    const float *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    const uint16_t *q_w, *k_w;
    float* q_out;
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    double c_hi, c_lo;   // 2 * log2(theta) / head_dim as a sum of two doubles
    double eps;
    uint32_t q_heads, kv_heads, capacity, pairs, vec;   // vec: inputs may be read 16 bytes at a time
};

__device__ __forceinline__ double warp_sum(double a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}
__device__ __forceinline__ double warp_max(double a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = fmax(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}

// V consecutive floats at p. Plain loads: q may be written in place by this very launch (each warp writes a head that
// it has read), and __ldg is for what no one writes meanwhile.
template <int V>
__device__ __forceinline__ void load_vals(const float* p, bool vec, float (&x)[V]) {
    if (vec) {
        if constexpr (V == 2) {
            const float2 t = *reinterpret_cast<const float2*>(p);
            x[0] = t.x, x[1] = t.y;
        } else {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) {
                const float4 t = reinterpret_cast<const float4*>(p)[j];
                x[4 * j] = t.x, x[4 * j + 1] = t.y, x[4 * j + 2] = t.z, x[4 * j + 3] = t.w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = p[j];
    }
}

// |u| >= 0 to its e4m3 code: steps of 2^(e-3) in [2^e, 2^(e+1)), of 2^-9 below 2^-6; at most 448.
__device__ __forceinline__ uint32_t e4m3_code(double u) {
    const uint32_t hi = static_cast<uint32_t>(__double2hiint(u));
    int e = static_cast<int>((hi >> 20) & 0x7FFu) - 1023;
    e = max(e, -6);
    const double scaled = fabs(u) * __hiloint2double((1023 + 3 - e) << 20, 0);   // exact
    const int r = __double2int_rn(scaled);                                       // 0..16
    const int code = min((e + 7) * 8 + r - 8, 0x7E);
    return static_cast<uint32_t>(code) | ((hi >> 24) & 0x80u);
}

template <int HD, int FMT>
__global__ void __launch_bounds__(kWriteWarps * 32) kv_write(const __grid_constant__ WriteArgs a,
                                                             const __grid_constant__ RowU32 pos,
                                                             const __grid_constant__ RowU32 seq) {
    constexpr int V = HD / 64;   // values per lane and half: pairs (d, d + HD/2) stay in one lane
    __shared__ double2 rot[HD / 2];
    const uint32_t row = blockIdx.x, p = pos.v[row];
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t step = kWriteWarps * gridDim.y;

    auto source = [&](uint32_t h) {
        if (h < a.q_heads) return a.q + row * a.q_stride + static_cast<size_t>(h) * HD;
        h -= a.q_heads;
        if (h < a.kv_heads) return a.k + row * a.k_stride + static_cast<size_t>(h) * HD;
        return a.v + row * a.v_stride + static_cast<size_t>(h - a.kv_heads) * HD;
    };
    float x0[V], x1[V];
    uint32_t h = blockIdx.y * kWriteWarps + warp;
    if (h < heads) {
        load_vals<V>(source(h) + lane * V, a.vec, x0);
        load_vals<V>(source(h) + HD / 2 + lane * V, a.vec, x1);
    }
    if (blockIdx.y * kWriteWarps < a.q_heads + a.kv_heads) {
        for (uint32_t i = threadIdx.x; i < a.pairs; i += kWriteWarps * 32) {
            // theta^(-2i/hd) = 2^-(i c), i c carried to ~2^-100 so that far positions' angles hold
            const double t = static_cast<double>(i) * a.c_hi;
            const double lo = fma(static_cast<double>(i), a.c_hi, -t) + static_cast<double>(i) * a.c_lo;
            const double f = exp2(-t);
            const double freq = fma(f, -0.69314718055994530942 * lo, f);
            double s, c;
            sincos(static_cast<double>(p) * freq, &s, &c);
            rot[i] = make_double2(c, s);
        }
    }
    __syncthreads();
    const uint32_t slot = p % a.capacity;
    while (h < heads) {
        double y0[V], y1[V], ss = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            y0[j] = x0[j], y1[j] = x1[j];
            ss = fma(y0[j], y0[j], ss);
            ss = fma(y1[j], y1[j], ss);
        }
        const uint32_t now = h;
        h += step;
        if (h < heads) {
            load_vals<V>(source(h) + lane * V, a.vec, x0);
            load_vals<V>(source(h) + HD / 2 + lane * V, a.vec, x1);
        }
        const double inv = 1.0 / sqrt(warp_sum(ss) * (1.0 / HD) + a.eps);
        const bool is_q = now < a.q_heads, is_k = !is_q && now < a.q_heads + a.kv_heads;
        const uint16_t* w = is_q ? a.q_w : is_k ? a.k_w : nullptr;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            y0[j] *= inv, y1[j] *= inv;
            if (w) {
                y0[j] *= __uint_as_float(static_cast<uint32_t>(__ldg(w + lane * V + j)) << 16);
                y1[j] *= __uint_as_float(static_cast<uint32_t>(__ldg(w + HD / 2 + lane * V + j)) << 16);
            }
        }
        if (is_q || is_k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (static_cast<uint32_t>(lane * V + j) < a.pairs) {
                    const double2 cs = rot[lane * V + j];
                    const double r0 = y0[j] * cs.x - y1[j] * cs.y;
                    y1[j] = y0[j] * cs.y + y1[j] * cs.x;
                    y0[j] = r0;
                }
            }
        }
        if (is_q) {
            float* o = a.q_out + (static_cast<size_t>(row) * a.q_heads + now) * HD + lane * V;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float f[V];
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = static_cast<float>(half ? y1[j] : y0[j]);
                if constexpr (V == 2) {
                    *reinterpret_cast<float2*>(o + half * (HD / 2)) = make_float2(f[0], f[1]);
                } else {
#pragma unroll
                    for (int j = 0; j < V / 4; ++j)
                        reinterpret_cast<float4*>(o + half * (HD / 2))[j] =
                            make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                }
            }
            continue;
        }
        double top = 0.0;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            top = fmax(top, fmax(fabs(y0[j]), fabs(y1[j])));
            finite = finite && isfinite(y0[j]) && isfinite(y1[j]);
        }
        finite = __all_sync(0xffffffffu, finite);
        top = warp_max(top);
        constexpr double kMost = FMT == GTM_KV_INT8 ? 127.0 : 448.0;
        const float scale = finite ? fmaxf(static_cast<float>(top / kMost), kKvTiny) : __int_as_float(0x7FC00000);
        const double s = scale, rs = 1.0 / s;
        uint32_t code[2][V];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double y = half ? y1[j] : y0[j];
                const double u0 = y * rs;
                const double u = fma(fma(-u0, s, y), rs, u0);   // y / s, rounded once
                if constexpr (FMT == GTM_KV_INT8)
                    code[half][j] = static_cast<uint32_t>(max(-127, min(127, __double2int_rn(u)))) & 0xFFu;
                else
                    code[half][j] = e4m3_code(u);
                if (!finite) code[half][j] = 0;
            }
        const uint32_t kvh = now - a.q_heads - (is_k ? 0 : a.kv_heads);
        const size_t ring = (static_cast<size_t>(seq.v[row]) * a.capacity + slot) * a.kv_heads + kvh;
        uint8_t* o = (is_k ? a.k_codes : a.v_codes) + ring * HD + lane * V;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint8_t* d = o + half * (HD / 2);
            if constexpr (V == 2) {
                *reinterpret_cast<uint16_t*>(d) = static_cast<uint16_t>(code[half][0] | (code[half][1] << 8));
            } else {
                uint32_t wd[V / 4];
#pragma unroll
                for (int j = 0; j < V / 4; ++j)
                    wd[j] = code[half][4 * j] | (code[half][4 * j + 1] << 8) | (code[half][4 * j + 2] << 16) |
                            (code[half][4 * j + 3] << 24);
                if constexpr (V == 4)
                    *reinterpret_cast<uint32_t*>(d) = wd[0];
                else
                    *reinterpret_cast<uint2*>(d) = make_uint2(wd[0], wd[1]);
            }
        }
        if (lane == 0)
            (is_k ? a.k_scale : a.v_scale)[(static_cast<size_t>(seq.v[row]) * a.kv_heads + kvh) * a.capacity + slot] = scale;
    }
}

// kv_read: a CTA reads kReadRows positions of the keys or of the values (blockIdx.y), four codes a thread and
// load: a warp takes 128 bytes in and 512 out, the loads of all its rows before the first store. Bound by
// HBM, four fifths of it stores: 131,071 positions of 2 heads of 512 (1.34 GB) 214 us, 6.28 TB/s; a
// 1,000 positions of 8 heads of 256 5.8 us, half of it launch. Sixteen codes a thread wrote 64-byte pieces: 277 us.
constexpr int kReadRows = 8;
struct ReadArgs {
    const uint8_t* codes[2];
    const float* scale[2];
    float* out[2];
    uint32_t count, start, capacity, words, shift;   // start: ring row of the first position; words
                                                               // of four codes in a row, 2^shift of them a vector
};

template <int FMT>
__device__ __forceinline__ float2 code_pair(uint32_t two) {   // the low 16 bits: two codes
    if constexpr (FMT == GTM_KV_INT8) {
        return make_float2(static_cast<float>(static_cast<int8_t>(two & 0xFFu)),
                           static_cast<float>(static_cast<int8_t>((two >> 8) & 0xFFu)));
    } else {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
        return __half22float2(__half2(h));
    }
}

template <int FMT>
__global__ void __launch_bounds__(256) kv_read(const __grid_constant__ ReadArgs a) {
    const int which = a.out[0] && blockIdx.y == 0 ? 0 : 1;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.codes[which]);
    float4* out = reinterpret_cast<float4*>(a.out[which]);
    const uint32_t t0 = blockIdx.x * kReadRows;
    for (uint32_t w = threadIdx.x; w < a.words; w += 256) {
        const float* scale = a.scale[which] + static_cast<size_t>(w >> a.shift) * a.capacity;
        uint32_t word[kReadRows];
        float s[kReadRows];
#pragma unroll
        for (int r = 0; r < kReadRows; ++r) {
            uint64_t slot = static_cast<uint64_t>(a.start) + min(t0 + r, a.count - 1);
            if (slot >= a.capacity) slot -= a.capacity;
            word[r] = __ldg(codes + slot * a.words + w);
            s[r] = __ldg(scale + slot);
        }
#pragma unroll
        for (int r = 0; r < kReadRows; ++r) {
            const float2 lo = code_pair<FMT>(word[r]), hi = code_pair<FMT>(word[r] >> 16);
            if (t0 + r < a.count)
                __stcs(out + static_cast<size_t>(t0 + r) * a.words + w, make_float4(lo.x * s[r], lo.y * s[r], hi.x * s[r], hi.y * s[r]));
        }
    }
}

// Whether two rows of a step name the same ring row (512 keys in 1,024 places, linear probing).
bool ring_row_twice(const uint32_t* seqs, const uint32_t* positions, uint32_t n, uint32_t capacity) {
    uint64_t seen[1024];
    for (uint64_t& s : seen) s = ~0ull;
    for (uint32_t i = 0; i < n; ++i) {
        const uint64_t key = static_cast<uint64_t>(seqs[i]) * capacity + positions[i] % capacity;
        uint32_t at = static_cast<uint32_t>((key * 0x9E3779B97F4A7C15ull) >> 54);
        while (seen[at] != ~0ull) {
            if (seen[at] == key) return true;
            at = (at + 1) & 1023u;
        }
        seen[at] = key;
    }
    return false;
}

// Whether `out` touches a row of x (n rows of `width` floats, `stride` apart).
bool rows_touch(const float* x, uint64_t stride, uint64_t width, uint32_t n, const float* out, uint64_t out_floats) {
    if (!overlap(x, ((n - 1) * stride + width) * 4, out, out_floats * 4)) return false;
    for (uint32_t i = 0; i < n; ++i)
        if (overlap(x + i * stride, width * 4, out, out_floats * 4)) return true;
    return false;
}

template <int HD>
void launch_write(const WriteArgs& a, const RowU32& pos, const RowU32& seq, uint32_t n, uint32_t fmt, cudaStream_t st) {
    // A CTA per row forms each angle once; few rows are split over their heads (a CTA per 8, an
    // angle formed per CTA) until about four CTAs per SM run.
    const uint32_t most = (a.q_heads + 2 * a.kv_heads + kWriteWarps - 1) / kWriteWarps;
    const uint32_t want = 592 / n;
    const dim3 grid(n, want < 1 ? 1 : (want < most ? want : most));
    if (fmt == GTM_KV_INT8)
        kv_write<HD, GTM_KV_INT8><<<grid, kWriteWarps * 32, 0, st>>>(a, pos, seq);
    else
        kv_write<HD, GTM_KV_E4M3><<<grid, kWriteWarps * 32, 0, st>>>(a, pos, seq);
}

}  // namespace
}  // namespace gtm

using namespace gtm;

extern "C" {

GTM_API int gtm_qkv_cache_rows(const GtmKvCache* c, uint32_t q_heads, uint32_t n, const float* q, const float* k,
                               const float* v, uint64_t q_stride, uint64_t k_stride, uint64_t v_stride,
                               const uint16_t* q_w, const uint16_t* k_w, float eps, uint32_t rotated_pairs, float theta,
                               const uint32_t* positions, const uint32_t* seqs, float* q_out, void* stream) {
    const char* fn = "gtm_qkv_cache_rows";
    int rc = check_kv(fn, "cache", c);
    if (rc) return rc;
    if (n == 0) {
        clear_error();
        return GTM_OK;
    }
    if (n > kMaxBatchRows) return set_error(GTM_ERR_INVALID, "%s: n=%u rows (at most %u)", fn, n, kMaxBatchRows);
    if (!q || !k || !v || !q_out || !positions || !seqs) return set_error(GTM_ERR_INVALID, "%s: null pointer", fn);
    if (q_heads == 0 || q_heads > 65535u) return set_error(GTM_ERR_UNSUPPORTED, "%s: q_heads=%u (1..65535)", fn, q_heads);
    const uint64_t q_width = static_cast<uint64_t>(q_heads) * c->head_dim, kv_width = static_cast<uint64_t>(c->kv_heads) * c->head_dim;
    if (n > 1 && (q_stride < q_width || k_stride < kv_width || v_stride < kv_width))
        return set_error(GTM_ERR_INVALID, "%s: row strides %llu, %llu, %llu below the rows' widths", fn,
                         (unsigned long long)q_stride, (unsigned long long)k_stride, (unsigned long long)v_stride);
    if (rotated_pairs > c->head_dim / 2)
        return set_error(GTM_ERR_INVALID, "%s: rotated_pairs %u > head_dim / 2", fn, rotated_pairs);
    if (!(theta > 0.0f) || !std::isfinite(theta) || !(eps >= 0.0f) || !std::isfinite(eps))
        return set_error(GTM_ERR_INVALID, "%s: theta must be finite and > 0, eps finite and >= 0", fn);
    if (!ptr_aligned(q, 4) || !ptr_aligned(k, 4) || !ptr_aligned(v, 4) || !ptr_aligned(q_out, 16) || !ptr_aligned(q_w, 2) ||
        !ptr_aligned(k_w, 2))
        return set_error(GTM_ERR_MISALIGNED, "%s: q_out needs 16-byte alignment, inputs 4, weights 2", fn);
    if (q_out == q && n > 1 && q_stride != q_width)
        return set_error(GTM_ERR_INVALID, "%s: in place needs q_stride = q_heads * head_dim", fn);
    RowU32 pos, seq;
    for (uint32_t i = 0; i < n; ++i) {
        if (seqs[i] >= c->num_seqs)
            return set_error(GTM_ERR_INVALID, "%s: row %u names sequence %u of %u", fn, i, seqs[i], c->num_seqs);
        pos.v[i] = positions[i];
        seq.v[i] = seqs[i];
    }
    if (ring_row_twice(seqs, positions, n, c->capacity))
        return set_error(GTM_ERR_INVALID, "%s: two rows write the same ring row of one sequence", fn);
    // a head's warp writes q_out while others still read: only where each reads what it writes, in place, is that sound
    if ((q_out != q && rows_touch(q, q_stride, q_width, n, q_out, n * q_width)) ||
        rows_touch(k, k_stride, kv_width, n, q_out, n * q_width) || rows_touch(v, v_stride, kv_width, n, q_out, n * q_width))
        return set_error(GTM_ERR_INVALID, "%s: q_out overlaps an input's rows (it may be q itself)", fn);
    WriteArgs a;
    a.q = q, a.k = k, a.v = v;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
    a.q_w = q_w, a.k_w = k_w;
    a.q_out = q_out;
    a.k_codes = static_cast<uint8_t*>(c->k_dev), a.v_codes = static_cast<uint8_t*>(c->v_dev);
    a.k_scale = c->k_scale_dev, a.v_scale = c->v_scale_dev;
    const long double step = 2.0L * log2l(static_cast<long double>(theta)) / c->head_dim;
    a.c_hi = static_cast<double>(step);
    a.c_lo = static_cast<double>(step - static_cast<long double>(a.c_hi));
    a.eps = eps;
    a.q_heads = q_heads, a.kv_heads = c->kv_heads, a.capacity = c->capacity, a.pairs = rotated_pairs;
    a.vec = ptr_aligned(q, 16) && ptr_aligned(k, 16) && ptr_aligned(v, 16) &&
            (n == 1 || (q_stride % 4 == 0 && k_stride % 4 == 0 && v_stride % 4 == 0));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->head_dim == 128)
        launch_write<128>(a, pos, seq, n, c->format, st);
    else if (c->head_dim == 256)
        launch_write<256>(a, pos, seq, n, c->format, st);
    else
        launch_write<512>(a, pos, seq, n, c->format, st);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    clear_error();
    return GTM_OK;
}

GTM_API int gtm_kv_read(const GtmKvCache* c, uint32_t seq, uint32_t first, uint32_t count, float* k_out, float* v_out,
                        void* stream) {
    const char* fn = "gtm_kv_read";
    int rc = check_kv(fn, "cache", c);
    if (rc) return rc;
    if (seq >= c->num_seqs) return set_error(GTM_ERR_INVALID, "%s: sequence %u of %u", fn, seq, c->num_seqs);
    if (count > c->capacity || static_cast<uint64_t>(first) + count > (1ull << 32))
        return set_error(GTM_ERR_INVALID, "%s: %u positions from %u in a ring of %u rows", fn, count, first, c->capacity);
    if (!k_out && !v_out && count) return set_error(GTM_ERR_INVALID, "%s: null pointer", fn);
    if (!ptr_aligned(k_out, 16) || !ptr_aligned(v_out, 16))
        return set_error(GTM_ERR_MISALIGNED, "%s: outputs need 16-byte alignment", fn);
    if (count == 0) {
        clear_error();
        return GTM_OK;
    }
    ReadArgs a;
    const size_t codes = static_cast<size_t>(seq) * c->capacity * c->kv_heads * c->head_dim;
    const size_t scales = static_cast<size_t>(seq) * c->kv_heads * c->capacity;
    a.codes[0] = static_cast<const uint8_t*>(c->k_dev) + codes, a.codes[1] = static_cast<const uint8_t*>(c->v_dev) + codes;
    a.scale[0] = c->k_scale_dev + scales, a.scale[1] = c->v_scale_dev + scales;
    a.out[0] = k_out, a.out[1] = v_out;
    a.words = c->kv_heads * (c->head_dim / 4);
    a.shift = c->head_dim == 128 ? 5 : c->head_dim == 256 ? 6 : 7;
    a.count = count;
    a.start = first % c->capacity;
    a.capacity = c->capacity;
    const dim3 grid((count - 1) / kReadRows + 1, k_out && v_out ? 2 : 1);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->format == GTM_KV_INT8)
        kv_read<GTM_KV_INT8><<<grid, 256, 0, st>>>(a);
    else
        kv_read<GTM_KV_E4M3><<<grid, 256, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(fn, e);
    clear_error();
    return GTM_OK;
}

}  // extern "C"
