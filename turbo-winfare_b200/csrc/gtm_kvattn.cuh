// Shared by the attention kernels over the one-byte KV caches: a row's positions, the codes as fp16
// pairs, and the launch of the prefix part.
#pragma once
#include <cuda_fp16.h>

#include "gtm_kvcache.cuh"

namespace gtm {

constexpr uint32_t kKvMaxGroup = 8;
constexpr float kLog2e = 1.4426950408889634f;

// One side (prefix or own cache) as the kernels address it.
struct Side {
    const uint8_t *k, *v;
    const float *ks, *vs;
    uint32_t capacity;
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

// A carried weight p = exp2(s2 - m) * vs is at most 2^kWeightTop (61,148), which fp16 (65,504) has room for. Its two
// limbs are off by up to 2^-25 whatever p is, so the top is put as high as it goes: a weight is off by up to 2^-40.9 of
// the largest one (2^-32.9 in kv_shared, whose m may stay while weights grow). With the largest at 1, keys whose scores
// were 18 below it (2^-26) were lost, however many they were.
constexpr float kWeightTop = 15.9f;
// log2 vs as the stabiliser takes it: from 2^-88 on, so that exp2(s2 - m) <= 2^(16 + 88), and 2^23 of them sum up in
// fp32. Values of smaller scales (2^-100 is the least) still have p up to 2^3.
__device__ __forceinline__ float log2_vs(float vs) { return log2f(fmaxf(vs, 3.2311742677852644e-27f)); }

// A query head is split with its largest value in [2^14, 2^15), as its limbs, too, end at 2^-25: from [1, 2) on,
// one value thousands of times the others cost those their low bits. The power of two, from the largest |q|, and
// the factors 2^(14 - e) and 2^(e - 14).
__device__ __forceinline__ int query_exponent(float top) {
    return max(-112, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
}
__device__ __forceinline__ float query_down(int e) { return __int_as_float((141 - e) << 23); }
__device__ __forceinline__ float query_up(int e) { return __int_as_float((113 + e) << 23); }

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Code words (4 codes) as half2 pairs. Int8: 1024 + (code + 128) is the half 0x6400 | byte, minus
// 1152. E4m3: sign and 7 bits moved to a half's sign, exponent and top mantissa bits: value * 2^-8,
// exact, subnormals included.
template <int FMT>
__device__ __forceinline__ uint32_t bias_codes(uint32_t w) {
    return FMT == GTM_KV_INT8 ? w ^ 0x80808080u : w;
}
__device__ __forceinline__ uint32_t hsub1152(uint32_t h) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t e4m3_halves(uint32_t v) {   // codes in bytes 1 and 3
    return (v & 0x80008000u) | ((v >> 1) & 0x3F803F80u);
}
// codes 2i, 2i + 1 of one (biased) word
template <int FMT, int I>
__device__ __forceinline__ uint32_t pair_in_word(uint32_t w) {
    if constexpr (FMT == GTM_KV_INT8) return hsub1152(__byte_perm(w, 0x64646464u, I ? 0x4342 : 0x4140));
    return e4m3_halves(__byte_perm(w, 0u, I ? 0x3424 : 0x1404));
}
// code i of word a (low half) and of word b (high half)
template <int FMT>
__device__ __forceinline__ uint32_t pair_of_words(uint32_t a, uint32_t b, int i) {
    if constexpr (FMT == GTM_KV_INT8) {
        const uint32_t x = __byte_perm(a, b, i | ((4 + i) << 4));
        return hsub1152(__byte_perm(x, 0x64646464u, 0x4140));
    }
    return e4m3_halves(__byte_perm(a, b, (i << 4) | ((4 + i) << 12)));
}

// What kv_shared leaves for the merge: the partial results of unit u (a kv head and 64 of the rows x
// group query heads) made by CTA c are at slot c + u.
constexpr int kSharedRows = 64;                                                   // query rows of a unit
constexpr uint32_t kMaxUnitsPerHead = kMaxBatchRows * kKvMaxGroup / kSharedRows;   // 64
struct SharedPlan {
    float* part;          // [slot][64][head_dim]
    float2* ml;           // [slot][64]
    uint32_t per;         // tiles per CTA
    uint32_t units;       // units per kv head (0: no shared part)
    uint32_t start[kMaxUnitsPerHead + 1];   // first tile of a head's units, then the head's tiles
};

// Slots that any plan of at most n rows takes; the plan for these rows; the launch. `part` and `ml`
// of the plan are set by the caller between the two.
size_t shared_slots(uint32_t q_heads, uint32_t kv_heads, uint32_t n, int num_sms);
struct SharedCall {
    const GtmKvCache* prefix;
    uint32_t prefix_seq, prefix_len, q_heads, kv_heads, head_dim, n, window;
    const float* q;
    int* err;          // the workspace's error word
    bool test_wait;    // gtm_attention_kv_test_wait
};
void plan_shared(const SharedCall& c, const RowU32& pos, int num_sms, SharedPlan& plan);
int launch_shared(const SharedCall& c, const RowU32& pos, const SharedPlan& plan, int num_sms, cudaStream_t st);

}  // namespace gtm
