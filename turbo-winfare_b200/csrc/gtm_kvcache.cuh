// The one-byte KV caches of include/gtmoe_attention.h: argument checks and code formats shared by
// the translation units that write, read and attend them.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "gtm_internal.h"
#include "gtmoe_attention.h"

namespace gtm {

// Per-row values of a launch, passed by value (no host-to-device copy, checked on the host).
struct RowU32 {
    uint32_t v[kMaxBatchRows];
};

constexpr float kKvTiny = 7.8886090522101181e-31f;   // 2^-100, the least scale of a vector

inline bool ptr_aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// Whether [a, a + na) and [b, b + nb) share bytes.
inline bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// GTM_OK, or the error of a cache descriptor that no kernel may be given.
inline int check_kv(const char* fn, const char* what, const GtmKvCache* c) {
    if (!c) return set_error(GTM_ERR_INVALID, "%s: null %s", fn, what);
    if (!c->k_dev || !c->v_dev || !c->k_scale_dev || !c->v_scale_dev)
        return set_error(GTM_ERR_INVALID, "%s: null pointer in the %s", fn, what);
    if (c->format != GTM_KV_INT8 && c->format != GTM_KV_E4M3)
        return set_error(GTM_ERR_UNSUPPORTED, "%s: %s format %u", fn, what, c->format);
    if (c->head_dim != 128 && c->head_dim != 256 && c->head_dim != 512)
        return set_error(GTM_ERR_UNSUPPORTED, "%s: %s head_dim %u (128, 256 or 512)", fn, what, c->head_dim);
    if (c->num_seqs == 0 || c->capacity == 0 || c->kv_heads == 0 || c->reserved != 0)
        return set_error(GTM_ERR_INVALID, "%s: %s of %u sequences, %u positions, %u heads, reserved %u", fn, what,
                         c->num_seqs, c->capacity, c->kv_heads, c->reserved);
    if (c->kv_heads > 65535u) return set_error(GTM_ERR_UNSUPPORTED, "%s: %s of %u heads (at most 65535)", fn, what, c->kv_heads);
    if (!ptr_aligned(c->k_dev, 16) || !ptr_aligned(c->v_dev, 16) || !ptr_aligned(c->k_scale_dev, 4) ||
        !ptr_aligned(c->v_scale_dev, 4))
        return set_error(GTM_ERR_MISALIGNED, "%s: %s codes need 16-byte alignment, scales 4", fn, what);
    return GTM_OK;
}

}  // namespace gtm
