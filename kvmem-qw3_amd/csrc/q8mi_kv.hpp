// The paged key / value cache as the kernels see it: element types, row addresses, host checks.
#pragma once

#include <math.h>

#include "q8mi_device.hpp"
#include "q8mi_internal.hpp"

namespace q8mi {

constexpr uint32_t kMaxPageSize = 65536;

__host__ __device__ inline uint32_t kv_element_bytes(int dtype) { return dtype == Q8MI_KV_E4M3 ? 1 : 2; }

// Q8MI_OK when the descriptor is one the kernels serve.
inline int check_kv_cache(const char *what, const q8mi_kv_cache *c) {
    if (c == nullptr || c->k == nullptr || c->v == nullptr) return fail(Q8MI_REJECTED, "%s: null cache", what);
    if (c->dtype != Q8MI_KV_BF16 && c->dtype != Q8MI_KV_F16 && c->dtype != Q8MI_KV_E4M3)
        return fail(Q8MI_REJECTED, "%s: cache type %d", what, c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(Q8MI_REJECTED, "%s: head_dim %u is not 64, 128 or 256", what, c->head_dim);
    if (c->pages == 0 || c->pages > 0x7fffffffu || c->page_size == 0 || c->page_size > kMaxPageSize || c->kv_heads == 0)
        return fail(Q8MI_REJECTED, "%s: cache of %u pages of %u tokens, %u heads", what, c->pages, c->page_size, c->kv_heads);
    const uint64_t es = kv_element_bytes(c->dtype);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 != 0 ||
        (c->stride_page * es) % 16 != 0 || (c->stride_head * es) % 16 != 0 || (c->stride_token * es) % 16 != 0 ||
        c->stride_token < c->head_dim)
        return fail(Q8MI_REJECTED, "%s: cache rows must begin on 16-byte boundaries, stride_token >= head_dim", what);
    if (c->dtype == Q8MI_KV_E4M3 &&
        !(isfinite(c->k_scale) && isfinite(c->v_scale) && c->k_scale > 0.0f && c->v_scale > 0.0f))
        return fail(Q8MI_REJECTED, "%s: e4m3 scales must be finite and above zero", what);
    return Q8MI_OK;
}

// Rows of activations in memory, in bytes: `count` rows of `width`, `stride` apart (no less than width where there are several).
struct RowSet {
    uintptr_t base;
    uint64_t count, stride, width;
    uintptr_t end() const { return base + (count - 1) * stride + width; }
};
// Whether two sets of rows share a byte.  Sets that lie side by side in one buffer (one row's queries beside its outputs) do not.
inline bool rows_meet(const RowSet &a, const RowSet &b) {
    if (a.end() <= b.base || b.end() <= a.base) return false;
    if (a.count > 1 && a.stride == b.stride) {   // one answer for all rows: where b's row lies behind the a row before it
        const uint64_t s = a.stride;
        const uint64_t behind = b.base >= a.base ? (b.base - a.base) % s : (s - (a.base - b.base) % s) % s;
        return behind < a.width || behind + b.width > s;
    }
    for (uint64_t i = 0; i < a.count; ++i) {
        const uintptr_t lo = a.base + i * a.stride, hi = lo + a.width;
        const uint64_t k = lo < b.base + b.width ? 0 : (lo - b.base - b.width) / b.stride + 1;   // the first of b's that ends behind lo
        if (k < b.count && b.base + k * b.stride < hi) return true;
    }
    return false;
}

// Two floats as bf16, nearest even (v_cvt_pk_bf16_f32), the first in the lower half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    v2bf r;
    r.x = static_cast<__bf16>(a);
    r.y = static_cast<__bf16>(b);
    return __builtin_bit_cast(uint32_t, r);
}

// Four floats as four elements of a cache row (nearest even; e4m3: the quotient by the scale, clamped, NaN kept).
__device__ __forceinline__ void store_kv4(void *row, uint32_t element, int dtype, float scale, const float (&v)[4]) {
    if (dtype == Q8MI_KV_E4M3) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = v[i] / scale;
            t[i] = q != q ? q : fminf(fmaxf(q, -448.0f), 448.0f);
        }
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
        *reinterpret_cast<int *>(static_cast<uint8_t *>(row) + element) = w;
        return;
    }
    uint2 w;
    if (dtype == Q8MI_KV_BF16) {
        w = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = float_to_half_bits(v[i]);
        w = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(row) + element) = w;
}

}  // namespace q8mi
