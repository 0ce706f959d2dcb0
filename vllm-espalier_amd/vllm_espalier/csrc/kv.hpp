// What the kernels over a paged cache of keys and values share: its 16- and 8-bit elements, and the host's checks of it.
#pragma once

#include "../../../include/espalier.h"
#include "common.hpp"

#include <algorithm>
#include <utility>

namespace esp {

constexpr int E4M3 = ESP_E4M3;
constexpr float E4M3_MAX = 448.0f;

// Bytes of an element
__host__ __device__ constexpr int kv_bytes(int dtype) { return dtype == E4M3 ? 1 : 2; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Two floats as bf16 or fp16, to nearest even
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// Two floats as e4m3 in the low (or, HI, the high) half of w, to nearest even, those past the largest (infinities too) as the
// largest, a NaN as a NaN
template <bool HI>
__device__ __forceinline__ int pack_e4m3(float a, float b, int w) {
    a = a > E4M3_MAX ? E4M3_MAX : a < -E4M3_MAX ? -E4M3_MAX : a;      // (a NaN compares false and stays)
    b = b > E4M3_MAX ? E4M3_MAX : b < -E4M3_MAX ? -E4M3_MAX : b;
    return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, HI);
}

}  // namespace esp

namespace esp_host {

// nullptr, or what is wrong with a cache. `align`: the bytes that its rows of D elements are aligned to
inline const char* kv_cache_error(const esp_kv_cache* c, int dtype) {
    if (!c) return "null cache";
    if (c->dtype != dtype && c->dtype != ESP_E4M3) return "a cache has the rows' dtype or e4m3";
    if (c->dim != 64 && c->dim != 128 && c->dim != 256) return "heads of 64, 128 or 256 elements";
    if (c->heads < 1 || c->heads > 1024) return "1 to 1024 heads in the cache";
    if (c->pages < 1 || c->pages >= (int64_t(1) << 31)) return "1 to 2^31 - 1 pages";
    if (c->page < 16 || c->page > 65536 || c->page % 16) return "pages of a multiple of 16 tokens, at most 65536";
    if (!c->k || !c->v) return "null pointer";
    if ((c->dtype == ESP_E4M3) != (c->k_scale != nullptr) || (c->dtype == ESP_E4M3) != (c->v_scale != nullptr))
        return "an e4m3 cache has a scale a head for k and for v, one of 16 bits has none";
    const int64_t size = esp::kv_bytes(c->dtype);
    const int64_t strides[6] = {c->k_page, c->k_token, c->k_head, c->v_page, c->v_token, c->v_head};
    for (const int64_t s : strides) {
        if (s < 0 || s >= (int64_t(1) << 40)) return "cache strides of 0 to 2^40 elements";
        if (s * size % 16) return "cache rows must be aligned to 16 bytes";
    }
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return "cache rows must be aligned to 16 bytes";
    if (c->k_token < c->dim || c->v_token < c->dim) return "the cache's tokens overlap";
    if (c->k_token >= (1 << 24) || c->v_token >= (1 << 24)) return "a token's stride of at most 2^24 elements";
    return nullptr;
}

// Whether two of the cache's elements share a place (no call may write into such a one): a dimension's stride must be past all that the
// ones of smaller strides span
inline bool kv_overlaps(int64_t dim, int64_t pages, int64_t page_stride, int64_t page, int64_t token_stride, int64_t heads, int64_t head_stride) {
    int64_t sizes[3] = {pages, page, heads}, strides[3] = {page_stride, token_stride, head_stride}, span = dim;
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (strides[j] < strides[i]) {
                std::swap(strides[i], strides[j]);
                std::swap(sizes[i], sizes[j]);
            }
    for (int i = 0; i < 3; ++i) {
        if (sizes[i] == 1) continue;
        if (strides[i] < span) return true;
        span += strides[i] * (sizes[i] - 1);
    }
    return false;
}

// Whether k and v of one layout (kv_overlaps is false of it) share an element: whether what lies between their first ones, v - k elements,
// is a difference of two places. The largest stride first: all that the smaller ones span is less than it, so one of two multiples of it
// is in the difference, if any
inline bool kv_share(int64_t between, int64_t dim, int64_t pages, int64_t page_stride, int64_t page, int64_t token_stride, int64_t heads,
                     int64_t head_stride) {
    std::pair<int64_t, int64_t> by[3] = {{page_stride, pages}, {token_stride, page}, {head_stride, heads}};
    std::sort(by, by + 3);
    const auto reached = [&](const auto& self, int level, int64_t d) -> bool {
        if (level < 0) return d > -dim && d < dim;
        const auto [stride, n] = by[level];
        if (n == 1) return self(self, level - 1, d);
        const int64_t q = d >= 0 ? d / stride : -((-d + stride - 1) / stride);
        for (int64_t k = q; k <= q + 1; ++k)
            if (k > -n && k < n && self(self, level - 1, d - k * stride)) return true;
        return false;
    };
    return reached(reached, 2, between);
}

}  // namespace esp_host
