// What the kernels over rows of logits share: loads of rows that start at any element, the order of logits and their indices, and
// the exponentials at a temperature.
#pragma once

#include "common.hpp"
#include "norm.hpp"

namespace esp {

// unaligned 16-byte loads: rows start at any element (an odd vocabulary)
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// elements i .. i + 8 of a row
template <int DT>
__device__ __forceinline__ void load_whole_group(const void* row, int i, float (&v)[8]) {
    if constexpr (DT == F32) {
        const f32x4_a4* p = reinterpret_cast<const f32x4_a4*>(static_cast<const float*>(row) + i);
        const f32x4_a4 a = p[0], b = p[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = a[k];
            v[4 + k] = b[k];
        }
    } else {
        const u32x4_a2 u = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(row) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = from16((uint16_t)(u[k] & 0xFFFFu), DT == BF16);
            v[2 * k + 1] = from16((uint16_t)(u[k] >> 16), DT == BF16);
        }
    }
}

// elements i .. i + 8 of a row of V, `past` past its end
template <int DT>
__device__ __forceinline__ void load_group(const void* row, int i, int V, float past, float (&v)[8]) {
    if (i + 8 <= V) {
        load_whole_group<DT>(row, i, v);
    } else {                                                 // eight loads at once here too, and none wholly past the end
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = past;
        if (i < V) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = load_elem(row, DT, (size_t)min(i + k, V - 1));
                if (i + k < V) v[k] = f;
            }
        }
    }
}

// f's order among all floats as an unsigned integer, zeros of both signs alike, NaN above everything; above the complemented
// index, so that the largest key is the largest value at its lowest index
__device__ __forceinline__ unsigned long long key32(float f, int idx) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.0f);
    const uint32_t o = f != f ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((unsigned long long)o << 32) | (uint32_t)~(uint32_t)idx;
}

template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ float dpp_of(float v) {           // -inf where the row mask excludes the lane
    return __builtin_bit_cast(float, dpp_u32<CTRL, ROW_MASK>(__builtin_bit_cast(uint32_t, v), 0xFF800000u));
}
// the wave's maximum, in every lane; a NaN is passed over
__device__ __forceinline__ float wave_max_f32(float v) {
    v = fmaxf(v, dpp_of<0xB1>(v));
    v = fmaxf(v, dpp_of<0x4E>(v));
    v = fmaxf(v, dpp_of<0x141>(v));
    v = fmaxf(v, dpp_of<0x140>(v));
    v = fmaxf(v, dpp_of<0x142, 0xA>(v));
    v = fmaxf(v, dpp_of<0x143, 0xC>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, v), 63));
}
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)k, m), hi = (uint32_t)__shfl_xor((int)(k >> 32), m);
        const unsigned long long o = ((unsigned long long)hi << 32) | lo;
        k = o > k ? o : k;
    }
    return k;
}

// Below this temperature a request is greedy
constexpr float GREEDY_BELOW = 1e-5f;

// 1 / temperature (1 for a greedy request, whose log-probabilities are those of temperature 1). An infinite temperature
// keeps a factor above zero: a masked logit's -inf stays one.
__device__ __forceinline__ bool is_greedy(float temperature) { return !(temperature >= GREEDY_BELOW); }
__device__ __forceinline__ double inv_temperature(float temperature) {
    if (is_greedy(temperature)) return 1.0;
    const double inv = 1.0 / (double)temperature;
    return inv > 1e-30 ? inv : 1e-30;
}
// log2(e) / temperature as two floats: one float's rounding would shift every exponent of a row the same way. Both are
// positive (hi rounded down, lo above zero), so a masked logit's -inf stays -inf in either product.
__device__ __forceinline__ void exponent_factor(double inv_t, float& hi, float& lo) {
    const double c = inv_t * 1.4426950408889634;
    hi = (float)c;
    if ((double)hi > c) hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, hi) - 1u);
    lo = fmaxf((float)(c - (double)hi), 1e-37f);
}
__device__ __forceinline__ float exp_scaled(float d, float hi, float lo) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi, d * lo));
}

}  // namespace esp
