// The norms after and before a block, with the block's gate and the residual scale, on gfx950:
//   d = d1 + d2,  u = (d * inv(d)) * w_post,  z = h + (scale * f(g)) * u,  h_out = z in the model dtype,
//   out = (h_out * inv(h_out)) * w_pre,       inv(v) = 1 / sqrt(mean(v^2) + eps)
// add_rmsnorm (step.hip) is its form without a norm behind the block; with one delta, no gate and scale 1 the two give the
// same bits.
//
// Every sum runs in norm.hpp's order (lane slices, DPP inside a wave, the four waves' sums in index order), in fp32, so a
// row's bits depend on that row alone.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "norm.hpp"

namespace esp {

enum GateKind : int { GATE_NONE = 0, GATE_ROW = 1, GATE_ELEMENT = 2 };    // none; one value a row; one an element

struct SandwichArgs {
    const uint16_t *h, *d1, *d2, *w_post, *gate, *w_pre;
    int64_t gate_row;              // elements between two rows' gates (0: all rows share them)
    uint16_t *h_out, *out;
    int D, gate_kind, sigmoid, bf;
    float scale, eps;
};

__device__ __forceinline__ void unpack8_16(uint4 u, bool bf, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = from16((uint16_t)(w[k] & 0xFFFFu), bf);
        v[2 * k + 1] = from16((uint16_t)(w[k] >> 16), bf);
    }
}

// the factor of a gate value: itself, or its sigmoid (1 / (1 + inf) = 0 far below zero)
__device__ __forceinline__ float gate_of(float g, int sigmoid) { return sigmoid ? 1.0f / (1.0f + __expf(-g)) : g; }

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
template <bool NT>
__device__ __forceinline__ void store16(uint16_t* p, uint4 v) {
    const u32x4_t u = {v.x, v.y, v.z, v.w};
    if constexpr (NT) __builtin_nontemporal_store(u, reinterpret_cast<u32x4_t*>(p));
    else *reinterpret_cast<u32x4_t*>(p) = u;
}

// One workgroup of 256 a row; thread t holds elements (c * 256 + t) * 8 .. + 8. Bound by memory from a few hundred rows on (8192 x
// 4096 with a gate an element, 336 MB: 64 us, 5.2 TB/s; a copy of such a size reaches 4.7 to 5.5), below by the launch and its chain
// of round trips: each operand's load is waited for before the next one's begins, d1, d2, w_post, gate, h and w_pre, three to six for a
// chunk of 2048 and, chunk after chunk, up to four times as many for 8192. One row, graph replays: 2048 with one delta and a channel
// gate 3.7 us, with two deltas and a gate an element 4.1; 8192 8.3 and 9.7 (add_rmsnorm, which issues a row's loads together, 3.3 and
// 6.7). NT: outputs stored past the L2, see the launch.
template <bool NT>
__global__ __launch_bounds__(256) void sandwich_rmsnorm_kernel(const SandwichArgs a) {
    __shared__ float part[2][4];
    const int t = threadIdx.x, wave = t >> 6;
    const size_t o = (size_t)blockIdx.x * a.D;
    const bool bf = a.bf;
    float u[NORM_CHUNKS][8];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NORM_CHUNKS; ++c) {
        const int i = (c * 256 + t) * 8;
        if (i < a.D) {
            unpack8_16(*reinterpret_cast<const uint4*>(a.d1 + o + i), bf, u[c]);
            if (a.d2) {
                float b[8];
                unpack8_16(*reinterpret_cast<const uint4*>(a.d2 + o + i), bf, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[c][j] += b[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += u[c][j] * u[c][j];
        }
    }
    if (a.w_post) {
        ss = wave_sum_f32(ss);
        if ((t & 63) == 0) part[0][wave] = ss;
        __syncthreads();
        const float inv = norm_inv(part[0], a.D, a.eps);
#pragma unroll
        for (int c = 0; c < NORM_CHUNKS; ++c) {
            const int i = (c * 256 + t) * 8;
            if (i < a.D) {
                float w[8];
                unpack8_16(*reinterpret_cast<const uint4*>(a.w_post + i), bf, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[c][j] = (u[c][j] * inv) * w[j];
            }
        }
    }
    float row_factor = a.scale;
    if (a.gate_kind == GATE_ROW) row_factor *= gate_of(from16(a.gate[(int64_t)blockIdx.x * a.gate_row], bf), a.sigmoid);
    uint4 zq[NORM_CHUNKS];
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < NORM_CHUNKS; ++c) {
        const int i = (c * 256 + t) * 8;
        if (i < a.D) {
            float f[8], z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = row_factor;
            if (a.gate_kind == GATE_ELEMENT) {
                float g[8];
                unpack8_16(*reinterpret_cast<const uint4*>(a.gate + (int64_t)blockIdx.x * a.gate_row + i), bf, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] *= gate_of(g[j], a.sigmoid);
            }
            unpack8_16(*reinterpret_cast<const uint4*>(a.h + o + i), bf, z);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = z[j] + f[j] * u[c][j];
            zq[c] = pack8_16(z, bf);
            unpack8_16(zq[c], bf, z);                     // the second norm is that of the residual as it is stored
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += z[j] * z[j];
        }
    }
    ss = wave_sum_f32(ss);
    if ((t & 63) == 0) part[1][wave] = ss;
    __syncthreads();
    const float inv = norm_inv(part[1], a.D, a.eps);
#pragma unroll
    for (int c = 0; c < NORM_CHUNKS; ++c) {
        const int i = (c * 256 + t) * 8;
        if (i < a.D) {
            store16<NT>(a.h_out + o + i, zq[c]);
            store16<NT>(a.out + o + i, norm_scale8(zq[c], *reinterpret_cast<const uint4*>(a.w_pre + i), inv, bf));
        }
    }
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

extern "C" int esp_sandwich_rmsnorm(const void* h, const void* d1, const void* d2, const void* w_post, const void* gate,
                                    int64_t gate_row, int64_t gate_col, int gate_sigmoid, double scale, const void* w_pre,
                                    void* h_out, void* out, int64_t T, int64_t D, double eps, int dtype, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16, "sandwich_rmsnorm: dtype must be bf16 or fp16");
    ESP_REQUIRE(D > 0 && D % 8 == 0 && D <= NORM_MAX_D, "sandwich_rmsnorm: D must be a positive multiple of 8, at most %d",
                NORM_MAX_D);
    ESP_REQUIRE(T < (1 << 24), "sandwich_rmsnorm: at most 2^24 - 1 rows");
    if (T <= 0) return esp_host::ok();                       // (no rows have no address)
    ESP_REQUIRE(h && d1 && w_pre && h_out && out, "sandwich_rmsnorm: null pointer");
    ESP_REQUIRE(((uintptr_t)h | (uintptr_t)d1 | (uintptr_t)d2 | (uintptr_t)w_post | (uintptr_t)w_pre | (uintptr_t)h_out |
                 (uintptr_t)out) % 16 == 0, "sandwich_rmsnorm: every tensor must be 16-byte aligned");
    ESP_REQUIRE(gate_row >= 0 && (gate_col == 0 || gate_col == 1),
                "sandwich_rmsnorm: a gate has a row stride of at least 0 and a column stride of 0 (one a row) or 1");
    ESP_REQUIRE(!gate || (gate_col == 0 ? (uintptr_t)gate % 2 == 0 : ((uintptr_t)gate % 16 == 0 && gate_row % 8 == 0)),
                "sandwich_rmsnorm: a gate an element must have 16-byte aligned rows");
    // A workgroup has read all of its row but w_pre when it stores it: an output may lie where its own row's inputs do
    const auto meet = [](const void* p, int64_t n, const void* q, int64_t m) { return q && esp_host::rows_meet(p, 0, n, q, 0, m, 1); };
    for (const void* o : {h_out, out}) {
        for (const void* i : {h, d1, d2})
            ESP_REQUIRE(i == o || T == 1 || !meet(o, T * D * 2, i, T * D * 2),
                        "sandwich_rmsnorm: an output overlaps other rows of an input");
        ESP_REQUIRE(!meet(o, T * D * 2, w_post, D * 2) && !meet(o, T * D * 2, w_pre, D * 2),
                    "sandwich_rmsnorm: an output overlaps a weight");
        const int64_t g = gate_col ? D * 2 : 2;
        const bool own_row = gate_row == D && (uintptr_t)gate - (uintptr_t)o <= (uintptr_t)(D * 2 - g);
        ESP_REQUIRE(!gate || T == 1 || own_row ||
                        !(gate_row ? esp_host::rows_meet(o, D * 2, D * 2, gate, gate_row * 2, g, T) : meet(o, T * D * 2, gate, g)),
                    "sandwich_rmsnorm: an output overlaps the gate");
    }
    ESP_REQUIRE(!meet(h_out, T * D * 2, out, T * D * 2), "sandwich_rmsnorm: the two outputs overlap");
    SandwichArgs a;
    a.h = static_cast<const uint16_t*>(h);
    a.d1 = static_cast<const uint16_t*>(d1);
    a.d2 = static_cast<const uint16_t*>(d2);
    a.w_post = static_cast<const uint16_t*>(w_post);
    a.gate = static_cast<const uint16_t*>(gate);
    a.w_pre = static_cast<const uint16_t*>(w_pre);
    a.gate_row = gate_row;
    a.h_out = static_cast<uint16_t*>(h_out);
    a.out = static_cast<uint16_t*>(out);
    a.D = (int)D;
    a.gate_kind = !gate ? GATE_NONE : gate_col ? GATE_ELEMENT : GATE_ROW;
    a.sigmoid = gate_sigmoid;
    a.bf = dtype == ESP_BF16;
    a.scale = (float)scale;
    a.eps = (float)eps;
    // Outputs past an XCD's L2 (4 MiB) are stored past it, and push out less of what the launch reads: 1531 x 4096 11.7 -> 8.3 us,
    // 8192 x 4096 67.5 -> 64.4; smaller ones, where it makes no difference, stay for the next launch to read
    const auto kernel = T * D * 2 >= 4 << 20 ? sandwich_rmsnorm_kernel<true> : sandwich_rmsnorm_kernel<false>;
    kernel<<<(unsigned)T, 256, 0, (hipStream_t)stream>>>(a);
    return esp_host::launch_check("sandwich_rmsnorm");
}
