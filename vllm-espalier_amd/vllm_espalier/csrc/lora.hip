// Low-rank adapters of many requests beside a shared projection, on gfx950:
//   out[m, n] = y[m, n] + sum_{j < r} t[m, j] B[a][n][j],   t[m, j] = scale[a][s] * sum_k x[m, k] A[a][s][j][k]
// for row m of adapter a = rows[m] and column n of the layer's matrix s (r = ranks[a][s]); rows of no adapter keep y.
//
// Two launches: the rows' products with A (fp32, in K splits), then those with B and the sum. Both take tiles of 16
// consecutive rows and, inside a tile, one adapter after the other (the tile's distinct ones, found by a few lane
// exchanges): a matrix instruction's columns are the rows, so each row keeps the column that its own adapter made and no
// sorting or grouping launch is needed, whatever the order of the rows. Where a batch is small its distinct adapters are
// spread over workgroups.
//
// t keeps 32 bits between the launches and enters the second product as a 16-bit high part and the 16-bit rest, side by
// side in one instruction's k (16 ranks of each), so nothing of it is lost but the rest's own rounding (2^-17 for bf16). fp16's narrow
// range is kept out of it: a row of t is first scaled by a power of two to below 2.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "norm.hpp"

namespace esp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int LORA_ROWS = 16;                  // rows a tile
constexpr int LORA_CHUNK = 512;               // k a partial sum of t: t is the chunks' sums added in order
constexpr int LORA_MAX_SHARDS = 4;
constexpr int LORA_MAX_RANK = 256;

struct LoraArgs {
    const uint16_t* x;
    int64_t x_stride;
    const uint16_t* y;
    int64_t y_stride;
    uint16_t* out;
    int64_t out_stride;
    const int32_t *rows, *ranks;
    const float* scales;
    const uint16_t *a, *b;
    float* t;                                  // [SK][T][S * R]
    int T, K, S, N, R, slots, SK, spread;      // spread: workgroups that share a row tile's adapters
    int n_cols[LORA_MAX_SHARDS], tiles0[LORA_MAX_SHARDS + 1];   // a matrix's columns, and its first 64-column tile
};

// D += P Q^T over 32 k, P's 16 rows and Q's 16 rows 8 k a lane: lane l holds row l & 15, k of its group l >> 4; it gets
// D[4 * (l >> 4) + i][l & 15]
template <int DT>
__device__ __forceinline__ f32x4 mfma32(uint4 p, uint4 q, f32x4 acc) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), acc, 0, 0,
                                                      0);
}

// 8 elements at an 8-byte aligned address (16 with wide)
__device__ __forceinline__ uint4 load8(const uint16_t* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + 4);
    return make_uint4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ bool wide_rows(const void* p, int64_t stride) {
    return (uintptr_t)p % 16 == 0 && stride % 8 == 0;
}

// The adapter of row row0 + (lane & 15), -1 for none or no such row; leaders: the lanes (0 to 15) that are the first of
// their adapter in the tile
__device__ __forceinline__ int tile_adapter(const LoraArgs& a, int row0, uint32_t& leaders) {
    const int lane = threadIdx.x & 63, m = lane & 15;
    int id = -1;
    if (row0 + m < a.T) {
        id = a.rows[row0 + m];
        if (id < 0 || id >= a.slots) id = -1;
    }
    bool first = id >= 0;
#pragma unroll
    for (int k = 0; k < 15; ++k) {
        const int o = __builtin_amdgcn_readlane(id, k);
        if (k < m && o == id) first = false;
    }
    leaders = (uint32_t)__ballot(first && lane < 16);
    return id;
}

// t of a row tile, 16 ranks (blockIdx.y: matrix and rank tile) and one chunk of 512 k (blockIdx.z): a wave 128 k of it, the
// four waves' sums added in order
template <int DT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraArgs a) {
    __shared__ f32x4 part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const int row0 = (int)(blockIdx.x / a.spread) * LORA_ROWS, d = blockIdx.x % a.spread;
    const int s = blockIdx.y / (a.R / 16), j0 = (int)(blockIdx.y % (a.R / 16)) * 16;
    uint32_t leaders;
    const int id = tile_adapter(a, row0, leaders);
    const bool wide = wide_rows(a.x, a.x_stride);
    const uint16_t* xr = a.x + (int64_t)min(row0 + m, a.T - 1) * a.x_stride + 16 * g;
    const int k0 = (int)blockIdx.z * LORA_CHUNK + wave * (LORA_CHUNK / 4);
    for (int nth = 0; leaders; ++nth) {
        const int who = __builtin_amdgcn_readlane(id, __builtin_ctz(leaders));
        leaders &= leaders - 1;
        if (nth % a.spread != d || j0 >= a.ranks[who * a.S + s]) continue;
        const uint16_t* ar = a.a + (((size_t)who * a.S + s) * a.R + j0 + m) * a.K + 16 * g;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < LORA_CHUNK / 4 / 64; ++st) {
            const int k = k0 + 64 * st;
            uint4 p[2], q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) p[h] = q[h] = make_uint4(0u, 0u, 0u, 0u);
            if (k + 16 * g < a.K) {                          // K is a multiple of 16: a lane's 16 k are in or out
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    p[h] = *reinterpret_cast<const uint4*>(ar + k + 8 * h);
                    q[h] = load8(xr + k + 8 * h, wide);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma32<DT>(p[h], q[h], acc);
        }
        part[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && id == who) {
            const f32x4 sum = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
            *reinterpret_cast<f32x4*>(a.t + (((size_t)blockIdx.z * a.T + row0 + m) * a.S + s) * a.R + j0 + 4 * g) = sum;
        }
        __syncthreads();                                     // part is written again
    }
}

__device__ __forceinline__ f32x4 lora_t4(const LoraArgs& a, const float* t, float scale) {
    f32x4 v = *reinterpret_cast<const f32x4*>(t);
    for (int z = 1; z < a.SK; ++z) v += *reinterpret_cast<const f32x4*>(t + (size_t)z * a.T * a.S * a.R);
    return v * scale;
}

// 8 floats as the 16-bit high parts (low: what they leave)
template <int DT>
__device__ __forceinline__ uint4 split8(const float (&v)[8], bool low) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint16_t h[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float f = v[2 * k + e];
            h[e] = to16(f, DT == BF16);
            if (low) {
                const float hi = from16(h[e], DT == BF16), rest = f - hi;
                h[e] = to16(rest == rest && fabsf(rest) < INFINITY ? rest : 0.f, DT == BF16);
            }
        }
        w[k] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 64 columns of one matrix (a wave each) of a row tile: the products of t with B, added to y. Rows of B enter in the order
// that gives a lane 16 columns in a row of its row of y: instruction q's row 4 c + i is column 16 c + 4 q + i.
template <int DT>
__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraArgs a) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int row0 = (int)(blockIdx.x / a.spread) * LORA_ROWS, d = blockIdx.x % a.spread;
    const int ct = (int)blockIdx.y * 4 + (int)(threadIdx.x >> 6);
    if (ct >= a.tiles0[a.S]) return;
    int s = 0, c0 = 0;                                       // c0: the matrix's first column in y
    while (ct >= a.tiles0[s + 1]) c0 += a.n_cols[s++];
    const int n0 = (ct - a.tiles0[s]) * 64;
    uint32_t leaders;
    const int id = tile_adapter(a, row0, leaders);
    const float* tr = a.t + ((size_t)min(row0 + m, a.T - 1) * a.S + s) * a.R + 8 * (g & 1);
    bool mine = false;
    f32x4 sum[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] = {0.f, 0.f, 0.f, 0.f};
    const int br = n0 + 16 * (m >> 2) + (m & 3);             // this lane's row of B for q = 0
    const bool b_in = n0 + 16 * (m >> 2) < a.n_cols[s];      // columns are multiples of 16
    for (int nth = 0; leaders; ++nth) {
        const int who = __builtin_amdgcn_readlane(id, __builtin_ctz(leaders));
        leaders &= leaders - 1;
        if (nth % a.spread != d) continue;
        const int r = min(a.ranks[who * a.S + s], a.R);
        const float scale = a.scales[who * a.S + s];
        int e = 0;
        if constexpr (DT == F16) {
            float top = 0.f;
            for (int js = 0; js < r; js += 16) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = lora_t4(a, tr + js + 4 * h, scale);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (js + 8 * (g & 1) + 4 * h + i < r) top = fmaxf(top, fabsf(v[i]));
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            if (top > 0.f && top < INFINITY) e = __builtin_amdgcn_frexp_expf(top);
        }
        f32x4 acc[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] = {0.f, 0.f, 0.f, 0.f};
        const uint16_t* bp = a.b + ((size_t)who * a.N + c0 + br) * a.R + 8 * (g & 1);
        for (int js = 0; js < r; js += 16) {
            const int left = r - js - 8 * (g & 1);           // ranks of this lane's 8 that the adapter has
            float v[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 t4 = lora_t4(a, tr + js + 4 * h, scale);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * h + i] = 4 * h + i < left ? (DT == F16 ? ldexpf(t4[i], -e) : t4[i]) : 0.f;
            }
            const uint4 tq = split8<DT>(v, g >= 2);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint4 bq = make_uint4(0u, 0u, 0u, 0u);
                if (b_in) bq = *reinterpret_cast<const uint4*>(bp + (size_t)4 * q * a.R + js);
                if (left < 8) {                              // what lies past the rank is not used, whatever it holds
                    uint32_t w[4] = {bq.x, bq.y, bq.z, bq.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (2 * i >= left) w[i] = 0u;
                        else if (2 * i + 1 >= left) w[i] &= 0xFFFFu;
                    }
                    bq = make_uint4(w[0], w[1], w[2], w[3]);
                }
                acc[q] = mfma32<DT>(bq, tq, acc[q]);
            }
        }
        if (id == who) {
            mine = true;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[q][i] = DT == F16 ? ldexpf(acc[q][i], e) : acc[q][i];
        }
    }
    const int row = row0 + m, n = n0 + 16 * g;
    if (id < 0) mine = d == 0 && a.out != a.y;               // no adapter: y as it is
    if (!mine || row >= a.T || n >= a.n_cols[s]) return;
    const uint16_t* yp = a.y + (int64_t)row * a.y_stride + c0 + n;
    uint16_t* op = a.out + (int64_t)row * a.out_stride + c0 + n;
    const bool wide_y = wide_rows(a.y, a.y_stride), wide_o = wide_rows(a.out, a.out_stride);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint4 u = load8(yp + 8 * h, wide_y);
        if (id >= 0) {
            float v[8];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint16_t bits = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                v[i] = from16(bits, DT == BF16) + sum[2 * h + (i >> 2)][i & 3];
            }
            u = pack8_16(v, DT == BF16);
        }
        if (wide_o) {
            *reinterpret_cast<uint4*>(op + 8 * h) = u;
        } else {
            *reinterpret_cast<uint2*>(op + 8 * h) = make_uint2(u.x, u.y);
            *reinterpret_cast<uint2*>(op + 8 * h + 4) = make_uint2(u.z, u.w);
        }
    }
}

constexpr int LORA_SPREAD_ROWS = 256;          // up to this many rows a tile's adapters run in workgroups of their own

template <int DT>
int lora_launch(const LoraArgs& a, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.T + LORA_ROWS - 1) / LORA_ROWS) * a.spread;
    lora_shrink_kernel<DT><<<dim3(tiles, (unsigned)(a.S * (a.R / 16)), (unsigned)a.SK), 256, 0, st>>>(a);
    lora_expand_kernel<DT><<<dim3(tiles, (unsigned)((a.tiles0[a.S] + 3) / 4)), 256, 0, st>>>(a);
    return esp_host::launch_check("lora");
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

static int64_t lora_splits(int64_t K) { return (K + LORA_CHUNK - 1) / LORA_CHUNK; }

extern "C" int64_t esp_lora_scratch(int64_t T, int64_t K, int64_t n_shards, int64_t R) {
    if (T <= 0 || K <= 0 || n_shards <= 0 || R <= 0) return 0;
    return lora_splits(K) * T * n_shards * R;
}

extern "C" int esp_lora(const void* x, int64_t x_stride, const void* y, int64_t y_stride, void* out, int64_t out_stride,
                        const int32_t* rows, int64_t T, int64_t K, int64_t n_shards, const int64_t* n_cols, const void* A,
                        const void* B, const int32_t* ranks, const float* scales, int64_t slots, int64_t R, int dtype,
                        float* scratch, int64_t scratch_numel, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16, "lora: dtype must be bf16 or fp16");
    ESP_REQUIRE(T >= 0 && T < (1 << 24), "lora: at most 2^24 - 1 rows");
    ESP_REQUIRE(n_shards >= 1 && n_shards <= LORA_MAX_SHARDS, "lora: 1 to %d matrices", LORA_MAX_SHARDS);
    ESP_REQUIRE(K > 0 && K % 16 == 0 && K <= (1 << 20), "lora: K must be a positive multiple of 16, at most 2^20");
    ESP_REQUIRE(R > 0 && R % 16 == 0 && R <= LORA_MAX_RANK, "lora: the rank rows must be a multiple of 16, at most %d",
                LORA_MAX_RANK);
    ESP_REQUIRE(slots >= 1 && slots <= (1 << 20), "lora: 1 to 2^20 adapters");
    ESP_REQUIRE(n_cols, "lora: null pointer");
    LoraArgs a;
    int64_t N = 0;
    a.tiles0[0] = 0;
    for (int64_t s = 0; s < n_shards; ++s) {
        ESP_REQUIRE(n_cols[s] > 0 && n_cols[s] % 16 == 0 && n_cols[s] <= (1 << 21),
                    "lora: columns must be positive multiples of 16, at most 2^21 a matrix");
        a.n_cols[s] = (int)n_cols[s];
        a.tiles0[s + 1] = a.tiles0[s] + (int)((n_cols[s] + 63) / 64);
        N += n_cols[s];
    }
    if (T == 0) return esp_host::ok();
    ESP_REQUIRE(x && y && out && rows && A && B && ranks && scales && scratch, "lora: null pointer");
    ESP_REQUIRE(T == 1 || (x_stride >= K && y_stride >= N && out_stride >= N), "lora: rows overlap");
    ESP_REQUIRE(out != y || T == 1 || out_stride == y_stride, "lora: in place, out must have y's row stride");
    ESP_REQUIRE(((uintptr_t)x | (uintptr_t)y | (uintptr_t)out) % 8 == 0 &&
                    (T == 1 || (x_stride % 4 == 0 && y_stride % 4 == 0 && out_stride % 4 == 0)),
                "lora: x, y and out must be 8-byte aligned with row strides a multiple of 4 elements");
    ESP_REQUIRE(((uintptr_t)A | (uintptr_t)B | (uintptr_t)scratch) % 16 == 0,
                "lora: the adapters and the scratch must be 16-byte aligned");
    ESP_REQUIRE(scratch_numel >= esp_lora_scratch(T, K, n_shards, R), "lora: the scratch needs esp_lora_scratch floats");
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.y = static_cast<const uint16_t*>(y);
    a.y_stride = y_stride;
    a.out = static_cast<uint16_t*>(out);
    a.out_stride = out_stride;
    a.rows = rows;
    a.ranks = ranks;
    a.scales = scales;
    a.a = static_cast<const uint16_t*>(A);
    a.b = static_cast<const uint16_t*>(B);
    a.t = scratch;
    a.T = (int)T;
    a.K = (int)K;
    a.S = (int)n_shards;
    a.N = (int)N;
    a.R = (int)R;
    a.slots = (int)slots;
    a.SK = (int)lora_splits(K);
    a.spread = T > LORA_SPREAD_ROWS ? 1 : (int)(T < LORA_ROWS ? T : LORA_ROWS);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == ESP_BF16 ? lora_launch<BF16>(a, st) : lora_launch<F16>(a, st);
}
