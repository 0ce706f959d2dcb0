// Low-rank adapters of many requests beside a shared projection, on gfx950:
//   out[m, n] = y[m, n] + sum_{j < r} t[m, j] B[a][n][j],   t[m, j] = scale[a][s] * sum_k x[m, k] A[a][s][j][k]
// for row m of adapter a = rows[m] and column n of the layer's matrix s (r = ranks[a][s]); rows of no adapter keep y.
//
// Two launches: the rows' products with A, then those with B and the sum; one for a few rows and ranks. All take tiles of 16 to 64
// consecutive rows and, inside a tile, one adapter after the other (the tile's distinct ones, found by ballots): the rows are one
// side of a matrix instruction, so each row keeps what its own adapter made of it and no sorting or grouping launch is needed,
// whatever the order of the rows. Where a batch is small its distinct adapters are spread over workgroups.
//
// The adapters are laid out as the instructions read them (LoraArgs): a wave's load is one KiB in a row. The quarter of a wave
// that a CU looks up at once then meets two lines; 16 rows of a plain matrix are 16 lines, and came in at 10 bytes a clock.
//
// t is summed in fp32 and enters the second product as a 16-bit high part and the 16-bit rest, side by side in one instruction's
// k (16 ranks of each), so nothing of it is lost but the rest's own rounding (2^-17 for bf16). fp16's narrow range is kept out of
// it: 16 ranks of a row are first scaled by a power of two to below 1, and their products scaled back.
//
// The order of t's sum is fixed: K in 16 runs of whole 32-k units, a run in its units' order, the runs four by four in order, and
// of the four fours the first two and the last two; so a row's bits depend on that row and its adapter alone.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int LORA_RUNS = 16;                  // runs of k that t is summed in
constexpr int LORA_MAX_SHARDS = 4;
constexpr int LORA_MAX_RANK = 256;
constexpr int LORA_COLS = 128;                 // columns a wave of the second product

struct LoraArgs {
    const uint16_t* x;
    int64_t x_stride;
    const uint16_t* y;
    int64_t y_stride;
    uint16_t* out;
    int64_t out_stride;
    const int32_t *rows, *ranks;
    const float* scales;
    const uint4* a;                            // [slots][S][R / 16][units][64]: lane l of a unit rank l % 16, k 8 (l / 16) .. + 8
    const uint4* b;                            // [slots][col_tiles][R / 16][8][32]: lane l of instruction c column 8 (l % 16) + c,
                                               // ranks 8 (l / 16) .. + 8
    float* part;                               // few rows: [4][row tiles][S * R / 16][16 rows][16 ranks], t's sums of four runs
    uint4* t;                                  // many: [row tiles][S * R / 16][64], finished: lane l row l % 16, ranks 8 (l / 16
                                               // % 2) .. + 8, the high parts (l < 32) or the rests
    int* e;                                    // [row tiles][S * R / 16][16]: fp16's exponents
    int T, K, S, R, slots, spread;             // spread: workgroups that share a row tile's adapters (few rows)
    int n_cols[LORA_MAX_SHARDS], tiles0[LORA_MAX_SHARDS + 1];   // a matrix's columns, and its first tile of LORA_COLS
};

// D += P Q^T over 32 k, P's 16 rows and Q's 16 rows 8 k a lane: lane l holds row l % 16, k of its group l / 16; it gets
// D[4 * (l / 16) + i][l % 16]
template <int DT>
__device__ __forceinline__ f32x4 mfma32(uint4 p, uint4 q, f32x4 acc) {
    if constexpr (DT == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), acc,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), acc, 0, 0,
                                                      0);
}

// 8 elements at an 8-byte aligned address: one 16-byte access, which the hardware asks no more of
typedef uint32_t u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));
__device__ __forceinline__ uint4 load8(const uint16_t* p) {
    const u32x4_a8 v = *reinterpret_cast<const u32x4_a8*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store8(uint16_t* p, uint4 v) {
    *reinterpret_cast<u32x4_a8*>(p) = u32x4_a8{v.x, v.y, v.z, v.w};
}

// past the L2's present contents: 42 MB of a prompt's outputs pushed out what its other workgroups read again (the expanding
// launch of 4096 rows through 2048 -> 5120 25.9 -> 21.8 us, and the one before it ran 8 % faster)
__device__ __forceinline__ void store8_nt(uint16_t* p, uint4 v) {
    __builtin_nontemporal_store(u32x4_a8{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_a8*>(p));
}

// a value that every lane of the wave reads, through the scalar cache (nothing writes it while the kernel runs)
template <typename T>
__device__ __forceinline__ T load_uniform(const T* p) {
    return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// The distinct adapters of a tile of 16 * MG rows (a lane each), one after the other: next() gives an adapter and the mask of
// its rows, those of `rest` that are left; an id outside [0, slots) is none
template <int MG>
struct TileAdapters {
    int id;
    uint64_t rest;
    __device__ __forceinline__ TileAdapters(const LoraArgs& a, int row0) {
        const int lane = threadIdx.x & 63;
        id = -1;
        if (lane < 16 * MG && row0 + lane < a.T) id = a.rows[row0 + lane];
        if (id >= a.slots) id = -1;
        rest = __ballot(id >= 0);
    }
    __device__ __forceinline__ int next(uint64_t& mask) {
        const int who = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
        mask = __ballot(id == who) & rest;
        rest &= ~mask;
        return who;
    }
};

__device__ __forceinline__ int lora_rank(const LoraArgs& a, int who, int s) {
    return min(load_uniform(a.ranks + (int64_t)who * a.S + s), a.R);
}

// 4 floats as their 16-bit high parts (hi) and what those leave (lo)
template <int DT>
__device__ __forceinline__ void split4(const f32x4& v, uint2& hi, uint2& lo) {
    uint16_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = to16(v[i], DT == BF16);
        const float rest = v[i] - from16(h[i], DT == BF16);
        l[i] = to16(fabsf(rest) < INFINITY ? rest : 0.f, DT == BF16);    // an infinity's or NaN's rest is nothing
    }
    hi = make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
    lo = make_uint2((uint32_t)l[0] | ((uint32_t)l[1] << 16), (uint32_t)l[2] | ((uint32_t)l[3] << 16));
}

// 16 bytes a lane of a KiB that starts where all lanes have it alike, its address in scalar registers
__device__ __forceinline__ uint4 load_kib(const char* p, int lane) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32));
    typedef const __attribute__((address_space(1))) char* global;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 r = *(const __attribute__((address_space(1))) u32x4*)((global)(uintptr_t)((hi << 32) | lo) + (uint32_t)(lane * 16));
    return make_uint4(r.x, r.y, r.z, r.w);
}

// Item of workgroup `block` of n: workgroups go to the eight XCDs in turn, and each XCD takes a run of consecutive items (row tiles,
// and the shares or column tiles of each), so that one tile's rows and the adapters of few requests pass through its L2
__device__ __forceinline__ int xcd_tile(int block, int n) {
    const int per = n / 8, more = n % 8, xcd = block % 8;
    return xcd * per + min(xcd, more) + block / 8;
}

// The power of two to scale 16 ranks of a row by whose largest magnitude is top
__device__ __forceinline__ int lora_exponent(float top) {
    return top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
}

// ------------------------------------------------------------------------------------------------------------------
// The first product, few rows: the sums of runs 4 z .. 4 z + 3 for 16 rows and LORA_FEW tiles of 16 ranks, a wave a run, in fp32.
// blockIdx.x the row tile and, spread, its adapters; blockIdx.y the matrix and rank tiles, blockIdx.z the runs: a batch's adapters
// are read once and come in through many CUs. Bound by its three dependent round trips (rows, ranks, operands): 32 rows of 24
// adapters, ranks up to 64 of 4096, 5.2 us for 5.3 MB; 509 rows of 3 adapters of rank 32 of 2048 5.2 us.
// ------------------------------------------------------------------------------------------------------------------
constexpr int LORA_FEW = 2;                    // rank tiles whose loads are all in flight at once

template <int DT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraArgs a) {
    __shared__ f32x4 part[4][LORA_FEW][64];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int tile_at = blockIdx.x / a.spread, d = blockIdx.x % a.spread;
    const int rt = a.R / 16, of = (rt + LORA_FEW - 1) / LORA_FEW, s = blockIdx.y / of, j0 = blockIdx.y % of * LORA_FEW;
    const int units = (a.K + 31) / 32, run = (units + LORA_RUNS - 1) / LORA_RUNS;
    const int u0 = (4 * (int)blockIdx.z + wave) * run, u1 = min(units, u0 + run);
    TileAdapters<1> tile(a, 16 * tile_at);
    for (int nth = 0; tile.rest; nth = nth + 1 == a.spread ? 0 : nth + 1) {
        uint64_t mask;
        const int who = tile.next(mask);
        if (nth != d) continue;
        const int n = (lora_rank(a, who, s) + 15) / 16 - j0;
        if (n <= 0) continue;
        const char* ab = reinterpret_cast<const char*>(a.a + (((int64_t)who * a.S + s) * rt + j0) * units * 64);
        // rows of other adapters read the first of this one's instead: no line comes in for them
        const bool mine = (mask >> m) & 1;
        const int mr = mine ? m : __builtin_ctzll(mask);
        const uint16_t* xp = a.x + (int64_t)(16 * tile_at + mr) * a.x_stride + 8 * g;
        f32x4 acc[LORA_FEW];
#pragma unroll
        for (int j = 0; j < LORA_FEW; ++j) acc[j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int u = u0; u < u1; u += 4) {
            uint4 x[4], p[LORA_FEW][4];
#pragma unroll
            for (int j = 0; j < LORA_FEW; ++j)               // units past the run's: its last one again, tiles past the adapter's:
#pragma unroll
                for (int i = 0; i < 4; ++i)                  // its last one; not used
                    p[j][i] = *reinterpret_cast<const uint4*>(ab + ((int64_t)min(j, n - 1) * units + min(u + i, u1 - 1)) * 1024 +
                                                              lane * 16u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 32 * min(u + i, u1 - 1);
                x[i] = load8(xp + min(k, a.K - 8 - 8 * g));
                if (k + 8 * g >= a.K) x[i] = make_uint4(0u, 0u, 0u, 0u);
            }
            __builtin_amdgcn_sched_barrier(0);               // every load before the first use
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (u + i < u1)
#pragma unroll
                    for (int j = 0; j < LORA_FEW; ++j) acc[j] = mfma32<DT>(p[j][i], x[i], acc[j]);
        }
#pragma unroll
        for (int j = 0; j < LORA_FEW; ++j) part[wave][j][lane] = acc[j];
        __syncthreads();
        if (wave < min(n, LORA_FEW) && mine)
            *reinterpret_cast<f32x4*>(a.part + (((((int64_t)blockIdx.z * ((a.T + 15) / 16) + tile_at) * a.S + s) * rt + j0 + wave) *
                                                    16 + m) * 16 + 4 * g) =
                ((part[0][wave][lane] + part[1][wave][lane]) + part[2][wave][lane]) + part[3][wave][lane];
        if (tile.rest) __syncthreads();                      // part is written again
    }
}

// Many rows. An adapter's rank tiles, matrix after matrix, a lane each: the tile's place among the layer's S * R / 16, how many of its
// ranks the adapter has, and their scale
struct RankTiles {
    int total, place, ranks;
    float scale;
    __device__ __forceinline__ RankTiles(const LoraArgs& a, int who) : total(0), place(0), ranks(0), scale(0.f) {
        const int lane = threadIdx.x & 63, rt = a.R / 16;
        int r[LORA_MAX_SHARDS];
        float f[LORA_MAX_SHARDS];
#pragma unroll
        for (int s = 0; s < LORA_MAX_SHARDS; ++s) {
            r[s] = load_uniform(a.ranks + (int64_t)who * a.S + min(s, a.S - 1));
            f[s] = load_uniform(a.scales + (int64_t)who * a.S + min(s, a.S - 1));
        }
        asm volatile("" : "+s"(r[0]), "+s"(r[1]), "+s"(r[2]), "+s"(r[3]), "+s"(f[0]), "+s"(f[1]), "+s"(f[2]), "+s"(f[3]));
#pragma unroll                                               // (all eight on their way before the first is waited for)
        for (int s = 0; s < LORA_MAX_SHARDS; ++s)
            if (s < a.S) {
                const int n = min(max(r[s], 0), a.R);
                if (lane >= total) {
                    place = s * rt + lane - total;
                    ranks = n - 16 * (lane - total);
                    scale = f[s];
                }
                total += (n + 15) / 16;
            }
    }
    __device__ __forceinline__ int place_of(int i) const { return __builtin_amdgcn_readlane(place, i); }
    __device__ __forceinline__ int ranks_of(int i) const { return __builtin_amdgcn_readlane(ranks, i); }
    __device__ __forceinline__ float scale_of(int i) const {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), i));
    }
};

// The runs' sums of NS tiles of 16 ranks x 16 rows, as the matrix instruction leaves them but for the lanes' order, which keeps apart
// in the banks what lora_sum reads at once: rank l % 16 of row m = 4 (wave % 4) + l / 16 of tile q = wave / 4, in every lane l
template <int NS>
using LoraSums = f32x4[LORA_RUNS][NS][64];
__device__ __forceinline__ int sums_lane(int l) { return l ^ (l >> 4 << 2); }
template <int NS>
__device__ __forceinline__ float lora_sum(const LoraSums<NS>& sums, int q, int m, int l) {
    const int g = (l >> 2) & 3;
    const float* from = reinterpret_cast<const float*>(&sums[0][q][16 * g + (m ^ (4 * g))]) + (l & 3);
    float v[LORA_RUNS], four[4];
#pragma unroll
    for (int z = 0; z < LORA_RUNS; ++z) v[z] = from[z * 256 * NS];
#pragma unroll
    for (int z = 0; z < 4; ++z) four[z] = ((v[4 * z] + v[4 * z + 1]) + v[4 * z + 2]) + v[4 * z + 3];
    return (four[0] + four[1]) + (four[2] + four[3]);
}

// That sum into t: scaled, none of the ranks past `left`, split
template <int DT>
__device__ __forceinline__ void lora_put(const LoraArgs& a, float sum, float scale, int left, int64_t tile_to, int m, int l, bool mine) {
    sum *= scale;
    if ((l & 15) >= left) sum = 0.f;
    if constexpr (DT == F16) {
        float top = fabsf(sum);                              // of the row's 16 lanes; a NaN is passed over
        top = fmaxf(top, dpp_f32<0xB1>(top));
        top = fmaxf(top, dpp_f32<0x4E>(top));
        top = fmaxf(top, dpp_f32<0x141>(top));
        top = fmaxf(top, dpp_f32<0x140>(top));
        const int e = lora_exponent(top);
        sum = ldexpf(sum, -e);
        if ((l & 15) == 0 && mine) a.e[tile_to * 16 + m] = e;
    }
    const uint32_t hi = to16(sum, DT == BF16);
    const float rest = sum - from16((uint16_t)hi, DT == BF16);
    const uint32_t lo = to16(fabsf(rest) < INFINITY ? rest : 0.f, DT == BF16);
    // even lanes store two ranks' high parts, odd ones the two rests
    const uint32_t other = dpp_u32<0xB1>(l & 1 ? hi : lo, 0u);
    const uint32_t two = l & 1 ? other | (lo << 16) : hi | (other << 16);
    const int g = (l >> 2) & 3;
    if (mine)
        reinterpret_cast<uint32_t*>(a.t + tile_to * 64)[4 * (16 * (g >> 1) + m) + 2 * (g & 1) + ((l >> 1) & 1) + (l & 1) * 128] = two;
}

// ------------------------------------------------------------------------------------------------------------------
// The first product, many rows, K up to 8192: 16 G rows against `per` of an adapter's rank tiles (blockIdx.x: the row tile and its
// share of the rank tiles), sixteen waves, a run of the k each. t leaves finished and split. A workgroup has a CU to itself, whose
// intake bounds it (~25 bytes a ns from memory, ~50 from the L2), so it takes x in once and keeps it in registers, G C = 4 KiB of it
// a wave, whatever the ranks and adapters that follow, and the shares are as many as there are CUs for: 64 rows against 48 ranks of
// 2048 are 448 KiB (256 of x, 192 of A), where 32 rows against 96 are 512. x comes in 256 bytes of a row at a time and turns into
// operands through the wave's own 4 KiB of shared memory (16-byte units of a row in the place of their number xor the row's: no two
// lanes of a quarter-wave meet in a bank either way). The next rank tile is in flight while one is multiplied and summed over the waves; the sums of a tile are
// finished by all waves, a rank a lane (the same xor keeps its reads apart). 4096 rows of 2048 against 48 and 192 ranks: 16.4 us.
// ------------------------------------------------------------------------------------------------------------------
constexpr int LORA_ALL_SMEM = 2 * LORA_RUNS * 4096;

template <int DT, int G, int C>
__global__ __launch_bounds__(1024) void lora_shrink_all_kernel(const LoraArgs a, int shares, int per) {
    extern __shared__ uint4 xs[];                            // [LORA_RUNS][256] for x, then every other round's sums
    typedef LoraSums<G> Sums;                                // of a round's row groups
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int item = xcd_tile(blockIdx.x, gridDim.x), tile_at = item / shares, first = item % shares * per;
    const int row0 = tile_at * 16 * G, rt = a.R / 16;
    const int units = (a.K + 31) / 32, run = (units + LORA_RUNS - 1) / LORA_RUNS;      // (at most 4 C)
    const int u0 = wave * run, u1 = min(units, u0 + run);
    TileAdapters<G> tile(a, row0);
    uint4 x[G][C][4];
    {
        const int m = lane & 15, g = lane >> 4;
        const char* xb = reinterpret_cast<const char*>(a.x + row0 * a.x_stride);
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)                  // row 4 i + g of group q, k 32 (u0 + 4 c) + 8 m .. + 8
                    x[q][c][i] = load8(reinterpret_cast<const uint16_t*>(
                        xb + ((uint32_t)(min(16 * q + 4 * i + g, a.T - 1 - row0) * (int)a.x_stride) * 2u +
                              (uint32_t)min(32 * (u0 + 4 * c) + 8 * m, min(32 * u1, a.K) - 8) * 2u)));
    }
    bool fresh = true;
    int round = 1;
    while (tile.rest) {
        uint64_t mask;
        const int who = tile.next(mask);
        const RankTiles tiles(a, who);
        if (first >= tiles.total) continue;
        const int last = min(tiles.total, first + per) - 1;
        const char* ab = reinterpret_cast<const char*>(a.a + (int64_t)who * a.S * rt * units * 64);
        const auto load_a = [&](int i0, int c, uint4(&p)[4]) __attribute__((always_inline)) {
            const char* ap = ab + (int64_t)tiles.place_of(min(i0, last)) * (units * 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = load_kib(ap + min(u0 + 4 * c + i, u1 - 1) * 1024, lane);
        };
        uint4 p[4];
        load_a(first, 0, p);
        __builtin_amdgcn_sched_barrier(0);
        if (fresh) {
            int l = lane;
            asm volatile("" : "+v"(l));                      // (addresses made here, not kept in registers)
            const int m = l & 15, g = l >> 4;
            uint4* own = xs + 256 * wave;
#pragma unroll
            for (int q = 0; q < G; ++q)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const bool past = 32 * (u0 + 4 * c) + 8 * m >= a.K;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        own[(4 * i + g) * 16 + (m ^ (4 * i + g))] = past ? make_uint4(0u, 0u, 0u, 0u) : x[q][c][i];
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[q][c][i] = own[m * 16 + ((4 * i + g) ^ m)];
                    __builtin_amdgcn_wave_barrier();
                }
            fresh = false;
        }
#pragma unroll 1
        for (int i0 = first; i0 <= last; ++i0) {
            f32x4 acc[G];
            uint4 next[4];
#pragma unroll
            for (int q = 0; q < G; ++q) acc[q] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                load_a(c + 1 < C ? i0 : i0 + 1, (c + 1) % C, next);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (u0 + 4 * c + i < u1)
#pragma unroll
                        for (int q = 0; q < G; ++q) acc[q] = mfma32<DT>(p[i], x[q][c][i], acc[q]);
                if (c + 1 < C)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = next[i];
            }
            Sums& sums = *reinterpret_cast<Sums*>(xs + (round++ & 1) * (LORA_RUNS * 256));
            int l = lane;
            asm volatile("" : "+v"(l));
#pragma unroll
            for (int j = 0; j < G; ++j) sums[wave][j][sums_lane(l)] = acc[j];
            lds_barrier();                                   // (the sums before the last ones are read: who does came here after it)
            const int q = (wave >> 2) % G, m = 4 * (wave & 3) + (l >> 4);
            const float sum = lora_sum<G>(sums, q, m, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {                    // (before the store, which would be waited for with them)
                p[i] = next[i];
                asm volatile("" : "+v"(p[i].x), "+v"(p[i].y), "+v"(p[i].z), "+v"(p[i].w));
            }
            lora_put<DT>(a, sum, tiles.scale_of(i0), tiles.ranks_of(i0),
                         ((int64_t)tile_at * G + q) * a.S * rt + tiles.place_of(i0), m, l,
                         wave < 4 * G && (mask >> (16 * q + m)) & 1);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// The first product, many rows, K past 8192: 16 rows against all of an adapter's rank tiles, two a round, sixteen waves, a run of the
// k each; x, which no wave can hold, comes in again every round. blockIdx.y: a row tile's first, third, ... adapter or the others.
// Bound by that intake of x: 14336 -> 4096, three adapters in runs, 2048 rows against 16 ranks 17.6 us (59 MB of x, 3.3 TB/s), 4096 rows
// 42.2 (2.8 TB/s), against 16 and 64 ranks, two rounds for a third of the rows, 56.2.
// ------------------------------------------------------------------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(1024) void lora_shrink_long_kernel(const LoraArgs a, int, int) {
    extern __shared__ uint4 xs[];                            // [LORA_RUNS][256], then the sums of two rounds
    typedef LoraSums<2> Sums;                                // of a round's two tiles
    Sums* part = reinterpret_cast<Sums*>(xs + LORA_RUNS * 256);
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int tile_at = xcd_tile(blockIdx.x, gridDim.x), row0 = tile_at * 16, rt = a.R / 16;
    const int units = (a.K + 31) / 32, run = (units + LORA_RUNS - 1) / LORA_RUNS, chunks = (run + 3) / 4;
    const int u0 = wave * run, u1 = min(units, u0 + run);
    const char* xb = reinterpret_cast<const char*>(a.x + row0 * a.x_stride);
    uint32_t xrow[4];                                        // bytes to rows g, 4 + g, 8 + g, 12 + g
#pragma unroll
    for (int i = 0; i < 4; ++i) xrow[i] = (uint32_t)(min(4 * i + g, a.T - 1 - row0) * (int)a.x_stride) * 2u;
    uint4* own = xs + 256 * wave;
    TileAdapters<1> tile(a, row0);
    int round = 0;
    for (int nth = 0; tile.rest; ++nth) {
        uint64_t mask;
        const int who = tile.next(mask);
        if ((nth & 1) != (int)blockIdx.y) continue;
        const RankTiles tiles(a, who);
        if (tiles.total == 0) continue;
        const char* ab = reinterpret_cast<const char*>(a.a + (int64_t)who * a.S * rt * units * 64);
        const auto load_a = [&](int i0, int c, uint4(&p)[2][4]) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {                    // past the last one: that one again, and not used
                const char* ap = ab + (int64_t)tiles.place_of(min(i0 + j, tiles.total - 1)) * (units * 1024);
#pragma unroll
                for (int i = 0; i < 4; ++i) p[j][i] = load_kib(ap + (int64_t)min(u0 + 4 * c + i, u1 - 1) * 1024, lane);
            }
        };
        uint4 x[4], p[2][4];
        load_a(0, 0, p);
#pragma unroll 1
        for (int i0 = 0; i0 < tiles.total; i0 += 2) {
            f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                const int u = u0 + 4 * c;
#pragma unroll
                for (int i = 0; i < 4; ++i) {                // row 4 i + g, k 32 u + 8 m .. + 8
                    const int k = 32 * u + 8 * m;            // (of a row that is not the adapter's too: its t is not kept)
                    x[i] = load8(reinterpret_cast<const uint16_t*>(xb + (xrow[i] + (uint32_t)min(k, a.K - 8) * 2u)));
                    if (k >= a.K) x[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                const bool more = c + 1 < chunks;
                uint4 next[2][4];
                load_a(more ? i0 : i0 + 2, more ? c + 1 : 0, next);
                __builtin_amdgcn_sched_barrier(0);           // every load before the first use
#pragma unroll
                for (int i = 0; i < 4; ++i) own[(4 * i + g) * 16 + (m ^ (4 * i + g))] = x[i];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = own[m * 16 + ((4 * i + g) ^ m)];
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (u + i < u1)
#pragma unroll
                        for (int j = 0; j < 2; ++j) acc[j] = mfma32<DT>(p[j][i], x[i], acc[j]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[j][i] = next[j][i];
            }
            Sums& sums = part[round++ & 1];
#pragma unroll
            for (int j = 0; j < 2; ++j) sums[wave][j][sums_lane(lane)] = acc[j];
            lds_barrier();
            const int q = (wave >> 2) & 1, at = min(i0 + q, tiles.total - 1), row = 4 * (wave & 3) + g;
            lora_put<DT>(a, lora_sum<2>(sums, q, row, lane), tiles.scale_of(at), tiles.ranks_of(at),
                         (int64_t)tile_at * a.S * rt + tiles.place_of(at), row, lane,
                         wave < 8 && i0 + q < tiles.total && (mask >> row) & 1);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// The second product
// ------------------------------------------------------------------------------------------------------------------
// 8 columns of a row: y's, with what the adapter adds (only where it has ranks: y + 0 is not y's bits for -0 and NaN)
template <int DT>
__device__ __forceinline__ uint4 lora_add8(uint4 y, const float (&add)[8]) {
    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from16((uint16_t)(w[i >> 1] >> (16 * (i & 1))), DT == BF16) + add[i];
    return pack8_16(v, DT == BF16);
}

// One rank tile's products: instruction c's are column 8 (lane % 16) + c of rows 4 (lane / 16) .. + 4
template <int DT>
__device__ __forceinline__ void lora_rank_tile(const uint4& t, const int (&e)[4], const uint4 (&b)[8], f32x4 (&acc)[8]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        if constexpr (DT == F16) {
            const f32x4 v = mfma32<DT>(t, b[c], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[c][i] += ldexpf(v[i], e[i]);
        } else {
            acc[c] = mfma32<DT>(t, b[c], acc[c]);
        }
    }
}

// The matrix that column tile ct lies in: its number, first column of y, and the tile's columns
struct LoraCols {
    int s, c0, cols;
    __device__ __forceinline__ LoraCols(const LoraArgs& a, int ct) : s(0), c0(0) {
        while (ct >= a.tiles0[s + 1]) c0 += a.n_cols[s++];
        const int n0 = (ct - a.tiles0[s]) * LORA_COLS;
        c0 += n0;
        cols = min(a.n_cols[s] - n0, LORA_COLS);
    }
};

// v of the lanes below 32 plus v of those 32 above, in all of them
__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// This lane's operand of a rank tile of t: 8 ranks v of 16 of row lane % 16, the high parts (lanes below 32) or the rests; e: fp16's
// exponents of rows 4 (lane / 16) .. + 4
template <int DT>
__device__ __forceinline__ uint4 lora_operand(f32x4 (&v)[2], float scale, int left, int (&e)[4]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[h][i] = 4 * h + i < left ? v[h][i] * scale : 0.f;
    if constexpr (DT == F16) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(v[0][i]), fabsf(v[1][i])));
        const int mine = lora_exponent(fmaxf(top, __shfl_xor(top, 16)));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[h][i] = ldexpf(v[h][i], -mine);
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __shfl(mine, 4 * (lane >> 4) + i);
    }
    uint2 hi[2], lo[2];
    split4<DT>(v[0], hi[0], lo[0]);
    split4<DT>(v[1], hi[1], lo[1]);
    return lane >= 32 ? make_uint4(lo[0].x, lo[0].y, lo[1].x, lo[1].y) : make_uint4(hi[0].x, hi[0].y, hi[1].x, hi[1].y);
}

// lora_operand from lora_shrink_kernel's four sums, of which the lanes below 32 hold the first two and those above the last two
template <int DT>
__device__ __forceinline__ uint4 lora_t8(const f32x4 (&p)[2][2], float scale, int left, int (&e)[4]) {
    f32x4 v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        v[h] = p[0][h] + p[1][h];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[h][i] = add_halves(v[h][i]);
    }
    return lora_operand<DT>(v, scale, left, e);
}

// Few rows: a wave 128 columns of a row tile (and, spread, its adapters). The same 32 rows, 2048 columns: 5.9 us for 2.5 MB, the same
// round trips; loading before the ranks are known gained nothing, four rank tiles at once (308 registers) lost.
template <int DT>
__global__ __launch_bounds__(64) void lora_expand_kernel(const LoraArgs a) {
    const int lane = threadIdx.x, m = lane & 15, g = lane >> 4, rt = a.R / 16, ct = blockIdx.y;
    const int tile_at = blockIdx.x / a.spread, d = blockIdx.x % a.spread;
    const LoraCols col(a, ct);
    const bool in = 8 * m < col.cols;
    const int64_t row0 = 16 * tile_at + 4 * g, z_at = (int64_t)((a.T + 15) / 16) * a.S * rt * 256;
    const uint16_t* yp = a.y + row0 * a.y_stride + col.c0 + 8 * m;
    uint16_t* op = a.out + row0 * a.out_stride + col.c0 + 8 * m;
    TileAdapters<1> tile(a, 16 * tile_at);
    if (d == 0 && a.out != a.y) {                            // rows of no adapter: y as it is
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && !((tile.rest >> (4 * g + i)) & 1) && row0 + i < a.T) store8(op + i * a.out_stride, load8(yp + i * a.y_stride));
    }
    for (int nth = 0; tile.rest; nth = nth + 1 == a.spread ? 0 : nth + 1) {
        uint64_t mask;
        const int who = tile.next(mask);
        if (nth != d) continue;
        const int r = lora_rank(a, who, col.s);
        const float scale = load_uniform(a.scales + (int64_t)who * a.S + col.s);
        const int mr = (mask >> m) & 1 ? m : __builtin_ctzll(mask);
        const uint32_t own = (uint32_t)mask >> (4 * g);      // this lane's rows 4 g .. + 4
        const uint4* bp = a.b + ((int64_t)who * a.tiles0[a.S] + ct) * rt * 256 + (lane & 31);
        const float* pp = a.part + 2 * (g >> 1) * z_at + (((int64_t)tile_at * a.S + col.s) * rt * 16 + mr) * 16 + 8 * (g & 1);
        uint4 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && ((own >> i) & 1)) y[i] = load8(yp + i * a.y_stride);
        f32x4 acc[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int j0 = 0; 16 * j0 < r; j0 += LORA_FEW) {
            f32x4 p[LORA_FEW][2][2];
            uint4 b[LORA_FEW][8];
#pragma unroll
            for (int j = 0; j < LORA_FEW; ++j)
                if (16 * (j0 + j) < r) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) b[j][c] = bp[(j0 + j) * 256 + 32 * c];
#pragma unroll
                    for (int z = 0; z < 2; ++z)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            p[j][z][h] = *reinterpret_cast<const f32x4*>(pp + z * z_at + (j0 + j) * 256 + 4 * h);
                }
#pragma unroll
            for (int j = 0; j < LORA_FEW; ++j)
                if (16 * (j0 + j) < r) {
                    int e[4];
                    const uint4 t = lora_t8<DT>(p[j], scale, r - 16 * (j0 + j) - 8 * (g & 1), e);
                    lora_rank_tile<DT>(t, e, b[j], acc);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && ((own >> i) & 1)) {
                const float add[8] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i], acc[4][i], acc[5][i], acc[6][i], acc[7][i]};
                store8(op + i * a.out_stride, r > 0 ? lora_add8<DT>(y[i], add) : y[i]);
            }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Both products in one launch, for a few rows and ranks: sixteen waves make t of a row tile and adapter (blockIdx.x), a run of the
// k each, and four of them go on to 128 columns of one matrix each (blockIdx.y). Every workgroup makes its t itself: at 16 ranks of
// 2048 it takes in 64 KiB of A, which costs less than a launch more and the way through memory. One row, 2048 -> 4096 + 512 + 512,
// rank 16: 4.7 us, a launch and four dependent round trips.
// ------------------------------------------------------------------------------------------------------------------
constexpr int LORA_ONE_TILES = 2;              // rank tiles

template <int DT>
__global__ __launch_bounds__(1024) void lora_one_kernel(const LoraArgs a) {
    __shared__ f32x4 part[LORA_ONE_TILES][LORA_RUNS][64];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, rt = a.R / 16;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    int s = 0, c0 = 0, block = blockIdx.y, tiles;            // the matrix, its first column, and four of its column tiles
    while (block >= ((tiles = a.tiles0[s + 1] - a.tiles0[s]) + 3) / 4) {
        block -= (tiles + 3) / 4;
        c0 += a.n_cols[s++];
    }
    const int ct = 4 * block + wave, n0 = ct * LORA_COLS;
    const bool expands = wave < 4 && ct < tiles, in = expands && n0 + 8 * m < a.n_cols[s];
    const uint16_t* yp = a.y + 4 * g * a.y_stride + c0 + n0 + 8 * m;
    uint16_t* op = a.out + 4 * g * a.out_stride + c0 + n0 + 8 * m;
    uint4 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (in && 4 * g + i < a.T) y[i] = load8(yp + i * a.y_stride);
    TileAdapters<1> tile(a, 0);
    if (blockIdx.x == 0 && a.out != a.y) {                   // rows of no adapter: y as it is
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && !((tile.rest >> (4 * g + i)) & 1) && 4 * g + i < a.T) store8(op + i * a.out_stride, y[i]);
    }
    const int units = (a.K + 31) / 32, run = (units + LORA_RUNS - 1) / LORA_RUNS;
    const int u0 = wave * run, u1 = min(units, u0 + run);
    for (int nth = 0; tile.rest; ++nth) {
        uint64_t mask;
        const int who = tile.next(mask);
        if (nth != (int)blockIdx.x) continue;
        const int r = lora_rank(a, who, s), nt = (r + 15) / 16;
        const float scale = load_uniform(a.scales + (int64_t)who * a.S + s);
        const uint4* bp = a.b + ((int64_t)who * a.tiles0[a.S] + a.tiles0[s] + ct) * rt * 256 + (lane & 31);
        uint4 b[LORA_ONE_TILES][8];
        if (expands)
#pragma unroll
            for (int c = 0; c < 8; ++c) b[0][c] = bp[32 * c];
        const int mr = (mask >> m) & 1 ? m : __builtin_ctzll(mask);     // rows of others: the first of this one's
        const uint16_t* xp = a.x + (int64_t)mr * a.x_stride + 8 * g;
        const char* ab = reinterpret_cast<const char*>(a.a + ((int64_t)who * a.S + s) * rt * units * 64);
        f32x4 sum[LORA_ONE_TILES];
#pragma unroll
        for (int j = 0; j < LORA_ONE_TILES; ++j) sum[j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int u = u0; u < u1; u += 4) {
            uint4 x[4], p[LORA_ONE_TILES][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {                    // units past the run's: its last one again, and not used
                const int v = min(u + i, u1 - 1);
#pragma unroll
                for (int j = 0; j < LORA_ONE_TILES; ++j)
                    if (j == 0 || j < nt) p[j][i] = *reinterpret_cast<const uint4*>(ab + ((int64_t)j * units + v) * 1024 + lane * 16u);
                x[i] = load8(xp + min(32 * v, a.K - 8 - 8 * g));
                if (32 * v + 8 * g >= a.K) x[i] = make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int j = 0; j < LORA_ONE_TILES; ++j)
                if (j < nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (u + i < u1) sum[j] = mfma32<DT>(p[j][i], x[i], sum[j]);
        }
#pragma unroll
        for (int j = 0; j < LORA_ONE_TILES; ++j) part[j][wave][lane] = sum[j];
        if (expands && nt > 1)
#pragma unroll
            for (int c = 0; c < 8; ++c) b[1][c] = bp[256 + 32 * c];
        lds_barrier();
        if (!expands) return;                                // (a workgroup has one adapter)
        f32x4 acc[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < LORA_ONE_TILES; ++j)
            if (j < nt) {
                f32x4 v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {                // ranks 8 (g % 2) + 4 h .. + 4 of row m
                    const f32x4* from = &part[j][0][(2 * (g & 1) + h) * 16 + m];
                    f32x4 four[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z)
                        four[z] = ((from[256 * z] + from[256 * z + 64]) + from[256 * z + 128]) + from[256 * z + 192];
                    v[h] = (four[0] + four[1]) + (four[2] + four[3]);
                }
                int e[4];
                const uint4 t = lora_operand<DT>(v, scale, r - 16 * j - 8 * (g & 1), e);
                lora_rank_tile<DT>(t, e, b[j], acc);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && ((mask >> (4 * g + i)) & 1)) {
                const float add[8] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i], acc[4][i], acc[5][i], acc[6][i], acc[7][i]};
                store8(op + i * a.out_stride, r > 0 ? lora_add8<DT>(y[i], add) : y[i]);
            }
        return;
    }
}

constexpr int LORA_HELD = 4;                   // rank tiles of B in shared memory at once

// Many rows: a workgroup of 64 rows (16 a wave) and 128 columns, an adapter's B for them in shared memory. Bound by memory: y comes in
// and out goes out, 84 MB for 4096 rows of 5120 columns in 20.6 us (4.1 TB/s) under the profiler. All waves of a SIMD busy matters more than
// loads in flight: 5 or 6 waves a SIMD by spilling 23 and 36 us, several column tiles a workgroup 31 to 55. An XCD's workgroups go
// through the columns of a row tile first, so that whole rows of y pass at a time (the rows first: 22.1 us).
template <int DT>
__global__ __launch_bounds__(256, DT == BF16 ? 4 : 3) void lora_expand_all_kernel(const LoraArgs a) {
    __shared__ uint4 bs[LORA_HELD][256];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int cts = a.tiles0[a.S], item = xcd_tile(blockIdx.x, gridDim.x), tile_at = item / cts, ct = item % cts;
    const int row0 = tile_at * 64, rt = a.R / 16;
    const LoraCols col(a, ct);
    const uint16_t* yp = a.y + (int64_t)(row0 + 16 * wave) * a.y_stride + col.c0 + 8 * m;
    uint16_t* op = a.out + (int64_t)(row0 + 16 * wave) * a.out_stride + col.c0 + 8 * m;
    const bool in = 8 * m < col.cols;
    uint4 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = make_uint4(0u, 0u, 0u, 0u);
        if (in && row0 + 16 * wave + 4 * g + i < a.T) y[i] = load8(yp + (4 * g + i) * a.y_stride);
    }
    TileAdapters<4> tile(a, row0);
    const uint64_t some = tile.rest;
    while (tile.rest) {
        uint64_t mask;
        const int who = tile.next(mask);
        const int r = lora_rank(a, who, col.s), nt = (r + 15) / 16;
        const uint4* bp = a.b + ((int64_t)who * cts + ct) * rt * 256 + threadIdx.x;
        const uint32_t rows = (uint32_t)(mask >> (16 * wave)) & 0xFFFFu;
        const int64_t at = ((int64_t)min(tile_at * 4 + wave, (a.T - 1) / 16) * a.S + col.s) * rt;
        f32x4 acc[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int j0 = 0; j0 < nt; j0 += LORA_HELD) {
            uint4 b[LORA_HELD], t[LORA_HELD];
            int4 e[LORA_HELD];
#pragma unroll
            for (int j = 0; j < LORA_HELD; ++j) {            // past the last one: that one again
                const int jt = min(j0 + j, nt - 1);
                b[j] = bp[jt * 256];
                t[j] = a.t[(at + jt) * 64 + lane];
                if (DT == F16) e[j] = *reinterpret_cast<const int4*>(a.e + (at + jt) * 16 + 4 * g);
            }
#pragma unroll
            for (int j = 0; j < LORA_HELD; ++j) bs[j][threadIdx.x] = b[j];
            __syncthreads();
            if (rows) {
#pragma unroll
                for (int j = 0; j < LORA_HELD; ++j)
                    if (j0 + j < nt) {
                        uint4 bc[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) bc[c] = bs[j][32 * c + (lane & 31)];
                        int ej[4] = {0, 0, 0, 0};
                        if constexpr (DT == F16) {
                            ej[0] = e[j].x; ej[1] = e[j].y; ej[2] = e[j].z; ej[3] = e[j].w;
                        }
                        lora_rank_tile<DT>(t[j], ej, bc, acc);
                    }
            }
            __syncthreads();                                 // bs is written again
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (in && ((rows >> (4 * g + i)) & 1)) {
                const float add[8] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i], acc[4][i], acc[5][i], acc[6][i], acc[7][i]};
                store8_nt(op + (4 * g + i) * a.out_stride, r > 0 ? lora_add8<DT>(y[i], add) : y[i]);
            }
    }
    if (a.out != a.y) {                                      // rows of no adapter: y as it is
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 16 * wave + 4 * g + i;
            if (in && !((some >> row) & 1) && row0 + row < a.T) store8_nt(op + (4 * g + i) * a.out_stride, y[i]);
        }
    }
}

// The one launch's workgroups a row tile and adapter
static int lora_one_blocks(const LoraArgs& a) {
    int blocks = 0;
    for (int s = 0; s < a.S; ++s) blocks += (a.tiles0[s + 1] - a.tiles0[s] + 3) / 4;
    return blocks;
}

// Whether both products run in one launch: one row tile, at most 64 Ki elements of A a matrix, which every workgroup takes in, and
// no more workgroups than CUs. us in two launches / in one, one row: 2048 -> 4096 + 512 + 512, rank 16 6.2 / 4.6, rank 32 6.6 / 5.9;
// 4096 -> 2048 6.5 / 5.3 and 6.9 / 7.1; 8192 -> 8192, rank 16 7.5 / 7.3; 2048 -> 50048, rank 16, two and four rows 6.4 / 4.8 and
// 7.0 / 8.5
static bool lora_one(const LoraArgs& a) {
    return a.T <= 16 && a.R <= 16 * LORA_ONE_TILES && (int64_t)a.R * a.K <= 1 << 16 && a.T * lora_one_blocks(a) <= 256;
}

template <int DT>
int lora_launch(const LoraArgs& a, bool all, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.T + 15) / 16), cols = (unsigned)a.tiles0[a.S];
    if (all) {
        const int rank_tiles = a.S * (a.R / 16), chunks = a.K <= 2048 ? 1 : a.K <= 4096 ? 2 : 4;
        int groups = a.K <= 8192 ? 4 / chunks : 1;
        // half the rows where there are few tiles, so that more CUs have one. us of both launches, 4 / 2 groups: 2048 -> 4096 + 512 +
        // 512, rank 16, 2048 rows 20.6 / 18.9, 8192 rows 46.8 / 47.9; 2048 -> 2048, rank 128, 1536 rows 13.0 / 12.3, 8192 rows 43 / 48
        if (groups > 1 && (a.T + 16 * groups - 1) / (16 * groups) * rank_tiles < 256) groups /= 2;
        const int row_tiles = (a.T + 16 * groups - 1) / (16 * groups);
        const int want = std::min(rank_tiles, std::max(1, 256 / row_tiles));         // a workgroup a CU
        const int per = (rank_tiles + want - 1) / want, shares = (rank_tiles + per - 1) / per;
        const auto shrink = a.K > 8192                    ? lora_shrink_long_kernel<DT>
                            : chunks == 4                 ? lora_shrink_all_kernel<DT, 1, 4>
                            : chunks == 2 && groups == 2  ? lora_shrink_all_kernel<DT, 2, 2>
                            : chunks == 2                 ? lora_shrink_all_kernel<DT, 1, 2>
                            : groups == 4                 ? lora_shrink_all_kernel<DT, 4, 1>
                                                          : lora_shrink_all_kernel<DT, 2, 1>;
        if (hipFuncSetAttribute((const void*)shrink, hipFuncAttributeMaxDynamicSharedMemorySize, LORA_ALL_SMEM) != hipSuccess)
            return esp_host::fail(ESP_ERR_HIP, "lora: no %d bytes of shared memory", LORA_ALL_SMEM);
        shrink<<<a.K > 8192 ? dim3(tiles, 2) : dim3(row_tiles * shares), 1024, LORA_ALL_SMEM, st>>>(a, shares, per);
        lora_expand_all_kernel<DT><<<(tiles + 3) / 4 * cols, 256, 0, st>>>(a);
    } else if (lora_one(a)) {
        lora_one_kernel<DT><<<dim3(a.T, lora_one_blocks(a)), 1024, 0, st>>>(a);
    } else {
        const unsigned x = tiles * a.spread, ranks = (unsigned)((a.R / 16 + LORA_FEW - 1) / LORA_FEW);
        lora_shrink_kernel<DT><<<dim3(x, a.S * ranks, LORA_RUNS / 4), 256, 0, st>>>(a);
        lora_expand_kernel<DT><<<dim3(x, cols), 64, 0, st>>>(a);
    }
    return esp_host::launch_check("lora");
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

// Whether T rows run as the launches for many rows. They take longer to begin with and less a row, column and rank; but a workgroup of
// theirs goes through all adapters of its 64 rows one after the other, where the few's are dealt out. How many a batch mixes the host
// does not know, only how many there are: up to 16, the rows and the work decide (they cross between 4 and 8 Mi); past 16, a mixed
// batch would lose up to 90 us where a batch of few adapters gains up to 11, so the few's run until 1152 rows, where their own cost
// a row has caught up. us for T rows, few / many (bf16, graph replays): the adapters in runs of rows; 32 rows of any behind a prompt of
// two; all in random order:
//   2048 -> 4096 + 512 + 512, ranks 16, 3 adapters: 8/9  13/14  14/14 at 384, 10/10  15/14  17/15 at 768, 15/10  19/15  25/16 at 1151
//     8 adapters: 8/12  23/26  24/28 at 384, 11/10  26/31  30/31 at 768, 16/13  28/28  44/34 at 1151
//     16 adapters: 9/10  34/52  38/54 at 512, 12/12  34/44  42/53 at 768, 20/13  36/49  59/56 at 1151
//     32 adapters: 11/19  37/76  42/84 at 384, 15/14  40/70  48/85 at 768, 20/15  42/70  70/92 at 1151
//   ranks 16 and 64, 3 adapters: 11/10  15/14  16/15 at 384, 15/11  20/19  23/20 at 768, 20/13  24/20  32/22 at 1151
//     8 adapters: 12/12  32/34  36/36 at 384, 18/12  36/43  46/44 at 768, 23/16  36/39  67/46 at 1151
//     16 adapters: 15/11  50/61  60/64 at 512, 18/16  46/61  68/79 at 768, 26/18  50/69  97/84 at 1151
//     32 adapters: 18/25  47/84  65/98 at 384, 21/21  57/101  86/125 at 768, 28/21  55/98  128/137 at 1151
//   2048 -> 2048, rank 128, 8 adapters: 16/15  31/50  37/52 at 384, 18/14  55/51  62/52 at 768, 22/17  53/59  76/59 at 1151
//     32 adapters: 17/37  43/116  67/157 at 384, 25/26  76/105  122/165 at 768, 31/25  92/153  153/187 at 1151
//   512 -> 2048, ranks 64, 3 adapters: 10/9  13/15  14/15 at 384, 10/10  17/15  18/16 at 768; 8 adapters: 10/12  20/29  21/30 at 384,
//     10/11  26/26  36/30 at 768, 13/13  35/30  43/32 at 1151
//   2048 -> 512 + 512, ranks 32, 8 adapters: 8/12  16/27  16/28 at 384, 10/10  16/24  19/29 at 768, 13/12  21/28  24/28 at 1151
constexpr int64_t LORA_MANY_ROWS = 1152;       // from here on whatever the adapters
static bool lora_many(int64_t T, int64_t N, int64_t rank_tiles, int64_t slots) {
    return T >= LORA_MANY_ROWS || (slots <= 16 && T >= 384 && T * N * rank_tiles >= 6 << 20);
}

// The workgroups that a row tile's adapters are dealt to (few rows): up to one a row, and no more than 32 over all tiles, since
// one that finds nothing costs 2 ns too (a tile of one adapter leaves the others empty). 2048 -> 4096 + 512 + 512, ranks 16 and 64
// of 32 adapters in random rows, 16 / 32 / 64 workgroups: 16 / 13 / 13 us for 32 rows, 64 / 45 / 51 for 256; in 3 runs of rows
// 9.8 / 11.3 / 11.3 and 13.0 / 13.2 / 18.5. Two even so where the second product has few columns (1280 of its waves), so that a
// prompt's tiles of two requests do not take twice as long: 512 rows in 3 runs, one and two: 4096 -> 2048 11.0 and 8.8 us,
// 2048 -> 512 + 512 10.3 and 8.7; 2048 -> 4096 + 512 + 512 11.7 and 13.8
static int lora_spread(int64_t T, int64_t cols) {
    const int64_t tiles = (T + 15) / 16;
    const int64_t spread = std::max<int64_t>(32 / tiles, 2 * tiles * cols <= 1280 ? 2 : 1);
    return (int)std::min<int64_t>({16, T, spread});
}

extern "C" int64_t esp_lora_scratch(int64_t T, int64_t N, int64_t n_shards, int64_t R) {
    if (T <= 0 || N <= 0 || n_shards <= 0 || R <= 0) return 0;
    const int64_t rows = (T + 15) / 16 * 16, ranks = n_shards * ((R + 15) / 16);
    // (below LORA_MANY_ROWS either launches may run, as the slots are, and the few's need more)
    return T >= LORA_MANY_ROWS ? rows * ranks * 17 : rows * ranks * 16 * (LORA_RUNS / 4);
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
        a.tiles0[s + 1] = a.tiles0[s] + (int)((n_cols[s] + LORA_COLS - 1) / LORA_COLS);
        N += n_cols[s];
    }
    ESP_REQUIRE(a.tiles0[n_shards] <= 65535, "lora: at most 65535 blocks of %d columns", LORA_COLS);
    ESP_REQUIRE((T + 63) / 64 * a.tiles0[n_shards] < (1 << 24), "lora: at most 2^24 - 1 blocks of 64 rows and %d columns", LORA_COLS);
    if (T == 0) return esp_host::ok();
    ESP_REQUIRE(x && y && out && rows && A && B && ranks && scales && scratch, "lora: null pointer");
    ESP_REQUIRE(T == 1 || (x_stride >= K && y_stride >= N && out_stride >= N), "lora: rows overlap");
    ESP_REQUIRE(T == 1 || (x_stride <= (1 << 24) && y_stride <= (1 << 24) && out_stride <= (1 << 24)),
                "lora: row strides of at most 2^24 elements");
    ESP_REQUIRE(out != y || T == 1 || out_stride == y_stride, "lora: in place, out must have y's row stride");
    ESP_REQUIRE(((uintptr_t)x | (uintptr_t)y | (uintptr_t)out) % 8 == 0 &&
                    (T == 1 || (x_stride % 4 == 0 && y_stride % 4 == 0 && out_stride % 4 == 0)),
                "lora: x, y and out must be 8-byte aligned with row strides a multiple of 4 elements");
    ESP_REQUIRE(((uintptr_t)A | (uintptr_t)B | (uintptr_t)scratch) % 16 == 0,
                "lora: the adapters and the scratch must be 16-byte aligned");
    ESP_REQUIRE(scratch_numel >= esp_lora_scratch(T, N, n_shards, R), "lora: the scratch needs esp_lora_scratch floats");
    ESP_REQUIRE(!esp_host::rows_meet(out, out_stride * 2, N * 2, x, x_stride * 2, K * 2, T),
                "lora: out overlaps x, which other workgroups still read");
    ESP_REQUIRE(out == y || !esp_host::rows_meet(out, out_stride * 2, N * 2, y, y_stride * 2, N * 2, T),
                "lora: out overlaps y without being y");
    const bool all = lora_many(T, N, n_shards * (R / 16), slots);
    const int64_t tiles = (T + 15) / 16;
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.y = static_cast<const uint16_t*>(y);
    a.y_stride = y_stride;
    a.out = static_cast<uint16_t*>(out);
    a.out_stride = out_stride;
    a.rows = rows;
    a.ranks = ranks;
    a.scales = scales;
    a.a = static_cast<const uint4*>(A);
    a.b = static_cast<const uint4*>(B);
    a.part = scratch;
    a.t = reinterpret_cast<uint4*>(scratch);
    a.e = reinterpret_cast<int*>(scratch) + tiles * n_shards * R * 16;
    a.T = (int)T;
    a.K = (int)K;
    a.S = (int)n_shards;
    a.R = (int)R;
    a.slots = (int)slots;
    a.spread = lora_spread(T, a.tiles0[n_shards]);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == ESP_BF16 ? lora_launch<BF16>(a, all, st) : lora_launch<F16>(a, all, st);
}
