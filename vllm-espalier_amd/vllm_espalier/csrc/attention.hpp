// What the kernels of the attention over a paged cache share (attention.hip for few rows a request, attention_prompt.hip for many):
// which keys of which rows a workgroup takes, conversions, and the join of a row's pieces.
#pragma once

#include "kv.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int STEP = 32;                       // keys a wave takes at once
constexpr int WAVES = 4;
constexpr int FEW_ROWS = 32;                   // requests of up to this many rows a head of the cache are attention.hip's, a tile each,
constexpr int PROMPT_ROWS = 128;               // those of more attention_prompt.hip's, in tiles of this many
constexpr int PIECE = WAVES * STEP;            // pieces are multiples of this many keys
constexpr int TARGET = 512;                    // pieces that a batch is cut into, about: two workgroups a CU

struct AttendArgs {
    const uint16_t* q;
    int64_t q_row, q_head;                      // elements
    uint16_t* out;
    int64_t o_row, o_head;
    const char *k, *v;
    int64_t k_page, k_token, k_head, v_page, v_token, v_head, pages;       // bytes
    const float *ks, *vs;
    const int32_t* tables;
    int64_t table_row;
    const int32_t *lengths, *first, *n_new;
    float* part;                                // [rows][D]: a piece's rows one after the other
    float2* stats;                              // [rows]: a row's maximum and sum
    int2* plan;                                 // [B]: a request's first row in scratch and its pieces a tile
    int tile_rows, first_row;                   // of attention.hip's tiles; attention_prompt.hip's first row in scratch
    int B, T, Hkv, group, max_new, window, split, capacity;                // capacity: tokens that a table can name
    int page16, page_shift;                     // tokens of a page / 16, and its reciprocal: 2 n page_mul >> (32 + page_shift)
    uint32_t page_mul;
    float scale;                                // scale * log2(e)
};

template <typename T>
__device__ __forceinline__ T load_uniform(const T* p) {       // through the scalar cache: nothing writes it while the kernel runs
    return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// ---- which piece a workgroup has

// A request: its rows, and the keys [lo, hi) that any of them sees, lo down to a whole step
struct Request {
    int n, first, length, lo, hi;
};
__device__ __forceinline__ Request request(const AttendArgs& a, int n, int first, int length) {
    Request r = {n, first, max(length, 0), 0, 0};
    if (n < 0 || n > a.max_new || first < 0 || first > a.T - n) r.n = 0;        // no such request
    r.hi = min(r.length, a.capacity);
    if (a.window) r.lo = max(0, min(r.hi, r.length - r.n + 1 - a.window)) & ~(STEP - 1);
    return r;
}
__device__ __forceinline__ Request request_of(const AttendArgs& a, int b) {              // any lane's
    return b < a.B ? request(a, a.n_new ? a.n_new[b] : 1, a.first ? a.first[b] : b, a.lengths[b]) : Request{0, 0, 0, 0, 0};
}
__device__ __forceinline__ Request uniform_request(const AttendArgs& a, int b) {
    return request(a, a.n_new ? load_uniform(a.n_new + b) : 1, a.first ? load_uniform(a.first + b) : b, load_uniform(a.lengths + b));
}

struct Piece {
    int b, tile, head, at, pieces;              // at: which of the tile's pieces
    int64_t row;                                // its first row in scratch
    int size;                                   // keys a piece
};

__device__ __forceinline__ int wave_scan(int v) {             // inclusive sum over the lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Piece `item` of the requests that are tiles of ROWS rows, found by every wave for itself: the requests' lengths give the size of
// the pieces (a.split, or so that there are about TARGET of them) and the requests' first ones. false: there are fewer
template <int ROWS>
__device__ __forceinline__ bool piece_of(const AttendArgs& a, int item, Piece& p) {
    constexpr bool MANY = ROWS == PROMPT_ROWS;
    const int lane = threadIdx.x & 63;
    const auto mine_of = [&](int b) __attribute__((always_inline)) {
        Request r = request_of(a, b);
        if ((r.n * a.group > FEW_ROWS) != MANY) r.n = 0;
        return r;
    };
    // (a prompt has tiles enough to run apart, and is not cut where rows are to be their own)
    int size = MANY && a.split ? 1 << 28 : a.split;
    if (!size) {
        double keys = 0.0;                                     // exact: below 2^53
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const Request r = mine_of(b0 + lane);
            keys += (double)((r.n * a.group + ROWS - 1) / ROWS) * (double)(r.hi - r.lo);
        }
        keys = wave_sum_f64_dpp(keys) * a.Hkv;
        size = ((int)fmin(keys / TARGET, (double)(1 << 28)) / PIECE + 1) * PIECE;
    }
    int before = 0, rows = MANY ? a.first_row : 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const Request r = mine_of(b0 + lane);
        const int tiles = (r.n * a.group + ROWS - 1) / ROWS, pieces = max(1, (r.hi - r.lo + size - 1) / size);
        const int mine = tiles * a.Hkv * pieces, in_scratch = pieces > 1 ? mine * ROWS : 0;
        const int upto = wave_scan(mine), rows_upto = wave_scan(in_scratch);
        const uint64_t hit = __ballot(item >= before + upto - mine && item < before + upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, l); };
            const int in = item - before - of(upto - mine), per_tile = of(pieces);
            p.b = b0 + l;
            p.size = size;
            p.pieces = per_tile;
            // the tiles of a head and piece read the same keys: next to one another
            const int n_tiles = of(tiles);
            p.tile = n_tiles - 1 - in % n_tiles;               // the last rows see the most
            p.at = in / n_tiles % per_tile;
            p.head = in / n_tiles / per_tile;
            const int base = rows + of(rows_upto - in_scratch);
            p.row = base + (int64_t)((p.head * n_tiles + p.tile) * per_tile + p.at) * ROWS;
            if (in == 0 && threadIdx.x == 0) a.plan[p.b] = make_int2(base, per_tile);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        rows += __builtin_amdgcn_readlane(rows_upto, 63);
    }
    return false;
}

// ---- the products

template <bool BF>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {              // to nearest even
    const f32x2 v = {a, b};
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
// two e4m3 values of w's low (HI: high) half as two of dtype, exact
template <bool BF, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// the largest over the four 16-lane rows of a wave, each lane with those at its place; their sum
__device__ __forceinline__ float rows_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
    const uint32_t w = __builtin_bit_cast(uint32_t, v);
    s = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
    const uint32_t w = __builtin_bit_cast(uint32_t, v);
    s = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}

// whether any of the values in w is a NaN or an infinity (e4m3 has no infinities)
template <bool BF, bool E8>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    if constexpr (E8) return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
    return (w & E) == E || (w >> 16 & E) == E;
}

// w with zeros for the values that are none
template <bool BF, bool E8>
__device__ __forceinline__ uint32_t finite(uint32_t w) {
    if constexpr (E8) return w & ~((((w & 0x7F7F7F7Fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xFFu);
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
    return w & ~(((w & E) == E ? 0xFFFFu : 0u) | ((w >> 16 & E) == E ? 0xFFFF0000u : 0u));
}

// The page of 16 keys (-1: the table does not have it, or it does not exist) and their place in it
struct Page {
    int64_t page;
    int off;
};
__device__ __forceinline__ Page page_of(const AttendArgs& a, const int32_t* table, int key) {
    const uint32_t n = (uint32_t)key >> 4, at = __umulhi(2 * n, a.page_mul) >> a.page_shift;
    const bool in = key < a.capacity;
    const int id = load_uniform(table + (in ? at : 0));
    return {in && id >= 0 && id < a.pages ? id : -1, (int)(n - at * (uint32_t)a.page16) * 16};
}

// What a product cannot say: where only some of a tile's rows see a key, its values that are NaN or infinite went in as zeros (a
// weight of zero would have made NaNs of them for every row). If there were any, the tile's outputs are gone over once more, after
// they are stored, and those of the rows that see one become NaN. All threads of the workgroup
template <int D, bool BF, bool E8, int ROWS>
__device__ __forceinline__ void mark_not_finite(const AttendArgs& a, const Piece& pc, const Request& r, const int32_t* table, int k0,
                                                int end) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const char* vb = a.v + pc.head * a.v_head;
    const int d = threadIdx.x;
    if (d >= D) return;
    for (int key = k0; key < end; ++key) {
        const Page p = page_of(a, table, key & ~15);
        if (p.page < 0) continue;
        const char* row = vb + p.page * a.v_page + (p.off + (key & 15)) * a.v_token;
        const uint32_t v = E8 ? *reinterpret_cast<const uint8_t*>(row + d) : *reinterpret_cast<const uint16_t*>(row + 2 * d);
        if (!not_finite<BF, E8>(v)) continue;
        for (int t = 0; t < ROWS; ++t) {
            const int n = pc.tile * ROWS + t, i = n / a.group, pos = r.length - r.n + i;
            if (i >= r.n || key > pos || (a.window && key <= pos - a.window)) continue;
            if (pc.pieces == 1)
                a.out[(int64_t)(r.first + i) * a.o_row + (int64_t)(pc.head * a.group + n % a.group) * a.o_head + d] = BF ? 0x7FC0 : 0x7E00;
            else
                a.part[(pc.row + t) * D + d] = __builtin_nanf("");
        }
    }
}

// Output row `row` (token i, head) of request b from its pieces: D / 4 lanes a piece, the pieces in order within every
// 256 / (D / 4)-th, then those sums in order
template <int D, bool BF, bool E8>
__device__ __forceinline__ void join_row(const AttendArgs& a, const Request& r, int2 plan, int i, int head) {
    constexpr int LANES = D / 4, SIDE = 256 / LANES;
    __shared__ float4 sh[SIDE][LANES];
    __shared__ float sh_m[4], sides[SIDE];
    const int pieces = plan.y, rows = r.n * a.group > FEW_ROWS ? PROMPT_ROWS : a.tile_rows;
    const int row = i * a.group + head % a.group, tiles = (r.n * a.group + rows - 1) / rows;
    const int64_t at = plan.x + (int64_t)((head / a.group * tiles + row / rows) * pieces) * rows + row % rows;
    const float* part = a.part + at * D;
    const float2* stats = a.stats + at;
    float m = -INFINITY;
    for (int p = threadIdx.x; p < pieces; p += 256) m = fmaxf(m, stats[(int64_t)p * rows].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) sh_m[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
    const float base = m == -INFINITY ? 0.f : m;
    const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int p = side; p < pieces; p += SIDE) {
        const float2 s = stats[(int64_t)p * rows];
        const float4 v = *reinterpret_cast<const float4*>(part + (int64_t)p * rows * D + 4 * lane);
        const float w = __builtin_amdgcn_exp2f(s.x - base);
        l += s.y * w;
        o.x += v.x * w;
        o.y += v.y * w;
        o.z += v.z * w;
        o.w += v.w * w;
    }
    sh[side][lane] = o;
    if (lane == 0) sides[side] = l;
    __syncthreads();
    if (side == 0) {
        l = sides[0];
#pragma unroll
        for (int k = 1; k < SIDE; ++k) {
            const float4 v = sh[k][lane];
            l += sides[k];
            o.x += v.x;
            o.y += v.y;
            o.z += v.z;
            o.w += v.w;
        }
        const float vscale = E8 ? a.vs[head / a.group] : 1.f;
        const float f = l > 0.f ? vscale / l : l == 0.f ? 0.f : __builtin_nanf("");
        *reinterpret_cast<uint2*>(a.out + (int64_t)(r.first + i) * a.o_row + (int64_t)head * a.o_head + 4 * lane) =
            make_uint2(pack2<BF>(o.x * f, o.y * f), pack2<BF>(o.z * f, o.w * f));
    }
    __syncthreads();                                          // the LDS is the next row's
}

// The rows of requests with more than one piece, a workgroup every gridDim.x-th of them
template <int D, bool BF, bool E8>
__global__ __launch_bounds__(256) void join_kernel(const AttendArgs a) {
    const int lane = threadIdx.x & 63, heads = a.Hkv * a.group;
    int before = 0, row = blockIdx.x;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        const Request r = request_of(a, b);
        int mine = 0;
        if (r.n > 0 && a.plan[b].y > 1) mine = r.n * heads;
        const int upto = wave_scan(mine), all = before + __builtin_amdgcn_readlane(upto, 63);
        for (; row < all; row += gridDim.x) {
            const int l = __builtin_ctzll(__ballot(row < before + upto));
            const int in = row - before - __builtin_amdgcn_readlane(upto - mine, l);
            join_row<D, BF, E8>(a, uniform_request(a, b0 + l), a.plan[b0 + l], in / heads, in % heads);
        }
        before = all;
    }
}

// ---- the host's side

struct AttendSizes {
    int64_t few, many, rows, part, stats, bytes;              // workgroups of either kernel; rows in scratch; byte offsets
    int tile_rows, first_row;
    AttendSizes(int64_t B, int64_t T, int64_t max_new, int64_t group, int64_t Hkv, int64_t D, int64_t capacity, int64_t split) {
        tile_rows = max_new * group <= 16 ? 16 : FEW_ROWS;
        const int64_t size = split ? split : PIECE, most = std::max<int64_t>(1, (capacity + size - 1) / size);   // pieces a tile
        // chosen pieces: the sum of ceil(k / size) over all tiles is at most TARGET more than there are tiles, and that of the
        // tiles with k > size, whose pieces go to scratch, at most twice the sum of k / size
        few = B * Hkv * most;
        int64_t slots = most > 1 ? few : 0;
        if (!split) {
            few = std::min(few, B * Hkv + TARGET);
            slots = std::min<int64_t>(slots, 2 * TARGET);
        }
        first_row = 0;
        rows = slots * tile_rows;
        many = 0;
        if (max_new * group > FEW_ROWS) {
            // requests' rows are apart, so there are no more tiles than all rows make, and a part of one more each
            many = std::min(B * ((max_new * group + PROMPT_ROWS - 1) / PROMPT_ROWS), T * group / PROMPT_ROWS + B) * Hkv;
            first_row = (int)std::min<int64_t>(rows, 1 << 30);
            if (!split && most > 1) {
                many += TARGET;
                rows += 2 * TARGET * PROMPT_ROWS;
            }
        }
        part = (B * 8 + 15) / 16 * 16;
        stats = part + rows * D * 4;
        bytes = stats + rows * 8;
    }
};

// attention_prompt.hip: tiles of PROMPT_ROWS rows
void attend_prompt(const AttendArgs& a, const AttendSizes& z, int D, bool bf, bool e8, hipStream_t st);

}  // namespace esp
