// What the kernels of the attention over a paged cache share (attention.hip for few rows a request, attention_prompt.hip for many):
// which keys of which rows a workgroup takes, conversions, and the join of a row's pieces.
#pragma once

#include "kv.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int STEP = 32;                       // keys a wave takes at once
constexpr int WAVES = 4;
constexpr int FEW_ROWS = 32;                   // requests of up to this many rows a head of the cache are attention.hip's, a tile each,
constexpr int PROMPT_ROWS = 128;               // those of more attention_prompt.hip's, in tiles of this many
constexpr int PIECE = WAVES * STEP;            // pieces are multiples of this many keys
constexpr int PROMPT_SLOTS = 512;              // workgroups that fit at once: attention_prompt.hip's (two a CU)
constexpr int LONG_SLOTS = 256, LONG_TILES = 16;    // and attention.hip's where a batch has few tiles, whose rows would have many pieces

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
    float* part;                                // [a tile's rows][its pieces][D]
    float2* stats;                              // a row's maximum and sum in a piece
    int2* plan;                                 // [B]: a request's first place in scratch and its pieces a tile
    int slots;                                  // workgroups of attention.hip that fit at once
    int many;                                   // of attention_prompt.hip's launch, those for requests of many rows
    int tile_rows, first_row;                   // of attention.hip's tiles; attention_prompt.hip's first place in scratch
    int64_t rows;                               // places in scratch
    int B, T, Hkv, group, max_new, window, split, capacity;                // capacity: tokens that a table can name
    int page16, page_shift;                     // tokens of a page / 16, and its reciprocal: 2 n page_mul >> (32 + page_shift)
    uint32_t page_mul;
    float scale;                                // scale * log2(e)
};

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

struct Piece {
    Request r;
    int b, tile, head, at, pieces;              // at: which of the tile's pieces
    int64_t row;                                // its first row's place in scratch, a row's pieces are next to one another
    int size;                                   // keys a piece
};

__device__ __forceinline__ int wave_scan(int v) {             // inclusive sum over the lanes: rows of 16, then over the rows
    v += (int)dpp_u32<0x111>((uint32_t)v, 0u);                // row_shr 1, 2, 4, 8
    v += (int)dpp_u32<0x112>((uint32_t)v, 0u);
    v += (int)dpp_u32<0x114>((uint32_t)v, 0u);
    v += (int)dpp_u32<0x118>((uint32_t)v, 0u);
    v += (int)dpp_u32<0x142, 0xA>((uint32_t)v, 0u);           // row_bcast:15 into rows 1, 3
    v += (int)dpp_u32<0x143, 0xC>((uint32_t)v, 0u);           // row_bcast:31 into rows 2, 3
    return v;
}

// n / d of non-negative numbers with a quotient below 2^22 (its relative error is 2^-22 at most: the reciprocal's quotient is off by
// one at most), or n below 2^24 and d a power of two
__device__ __forceinline__ int quotient(int n, int d) {
    int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
    const int r = n - q * d;
    q += r >= d ? 1 : r < 0 ? -1 : 0;
    return q;
}

// Whether what was found lies in the request and in scratch. It does, but where requests that claim the same rows make more tiles than
// all rows have
__device__ __forceinline__ bool sound(const AttendArgs& a, const Piece& p, int tiles, int rows, int base, int first) {
    return p.tile >= 0 && p.tile < tiles && p.head >= 0 && p.head < a.Hkv && p.at >= 0 && p.at < p.pieces &&
           (p.pieces == 1 || (base >= first && base + (int64_t)tiles * a.Hkv * p.pieces * rows <= a.rows));
}

// The same of up to 64 requests, a lane each (r, pieces of `size` keys), those of the tiles that see the most keys first, so that the
// last workgroups are short ones: item counts down the tiles that see more than 64 x keys, for the x at which they are more than
// item (-1: all tiles). Heads next to one another: with the workgroups dealt to the XCDs in turn, an XCD's L2 has a few heads' keys.
template <int ROWS>
__device__ __forceinline__ bool piece_by_length(const AttendArgs& a, int item, int size, const Request& r, Piece& p) {
    const int lane = threadIdx.x & 63;
    const int tiles = (r.n * a.group + ROWS - 1) / ROWS, pieces = max(1, quotient(r.hi - r.lo + size - 1, size));
    const float per_key = (float)a.group / ROWS;              // tiles a key further down
    const auto above = [&](int x) __attribute__((always_inline)) {           // the request's tiles that see more
        return x < 0 ? tiles : max(0, min(tiles, (int)ceilf((float)min(r.hi - 64 * x, 1 << 24) * per_key)));
    };
    const auto all = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
    if (item >= all(tiles * a.Hkv * pieces)) return false;
    int x = -1, end = (int)(wave_max_u32((uint32_t)r.hi) >> 6) + 1;
    while (end - x > 1) {
        const int mid = (x + end) >> 1;
        if (all(above(mid) * a.Hkv * pieces) > item) x = mid;
        else end = mid;
    }
    const int higher = above(x + 1), rest = item - all(higher * a.Hkv * pieces);
    const int mine = (above(x) - higher) * a.Hkv * pieces, upto = wave_scan(mine);
    const int in_scratch = pieces > 1 ? tiles * a.Hkv * pieces * ROWS : 0, rows_upto = wave_scan(in_scratch);
    const uint64_t hit = __ballot(rest < upto);
    if (!hit) return false;
    const int l = __builtin_ctzll(hit);
    const auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, l); };
    const int in = rest - of(upto - mine), stack = __builtin_amdgcn_readfirstlane(quotient(in, a.Hkv));
    p.r = {of(r.n), of(r.first), of(r.length), of(r.lo), of(r.hi)};
    p.b = l;
    p.size = size;
    p.pieces = of(pieces);
    p.head = in - stack * a.Hkv;
    const int level = __builtin_amdgcn_readfirstlane(quotient(stack, p.pieces));
    p.at = stack - level * p.pieces;
    p.tile = of(tiles) - 1 - of(higher) - level;
    const int base = a.first_row + of(rows_upto - in_scratch);
    p.row = base + (int64_t)(p.head * of(tiles) + p.tile) * p.pieces * ROWS + p.at;
    if (!sound(a, p, of(tiles), ROWS, base, a.first_row)) return false;
    if (p.tile == 0 && p.head == 0 && p.at == 0 && threadIdx.x == 0) a.plan[l] = make_int2(base, p.pieces);
    return true;
}

// Piece `item` of the requests that are tiles of ROWS rows, found by every wave for itself from the requests' lengths: the size of the
// pieces (a.split, or the smallest, about, with which all pieces fit on the CUs at once) and the requests' first ones. false: there are
// fewer. 32 requests of up to 8171 keys, 273 MB: 53 us with pieces that fit, 57 with smaller and 66 with larger ones
template <int ROWS>
__device__ __forceinline__ bool piece_of(const AttendArgs& a, int item, Piece& p) {
    constexpr bool MANY = ROWS == PROMPT_ROWS;
    const int lane = threadIdx.x & 63;
    const auto mine_of = [&](int b) __attribute__((always_inline)) {
        Request r = request_of(a, b);
        if ((r.n * a.group > FEW_ROWS) != MANY) r.n = 0;
        return r;
    };
    const auto tiles_of = [&](const Request& r) __attribute__((always_inline)) { return (r.n * a.group + ROWS - 1) / ROWS * a.Hkv; };
    const Request r0 = mine_of(lane);                         // the first 64, loaded once
    const auto request_at = [&](int b0) __attribute__((always_inline)) { return b0 ? mine_of(b0 + lane) : r0; };
    // Requests of more than FEW_ROWS rows are not cut where rows are to be their own: a prompt has tiles enough to run apart. One of few tiles
    // has not (5 tokens of 32/4 heads over 8000: 178 us for 18 by the lengths), which is what its rows' own bits cost it
    int size = MANY && a.split ? 1 << 28 : a.split;
    if (!size) {
        double keys = 0.0;                                     // exact: below 2^53
        int tiles = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const Request r = request_at(b0);
            const int mine = tiles_of(r);
            keys += (double)mine * (double)(r.hi - r.lo);
            tiles += mine;
        }
        keys = wave_sum_f64_dpp(keys);
        tiles = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
        const int slots = MANY ? PROMPT_SLOTS : tiles <= LONG_TILES ? min(LONG_SLOTS, a.slots) : a.slots;
        // a tile's last piece is half a piece, on average; then a little more at a time
        const float most = (float)max(slots - tiles / 2, slots / 4);
        size = ((int)fminf((float)keys * __builtin_amdgcn_rcpf(most), (float)(1 << 28)) / PIECE + 1) * PIECE;
        for (int k = 0; k < 4 && !MANY && tiles < slots; ++k) {
            int pieces = 0;
            for (int b0 = 0; b0 < a.B; b0 += 64) {
                const Request r = request_at(b0);
                pieces += tiles_of(r) * max(1, quotient(r.hi - r.lo + size - 1, size));
            }
            if (__builtin_amdgcn_readlane(wave_scan(pieces), 63) <= slots) break;
            size += (size / (16 * PIECE) + 1) * PIECE;
        }
    }
    if (MANY && a.B <= 64) return piece_by_length<ROWS>(a, item, size, r0, p);
    int before = 0, rows = MANY ? a.first_row : 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const Request r = request_at(b0);
        const int tiles = (r.n * a.group + ROWS - 1) / ROWS, pieces = max(1, quotient(r.hi - r.lo + size - 1, size));
        const int mine = tiles * a.Hkv * pieces, in_scratch = pieces > 1 ? mine * ROWS : 0;
        const int upto = wave_scan(mine), rows_upto = wave_scan(in_scratch);
        const uint64_t hit = __ballot(item >= before + upto - mine && item < before + upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, l); };
            const int in = item - before - of(upto - mine), per_tile = of(pieces);
            p.r = {of(r.n), of(r.first), of(r.length), of(r.lo), of(r.hi)};
            p.b = b0 + l;
            p.size = size;
            p.pieces = per_tile;
            // the tiles of a head and piece read the same keys: next to one another
            const int n_tiles = of(tiles);
            const int stack = MANY ? __builtin_amdgcn_readfirstlane(quotient(in, n_tiles)) : in;
            p.tile = MANY ? n_tiles - 1 - (in - stack * n_tiles) : 0;
            p.head = __builtin_amdgcn_readfirstlane(quotient(stack, per_tile));
            p.at = stack - p.head * per_tile;
            const int base = rows + of(rows_upto - in_scratch);
            p.row = base + (int64_t)(p.head * n_tiles + p.tile) * per_tile * ROWS + p.at;
            if (!sound(a, p, n_tiles, ROWS, base, MANY ? a.first_row : 0)) return false;
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
// two e4m3 values of w's low (HI: high) half as two of dtype, exact
template <bool BF, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// What the exponents of a row's weights are taken from, by its running maximum m (-inf where it has seen nothing). bf16 weights: m. fp16 has
// ten binary places down to 2^-14 only: over m - 13 a weight is off by at most half a step of itself down to 2^-27 of the largest, and by
// 2^-38 of that below (over m, thousands of keys some 2^-25 below one whose value is small would come out as nothing, though their weights
// are in the sum). Weights stay below 2^15.5 so, prompts' LAG among them, while scores are below 2^22; past that, where fp32's own steps
// move an exponent by whole numbers, over m. Sums, outputs and statistics are over the same, and it cancels.
template <bool BF>
__device__ __forceinline__ float reference(float m) {
    if constexpr (BF) return m;
    return m - (fabsf(m) < 4194304.0f ? 13.0f : 0.0f);
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

// The same by every lane for a key of its own: a wave looks its next pages up together, ahead of their turn
struct Place {
    int page, off;
};
__device__ __forceinline__ Place place_of(const AttendArgs& a, const int32_t* table, int key) {
    const uint32_t n = (uint32_t)key >> 4, at = __umulhi(2 * n, a.page_mul) >> a.page_shift;
    const bool in = key < a.capacity;
    const int id = table[in ? at : 0];
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
                a.part[(pc.row + t * pc.pieces) * D + d] = __builtin_nanf("");
        }
    }
}

// Output row (token i, head) of a request from its pieces: D / 4 lanes a piece, the pieces in order within every SIDE-th with a running
// maximum, then those sums in order; AHEAD pieces of a thread are on their way at once
template <int D, bool BF, bool E8, int THREADS, int AHEAD>
__device__ __forceinline__ void join_row(const AttendArgs& a, const Request& r, int first_row, int pieces, int i, int head) {
    constexpr int LANES = D / 4, SIDE = THREADS / LANES;
    __shared__ float4 sh[SIDE][LANES];
    __shared__ float2 sides[SIDE];
    const int rows = r.n * a.group > FEW_ROWS ? PROMPT_ROWS : a.tile_rows;
    const int kv = __builtin_amdgcn_readfirstlane(quotient(head, a.group)), row = i * a.group + head - kv * a.group;
    const int tiles = (r.n * a.group + rows - 1) / rows;
    const int64_t at = first_row + ((int64_t)(kv * tiles + row / rows) * rows + row % rows) * pieces;
    const int lane = threadIdx.x % LANES, side = threadIdx.x / LANES;
    const float* part = a.part + at * D + 4 * lane;
    const float2* stats = a.stats + at;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = side; p0 < pieces; p0 += SIDE * AHEAD) {
        float2 s[AHEAD];
        float4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {                     // (the last ones again where there are no more)
            const int p = min(p0 + SIDE * k, pieces - 1);
            s[k] = stats[p];
            v[k] = *reinterpret_cast<const float4*>(part + p * D);
        }
        float next = m;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (p0 + SIDE * k < pieces) next = fmaxf(next, s[k].x);
        const float base = next == -INFINITY ? 0.f : next, alpha = __builtin_amdgcn_exp2f(m - base);
        m = next;
        l *= alpha;
        o.x *= alpha;
        o.y *= alpha;
        o.z *= alpha;
        o.w *= alpha;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p0 + SIDE * k >= pieces) break;
            const float w = __builtin_amdgcn_exp2f(s[k].x - base);
            l += s[k].y * w;
            o.x += v[k].x * w;
            o.y += v[k].y * w;
            o.z += v[k].z * w;
            o.w += v[k].w * w;
        }
    }
    sh[side][lane] = o;
    if (lane == 0) sides[side] = make_float2(m, l);
    __syncthreads();
    if (side == 0) {
#pragma unroll
        for (int k = 1; k < SIDE; ++k) m = fmaxf(m, sides[k].x);
        const float base = m == -INFINITY ? 0.f : m;
        l = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < SIDE; ++k) {
            const float4 v = sh[k][lane];
            const float w = __builtin_amdgcn_exp2f(sides[k].x - base);
            l += sides[k].y * w;
            o.x += v.x * w;
            o.y += v.y * w;
            o.z += v.z * w;
            o.w += v.w * w;
        }
        const float vscale = E8 ? a.vs[kv] : 1.f;
        const float f = l > 0.f ? vscale / l : l == 0.f ? 0.f : __builtin_nanf("");
        *reinterpret_cast<uint2*>(a.out + (int64_t)(r.first + i) * a.o_row + (int64_t)head * a.o_head + 4 * lane) =
            make_uint2(pack2<BF>(o.x * f, o.y * f), pack2<BF>(o.z * f, o.w * f));
    }
    __syncthreads();                                          // the LDS is the next row's
}

// The rows of requests with more than one piece, a workgroup every gridDim.x-th of them
template <int D, bool BF, bool E8, int THREADS, int AHEAD>
__global__ __launch_bounds__(THREADS) void join_kernel(const AttendArgs a) {
    const int lane = threadIdx.x & 63, heads = a.Hkv * a.group;
    int before = 0, row = blockIdx.x;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        const int2 plan = b < a.B ? a.plan[b] : make_int2(0, 0);              // (of no request: anything)
        const Request r = request_of(a, b);
        const int rows = r.n * a.group > FEW_ROWS ? PROMPT_ROWS : a.tile_rows, tiles = (r.n * a.group + rows - 1) / rows;
        const bool joined = r.n > 0 && plan.x >= 0 && plan.y > 1 && plan.x + (int64_t)tiles * a.Hkv * plan.y * rows <= a.rows;
        const int mine = joined ? r.n * heads : 0, upto = wave_scan(mine);
        const int all = before + __builtin_amdgcn_readlane(upto, 63);
        for (; row < all; row += gridDim.x) {
            const uint64_t hit = __ballot(row < before + upto);
            if (!hit) return;
            const int l = __builtin_ctzll(hit);
            const auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, l); };
            const int in = row - before - of(upto - mine), i = __builtin_amdgcn_readfirstlane((int)((uint32_t)in / (uint32_t)heads));
            if (in < 0 || i >= of(r.n)) return;
            join_row<D, BF, E8, THREADS, AHEAD>(a, {of(r.n), of(r.first), 0, 0, 0}, of(plan.x), of(plan.y), i, in - i * heads);
        }
        before = all;
    }
}

// ---- the host's side

struct AttendSizes {
    int64_t few, many, rows, part, stats, bytes;              // workgroups of either kernel; rows in scratch; byte offsets
    int tile_rows, first_row, slots;
    AttendSizes(int64_t B, int64_t T, int64_t max_new, int64_t group, int64_t Hkv, int64_t D, int64_t capacity, int64_t split) {
        tile_rows = max_new * group <= 16 ? 16 : FEW_ROWS;
        slots = 256 * (D == 256 ? 1 : D == 128 && tile_rows == FEW_ROWS ? 2 : 3);
        const int64_t size = split ? split : PIECE, most = std::max<int64_t>(1, (capacity + size - 1) / size);   // pieces a tile
        // the size chosen is at least keys / slots: the sum of ceil(k / size) over all tiles is at most `slots` more than there are
        // tiles, and that of the tiles with k > size, whose pieces go to scratch, at most twice the sum of k / size
        few = B * Hkv * most;
        int64_t in_scratch = most > 1 ? few : 0;
        if (!split) {
            few = std::min(few, B * Hkv + slots);
            in_scratch = std::min<int64_t>(in_scratch, 2 * slots);
        }
        first_row = 0;
        rows = in_scratch * tile_rows;
        many = 0;
        if (max_new * group > FEW_ROWS) {
            // requests' rows are apart, so there are no more tiles than all rows make, and a part of one more each
            many = std::min(B * ((max_new * group + PROMPT_ROWS - 1) / PROMPT_ROWS), T * group / PROMPT_ROWS + B) * Hkv;
            first_row = (int)std::min<int64_t>(rows, 1 << 30);
            if (!split && most > 1) {
                many += PROMPT_SLOTS;
                rows += 2 * PROMPT_SLOTS * PROMPT_ROWS;
            }
        }
        part = (B * 8 + 15) / 16 * 16;
        stats = part + rows * D * 4;
        bytes = stats + rows * 8;
    }
};

// attention_prompt.hip: tiles of PROMPT_ROWS rows, and, FEW_TOO, the requests of few rows as well: a prompt of 2048 new tokens beside
// 31 requests of one over 4000, heads 32/8 of 128, takes 149 us in one launch and 171 in two (the same prompt alone 62 and 64), 512
// beside 31 over 2000 77 and 85. With workgroups of both kinds in turn, by eights, the second is 93 (the requests of one token, bound
// by memory, want all slots at once). Heads of 256 would lose: 174 us for 168 at 4 prompts of 1024 over 2048 (registers spill).
template <int D>
constexpr bool FEW_TOO = D != 256;
void attend_prompt(const AttendArgs& a, const AttendSizes& z, int D, bool bf, bool e8, hipStream_t st);

}  // namespace esp
