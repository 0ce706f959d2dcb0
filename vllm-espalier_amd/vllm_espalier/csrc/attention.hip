// Attention of new tokens over a paged cache of keys and values, on gfx950: one token of a request, a token and its drafts, or a
// prompt, behind whatever the cache holds of the request already. Row i of a request's n new tokens stands at position
// p = length - n + i and sees the keys j with max(0, p - window + 1) <= j <= p (no window: all up to its own):
//   o = sum_j softmax_j(scale * q k_j) v_j,   zeros where a row sees nothing.
//
// A request's rows that share a head of the cache (its new tokens times the query heads of the group) are tiles of ROWS rows; the
// keys that a tile sees are cut into pieces, and a workgroup takes a piece of a tile: its four waves take 32 keys in turn, each with
// a running maximum and sum of its own, joined at the end. Tiles of one piece are written at once, the others' pieces go to scratch
// (fp32) and a second launch joins them, in their order.
//
// All in registers: with S^T = K Q^T (keys are the rows of the product, queries its columns) a lane loads 8 consecutive elements of
// a key, 16 bytes, as the matrix instruction wants them, and is left with the scores of one query. For O^T = V^T P^T its scores are
// again what the instruction wants, if the 8 keys that it takes of 32 are the lane's own: 4 of the first 16 and 4 of the second,
// since the order of the summed index is free. V^T wants 8 keys of one element in a lane: the lane loads the same 16 bytes of 8
// keys (16 lanes: a whole row) and swaps pairs of halves, 32 v_perm for 8 x 8 elements; the element of operand e in lane l is
// 8 l + e, which is where the output puts it.
//
// Scores, statistics and sums are fp32; the weights are rounded to the rows' dtype for the second product (off by at most half a
// step of themselves; their sum is that of the unrounded ones), e4m3 keys and values are exact in either dtype.
#include "kv.hpp"
#include "norm.hpp"

namespace esp {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int STEP = 32;                       // keys a wave takes at once
constexpr int WAVES = 4;
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
    float* part;                                // [pieces][ROWS][D], then [pieces][ROWS][2]: a row's maximum and sum
    float* stats;
    int2* plan;                                 // [B]: a request's first piece in scratch and its pieces a tile
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
    int64_t slot;                               // its place in scratch
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

// Piece `item` of the batch, found by every wave for itself: the requests' lengths give the size of the pieces (a.split, or so
// that there are about TARGET of them) and the requests' first ones. false: there are fewer
template <int ROWS>
__device__ __forceinline__ bool piece_of(const AttendArgs& a, int item, Piece& p) {
    const int lane = threadIdx.x & 63;
    int size = a.split;
    if (!size) {
        double keys = 0.0;                                     // exact: below 2^53
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const Request r = request_of(a, b0 + lane);
            keys += (double)((r.n * a.group + ROWS - 1) / ROWS) * (double)(r.hi - r.lo);
        }
        keys = wave_sum_f64_dpp(keys) * a.Hkv;
        size = ((int)fmin(keys / TARGET, (double)(1 << 28)) / PIECE + 1) * PIECE;
    }
    int before = 0, slots = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const Request r = request_of(a, b0 + lane);
        const int tiles = (r.n * a.group + ROWS - 1) / ROWS, pieces = max(1, (r.hi - r.lo + size - 1) / size);
        const int mine = tiles * a.Hkv * pieces, in_scratch = pieces > 1 ? mine : 0;
        const int upto = wave_scan(mine), slots_upto = wave_scan(in_scratch);
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
            p.tile = in % n_tiles;
            p.at = in / n_tiles % per_tile;
            p.head = in / n_tiles / per_tile;
            const int base = slots + of(slots_upto - in_scratch);
            p.slot = base + (int64_t)(p.head * n_tiles + p.tile) * per_tile + p.at;
            if (in == 0 && threadIdx.x == 0) a.plan[p.b] = make_int2(base, per_tile);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        slots += __builtin_amdgcn_readlane(slots_upto, 63);
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

// The pages of 16 keys each, of which a step has two: a page that the table does not have, or that does not exist, is none
struct Pages {
    int64_t page[2];                            // -1: none
    int off[2];                                 // keys into the page
};
__device__ __forceinline__ Pages pages_of(const AttendArgs& a, const int32_t* table, int key) {
    Pages p;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint32_t n = (uint32_t)(key + 16 * u) >> 4;
        const uint32_t at = __umulhi(2 * n, a.page_mul) >> a.page_shift;
        const bool in = key + 16 * u < a.capacity;
        const int id = load_uniform(table + (in ? at : 0));
        p.page[u] = in && id >= 0 && id < a.pages ? id : -1;
        p.off[u] = (int)(n - at * (uint32_t)a.page16) * 16;
    }
    return p;
}

// A wave's 32 keys or values. Keys: operand c of tile u holds elements 32 c + 8 g .. + 8 of key l (16 bits), or, two operands a
// load, 64 (c / 2) + 16 g + 8 (c % 2) .. + 8 (8 bits). Values: words of elements E l .. + E (in halves of 128) of keys 4 g + j
template <int D, bool E8>
struct Keys {
    u32x4 w[2][E8 ? D / 64 : D / 32];
};
template <int D, bool E8>
struct Values {
    static constexpr int HALVES = D == 256 ? 2 : 1, E = D == 64 ? 4 : 8, WORDS = E8 ? E / 4 : E / 2;
    uint32_t w[8][HALVES][WORDS];
};

template <int D, bool E8>
__device__ __forceinline__ void load_keys(const AttendArgs& a, const char* base, const Pages& p, int lane, Keys<D, E8>& k) {
    const int to = (lane & 15) * (int)a.k_token + (lane >> 4) * 16;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const char* row = base + (p.page[u] < 0 ? 0 : p.page[u]) * a.k_page + p.off[u] * a.k_token;
#pragma unroll
        for (int c = 0; c < (E8 ? D / 64 : D / 32); ++c) k.w[u][c] = *reinterpret_cast<const u32x4*>(row + to + c * 64);
    }
}
template <int D, bool E8>
__device__ __forceinline__ void load_values(const AttendArgs& a, const char* base, const Pages& p, int lane, Values<D, E8>& v) {
    using V = Values<D, E8>;
    const int to = (lane >> 4) * 4 * (int)a.v_token + (lane & 15) * V::WORDS * 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const char* row = base + (p.page[j / 4] < 0 ? 0 : p.page[j / 4]) * a.v_page + (p.off[j / 4] + j % 4) * a.v_token;
#pragma unroll
        for (int h = 0; h < V::HALVES; ++h) {
            const char* at = row + to + h * (E8 ? 128 : 256);
            if constexpr (V::WORDS == 4) {
                const uint4 t = *reinterpret_cast<const uint4*>(at);
                v.w[j][h][0] = t.x; v.w[j][h][1] = t.y; v.w[j][h][2] = t.z; v.w[j][h][3] = t.w;
            } else if constexpr (V::WORDS == 2) {
                const uint2 t = *reinterpret_cast<const uint2*>(at);
                v.w[j][h][0] = t.x; v.w[j][h][1] = t.y;
            } else {
                v.w[j][h][0] = *reinterpret_cast<const uint32_t*>(at);
            }
        }
    }
}

// What a wave has of its tile: a running maximum and (this lane's keys') sum of a query, and the unscaled output
template <int D, int NT>
struct State {
    static constexpr int OPS = D / 16;                        // operands of V^T
    float m[NT], l[NT];
    f32x4 o[NT][OPS];
};

// halves e % 2 of rows 2 t, 2 t + 1: operand e of V^T, from the words of 8 keys that hold its element
__device__ __forceinline__ u32x4 turned(const uint32_t (&w)[8], int e) {
    u32x4 r;
#pragma unroll
    for (int t = 0; t < 4; ++t) r[t] = __builtin_amdgcn_perm(w[2 * t + 1], w[2 * t], e % 2 ? 0x07060302u : 0x05040100u);
    return r;
}

// One step of 32 keys from `key`. edge: some of them are not every row's. hi, lo: the keys [lo, hi) that the lane's query sees
template <int D, bool BF, bool E8, int NT>
__device__ __forceinline__ void step(const u32x4 (&q)[NT][D / 32], const Keys<D, E8>& k, Values<D, E8>& v, bool edge, int key,
                                     const Pages& p, const int (&lo)[NT], const int (&hi)[NT], int any_lo, int any_hi, float scale,
                                     State<D, NT>& st) {
    using V = Values<D, E8>;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    f32x4 s[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[t][u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            u32x4 kw;
            if constexpr (E8) {
                const u32x4 w = k.w[u][c / 2];
                const uint32_t x = w[c % 2 * 2], y = w[c % 2 * 2 + 1];
                kw = {widen2<BF, false>(x), widen2<BF, true>(x), widen2<BF, false>(y), widen2<BF, true>(y)};
            } else {
                kw = k.w[u][c];
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][u] = mfma<BF>(kw, q[t][c], s[t][u]);
        }
    bool odd = false;                                         // a NaN or an infinity: some rows may see it and others not
    if (edge) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = key + 16 * u + 4 * g + i;
                const bool none = p.page[u] < 0;
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    if (none || at < lo[t] || at >= hi[t]) s[t][u][i] = -INFINITY;
                const uint32_t keep = none || at < any_lo || at >= any_hi ? 0u : ~0u;    // nobody's value: 0 * NaN would be a NaN
#pragma unroll
                for (int h = 0; h < V::HALVES; ++h)
#pragma unroll
                    for (int w = 0; w < V::WORDS; ++w) {
                        v.w[4 * u + i][h][w] &= keep;
                        odd |= not_finite<BF, E8>(v.w[4 * u + i][h][w]);
                    }
            }
        odd = __any(odd);
    }
    u32x4 pw[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float m = st.m[t];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, s[t][u][i] * scale);
        m = rows_max(m);
        const float base = m == -INFINITY ? 0.f : m;
        if (__any(m != st.m[t])) {
            const float alpha = __builtin_amdgcn_exp2f(st.m[t] - base);
            st.l[t] *= alpha;
#pragma unroll
            for (int e = 0; e < State<D, NT>::OPS; ++e) st.o[t][e] *= alpha;
            st.m[t] = m;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][i], scale, -base));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][i + 1], scale, -base));
                st.l[t] += x + y;
                pw[t][2 * u + i / 2] = pack2<BF>(x, y);
            }
    }
#pragma unroll
    for (int h = 0; h < V::HALVES; ++h)
#pragma unroll
        for (int i = 0; i < V::E / 2; ++i) {                  // elements 2 i, 2 i + 1 of the lane's
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (E8) w[j] = i % 2 ? widen2<BF, true>(v.w[j][h][i / 2]) : widen2<BF, false>(v.w[j][h][i / 2]);
                else w[j] = v.w[j][h][i];
            }
            if (!odd) {
#pragma unroll
                for (int e = 2 * i; e < 2 * i + 2; ++e) {
                    const u32x4 vw = turned(w, e);
#pragma unroll
                    for (int t = 0; t < NT; ++t) st.o[t][h * 8 + e] = mfma<BF>(vw, pw[t], st.o[t][h * 8 + e]);
                }
            } else {                                          // rarely: a product a query, without the values that it does not see
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    for (int c = 0; c < 16; ++c) {
                        const int from = __builtin_amdgcn_readlane(lo[t], c), to = __builtin_amdgcn_readlane(hi[t], c);
                        uint32_t x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int at = key + 16 * (j / 4) + 4 * g + j % 4;
                            x[j] = at < from || at >= to ? 0 : w[j];
                        }
#pragma unroll
                        for (int e = 2 * i; e < 2 * i + 2; ++e) {
                            const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                            const f32x4 r = mfma<BF>(turned(x, e), pw[t], zero);
                            if ((lane & 15) == c) st.o[t][h * 8 + e] += r;
                        }
                    }
            }
        }
}

template <int D, bool BF, bool E8, int NT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_kernel(const AttendArgs a) {
    constexpr int ROWS = 16 * NT, OPS = D / 16;
    Piece pc;
    if (!piece_of<ROWS>(a, (int)blockIdx.x, pc)) return;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, g = lane >> 4;
    const Request r = uniform_request(a, pc.b);
    const int k0 = r.lo + pc.at * pc.size, k1 = min(k0 + pc.size, r.hi);
    const int32_t* table = a.tables + pc.b * a.table_row;
    const char *kb = a.k + pc.head * a.k_head, *vb = a.v + pc.head * a.v_head;

    // the lane's queries and the keys that they see
    u32x4 q[NT][D / 32];
    int lo[NT], hi[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = pc.tile * ROWS + 16 * t + (lane & 15), i = row / a.group, gh = row % a.group;
        const bool here = i < r.n;
        hi[t] = here ? max(0, min(r.length - r.n + i + 1, r.hi)) : 0;
        lo[t] = a.window && here ? max(0, r.length - r.n + i + 1 - a.window) : 0;
        const uint16_t* p = a.q + (int64_t)(r.first + (here ? i : 0)) * a.q_row + (int64_t)(pc.head * a.group + gh) * a.q_head;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            q[t][c] = *reinterpret_cast<const u32x4*>(p + (E8 ? c / 2 * 64 + g * 16 + c % 2 * 8 : c * 32 + g * 8));
    }
    // the keys that all of the tile's rows see, and those that any of them does
    const int i0 = pc.tile * ROWS / a.group, i1 = min((pc.tile * ROWS + ROWS - 1) / a.group, r.n - 1);
    const int all_hi = min(r.length - r.n + i0 + 1, r.hi), any_hi = max(0, min(r.length - r.n + i1 + 1, r.hi));
    const int all_lo = a.window ? max(0, r.length - r.n + i1 + 1 - a.window) : 0;
    const int any_lo = a.window ? max(0, r.length - r.n + i0 + 1 - a.window) : 0;

    State<D, NT> st;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        st.m[t] = -INFINITY;
        st.l[t] = 0.f;
#pragma unroll
        for (int e = 0; e < OPS; ++e) st.o[t][e] = {0.f, 0.f, 0.f, 0.f};
    }
    const float scale = E8 ? a.scale * load_uniform(a.ks + pc.head) : a.scale;
    const int end = min(k1, any_hi);
    int key = k0 + STEP * wave;
    if (any_lo > key) key += (any_lo - key) / PIECE * PIECE;
    for (; key < end; key += PIECE) {
        const Pages p = pages_of(a, table, key);
        Keys<D, E8> k;
        Values<D, E8> v;
        load_keys<D, E8>(a, kb, p, lane, k);
        load_values<D, E8>(a, vb, p, lane, v);
        const bool edge = key < all_lo || key + STEP > all_hi || p.page[0] < 0 || p.page[1] < 0;
        step<D, BF, E8, NT>(q, k, v, edge, key, p, lo, hi, any_lo, any_hi, scale, st);
    }

    // the four waves' shares: scaled to one maximum, summed in two rounds through the LDS
    __shared__ float sh_m[WAVES][ROWS], sh_l[WAVES][ROWS];
    __shared__ f32x4 sh_o[2][NT * OPS][64];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        st.l[t] = rows_sum(st.l[t]);
        if (g == 0) {
            sh_m[wave][16 * t + lane] = st.m[t];
            sh_l[wave][16 * t + lane] = st.l[t];
        }
    }
    __syncthreads();
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int c = 16 * t + (lane & 15);
        m[t] = fmaxf(fmaxf(sh_m[0][c], sh_m[1][c]), fmaxf(sh_m[2][c], sh_m[3][c]));
        const float base = m[t] == -INFINITY ? 0.f : m[t];
        l[t] = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) l[t] += sh_l[w][c] * __builtin_amdgcn_exp2f(sh_m[w][c] - base);
        const float alpha = __builtin_amdgcn_exp2f(st.m[t] - base);
#pragma unroll
        for (int e = 0; e < OPS; ++e) st.o[t][e] *= alpha;
    }
#pragma unroll
    for (int round = 2; round > 0; round >>= 1) {             // waves 2, 3 to 0, 1; then wave 1 to 0
        if (wave >= round && wave < 2 * round)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < OPS; ++e) sh_o[wave - round][t * OPS + e][lane] = st.o[t][e];
        __syncthreads();
        if (wave < round)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < OPS; ++e) st.o[t][e] += sh_o[wave][t * OPS + e][lane];
        __syncthreads();
    }
    if (wave != 0) return;
    const float vscale = E8 ? load_uniform(a.vs + pc.head) : 1.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = pc.tile * ROWS + 16 * t + (lane & 15), i = row / a.group, gh = row % a.group;
        if (i >= r.n) continue;
        // operand e of half h, output i of row group g: element 128 h + E (4 g + i) + e
        constexpr int E = Values<D, E8>::E, HALVES = Values<D, E8>::HALVES;
        if (pc.pieces == 1) {
            const float f = l[t] > 0.f ? vscale / l[t] : l[t] == 0.f ? 0.f : __builtin_nanf("");
            uint16_t* to = a.out + (int64_t)(r.first + i) * a.o_row + (int64_t)(pc.head * a.group + gh) * a.o_head;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t w[E / 2];
#pragma unroll
                    for (int e = 0; e < E; e += 2) w[e / 2] = pack2<BF>(st.o[t][h * 8 + e][u] * f, st.o[t][h * 8 + e + 1][u] * f);
                    uint16_t* at = to + 128 * h + E * (4 * g + u);
                    if constexpr (E == 8) *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
                    else *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
                }
        } else {
            float* to = a.part + (pc.slot * ROWS + 16 * t + (lane & 15)) * D;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<float4*>(to + 128 * h + E * (4 * g + u) + e) =
                            make_float4(st.o[t][h * 8 + e][u], st.o[t][h * 8 + e + 1][u], st.o[t][h * 8 + e + 2][u],
                                        st.o[t][h * 8 + e + 3][u]);
            if (g == 0) *reinterpret_cast<float2*>(a.stats + (pc.slot * ROWS + 16 * t + lane) * 2) = make_float2(m[t], l[t]);
        }
    }
}

// The pieces of one row joined: a workgroup a row of a request with more than one; D / 4 lanes a piece, the pieces in order within
// every 256 / (D / 4)-th, then those sums in order
template <int D, bool BF, bool E8, int NT>
__global__ __launch_bounds__(256) void join_kernel(const AttendArgs a) {
    constexpr int ROWS = 16 * NT, LANES = D / 4, SIDE = 256 / LANES;
    __shared__ float4 sh[SIDE][LANES];
    __shared__ float sh_m[4], sh_l[4];
    const int heads = a.Hkv * a.group, head = blockIdx.x % heads, i = blockIdx.x / heads % a.max_new,
              b = blockIdx.x / heads / a.max_new;
    const Request r = uniform_request(a, b);
    if (i >= r.n) return;
    const int2 plan = a.plan[b];
    const int pieces = plan.y;
    if (pieces == 1) return;
    const int row = i * a.group + head % a.group, tiles = (r.n * a.group + ROWS - 1) / ROWS;
    const int64_t slot = plan.x + (int64_t)(head / a.group * tiles + row / ROWS) * pieces;
    const float* part = a.part + (slot * ROWS + row % ROWS) * D;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + slot * ROWS + row % ROWS;
    float m = -INFINITY;
    for (int p = threadIdx.x; p < pieces; p += 256) m = fmaxf(m, stats[(int64_t)p * ROWS].x);
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
        const float2 s = stats[(int64_t)p * ROWS];
        const float4 v = *reinterpret_cast<const float4*>(part + (int64_t)p * ROWS * D + 4 * lane);
        const float w = __builtin_amdgcn_exp2f(s.x - base);
        l += s.y * w;
        o.x += v.x * w;
        o.y += v.y * w;
        o.z += v.z * w;
        o.w += v.w * w;
    }
    sh[side][lane] = o;
    __shared__ float sides[SIDE];
    if (lane == 0) sides[side] = l;
    __syncthreads();
    if (side != 0) return;
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

// ---- the host's side

// Rows a tile: 32 where a request has more than 16
inline int attend_rows(int64_t max_new, int64_t group) { return max_new * group > 16 ? 32 : 16; }

struct AttendSizes {
    int64_t tiles, items, slots, part, stats, bytes;          // offsets in bytes behind the plan
    AttendSizes(int64_t B, int64_t max_new, int64_t group, int64_t Hkv, int64_t D, int64_t capacity, int64_t split) {
        const int64_t rows = attend_rows(max_new, group);
        tiles = (max_new * group + rows - 1) / rows * Hkv;
        const int64_t size = split ? split : PIECE, most = (capacity + size - 1) / size;      // pieces a tile, at most
        items = B * tiles * std::max<int64_t>(1, most);
        slots = most > 1 ? items : 0;
        if (!split) {                                          // sum of ceil(k / size) over all tiles: at most TARGET + tiles
            items = std::min(items, B * tiles + TARGET);
            slots = std::min<int64_t>(slots, 2 * TARGET);      // of those with k > size: at most twice sum of k / size
        }
        part = (B * 8 + 15) / 16 * 16;
        stats = part + slots * rows * D * 4;
        bytes = stats + slots * rows * 8;
    }
};

template <int D, bool BF, bool E8, int NT>
void attend_launch(const AttendArgs& a, const AttendSizes& z, hipStream_t st) {
    attend_kernel<D, BF, E8, NT><<<(unsigned)z.items, 256, 0, st>>>(a);
    if (z.slots) join_kernel<D, BF, E8, NT><<<(unsigned)((int64_t)a.B * a.max_new * a.Hkv * a.group), 256, 0, st>>>(a);
}
template <int D, bool BF, bool E8>
void attend_tiles(const AttendArgs& a, const AttendSizes& z, hipStream_t st) {
    attend_rows(a.max_new, a.group) == 16 ? attend_launch<D, BF, E8, 1>(a, z, st) : attend_launch<D, BF, E8, 2>(a, z, st);
}
template <int D>
void attend_types(const AttendArgs& a, const AttendSizes& z, bool bf, bool e8, hipStream_t st) {
    if (bf) e8 ? attend_tiles<D, true, true>(a, z, st) : attend_tiles<D, true, false>(a, z, st);
    else e8 ? attend_tiles<D, false, true>(a, z, st) : attend_tiles<D, false, false>(a, z, st);
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

constexpr int64_t ATTEND_CAPACITY = int64_t(1) << 28;

extern "C" int64_t esp_paged_attention_scratch(int64_t B, int64_t max_new, int64_t Hq, const esp_kv_cache* cache,
                                               int64_t max_pages, int64_t split) {
    if (!cache || B <= 0 || B > (1 << 20) || max_new <= 0 || max_new >= (1 << 24) || cache->heads < 1 || Hq < cache->heads ||
        Hq % cache->heads || Hq > 65536 || cache->page < 1 || max_pages < 0 || max_pages * cache->page > ATTEND_CAPACITY ||
        split < 0 || split % PIECE)
        return 0;
    return AttendSizes(B, max_new, Hq / cache->heads, cache->heads, cache->dim, max_pages * cache->page, split).bytes;
}

extern "C" int esp_paged_attention(const void* q, int64_t q_row, int64_t q_head, int64_t T, int64_t Hq, int dtype,
                                   const esp_kv_cache* cache, const int32_t* tables, int64_t table_row, int64_t max_pages,
                                   const int32_t* lengths, const int32_t* first, const int32_t* n_new, int64_t B,
                                   int64_t max_new, double scale, int64_t window, int64_t split, void* out, int64_t out_row,
                                   int64_t out_head, void* scratch, int64_t scratch_bytes, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16, "paged_attention: dtype must be bf16 or fp16");
    const char* wrong = esp_host::kv_cache_error(cache, dtype);
    ESP_REQUIRE(!wrong, "paged_attention: %s", wrong);
    const esp_kv_cache& c = *cache;
    ESP_REQUIRE(T >= 0 && T < (1 << 24) && B >= 0 && B <= (1 << 20), "paged_attention: at most 2^24 - 1 rows of at most 2^20 requests");
    ESP_REQUIRE(Hq >= c.heads && Hq % c.heads == 0 && Hq <= 65536,
                "paged_attention: the query heads must be a multiple of the cache's, at most 65536");
    ESP_REQUIRE(max_new >= 1 && max_new < (1 << 24), "paged_attention: 1 to 2^24 - 1 new tokens a request");
    ESP_REQUIRE(scale > 0 && scale < 1e30, "paged_attention: the scale must be positive");
    ESP_REQUIRE(window >= 0 && window < (int64_t(1) << 30), "paged_attention: the window must be at least 0 (none), below 2^30");
    ESP_REQUIRE(split >= 0 && split % PIECE == 0 && split < (int64_t(1) << 30), "paged_attention: split must be a multiple of %d (0: by the lengths)", PIECE);
    ESP_REQUIRE(max_pages >= 0 && max_pages * c.page <= ATTEND_CAPACITY, "paged_attention: tables of at most 2^28 tokens");
    if (T == 0 || B == 0) return esp_host::ok();
    ESP_REQUIRE(q && out && lengths && (tables || max_pages == 0) && scratch, "paged_attention: null pointer");
    ESP_REQUIRE(max_pages >= 1, "paged_attention: tables of at least one page");
    ESP_REQUIRE(B == 1 || table_row >= max_pages, "paged_attention: the tables' rows overlap");
    const int64_t strides[4] = {q_row, q_head, out_row, out_head};
    for (const int64_t s : strides)
        ESP_REQUIRE(s >= 0 && s < (int64_t(1) << 32) && s % 8 == 0, "paged_attention: strides must be multiples of 8 elements, below 2^32");
    ESP_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) % 16 == 0, "paged_attention: rows and scratch must be 16-byte aligned");
    ESP_REQUIRE((Hq == 1 || out_head >= c.dim) && (T == 1 || out_row >= (Hq - 1) * out_head + c.dim),
                "paged_attention: the output's rows overlap");
    const int64_t group = Hq / c.heads;
    ESP_REQUIRE(max_new * group < (1 << 24), "paged_attention: at most 2^24 - 1 rows a request and head of the cache");
    // other workgroups still read the queries when one writes its rows
    ESP_REQUIRE(!esp_host::rows_meet(out, out_row * 2, ((Hq - 1) * out_head + c.dim) * 2, q, q_row * 2,
                                     ((Hq - 1) * q_head + c.dim) * 2, T), "paged_attention: the output overlaps q");
    const AttendSizes z(B, max_new, group, c.heads, c.dim, max_pages * c.page, split);
    ESP_REQUIRE(z.items < (1 << 24) && B * max_new * Hq < (int64_t(1) << 31), "paged_attention: at most 2^24 - 1 pieces of tiles");
    ESP_REQUIRE(scratch_bytes >= z.bytes, "paged_attention: the scratch needs esp_paged_attention_scratch bytes");
    AttendArgs a;
    a.q = static_cast<const uint16_t*>(q);
    a.q_row = q_row;
    a.q_head = q_head;
    a.out = static_cast<uint16_t*>(out);
    a.o_row = out_row;
    a.o_head = out_head;
    const int64_t size = kv_bytes(c.dtype);
    a.k = static_cast<const char*>(c.k);
    a.v = static_cast<const char*>(c.v);
    a.k_page = c.k_page * size;
    a.k_token = c.k_token * size;
    a.k_head = c.k_head * size;
    a.v_page = c.v_page * size;
    a.v_token = c.v_token * size;
    a.v_head = c.v_head * size;
    a.pages = c.pages;
    a.ks = c.k_scale;
    a.vs = c.v_scale;
    a.tables = tables;
    a.table_row = table_row;
    a.lengths = lengths;
    a.first = first;
    a.n_new = n_new;
    char* base = static_cast<char*>(scratch);
    a.plan = reinterpret_cast<int2*>(base);
    a.part = reinterpret_cast<float*>(base + z.part);
    a.stats = reinterpret_cast<float*>(base + z.stats);
    a.B = (int)B;
    a.T = (int)T;
    a.Hkv = (int)c.heads;
    a.group = (int)group;
    a.max_new = (int)max_new;
    a.window = (int)window;
    a.split = (int)split;
    a.capacity = (int)(max_pages * c.page);
    a.page16 = (int)(c.page / 16);
    a.page_shift = 31 - __builtin_clz((unsigned)a.page16);
    a.page_mul = (uint32_t)(((uint64_t(1) << (31 + a.page_shift)) + a.page16 - 1) / a.page16);
    a.scale = (float)(scale * 1.4426950408889634);
    const hipStream_t st = (hipStream_t)stream;
    const bool bf = dtype == ESP_BF16, e8 = c.dtype == ESP_E4M3;
    if (c.dim == 64) attend_types<64>(a, z, bf, e8, st);
    else if (c.dim == 128) attend_types<128>(a, z, bf, e8, st);
    else attend_types<256>(a, z, bf, e8, st);
    return esp_host::launch_check("paged_attention");
}
