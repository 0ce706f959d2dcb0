// The kernels' program for a request of up to FEW_ROWS rows a head of the cache (attention.hip's comment), which attention_prompt.hip's
// launch runs too, for the requests of few rows in its batch.
#pragma once

#include "attention.hpp"

namespace esp {

// The pages of a step's two times 16 keys (-1: none), and the keys' places in them
struct Pages {
    int page[2], off[2];
};

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
        const char* row = base + (int64_t)max(p.page[u], 0) * a.k_page + p.off[u] * a.k_token;
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
        const char* row = base + (int64_t)max(p.page[j / 4], 0) * a.v_page + (p.off[j / 4] + j % 4) * a.v_token;
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

// The scores of 32 keys
template <int D, bool BF, bool E8, int NT>
__device__ __forceinline__ void scores(const u32x4 (&q)[NT][D / 32], const Keys<D, E8>& k, f32x4 (&s)[NT][2]) {
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
}

// 32 keys from `key` by their scores and values; whether values went in as zeros (mark_not_finite). edge: some of them are not every row's. hi, lo: the keys [lo, hi) that the lane's query sees
template <int D, bool BF, bool E8, int NT>
__device__ __forceinline__ bool weigh(f32x4 (&s)[NT][2], Values<D, E8>& v, bool edge, int key, const Pages& p, const int (&lo)[NT],
                                      const int (&hi)[NT], int any_lo, int any_hi, float scale, State<D, NT>& st) {
    using V = Values<D, E8>;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    bool odd = false;
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
                        const uint32_t x = v.w[4 * u + i][h][w] & keep, f = finite<BF, E8>(x);
                        odd |= f != x;
                        v.w[4 * u + i][h][w] = f;
                    }
            }
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
        const float base = m == -INFINITY ? 0.f : reference<BF>(m);
        if (__any(m != st.m[t])) {
            const float alpha = __builtin_amdgcn_exp2f(reference<BF>(st.m[t]) - base);
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
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                const u32x4 vw = turned(w, e);
#pragma unroll
                for (int t = 0; t < NT; ++t) st.o[t][h * 8 + e] = mfma<BF>(vw, pw[t], st.o[t][h * 8 + e]);
            }
        }
    return odd;
}

// Piece `item` of the requests of few rows, by a workgroup. lds: 32 rows of D floats, the shares of two waves
template <int D, int NT>
constexpr int FEW_LDS = 2 * NT * (D / 16) * 64 * 16;
template <int D, bool BF, bool E8, int NT>
__device__ __forceinline__ void attend_few(const AttendArgs& a, int item, char* lds) {
    constexpr int ROWS = 16 * NT, OPS = D / 16;
    // All arguments at once: left to where they are used, they come one after the other, a trip to memory each (one token over 113, in turn without:
    // 6.45 -> 6.2 us a pass)
    asm volatile("" ::"s"(a.lengths), "s"(a.first), "s"(a.n_new), "s"(a.tables), "s"(a.table_row), "s"(a.q), "s"(a.q_row), "s"(a.q_head),
                 "s"(a.k), "s"(a.v), "s"(a.k_page), "s"(a.k_token), "s"(a.k_head), "s"(a.v_page), "s"(a.v_token), "s"(a.v_head),
                 "s"(a.pages), "s"(a.B), "s"(a.T), "s"(a.Hkv), "s"(a.group), "s"(a.max_new), "s"(a.window), "s"(a.split), "s"(a.capacity),
                 "s"(a.page16), "s"(a.page_shift), "s"(a.page_mul), "s"(a.slots));
    Piece pc;
    if (!piece_of<ROWS>(a, item, pc)) return;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, g = lane >> 4;
    const Request& r = pc.r;
    // (readfirstlane: what all lanes share is kept in scalar registers)
    const auto shared = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
    const int k0 = shared(r.lo + pc.at * pc.size), k1 = shared(min(k0 + pc.size, r.hi));
    const int32_t* table = a.tables + pc.b * a.table_row;
    const char *kb = a.k + pc.head * a.k_head, *vb = a.v + pc.head * a.v_head;

    // the lane's queries and the keys that they see
    u32x4 q[NT][D / 32];
    int lo[NT], hi[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = 16 * t + (lane & 15), i = quotient(row, a.group), gh = row - i * a.group;
        const bool here = i < r.n;
        hi[t] = here ? max(0, min(r.length - r.n + i + 1, r.hi)) : 0;
        lo[t] = a.window && here ? max(0, r.length - r.n + i + 1 - a.window) : 0;
        const uint16_t* p = a.q + (int64_t)(r.first + (here ? i : 0)) * a.q_row + (int64_t)(pc.head * a.group + gh) * a.q_head;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            q[t][c] = *reinterpret_cast<const u32x4*>(p + (E8 ? c / 2 * 64 + g * 16 + c % 2 * 8 : c * 32 + g * 8));
    }
    // the keys that all of the tile's rows see, and those that any of them does
    const int i0 = 0, i1 = r.n - 1;                           // (a request is one tile)
    const int all_hi = shared(min(r.length - r.n + i0 + 1, r.hi)), any_hi = shared(max(0, min(r.length - r.n + i1 + 1, r.hi)));
    const int all_lo = shared(a.window ? max(0, r.length - r.n + i1 + 1 - a.window) : 0);
    const int any_lo = shared(a.window ? max(0, r.length - r.n + i0 + 1 - a.window) : 0);

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
    bool odd = false;
    int key = k0 + STEP * wave;
    if (any_lo > key) key += (any_lo - key) / PIECE * PIECE;
    // Lane 2 i + u: the page of the wave's 16 keys u of step i from where it was last asked, 32 steps at once
    Place ahead = {};
    int steps = 0;
    const auto pages_at = [&](int from) __attribute__((always_inline)) {
        if (steps == 0) ahead = place_of(a, table, from + (lane >> 1) * PIECE + 16 * (lane & 1));
        Pages p;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            p.page[u] = __builtin_amdgcn_readlane(ahead.page, 2 * steps + u);
            p.off[u] = __builtin_amdgcn_readlane(ahead.off, 2 * steps + u);
        }
        steps = (steps + 1) & 31;
        return p;
    };
    if (key < end) {
        Pages p = pages_at(key);
        Keys<D, E8> k;
        Values<D, E8> v;
        load_keys<D, E8>(a, kb, p, lane, k);
        load_values<D, E8>(a, vb, p, lane, v);
        while (true) {                                        // the next keys are on their way while these are weighed, the next
            const int next = key + PIECE;                     // values as soon as these are added up
            const bool more = next < end;
            f32x4 s[NT][2];
            scores<D, BF, E8, NT>(q, k, s);
            const Pages now = p;
            if (more) {
                p = pages_at(next);
                load_keys<D, E8>(a, kb, p, lane, k);
            }
            const bool edge = key < all_lo || key + STEP > all_hi || now.page[0] < 0 || now.page[1] < 0;
            odd |= weigh<D, BF, E8, NT>(s, v, edge, key, now, lo, hi, any_lo, any_hi, scale, st);
            if (!more) break;
            load_values<D, E8>(a, vb, p, lane, v);
            key = next;
        }
    }

    // the four waves' shares: scaled to one maximum, summed in two rounds through the LDS
    __shared__ float sh_m[WAVES][ROWS], sh_l[WAVES][ROWS];
    f32x4(*sh_o)[NT * OPS][64] = reinterpret_cast<f32x4(*)[NT * OPS][64]>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        st.m[t] = reference<BF>(st.m[t]);                     // (from here on what the sums are over)
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
    const float vscale = E8 ? load_uniform(a.vs + pc.head) : 1.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = 16 * t + (lane & 15), i = quotient(row, a.group), gh = row - i * a.group;
        if (wave != 0 || i >= r.n) continue;
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
            const int64_t at = pc.row + (16 * t + (lane & 15)) * pc.pieces;
            float* to = a.part + at * D;
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<float4*>(to + 128 * h + E * (4 * g + u) + e) =
                            make_float4(st.o[t][h * 8 + e][u], st.o[t][h * 8 + e + 1][u], st.o[t][h * 8 + e + 2][u],
                                        st.o[t][h * 8 + e + 3][u]);
            if (g == 0) a.stats[at] = make_float2(m[t], l[t]);
        }
    }
    if (__syncthreads_or(odd)) mark_not_finite<D, BF, E8, ROWS>(a, pc, r, table, k0, end);
}

}  // namespace esp
