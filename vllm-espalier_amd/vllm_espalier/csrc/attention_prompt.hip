// Attention over a paged cache for requests of many rows (prompts): attention.hip's mathematics in tiles of 128 rows.
//
// A workgroup takes 128 rows of a request and head of the cache, a wave 32 of them, and walks over the keys 64 at a time: keys and
// values come into the LDS (16-bit caches: straight from memory, e4m3: through registers, widened), the next 64 while these are used. As
// there, S^T = K Q^T leaves a wave's lanes with the scores of one query each (32 x 32 products: half a query, 16 of its 32 keys), and
// they are what O^T = V^T P^T wants; V^T comes from the LDS by its transposed reads, 4 keys of an element at a time. A query's
// statistics are two lanes' business.
//
// The maximum that the weights are taken from may lie up to LAG below the largest score (as exponents of 2): sums and outputs, fp32, keep
// their relative errors, and the outputs are rarely scaled.
//
// LDS rows are the head's elements in pieces of 16 bytes, piece c of key r at c ^ spread(r): the 16 keys that a read of K goes through
// at one piece lie in different banks, and so do the 4 keys of 64 bytes that a transposed read goes through.
//
// What bounds it is neither products nor memory alone but a wave's order: its products (34 % of the cycles), then its softmax (41 %
// on the vector units), with two waves a SIMD to fill in for each other, which is what the registers of 32 x 128 outputs leave.
// Three requests of up to 2048 new tokens over up to 4096, heads 32/4 of 128, bf16 (105 GFLOP of visible pairs): 134 to 139 us
// a pass with its join (0.78 PFLOP/s; a kernel trace, which slows it, has 143 at least), where the tiles that see most decide the end;
// one of 4096 over 8192, heads 32/8 (412 GFLOP), 445 us (0.93 PFLOP/s).
// A large matrix product reaches 1.5.
#include "attention_few.hpp"

namespace esp {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
using global_void_ptr = const __attribute__((address_space(1))) void*;
using lds_void_ptr = __attribute__((address_space(3))) void*;

constexpr int TILE = 64;                       // keys in the LDS
// (fp16: what reference() leaves of its range. The outputs are scaled more often: 4 prompts of 1024 over 3071, 32/4 heads of 64 125 us for
// 123 with 8, 16/2 of 256 252 for 235)
template <bool BF>
constexpr float LAG = BF ? 8.0f : 2.0f;

__device__ const uint4 no_keys[1] = {};        // what keys that nobody sees are read from

template <int D>
__device__ __forceinline__ int spread(int r) {
    return D == 64 ? (r >> 1 & 1) * 4 + (r >> 2 & 3) : (r & 3) * 4 + (r >> 2 & 3);
}

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// the other half's value
__device__ __forceinline__ float halves_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}

// A wave's 16 keys of a tile: pieces straight into the LDS, or 8-bit ones into registers and from there
template <int D, bool E8>
struct Loader {
    static constexpr int ROW = D * 2, N = E8 ? D / 64 : D / 32, UNITS = E8 ? D / 16 : D / 8;      // LDS bytes a row; loads; their pieces a row
    u32x4 held[E8 ? 2 * N : 1];
    uint32_t k_at[N], v_at[N];                                // where the lane reads, from the first key

    __device__ __forceinline__ explicit Loader(const AttendArgs& a) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int unit = i * 64 + (int)(threadIdx.x & 63), r = unit / UNITS, c = unit % UNITS;
            k_at[i] = r * (int)a.k_token + (E8 ? c : c ^ spread<D>(r)) * 16;
            v_at[i] = r * (int)a.v_token + (E8 ? c : c ^ spread<D>(r)) * 16;
        }
    }
    // part: only the keys in [lo, hi) of them, and none without a page, are anybody's
    __device__ __forceinline__ void load(const AttendArgs& a, const char* kb, const char* vb, int page, int off, bool part, int key, int lo,
                                         int hi, char* lds) {
        const char *k = kb + (int64_t)max(page, 0) * a.k_page + off * a.k_token, *v = vb + (int64_t)max(page, 0) * a.v_page + off * a.v_token;
        const auto one = [&](int i, const char* ks, const char* vs) __attribute__((always_inline)) {
            if constexpr (E8) {
                held[i] = *reinterpret_cast<const u32x4*>(ks);
                held[N + i] = *reinterpret_cast<const u32x4*>(vs);
            } else {
                __builtin_amdgcn_global_load_lds((global_void_ptr)ks, (lds_void_ptr)(lds + i * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((global_void_ptr)vs, (lds_void_ptr)(lds + TILE * ROW + i * 1024), 16, 0, 0);
            }
        };
        if (!part) {
#pragma unroll
            for (int i = 0; i < N; ++i) one(i, k + k_at[i], v + v_at[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = key + (i * 64 + (int)(threadIdx.x & 63)) / UNITS;
                const bool none = page < 0 || at < lo || at >= hi;
                const char* zeros = reinterpret_cast<const char*>(no_keys);
                one(i, none ? zeros : k + k_at[i], none ? zeros : v + v_at[i]);
            }
        }
    }
    template <bool BF>
    __device__ __forceinline__ void store(char* lds) const {
        if constexpr (E8) {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) {
                const int unit = i % N * 64 + lane, r = unit / (D / 16), c = unit % (D / 16);
                char* row = lds + (i < N ? 0 : TILE * ROW) + r * ROW;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = held[i][2 * h], y = held[i][2 * h + 1];
                    const u32x4 w = {widen2<BF, false>(x), widen2<BF, true>(x), widen2<BF, false>(y), widen2<BF, true>(y)};
                    *reinterpret_cast<u32x4*>(row + ((2 * c + h) ^ spread<D>(r)) * 16) = w;
                }
            }
        }
    }
};

// (three waves a SIMD hold the plain heads of 64 by themselves in bf16; fp16, one register over, has to be told)
template <int D, bool BF, bool E8>
__global__ __launch_bounds__(256, D == 256 ? 1 : D == 64 && !E8 && !BF ? 3 : 2) void attend_prompt_kernel(const AttendArgs a) {
    constexpr int ROWS = PROMPT_ROWS, ROW = D * 2, KK = D / 16, DB = D / 32, BUFFER = 2 * TILE * ROW;
    constexpr int K_AHEAD = D == 256 ? 1 : 2, V_AHEAD = D == 256 ? 2 : 4;     // steps that operands are read ahead of their products
    // two buffers, each an object of its own and each step of the loop with its own: a read of one is then known not to wait for what
    // is on its way into the other
    __shared__ __attribute__((aligned(1024))) char lds0[BUFFER], lds1[BUFFER];
    if constexpr (FEW_TOO<D>) {
        static_assert(FEW_LDS<D, 2> <= BUFFER, "the few rows' shares");
        if ((int)blockIdx.x >= a.many) {                      // behind the others: they fill in where these end
            attend_few<D, BF, E8, 2>(a, (int)blockIdx.x - a.many, lds0);
            return;
        }
    }
    Piece pc;
    if (!piece_of<ROWS>(a, (int)blockIdx.x, pc)) return;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, h = lane >> 5;
    const Request& r = pc.r;
    const int32_t* table = a.tables + pc.b * a.table_row;
    const char *kb = a.k + pc.head * a.k_head, *vb = a.v + pc.head * a.v_head;

    // the lane's query, the keys that it sees, those that all and any of the wave's do, and those that any of the workgroup's do
    const int before = r.length - r.n + 1, row0 = pc.tile * ROWS + 32 * wave, row = row0 + (lane & 31), i = quotient(row, a.group), gh = row - i * a.group;
    const bool here = i < r.n, some = row0 < r.n * a.group;
    // (readfirstlane: what all lanes share is kept in scalar registers)
    const auto shared = [](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(v); };
    const auto upto = [&](int t) __attribute__((always_inline)) { return max(0, min(before + t, r.hi)); };
    const auto from = [&](int t) __attribute__((always_inline)) { return a.window ? max(0, before + t - a.window) : 0; };
    const int hi = here ? upto(i) : 0, lo = here ? from(i) : 0;
    const int i0 = shared(quotient(row0, a.group)), i1 = min(shared(quotient(row0 + 31, a.group)), r.n - 1);
    const int wg_i0 = shared(quotient(pc.tile * ROWS, a.group)), wg_i1 = min(shared(quotient(pc.tile * ROWS + ROWS - 1, a.group)), r.n - 1);
    const int all_hi = shared(upto(i0)), any_hi = shared(upto(i1)), all_lo = shared(from(i1)), any_lo = shared(from(i0));
    const int wg_hi = shared(upto(wg_i1)), wg_lo = shared(from(wg_i0));
    u32x4 q[KK];
    {
        const uint16_t* p = a.q + (int64_t)(r.first + (here ? i : 0)) * a.q_row + (int64_t)(pc.head * a.group + gh) * a.q_head;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) q[kk] = *reinterpret_cast<const u32x4*>(p + kk * 16 + h * 8);
    }
    const int k0 = shared(r.lo + pc.at * pc.size), end = shared(min(min(k0 + pc.size, r.hi), wg_hi));
    const int start = shared(k0 + (wg_lo > k0 ? (wg_lo - k0) / TILE * TILE : 0));

    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[db][j] = 0.f;
    float m = -INFINITY, l = 0.f, over = -INFINITY;          // over: reference(m), of fp16 (made from m for every tile it costs 27 registers)
    const float scale = E8 ? a.scale * load_uniform(a.ks + pc.head) : a.scale;

    // where the lane reads: K operand kk of key lane % 32; V^T, elements 32 db + lane % 32, keys 4 h .. of 16 (and 8 further on)
    const int kr = (lane & 31) * ROW, kf = spread<D>(lane & 31);
    const int vi = lane & 15, vr = (4 * h + (vi >> 2)) * ROW, vf = spread<D>(4 * h + (vi >> 2)), vp = (lane >> 4 & 1) * 2 + (vi >> 1 & 1);
    const auto read_k = [&](const char* buf, int kb32, int kk) __attribute__((always_inline)) {
        return *reinterpret_cast<const u32x4*>(buf + kb32 * 32 * ROW + kr + (((2 * kk + h) ^ kf) << 4));
    };
    const auto read_v = [&](const char* buf, int st, int db) __attribute__((always_inline)) {
        const char* at = buf + TILE * ROW + st * 16 * ROW + vr + (vi & 1) * 8;
        const int c = (db * 4 + vp) ^ vf;
        typedef __attribute__((address_space(3))) s16x4* tr_ptr;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + (c << 4)));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(at + 8 * ROW + ((c ^ 2) << 4)));
        const uint2 u = __builtin_bit_cast(uint2, x), w = __builtin_bit_cast(uint2, y);
        return u32x4{u.x, u.y, w.x, w.y};
    };

    Loader<D, E8> loader(a);
    const int mine = 16 * wave;                               // the wave's keys of a tile
    // Lane i: the page of the wave's keys of tile i from where it was last asked, and which of the tile's 16 keys have none
    Place ahead = {};
    int none_ahead = 0, tiles = 0;
    const auto load = [&](int key, char* lds) __attribute__((always_inline)) {
        if (tiles == 0) {
            none_ahead = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const Place p = place_of(a, table, key + lane * TILE + 16 * u);
                if (p.page < 0) none_ahead |= 1 << u;
                if (u == wave) ahead = p;
            }
        }
        const int none = __builtin_amdgcn_readlane(none_ahead, tiles);
        const bool part = none || key < wg_lo || key + TILE > wg_hi;
        loader.load(a, kb, vb, __builtin_amdgcn_readlane(ahead.page, tiles), __builtin_amdgcn_readlane(ahead.off, tiles), part, key + mine,
                    wg_lo, wg_hi, lds + mine * ROW);
        tiles = (tiles + 1) & 63;
        return none;
    };
    int none_next = 0;
    if (start < end) {
        none_next = load(start, lds0);
        loader.template store<BF>(lds0 + mine * ROW);
    }
    const int wg_all_hi = shared(upto(wg_i0)), wg_all_lo = shared(from(wg_i1));
    bool odd = false;                                         // a NaN or an infinity among values that some rows see and others do not
    const auto tile = [&](int key, char* buf, char* other) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);                        // this wave's part of the tile has come
        if (key < wg_all_lo || key + TILE > wg_all_hi || none_next) {
            u32x4* v = reinterpret_cast<u32x4*>(buf + (TILE + mine) * ROW) + lane;
#pragma unroll
            for (int c = 0; c < ROW / 64; ++c) {
                const u32x4 w = v[c * 64];
                const u32x4 f = {finite<BF, false>(w[0]), finite<BF, false>(w[1]), finite<BF, false>(w[2]), finite<BF, false>(w[3])};
                odd |= f[0] != w[0] || f[1] != w[1] || f[2] != w[2] || f[3] != w[3];
                v[c * 64] = f;
            }
        }
        __syncthreads();                                      // and everybody's; the other buffer is read by nobody any more
        const int next = key + TILE;
        const int none = none_next;                           // which 16 keys have no page
        if (next < end) none_next = load(next, other);
        if (some && key < any_hi && key + TILE > any_lo) {
            f32x16 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[u][j] = 0.f;
            u32x4 k[K_AHEAD + 1][2];                          // operands some steps ahead
#pragma unroll
            for (int kk = 0; kk < K_AHEAD; ++kk)
#pragma unroll
                for (int u = 0; u < 2; ++u) k[kk][u] = read_k(buf, u, kk);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (kk + K_AHEAD < KK)
#pragma unroll
                    for (int u = 0; u < 2; ++u) k[(kk + K_AHEAD) % (K_AHEAD + 1)][u] = read_k(buf, u, kk + K_AHEAD);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 2; ++u) s[u] = mfma32<BF>(k[kk % (K_AHEAD + 1)][u], q[kk], s[u]);
            }
            u32x4 v[V_AHEAD + 1];
#pragma unroll
            for (int n = 0; n < V_AHEAD; ++n) v[n] = read_v(buf, n / DB, n % DB);
            const bool edge = key < all_lo || key + TILE > all_hi || none;
            if (edge) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int t = 32 * u + 8 * (j / 4) + 4 * h + j % 4;
                        if (key + t < lo || key + t >= hi || (none >> (2 * u + j / 8) & 1)) s[u][j] = -INFINITY;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int j = 1; j < 16; ++j) top = fmaxf(top, s[0][j]);
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, s[1][j]);
            top = halves_max(top) * scale;
            if (__any(top > m + LAG<BF>)) {
                const float next_m = fmaxf(m, top);
                const float next = reference<BF>(next_m), alpha = __builtin_amdgcn_exp2f((BF ? m : over) - (next == -INFINITY ? 0.f : next));
                m = next_m;
                over = next;
                l *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db] *= alpha;
            }
            const float base = (BF ? m : over) == -INFINITY ? 0.f : BF ? m : over;
            u32x4 p[4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], scale, -base));
                    const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j + 1], scale, -base));
                    l += x + y;
                    p[2 * u + j / 8][j % 8 / 2] = pack2<BF>(x, y);
                }
#pragma unroll
            for (int n = 0; n < 4 * DB; ++n) {
                if (n + V_AHEAD < 4 * DB) v[(n + V_AHEAD) % (V_AHEAD + 1)] = read_v(buf, (n + V_AHEAD) / DB, (n + V_AHEAD) % DB);
                if constexpr (D != 64) __builtin_amdgcn_sched_barrier(0);      // (there the registers hold more: 87 -> 82 us)
                o[n % DB] = mfma32<BF>(v[n % (V_AHEAD + 1)], p[n / DB], o[n % DB]);
            }
        }
        if (next < end) loader.template store<BF>(other + mine * ROW);
    };
    for (int key = start; key < end; key += 2 * TILE) {
        tile(key, lds0, lds1);
        if (key + TILE < end) tile(key + TILE, lds1, lds0);
    }

    l = halves_sum(l);
    const float vscale = E8 ? load_uniform(a.vs + pc.head) : 1.f;
    // output j of block db: element 32 db + 8 (j / 4) + 4 h + j % 4
    if (here && pc.pieces == 1) {
        const float f = l > 0.f ? vscale / l : l == 0.f ? 0.f : __builtin_nanf("");
        uint16_t* to = a.out + (int64_t)(r.first + i) * a.o_row + (int64_t)(pc.head * a.group + gh) * a.o_head + 4 * h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<uint2*>(to + 32 * db + 2 * j) =
                    make_uint2(pack2<BF>(o[db][j] * f, o[db][j + 1] * f), pack2<BF>(o[db][j + 2] * f, o[db][j + 3] * f));
    } else if (here) {
        const int64_t at = pc.row + (32 * wave + (lane & 31)) * pc.pieces;
        float* to = a.part + at * D + 4 * h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<float4*>(to + 32 * db + 2 * j) = make_float4(o[db][j], o[db][j + 1], o[db][j + 2], o[db][j + 3]);
        if (h == 0) a.stats[at] = make_float2(BF ? m : over, l);
    }
    if (__syncthreads_or(odd)) mark_not_finite<D, BF, E8, ROWS>(a, pc, r, table, start, end);
}

template <int D, bool BF, bool E8>
void prompt_launch(const AttendArgs& a, const AttendSizes& z, hipStream_t st) {
    attend_prompt_kernel<D, BF, E8><<<(unsigned)(z.many + (FEW_TOO<D> ? z.few : 0)), 256, 0, st>>>(a);
}
template <int D>
void prompt_types(const AttendArgs& a, const AttendSizes& z, bool bf, bool e8, hipStream_t st) {
    if (bf) e8 ? prompt_launch<D, true, true>(a, z, st) : prompt_launch<D, true, false>(a, z, st);
    else e8 ? prompt_launch<D, false, true>(a, z, st) : prompt_launch<D, false, false>(a, z, st);
}

void attend_prompt(const AttendArgs& a, const AttendSizes& z, int D, bool bf, bool e8, hipStream_t st) {
    if (D == 64) prompt_types<64>(a, z, bf, e8, st);
    else if (D == 128) prompt_types<128>(a, z, bf, e8, st);
    else prompt_types<256>(a, z, bf, e8, st);
}

}  // namespace esp
