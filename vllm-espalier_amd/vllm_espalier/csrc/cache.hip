// New keys and values into a paged cache, with the norms of queries and keys a head and the rotation of positions on the way, on
// gfx950. For a row x of a head of D elements (queries and keys):
//   u = (x * inv(x)) * w,  inv(x) = 1 / sqrt(mean(x^2) + eps)   (u = x without a norm)
//   (a, b) -> s * (a cos t - b sin t, b cos t + a sin t)        for the pairs f < half of its first 2 half elements,
//   t = position(axis of f) * inv_freq[f]
// in fp32, rounded once where it is stored: queries to their output, keys and the values (as they are) to their token's slot.
//
// One launch. A lane holds 8 elements (16 bytes) of a row, so a wave holds 512 / D rows and a row's sum runs over the lanes of
// its own; the partner of a half-split pair lies half / 8 lanes further. The angles of a token are shared by all of its rows:
// a workgroup makes them first, into the LDS, in fp64 up to the fraction of a turn (a far position leaves few of 32 bits for it).
// A lane keeps the two factors of each of its elements for all rows of a kind, its weight times the cosine and its partner's times
// the sine, so that an element is inv * (x * a + partner * b), with the partners exchanged as they were loaded, two to a word.
#include "kv.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t q_row, k_row, v_row, o_row;                       // elements
    uint32_t q_head, k_head, v_head, o_head;
    uint16_t* out;
    char *kc, *vc;
    int64_t kc_page, kc_token, kc_head, vc_page, vc_token, vc_head, pages;
    const int64_t *slots, *positions;
    int64_t pos_axis;                                          // elements between two axes' positions
    const double* inv_freq;
    const int32_t* axes;                                       // the axis of a frequency; null: the first
    const uint16_t *wq, *wk;
    const float *ks, *vs;
    int T, Hq, Hkv, n_axes, half, page, adjacent;
    float eps, rot_scale;
};

// the sum over the LANES lanes of a row (8, 16 or 32 neighbours), in every one of them
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_f32<0xB1>(v);                                     // quad_perm [1,0,3,2]
    v += dpp_f32<0x4E>(v);                                     // quad_perm [2,3,0,1]
    v += dpp_f32<0x141>(v);                                    // row_half_mirror
    if constexpr (LANES >= 16) v += dpp_f32<0x140>(v);         // row_mirror
    if constexpr (LANES >= 32) v += xor_lane32<16>(v);
    return v;
}

__device__ __forceinline__ void unpack8(uint4 u, bool bf, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = from16((uint16_t)(w[k] & 0xFFFFu), bf);
        v[2 * k + 1] = from16((uint16_t)(w[k] >> 16), bf);
    }
}

// What a lane needs of one kind of rows: its factors (see above), and where its partners are
struct Turn {
    float a[8], b[8];
    int from;                                                 // the partner's lane times 4, of a half-split pair
    bool turns;
};
struct Weights {                                              // a lane's, and its partner's
    uint4 own, other;
};
template <int D>
__device__ __forceinline__ Weights weights_of(const AppendArgs& p, const uint16_t* weight, int lane) {
    const int d = lane % (D / 8) * 8, half = p.half;
    const int other = d < 2 * half && !p.adjacent ? (d < half ? d + half : d - half) : d;
    Weights w = {};
    if (weight) w = {*reinterpret_cast<const uint4*>(weight + d), *reinterpret_cast<const uint4*>(weight + other)};
    return w;
}
template <int D, bool BF>
__device__ __forceinline__ Turn turn_of(const AppendArgs& p, const float2* turn, const uint16_t* weight, const Weights& u, int lane) {
    const int d = lane % (D / 8) * 8, half = p.half;
    Turn t;
    t.turns = d < 2 * half;
    const bool low = d < half;
    t.from = t.turns && !p.adjacent ? (lane + (low ? half / 8 : -(half / 8))) * 4 : lane * 4;
    float w[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[j] = 1.f;
    if (weight) {
        unpack8(u.own, BF, w);
        unpack8(u.other, BF, v);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 cs = !t.turns ? make_float2(1.f, 0.f) : p.adjacent ? turn[d / 2 + j / 2] : turn[d % half + j];
        const bool first = p.adjacent ? j % 2 == 0 : low;
        t.a[j] = w[j] * cs.x;
        t.b[j] = t.turns ? (p.adjacent ? v[j ^ 1] : v[j]) * (first ? -cs.y : cs.y) : -0.0f;      // (a zero keeps its sign)
    }
    return t;
}
// Rows as loaded, through their norm and turn
template <int D, bool BF>
__device__ __forceinline__ void turned(const AppendArgs& p, const Turn& t, bool norm, uint4 raw, float (&x)[8]) {
    unpack8(raw, BF, x);
    float o[8];
    if (p.adjacent) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t.turns ? x[j ^ 1] : 0.f;
    } else {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u[k] = (uint32_t)__builtin_amdgcn_ds_bpermute(t.from, (int)w[k]);
            u[k] = t.turns ? u[k] : 0u;                       // (0 * infinity would be a NaN)
        }
        unpack8(make_uint4(u[0], u[1], u[2], u[3]), BF, o);
    }
    float inv = 1.f;
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
        inv = __builtin_amdgcn_rsqf(row_sum<D / 8>(ss) * (1.0f / D) + p.eps);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf(o[j], t.b[j], x[j] * t.a[j]) * inv;
}

// x / scale from 1 / scale, to nearest: many quotients of 16-bit values lie on the borders of 8-bit ones, and the product alone, off by
// one last place, would put them on either side (beyond what eight bits hold it does, infinities among it; a zero keeps its sign)
__device__ __forceinline__ float quotient_of(float x, float scale, float over) {
    const float q = x * over;
    return q != 0.0f && fabsf(q) <= 1024.0f ? __builtin_fmaf(__builtin_fmaf(-q, scale, x), over, q) : q;
}

// one of three values by a row's kind (by value: the arguments stay where they are)
template <typename T>
__device__ __forceinline__ T of_kind(int kind, T q, T k, T v) {
    return kind == 0 ? q : kind == 1 ? k : v;
}

// The rows of TOKENS tokens, a wave's worth of one kind (queries, keys, values) at a time: a workgroup takes all of TOKENS tokens' (a
// wave a token; TOKENS 4), or a share of one token's (TOKENS 1: gridDim.y of them)
template <int D, bool BF, bool E8, int TOKENS>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
    constexpr int LANES = D / 8, ROWS = 64 / LANES;           // lanes a row, rows a wave
    __shared__ float2 turn[TOKENS][D / 2];                    // (cos, sin) of a token's angles
    const int t0 = blockIdx.x * TOKENS, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int token = TOKENS == 1 ? 0 : wave, t = min(t0 + token, a.T - 1), d = lane % LANES * 8, sub = lane / LANES;
    const int q_passes = (a.Hq + ROWS - 1) / ROWS, kv_passes = (a.Hkv + ROWS - 1) / ROWS, passes = q_passes + 2 * kv_passes;
    const int first = TOKENS == 1 ? (int)(blockIdx.y * 4) + wave : (int)blockIdx.y, step = (int)gridDim.y * (TOKENS == 1 ? 4 : 1);
    // a pass's rows as they are in memory (those past the last head: the last head's again)
    const uint16_t *q_at = a.q + t * a.q_row, *k_at = a.k + t * a.k_row, *v_at = a.v + t * a.v_row;
    const auto kind_of = [&](int g) __attribute__((always_inline)) { return (g >= q_passes) + (g >= q_passes + kv_passes); };
    const auto head_of = [&](int g, int kind) __attribute__((always_inline)) {
        return (g - of_kind(kind, 0, q_passes, q_passes + kv_passes)) * ROWS + sub;
    };
    const auto raw_of = [&](int g) __attribute__((always_inline)) {
        const int kind = kind_of(g);
        const uint32_t head = min(head_of(g, kind), of_kind(kind, a.Hq, a.Hkv, a.Hkv) - 1);
        return *reinterpret_cast<const uint4*>(of_kind(kind, q_at, k_at, v_at) +
                                               (uint64_t)head * of_kind(kind, a.q_head, a.k_head, a.v_head) + d);
    };
    uint4 raw = make_uint4(0, 0, 0, 0);
    Weights weights = {};
    if (first < passes) {                                     // on their way while the angles are made
        raw = raw_of(first);
        weights = weights_of<D>(a, of_kind(kind_of(first), a.wq, a.wk, a.wk), lane);
    }
    const int64_t slot = load_uniform(a.slots + t);
    for (int i = threadIdx.x; i < TOKENS * a.half; i += 256) {
        const int at = min(t0 + (TOKENS == 1 ? 0 : i / a.half), a.T - 1), f = TOKENS == 1 ? i : i % a.half;
        const int axis = a.axes ? min(max(a.axes[f], 0), a.n_axes - 1) : 0;
        const double r = (double)a.positions[axis * a.pos_axis + at] * a.inv_freq[f] * 0.15915494309189535;     // turns
        const float share = (float)(r - rint(r));             // the hardware's sine and cosine: off by 2^-22 at most
        turn[TOKENS == 1 ? 0 : i / a.half][f] =
            make_float2(__builtin_amdgcn_cosf(share) * a.rot_scale, __builtin_amdgcn_sinf(share) * a.rot_scale);
    }
    const bool kept = slot >= 0 && slot < a.pages * a.page;
    int64_t page = 0, off = 0;
    if (kept) {
        if (slot >> 32 == 0) {
            page = (uint32_t)slot / (uint32_t)a.page;
            off = (uint32_t)slot % (uint32_t)a.page;
        } else {
            page = slot / a.page;
            off = slot % a.page;
        }
    }
    char *kc = a.kc + page * a.kc_page + off * a.kc_token, *vc = a.vc + page * a.vc_page + off * a.vc_token;
    __syncthreads();
    if (t0 + token >= a.T) return;
    uint16_t* out = a.out + t * a.o_row + d;
    Turn mine;
    int have = -1;                                            // the kind that `mine` is of
    for (int g = first; g < passes; g += step) {
        const int kind = kind_of(g), head = head_of(g, kind);
        const uint4 now = raw;
        if (g + step < passes) raw = raw_of(g + step);
        float x[8];
        const uint16_t* weight = of_kind(kind, a.wq, a.wk, a.wk);
        if (kind < 2) {
            if (kind != have) {
                if (have >= 0) weights = weights_of<D>(a, weight, lane);
                mine = turn_of<D, BF>(a, turn[token], weight, weights, lane);
                have = kind;
            }
            turned<D, BF>(a, mine, weight != nullptr, now, x);
        } else {
            unpack8(now, BF, x);
        }
        if (head >= of_kind(kind, a.Hq, a.Hkv, a.Hkv) || (kind && !kept)) continue;
        char* row = of_kind(kind, reinterpret_cast<char*>(out + (uint64_t)(uint32_t)head * a.o_head), kc + head * a.kc_head,
                            vc + head * a.vc_head);
        if (kind) row += d * (E8 ? 1 : 2);
        if (E8 && kind) {
            const float scale = of_kind(kind, a.ks, a.ks, a.vs)[head], over = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = quotient_of(x[j], scale, over);
            const int w = pack_e4m3<true>(x[2], x[3], pack_e4m3<false>(x[0], x[1], 0));
            *reinterpret_cast<int2*>(row) = make_int2(w, pack_e4m3<true>(x[6], x[7], pack_e4m3<false>(x[4], x[5], 0)));
        } else {                                              // (values as they came)
            *reinterpret_cast<uint4*>(row) =
                kind == 2 ? now : make_uint4(pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7]));
        }
    }
}

template <int D, bool BF, bool E8>
void append_launch(const AppendArgs& a, hipStream_t st) {
    constexpr int ROWS = 512 / D;
    const int passes = (a.Hq + ROWS - 1) / ROWS + 2 * ((a.Hkv + ROWS - 1) / ROWS);
    // From 256 tokens on four share a workgroup, whose angles a wave's worth of threads makes at once; as many shares of their rows
    // as fill the CUs, two passes at least. 8192 tokens of 32 + 2 x 4 heads of 128 (168 MB): 42 us, 4.0 TB/s (73 us a token a workgroup);
    // 1531: 15 us (21 us); 300: 6.5 us (5.5 us); one: 3.6 us by the kernel trace (3.4 at least), bound by its chain of loads
    if (a.T >= 256) {
        const int shares = std::max(1, std::min((passes + 1) / 2, 8192 / a.T));
        append_kernel<D, BF, E8, 4><<<dim3((unsigned)((a.T + 3) / 4), (unsigned)shares), 256, 0, st>>>(a);
    } else {
        append_kernel<D, BF, E8, 1><<<dim3((unsigned)a.T, (unsigned)((passes + 3) / 4)), 256, 0, st>>>(a);
    }
}
template <bool BF, bool E8>
void append_dim(const AppendArgs& a, int D, hipStream_t st) {
    D == 64 ? append_launch<64, BF, E8>(a, st) : D == 128 ? append_launch<128, BF, E8>(a, st) : append_launch<256, BF, E8>(a, st);
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

extern "C" int esp_cache_append(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                                const void* v, int64_t v_row, int64_t v_head, int64_t T, int64_t Hq, int dtype,
                                const esp_kv_cache* cache, const int64_t* slots, const int64_t* positions, int64_t pos_axis,
                                int64_t n_axes, const double* inv_freq, const int32_t* axes, int64_t half, int adjacent,
                                double rot_scale, const void* q_weight, const void* k_weight, double eps, void* out,
                                int64_t out_row, int64_t out_head, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16, "cache_append: dtype must be bf16 or fp16");
    const char* wrong = esp_host::kv_cache_error(cache, dtype);
    ESP_REQUIRE(!wrong, "cache_append: %s", wrong);
    const esp_kv_cache& c = *cache;
    ESP_REQUIRE(!esp_host::kv_overlaps(c.dim, c.pages, c.k_page, c.page, c.k_token, c.heads, c.k_head) &&
                    !esp_host::kv_overlaps(c.dim, c.pages, c.v_page, c.page, c.v_token, c.heads, c.v_head),
                "cache_append: elements of the cache overlap");
    ESP_REQUIRE(c.k_page != c.v_page || c.k_token != c.v_token || c.k_head != c.v_head ||
                    !esp_host::kv_share(((intptr_t)c.v - (intptr_t)c.k) / kv_bytes(c.dtype), c.dim, c.pages, c.k_page, c.page, c.k_token, c.heads, c.k_head),
                "cache_append: k and v of the cache overlap");
    ESP_REQUIRE(T >= 0 && T < (1 << 24), "cache_append: at most 2^24 - 1 rows");
    ESP_REQUIRE(Hq >= 0 && Hq <= 1024, "cache_append: at most 1024 query heads");
    ESP_REQUIRE(half >= 0 && half % 8 == 0 && 2 * half <= c.dim,
                "cache_append: half the rotated elements must be a multiple of 8, at most half a head's");
    ESP_REQUIRE(n_axes >= 1 && n_axes <= 16 && pos_axis >= 0, "cache_append: 1 to 16 axes");
    if (T == 0) return esp_host::ok();
    ESP_REQUIRE((Hq == 0 || (q && out)) && k && v && slots && (half == 0 || (positions && inv_freq)), "cache_append: null pointer");
    ESP_REQUIRE(n_axes == 1 || axes || half == 0, "cache_append: several axes need the axis of each frequency");
    ESP_REQUIRE(n_axes == 1 || pos_axis >= T, "cache_append: the axes' positions overlap");
    const int64_t strides[8] = {q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head};
    for (const int64_t s : strides)
        ESP_REQUIRE(s >= 0 && s < (int64_t(1) << 32) && s % 8 == 0, "cache_append: strides must be multiples of 8 elements, below 2^32");
    ESP_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)q_weight | (uintptr_t)k_weight) % 16 == 0,
                "cache_append: rows and weights must be 16-byte aligned");
    ESP_REQUIRE((Hq <= 1 || out_head >= c.dim) && (T == 1 || out_row >= (Hq - 1) * out_head + c.dim || Hq == 0),
                "cache_append: the output's rows overlap");
    // A wave has read its rows when it stores them: queries may be turned in place, and nothing else may be overwritten
    const auto wide = [&](int64_t heads, int64_t head) { return ((heads - 1) * head + c.dim) * 2; };
    if (Hq) {
        ESP_REQUIRE((out == q && (T == 1 || out_row == q_row) && (Hq == 1 || out_head == q_head)) ||
                        !esp_host::rows_meet(out, out_row * 2, wide(Hq, out_head), q, q_row * 2, wide(Hq, q_head), T),
                    "cache_append: the output overlaps q without being q");
        ESP_REQUIRE(!esp_host::rows_meet(out, out_row * 2, wide(Hq, out_head), k, k_row * 2, wide(c.heads, k_head), T) &&
                        !esp_host::rows_meet(out, out_row * 2, wide(Hq, out_head), v, v_row * 2, wide(c.heads, v_head), T),
                    "cache_append: the output overlaps k or v");
    }
    AppendArgs a;
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.q_row = q_row;
    a.q_head = (uint32_t)q_head;
    a.k_row = k_row;
    a.k_head = (uint32_t)k_head;
    a.v_row = v_row;
    a.v_head = (uint32_t)v_head;
    a.out = static_cast<uint16_t*>(out);
    a.o_row = out_row;
    a.o_head = (uint32_t)out_head;
    const int64_t size = kv_bytes(c.dtype);
    a.kc = static_cast<char*>(c.k);
    a.vc = static_cast<char*>(c.v);
    a.kc_page = c.k_page * size;
    a.kc_token = c.k_token * size;
    a.kc_head = c.k_head * size;
    a.vc_page = c.v_page * size;
    a.vc_token = c.v_token * size;
    a.vc_head = c.v_head * size;
    a.pages = c.pages;
    a.slots = slots;
    a.positions = positions;
    a.pos_axis = pos_axis;
    a.inv_freq = inv_freq;
    a.axes = axes;
    a.wq = static_cast<const uint16_t*>(q_weight);
    a.wk = static_cast<const uint16_t*>(k_weight);
    a.ks = c.k_scale;
    a.vs = c.v_scale;
    a.T = (int)T;
    a.Hq = (int)Hq;
    a.Hkv = (int)c.heads;
    a.n_axes = (int)n_axes;
    a.half = (int)half;
    a.page = (int)c.page;
    a.adjacent = adjacent;
    a.eps = (float)eps;
    a.rot_scale = (float)rot_scale;
    const hipStream_t st = (hipStream_t)stream;
    const bool bf = dtype == ESP_BF16, e8 = c.dtype == ESP_E4M3;
    if (bf) e8 ? append_dim<true, true>(a, (int)c.dim, st) : append_dim<true, false>(a, (int)c.dim, st);
    else e8 ? append_dim<false, true>(a, (int)c.dim, st) : append_dim<false, false>(a, (int)c.dim, st);
    return esp_host::launch_check("cache_append");
}
