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
#include "kv.hpp"
#include "norm.hpp"

namespace esp {

struct AppendArgs {
    const uint16_t *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;      // elements
    uint16_t* out;
    int64_t o_row, o_head;
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

// Eight elements of a row into the cache, over the head's scale where it has one
template <bool BF, bool E8>
__device__ __forceinline__ void store_cache(char* row, int d, const float (&v)[8], const float* scale, int head) {
    if constexpr (E8) {
        const float s = scale[head];
        float u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = v[j] / s;
        int2 w = {0, 0};
        w.x = pack_e4m3<true>(u[2], u[3], pack_e4m3<false>(u[0], u[1], 0));
        w.y = pack_e4m3<true>(u[6], u[7], pack_e4m3<false>(u[4], u[5], 0));
        *reinterpret_cast<int2*>(row + d) = w;
    } else {
        *reinterpret_cast<uint4*>(row + 2 * d) = pack8_16(v, BF);
    }
}

// The rows of TOKENS tokens: a workgroup takes all rows of TOKENS tokens (a wave a token; TOKENS 4), or a share of one token's
// (TOKENS 1: gridDim.y of them)
template <int D, bool BF, bool E8, int TOKENS>
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs a) {
    constexpr int LANES = D / 8, ROWS = 64 / LANES;           // lanes a row, rows a wave
    __shared__ float2 turn[TOKENS][D / 2];                    // (cos, sin) of a token's angles
    const int t0 = blockIdx.x * TOKENS, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < TOKENS * a.half; i += 256) {
        const int t = min(t0 + i / a.half, a.T - 1), f = i % a.half;
        const int axis = a.axes ? min(max(a.axes[f], 0), a.n_axes - 1) : 0;
        const double r = (double)a.positions[axis * a.pos_axis + t] * a.inv_freq[f] * 0.15915494309189535;      // turns
        float s, c;
        sincospif(2.0f * (float)(r - rint(r)), &s, &c);
        turn[i / a.half][f] = make_float2(c * a.rot_scale, s * a.rot_scale);
    }
    __syncthreads();
    const int token = TOKENS == 1 ? 0 : wave, t = t0 + token;
    if (t >= a.T) return;
    const int heads = a.Hq + 2 * a.Hkv, d = lane % LANES * 8;
    const int64_t slot = a.slots[t];
    const bool kept = slot >= 0 && slot < a.pages * a.page;
    const int64_t page = kept ? slot / a.page : 0, off = kept ? slot % a.page : 0;
    const int first = TOKENS == 1 ? (int)(blockIdx.y * 4 + wave) : 0, step = TOKENS == 1 ? (int)gridDim.y * 4 : 1;
    for (int g = first; g * ROWS < heads; g += step) {
        const int row = g * ROWS + lane / LANES;              // queries, then keys, then values
        const int kind = row < a.Hq ? 0 : row < a.Hq + a.Hkv ? 1 : 2;
        const int head = kind == 0 ? row : kind == 1 ? row - a.Hq : row - a.Hq - a.Hkv;
        const bool here = row < heads;
        float x[8];
        if (here) {
            const uint16_t* p = kind == 0 ? a.q + t * a.q_row + head * a.q_head
                              : kind == 1 ? a.k + t * a.k_row + head * a.k_head : a.v + t * a.v_row + head * a.v_head;
            unpack8(*reinterpret_cast<const uint4*>(p + d), BF, x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
        }
        const uint16_t* w = kind == 0 ? a.wq : kind == 1 ? a.wk : nullptr;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
        ss = row_sum<LANES>(ss);
        if (w) {
            float wv[8];
            unpack8(*reinterpret_cast<const uint4*>(w + d), BF, wv);
            const float inv = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (x[j] * inv) * wv[j];
        }
        if (a.adjacent) {
            if (kind < 2 && d < 2 * a.half) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float2 cs = turn[token][d / 2 + j / 2];
                    const float p = x[j], o = x[j + 1];
                    x[j] = p * cs.x - o * cs.y;
                    x[j + 1] = o * cs.x + p * cs.y;
                }
            }
        } else {
            const bool low = d < a.half;
            const int from = (lane + (low ? a.half / 8 : -(a.half / 8))) * 4;
            const bool turns = kind < 2 && d < 2 * a.half;
            const int f = turns ? d % a.half : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float o = __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(from, __builtin_bit_cast(int, x[j])));
                if (turns) {
                    const float2 cs = turn[token][f + j];
                    x[j] = low ? x[j] * cs.x - o * cs.y : x[j] * cs.x + o * cs.y;
                }
            }
        }
        if (!here) continue;
        if (kind == 0) *reinterpret_cast<uint4*>(a.out + t * a.o_row + head * a.o_head + d) = pack8_16(x, BF);
        else if (kept && kind == 1) store_cache<BF, E8>(a.kc + page * a.kc_page + off * a.kc_token + head * a.kc_head, d, x, a.ks, head);
        else if (kept) store_cache<BF, E8>(a.vc + page * a.vc_page + off * a.vc_token + head * a.vc_head, d, x, a.vs, head);
    }
}

template <int D, bool BF, bool E8>
void append_launch(const AppendArgs& a, hipStream_t st) {
    constexpr int ROWS = 512 / D;
    const int heads = a.Hq + 2 * a.Hkv, passes = (heads + ROWS - 1) / ROWS;
    if (a.T >= 1024) append_kernel<D, BF, E8, 4><<<(unsigned)((a.T + 3) / 4), 256, 0, st>>>(a);
    else append_kernel<D, BF, E8, 1><<<dim3((unsigned)a.T, (unsigned)((passes + 3) / 4)), 256, 0, st>>>(a);
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
    a.q_head = q_head;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    a.out = static_cast<uint16_t*>(out);
    a.o_row = out_row;
    a.o_head = out_head;
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
