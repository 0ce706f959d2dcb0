// Verification of drafted tokens against the target's logits from given random numbers (speculative decoding), on gfx950.
//
// Request b has n drafts x_0 .. x_{n-1}; rows f .. f + n of the logits are the target's at those positions and one further.
// With p_j = softmax(row f + j / temperature) and q_j what the draft was drawn from (one-hot at x_j when no probabilities
// are given), draft j is accepted iff u_j * q_j(x_j) < p_j(x_j). At the first one that is not, the token is drawn from what
// p_j has over q_j, w = max(p_j - q_j, 0) (p_j itself where that is nothing); behind n accepted drafts it is drawn from p_n.
// Drawing is a race: argmax of w_v / e_v with e_v exponential random numbers, the lowest index among equal ones. A request
// whose temperature is below 1e-5 is greedy: a draft is accepted iff it is the row's argmax, which is also the token drawn.
//
// Bound by reading the logits: a row is split over many waves, each taking the maximum and the sum of exponentials of its
// piece from registers, so every logit is read once for the statistics of all rows; the second reading is one row a request.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "norm.hpp"

namespace esp {

constexpr float GREEDY_BELOW = 1e-5f;
constexpr int VERIFY_VECS = 2;                 // 16-byte loads of logits a lane, all in flight

// one wave's piece of one row: the largest logit (NaN if there is one), the sum of exp((l - m) / temperature), the index of m
struct Piece {
    float m, s;
    int idx, pad;
};

// what the race of a request needs, written by the decision
struct Drawn {
    int row;              // the logits row, -1: nothing to draw
    int j;                // the token's place
    int draft;            // the rejected draft, -1: none was (the row behind the last draft)
    float m, c_hi, c_lo, rz;
    double log_z;
};

struct VerifyArgs {
    const void* logits;
    int64_t stride, R;
    int V, B, G, pieces;
    const int32_t *first, *n_drafts, *drafts;
    const float *uniform, *race, *temperature, *probs;
    int64_t race_stride, probs_request, probs_row;
    int32_t *tokens, *counts;
    float* logprobs;
    Piece* part;                                // [B][G + 1][pieces]
    unsigned long long* keys;                   // [B][pieces][2]
    Drawn* drawn;                               // [B]
};

// unaligned 16-byte loads: rows start at any element (an odd vocabulary)
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Elems {
    static constexpr int VEC = DT == F32 ? 4 : 8;
    static __device__ __forceinline__ float at(const void* row, int i) { return load_elem(row, DT, (size_t)i); }
    // elements i .. i + VEC of a row of V, -inf past its end
    static __device__ __forceinline__ void load(const void* row, int i, int V, float (&v)[VEC]) {
        if (i + VEC <= V) {
            if constexpr (DT == F32) {
                const f32x4_a4 u = *reinterpret_cast<const f32x4_a4*>(static_cast<const float*>(row) + i);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
            } else {
                const u32x4_a2 u = *reinterpret_cast<const u32x4_a2*>(static_cast<const uint16_t*>(row) + i);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[2 * k] = from16((uint16_t)(w[k] & 0xFFFFu), DT == BF16);
                    v[2 * k + 1] = from16((uint16_t)(w[k] >> 16), DT == BF16);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = i + k < V ? at(row, i + k) : -INFINITY;
        }
    }
};

// f's order among all floats as an unsigned integer, zeros of both signs alike, NaN above everything
__device__ __forceinline__ uint32_t order32(float f) {
    if (f != f) return 0xFFFFFFFFu;
    const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key32(float f, int idx) {
    return ((unsigned long long)order32(f) << 32) | (uint32_t)~(uint32_t)idx;
}

__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)k, m), hi = (uint32_t)__shfl_xor((int)(k >> 32), m);
        const unsigned long long o = ((unsigned long long)hi << 32) | lo;
        k = o > k ? o : k;
    }
    return k;
}

// 1 / temperature (1 for a greedy request, whose log-probabilities are those of temperature 1). An infinite temperature
// keeps a factor above zero: a masked logit's -inf stays one.
__device__ __forceinline__ bool is_greedy(float temperature) { return !(temperature >= GREEDY_BELOW); }
__device__ __forceinline__ double inv_temperature(float temperature) {
    if (is_greedy(temperature)) return 1.0;
    const double inv = 1.0 / (double)temperature;
    return inv > 1e-30 ? inv : 1e-30;
}
// log2(e) / temperature as two floats: one float's rounding would shift every exponent of a row the same way. Both are
// positive (hi rounded down, lo above zero), so a masked logit's -inf stays -inf in either product.
__device__ __forceinline__ void exponent_factor(double inv_t, float& hi, float& lo) {
    const double c = inv_t * 1.4426950408889634;
    hi = (float)c;
    if ((double)hi > c) hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, hi) - 1u);
    lo = fmaxf((float)(c - (double)hi), 1e-37f);
}
__device__ __forceinline__ float exp_scaled(float d, float hi, float lo) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, hi, d * lo));
}

// the drafts of request b, -1 where there is no such request (or its rows lie outside the logits)
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
    const int n = a.n_drafts[b];
    const int64_t f = a.first[b];
    return n >= 0 && n <= a.G && f >= 0 && f + n < a.R ? n : -1;
}
__device__ __forceinline__ const void* logits_row(const VerifyArgs& a, int64_t row, int dt) {
    return static_cast<const char*>(a.logits) + row * a.stride * (dt == F32 ? 4 : 2);
}

// The statistics of one piece (64 * VERIFY_VECS vectors) of one row: a wave each, blockIdx.x a row of a request
template <int DT>
__global__ __launch_bounds__(256) void verify_stats_kernel(const VerifyArgs a) {
    constexpr int VEC = Elems<DT>::VEC;
    const int b = blockIdx.x / (a.G + 1), j = blockIdx.x % (a.G + 1);
    const int piece = blockIdx.y * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = drafts_of(a, b);
    if (j > n || piece >= a.pieces) return;
    const void* row = logits_row(a, (int64_t)a.first[b] + j, DT);
    float hi, lo;
    exponent_factor(inv_temperature(a.temperature[b]), hi, lo);
    const int i0 = (piece * VERIFY_VECS * 64 + lane) * VEC;
    float v[VERIFY_VECS][VEC];
#pragma unroll
    for (int u = 0; u < VERIFY_VECS; ++u) Elems<DT>::load(row, i0 + u * 64 * VEC, a.V, v[u]);
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < VERIFY_VECS; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) m = fmaxf(m, v[u][k]);
    m = wave_max_f32(m);                                    // NaN is passed over here and found in the sum
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < VERIFY_VECS; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += exp_scaled(v[u][k] - base, hi, lo);
    s = wave_sum_f32(s);
    const bool odd = s != s;                                // a NaN or +inf among the logits
    int idx = 0x7FFFFFFF;
    bool nan = false;
#pragma unroll
    for (int u = VERIFY_VECS - 1; u >= 0; --u)
#pragma unroll
        for (int k = VEC - 1; k >= 0; --k)
            if (v[u][k] == m) idx = i0 + u * 64 * VEC + k;  // (a -inf past the row's end has the highest indices)
    if (odd) {
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int u = VERIFY_VECS - 1; u >= 0; --u)
#pragma unroll
            for (int k = VEC - 1; k >= 0; --k)
                if (v[u][k] != v[u][k]) at = i0 + u * 64 * VEC + k;
        nan = __ballot(at != 0x7FFFFFFF) != 0;
        if (nan) idx = at;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_xor(idx, d);
        idx = o < idx ? o : idx;
    }
    if (lane == 0) a.part[(size_t)blockIdx.x * a.pieces + piece] = {nan ? __builtin_nanf("") : m, s, idx, 0};
}

// One workgroup a request: every row's statistics from its pieces (a wave a row), then the drafts in order
template <int DT>
__global__ __launch_bounds__(256) void verify_decide_kernel(const VerifyArgs a) {
    extern __shared__ double row_z[];                        // [G + 1] sums, then maxima and argmaxima
    float* row_m = reinterpret_cast<float*>(row_z + a.G + 1);
    int* row_best = reinterpret_cast<int*>(row_m + a.G + 1);
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    const int n = drafts_of(a, b);
    const double inv_t = inv_temperature(a.temperature[b]);
    for (int j = threadIdx.x >> 6; j <= n; j += 4) {
        const Piece* p = a.part + ((size_t)b * (a.G + 1) + j) * a.pieces;
        unsigned long long key = 0;
        float m = -INFINITY;
        for (int i = lane; i < a.pieces; i += 64) {
            const Piece q = p[i];
            const unsigned long long k = key32(q.m, q.idx);
            key = k > key ? k : key;
            m = fmaxf(m, q.m);
        }
        key = wave_max_key(key);
        m = wave_max_f32(m);
        double z = 0.0;
        for (int i = lane; i < a.pieces; i += 64) {
            const Piece q = p[i];
            if (q.s != 0.f) z += (double)q.s * exp(((double)q.m - (double)m) * inv_t);
        }
        z = wave_sum_f64_dpp(z);
        if (lane == 0) {
            row_z[j] = z;
            row_m[j] = m;
            row_best[j] = (int)~(uint32_t)key;
        }
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    const size_t o = (size_t)b * (a.G + 1);
    Drawn d = {-1, 0, -1, 0.f, 0.f, 0.f, 0.f, 0.0};
    int emitted = 0;
    if (n >= 0) {
        const bool greedy = is_greedy(a.temperature[b]);
        for (int j = 0; j <= n; ++j) {
            const void* row = logits_row(a, (int64_t)a.first[b] + j, DT);
            const double z = row_z[j], m = row_m[j];
            const bool some = z > 0.0 && z < INFINITY;       // false too for a NaN: no distribution
            const double log_z = some ? log(z) : 0.0;
            const int x = j < n ? a.drafts[(size_t)b * a.G + j] : -1;
            const bool in = x >= 0 && x < a.V;
            int token = -1;
            if (greedy) {
                token = row_best[j];
                if (j < n && x == token) {
                    a.tokens[o + j] = token;
                    a.logprobs[o + j] = some ? (float)((Elems<DT>::at(row, token) - m) * inv_t - log_z) : 0.f;
                    ++emitted;
                    continue;
                }
                a.tokens[o + j] = token;
                a.logprobs[o + j] = some ? (float)((Elems<DT>::at(row, token) - m) * inv_t - log_z) : 0.f;
                ++emitted;
                break;
            }
            if (in && some && j < n) {
                const double arg = (Elems<DT>::at(row, x) - m) * inv_t;
                const double q = a.probs ? (double)a.probs[b * a.probs_request + j * a.probs_row + x] : 1.0;
                if ((double)a.uniform[(size_t)b * a.G + j] * q < exp(arg) / z) {
                    a.tokens[o + j] = x;
                    a.logprobs[o + j] = (float)(arg - log_z);
                    ++emitted;
                    continue;
                }
            }
            if (some) {
                d.row = a.first[b] + j;
                d.j = j;
                d.draft = j < n ? x : -1;
                d.m = row_m[j];
                exponent_factor(inv_t, d.c_hi, d.c_lo);
                d.rz = (float)(1.0 / z);
                d.log_z = log_z;
                ++emitted;
            }
            break;
        }
    }
    a.drawn[b] = d;
    a.counts[b] = emitted;
    for (int j = emitted - (d.row >= 0); j <= a.G; ++j) {    // the race's token overwrites its place
        a.tokens[o + j] = -1;
        a.logprobs[o + j] = 0.f;
    }
}

// The race over one piece of request blockIdx.x's row: the largest key of w / e, and that of p / e
template <int DT>
__global__ __launch_bounds__(256) void verify_race_kernel(const VerifyArgs a) {
    constexpr int VEC = Elems<DT>::VEC;
    const int b = blockIdx.x, piece = blockIdx.y * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (piece >= a.pieces) return;
    const Drawn d = a.drawn[b];
    if (d.row < 0) return;
    const int n = drafts_of(a, b);
    const void* row = logits_row(a, d.row, DT);
    const float* e = a.race + b * a.race_stride;
    const float* q = a.probs && d.j < n ? a.probs + b * a.probs_request + d.j * a.probs_row : nullptr;
    const int i0 = (piece * VERIFY_VECS * 64 + lane) * VEC;
    unsigned long long best_w = 0, best_p = 0;
#pragma unroll
    for (int u = 0; u < VERIFY_VECS; ++u) {
        const int i = i0 + u * 64 * VEC;
        float v[VEC];
        Elems<DT>::load(row, i, a.V, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (i + k >= a.V) break;
            const float p = exp_scaled(v[k] - d.m, d.c_hi, d.c_lo) * d.rz;
            float w = p;
            if (q) w = p - q[i + k];
            else if (d.draft == i + k) w = 0.f;
            const float kp = p / e[i + k], kw = w / e[i + k];
            if (p > 0.f && kp == kp) best_p = max(best_p, key32(kp, i + k));
            if (w > 0.f && kw == kw) best_w = max(best_w, key32(kw, i + k));
        }
    }
    best_w = wave_max_key(best_w);
    best_p = wave_max_key(best_p);
    if (lane == 0) {
        unsigned long long* k = a.keys + ((size_t)b * a.pieces + piece) * 2;
        k[0] = best_w;
        k[1] = best_p;
    }
}

// The winner of every request's race: a wave a request
template <int DT>
__global__ __launch_bounds__(64) void verify_finish_kernel(const VerifyArgs a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const Drawn d = a.drawn[b];
    if (d.row < 0) return;
    unsigned long long w = 0, p = 0;
    for (int i = lane; i < a.pieces; i += 64) {
        const unsigned long long* k = a.keys + ((size_t)b * a.pieces + i) * 2;
        w = max(w, k[0]);
        p = max(p, k[1]);
    }
    w = wave_max_key(w);
    p = wave_max_key(p);
    if (lane != 0) return;
    const unsigned long long key = w ? w : p;
    const size_t o = (size_t)b * (a.G + 1) + d.j;
    if (!key) {                                              // every random number of the row is unusable
        a.counts[b] = d.j;
        return;
    }
    const int token = (int)~(uint32_t)key;
    const double inv_t = inv_temperature(a.temperature[b]);
    a.tokens[o] = token;
    a.logprobs[o] = (float)(((double)Elems<DT>::at(logits_row(a, d.row, DT), token) - (double)d.m) * inv_t - d.log_z);
}

template <int DT>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
    const unsigned blocks = (unsigned)((a.pieces + 3) / 4);
    verify_stats_kernel<DT><<<dim3((unsigned)(a.B * (a.G + 1)), blocks), 256, 0, st>>>(a);
    verify_decide_kernel<DT><<<(unsigned)a.B, 256, (size_t)(a.G + 1) * 16, st>>>(a);
    verify_race_kernel<DT><<<dim3((unsigned)a.B, blocks), 256, 0, st>>>(a);
    verify_finish_kernel<DT><<<(unsigned)a.B, 64, 0, st>>>(a);
    return esp_host::launch_check("verify");
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

static int64_t verify_pieces(int64_t V, int dtype) {
    const int64_t one = 64 * VERIFY_VECS * (dtype == ESP_F32 ? 4 : 8);
    return (V + one - 1) / one;
}

extern "C" int64_t esp_verify_scratch(int64_t B, int64_t G, int64_t V, int dtype) {
    if (B <= 0 || G < 0 || V <= 0 || B > (1 << 20) || G > 1024 || V > (1 << 24)) return 0;
    const int64_t np = verify_pieces(V, dtype);
    return B * (G + 1) * np * (int64_t)sizeof(Piece) + B * np * 16 + B * (int64_t)sizeof(Drawn);
}

extern "C" int esp_verify(const void* logits, int dtype, int64_t stride, int64_t R, int64_t V, const int32_t* first,
                          const int32_t* n_drafts, const int32_t* drafts, int64_t B, int64_t G, const float* uniform,
                          const float* race, int64_t race_stride, const float* temperature, const float* probs,
                          int64_t probs_request, int64_t probs_row, int32_t* tokens, int32_t* counts, float* logprobs,
                          void* scratch, int64_t scratch_bytes, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16 || dtype == ESP_F32, "verify: dtype must be bf16, fp16 or fp32");
    ESP_REQUIRE(B >= 0 && B <= (1 << 20) && G >= 0 && G <= 1024, "verify: at most 2^20 requests of at most 1024 drafts");
    ESP_REQUIRE(R >= 0 && R < (1ll << 31) && V > 0 && V <= (1 << 24), "verify: need R < 2^31 rows and 0 < V <= 2^24");
    if (B == 0) return esp_host::ok();
    ESP_REQUIRE(B * (G + 1) <= (1 << 23), "verify: at most 2^23 rows over all requests");
    ESP_REQUIRE((logits || R == 0) && first && n_drafts && race && temperature && tokens && counts && logprobs && scratch &&
                    (G == 0 || (drafts && uniform)), "verify: null pointer");
    ESP_REQUIRE((R <= 1 || stride >= V) && (B <= 1 || race_stride >= V), "verify: rows overlap");
    ESP_REQUIRE(probs_request >= 0 && probs_row >= 0, "verify: negative stride");
    ESP_REQUIRE((uintptr_t)logits % (dtype == ESP_F32 ? 4 : 2) == 0 && (uintptr_t)scratch % 16 == 0,
                "verify: logits must be aligned to an element, the scratch to 16 bytes");
    ESP_REQUIRE(scratch_bytes >= esp_verify_scratch(B, G, V, dtype), "verify: the scratch needs esp_verify_scratch bytes");
    VerifyArgs a;
    a.logits = logits;
    a.stride = stride;
    a.R = R;
    a.V = (int)V;
    a.B = (int)B;
    a.G = (int)G;
    a.pieces = (int)verify_pieces(V, dtype);
    a.first = first;
    a.n_drafts = n_drafts;
    a.drafts = drafts;
    a.uniform = uniform;
    a.race = race;
    a.temperature = temperature;
    a.probs = G ? probs : nullptr;
    a.race_stride = race_stride;
    a.probs_request = probs_request;
    a.probs_row = probs_row;
    a.tokens = tokens;
    a.counts = counts;
    a.logprobs = logprobs;
    a.part = static_cast<Piece*>(scratch);
    a.keys = reinterpret_cast<unsigned long long*>(a.part + B * (G + 1) * a.pieces);
    a.drawn = reinterpret_cast<Drawn*>(a.keys + B * a.pieces * 2);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == ESP_F32 ? verify_launch<F32>(a, st) : dtype == ESP_BF16 ? verify_launch<BF16>(a, st)
                                                                            : verify_launch<F16>(a, st);
}
