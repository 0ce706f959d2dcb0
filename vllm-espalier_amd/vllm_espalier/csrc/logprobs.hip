// Log-probabilities of given tokens, with their ranks, the rows' entropies and the likeliest alternatives, on gfx950. With
// p = softmax(row / T), m the row's largest logit, d = l - m, z = sum exp(d / T):
//   log p_t = d_t / T - log z,   -sum p log p = log z - (sum exp(d / T) d / T) / z.
// Tokens are ordered by their logits, equal ones by their indices; a token's rank is its place in that order.
//
// Two launches. The first reads every row once: a wave takes 1024 logits into registers and leaves their maximum, their sums and
// how many of them come before the row's token, so no workgroup waits for another. The second puts a row together, a workgroup a
// row, and finds the alternatives without another pass over it: the k first tokens lie in the k pieces whose largest logits are
// the first (each other piece has k elements before all of its own), and in there in the k lanes of 16 logits for which the same
// holds. So it reads k pieces again, and keeps one key a lane. Keys hold the index: they are all different, and a key's place is
// the number of larger ones.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "logits.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

constexpr int TOP_MAX = 64;
constexpr int PIECE = 1024;                    // logits a wave takes: 16 a lane, 8 from 8 l and 8 from 512 + 8 l
constexpr int PIECES_MAX = 1024;

struct LogitsPiece {
    float m, s, w;                             // largest logit (a NaN if there is one), sum of e = exp((l - m) / T), sum of e (l - m)
    int above;                                 // logits before the row's token
};

struct LogprobsArgs {
    const void* logits;
    int64_t stride;
    int R, V, pieces, top;
    const int32_t* tokens;
    const float* temperature;
    float* logprobs;
    int32_t* ranks;
    float* entropies;
    int32_t* top_ids;
    float* top_logprobs;
    LogitsPiece* part;                         // [R][pieces]
};

template <int DT>
__device__ __forceinline__ const void* row_of(const LogprobsArgs& a, int64_t r) {
    return static_cast<const char*>(a.logits) + r * a.stride * (DT == F32 ? 4 : 2);
}
__device__ __forceinline__ double inv_temperature_of(const LogprobsArgs& a, int r) {
    return a.temperature ? inv_temperature(load_uniform(a.temperature + r)) : 1.0;
}

// The statistics of the rows: a wave a piece, four to a workgroup
template <int DT>
__global__ __launch_bounds__(256) void logprobs_stats_kernel(const LogprobsArgs a) {
    const int quads = (a.pieces + 3) / 4, r = blockIdx.x / quads, lane = threadIdx.x & 63;
    const int piece = (int)(blockIdx.x % quads) * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (piece >= a.pieces) return;
    const void* row = row_of<DT>(a, r);
    const int i0 = piece * PIECE + lane * 8;
    float v[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) load_group<DT>(row, i0 + u * 512, a.V, -INFINITY, v[u]);
    const int token = load_uniform(a.tokens + r);
    const bool given = token >= 0 && token < a.V;
    const float mine = load_elem(row, DT, (size_t)(given ? token : 0));
    float hi, lo;
    exponent_factor(inv_temperature_of(a, r), hi, lo);
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, v[u][k]);
    m = wave_max_f32(m);                                    // NaN is passed over here and found in the sum
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f, w = 0.f;
    int above = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float d = v[u][k] - base, e = exp_scaled(d, hi, lo);
            s += e;
            w += e * fmaxf(d, -3.0e38f);                    // a masked logit: 0 times a number
            above += v[u][k] > mine || (v[u][k] == mine && i0 + u * 512 + k < token);
        }
    s = wave_sum_f32(s);
    w = wave_sum_f32(w);
    bool nan = false;
    if (s != s || mine != mine) {                           // a NaN, or +inf: counted by their order
        above = 0;
        const unsigned long long key = key32(mine, token);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int i = i0 + u * 512 + k;
                nan |= v[u][k] != v[u][k];
                above += i < a.V && key32(v[u][k], i) > key;
            }
        nan = __any(nan);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) above += __shfl_xor(above, d);
    if (lane == 0) a.part[(size_t)r * a.pieces + piece] = {nan ? __builtin_nanf("") : m, s, w, given ? above : 0};
}

// How many of the n keys are larger
__device__ __forceinline__ int place_of(unsigned long long key, const unsigned long long* keys, int n) {
    int larger = 0;
    for (int i = 0; i < n; ++i) larger += keys[i] > key;
    return larger;
}

struct LogprobsRow {
    double z, w;                               // over the row's maximum
    float m;
    int above;
};

// A row from its pieces, and its alternatives
template <int DT>
__global__ __launch_bounds__(256) void logprobs_row_kernel(const LogprobsArgs a) {
    __shared__ unsigned long long keys[TOP_MAX * 64];       // of pieces, then of lanes, then of logits
    __shared__ int chosen[TOP_MAX];
    __shared__ unsigned long long least[4];
    __shared__ LogprobsRow part[4];
    __shared__ int count;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const LogitsPiece* p = a.part + (size_t)r * a.pieces;
    const void* row = row_of<DT>(a, r);
    const int token = load_uniform(a.tokens + r);
    const bool given = token >= 0 && token < a.V;
    const float mine = load_elem(row, DT, (size_t)(given ? token : 0));
    const double inv_t = inv_temperature_of(a, r);
    // a thread's pieces t, t + 256, ..: the maximum, then the sums over it
    LogitsPiece held[PIECES_MAX / 256];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PIECES_MAX / 256; ++k) {
        held[k] = t + 256 * k < a.pieces ? p[t + 256 * k] : LogitsPiece{-INFINITY, 0.f, 0.f, 0};
        m = fmaxf(m, held[k].m);
    }
    m = wave_max_f32(m);
    if (lane == 0) part[wave].m = m;
    if (t == 0) count = 0;
    __syncthreads();
    m = fmaxf(fmaxf(part[0].m, part[1].m), fmaxf(part[2].m, part[3].m));
    const double base = m == -INFINITY ? 0.0 : (double)m;
    double z = 0.0, w = 0.0, above = 0.0;
#pragma unroll
    for (int k = 0; k < PIECES_MAX / 256; ++k)
        if (held[k].s != 0.f) {
            const double d = (double)held[k].m - base, e = exp(d * inv_t);
            z += (double)held[k].s * e;
            w += ((double)held[k].w + (double)held[k].s * d) * e;
        }
#pragma unroll
    for (int k = 0; k < PIECES_MAX / 256; ++k) above += held[k].above;
    z = wave_sum_f64_dpp(z);
    w = wave_sum_f64_dpp(w);
    above = wave_sum_f64_dpp(above);
    if (lane == 0) {
        part[wave].z = z;
        part[wave].w = w;
        part[wave].above = (int)above;
    }
    if (a.top)
        for (int i = t; i < a.pieces; i += 256) keys[i] = key32(p[i].m, i);
    __syncthreads();
    z = ((part[0].z + part[1].z) + part[2].z) + part[3].z;
    w = ((part[0].w + part[1].w) + part[2].w) + part[3].w;
    const bool some = z > 0.0 && z < INFINITY;
    const double log_z = some ? log(z) : (double)__builtin_nanf("");
    if (t == 0) {
        a.logprobs[r] = given ? (float)(((double)mine - base) * inv_t - log_z) : 0.f;
        if (a.ranks) a.ranks[r] = given ? 1 + part[0].above + part[1].above + part[2].above + part[3].above : 0;
        if (a.entropies) a.entropies[r] = (float)(log_z - w * inv_t / z);
    }
    if (!a.top) return;
    // the pieces that the alternatives lie in
    const int n_pieces = min(a.pieces, a.top);
    for (int i = t; i < a.pieces; i += 256) {
        const int at = place_of(keys[i], keys, a.pieces);
        if (at < n_pieces) chosen[at] = i;
    }
    __syncthreads();
    // the first key of each of their lanes
    unsigned long long first = ~0ull;
    for (int c = wave; c < n_pieces; c += 4) {
        const int i0 = chosen[c] * PIECE + lane * 8;
        unsigned long long key = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float v[8];
            load_group<DT>(row, i0 + u * 512, a.V, 0.f, v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i0 + u * 512 + k < a.V) key = max(key, key32(v[k], i0 + u * 512 + k));
        }
        keys[c * 64 + lane] = key;
        first = min(first, wave_max_key(key));
    }
    if (lane == 0) least[wave] = first;
    __syncthreads();
    // (with fewer pieces than alternatives there is nothing that a key has to reach)
    unsigned long long bar = n_pieces < a.top ? 1 : min(min(least[0], least[1]), min(least[2], least[3]));
    unsigned long long mine_keys[TOP_MAX / 4];
#pragma unroll
    for (int k = 0; k < TOP_MAX / 4; ++k) mine_keys[k] = t + 256 * k < n_pieces * 64 ? keys[t + 256 * k] : 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TOP_MAX / 4; ++k)
        if (mine_keys[k] >= bar) keys[atomicAdd(&count, 1)] = mine_keys[k];
    __syncthreads();
    const int n_lanes = count;
    __syncthreads();
    if (t == 0) {
        count = 0;
        least[0] = 1;
    }
    __syncthreads();
    for (int i = t; i < n_lanes; i += 256) {
        const unsigned long long key = keys[i];
        const int at = place_of(key, keys, n_lanes);
        if (at < a.top) {
            const int id = (int)~(uint32_t)key;
            chosen[at] = id - id % 512 % 8 - (id % PIECE >= 512 ? 512 : 0);     // the first of the lane's logits
            if (at == a.top - 1) least[0] = key;
        }
    }
    __syncthreads();
    // their logits
    bar = least[0];
    const int n_chosen = min(n_lanes, a.top);
    for (int i = t; i < n_chosen * 16; i += 256) {
        const int id = chosen[i / 16] + (i % 16 >= 8 ? 512 : 0) + i % 8;
        const unsigned long long key = id < a.V ? key32(load_elem(row, DT, (size_t)id), id) : 0;
        if (key >= bar) keys[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    const int n = count;
    for (int i = t; i < n; i += 256) {
        const unsigned long long key = keys[i];
        const int at = place_of(key, keys, n);
        if (at < a.top) {
            const int id = (int)~(uint32_t)key;
            a.top_ids[(size_t)r * a.top + at] = id;
            a.top_logprobs[(size_t)r * a.top + at] = (float)(((double)load_elem(row, DT, (size_t)id) - base) * inv_t - log_z);
        }
    }
}

template <int DT>
int logprobs_launch(const LogprobsArgs& a, hipStream_t st) {
    logprobs_stats_kernel<DT><<<(unsigned)((int64_t)a.R * ((a.pieces + 3) / 4)), 256, 0, st>>>(a);
    logprobs_row_kernel<DT><<<(unsigned)a.R, 256, 0, st>>>(a);
    return esp_host::launch_check("token_logprobs");
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

extern "C" int64_t esp_token_logprobs_scratch(int64_t R, int64_t V, int64_t top) {
    if (R <= 0 || V <= 0 || R >= (int64_t(1) << 31) || V > (1 << 20) || top < 0) return 0;
    return R * ((V + PIECE - 1) / PIECE) * (int64_t)sizeof(LogitsPiece);
}

extern "C" int esp_token_logprobs(const void* logits, int dtype, int64_t stride, int64_t R, int64_t V, const int32_t* tokens,
                                  const float* temperature, int64_t top, float* logprobs, int32_t* ranks, float* entropies,
                                  int32_t* top_ids, float* top_logprobs, void* scratch, int64_t scratch_bytes, void* stream) {
    ESP_REQUIRE(dtype == ESP_BF16 || dtype == ESP_F16 || dtype == ESP_F32, "token_logprobs: dtype must be bf16, fp16 or fp32");
    ESP_REQUIRE(R >= 0 && R < (int64_t(1) << 31) && V > 0 && V <= (1 << 20), "token_logprobs: need R < 2^31 rows and 0 < V <= 2^20");
    ESP_REQUIRE(top >= 0 && top <= TOP_MAX && top <= V, "token_logprobs: at most %d alternatives, and no more than V", TOP_MAX);
    if (R == 0) return esp_host::ok();
    const int64_t pieces = (V + PIECE - 1) / PIECE;
    ESP_REQUIRE(R * ((pieces + 3) / 4) < (1 << 24), "token_logprobs: at most 2^24 - 1 blocks of 4096 logits over all rows");
    ESP_REQUIRE(logits && tokens && logprobs && scratch && (top == 0 || (top_ids && top_logprobs)), "token_logprobs: null pointer");
    ESP_REQUIRE(R == 1 || stride >= V, "token_logprobs: rows overlap");
    ESP_REQUIRE((uintptr_t)logits % (dtype == ESP_F32 ? 4 : 2) == 0 && (uintptr_t)scratch % 16 == 0,
                "token_logprobs: logits must be aligned to an element, the scratch to 16 bytes");
    ESP_REQUIRE(scratch_bytes >= esp_token_logprobs_scratch(R, V, top), "token_logprobs: the scratch needs esp_token_logprobs_scratch bytes");
    LogprobsArgs a;
    a.logits = logits;
    a.stride = stride;
    a.R = (int)R;
    a.V = (int)V;
    a.pieces = (int)pieces;
    a.top = (int)top;
    a.tokens = tokens;
    a.temperature = temperature;
    a.logprobs = logprobs;
    a.ranks = ranks;
    a.entropies = entropies;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.part = static_cast<LogitsPiece*>(scratch);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == ESP_F32 ? logprobs_launch<F32>(a, st) : dtype == ESP_BF16 ? logprobs_launch<BF16>(a, st)
                                                                             : logprobs_launch<F16>(a, st);
}
