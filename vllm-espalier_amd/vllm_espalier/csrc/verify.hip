// Verification of drafted tokens against the target's logits from given random numbers (speculative decoding), on gfx950.
//
// Request b has n drafts x_0 .. x_{n-1}; rows f .. f + n of the logits are the target's at those positions and one further.
// With p_j = softmax(row f + j / temperature) and q_j what the draft was drawn from (one-hot at x_j when no probabilities
// are given), draft j is accepted iff u_j * q_j(x_j) < p_j(x_j). At the first one that is not, the token is drawn from what
// p_j has over q_j, w = max(p_j - q_j, 0) (p_j itself where that is nothing); behind n accepted drafts it is drawn from p_n.
// Drawing is a race: argmax of w_v / e_v with e_v exponential random numbers, the lowest index among equal ones. A request
// whose temperature is below 1e-5 is greedy: a draft is accepted iff it is the row's argmax, which is also the token drawn.
//
// Two launches. The first reads every row once: a wave takes 1024 logits into registers and leaves their maximum and their sum of
// exponentials (a greedy request's: the place of the maximum too), so no workgroup waits for another and nothing is rescaled. The
// second runs over the one row of a request that is drawn from: each of its workgroups puts the request's rows together from the
// waves' pieces and decides the drafts for itself (a few hundred bytes out of the L2, a wave a row, while its random numbers are
// on the way), then races its share of the entries, 4096 at a time; the last of a request's to arrive writes the outcome.
#include "../../../include/espalier.h"
#include "common.hpp"
#include "logits.hpp"
#include "norm.hpp"

#include <algorithm>

namespace esp {

constexpr int PIECE_GROUPS = 2;                // groups of 8 logits a lane of a wave's piece, all in flight
// (2048 a wave: 7.0 us instead of 5.0 for the four rows of one request, 79 / 76 for 768)
constexpr int PIECE = 64 * 8 * PIECE_GROUPS;
constexpr int RACE_GROUPS = 2;                 // groups of 8 entries a thread of a race
constexpr int RACE = 256 * 8 * RACE_GROUPS;

// one wave's piece of one row: the largest logit and the sum of exp((l - m) / temperature), NaN where a logit is NaN or +inf
struct Piece {
    float m, s;
};

struct VerifyArgs {
    const void* logits;
    int64_t stride, R;
    int V, B, G, pieces, races, chunks;         // races: workgroups a request, that share its chunks of RACE entries
    const int32_t *first, *n_drafts, *drafts;
    const float *uniform, *race, *temperature, *probs;
    int64_t race_stride, probs_request, probs_row;
    int32_t *tokens, *counts;
    float* logprobs;
    unsigned long long* keys;                   // [B][races]
    float* winners;                             // [B][races]: the keys' logits
    Piece* part;                                // [B][G + 1][pieces]
    int* best;                                  // [B][G + 1][pieces]: the place of m (the first NaN, if any), greedy requests
    int* arrived;                               // [B][CNT_STRIDE], made zero by the first launch
};

// the drafts of request b, -1 where there is no such request (or its rows lie outside the logits)
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
    const int n = load_uniform(a.n_drafts + b);
    const int64_t f = load_uniform(a.first + b);
    return n >= 0 && n <= a.G && f >= 0 && f + n < a.R ? n : -1;
}
template <int DT>
__device__ __forceinline__ const void* logits_row(const VerifyArgs& a, int64_t row) {
    return static_cast<const char*>(a.logits) + row * a.stride * (DT == F32 ? 4 : 2);
}

// The statistics of the rows: a wave a piece, four to a workgroup. Bound by memory: 768 rows of 151936 fp32 logits (467 MB) 78 us, 6.0
// TB/s; four rows of one request, in bf16, 3.5 us
template <int DT>
__global__ __launch_bounds__(256) void verify_stats_kernel(const VerifyArgs a) {
    const int quads = (a.pieces + 3) / 4, at = blockIdx.x / quads, b = at / (a.G + 1), j = at % (a.G + 1);
    const int lane = threadIdx.x & 63;
    const int piece = (int)(blockIdx.x % quads) * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (j == 0 && piece == 0 && lane == 0) a.arrived[(size_t)b * CNT_STRIDE] = 0;
    if (j > drafts_of(a, b) || piece >= a.pieces) return;
    const void* row = logits_row<DT>(a, (int64_t)load_uniform(a.first + b) + j);
    const float temperature = load_uniform(a.temperature + b);
    const int i0 = piece * PIECE + lane * 8;
    float v[PIECE_GROUPS][8];
#pragma unroll
    for (int u = 0; u < PIECE_GROUPS; ++u) load_group<DT>(row, i0 + u * 512, a.V, -INFINITY, v[u]);
    float hi, lo;
    exponent_factor(inv_temperature(temperature), hi, lo);
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < PIECE_GROUPS; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, v[u][k]);
    m = wave_max_f32(m);                                    // NaN is passed over here and found in the sum
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < PIECE_GROUPS; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) s += exp_scaled(v[u][k] - base, hi, lo);
    s = wave_sum_f32(s);
    const size_t to = (size_t)at * a.pieces + piece;
    if (lane == 0) a.part[to] = {m, s};
    if (!is_greedy(temperature)) return;
    const bool nan = s != s;                                // a NaN or +inf; the first NaN, if there is one, is the largest
    int idx = 0x7FFFFFFF, nan_at = 0x7FFFFFFF;
#pragma unroll
    for (int u = PIECE_GROUPS - 1; u >= 0; --u)
#pragma unroll
        for (int k = 7; k >= 0; --k) {
            if (v[u][k] == m) idx = i0 + u * 512 + k;       // (a -inf past the row's end has the highest indices)
            if (nan && v[u][k] != v[u][k]) nan_at = i0 + u * 512 + k;
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        idx = min(idx, __shfl_xor(idx, d));
        nan_at = min(nan_at, __shfl_xor(nan_at, d));
    }
    if (lane == 0) {
        const bool has = nan_at != 0x7FFFFFFF;
        a.best[to] = has ? nan_at : idx;
        if (has) a.part[to].m = __builtin_nanf("");
    }
}

// What a workgroup knows of each of its request's rows
struct Row {
    double z;                                   // the sum of exponentials over m, no finite positive number: no distribution
    double arg;                                 // (the logit of the draft, or of a greedy row's argmax, - m) / temperature
    float m;
    int token;                                  // the draft, if it is accepted, else -1; the argmax of a greedy row
};

__device__ __forceinline__ bool distribution(double z) { return z > 0.0 && z < INFINITY; }

// Row j of request b from its pieces, by one wave; the decision about its draft (j < n)
template <int DT>
__device__ __forceinline__ Row verify_row(const VerifyArgs& a, int b, int j, int n, bool greedy, double inv_t, float hi, float lo) {
    const int lane = threadIdx.x & 63;
    const size_t at = (size_t)b * (a.G + 1) + j;
    const Piece* p = a.part + at * a.pieces;
    constexpr int HELD = 4;                                  // pieces a lane keeps (a vocabulary of 262144); more are read twice
    Piece held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) held[k] = lane + 64 * k < a.pieces ? p[lane + 64 * k] : Piece{-INFINITY, 0.f};
    const int x = j < n ? load_uniform(a.drafts + (size_t)b * a.G + j) : -1;
    const bool in = x >= 0 && x < a.V;
    const void* row = logits_row<DT>(a, (int64_t)load_uniform(a.first + b) + j);
    float lx = 0.f, u = 0.f, q = 1.f;
    if (in && !greedy) {
        lx = load_elem(row, DT, (size_t)x);
        u = load_uniform(a.uniform + (size_t)b * a.G + j);
        if (a.probs) q = load_uniform(a.probs + b * a.probs_request + j * a.probs_row + x);
    }
    Row r;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < HELD; ++k) m = fmaxf(m, held[k].m);
    for (int i = lane + 64 * HELD; i < a.pieces; i += 64) m = fmaxf(m, p[i].m);
    r.m = m = wave_max_f32(m);
    double z = 0.0;
    const auto add = [&](const Piece& v) __attribute__((always_inline)) {
        if (v.s != 0.f) z += (double)(v.s * exp_scaled(v.m - m, hi, lo));
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) add(held[k]);
    for (int i = lane + 64 * HELD; i < a.pieces; i += 64) add(p[i]);
    r.z = z = wave_sum_f64_dpp(z);
    if (greedy) {
        unsigned long long key = 0;
        for (int i = lane; i < a.pieces; i += 64) key = max(key, key32(p[i].m, a.best[at * a.pieces + i]));
        r.token = (int)~(uint32_t)wave_max_key(key);
        lx = load_elem(row, DT, (size_t)r.token);
    } else {
        r.token = -1;
    }
    r.arg = ((double)lx - (double)m) * inv_t;
    if (in && !greedy && distribution(z) && (double)u * (double)q < exp(r.arg) / z) r.token = x;
    return r;
}

// This thread's entries of the race from entry i0 on (RACE_GROUPS groups of 8, 2048 apart) into its best: the largest w / e with w
// above 0, w = p without draft probabilities q (0 at the draft itself), else p - q. In fp32 with the hardware's exponential and
// reciprocal, since only the keys' order is wanted: two that are nearer than about 2^-19 of p may change places
struct Best {
    float key, logit;
    int idx;
};
template <int DT>
__device__ __forceinline__ void race_best(const VerifyArgs& a, const void* row, const float* q, int draft, float m, float hi,
                                          float lo, float rz, int i0, const float (&ev)[RACE_GROUPS][8], Best& best) {
    float v[RACE_GROUPS][8], qv[RACE_GROUPS][8];
#pragma unroll
    for (int u = 0; u < RACE_GROUPS; ++u) {
        load_group<DT>(row, i0 + u * 2048, a.V, -INFINITY, v[u]);
        if (q) load_group<F32>(q, i0 + u * 2048, a.V, 0.f, qv[u]);
    }
#pragma unroll
    for (int u = 0; u < RACE_GROUPS; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + u * 2048 + k;
            float w = exp_scaled(v[u][k] - m, hi, lo) * rz;
            if (q) w -= qv[u][k];
            else if (i == draft) w = 0.f;
            const float key = w * __builtin_amdgcn_rcpf(ev[u][k]);
            if (w > 0.f && key > best.key) best = {key, v[u][k], i};     // in the order of the indices: the lowest of equal
        }                                                                // ones stays
}

// A request's outcome: tokens, counts and log-probabilities from its rows (rows below `taken` accepted, the token of row `taken`
// drawn, -1: none)
__device__ __forceinline__ void verify_write(const VerifyArgs& a, int b, const Row* rows, int taken, int drawn, double drawn_arg) {
    const size_t o = (size_t)b * (a.G + 1);
    for (int j = threadIdx.x; j <= a.G; j += 256) {
        const int token = j < taken ? rows[j].token : j == taken ? drawn : -1;
        const bool some = token >= 0 && distribution(rows[j].z);
        a.tokens[o + j] = token;
        a.logprobs[o + j] = some ? (float)((j < taken ? rows[j].arg : drawn_arg) - log(rows[j].z)) : 0.f;
    }
    if (threadIdx.x == 0) a.counts[b] = taken + (drawn >= 0);
}

// The largest key of the workgroup, and its logit
struct Winner {
    unsigned long long key[4];
    float logit;
};
__device__ __forceinline__ unsigned long long block_max_key(unsigned long long mine, float logit, Winner& sh) {
    const unsigned long long k = wave_max_key(mine);
    if ((threadIdx.x & 63) == 0) sh.key[threadIdx.x >> 6] = k;
    __syncthreads();
    const unsigned long long all = max(max(sh.key[0], sh.key[1]), max(sh.key[2], sh.key[3]));
    if (all && mine == all) sh.logit = logit;                // one thread: a key holds its index
    __syncthreads();
    return all;
}

// The drafts' decisions and a request's race: a.races workgroups a request, each of which takes every a.races-th chunk. For many
// requests bound by memory (128 of 151936: e, q and a row, of which the MALL may hold some, 233 MB in 44 us), for few by its chain:
// pieces, draft, row, hand-off, 7.9 us for one
template <int DT>
__global__ __launch_bounds__(256) void verify_race_kernel(const VerifyArgs a) {
    extern __shared__ Row rows[];                            // [G + 1]
    __shared__ Winner sh;
    __shared__ int last;
    const int b = blockIdx.x / a.races, at = blockIdx.x % a.races;
    const int n = drafts_of(a, b);
    const float temperature = load_uniform(a.temperature + b);
    const bool greedy = is_greedy(temperature);
    if ((n < 0 || greedy) && at != 0) return;
    if (n < 0) {
        verify_write(a, b, rows, 0, -1, 0.0);
        return;
    }
    const float* e = a.race + b * a.race_stride;
    const int i0 = (int)threadIdx.x * 8;
    float ev[RACE_GROUPS][8];
    const auto load_e = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < RACE_GROUPS; ++u) load_group<F32>(e, c * RACE + i0 + u * 2048, a.V, 1.f, ev[u]);
    };
    if (!greedy) load_e(at);
    const double inv_t = inv_temperature(temperature);
    float hi, lo;
    exponent_factor(inv_t, hi, lo);
    for (int j = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); j <= n; j += 4) {
        const Row r = verify_row<DT>(a, b, j, n, greedy, inv_t, hi, lo);
        if ((threadIdx.x & 63) == 0) rows[j] = r;
    }
    __syncthreads();
    const int32_t* drafts = a.drafts + (size_t)b * a.G;
    int taken = 0;
    while (taken < n && (greedy ? rows[taken].token == load_uniform(drafts + taken) : rows[taken].token >= 0)) ++taken;
    taken = __builtin_amdgcn_readfirstlane(taken);
    const Row r = rows[taken];
    if (greedy || !distribution(r.z)) {                      // nothing to race for
        if (at == 0) verify_write(a, b, rows, taken, greedy ? r.token : -1, r.arg);
        return;
    }
    const void* row = logits_row<DT>(a, (int64_t)load_uniform(a.first + b) + taken);
    const float* q = a.probs && taken < n ? a.probs + b * a.probs_request + taken * a.probs_row : nullptr;
    const int draft = taken < n ? load_uniform(drafts + taken) : -1;
    const float rz = (float)(1.0 / r.z);
    Best best = {-INFINITY, 0.f, -1};
    for (int c = at; c < a.chunks; c += a.races) {
        if (c != at) load_e(c);
        race_best<DT>(a, row, q, draft, r.m, hi, lo, rz, c * RACE + i0, ev, best);
    }
    unsigned long long key = block_max_key(best.idx < 0 ? 0ull : key32(best.key, best.idx), best.logit, sh);
    if (a.races > 1) {
        const size_t to = (size_t)b * a.races;
        if (threadIdx.x == 0) {
            store_dev(a.winners + to + at, sh.logit);
            store_dev(a.keys + to + at, key);
        }
        if (!arrive_last(a.arrived + (size_t)b * CNT_STRIDE, a.races, &last)) return;
        key = 0;
        float logit = 0.f;
        for (int i = threadIdx.x; i < a.races; i += 256) {
            const unsigned long long k = load_dev(a.keys + to + i);
            const float l = load_dev(a.winners + to + i);
            if (k > key) {
                key = k;
                logit = l;
            }
        }
        key = block_max_key(key, logit, sh);
    }
    if (!key && taken < n) {                                 // q covers p (or the draft was all of it): p itself, rarely
        for (int c = 0; c < a.chunks; ++c) {
            load_e(c);
            race_best<DT>(a, row, nullptr, -1, r.m, hi, lo, rz, c * RACE + i0, ev, best);
        }
        key = block_max_key(best.idx < 0 ? 0ull : key32(best.key, best.idx), best.logit, sh);
    }
    // no key: every random number of the row is unusable
    verify_write(a, b, rows, taken, key ? (int)~(uint32_t)key : -1, ((double)sh.logit - (double)r.m) * inv_t);
}

template <int DT>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
    verify_stats_kernel<DT><<<(unsigned)(a.B * (a.G + 1) * ((a.pieces + 3) / 4)), 256, 0, st>>>(a);
    verify_race_kernel<DT><<<(unsigned)(a.B * a.races), 256, (size_t)(a.G + 1) * sizeof(Row), st>>>(a);
    return esp_host::launch_check("verify");
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

// A request's race is shared by as many workgroups as it has chunks of entries, but 1280 over all requests (five a CU, what
// fits at once): each of them decides the drafts first, which takes longer than a chunk. The launch of 128 requests
// of 151936 fp32 logits, 5 drafts and draft probabilities: 51.5 us with 38 workgroups a request, 49.5 with 19, 48.5 with 10
constexpr int64_t VERIFY_RACES = 1280;

struct VerifySizes {
    int64_t pieces, chunks, races, winners, part, best, arrived, bytes;       // byte offsets behind the keys
    VerifySizes(int64_t B, int64_t G, int64_t V) {
        pieces = (V + PIECE - 1) / PIECE;
        chunks = (V + RACE - 1) / RACE;
        const int64_t loops = std::max<int64_t>(1, (B * chunks + VERIFY_RACES - 1) / VERIFY_RACES);
        races = (chunks + loops - 1) / loops;
        winners = B * races * 8;
        part = winners + (B * races * 4 + 7) / 8 * 8;
        best = part + B * (G + 1) * pieces * (int64_t)sizeof(Piece);
        arrived = best + B * (G + 1) * pieces * 4;
        bytes = arrived + B * CNT_STRIDE * 4;
    }
};

extern "C" int64_t esp_verify_scratch(int64_t B, int64_t G, int64_t V) {
    if (B <= 0 || G < 0 || V <= 0 || B > (1 << 20) || G > 1024 || V > (1 << 24)) return 0;
    return VerifySizes(B, G, V).bytes;
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
    const VerifySizes z(B, G, V);
    ESP_REQUIRE(B * (G + 1) * ((z.pieces + 3) / 4) < (1 << 24), "verify: at most 2^24 - 1 blocks of 4096 logits over all rows");
    ESP_REQUIRE((logits || R == 0) && first && n_drafts && race && temperature && tokens && counts && logprobs && scratch &&
                    (G == 0 || (drafts && uniform)), "verify: null pointer");
    ESP_REQUIRE((R <= 1 || stride >= V) && (B <= 1 || race_stride >= V), "verify: rows overlap");
    ESP_REQUIRE(probs_request >= 0 && probs_row >= 0, "verify: negative stride");
    ESP_REQUIRE((uintptr_t)logits % (dtype == ESP_F32 ? 4 : 2) == 0 && (uintptr_t)scratch % 16 == 0,
                "verify: logits must be aligned to an element, the scratch to 16 bytes");
    ESP_REQUIRE(scratch_bytes >= z.bytes, "verify: the scratch needs esp_verify_scratch bytes");
    VerifyArgs a;
    a.logits = logits;
    a.stride = stride;
    a.R = R;
    a.V = (int)V;
    a.B = (int)B;
    a.G = (int)G;
    a.pieces = (int)z.pieces;
    a.races = (int)z.races;
    a.chunks = (int)z.chunks;
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
    char* base = static_cast<char*>(scratch);
    a.keys = reinterpret_cast<unsigned long long*>(base);
    a.winners = reinterpret_cast<float*>(base + z.winners);
    a.part = reinterpret_cast<Piece*>(base + z.part);
    a.best = reinterpret_cast<int*>(base + z.best);
    a.arrived = reinterpret_cast<int*>(base + z.arrived);
    const hipStream_t st = (hipStream_t)stream;
    return dtype == ESP_F32 ? verify_launch<F32>(a, st) : dtype == ESP_BF16 ? verify_launch<BF16>(a, st)
                                                                            : verify_launch<F16>(a, st);
}
