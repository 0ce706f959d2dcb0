// Log-probabilities of given tokens, with their ranks, the rows' entropies and the likeliest alternatives, on gfx950. With
// p = softmax(row / T), c = log2(e) / T and x = c l of a logit l:
//   log2 p_t = x_t - log2 z,   -sum p log2 p = log2 z - (sum 2^x x) / z,   z = sum 2^x.
// Tokens are ordered by their logits, equal ones by their indices; a token's rank is its place in that order.
//
// Two launches. The first reads every row once: a wave takes 1024 logits into registers and leaves their maximum, their sums and
// how many of them come before the row's token, so no workgroup waits for another. Sums are over 2^(x - K) with K the whole number
// nearest to the piece's largest x, so that an exponent costs one multiply-add. That is with c rounded down to fp32, hi: what it leaves
// out, x - K times off = (c - hi) / hi below 2^-23 and K times the same, comes back in the second launch. A piece's base is K (1 + off)
// there, in fp64 (K off passes 1 where logits times c pass 2^23: no first order of it would do), and off times x - K, a small number for
// every logit that counts, is taken into the sums by its first order, which is off times the sum of 2^(x - K) (x - K), which is there.
//
// The second launch puts a row together, a workgroup a row, and finds the alternatives without another pass over it: the k first
// tokens lie in the k pieces whose largest logits are the first (each other piece has k elements before all of its own), so it reads
// these again and keeps the logits that are no smaller than the least of the k maxima, mostly little more than k. A row of fewer pieces
// gets that bar from the largest logits of its lanes, 16 logits each. Where equal logits make them too many, the first key of each
// lane is kept instead, of which the same holds once more, and sorted. Keys hold the index: they are all different, and a key's place
// is the number of larger ones.
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
    float m, s, w;                             // the largest logit (a NaN if there is one), sums of e = 2^(x - K) and of e (x - K)
    int above;                                 // logits before the row's token
};

// K of a piece, where c m is a number of moderate size; elsewhere (rows of a type's lowest values) the sums are over x - c m
__device__ __forceinline__ bool whole_base(float m, float c, float& base) {
    base = rintf(m * c);
    return fabsf(m * c) < 16777216.0f;
}

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

// The statistics of the rows: a wave PER pieces, all on their way at once, four to a workgroup
template <int DT, int PER>
__global__ __launch_bounds__(256) void logprobs_stats_kernel(const LogprobsArgs a) {
    const int groups = (a.pieces + 4 * PER - 1) / (4 * PER), r = blockIdx.x / groups, lane = threadIdx.x & 63;
    const int piece0 = ((int)(blockIdx.x % groups) * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))) * PER;
    if (piece0 >= a.pieces) return;
    const void* row = row_of<DT>(a, r);
    float all[PER][2][8];
    if ((piece0 + PER) * PIECE <= a.V) {                    // (whole pieces without a branch between their loads)
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) load_whole_group<DT>(row, (piece0 + j) * PIECE + lane * 8 + u * 512, all[j][u]);
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) load_group<DT>(row, (piece0 + j) * PIECE + lane * 8 + u * 512, a.V, -INFINITY, all[j][u]);
    }
    const int token = load_uniform(a.tokens + r);
    const bool given = token >= 0 && token < a.V;
    const float mine = load_elem(row, DT, (size_t)(given ? token : 0));
    float hi, lo;
    exponent_factor(inv_temperature_of(a, r), hi, lo);
    const auto one = [&](int piece, const float (&v)[2][8]) __attribute__((always_inline)) {
        const int i0 = piece * PIECE + lane * 8;
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int k = 0; k < 8; ++k) m = fmaxf(m, v[u][k]);
        m = wave_max_f32(m);                                    // NaN is passed over here and found in the sum
        float s = 0.f, w = 0.f, base;
        if (whole_base(m, hi, base)) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float x = __builtin_fmaf(v[u][k], hi, -base);
                    const float e = __builtin_amdgcn_exp2f(x);
                    s += e;
                    w = __builtin_fmaf(e, fmaxf(x, -1024.0f), w);      // a masked logit: 0 times a number
                }
        } else {
            base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float d = v[u][k] - base, e = exp_scaled(d, hi, lo);
                    s += e;
                    w = __builtin_fmaf(e, fmaxf(d * hi, -1024.0f), w);
                }
        }
        s = wave_sum_f32(s);
        w = wave_sum_f32(w);
        int above = 0;
        const int begin = piece * PIECE;
        if (token < begin) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) above += __popcll(__ballot(v[u][k] > mine));
        } else if (token >= begin + PIECE) {                    // (never of a piece that ends past the row)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k) above += __popcll(__ballot(v[u][k] >= mine));
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    above += __popcll(__ballot(v[u][k] > mine || (v[u][k] == mine && i0 + u * 512 + k < token)));
        }
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
                    above += __popcll(__ballot(i < a.V && key32(v[u][k], i) > key));
                }
            nan = __any(nan);
        }
        if (lane == 0) a.part[(size_t)r * a.pieces + piece] = {nan ? __builtin_nanf("") : m, s, w, given ? above : 0};
    };
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (piece0 + j < a.pieces) one(piece0 + j, all[j]);
}

// Keys in the LDS: of all pieces, of the lanes of `top` pieces or of the logits of `top` lanes, whole powers of two, and a zero; at
// least some hundred logits
__host__ __device__ inline int keys_room(int pieces, int top) {
    int n = 512;
    while (n < pieces || n < top * 64) n *= 2;
    return n;
}
// the logit of a key (zeros of both signs alike)
__device__ __forceinline__ float logit_of(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, o & 0x80000000u ? (o == 0xFFFFFFFFu ? 0x7FC00000u : o & 0x7FFFFFFFu) : ~o);
}

// How many of the n keys are larger; a zero follows the last
__device__ __forceinline__ int place_of(unsigned long long key, const unsigned long long* keys, int n) {
    const ulonglong2* two = reinterpret_cast<const ulonglong2*>(keys);
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < (n + 1) / 2; ++i) larger += (two[i].x > key) + (two[i].y > key);
    return larger;
}

// The k-th largest of values[0 .. n) (a multiple of 256), a byte at a time from the top: how many have each value of
// it, of those that agree above it. bins: 256 counts and two more
template <int THREADS>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* values, int n, int k, int* bins) {
    const int t = threadIdx.x, lane = t & 63;
    uint32_t found = 0;
#pragma unroll
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (t < 256) bins[t] = 0;
        __syncthreads();
        for (int i = t; i < n; i += THREADS)
            if (shift == 24 || (values[i] ^ found) >> (shift + 8) == 0) atomicAdd(&bins[values[i] >> shift & 255], 1);
        __syncthreads();
        if (t < 64) {                                       // lane l: bins 255 - 4 l down
            int c[4], upto = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) upto += c[j] = bins[255 - 4 * lane - j];
            const int mine = upto;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(upto, d);
                if (lane >= d) upto += o;
            }
            int before = upto - mine;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < k && before + c[j] >= k) {
                    bins[256] = 255 - 4 * lane - j;
                    bins[257] = k - before;
                }
                before += c[j];
            }
        }
        __syncthreads();
        found |= (uint32_t)bins[256] << shift;
        k = bins[257];
        __syncthreads();
    }
    return found;
}

// keys[0 .. n), n a power of two, from the largest down
template <int THREADS>
__device__ __forceinline__ void sort_keys(unsigned long long* keys, int n) {
    for (int size = 2; size <= n; size *= 2)
        for (int log = 30 - __clz(size); log >= 0; --log) {
            const int step = 1 << log;
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
                const int lo = (i >> log) * 2 * step + (i & (step - 1)), hi = lo + step;
                const unsigned long long x = keys[lo], y = keys[hi];
                if ((x < y) == ((lo & size) == 0)) {
                    keys[lo] = y;
                    keys[hi] = x;
                }
            }
        }
    __syncthreads();
}
__device__ __forceinline__ int power_of_two(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

struct LogprobsRow {
    double z, w;
    float m;
    int above;
};

// A row from its pieces, and its alternatives: the logits that these are chosen from are on their way, of AHEAD pieces a wave at once,
// while the row's sums are made
template <int DT, int AHEAD, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_row_kernel(const LogprobsArgs a) {
    constexpr int WAVES = THREADS / 64, HELD = THREADS == 256 ? PIECES_MAX / 256 : 1;       // (512: at most 256 pieces)
    extern __shared__ __attribute__((aligned(16))) unsigned long long keys[];        // keys_room and two more
    __shared__ int chosen[TOP_MAX];
    __shared__ uint32_t bar;
    __shared__ LogprobsRow part[WAVES];
    __shared__ int count, nan, bins[258];
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const LogitsPiece* p = a.part + (size_t)r * a.pieces;
    const void* row = row_of<DT>(a, r);
    // a thread's pieces t, t + 256, ..
    LogitsPiece held[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k)
        held[k] = t + THREADS * k < a.pieces ? p[t + THREADS * k] : LogitsPiece{-INFINITY, 0.f, 0.f, 0};
    const int token = load_uniform(a.tokens + r);
    const bool given = token >= 0 && token < a.V;
    const float mine = load_elem(row, DT, (size_t)(given ? token : 0));
    const int n_pieces = min(a.pieces, a.top);
    if (a.top) {                                            // the pieces that the alternatives lie in
#pragma unroll
        for (int k = 0; k < HELD; ++k)
            if (t + THREADS * k <= a.pieces) keys[t + THREADS * k] = t + THREADS * k < a.pieces ? key32(held[k].m, t + THREADS * k) : 0;
        if (t == 0) {
            keys[a.pieces] = 0;
            count = 0;
        }
        __syncthreads();
        for (int i = t; i < a.pieces; i += THREADS) {
            const unsigned long long key = keys[i];
            const int at = place_of(key, keys, a.pieces);
            if (at < n_pieces) chosen[at] = i;
            if (at == a.top - 1) bar = (uint32_t)(key >> 32);
            if (at == 0) nan = key >> 32 == 0xFFFFFFFFull;
        }
        __syncthreads();
    }
    float v[AHEAD][2][8];
    int first[AHEAD];
    const auto load_ahead = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (from + WAVES * j < n_pieces) {
                const int piece = __builtin_amdgcn_readfirstlane(chosen[from + WAVES * j]);
                first[j] = piece * PIECE + lane * 8;
                if ((piece + 1) * PIECE <= a.V) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) load_whole_group<DT>(row, first[j] + u * 512, v[j][u]);
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) load_group<DT>(row, first[j] + u * 512, a.V, 0.f, v[j][u]);
                }
            }
    };
    load_ahead(wave);
    if (n_pieces < a.top) {                                 // the bar from the lanes (those without a logit: 0)
        uint32_t* order = reinterpret_cast<uint32_t*>(keys);
        const int n = (n_pieces * 64 + 255) / 256 * 256;
        for (int i = n_pieces * 64 + t; i < n; i += THREADS) order[i] = 0;
        for (int from = wave; from < n_pieces; from += WAVES * AHEAD) {
            if (from != wave) load_ahead(from);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (from + WAVES * j < n_pieces) {
                    uint32_t most = 0;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (first[j] + u * 512 + k < a.V) most = max(most, (uint32_t)(key32(v[j][u][k], 0) >> 32));
                    order[(from + WAVES * j) * 64 + lane] = most;
                }
        }
        __syncthreads();
        const uint32_t b = kth_largest<THREADS>(order, n, min(a.top, n), bins);
        if (t == 0) bar = b;
        if (n_pieces > WAVES * AHEAD) load_ahead(wave);
        __syncthreads();
    }
    // the pieces' sums over 2^base, and those over the largest base
    const double inv_t = inv_temperature_of(a, r), c = inv_t * 1.4426950408889634;
    float hi, lo;
    exponent_factor(inv_t, hi, lo);
    const double off = (c - (double)hi) / (double)hi;
    double base[HELD], s[HELD], w[HELD];
    bool whole[HELD];
    float most = -INFINITY;
    int above = 0;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        float b;
        s[k] = held[k].s;
        w[k] = held[k].w;
        whole[k] = s[k] != 0.0 && whole_base(held[k].m, hi, b);
        base[k] = held[k].m == -INFINITY ? -INFINITY : (double)held[k].m * c;
        if (whole[k]) {
            base[k] = b;                                      // K; below, K (1 + off)
            s[k] += 0.6931471805599453 * off * w[k];
            w[k] += off * w[k];
        }
        most = fmaxf(most, held[k].m);
        above += held[k].above;
    }
    most = wave_max_f32(most);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) above += __shfl_xor(above, d);
    if (lane == 0) {
        part[wave].m = most;
        part[wave].above = above;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WAVES; ++k) most = fmaxf(most, part[k].m);
    float top_k;
    const bool top_whole = whole_base(most, hi, top_k);
    const double top = top_whole ? (double)top_k * (1.0 + off) : most == -INFINITY ? 0.0 : (double)most * c;
    double z = 0.0, sum_w = 0.0;
#pragma unroll
    for (int k = 0; k < HELD; ++k)
        if (s[k] != 0.0) {
            double d, e;
            if (whole[k] && top_whole) {                      // 2^(a whole number) times 2^(off times it), off times 150 at most where it counts
                const double between = base[k] - (double)top_k;
                d = between * (1.0 + off);
                e = __builtin_amdgcn_exp2f((float)between);
                e = e != 0.0 ? e * (1.0 + 0.6931471805599453 * off * between) : 0.0;
            } else {
                d = (whole[k] ? base[k] * (1.0 + off) : base[k]) - top;
                e = __builtin_amdgcn_exp2f((float)d);
            }
            z += s[k] * e;
            sum_w += e != 0.0 ? (w[k] + s[k] * d) * e : 0.0;
        }
    z = wave_sum_f64_dpp(z);
    sum_w = wave_sum_f64_dpp(sum_w);
    if (lane == 0) {
        part[wave].z = z;
        part[wave].w = sum_w;
    }
    // their logits from the bar on
    const uint32_t reach = bar;
    const float least = nan ? __builtin_nanf("") : logit_of((unsigned long long)reach << 32);      // (a NaN: all are looked at)
    const int room = keys_room(a.pieces, a.top);
    for (int from = wave; from < n_pieces; from += WAVES * AHEAD) {
        if (from != wave) load_ahead(from);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (from + WAVES * j < n_pieces)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (v[j][u][k] < least) continue;
                        const int i = first[j] + u * 512 + k;
                        const unsigned long long key = key32(v[j][u][k], i);
                        if (i < a.V && (uint32_t)(key >> 32) >= reach) {
                            const int at = atomicAdd(&count, 1);
                            if (at < room) keys[at] = key;
                        }
                    }
    }
    __syncthreads();
    z = part[0].z;
    sum_w = part[0].w;
    above = part[0].above;
#pragma unroll
    for (int k = 1; k < WAVES; ++k) {
        z += part[k].z;
        sum_w += part[k].w;
        above += part[k].above;
    }
    const bool some = z > 0.0 && z < INFINITY;
    // log2 z in two parts: a whole number, and that of a number in [1/2, 1)
    const double small = __builtin_amdgcn_frexp_mant(z);
    const double log_s = (double)__builtin_amdgcn_frexp_exp(z) + (double)__builtin_amdgcn_logf((float)small);
    const double less = some ? log_s : (double)__builtin_nanf("");       // (the largest logit's difference is exact, however large it is)
    const auto log_p = [&](float l) __attribute__((always_inline)) { return (float)(0.6931471805599453 * ((double)l * c - top - less)); };
    if (t == 0) {
        a.logprobs[r] = given ? log_p(mine) : 0.f;
        if (a.ranks) a.ranks[r] = given ? 1 + above : 0;
        if (a.entropies) a.entropies[r] = some ? (float)(0.6931471805599453 * (log_s - (double)((float)sum_w / (float)z))) : __builtin_nanf("");
    }
    if (!a.top) return;
    int n = count;
    if (n <= min(room, 1024)) {
        if (t == 0) keys[n] = 0;
        __syncthreads();
        for (int i = t; i < n; i += THREADS) {
            const unsigned long long key = keys[i];
            const int at = place_of(key, keys, n);
            if (at < a.top) {
                a.top_ids[(size_t)r * a.top + at] = (int)~(uint32_t)key;
                a.top_logprobs[(size_t)r * a.top + at] = log_p(logit_of(key));
            }
        }
        return;
    }
    // Too many: the first key of each lane of the pieces, sorted; then the logits of the first lanes, sorted
    __syncthreads();
    n = power_of_two(n_pieces * 64);
    for (int i = n_pieces * 64 + t; i < n; i += THREADS) keys[i] = 0;
    for (int from = wave; from < n_pieces; from += WAVES * AHEAD) {
        load_ahead(from);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (from + WAVES * j < n_pieces) {
                unsigned long long key = 0;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (first[j] + u * 512 + k < a.V) key = max(key, key32(v[j][u][k], first[j] + u * 512 + k));
                keys[(from + WAVES * j) * 64 + lane] = key;
            }
    }
    sort_keys<THREADS>(keys, n);
    if (t < a.top) {
        const int id = t < n && keys[t] ? (int)~(uint32_t)keys[t] : -1;
        chosen[t] = id < 0 ? -1 : id - id % 8 - (id % PIECE >= 512 ? 512 : 0);      // the first of the lane's logits
    }
    __syncthreads();
    n = power_of_two(a.top * 16);
    for (int i = t; i < n; i += THREADS) {
        const int begin = i < a.top * 16 ? chosen[i / 16] : -1, id = begin + (i % 16 >= 8 ? 512 : 0) + i % 8;
        keys[i] = begin >= 0 && id < a.V ? key32(load_elem(row, DT, (size_t)id), id) : 0;
    }
    sort_keys<THREADS>(keys, n);
    if (t < a.top) {
        a.top_ids[(size_t)r * a.top + t] = (int)~(uint32_t)keys[t];
        a.top_logprobs[(size_t)r * a.top + t] = log_p(logit_of(keys[t]));
    }
}

template <int DT>
int logprobs_launch(const LogprobsArgs& a, hipStream_t st) {
    // Two pieces a wave where there are waves enough (64 a CU): 2043 rows of 151935 bf16 logits (621 MB) 145 -> 124 us, 5.0 TB/s
    if ((int64_t)a.R * a.pieces < 32768) logprobs_stats_kernel<DT, 1><<<(unsigned)((int64_t)a.R * ((a.pieces + 3) / 4)), 256, 0, st>>>(a);
    else logprobs_stats_kernel<DT, 2><<<(unsigned)((int64_t)a.R * ((a.pieces + 7) / 8)), 256, 0, st>>>(a);
    const size_t lds = a.top ? (keys_room(a.pieces, a.top) + 2) * 8 : 0;
    // Twice the waves where rows are few and alternatives many (48 rows of 151936 with 20: 9.6 -> 8.0 us); a row's pieces are summed alike
    if (a.top <= 4) logprobs_row_kernel<DT, 1, 256><<<(unsigned)a.R, 256, lds, st>>>(a);
    else if (a.R <= 256 && a.pieces <= 256) logprobs_row_kernel<DT, 4, 512><<<(unsigned)a.R, 512, lds, st>>>(a);
    else logprobs_row_kernel<DT, 4, 256><<<(unsigned)a.R, 256, lds, st>>>(a);
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
