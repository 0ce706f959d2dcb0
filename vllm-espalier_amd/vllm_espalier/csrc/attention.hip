// Attention of new tokens over a paged cache of keys and values, on gfx950: one token of a request, a token and its drafts, or a
// prompt, behind whatever the cache holds of the request already. Row i of a request's n new tokens stands at position
// p = length - n + i and sees the keys j with max(0, p - window + 1) <= j <= p (no window: all up to its own):
//   o = sum_j softmax_j(scale * q k_j) v_j,   zeros where a row sees nothing.
//
// A request's rows that share a head of the cache (its new tokens times the query heads of the group) are tiles of ROWS rows; the
// keys that a tile sees are cut into pieces, and a workgroup takes a piece of a tile: its four waves take 32 keys in turn, each with
// a running maximum and sum of its own, joined at the end. Tiles of one piece are written at once, the others' pieces go to scratch
// (fp32) and a second launch joins them, in their order. Requests of more than 32 rows are attention_prompt.hip's.
//
// All in registers: with S^T = K Q^T (keys are the rows of the product, queries its columns) a lane loads 8 consecutive elements of
// a key, 16 bytes, as the matrix instruction wants them, and is left with the scores of one query. For O^T = V^T P^T its scores are
// again what the instruction wants, if the 8 keys that it takes of 32 are the lane's own: 4 of the first 16 and 4 of the second,
// since the order of the summed index is free. V^T wants 8 keys of one element in a lane: the lane loads the same 16 bytes of 8
// keys (16 lanes: a whole row) and swaps pairs of halves, 32 v_perm for 8 x 8 elements; the element of operand e in lane l is
// 8 l + e, which is where the output puts it.
//
// Scores, statistics and sums are fp32; the weights are rounded to the rows' dtype for the second product (off by at most half a
// step of themselves, fp16 ones down to 2^-27 of the largest: reference() in attention.hpp; their sum is that of the unrounded ones),
// e4m3 keys and values are exact in either dtype.
//
// What bounds it is reading the cache, once for all rows of a tile (a large copy reaches 4.9 TB/s): bf16, 32 requests of one new
// token over up to 8171, heads 32/4 of 128 (273 MB), take 54 us (5.0 TB/s) and the join 4.9; one over 131072 (268 MB) 49 us
// (5.4 TB/s) and 5.4; 64 over 4000, 8 heads of 64 (524 MB), 88 us (5.9 TB/s). An e4m3 cache is bound by its widening, heads of 256
// with two tiles' outputs by one workgroup a CU: 40 requests of up to 4 new tokens over up to 6001, heads 16/2, e4m3 (128 MB), 37 us
// (3.5 TB/s). One token over 113 is bound by its chain of loads: length, table, keys, values, 6.2 us
// in a table of up to 128 tokens; a wider one could hold a second piece, and the join's launch, of nothing here, makes it 8.8.
#include "attention_few.hpp"

namespace esp {

constexpr int64_t JOIN_GRID = 2048;            // workgroups of a join: what fits at once

template <int D, bool BF, bool E8, int NT>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_kernel(const AttendArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[FEW_LDS<D, NT>];
    attend_few<D, BF, E8, NT>(a, (int)blockIdx.x, lds);
}

template <int D, bool BF, bool E8>
void attend_launch(const AttendArgs& a, const AttendSizes& z, hipStream_t st) {
    if (z.many) attend_prompt(a, z, D, BF, E8, st);
    if (!z.many || !FEW_TOO<D>) {
        if (z.tile_rows == 16) attend_kernel<D, BF, E8, 1><<<(unsigned)z.few, 256, 0, st>>>(a);
        else attend_kernel<D, BF, E8, 2><<<(unsigned)z.few, 256, 0, st>>>(a);
    }
    const int64_t rows = (int64_t)a.B * a.max_new * a.Hkv * a.group;
    if (!z.rows) return;
    // Few tiles have many pieces a row (64 of one request of 131072 keys: 4.8 us, 5.8 with 256 threads); others, and rows whose bits
    // are to be their own, go by one order (1024 rows of up to 11 pieces: 4.3 us, 6.8 with 512 threads)
    const unsigned grid = (unsigned)std::min<int64_t>(rows, JOIN_GRID);
    if (!a.split && a.B * a.Hkv <= LONG_TILES) join_kernel<D, BF, E8, 512, 8><<<grid, 512, 0, st>>>(a);
    else join_kernel<D, BF, E8, 256, 2><<<grid, 256, 0, st>>>(a);
}
template <int D>
void attend_types(const AttendArgs& a, const AttendSizes& z, bool bf, bool e8, hipStream_t st) {
    if (bf) e8 ? attend_launch<D, true, true>(a, z, st) : attend_launch<D, true, false>(a, z, st);
    else e8 ? attend_launch<D, false, true>(a, z, st) : attend_launch<D, false, false>(a, z, st);
}

}  // namespace esp

// ======================================================================================================================
// C ABI
// ======================================================================================================================
using namespace esp;

constexpr int64_t ATTEND_CAPACITY = int64_t(1) << 28;

extern "C" int64_t esp_paged_attention_scratch(int64_t B, int64_t T, int64_t max_new, int64_t Hq, const esp_kv_cache* cache,
                                               int64_t max_pages, int64_t split) {
    if (!cache || T <= 0 || T >= (1 << 24) || B <= 0 || B > (1 << 20) || max_new <= 0 || max_new >= (1 << 24) || cache->heads < 1 || Hq < cache->heads ||
        Hq % cache->heads || Hq > 65536 || cache->page < 1 || max_pages < 0 || max_pages * cache->page > ATTEND_CAPACITY ||
        split < 0 || split % PIECE)
        return 0;
    return AttendSizes(B, T, max_new, Hq / cache->heads, cache->heads, cache->dim, max_pages * cache->page, split).bytes;
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
    ESP_REQUIRE(first || max_new == 1, "paged_attention: requests of more than one new token need their first rows");
    ESP_REQUIRE(B == 1 || table_row >= max_pages, "paged_attention: the tables' rows overlap");
    const int64_t strides[4] = {q_row, q_head, out_row, out_head};
    for (const int64_t s : strides)
        ESP_REQUIRE(s >= 0 && s < (int64_t(1) << 32) && s % 8 == 0, "paged_attention: strides must be multiples of 8 elements, below 2^32");
    ESP_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) % 16 == 0, "paged_attention: rows and scratch must be 16-byte aligned");
    ESP_REQUIRE((Hq == 1 || out_head >= c.dim) && (T == 1 || out_row >= (Hq - 1) * out_head + c.dim),
                "paged_attention: the output's rows overlap");
    const int64_t group = Hq / c.heads;
    ESP_REQUIRE(max_new * group < (1 << 23), "paged_attention: at most 2^23 - 1 rows a request and head of the cache");
    // other workgroups still read the queries when one writes its rows
    ESP_REQUIRE(!esp_host::rows_meet(out, out_row * 2, ((Hq - 1) * out_head + c.dim) * 2, q, q_row * 2,
                                     ((Hq - 1) * q_head + c.dim) * 2, T), "paged_attention: the output overlaps q");
    const AttendSizes z(B, T, max_new, group, c.heads, c.dim, max_pages * c.page, split);
    ESP_REQUIRE(z.few < (1 << 24) && z.many < (1 << 24) && z.rows < (1 << 30) && T * Hq < (int64_t(1) << 31),
                "paged_attention: at most 2^24 - 1 pieces of tiles, 2^31 - 1 rows of heads");
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
    a.stats = reinterpret_cast<float2*>(base + z.stats);
    a.slots = z.slots;
    a.tile_rows = z.tile_rows;
    a.first_row = z.first_row;
    a.rows = z.rows;
    a.many = (int)z.many;
    a.B = (int)B;
    a.T = (int)T;
    a.Hkv = (int)c.heads;
    a.group = (int)group;
    a.max_new = (int)max_new;
    a.window = (int)window;
    a.split = split ? (int)split : z.rows ? 0 : PIECE;            // (tables of one piece: there is nothing to choose)
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
