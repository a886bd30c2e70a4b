/* The paged 8-bit key/value cache (Q38KVPages, include/q38hip.h): index
 * arithmetic shared by its kernels and their launchers.  The index functions
 * are plain C++, so they are checked on the CPU too. */
#pragma once

#include <stdint.h>

#include "q38hip.h"

#if defined(__HIPCC__)
#define Q38_HD __host__ __device__ __forceinline__
#else
#define Q38_HD inline
#endif

namespace q38 {

/* GGML type ids of the element types of queries, keys, values and outputs */
constexpr int kElementF32 = 0, kElementF16 = 1, kElementBF16 = 30;

/* The rows of a call: sequence i of `count` owns rows row_starts[i] ..
 * row_starts[i + 1] - 1, or `rows_each` rows where row_starts is null. */
struct KVRows {
    const int32_t *sequences;
    const int32_t *row_starts;
    uint32_t count, total_rows, rows_each;
};

/* first row of sequence i (i <= count), never past total_rows */
Q38_HD uint32_t kv_row_start(const KVRows &rows, uint32_t i)
{
    if (!rows.row_starts) return i * rows.rows_each;
    const int32_t start = rows.row_starts[i];
    const uint32_t at = start < 0 ? 0u : (uint32_t)start;
    return at < rows.total_rows ? at : rows.total_rows;
}

/* Work slots of a ragged batch without a scan: sequence i starts at slot
 * floor(start * per_row / unit) + gap * i.  Floors differ by at least
 * ceil(rows * per_row / unit) - 1, so with gap 1 a sequence has a slot for
 * every `unit` of its rows * per_row items, with gap 2 one for every page its
 * rows touch; kv_slots(total) slots hold all of them. */
Q38_HD uint32_t kv_slot_base(uint32_t start, uint32_t i, uint32_t per_row, uint32_t unit, uint32_t gap)
{
    return (uint32_t)((uint64_t)start * per_row / unit) + gap * i;
}
Q38_HD uint64_t kv_slots(uint64_t total_rows, uint64_t count, uint64_t per_row, uint64_t unit, uint64_t gap)
{
    return total_rows * per_row / unit + gap * count;
}

/* a launch has fewer than 2^32 threads along each direction of its grid */
inline bool kv_launch_holds(uint64_t workgroups, uint32_t threads) { return workgroups * threads <= 0xffffffffull; }

/* of an append: threads of a workgroup (a page is T D / 4 quads, eight a thread; a
 * smaller page leaves threads of its one wavefront idle) */
inline uint32_t kv_append_threads(const Q38KVPages &cache)
{
    const uint32_t threads = cache.page_tokens * cache.head_dim / 32;
    return threads < 64 ? 64 : threads;
}

/* tokens of sequence `seq` that the table can hold; 0 for an id outside the cache */
Q38_HD uint32_t kv_tokens(const Q38KVPages &cache, int32_t seq)
{
    if (seq < 0 || (uint32_t)seq >= cache.sequences) return 0;
    const int32_t n = cache.lengths[seq];
    const uint32_t most = cache.table_entries * cache.page_tokens;
    return n <= 0 ? 0u : (uint32_t)n < most ? (uint32_t)n : most;
}

/* What slot `slot` holds of an append: with the rows begin .. end - 1 of a
 * sequence of `tokens` tokens, whose slots (of pages) begin at `base`, tokens
 * from .. to - 1 of its table entry `entry`; token t is row end - tokens +
 * entry * T + t.  Rows before the sequence's first token are left out.  Where
 * row offsets decrease, a sequence may be found for a slot before its own. */
struct KVPageRows {
    bool some;
    uint32_t entry, from, to;
};
Q38_HD KVPageRows kv_page_rows(uint32_t begin, uint32_t end, uint32_t tokens, uint32_t slot, uint32_t base,
                               uint32_t page_shift, uint32_t table_entries)
{
    if (end <= begin || !tokens || slot < base) return {false, 0, 0, 0};
    const uint32_t T = 1u << page_shift, rows = end - begin < tokens ? end - begin : tokens, first = tokens - rows;
    const uint32_t entry = (first >> page_shift) + (slot - base);
    if (entry >= table_entries || entry * T >= tokens) return {false, 0, 0, 0};
    const uint32_t at = entry * T;
    return {true, entry, (first > at ? first : at) - at, (tokens - at < T ? tokens - at : T)};
}

/* page of table entry `entry` of sequence `seq` (< sequences), or -1 where the
 * entry lies outside the table or names no page of the pool */
Q38_HD int32_t kv_page(const Q38KVPages &cache, uint32_t seq, uint32_t entry)
{
    if (entry >= cache.table_entries) return -1;
    const int32_t page = cache.tables[(uint64_t)seq * cache.table_entries + entry];
    return page >= 0 && (uint32_t)page < cache.pages ? page : -1;
}

/* bytes of one (layer, page), and where the keys (half 0) or values (half 1)
 * of a head begin in the layer's pages */
Q38_HD uint64_t kv_page_bytes(const Q38KVPages &cache)
{
    return 2ull * cache.kv_heads * cache.page_tokens * cache.head_dim;
}
Q38_HD uint64_t kv_block(const Q38KVPages &cache, int32_t page, uint32_t half, uint32_t head)
{
    return ((uint64_t)page * 2 + half) * cache.kv_heads + head;
}

/* least k >= kMinScaleExponent with |x| <= 127 * 2^k (int8) or 448 * 2^k
 * (e4m3) for every |x| up to the finite value with these bits */
constexpr int kMinScaleExponent = -100;
Q38_HD int kv_scale_exponent(uint32_t abs_bits, bool e4m3)
{
    /* 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8 */
    const int top = e4m3 ? 8 : 6;
    const uint32_t limit = e4m3 ? 0x600000u : 0x7E0000u;
    const int k = (int)(abs_bits >> 23) - 127 - top + ((abs_bits & 0x7FFFFFu) > limit ? 1 : 0);
    return k > kMinScaleExponent ? k : kMinScaleExponent;
}

struct KVAttention {
    Q38KVPages cache;      /* data and scales moved to the layer */
    KVRows rows;
    const void *query, *gate;
    void *output;
    float *partial;        /* the workspace (q38_kv_attention.h) */
    uint64_t query_row, query_head, output_row;
    uint32_t group, group_magic, page_shift;
    float workgroups_inverse;
    uint32_t columns;                      /* of a slot */
    uint32_t slots;                        /* at most that many */
    uint32_t workgroups, shift, least;     /* per key/value head; steps of a unit (log2); units of a workgroup at least */
    bool cut;                              /* slots may be, and what is cut is joined */
    int type;
    float scale;           /* softmax scale times log2(e) */
};
/* the split of a call: fills columns, slots, workgroups, shift and least;
 * returns the bytes of `partial` (0 where no slot is cut) */
uint64_t plan_kv_attention(KVAttention &call);

}  // namespace q38

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>

namespace q38 {

/* launchers (q38_kv_append.hip, q38_kv_attention*.hip, q38_kv_pages.hip); false when a launch failed */
bool launch_kv_append(const Q38KVPages &cache, uint32_t layer, const void *key, const void *value, int type,
                      uint64_t row_stride, const KVRows &rows, hipStream_t stream);

bool launch_kv_attention(const KVAttention &call, hipStream_t stream);

bool launch_kv_reset(const Q38KVPages &cache, hipStream_t stream);
uint64_t kv_workspace_bytes(const Q38KVPages &cache);
bool launch_kv_extend(const Q38KVPages &cache, const int32_t *sequences, const int32_t *rows, uint32_t count,
                      int32_t *workspace, hipStream_t stream);
bool launch_kv_fork(const Q38KVPages &cache, const int32_t *parents, const int32_t *children, const int32_t *lengths,
                    uint32_t count, hipStream_t stream);
bool launch_kv_truncate(const Q38KVPages &cache, const int32_t *sequences, const int32_t *lengths, uint32_t count,
                        hipStream_t stream);
bool launch_kv_compact(const Q38KVPages &cache, int32_t *workspace, hipStream_t stream);
bool launch_kv_copy(const Q38KVPages &cache, const int32_t *sources, const int32_t *targets, uint32_t count,
                    hipStream_t stream);

}  // namespace q38
#endif
