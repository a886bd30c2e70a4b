/* How a paged attention call is cut into work.  The host knows the sizes of
 * the call and of the cache, the device the lengths; the functions are plain
 * C++, so they are checked on the CPU too. */
#pragma once

#include "q38_kv.h"

namespace q38 {

constexpr int kKVStep = 64;               /* tokens of a step */
/* units of a slot beside those of its steps: queries, joining and output take
 * about as long as eight steps */
constexpr uint32_t kKVSlotOverhead = 8;

/* n / d of n d < 2^32, d < 2^16, from kv_magic(d) */
inline uint32_t kv_magic(uint32_t d) { return d == 1 ? 0 : (uint32_t)(0xffffffffu / d + 1); }
Q38_HD uint32_t kv_divide(uint32_t n, uint32_t magic)
{
    return magic ? (uint32_t)((uint64_t)n * magic >> 32) : n;
}

Q38_HD uint32_t kv_steps(uint32_t tokens) { return (tokens + kKVStep - 1) / kKVStep; }
/* units of a slot of a sequence with that many steps, 2^shift steps each */
Q38_HD uint32_t kv_slot_units(uint32_t steps, uint32_t shift)
{
    return ((steps + (1u << shift) - 1) >> shift) + kKVSlotOverhead;
}
/* units of a workgroup's range, ceil(units / workgroups) or `least`: units and
 * workgroups are below 2^31 and 2^16, the quotient by the inverse is one off at most */
Q38_HD uint32_t kv_chunk(uint32_t units, uint32_t workgroups, float workgroups_inverse, uint32_t least)
{
    if (units <= least * (uint64_t)workgroups) return least;
    uint32_t each = (uint32_t)((float)units * workgroups_inverse);
    while ((uint64_t)each * workgroups < units) each += each >> 22 ? each >> 22 : 1;
    return each;
}
Q38_HD uint32_t kv_small(uint32_t chunk)
{
    return chunk / 4 > kKVSlotOverhead + 4 ? chunk / 4 : kKVSlotOverhead + 4;
}

/* What a range of units begin .. end - 1 holds of the slot whose `each` units
 * (of `steps` steps) begin at `slot` < end: steps first .. last - 1.  A slot of
 * no steps is one piece without any. */
struct KVPiece {
    uint32_t first, last, units, each;        /* units that hold the slot's steps, and all of its units */
    bool some, first_piece, whole;
};
Q38_HD KVPiece kv_piece(uint32_t slot, uint32_t each, uint32_t steps, uint32_t begin, uint32_t end, uint32_t small,
                        uint32_t shift)
{
    uint32_t units = (steps + (1u << shift) - 1) >> shift;
    if (!units) units = 1;
    if (each <= small) return {0, steps, units, each, slot >= begin, true, true};
    const uint32_t low = begin > slot ? begin - slot : 0, high = end - slot < units ? end - slot : units;
    const uint64_t last = (uint64_t)high << shift;
    return {low << shift, last < steps ? (uint32_t)last : steps, units, each, low < high, low == 0, low == 0 && high == units};
}
/* pieces of a slot that is cut and ends (with all its units) before `behind` */
Q38_HD uint32_t kv_pieces(uint32_t units, uint32_t chunk, uint32_t behind, uint32_t each)
{
    const uint32_t slot = behind - each;
    return (slot + units - 1) / chunk - slot / chunk + 1;
}

/* Place of a workgroup's piece of a cut slot: its range begins in one such slot
 * at most and ends in one.  The p-th piece of a slot is kv_place_step(p) places
 * behind the first, as the ranges follow each other. */
Q38_HD uint32_t kv_place(uint32_t workgroup, bool first_piece) { return 2 * workgroup + (first_piece ? 1 : 0); }
Q38_HD uint32_t kv_place_step(uint32_t p) { return p ? 2 * p - 1 : 0; }

/* Column tiles (of 8 fp32 or 16 other columns): up to kv_token_tiles in a
 * workgroup whose wavefronts share the tokens (128-wide heads: a third tile's
 * registers would leave one wavefront to a SIMD), else one or kv_most_tiles in
 * each wavefront. */
constexpr int kv_token_tiles(int head_dim) { return head_dim == 128 ? 2 : 3; }
constexpr int kv_most_tiles(int head_dim) { return head_dim == 256 ? 1 : 2; }
/* Wavefronts of a workgroup.  One alone on a SIMD issues an instruction every
 * four cycles at most, so where the products are the bound two share it: 512
 * columns of 256-wide heads over 8191 tokens took 195 us with four wavefronts of
 * two tiles, 175 with eight of one. */
constexpr int kv_workgroup_waves(int head_dim, bool columns) { return columns && head_dim > 64 ? 8 : 4; }
/* Wavefronts that share a SIMD's registers: one has 512, of two each 256.  256-wide
 * heads over shared tokens fill the LDS with one workgroup. */
constexpr int kv_waves(int head_dim, bool columns) { return head_dim == 256 && !columns ? 1 : 2; }

struct KVShape {
    int tiles;
    bool columns;          /* tiles of each wavefront's own */
};
inline KVShape kv_shape(const KVAttention &a)
{
    const uint64_t tile = a.type == kElementF32 ? 8 : 16;
    /* columns of a sequence, on average over the call */
    const uint64_t columns = ((uint64_t)a.rows.total_rows * a.group + a.rows.count - 1) / a.rows.count;
    const uint64_t shared = (columns + tile - 1) / tile;
    if (shared <= (uint64_t)kv_token_tiles(a.cache.head_dim)) return {(int)shared, false};
    /* few columns: two tiles a wavefront would leave most wavefronts none (prompts of up to 300
     * rows at 16 heads of 64: 43 us with two, 36 with one) */
    return {columns <= 16 * tile ? 1 : kv_most_tiles(a.cache.head_dim), true};
}

}  // namespace q38
