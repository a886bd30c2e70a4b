/* Causal attention of packed prompts (q38hip_prompt_attention). */
#include <type_traits>

#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

/* First row of the sequence that owns `row`, or -1 where none does: the last
 * sequence that starts at or before it, so empty ones are passed over.  Always
 * in 0 .. row, whatever the words hold. */
__device__ __forceinline__ int sequence_start(const PromptAttention &a, uint32_t row)
{
    uint32_t low = 0, high = a.count + 1;       /* row_starts[low - 1] <= row < row_starts[high] */
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (a.row_starts[mid] <= (int)row) low = mid + 1;
        else high = mid;
    }
    if (low == 0 || low == a.count + 1) return -1;
    return min(max(a.row_starts[low - 1], 0), (int)row);
}

__device__ __forceinline__ float quad_sum_f32(float v)
{
    v += __int_as_float(dpp_move<0xB1>(0, __float_as_int(v)));
    return v + __int_as_float(dpp_move<0x4E>(0, __float_as_int(v)));
}
__device__ __forceinline__ float wave_sum_f32(float v)
{
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i);
    return v;
}

/* One row of one head by one wavefront, 64 keys at a time with a running maximum;
 * only keys and values that the row sees are read.  Four lanes form a score, each
 * from 16 of every 64 bytes of a key, so a load is 16 whole pieces of 64 bytes; then a
 * lane sums D / 64 neighbouring channels of the values. */
template <typename T, int D, bool kWhole>
__device__ __forceinline__ void attend_row(const PromptAttention &a, uint32_t row, uint32_t head, uint32_t lane)
{
    constexpr int E = 16 / (int)sizeof(T), C = D / (4 * E), kChannels = D / 64;
    const int start = sequence_start(a, row);
    if (start < 0) return;
    const auto sixteen = [=](const T *from) {
        if constexpr (kWhole) return *reinterpret_cast<const layer_u32x4 *>(from);
        T e[E];
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = from[i];
        return __builtin_bit_cast(layer_u32x4, e);
    };
    const uint32_t kv = head / (a.heads / a.kv_heads), part = lane % 4 * E, channel = lane * kChannels;
    const uint64_t query = (uint64_t)row * a.query_row + (uint64_t)head * a.query_head;
    const T *keys = static_cast<const T *>(a.key) + kv * D + part, *values = static_cast<const T *>(a.value) + kv * D + channel;
    float q[C][E], out[kChannels] = {}, top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const layer_u32x4 raw = sixteen(static_cast<const T *>(a.query) + query + part + c * 4 * E);
#pragma unroll
        for (int e = 0; e < E; ++e) q[c][e] = static_cast<float>(reinterpret_cast<const T *>(&raw)[e]) * a.scale;
    }
    for (uint32_t first = start; first <= row; first += 64) {
        float s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            s[u] = -INFINITY;
            if (first + u * 16 > row) continue;
            const uint32_t key = first + u * 16 + lane / 4;
            const T *from = keys + (uint64_t)min(key, row) * a.key_row;
            layer_u32x4 raw[C];
#pragma unroll
            for (int c = 0; c < C; ++c) raw[c] = sixteen(from + c * 4 * E);
            float dot[2] = {};
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    dot[c % 2] = fmaf(q[c][e], static_cast<float>(reinterpret_cast<const T *>(&raw[c])[e]), dot[c % 2]);
            const float score = quad_sum_f32(dot[0] + dot[1]);
            if (key <= row) s[u] = score;
        }
        const float higher = fmaxf(top, wave_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
        /* nothing but -infinity so far: differences would be NaN, weights are 0 */
        const float base = higher == -INFINITY ? 0.0f : higher, shrink = __builtin_amdgcn_exp2f(top - base);
        top = higher;
        total *= shrink;
#pragma unroll
        for (int u = 0; u < 4; ++u) total += s[u] = __builtin_amdgcn_exp2f(s[u] - base);
#pragma unroll
        for (int e = 0; e < kChannels; ++e) out[e] *= shrink;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (first + u * 16 > row) continue;
            /* behind the row itself its own value again, with the weight 0 */
            T v[16][kChannels];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const T *from = values + (uint64_t)min(first + u * 16 + j, row) * a.value_row;
                if constexpr (kWhole) {
                    struct Some { T e[kChannels]; } __attribute__((aligned(sizeof(T) * kChannels)));
                    const Some some = *reinterpret_cast<const Some *>(from);
#pragma unroll
                    for (int e = 0; e < kChannels; ++e) v[j][e] = some.e[e];
                } else {
#pragma unroll
                    for (int e = 0; e < kChannels; ++e) v[j][e] = from[e];
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float weight = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s[u]), j * 4));
#pragma unroll
                for (int e = 0; e < kChannels; ++e) out[e] = fmaf(weight, static_cast<float>(v[j][e]), out[e]);
            }
        }
    }
    /* the four lanes of a score each counted it */
    const float inverse = 4.0f / wave_sum_f32(total);
    T *to = static_cast<T *>(a.output) + (uint64_t)row * a.output_row + (uint64_t)head * D + channel;
#pragma unroll
    for (int e = 0; e < kChannels; ++e) {
        float v = out[e] * inverse;
        if (a.gate) {
            const float g = static_cast<float>(static_cast<const T *>(a.gate)[query + channel + e]);
            v *= __builtin_amdgcn_rcpf(1.0f + __expf(-g));
        }
        to[e] = static_cast<T>(v);
    }
}

/* a wavefront to a row and head */
template <typename T, int D, bool kWhole>
__global__ void __launch_bounds__(256) row_kernel(PromptAttention a)
{
    const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= a.rows * a.heads) return;
    attend_row<T, D, kWhole>(a, item / a.heads, item % a.heads, threadIdx.x & 63);
}

/* ---- tiles of the matrix unit ------------------------------------------------ */

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define Q38_LDS __attribute__((address_space(3)))

__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return (uint32_t)(uintptr_t)(Q38_LDS const void *)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at)
{
    return *(Q38_LDS const V *)(uintptr_t)at;
}
/* 16 bytes per lane from memory to LDS at `to` + 16 lane, without registers; the
 * compiler does not count it, so the kernel waits itself (tile_barrier) */
__device__ __forceinline__ void copy_to_lds(const void *from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
/* what this wavefront asked for is in LDS and what it read has returned; then so
 * for all of the workgroup */
__device__ __forceinline__ void tile_barrier()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* c + A B over 16 bytes of a row from each lane: A's rows and B's columns are
 * lane % 32, the inner index is the lane's half and the place in the 16 bytes, in both
 * alike.  Element r of c is row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32. */
template <typename T>
__device__ __forceinline__ f32x16 multiply(u32x4 rows, u32x4 columns, f32x16 c)
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, rows), y = __builtin_bit_cast(f32x4, columns);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, rows), __builtin_bit_cast(f16x8, columns), c, 0,
                                                      0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, rows), __builtin_bit_cast(bf16x8, columns), c,
                                                       0, 0, 0);
    }
}

/* the value of both halves of the wavefront, in both */
__device__ __forceinline__ float halves_max(float v)
{
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v)
{
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ int wave_min(int v)
{
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v = min(v, __shfl_xor(v, i));
    return v;
}

/* Sizes of a workgroup: kWaves wavefronts of 32 * kGroups columns, tiles of kKeys
 * keys.  A column is a row and one of the query heads that share a key/value head,
 * columns of a row next to each other, so all of a tile's columns read the same
 * keys and values. */
template <typename T, int D>
struct PromptTile {
    static constexpr int kGroups = 1;
    static constexpr int kWaves = 4;
    /* wavefronts of a SIMD, which share 512 registers a lane: two hide each other's
     * softmax, but the sums and queries of 256-wide heads alone take 192 */
    static constexpr int kPerUnit = D == 256 ? 1 : 2;
    static constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;
    static constexpr int kRowBytes = D * (int)sizeof(T);
    static constexpr int kHalf = kKeys * kRowBytes;          /* keys or values of a tile */
    static constexpr uint32_t kColumns = kWaves * 32 * kGroups;
};

/* Where 16-byte piece `piece` of row `row` lies in its row in LDS.  Keys are read
 * 16 bytes a lane, 16 rows together, so the turn is the row; 16-bit values are read
 * transposed, 64 bytes of four rows together, so the turn is the row modulo 4 in
 * units of 64 bytes.  Values of fp32 are read along their rows: no turn. */
template <int kRowBytes>
__device__ __forceinline__ uint32_t key_turn(uint32_t row)
{
    return kRowBytes >= 256 ? row & 15 : (row >> 1) & 7;
}
template <typename T, int kRowBytes>
__device__ __forceinline__ uint32_t value_turn(uint32_t row)
{
    if (sizeof(T) == 4) return 0;
    return kRowBytes >= 256 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

/* Causal attention of a tile of columns.
 *
 * S^T = K Q^T leaves each lane the scores of one column, and its result has, in
 * each half of the wavefront, the keys that the second product, O^T = V^T P^T, takes
 * from that half: the weights go from one product to the other in registers.  So
 * statistics and rescaling are per lane; one exchange between the halves joins a
 * maximum.  The maximum that weights are relative to is raised only where a score
 * exceeds it by more than 2^8: then the sums are rescaled. */
template <typename T, int D, bool kWhole>
__global__ void __launch_bounds__((PromptTile<T, D>::kWaves * 64), (PromptTile<T, D>::kPerUnit))
    prompt_kernel(PromptAttention a)
{
    using Tile = PromptTile<T, D>;
    constexpr int NQ = Tile::kGroups, kWaves = Tile::kWaves;
    constexpr int kRowBytes = Tile::kRowBytes, kKeys = Tile::kKeys, kHalf = Tile::kHalf;
    constexpr int kSteps = kRowBytes / 32;                   /* 16 bytes a lane each */
    __shared__ __align__(1024) uint8_t tiles[2][2][kHalf];
    __shared__ int ranges[kWaves][2];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t half = lane >> 5, low = lane & 31;
    const uint32_t group = a.heads / a.kv_heads, columns = a.rows * group;
    /* later tiles, which see more, first; workgroups of one key/value head eight apart
     * where they can be, on one die's cache */
    const uint32_t kv = blockIdx.x % a.kv_heads;
    const uint32_t first = (gridDim.x / a.kv_heads - 1 - blockIdx.x / a.kv_heads) * Tile::kColumns + wave * (32 * NQ);

    /* the columns' rows and where their sequences begin */
    uint32_t row[NQ], head[NQ];
    int start[NQ], owner[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const uint32_t column = min(first + q * 32 + low, columns - 1);
        row[q] = column / group;
        head[q] = kv * group + column - row[q] * group;
        start[q] = 0;
        owner[q] = -1;
    }
    const int row_first = (int)(min(first, columns - 1) / group), row_last = (int)(min(first + 32 * NQ - 1, columns - 1) / group);
    uint32_t at = 0;
    if (a.count > 64) {                                      /* the last sequence at or before the first row */
        uint32_t end = a.count + 1;
        while (at < end) {
            const uint32_t mid = (at + end) / 2;
            if (a.row_starts[mid] <= row_first) at = mid + 1;
            else end = mid;
        }
        at = at ? at - 1 : 0;
    }
    for (bool more = true; more && at <= a.count; at += 64) {
        const int begins = at + lane <= a.count ? a.row_starts[at + lane] : INT32_MAX;
        for (uint32_t i = 0; i < 64; ++i) {
            const int begin = __builtin_amdgcn_readlane(begins, i);
            if (begin > row_last) {
                more = false;
                break;
            }
#pragma unroll
            for (int q = 0; q < NQ; ++q)
                if (begin <= (int)row[q]) start[q] = begin, owner[q] = (int)(at + i);
        }
    }
    int lowest = INT32_MAX, highest = -1, latest = 0, earliest = INT32_MAX;
    bool owned[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        owned[q] = first + q * 32 + low < columns && owner[q] >= 0 && owner[q] < (int)a.count;
        start[q] = min(max(start[q], 0), (int)row[q]);
        if (owned[q]) {
            lowest = min(lowest, start[q]);
            latest = max(latest, start[q]);
            highest = max(highest, (int)row[q]);
            earliest = min(earliest, (int)row[q]);
        }
    }
    /* the wavefront's keys: some column sees lowest .. highest, all see latest .. earliest */
    lowest = __builtin_amdgcn_readfirstlane(wave_min(lowest));
    highest = -__builtin_amdgcn_readfirstlane(wave_min(-highest));
    latest = -__builtin_amdgcn_readfirstlane(wave_min(-latest));
    earliest = __builtin_amdgcn_readfirstlane(wave_min(earliest));
    if (lane == 0) ranges[wave][0] = lowest, ranges[wave][1] = highest;
    __syncthreads();
    int from = INT32_MAX, to = -1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) from = min(from, ranges[w][0]), to = max(to, ranges[w][1]);
    from = __builtin_amdgcn_readfirstlane(from);
    to = __builtin_amdgcn_readfirstlane(to);
    if (to < 0) return;

    /* queries, 16 bytes of each 32, in registers throughout; a negative scale turns their sign */
    u32x4 query[NQ][kSteps];
    uint64_t query_at[NQ];
    const float scale = fabsf(a.scale);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        query_at[q] = (uint64_t)row[q] * a.query_row + (uint64_t)head[q] * a.query_head;
        const T *p = static_cast<const T *>(a.query) + query_at[q];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            constexpr int E = 16 / (int)sizeof(T);
            if constexpr (kWhole) {
                query[q][u] = *reinterpret_cast<const u32x4 *>(p + (2 * u + half) * E);
            } else {
                T e[E];
#pragma unroll
                for (int i = 0; i < E; ++i) e[i] = p[(2 * u + half) * E + i];
                query[q][u] = __builtin_bit_cast(u32x4, e);
            }
            if (a.scale < 0) query[q][u] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
        }
    }

    const T *keys = static_cast<const T *>(a.key) + kv * D, *values = static_cast<const T *>(a.value) + kv * D;
    const uint32_t tiles_at = lds_address(tiles);
    /* the keys and values from `key` on into a buffer; behind the last that any column
     * sees, that one again (what lies behind the sequences may be anything) */
    const auto load = [&](int key, uint32_t buffer) {
        constexpr int kParts = kHalf / 1024;
        static_assert(kParts % kWaves == 0, "whole copies of each wavefront");
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const T *base = h ? values : keys;
            const uint64_t stride = h ? a.value_row : a.key_row;
#pragma unroll
            for (int i = 0; i < kParts / kWaves; ++i) {
                const uint32_t place = (i * kWaves + wave) * 1024 + lane * 16;
                const uint32_t r = place / kRowBytes, piece = place % kRowBytes / 16;
                const uint32_t turn = h ? value_turn<T, kRowBytes>(r) : key_turn<kRowBytes>(r);
                const T *p = base + (uint64_t)min(key + (int)r, to) * stride + (piece ^ turn) * (16 / sizeof(T));
                const uint32_t where = tiles_at + buffer * (2 * kHalf) + h * kHalf + (i * kWaves + wave) * 1024;
                if constexpr (kWhole) {
                    copy_to_lds(p, where);
                } else {
                    T e[16 / sizeof(T)];
#pragma unroll
                    for (int j = 0; j < 16 / (int)sizeof(T); ++j) e[j] = p[j];
                    *(Q38_LDS u32x4 *)(uintptr_t)(where + lane * 16) = __builtin_bit_cast(u32x4, e);
                }
            }
        }
    };

    f32x16 out[NQ][D / 32] = {};
    float top[NQ], total[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) top[q] = -INFINITY, total[q] = 0.0f;

    load(from, 0);
    uint32_t buffer = 0;
    for (int key = from; key <= to; key += kKeys, buffer ^= 1) {
        tile_barrier();
        if (key + kKeys <= to) load(key + kKeys, buffer ^ 1);
        if (key > highest || key + kKeys <= lowest) continue;
        const uint32_t key_at = tiles_at + buffer * (2 * kHalf), value_at = key_at + kHalf;
        f32x16 score[kKeys / 32][NQ] = {};
#pragma unroll
        for (int t = 0; t < kKeys / 32; ++t)
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
                const uint32_t r = t * 32 + low;
                const u32x4 k = lds_read<u32x4>(key_at + r * kRowBytes + ((2 * u + half) ^ key_turn<kRowBytes>(r)) * 16);
#pragma unroll
                for (int q = 0; q < NQ; ++q) score[t][q] = multiply<T>(k, query[q][u], score[t][q]);
            }
        if (key < latest || key + kKeys - 1 > earliest) {
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                const uint32_t span = row[q] - start[q], base = key + 4 * half - start[q];
#pragma unroll
                for (int t = 0; t < kKeys / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (base + (t * 32 + r / 4 * 8 + r % 4) > span) score[t][q][r] = -INFINITY;
            }
        }
        u32x4 weight[NQ][kKeys / 16];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            float most = score[0][q][0];
#pragma unroll
            for (int t = 0; t < kKeys / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, score[t][q][r]);
            most = halves_max(most) * scale;
            if (__any(most > top[q] + 8.0f)) {
                const float higher = fmaxf(top[q], most);
                const float shrink = __builtin_amdgcn_exp2f(top[q] - (higher == -INFINITY ? 0.0f : higher));
                top[q] = higher;
                total[q] *= shrink;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) out[q][d][r] *= shrink;
            }
            /* nothing but -infinity so far: differences would be NaN, weights are 0 */
            const float base = top[q] == -INFINITY ? 0.0f : top[q];
#pragma unroll
            for (int t = 0; t < kKeys / 32; ++t) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    score[t][q][r] = __builtin_amdgcn_exp2f(fmaf(score[t][q][r], scale, -base));
                    total[q] += score[t][q][r];
                }
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        T e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = static_cast<T>(score[t][q][s * 8 + j]);
                        weight[q][t * 2 + s] = __builtin_bit_cast(u32x4, e);
                    }
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            /* a transposed read: 16 lanes name four rows of 16 neighbours, four lanes a row,
             * and get a column of four each */
            const uint32_t i = lane & 15, d16 = lane >> 4 & 1;
#pragma unroll
            for (int s = 0; s < kKeys / 16; ++s)
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    s16x4 part[2];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t r = s * 16 + b * 8 + half * 4 + i / 4, piece = d * 4 + d16 * 2 + (i & 3) / 2;
                        const uint32_t place = r * kRowBytes + (piece ^ value_turn<T, kRowBytes>(r)) * 16 + (i & 1) * 8;
                        part[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Q38_LDS s16x4 *)(uintptr_t)(value_at + place));
                    }
                    const u32x4 v = __builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int q = 0; q < NQ; ++q) out[q][d] = multiply<T>(v, weight[q][s], out[q][d]);
                }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    const uint32_t place = (r / 4 * 8 + half * 4 + r % 4) * kRowBytes + (d * 32 + low) * 4;
                    const float v = lds_read<float>(value_at + place);
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        out[q][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, score[0][q][r], out[q][d], 0, 0, 0);
                }
        }
    }

    /* A weight of 0 times a value that is not finite is NaN, so such values of rows that a
     * column does not see have got into its sums.  Whatever came out not finite is done
     * again, row by row, from the rows that it sees. */
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const float inverse = 1.0f / halves_sum(total[q]);
        float nothing = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                out[q][d][r] *= inverse;
                nothing = fmaf(out[q][d][r], 0.0f, nothing);
            }
        const uint64_t found = __ballot(owned[q] && nothing != 0.0f);
        uint32_t again = (uint32_t)(found | found >> 32);
        if (owned[q] && !(again >> low & 1)) {
            T *to_row = static_cast<T *>(a.output) + (uint64_t)row[q] * a.output_row + (uint64_t)head[q] * D;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t channel = d * 32 + r * 8 + half * 4;
                    T e[4];
                    if (a.gate) {
                        const T *gate = static_cast<const T *>(a.gate) + query_at[q] + channel;
                        if constexpr (kWhole && sizeof(T) == 2) {
                            *reinterpret_cast<layer_u32x2 *>(e) = *reinterpret_cast<const layer_u32x2 *>(gate);
                        } else if constexpr (kWhole) {
                            *reinterpret_cast<u32x4 *>(e) = *reinterpret_cast<const u32x4 *>(gate);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) e[j] = gate[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v = out[q][d][r * 4 + j];
                        if (a.gate) v *= __builtin_amdgcn_rcpf(1.0f + __expf(-static_cast<float>(e[j])));
                        e[j] = static_cast<T>(v);
                    }
                    if constexpr (kWhole && sizeof(T) == 2) {
                        *reinterpret_cast<layer_u32x2 *>(to_row + channel) = *reinterpret_cast<const layer_u32x2 *>(e);
                    } else if constexpr (kWhole) {
                        *reinterpret_cast<u32x4 *>(to_row + channel) = *reinterpret_cast<const u32x4 *>(e);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) to_row[channel + j] = e[j];
                    }
                }
        }
        while (again) {
            const uint32_t column = first + q * 32 + __builtin_ctz(again);
            again &= again - 1;
            attend_row<T, D, kWhole>(a, column / group, kv * group + column % group, lane);
        }
    }
}

template <typename T, int D>
bool attention(const PromptAttention &a, hipStream_t stream)
{
    const auto whole = [](const void *p, uint64_t stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * sizeof(T) % 16 == 0;
    };
    const bool wide = whole(a.query, a.query_row) && whole(a.gate, a.query_head) && whole(a.key, a.key_row) &&
                      whole(a.value, a.value_row) && whole(a.output, a.output_row);
    /* Few rows have few keys.  A wavefront to a row and head, against tiles, in us: 24 heads of
     * 256, fp32, 37 rows 5.9 against 28, 128 rows 21 against 48, 500 rows 197 against 154; bf16
     * 64 rows 10.5 against 14.7, 128 rows 20.7 against 17.4; 32 heads of 128, bf16, 64 rows 7.1
     * against 8.5, 128 rows 13.8 against 9.8, fp32 128 rows 18.5 against 24, 200 rows 39
     * against 35. */
    if (a.rows <= (sizeof(T) == 4 ? 128 : 64))
        return launch_kernel(wide ? row_kernel<T, D, true> : row_kernel<T, D, false>, dim3(layer_up(a.rows * a.heads, 4)), dim3(256),
                             stream, a);
    const uint32_t columns = a.rows * (a.heads / a.kv_heads);
    const dim3 grid(layer_up(columns, PromptTile<T, D>::kColumns) * a.kv_heads);
    return launch_kernel(wide ? prompt_kernel<T, D, true> : prompt_kernel<T, D, false>, grid, dim3(PromptTile<T, D>::kWaves * 64), stream, a);
}

template <typename T>
bool attention(const PromptAttention &a, hipStream_t stream)
{
    return a.head_dim == 64 ? attention<T, 64>(a, stream) : a.head_dim == 128 ? attention<T, 128>(a, stream)
                                                                              : attention<T, 256>(a, stream);
}

}  // namespace

bool launch_prompt_attention(const PromptAttention &a, hipStream_t stream)
{
    return a.type == kLayerF32 ? attention<float>(a, stream) : a.type == kLayerF16 ? attention<_Float16>(a, stream)
                                                                                   : attention<__bf16>(a, stream);
}

}  // namespace q38
